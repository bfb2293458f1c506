"""Workloads of the wide layers: the norm, the product in 8 bits and the linear layer that keeps its input in 8 bits.

Four kinds of work ("op"):

* ``norm``   root-mean-square norm of ``x`` plus a residual: the output alone and the new residual (``infer``), or forward and
             backward (``train``);
* ``int8``   the product of 8-bit rows and 8-bit weights with a scale for each row of either;
* ``chain``  what serving runs of them: norm with the residual's addition and 8-bit rows out, then the product (``layers`` 1), or a whole
             block, in which the product's output goes through an activation, into 8-bit rows again and through a second product (2);
* ``keep``   a training step of a linear layer ``act(x) W^T + b`` whose input is kept as 8-bit rows for the backward.

8-bit rows: ``q = rint(v * (127 / a))`` and ``s = a / 127``, ``a`` the largest magnitude of the row ``v``.

``own`` false computes everything from elementary torch operations in float32, ``own`` true calls the package.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS = 1e-6


def _norm(name, rows, width, mode, dtype="bfloat16", residual=True, view=False):
    """``view``: the rows are columns of a wider buffer, as the pieces of one fused product's output are."""
    return {"name": name, "op": "norm", "rows": rows, "width": width, "mode": mode, "dtype": dtype, "residual": residual, "view": view}


def _int8(name, rows, k, n, dtype="bfloat16", bias=False, act="none"):
    return {"name": name, "op": "int8", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias, "act": act}


def _chain(name, rows, width, hidden, layers, dtype="bfloat16", act="gelu"):
    return {"name": name, "op": "chain", "rows": rows, "width": width, "hidden": hidden, "layers": layers, "dtype": dtype, "act": act}


def _keep(name, rows, k, n, dtype="bfloat16", act="gelu", bias=True, view=False):
    return {"name": name, "op": "keep", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "view": view}


def listed():
    return [
        # one token of a decoding step: latency
        _norm("norm infer 1 x 4096", 1, 4096, "infer"),
        # a training batch in its ordinary precision
        _norm("norm train 16384 x 4096", 16384, 4096, "train"),
        # a float32 network, an odd width and a ragged batch, no residual
        _norm("norm train f32 5003 x 777", 5003, 777, "train", dtype="float32", residual=False),
        # one token through the widest layer: the weights are read once, and that is the time
        _int8("int8 1 x 4096 x 16384", 1, 4096, 16384),
        # a handful of sequences decoded together, an odd number of them and of channels
        _int8("int8 19 x 5000 x 4098", 19, 5000, 4098, dtype="float16", bias=True),
        # a prompt of ordinary length
        _int8("int8 2048 x 4096 x 4096", 2048, 4096, 4096, bias=True, act="silu"),
        # the largest batch of prompts
        _int8("int8 16384 x 8192 x 8192", 16384, 8192, 8192),
        # a decoding step of eight sequences through a whole block
        _chain("block 8 x 2048 x 8192", 8, 2048, 8192, 2),
        # the entry of a block for a ragged batch of prompts
        _chain("norm and product 3001 x 2048 x 6144", 3001, 2048, 6144, 1, act="none"),
        # a small field's decoder beyond the width that is fused whole: many points, few channels
        _keep("keep 2^18 x 256 x 256", 2**18, 256, 256, act="relu"),
        # a training step of a wide network
        _keep("keep 16384 x 4096 x 4096", 16384, 4096, 4096),
        # odd sizes throughout, a ragged batch
        _keep("keep f16 1003 x 777 x 333", 1003, 777, 333, dtype="float16", act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, lo, hi):
    """Mostly multiples of 64 or 8, as layers are made; one in three any number."""
    v, unit = _log(rng, lo, hi), rng.choice((64, 8, 1))
    return max(lo, v // unit * unit)


def draw(rng):
    op = rng.choice(("norm", "int8", "int8", "chain", "keep", "keep"))
    half = rng.choice(("bfloat16", "bfloat16", "float16"))
    act = rng.choice(("none", "relu", "relu2", "silu", "gelu"))
    if op == "norm":
        case = _norm("", _log(rng, 1, 16384), _channels(rng, 16, 8192), rng.choice(("infer", "train", "train")),
                     dtype=rng.choice((half, half, "float32")), residual=rng.choice((True, False)), view=rng.choice((True, False)))
    elif op == "int8":
        case = _int8("", _log(rng, 1, 16384), _channels(rng, 16, 8192), _channels(rng, 16, 8192), dtype=rng.choice((half, half, "float32")),
                     bias=rng.choice((True, False)), act=act)
    elif op == "chain":
        layers = rng.choice((1, 2))
        case = _chain("", _log(rng, 1, 8192), _channels(rng, 64, 4096), _channels(rng, 64, 8192), layers, dtype=half, act="none" if layers == 1 else act)
    else:
        k, n = _channels(rng, 16, 4096), _channels(rng, 16, 4096)
        case = _keep("", min(_log(rng, 1, 2**18), max(1, 2**37 // (k * n))), k, n, dtype=half, act=act, bias=rng.choice((True, False)),
                     view=rng.choice((True, False)))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rows(gen, rows, width, dtype, view):
    """Rows of a hidden state: a few channels carry values far above the others', as trained networks' do."""
    wide = width + 64 if view else width
    x = _randn(gen, rows, wide) * torch.exp(0.5 * _randn(gen, wide))
    return x.to(dtype)[:, 32 : 32 + width] if view else x.to(dtype)


def _eight(v):
    """8-bit rows of ``v``: (q, s), in the type of ``v``."""
    a = v.abs().amax(-1, keepdim=True)
    return torch.round(v * (127.0 / a)), a / 127.0


def _weight8(gen, n, k):
    q, s = _eight(_randn(gen, n, k) * k**-0.5)
    return q.to(torch.int8), s.squeeze(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype, rows = case["op"], _DTYPES[case["dtype"]], case["rows"]
    s = {"case": case}
    if op == "norm":
        train = case["mode"] == "train"
        s["x"] = _rows(gen, rows, case["width"], dtype, case["view"]).requires_grad_(train)
        s["r"] = (3.0 * _randn(gen, rows, case["width"])).to(dtype).requires_grad_(train) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * _randn(gen, case["width"])).to(dtype).requires_grad_(train)
        if train:
            s["dy"] = _randn(gen, rows, case["width"]).to(dtype)
            s["ds"] = _randn(gen, rows, case["width"]).to(dtype) if case["residual"] else None
    elif op == "int8":
        q, scale = _eight(_rows(gen, rows, case["k"], torch.float32, False))
        s["q"], s["s"] = q.to(torch.int8), scale.squeeze(-1)
        s["w"], s["t"] = _weight8(gen, case["n"], case["k"])
        s["b"] = (0.1 * _randn(gen, case["n"])).to(dtype) if case["bias"] else None
    elif op == "chain":
        s["x"], s["r"] = _rows(gen, rows, case["width"], dtype, False), (3.0 * _randn(gen, rows, case["width"])).to(dtype)
        s["w"] = (1.0 + 0.2 * _randn(gen, case["width"])).to(dtype)
        s["w1"], s["t1"] = _weight8(gen, case["hidden"], case["width"])
        if case["layers"] == 2:
            s["w2"], s["t2"] = _weight8(gen, case["width"], case["hidden"])
    else:
        s["x"] = _rows(gen, rows, case["k"], dtype, case["view"]).requires_grad_()
        s["w"] = (_randn(gen, case["n"], case["k"]) * case["k"] ** -0.5).to(dtype).requires_grad_()
        s["b"] = (0.1 * _randn(gen, case["n"])).to(dtype).requires_grad_() if case["bias"] else None
        s["dy"] = _randn(gen, rows, case["n"]).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain form, 32 bits
def _act(z, act):
    if act == "relu":
        return torch.clamp_min(z, 0.0)
    if act == "relu2":
        return torch.clamp_min(z, 0.0) * z
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return z * (0.5 * torch.special.erfc(z * -(0.5**0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "relu2":
        return 2.0 * torch.clamp_min(z, 0.0)
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if act == "gelu":
        return 0.5 * torch.special.erfc(z * -(0.5**0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    return torch.ones_like(z)


def _normed(s):
    h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    return h, torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)


def _plain_norm(s, case):
    dtype, w = _DTYPES[case["dtype"]], s["w"].float()
    h, rstd = _normed(s)
    n = h * rstd
    out = {"y": (n * w).to(dtype)}
    if case["residual"]:
        out["stream"] = h.to(dtype)
    if case["mode"] == "train":
        dy = s["dy"].float()
        g = dy * w
        dh = rstd * (g - n * (g * n).mean(-1, keepdim=True))
        if case["residual"]:
            dh = dh + s["ds"].float()
            out["dr"] = dh.to(dtype)
        out["dx"] = dh.to(dtype)
        out["dw"] = (dy * n).sum(0).to(dtype)
    return out


def _product8(q, scale, w, t, b, act):
    y = (q.float() @ w.float().t()) * scale.unsqueeze(-1) * t
    return _act(y if b is None else y + b.float(), act)


def _plain_chain(s, case):
    dtype = _DTYPES[case["dtype"]]
    h, rstd = _normed(s)
    q, scale = _eight(h * rstd * s["w"].float())
    y = _product8(q, scale.squeeze(-1), s["w1"], s["t1"], None, case["act"]).to(dtype)
    if case["layers"] == 2:
        q, scale = _eight(y.float())
        y = _product8(q, scale.squeeze(-1), s["w2"], s["t2"], None, "none").to(dtype)
    return {"y": y, "stream": h.to(dtype)}


def _plain_keep(s, case):
    dtype, act = _DTYPES[case["dtype"]], case["act"]
    x, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
    y = _act(x, act) @ w.t()
    if s["b"] is not None:
        y = y + s["b"].float()
    q, scale = _eight(x)
    kept = q.to(torch.int8).float() * scale
    out = {"y": y.to(dtype), "dx": ((dy @ w) * _act_slope(kept, act)).to(dtype), "dw": (dy.t() @ _act(kept, act)).to(dtype)}
    if s["b"] is not None:
        out["db"] = dy.sum(0).to(dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------- the package's calls
def _own_norm(s, case):
    from triton_helpers_amd.layers.rms_norm import rms_norm

    x, r, w = s["x"], s["r"], s["w"]
    if case["mode"] == "infer":
        with torch.no_grad():
            y = rms_norm(x, w, _EPS, residual=r)
        return {"y": y} if r is None else {"y": y[0], "stream": y[1]}
    x.grad = w.grad = None
    if r is None:
        y = rms_norm(x, w, _EPS)
        y.backward(s["dy"])
        return {"y": y.detach(), "dx": x.grad, "dw": w.grad}
    r.grad = None
    y, stream = rms_norm(x, w, _EPS, residual=r)
    torch.autograd.backward((y, stream), (s["dy"], s["ds"]))
    return {"y": y.detach(), "stream": stream.detach(), "dr": r.grad, "dx": x.grad, "dw": w.grad}


def _own_int8(s, case):
    from triton_helpers_amd.layers.int8_linear import int8_linear

    return {"y": int8_linear(s["q"], s["s"], s["w"], s["t"], s["b"], activation=case["act"], dtype=_DTYPES[case["dtype"]])}


def _own_chain(s, case):
    from triton_helpers_amd.layers.int8_linear import int8_linear, quantize_rows
    from triton_helpers_amd.layers.rms_norm import rms_norm_int8

    dtype = _DTYPES[case["dtype"]]
    q, scale, stream = rms_norm_int8(s["x"], s["w"], _EPS, residual=s["r"])
    y = int8_linear(q, scale, s["w1"], s["t1"], activation=case["act"], dtype=dtype)
    if case["layers"] == 2:
        q, scale = quantize_rows(y)
        y = int8_linear(q, scale, s["w2"], s["t2"], dtype=dtype)
    return {"y": y, "stream": stream}


def _own_keep(s, case):
    from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear

    x, w, b = s["x"], s["w"], s["b"]
    x.grad = w.grad = None
    if b is not None:
        b.grad = None
    y = checkpointed_linear(x, w, b, activation=case["act"])
    y.backward(s["dy"])
    out = {"y": y.detach(), "dx": x.grad, "dw": w.grad}
    if b is not None:
        out["db"] = b.grad
    return out


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return {"norm": _own_norm, "int8": _own_int8, "chain": _own_chain, "keep": _own_keep}[op](state, case)
    with torch.no_grad():
        if op == "norm":
            return _plain_norm(state, case)
        if op == "int8":
            return {"y": _product8(state["q"], state["s"], state["w"], state["t"], state["b"], case["act"]).to(_DTYPES[case["dtype"]])}
        return (_plain_chain if op == "chain" else _plain_keep)(state, case)


# ---------------------------------------------------------------------------------------------------------------- the definition, 64 bits
def _d(t):
    return None if t is None else t.detach().double()


def _exact_act(z, act):
    """(act(z), act'(z))."""
    one = torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, 0 * one), torch.where(z > 0, one, 0 * one)
    if act == "relu2":
        return torch.where(z > 0, z**2, 0 * one), torch.where(z > 0, 2 * z, 0 * one)
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        phi = (1 + torch.erf(z / math.sqrt(2))) / 2
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, one


def _exact_eight(v):
    """What the 8-bit rows of v stand for."""
    step = v.abs().max(dim=-1, keepdim=True).values / 127
    return torch.round(v / step) * step


def _exact_norm(x, r, w):
    h = x if r is None else x + r
    n = h / torch.sqrt(torch.einsum("mk,mk->m", h, h).div(h.shape[1]).add(_EPS)).unsqueeze(1)
    return h, n, n * w


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "norm":
            x, r, w = _d(s["x"]), _d(s["r"]), _d(s["w"])
            h, n, y = _exact_norm(x, r, w)
            out = {"y": y}
            if r is not None:
                out["stream"] = h
            if case["mode"] == "train":
                dy = _d(s["dy"])
                g = dy * w
                root = torch.sqrt(h.pow(2).sum(1, keepdim=True) / h.shape[1] + _EPS)
                # y = h / root(h): the projection of g off n, over the root
                dh = (g - n * ((g * n).sum(1, keepdim=True) / h.shape[1])) / root
                if r is not None:
                    dh = dh + _d(s["ds"])
                    out["dr"] = dh
                out["dx"] = dh
                out["dw"] = torch.einsum("mk,mk->k", dy, n)
            return out
        if op == "int8":
            y = torch.mm(_d(s["q"]) * _d(s["s"])[:, None], (_d(s["w"]) * _d(s["t"])[:, None]).t())
            if s["b"] is not None:
                y = y + _d(s["b"])
            return {"y": _exact_act(y, case["act"])[0]}
        if op == "chain":
            h, _, v = _exact_norm(_d(s["x"]), _d(s["r"]), _d(s["w"]))
            y = _exact_act(_exact_eight(v) @ (_d(s["w1"]) * _d(s["t1"])[:, None]).t(), case["act"])[0]
            if case["layers"] == 2:
                # the activation is handed on in the layers' type, a part of the definition
                y = _exact_eight(y.to(_DTYPES[case["dtype"]]).double()) @ (_d(s["w2"]) * _d(s["t2"])[:, None]).t()
            return {"y": y, "stream": h}
        x, w, dy = _d(s["x"]), _d(s["w"]), _d(s["dy"])
        y = torch.mm(_exact_act(x, case["act"])[0], w.t())
        kept, slope = _exact_act(_exact_eight(x), case["act"])
        out = {"y": y if s["b"] is None else y + _d(s["b"]), "dx": torch.mm(dy, w) * slope, "dw": torch.mm(dy.t(), kept)}
        if s["b"] is not None:
            out["db"] = dy.sum(0)
        return out


# ---------------------------------------------------------------------------------------------------------------- what it takes
def work(case):
    op, rows = case["op"], case["rows"]
    size = 4 if case["dtype"] == "float32" else 2
    if op == "norm":
        values, two = rows * case["width"], 2 if case["residual"] else 1
        if case["mode"] == "infer":
            return {"bytes": 2 * two * values * size + case["width"] * size, "flops": 5 * values}
        # forward: the inputs in, the outputs out; backward: the upstream gradients in, the gradients out (x and the residual share one)
        return {"bytes": (2 * two + two + 1) * values * size + 2 * case["width"] * size, "flops": 15 * values}
    if op == "int8":
        k, n = case["k"], case["n"]
        return {"bytes": rows * k + n * k + 4 * (rows + n) + rows * n * size + (n * size if case["bias"] else 0), "flops": 2 * rows * k * n}
    if op == "chain":
        k, n, layers = case["width"], case["hidden"], case["layers"]
        last = n if layers == 1 else k
        return {"bytes": 3 * rows * k * size + k * size + layers * n * k + rows * last * size, "flops": 2 * layers * rows * k * n}
    k, n = case["k"], case["n"]
    return {"bytes": 2 * (rows * (k + n) + n * k) * size + (2 * n * size if case["bias"] else 0), "flops": 6 * rows * k * n}
