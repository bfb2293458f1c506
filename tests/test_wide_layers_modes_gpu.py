"""GPU: the wide layers beside torch's tracer, forward-mode derivatives and function transforms."""
import pytest
import torch

from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_amd.layers.int8_linear import Int8Linear, int8_linear, quantize_rows
from triton_helpers_amd.layers.rms_norm import rms_norm, rms_norm_int8
from triton_helpers_amd.layers.wide_mlp import WideMLP

pytestmark = pytest.mark.gpu
DEV = "cuda"
M, K, N = 70, 96, 40

INFERENCE = ["quantize_rows", "int8_linear", "rms_norm_int8", "rms_norm_int8 residual"]
TRAINED = ["rms_norm", "rms_norm residual", "checkpointed_linear"]


def operator(name, seed=0):
    """(operator, its tensor arguments): the input in front."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def u(*s):
        return torch.randn(*s, generator=g, device=DEV)

    def bytes_of(*s):
        return torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)

    if name == "quantize_rows":
        return quantize_rows, [u(M, K)]
    if name == "int8_linear":
        return lambda s, t, b, q, w: int8_linear(q, s, w, t, b, "gelu"), [u(M).abs() * 0.01, u(N).abs() * 0.01, u(N), bytes_of(M, K), bytes_of(N, K)]
    if name.startswith("rms_norm"):
        f = rms_norm_int8 if name.startswith("rms_norm_int8") else rms_norm
        if name.endswith("residual"):
            return lambda x, w, r: f(x, w, 1e-6, r), [u(M, K).bfloat16(), u(K), u(M, K)]
        return f, [u(M, K).bfloat16(), u(K)]
    return lambda x, w, b: checkpointed_linear(x, w, b, "gelu"), [u(M, K).bfloat16(), u(N, K).bfloat16(), u(N)]


def several(out):
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("name,train", [(n, False) for n in INFERENCE + TRAINED] + [(n, True) for n in TRAINED])
def test_a_traced_function_runs_the_operator(name, train):
    fn, args = operator(name)
    _, others = operator(name, seed=1)
    if train:
        args[1] = args[1].requires_grad_()

    def doubled(*a):
        return tuple(t.float() * 2 for t in several(fn(*a)))

    traced = torch.jit.trace(doubled, tuple(args), check_trace=False)
    assert "PythonOp" in str(traced.graph) or "^" in str(traced.graph)
    for _ in range(3):
        junk = [torch.full((M, K), 77.0, device=DEV).to(t) for t in (torch.float32, torch.bfloat16, torch.int8)]  # what a fresh allocation may hold
        del junk
        for a, b in zip(traced(*others), doubled(*others)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", INFERENCE + TRAINED)
def test_a_traced_function_checks_its_arguments(name):
    """Tensors of another shape or type than at the tracing are held against the operator's conditions before anything is launched."""
    fn, args = operator(name)
    traced = torch.jit.trace(lambda *a: several(fn(*a)), tuple(args), check_trace=False)
    for i in range(1, len(args)):  # (torch's interpreter hands the error on as its own)
        with pytest.raises(RuntimeError, match="must|not implemented|runs on|NotImplemented|Assertion"):
            traced(*args[:i], args[i][:-1], *args[i + 1 :])
    with pytest.raises(RuntimeError):
        traced(args[0].double(), *args[1:])


def test_traced_modules():
    torch.manual_seed(0)
    linear = Int8Linear.from_linear(torch.nn.Linear(K, N).to(DEV, torch.bfloat16), "relu")
    block = WideMLP(K, N).to(DEV, torch.bfloat16).to_int8()
    x, other = torch.randn(M, K, device=DEV).bfloat16(), torch.randn(M, K, device=DEV).bfloat16()
    for m, args, others in ((linear, (x,), (other,)), (block, (x, other), (other, x))):
        traced = torch.jit.trace(m, args, check_trace=False)
        for a, b in zip(several(traced(*others)), several(m(*others))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("mode", ["plain", "no_grad", "train"])
@pytest.mark.parametrize("name,which", [(n, i) for n in INFERENCE + TRAINED for i in range({"quantize_rows": 1, "rms_norm": 2, "rms_norm_int8": 2}.get(n, 3))])
def test_forward_mode_derivatives_are_refused(name, which, mode):
    """A tangent that no kernel carries on raises instead of getting lost."""
    import torch.autograd.forward_ad as fw

    fn, args = operator(name)
    if mode == "train" and name in TRAINED:
        args[1].requires_grad_()
    with fw.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            fn(*args)


@pytest.mark.parametrize("name", INFERENCE + TRAINED)
def test_function_transforms_are_refused(name):
    """Inside a transform the autograd Functions refuse, also where the operator's own arguments are plain tensors."""
    fn, args = operator(name)
    want = several(fn(*args))

    def total(s, *a):
        return sum((t.float() * s).sum() for t in several(fn(*a)))

    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: total(s, *args))(torch.ones(3, device=DEV))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda s: total(s, *args))(torch.ones((), device=DEV))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: total(1.0, x, *args[1:]))(torch.stack([args[0], args[0]]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: total(1.0, x, *args[1:]))(args[0])
    for a, b in zip(several(fn(*args)), want):
        assert torch.equal(a, b)


def _functions(name):
    """The operator on the native host path and as its Python Function."""
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear
    from triton_helpers_amd.layers.rms_norm.kernel import _rms_norm

    if name == "rms_norm":
        return [lambda x, w: rms_norm(x, w), lambda x, w: _rms_norm.apply(x, w, 1e-6, None)]
    if name == "rms_norm residual":
        return [lambda x, w, r: rms_norm(x, w, 1e-6, r)[0], lambda x, w, r: _rms_norm.apply(x, w, 1e-6, r)[0]]
    return [lambda x, w, b: checkpointed_linear(x, w, b, "gelu"), lambda x, w, b: _checkpointed_linear.apply(x, w, b, "gelu")]


REFUSED = "differentiable once"


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("name", TRAINED)
def test_a_second_derivative_beside_a_first_is_refused(name, python):
    """A penalty on a gradient next to an ordinary loss: the second derivative raises, whichever tensors the backward is asked for."""
    fn = _functions(name)[python]
    leaves = [t.requires_grad_() for t in operator(name)[1]]
    rows = leaves[:1] if name != "rms_norm residual" else [leaves[0], leaves[2]]

    def mixed(of, upstream=None):
        y = fn(*leaves)
        dy = torch.ones_like(y) if upstream is None else upstream
        first = torch.autograd.grad(y, of, dy, retain_graph=True)
        g = torch.autograd.grad(y, of, dy, create_graph=True)
        for a, b in zip(first, g):
            assert torch.equal(a, b.detach())
        assert all(t.requires_grad for t in g)
        return y.float().sum() + sum(t.float().square().sum() for t in g)

    for of in (rows, leaves[1:2]):
        with pytest.raises(RuntimeError, match=REFUSED):
            mixed(of).backward()
        asked = leaves if of is rows else rows  # (the weight's gradient does not depend on the weight)
        for leaf in asked[:2]:
            with pytest.raises(RuntimeError, match=REFUSED):
                torch.autograd.grad(mixed(of), leaf)
        y = fn(*leaves)
        dy = torch.randn_like(y).requires_grad_()
        with pytest.raises(RuntimeError, match=REFUSED):
            torch.autograd.grad(mixed(of, dy), dy)


@pytest.mark.parametrize("python", [False, True])
def test_gradients_that_are_constant_need_no_second_derivative(python):
    """Without an activation dx depends on the weight alone, and db on the upstream gradient: where these are constant nothing is lost, and nothing refused."""
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear
    from triton_helpers_amd.layers.rms_norm.kernel import _rms_norm

    linear = (lambda x, w, b, name="none": _checkpointed_linear.apply(x, w, b, name)) if python else checkpointed_linear
    norm = (lambda x, w, eps=1e-6, r=None: _rms_norm.apply(x, w, eps, r)) if python else rms_norm
    x, w, b = operator("checkpointed_linear")[1]
    x, b = x.requires_grad_(), b.requires_grad_()
    y = linear(x, w, b)
    g = torch.autograd.grad(y.float().sum(), (x, b), create_graph=True)
    assert not any(t.requires_grad for t in g)
    (y.float().sum() + sum(t.float().square().sum() for t in g)).backward()
    assert torch.equal(x.grad, g[0]) and torch.equal(b.grad, g[1])
    y = linear(x, w, b, "gelu")
    g, = torch.autograd.grad(y.float().sum(), b, create_graph=True)
    assert not g.requires_grad
    # the weight's part in dx, with x fixed
    w.requires_grad_()
    g, = torch.autograd.grad(linear(x, w, b).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match=REFUSED):
        torch.autograd.grad(g.float().sum(), w)
    # the new residual's own gradient goes to x and r as it is
    x, w, r = (t.requires_grad_() for t in operator("rms_norm residual")[1])
    stream = norm(x, w, 1e-6, r)[1]
    g = torch.autograd.grad(stream.float().sum(), (x, r), create_graph=True)
    assert not any(t.requires_grad for t in g) and all(torch.equal(t, torch.ones_like(t)) for t in g)
    ds = torch.randn_like(stream).requires_grad_()
    g = torch.autograd.grad(norm(x, w, 1e-6, r)[1], (x, r), ds, create_graph=True)
    with pytest.raises(RuntimeError, match=REFUSED):
        torch.autograd.grad(g[1].float().sum(), ds)


def test_a_second_derivative_under_autocast_is_refused():
    x, w, b = (t.float().requires_grad_() for t in operator("checkpointed_linear")[1])
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = checkpointed_linear(x, w, b, "silu")
    g = torch.autograd.grad(y.float().sum(), (x, w), create_graph=True)
    assert all(t.dtype == torch.float32 for t in g)
    for t, leaf in ((g[0], w), (g[1], x)):
        with pytest.raises(RuntimeError, match=REFUSED):
            torch.autograd.grad(t.sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match=REFUSED):
        (y.float().sum() + g[0].square().sum()).backward()


@pytest.mark.parametrize("python", [False, True])
def test_what_the_backward_reads_may_not_change(python):
    """Rows and weights that are kept as they are: a change between forward and backward raises.  Kept 8-bit rows are the layer's own."""
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear
    from triton_helpers_amd.layers.rms_norm.kernel import _rms_norm

    linear = (lambda x, w, b, name="none": _checkpointed_linear.apply(x, w, b, name)) if python else checkpointed_linear
    norm = (lambda x, w, eps=1e-6, r=None: _rms_norm.apply(x, w, eps, r)) if python else rms_norm
    x, w, r = (t.requires_grad_() for t in operator("rms_norm residual")[1])
    rows, weight = x * 1.0, w * 1.0
    for changed in (rows, weight):
        y = norm(rows, weight)
        with torch.no_grad():
            changed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.float().sum().backward()
    y, stream = norm(x, w, 1e-6, r)
    with torch.no_grad():
        stream.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    x, w, b = (t.requires_grad_() for t in operator("checkpointed_linear")[1])
    weight = w * 1.0
    y = linear(x * 1.0, weight, b, "gelu")
    with torch.no_grad():
        weight.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    want = torch.autograd.grad(linear(x, w, b, "gelu").float().sum(), (x, w))
    rows = x * 1.0
    y = linear(rows, w, b, "gelu")
    with torch.no_grad():
        rows.zero_()
    for a, c in zip(torch.autograd.grad(y.float().sum(), (x, w)), want):
        assert torch.equal(a, c)


def _transposed(t):
    return t.t().contiguous().t() if t.dim() == 2 else torch.stack([t, t + 1], -1)[..., 0]


def _shifted(t):
    return torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("hook", [_transposed, _shifted, lambda t: t.cpu().cuda(), None])
@pytest.mark.parametrize("m", [300, 4096])
def test_saved_tensors_in_other_places(m, hook, python):
    """What a saved-tensor hook hands back may have other strides and lie off 16-byte boundaries.

    Weights off 16-byte boundaries go to other kernels, which add up dW's products in another order: both float32 sums of m products are off by at
    most (m + 4) 2^-24 of the sum of their magnitudes, which is at most |dy|^T (|x| + a / 127) as |gelu(z)| <= |z| and the 8-bit rows are at most half a
    step, a / 254, and a rounding off; each is rounded once, by half a step."""
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear
    from triton_helpers_amd.layers.rms_norm.kernel import _rms_norm

    g = torch.Generator(device=DEV).manual_seed(m)
    x, w, dy = (torch.randn(*s, generator=g, device=DEV).bfloat16() for s in ((m, 64), (64, 64), (m, 64)))
    v = torch.randn(64, generator=g, device=DEV)

    def step(saved):
        leaves = [t.clone().requires_grad_() for t in (x, w, v)]
        xl, wl, vl = leaves
        with saved:
            y = _checkpointed_linear.apply(xl, wl, None, "gelu") if python else checkpointed_linear(xl, wl, None, "gelu")
            u = _rms_norm.apply(xl, vl, 1e-6, None) if python else rms_norm(xl, vl)
            z = (_rms_norm.apply(xl, vl, 1e-6, xl * 2) if python else rms_norm(xl, vl, 1e-6, xl * 2))[0]
        torch.autograd.backward((y, u, z), (dy, dy, dy))
        return [t.grad for t in leaves]

    want = step(torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    got = step(torch.autograd.graph.save_on_cpu() if hook is None else torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook))
    if hook is _shifted:
        h = x.double().abs() + x.double().abs().amax(-1, keepdim=True) / 127
        bound = 2 * (m + 4) * 2.0**-24 * (dy.double().abs().t() @ h) + 2 * 2.0**-8 * torch.maximum(got[1].double().abs(), want[1].double().abs())
        assert ((got.pop(1).double() - want.pop(1).double()).abs() <= bound).all()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", TRAINED)
def test_checkpointed_gradients(name):
    """A saved-tensor hook that recomputes (non-reentrant checkpointing) runs with autograd on inside the operator's backward."""
    from torch.utils.checkpoint import checkpoint

    fn, args = operator(name)

    def region(*a):  # the operator's tensors come out of a differentiable operation inside the checkpointed region
        return several(fn(*(t * 1.5 for t in a)))

    got = []
    for through in (region, lambda *a: checkpoint(region, *a, use_reentrant=False)):
        leaves = [t.detach().clone().requires_grad_() for t in args]
        out = through(*leaves)
        torch.autograd.backward(out, [torch.ones_like(t) for t in out])
        got.append([*(t.detach() for t in out), *(t.grad for t in leaves)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def _negated(t):
    """t as the imaginary part of a conjugate, whose memory holds -t; dense where it is one value."""
    v = torch.view_as_complex(torch.stack([t, -t], -1).contiguous()).conj().imag
    assert v.is_neg() and torch.equal(v, t) and (t.numel() > 1 or v.is_contiguous())
    return v


@pytest.mark.parametrize("shape", [(1, 1), (5, 1), (5, 8)])
def test_negated_views(shape):
    x, r, dy = (torch.rand(*shape, device=DEV) + 1 for _ in range(3))
    w = torch.rand(shape[1], device=DEV) + 1
    for a, b in zip(rms_norm(_negated(x), _negated(w), 1.0, _negated(r)), rms_norm(x, w, 1.0, r)):
        assert torch.equal(a, b)
    for a, b in zip(rms_norm_int8(_negated(x), _negated(w), 1.0, _negated(r)), rms_norm_int8(x, w, 1.0, r)):
        assert torch.equal(a, b)
    for a, b in zip(quantize_rows(_negated(x)), quantize_rows(x)):
        assert torch.equal(a, b)
    q, s = quantize_rows(x)
    assert torch.equal(int8_linear(q, _negated(s), q[:1], _negated(s[:1]), _negated(w[:1])), int8_linear(q, s, q[:1], s[:1], w[:1]))
    got = []
    for form in (_negated, lambda t: t):
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        y = rms_norm(form(leaves[0]), form(leaves[1]), 1.0)
        y.backward(form(dy))
        got.append([t.grad for t in leaves])
        half = [t.half().requires_grad_() for t in (x, x[:1], w[:1])]
        y = checkpointed_linear(*(form(t) for t in half), "silu")
        y.backward(form(torch.ones_like(y)))
        got[-1] += [y.detach(), *(t.grad for t in half)]
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("mode", [False, True])
@pytest.mark.parametrize("name", TRAINED)
def test_a_capture_beside_an_eager_graph_is_refused(name, mode):
    """Also where the Python Functions run (a default device is a mode): the forward refuses, while nothing has happened yet; afterwards the step replays."""
    from contextlib import nullcontext

    fn, args = operator(name)
    leaves = [t.requires_grad_() for t in args]

    def step():
        with torch.device(DEV) if mode else nullcontext():
            out = several(fn(*leaves))
        return [*out, *torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])]

    alive = fn(*leaves)
    with pytest.raises(RuntimeError, match="outside of this capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with torch.device(DEV) if mode else nullcontext():
                fn(*leaves)
    with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():  # nothing to be refused: no gradient is asked for
        with torch.device(DEV) if mode else nullcontext():
            fn(*leaves)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 4):
        with torch.no_grad():
            for t, v in zip(leaves, operator(name, seed)[1]):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_python_functions_with_arguments_left_out():
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear
    from triton_helpers_amd.layers.rms_norm.kernel import _rms_norm

    x, w, b = (t.requires_grad_() for t in operator("checkpointed_linear")[1])
    v = torch.rand(K, device=DEV).requires_grad_()
    for short, full, leaves in ((lambda: _checkpointed_linear.apply(x, w), lambda: checkpointed_linear(x, w), (x, w)),
                                (lambda: _checkpointed_linear.apply(x, w, b), lambda: checkpointed_linear(x, w, b), (x, w, b)),
                                (lambda: _rms_norm.apply(x, v), lambda: rms_norm(x, v), (x, v)),
                                (lambda: _rms_norm.apply(x, v, 0.5), lambda: rms_norm(x, v, 0.5), (x, v)),
                                (lambda: _rms_norm.apply(x, None), lambda: rms_norm(x, None), (x,))):
        got, want = short(), full()
        assert torch.equal(got, want)
        for a, c in zip(torch.autograd.grad(got.float().square().sum(), leaves), torch.autograd.grad(want.float().square().sum(), leaves)):
            assert torch.equal(a, c)
