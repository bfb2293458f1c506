"""GPU: the norm, the linear layers with 8-bit checkpoints and the 8-bit product run together, as blocks of a network."""
import pytest
import torch

from triton_helpers_amd.layers.int8_linear import int8_linear, quantize_rows
from triton_helpers_amd.layers.rms_norm import rms_norm, rms_norm_int8
from triton_helpers_amd.layers.wide_mlp import WideMLP

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _block(d, h, dtype, activation="gelu", bias=True):
    torch.manual_seed(d)
    m = WideMLP(d, h, activation, bias).to(DEV, dtype)
    with torch.no_grad():
        m.norm.weight.add_(torch.randn_like(m.norm.weight) * 0.2)
    return m


def _kept(t, on):
    """The rows that the 8-bit checkpoint of t stands for, with the gradient of t itself."""
    if not on:
        return t
    a = t.detach().abs().amax(-1, keepdim=True)
    q = torch.round(t.detach() * (127 / a)) * (a / 127)
    return t + (q - t.detach())


def _act(z, name):
    return {"gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "relu": torch.relu}[name](z)


def _plain(m, x, r, eight):
    """The block in 64 bits; eight: both linear layers see the 8-bit form of their inputs."""
    p = {k: v.detach().double() for k, v in m.named_parameters()}
    leaves = {"x": x.double(), "r": None if r is None else r.double(), **p}
    leaves = {k: None if v is None else v.requires_grad_() for k, v in leaves.items()}
    h = leaves["x"] if r is None else leaves["x"] + leaves["r"]
    y = h * (h.square().mean(-1, keepdim=True) + m.norm.eps).rsqrt() * leaves["norm.weight"]
    z = _kept(y, eight) @ leaves["up.weight"].t()
    z = z if m.up.bias is None else z + leaves["up.bias"]
    out = _act(_kept(z, eight), m.down.activation) @ leaves["down.weight"].t()
    out = out if m.down.bias is None else out + leaves["down.bias"]
    return leaves, out, h


def _near(got, want, share, what):
    """In the 2-norm: roundings of single values are independent of each other."""
    far = float((got.detach().double() - want.detach()).norm() / want.detach().norm())
    assert far <= share, f"{what}: {far:.3g} of the norm"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,d,h", [(1, 64, 128), (37, 200, 520), (1000, 777, 333), (2048, 512, 2048)])
@pytest.mark.parametrize("name,residual,bias", [("gelu", True, True), ("silu", False, False), ("relu", True, True)])
def test_training_step(rows, d, h, dtype, name, residual, bias):
    """A block's results and gradients against 64 bits whose linear layers see 8-bit rows in the gradient.  A value passes at most eight roundings
    to 16 bits of half a step u each and two to 8 bits, a step of which is at most a / 127 of the row's largest value, some 4.5 of
    its root mean square: 4.5 / 127 / sqrt(12) = 1 % of the norm, twice."""
    m = _block(d, h, dtype, name, bias)
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, r, do, ds = (torch.randn(rows, d, generator=g, device=DEV).to(dtype) for _ in range(4))
    r = r if residual else None
    xl, rl = x.clone().requires_grad_(), None if r is None else r.clone().requires_grad_()
    out, stream = m(xl, rl)
    torch.autograd.backward((out, stream) if residual else (out,), (do, ds) if residual else (do,))
    leaves, want, h64 = _plain(m, x, r, False)
    u = torch.finfo(dtype).eps / 2
    _near(out, want, 8 * u, "out")
    _near(stream, h64, u, "stream")
    torch.autograd.backward((want, h64) if residual else (want,), (do.double(), ds.double()) if residual else (do.double(),))
    share = 8 * u + 0.02
    # a gate of ReLU that the 8-bit row sees closed, or that 16-bit sums open, is a whole term: up to 1 % of them lie within half a step of zero
    share = share + (0.15 if name == "relu" else 0.0)
    got = {"x": xl.grad, **{k: v.grad for k, v in m.named_parameters()}}
    if residual:
        got["r"] = rl.grad
    for k, v in got.items():
        _near(v, leaves[k].grad, share, k)


@pytest.mark.parametrize("rows", [1, 5, 64, 65, 1000])
@pytest.mark.parametrize("d,h", [(96, 400), (777, 333), (2048, 1024)])
def test_serving(rows, d, h):
    """The 8-bit block is its operators one after another, and near the block that it was made from: four roundings to 8 bits, rows and
    weights of two layers, 1 % of the norm each as above (weights are uniform: less)."""
    m = _block(d, h, torch.bfloat16)
    eight = m.to_int8()
    x, r = torch.randn(rows, d, device=DEV).bfloat16(), torch.randn(rows, d, device=DEV)
    out, stream = eight(x, r)
    with torch.no_grad():
        q, s, again = rms_norm_int8(x, m.norm.weight, m.norm.eps, r)
        z = int8_linear(q, s, *quantize_rows(m.up.weight), m.up.bias, "gelu")
        want = int8_linear(*quantize_rows(z), *quantize_rows(m.down.weight), m.down.bias)
    assert torch.equal(out, want) and torch.equal(stream, again) and stream.dtype == torch.float32
    _, full, h64 = _plain(m, x, r, False)
    _near(out, full, 0.04 + 8 * 2.0**-9, "out")
    assert torch.equal(stream, x.float() + r)
    alone, same = eight(x)
    assert same is x
    with torch.no_grad():
        assert torch.equal(alone, eight.down(eight.up(*rms_norm_int8(x, m.norm.weight, m.norm.eps))))


def test_two_blocks_train_under_autocast():
    """Float32 parameters, a float32 residual stream, gradients for everything."""
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(WideMLP(72, 160) for _ in range(2)).to(DEV)
    x = torch.randn(300, 72, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out, stream = blocks[0](x)
        out, stream = blocks[1](out, stream)
        loss = (out.float() + stream).square().mean()
    loss.backward()
    assert out.dtype == torch.bfloat16 and stream.dtype == torch.float32
    for p in [x, *blocks.parameters()]:
        assert p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() and p.grad.any()


def test_serving_a_token_captured():
    m = _block(256, 1024, torch.bfloat16).to_int8()
    x, r = torch.randn(8, 256, device=DEV).bfloat16(), torch.randn(8, 256, device=DEV).bfloat16()
    m(x, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, stream = m(*m(x, r))
    for _ in range(3):
        x.normal_()
        r.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = m(*m(x, r))
        assert torch.equal(out, want[0]) and torch.equal(stream, want[1])


def test_training_captured_and_an_eager_graph_refused():
    """Two blocks' step replayed; while a graph of the same leaves from outside is alive, the captured forward refuses to begin."""
    blocks = [_block(72, 160, torch.bfloat16), _block(72, 160, torch.bfloat16, "silu")]
    leaves = [p for m in blocks for p in m.parameters()]
    x, target = torch.randn(50, 72, device=DEV).bfloat16(), torch.randn(50, 72, device=DEV).bfloat16()

    def forward():
        out, stream = blocks[1](*blocks[0](x))
        return out + stream

    alive = forward()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside of this capture"):
        with torch.cuda.graph(graph):
            forward()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward()
        grads = torch.autograd.grad(y, leaves, target)
    for _ in range(3):
        x.normal_()
        target.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = forward()
        assert torch.equal(y, want)
        for a, b in zip(grads, torch.autograd.grad(want, leaves, target)):
            assert torch.equal(a, b)


def test_command_line(tmp_path):
    from triton_helpers.layers.wide_mlp.__main__ import main

    tables = main(["benchmark", "-L", "64", "-D", "128", "-H", "256", "-w", "2", "-r", "5", "-o", str(tmp_path)])
    assert len(tables) == 1 and len(tables[0].header) == 10 and all(v > 0 for v in tables[0].rows[0])
    main(["benchmark", "-p", "baseline", "checkpointed", "-m", "fwd-bwd", "bwd", "-d", "bf16", "-L", "64", "-D", "128", "-H", "256", "-w", "2", "-r", "5"])
    with pytest.raises(ValueError, match="no backward"):
        main(["benchmark", "-p", "int8", "-m", "bwd", "-L", "64", "-D", "128", "-H", "256"])
    assert rms_norm(torch.ones(1, 8, device=DEV), None).shape == (1, 8)
