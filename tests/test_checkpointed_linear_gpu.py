"""GPU: the linear layer that keeps its input in 8 bits.

Most tests are exact: small whole numbers, rows whose largest magnitude is 127 (the 8-bit form is the row itself), sums below 2^24.  Nothing rounds
but the result, so it has to equal the exact sum rounded once.  With other values: U = 2^-24, u half a step of the 16-bit type, mass the sum of
magnitudes of the products.  An operand act(x) is rounded to 16 bits (u, and 8 U of its own computation beside 1.5e-7 |x| of a GELU), a sum
of K products adds (K + 4) U, the result's rounding u of itself; dx is multiplied by act'(x^), which is off by (5 + 2 |x|) U or 4e-7.
"""
import pytest
import torch

from triton_helpers_amd.layers.checkpointed_linear import CheckpointedLinear, checkpointed_linear
from triton_helpers_amd.layers.int8_linear import quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
HALF = [torch.bfloat16, torch.float16]


def whole(m, n, k, dtype, seed=0, bias=True):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def ints(*shape, most=2):
        return torch.randint(-most, most + 1, shape, generator=g, device=DEV).to(dtype)

    x = ints(m, k, most=3)
    x[torch.arange(m, device=DEV), torch.randint(0, k, (m,), generator=g, device=DEV)] = 127
    return x, ints(n, k), ints(n) if bias else None, ints(m, n)


def act(z, name):
    """(act(z), act'(z)) in 64 bits."""
    z = z.double()
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "relu2":
        return z.clamp_min(0) ** 2, 2 * z.clamp_min(0)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) * 0.3989422804014327
    return z, torch.ones_like(z)


def step(x, w, b, dy, name="none", f=checkpointed_linear):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = f(leaves[0], leaves[1], leaves[2], name)
    y.backward(dy)
    return [y.detach(), *(None if t is None else t.grad for t in leaves)]


def exact(x, w, b, dy, name="none"):
    h, slope = act(x, name)
    y = h @ w.double().t()
    out = [y if b is None else y + b.double(), (dy.double() @ w.double()) * slope, dy.double().t() @ h]
    out = [t.to(x.dtype) for t in out]
    return out + [None if b is None else dy.double().sum(0).to(x.dtype)]


def check_exact(got, want):
    for a, b, what in zip(got, want, ("y", "dx", "dw", "db")):
        assert (a is None) == (b is None), what
        if a is not None:
            assert a.dtype == b.dtype and a.shape == b.shape, what
            bad = (a != b).nonzero()
            assert bad.numel() == 0, f"{what}: {bad.shape[0]} of {a.numel()} differ, first at {bad[0].tolist()}"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m", [1, 2, 31, 32, 33, 64, 127, 128, 129, 500])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 8), (8, 1), (7, 5), (16, 32), (33, 31), (64, 96), (100, 128), (128, 129), (200, 264), (257, 777)])
def test_sizes(m, n, k, dtype):
    args = whole(m, n, k, dtype, seed=m + n + k, bias=n % 2 == 0)
    check_exact(step(*args), exact(*args))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k", [(4096, 4096, 128), (3000, 4000, 520), (1000, 3333, 4097), (20000, 256, 256), (50000, 72, 40), (33333, 129, 257), (70, 5000, 6000), (2048, 6150, 2056)])
@pytest.mark.parametrize("name", ["none", "relu"])
def test_large(m, n, k, dtype, name):
    args = whole(m, n, k, dtype, seed=m)
    check_exact(step(*args, name), exact(*args, name))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k", [(8000, 1500, 5000), (8001, 5001, 1500), (1180, 3784, 7299), (13577, 5960, 301), (12022, 3075, 1550)])
def test_large_tiles_with_split_sums(m, n, k, dtype):
    """Tiles that fill the chip unevenly: the sum of one of the products is cut into a few runs."""
    args = whole(m, n, k, dtype, seed=n)
    check_exact(step(*args, "relu"), exact(*args, "relu"))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m", [2047, 2048, 2049, 12287, 12288, 12319, 40001])
@pytest.mark.parametrize("n,k", [(8, 8), (64, 128), (128, 64), (136, 120), (120, 136), (256, 256), (248, 32), (16, 256), (128, 128), (264, 256), (256, 264)])
def test_many_rows_few_channels(m, n, k, dtype):
    """Around the sizes from which, and up to which, a workgroup keeps the layer's weights."""
    args = whole(m, n, k, dtype, seed=m + n, bias=k != 64)
    check_exact(step(*args, "relu"), exact(*args, "relu"))


def test_many_rows_parts():
    """Strided rows and weights, absent gradients, nothing kept, float32 gradients, where a workgroup keeps the weights."""
    m, n, k = 20011, 64, 72
    x, w, b, dy = whole(m, n, k, torch.bfloat16)
    want = exact(x, w, b, dy, "relu")
    wide = [torch.full((t.shape[0], t.shape[1] + 24), 99.0, device=DEV, dtype=t.dtype) for t in (x, w, dy)]
    for at in (8, 3):  # on and off 16-byte boundaries
        views = [v[:, at : at + t.shape[1]] for v, t in zip(wide, (x, w, dy))]
        for v, t in zip(views, (x, w, dy)):
            v.copy_(t)
        check_exact(step(views[0], views[1], b, views[2], "relu"), want)
        check_exact(step(views[0], w, b, dy, "relu"), want)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)):
        leaves = [t.clone().requires_grad_(bool(r)) for t, r in zip((x, w, b), need)]
        checkpointed_linear(*leaves, "relu").backward(dy)
        for t, r, g in zip(leaves, need, want[1:]):
            assert (t.grad is not None) == bool(r) and (not r or torch.equal(t.grad, g))
    with torch.no_grad():
        assert torch.equal(checkpointed_linear(x, w, b, "relu"), want[0])
        assert torch.equal(checkpointed_linear(x, w), (x.double() @ w.double().t()).bfloat16())
    bl, wl = b.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = checkpointed_linear(x, wl, bl, "relu")
    y.backward(dy)
    assert torch.equal(wl.grad.double(), dy.double().t() @ x.double().clamp_min(0)) and torch.equal(bl.grad.double(), dy.double().sum(0))
    # rows without an 8-bit form
    x[7, 3], x[m - 1, 0] = float("nan"), -float("inf")
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = checkpointed_linear(xl, wl, b, "gelu")
    y.backward(dy)
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[7] = keep[m - 1] = False
    assert torch.isnan(y[7]).all() and torch.isfinite(y[keep]).all() and torch.isnan(wl.grad).all()
    assert torch.isnan(xl.grad[~keep]).all() and torch.isfinite(xl.grad[keep]).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("name", ["none", "relu", "relu2", "silu", "gelu"])
@pytest.mark.parametrize("m,n,k", [(1, 70, 90), (300, 70, 90), (300, 136, 2500), (5000, 64, 48), (17000, 64, 48), (17000, 200, 256)])
def test_activations(m, n, k, dtype, name):
    g = torch.Generator(device=DEV).manual_seed(k)
    x, w, b, dy = ((torch.randn(*s, generator=g, device=DEV) * c).to(dtype) for s, c in (((m, k), 2), ((n, k), k**-0.5), ((n,), 1), ((m, n), 1)))
    y, dx, dw, db = step(x, w, b, dy, name)
    u = torch.finfo(dtype).eps / 2
    q, s = quantize_rows(x)
    kept = (s[:, None] * q).double()

    def hold(got, want, bound, what):
        excess = (got.double() - want).abs() - bound - u * want.abs() - (2.0**-25 if dtype == torch.float16 else 0)
        assert (excess <= 0).all(), f"{what}: {float(excess.max()):.3g} beyond"

    def operand(z):
        h, _ = act(z, name)
        return h, (0 if name == "none" else u) * h.abs() + (8 * U * h.abs() + 1.5e-7 * z.abs().double() if name in ("silu", "gelu", "relu2") else 0) + U * h.abs() \
            + (2.0**-25 if dtype == torch.float16 else 0)

    h, err = operand(x)
    wa, da = w.double().abs(), dy.double().abs()
    hold(y, h @ w.double().t() + b.double(), err @ wa.t() + (k + 4) * U * (h.abs() @ wa.t() + b.double().abs()), "y")
    # the rounded x^ is an operand even without an activation
    h, _ = act(kept, name)
    _, err = operand(kept)
    err = err + (u * h.abs() if name == "none" else 0)
    hold(dw, dy.double().t() @ h, da.t() @ err + (m + 4) * U * (da.t() @ h.abs()), "dw")
    _, slope = act(kept, name)
    inner, mass = dy.double() @ w.double(), da @ wa
    hold(dx, inner * slope, (n + 4) * U * mass * slope.abs() + inner.abs() * ((5 + 2 * kept.abs()) * U * (1 + slope.abs()) + 4e-7 * (1 + kept.abs())) * (name != "none"), "dx")
    hold(db, dy.double().sum(0), (m + 4) * U * da.sum(0), "db")


def test_gradients_against_differences():
    """The formulas above: the exact gradient of act(x) W^T + b where x^ is x, against central differences in 64 bits."""
    for name in ("none", "relu2", "silu", "gelu"):
        x, w, b, dy = (t.double() * 0.3 for t in whole(3, 4, 5, torch.float32))
        h, slope = act(x, name)
        dx, dw = (dy @ w) * slope, dy.t() @ h

        def total(x, w):
            return float(((act(x, name)[0] @ w.t() + b) * dy).sum())

        for i in range(3):
            for j in range(5):
                e = torch.zeros_like(x)
                e[i, j] = 1e-5
                assert abs((total(x + e, w) - total(x - e, w)) / 2e-5 - float(dx[i, j])) < 1e-5 * (1 + abs(float(dx[i, j])))
        for i in range(4):
            for j in range(5):
                e = torch.zeros_like(w)
                e[i, j] = 1e-5
                assert abs((total(x, w + e) - total(x, w - e)) / 2e-5 - float(dw[i, j])) < 1e-5 * (1 + abs(float(dw[i, j])))


@pytest.mark.parametrize("m", [40, 700])
def test_strides_and_alignment(m):
    """Columns of wider buffers on and off 16-byte boundaries for every operand; more dimensions; expanded and transposed tensors."""
    n, k = 136, 264
    for at in (0, 8, 3):
        x, w, b, dy = whole(m, n, k, torch.bfloat16, seed=at)
        wide = [torch.full((t.shape[0], t.shape[1] + 16), 99.0, device=DEV, dtype=t.dtype) for t in (x, w, dy)]
        views = [v[:, at : at + t.shape[1]] for v, t in zip(wide, (x, w, dy))]
        for v, t in zip(views, (x, w, dy)):
            v.copy_(t)
        check_exact(step(views[0], views[1], b, views[2], "relu"), exact(x, w, b, dy, "relu"))
    x, w, b, dy = whole(m, n, k, torch.float16)
    want = exact(x, w, b, dy)
    got = step(x.t().contiguous().t(), w.t().contiguous().t(), b, dy.t().contiguous().t())
    check_exact(got, want)
    got = step(x.view(m // 10, 10, k), w, b, dy.view(m // 10, 10, n))
    check_exact([got[0].flatten(0, 1), got[1].flatten(0, 1), *got[2:]], want)
    one = x[:1].expand(m, k).detach().requires_grad_()
    y = checkpointed_linear(one, w, b)
    y.sum().backward()  # an expanded upstream gradient
    check_exact([y.detach(), one.grad], exact(x[:1].expand(m, k), w, b, torch.ones_like(dy))[:2])
    vec = x[0].detach().requires_grad_()
    y = checkpointed_linear(vec, w, b)
    y.backward(dy[0])
    check_exact([y.detach(), vec.grad], [t[0] for t in exact(x[:1], w, b, dy[:1])[:2]])


def test_offsets_beyond_32_bits():
    m, n, k, stride = 2100, 64, 72, 2**20
    x, w, b, dy = whole(m, n, k, torch.bfloat16)
    base = torch.empty(m, stride, dtype=torch.bfloat16, device=DEV)
    xs, ds = base[:, 8 : 8 + k], base[:, 128 : 128 + n]
    xs.copy_(x)
    ds.copy_(dy)
    want = exact(x, w, b, dy, "relu")
    check_exact(step(xs, w, b, ds, "relu"), want)
    check_exact(step(x, w, b, dy, "relu"), want)
    ws = base[:n, 256 : 256 + k]
    ws.copy_(w)
    check_exact(step(x, ws, b, dy, "relu"), want)
    del base, xs, ds, ws
    m, n, k = 2**20 + 77, 2056, 24  # more results than 2^31; dW over many rows
    x, w, b, dy = whole(m, n, k, torch.bfloat16)
    y, dx, dw, db = step(x, w, b, dy, "relu")
    for at in (0, 2**20 - 8, m - 100):
        c = slice(at, at + 100)
        check_exact([y[c], dx[c]], exact(x[c], w, b, dy[c], "relu")[:2])
    del y, dx
    h = x.double().clamp_min(0)
    want = sum(dy[i : i + 2**17].double().t() @ h[i : i + 2**17] for i in range(0, m, 2**17))
    assert float((want.abs()).max()) < 2**24 and torch.equal(dw, want.to(torch.bfloat16))
    assert torch.equal(db, sum(dy[i : i + 2**17].double().sum(0) for i in range(0, m, 2**17)).to(torch.bfloat16))


def test_more_pieces_than_one_row_of_a_grid():
    """act(x^) and a copied dy of more than 2^28 pieces of 16 bytes; only the last rows have gradients."""
    m, n, k, tail = 2**21 + 3, 12, 1030, 45
    x, w, b, dy = whole(m, n, k, torch.bfloat16)
    dy[:-tail] = 0
    got = step(x, w, b, dy, "relu")
    want = exact(x[-tail:], w, b, dy[-tail:], "relu")
    check_exact([got[0][-tail:], got[1][-tail:], *got[2:]], want)
    assert got[1][:-tail].abs().max() == 0


def test_rows_that_are_not_finite():
    """They are NaN where they are used, and nothing else is."""
    for name in ("none", "relu", "gelu"):
        x, w, b, dy = whole(150, 40, 70, torch.bfloat16)
        x[7, 3], x[9, 0] = float("nan"), float("inf")
        w[:, 3] += (w[:, 3] == 0)  # a NaN times zero is one, too, but an infinity times zero would make two cases of one
        y, dx, dw, db = step(x, w, b, dy, name)
        keep = torch.ones(150, dtype=torch.bool, device=DEV)
        keep[7] = keep[9] = False
        assert torch.isnan(y[7]).all() and torch.isfinite(y[keep]).all() and not torch.isfinite(y[9]).any()
        assert torch.isnan(dw).all() and torch.isfinite(dx[keep]).all() and torch.isfinite(db).all()
        assert name == "none" or torch.isnan(dx[7]).all()
    # zeros, and an infinity that a closed gate holds back
    x, w, b, dy = whole(20, 40, 70, torch.bfloat16)
    x[3] = 0
    dy[5, 0] = float("inf")
    w[0] = 1
    y, dx, dw, _ = step(x, w, b, dy, "relu")
    assert torch.equal(y[3], b) and not dx[3].any()
    assert (dx[5][x[5] <= 0] == 0).all() and torch.isinf(dx[5][x[5] > 0]).all()


@pytest.mark.parametrize("name", ["none", "silu"])
def test_absent_gradients_and_no_rows(name):
    x, w, b, dy = whole(200, 48, 80, torch.bfloat16)
    full = step(x, w, b, dy, name)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)):
        leaves = [t.clone().requires_grad_(bool(r)) for t, r in zip((x, w, b), need)]
        checkpointed_linear(*leaves, name).backward(dy)
        for t, r, g in zip(leaves, need, full[1:]):
            assert (t.grad is not None) == bool(r) and (not r or torch.equal(t.grad, g))
    with torch.no_grad():
        assert torch.equal(checkpointed_linear(x, w, b, name), full[0])
        assert torch.equal(checkpointed_linear(x[:, 1:], w[:, 1:], b, name), checkpointed_linear(x[:, 1:].contiguous(), w[:, 1:].contiguous(), b, name))
    xl, wl, bl = x[:0].clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    checkpointed_linear(xl, wl, bl, name).sum().backward()
    assert xl.grad.shape == (0, 80) and not wl.grad.any() and not bl.grad.any()


def test_what_is_kept():
    """8 bits a value of the input, a scale a row and the weight: nothing else stays alive between forward and backward."""
    x, w, b, dy = whole(4096, 512, 1024, torch.bfloat16)
    wl = w.clone().requires_grad_()
    a = (x * 1).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = checkpointed_linear(a, wl, None, "gelu")
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held <= x.numel() + 4096 * 4 + 4096, held
    a.data.zero_()  # the input itself is not needed any more
    y.backward(dy)
    assert torch.equal(wl.grad, step(x, w, None, dy, "gelu")[2])


@pytest.mark.parametrize("dtype", HALF)
def test_autocast(dtype):
    m = CheckpointedLinear(72, 40, activation="relu").to(DEV)
    x, w, b, dy = whole(300, 40, 72, dtype)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    xl = x.float().requires_grad_()
    with torch.autocast("cuda", dtype=dtype):
        y = m(xl)
    y.backward(dy)
    want = exact(x, w, b, dy, "relu")
    assert y.dtype == dtype and torch.equal(y, want[0])
    assert xl.grad.dtype == torch.float32 and torch.equal(xl.grad, want[1].float())
    h = x.double().clamp_min(0)
    assert m.weight.grad.dtype == torch.float32 and torch.equal(m.weight.grad.double(), dy.double().t() @ h)  # not rounded on the way
    assert m.bias.grad.dtype == torch.float32 and torch.equal(m.bias.grad.double(), dy.double().sum(0))
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear

    leaves = [t.detach().clone().requires_grad_() for t in (xl, m.weight, m.bias)]
    with torch.autocast("cuda", dtype=dtype):
        y2 = _checkpointed_linear.apply(*leaves, "relu")
    y2.backward(dy)
    for a, c in zip((y2, *(t.grad for t in leaves)), (y, xl.grad, m.weight.grad, m.bias.grad)):
        assert a.dtype == c.dtype and torch.equal(a, c)


def test_python_function_gives_the_same():
    from triton_helpers_amd.layers.checkpointed_linear.kernel import _checkpointed_linear

    for bias in (True, False):
        x, w, b, dy = whole(333, 50, 60, torch.float16, bias=bias)
        for a, c in zip(step(x, w, b, dy, "gelu"), step(x, w, b, dy, "gelu", _checkpointed_linear.apply)):
            assert (a is None) == (c is None) and (a is None or torch.equal(a, c))


def test_the_same_bits_every_time_and_on_another_stream():
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w, dy = (torch.randn(*s, generator=g, device=DEV).bfloat16() for s in ((30000, 200), (100, 200), (30000, 100)))
    b = torch.randn(100, generator=g, device=DEV)
    want = step(x, w, b, dy, "gelu")
    assert want[3].dtype == torch.float32
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x, w, b, dy, "gelu")
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_captured():
    x, w, b, dy = whole(700, 72, 136, torch.bfloat16)
    static = [t.clone().requires_grad_() for t in (x, w, b)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(checkpointed_linear(*static, "relu"), static, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = checkpointed_linear(*static, "relu")
        grads = torch.autograd.grad(y, static, dy)
    for turn in range(3):
        x, w, b, _ = whole(700, 72, 136, torch.bfloat16, seed=50 + turn)
        with torch.no_grad():
            for t, v in zip(static, (x, w, b)):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        check_exact([y, *grads], exact(x, w, b, dy, "relu"))


def test_a_second_derivative_is_refused():
    x, w, b, dy = whole(8, 16, 24, torch.bfloat16)
    xl = x.clone().requires_grad_()
    g, = torch.autograd.grad(checkpointed_linear(xl, w, b, "gelu"), xl, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
