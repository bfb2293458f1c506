"""GPU: the norm with a residual and its 8-bit form against plain 64-bit formulas.

Tolerances.  U = 2^-24 is half a step of float32.  A sum over a row adds at most 64 products in a thread and 16 levels of a tree, so a
statistic is off by at most 100 U of the sum of magnitudes, and a result adds its own rounding, half a step of its type: eps / 2 of the value
(and half of the smallest step, where float16 values are subnormal).
"""
import pytest
import torch

from triton_helpers_amd.layers.rms_norm import RMSNorm, rms_norm, rms_norm_int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
EPS = 1e-6
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 1e-38, torch.float32: 1e-38}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, bound, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    excess = (got - want).abs() - bound
    assert (excess <= 0).all(), f"{what}: {float(excess.max()):.3g} beyond the bound at {int(excess.argmax())}"


def inputs(rows, width, dtype, rdtype=None, wdtype=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    x = (rand(rows, width) * 2).to(dtype)
    r = None if rdtype is None else (rand(rows, width) * 3).to(rdtype)
    w = None if wdtype is None else (1 + 0.3 * rand(width)).to(wdtype)
    return x, r, w, rand(rows, width).to(dtype), None if rdtype is None else rand(rows, width).to(rdtype)


def formula(x, r, w, eps=EPS):
    h = x.double() if r is None else x.double() + r.double()
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = h * rstd if w is None else h * rstd * w.double()
    return h, rstd, y


def check_forward(y, stream, x, r, w):
    h, _, want = formula(x, r, w)
    within(y, want, (half_step(y.dtype) + 100 * U) * want.abs() + TINY[y.dtype], "y")
    if r is not None:
        assert stream.dtype == r.dtype
        within(stream, h, (half_step(r.dtype) + 2 * U) * h.abs() + TINY[r.dtype], "stream")


def check_backward(x, r, w, dy, ds, kept, dx, dr, dw):
    """kept: the rounded rows that the backward works on."""
    _, rstd, _ = formula(x, r, w)
    n = kept.double() * rstd
    g = dy.double() if w is None else dy.double() * w.double()
    m = (g * n).mean(-1, keepdim=True)
    dh = rstd * (g - n * m)
    slack = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    if ds is not None:
        dh, slack = dh + ds.double(), slack + ds.double().abs()
    for got, name in ((dx, "dx"), (dr, "dr")):
        if got is not None:
            within(got, dh, half_step(got.dtype) * dh.abs() + 200 * U * slack + TINY[got.dtype], name)
    if dw is not None:
        want, mass = (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0)
        within(dw, want, half_step(dw.dtype) * want.abs() + (x.shape[0] + 120) * U * mass + TINY[dw.dtype], "dw")


def step(x, r, w, dy, ds):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, r, w)]
    out = rms_norm(leaves[0], leaves[2], EPS, leaves[1])
    y, stream = (out, None) if r is None else out
    if r is None:
        y.backward(dy)
    else:
        torch.autograd.backward((y, stream), (dy, ds))
    grads = [None if t is None else t.grad for t in leaves]
    return y.detach(), None if stream is None else stream.detach(), *grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 64, 65, 511, 512, 513, 777, 2048, 2049, 4096, 4100, 8192, 8193, 16384, 16392, 20001, 32768, 32769, 40003])
def test_widths(width, dtype):
    rows = 5 if width > 4096 else 67
    x, r, w, dy, ds = inputs(rows, width, dtype, dtype, dtype)
    y, stream, dx, dr, dw = step(x, r, w, dy, ds)
    check_forward(y, stream, x, r, w)
    check_backward(x, r, w, dy, ds, stream, dx, dr, dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 1023, 4097, 9001])
@pytest.mark.parametrize("width", [72, 4096])
def test_rows(rows, width, dtype):
    """Fewer and more rows than the backward has groups of threads; no residual."""
    x, _, w, dy, _ = inputs(rows, width, dtype, None, dtype, seed=rows)
    y, _, dx, _, dw = step(x, None, w, dy, None)
    check_forward(y, None, x, None, w)
    check_backward(x, None, w, dy, None, x, dx, None, dw)


@pytest.mark.parametrize("dtype,rdtype,wdtype", [
    (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16, torch.float32),
    (torch.float16, None, torch.bfloat16), (torch.float32, torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32, None), (torch.float32, None, None)])
@pytest.mark.parametrize("width", [100, 3000, 33000])
def test_mixed_types(dtype, rdtype, wdtype, width):
    x, r, w, dy, ds = inputs(11, width, dtype, rdtype, wdtype, seed=3)
    y, stream, dx, dr, dw = step(x, r, w, dy, ds)
    assert y.dtype == dtype and dx.dtype == dtype and (dr is None or dr.dtype == rdtype) and (dw is None or dw.dtype == wdtype)
    check_forward(y, stream, x, r, w)
    check_backward(x, r, w, dy, ds, x if r is None else stream, dx, dr, dw)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_against_differences(dtype):
    """The formula's gradient, which the other tests hold the kernels to, against central differences in 64 bits."""
    x, r, w, dy, ds = (t.double() for t in inputs(3, 12, dtype, dtype, dtype, seed=5))

    def total(x, r, w):
        h, _, y = formula(x, r, w)
        return (y * dy).sum() + (h * ds).sum()

    h, rstd, _ = formula(x, r, w)
    n, g = h * rstd, dy * w
    dh, dw = ds + rstd * (g - n * (g * n).mean(-1, keepdim=True)), (dy * n).sum(0)
    step_ = 1e-5
    for k in range(12):
        e = torch.zeros(12, dtype=torch.double, device=DEV)
        e[k] = step_
        assert abs(float(total(x, r, w + e) - total(x, r, w - e)) / (2 * step_) - float(dw[k])) < 1e-7
        for i in range(3):
            d = torch.zeros_like(x)
            d[i, k] = step_
            assert abs(float(total(x + d, r, w) - total(x - d, r, w)) / (2 * step_) - float(dh[i, k])) < 1e-7


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 9, 512, 777, 4096, 8200, 33001])
@pytest.mark.parametrize("residual", [False, True])
def test_eight_bit_rows(width, dtype, residual):
    x, r, w, _, _ = inputs(19, width, dtype, dtype if residual else None, dtype, seed=width)
    with torch.no_grad():
        out = rms_norm_int8(x, w, EPS, r)
    q, scale = out[:2]
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and q.shape == x.shape and scale.shape == x.shape[:-1]
    h, _, v = formula(x, r, w)
    a = v.abs().amax(-1)
    within(scale, a / 127, 100 * U * a / 127, "scale")
    # a value's place among the 127 steps is off by at most 127 * 200 U (its own error and the largest value's) when it is rounded
    within(scale[:, None].double() * q, v, (0.5 + 127 * 200 * U) * a[:, None] / 127 * (1 + 100 * U), "rows")
    assert int(q.abs().amax(-1).min()) == 127
    if residual:
        within(out[2], h, (half_step(dtype) + 2 * U) * h.abs() + TINY[dtype], "stream")


@pytest.mark.parametrize("width", [40, 3000, 33001])
def test_eight_bit_rows_without_a_form(width):
    x = torch.randn(6, width, device=DEV)
    w = torch.ones(width, device=DEV)
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, width - 1] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = 1e-45
    q, scale = rms_norm_int8(x, w, 1e-6)
    assert scale[0] == 0 and scale[4] == 0 and not q[0].any() and not q[4].any()
    assert torch.isnan(scale[1:4]).all() and not q[1:4].any()
    assert torch.isfinite(scale[5]) and q[5].abs().max() == 127
    y = rms_norm(x, w, 1e-6)
    assert torch.isnan(y[1:4]).any(-1).all() and torch.isfinite(y[5]).all() and not y[0].any()
    # an infinity in the weight makes every row one without a form, but for zeros, which become NaN themselves
    w[5] = float("inf")
    assert torch.isnan(rms_norm_int8(x, w, 1e-6)[1]).all()


def test_strides_and_alignment():
    """Rows of a wider buffer, off 16-byte boundaries, a transposed and an expanded tensor, more dimensions."""
    base = torch.randn(3, 10, 600, device=DEV).bfloat16()
    w = torch.randn(523, device=DEV).bfloat16()
    x = base[..., 5:528]
    got, stream = rms_norm(x, w, EPS, residual=base[..., 1:524])
    want, want_stream = rms_norm(x.contiguous(), w, EPS, residual=base[..., 1:524].contiguous())
    assert torch.equal(got, want) and torch.equal(stream, want_stream) and got.shape == x.shape
    check_forward(got, stream, x, base[..., 1:524], w)
    for v in (torch.randn(523, 7, device=DEV).bfloat16().t(), torch.randn(1, 523, device=DEV).bfloat16().expand(7, 523), torch.randn(523, device=DEV).bfloat16()):
        assert torch.equal(rms_norm(v, w, EPS), rms_norm(v.contiguous(), w, EPS))
        assert torch.equal(rms_norm_int8(v, w.float())[0], rms_norm_int8(v.contiguous(), w.float())[0])
    strided = torch.randn(523, 2, device=DEV).bfloat16()[:, 0]
    assert torch.equal(rms_norm(x, strided, EPS), rms_norm(x, strided.contiguous(), EPS))
    xl = x.detach().requires_grad_()
    rms_norm(xl, w, EPS).sum().backward()  # an expanded upstream gradient
    ones = x.detach().contiguous().requires_grad_()
    rms_norm(ones, w, EPS).backward(torch.ones(x.shape, device=DEV, dtype=x.dtype))
    assert torch.equal(xl.grad, ones.grad)


def test_offsets_beyond_32_bits():
    rows, stride, width = 2100, 2**20, 72
    base = torch.empty(rows, stride, dtype=torch.bfloat16, device=DEV)
    x = base[:, 8 : 8 + width]
    x.copy_(torch.randn(rows, width, device=DEV))
    w = torch.ones(width, device=DEV, dtype=torch.bfloat16)
    xl, cl = x.detach().requires_grad_(), x.contiguous().requires_grad_()
    dy = base[:, 8 + width : 8 + 2 * width]
    dy.copy_(torch.randn(rows, width, device=DEV))
    a, b = rms_norm(xl, w), rms_norm(cl, w)
    a.backward(dy)
    b.backward(dy.contiguous())
    assert torch.equal(a, b) and torch.equal(xl.grad, cl.grad)


def test_more_rows_than_one_launch_takes():
    rows = 2**21 + 37
    x = torch.randn(rows, 8, device=DEV, dtype=torch.bfloat16)
    r = torch.randn(rows, 8, device=DEV)
    w = torch.randn(8, device=DEV)
    y, s = rms_norm(x, w, EPS, r)
    q, scale, s8 = rms_norm_int8(x, w, EPS, r)
    check_forward(y, s, x, r, w)
    assert torch.equal(s8, s)
    for part in (slice(0, 50), slice(2**21 - 20, rows)):
        alone = rms_norm_int8(x[part], w, EPS, r[part])
        assert torch.equal(alone[0], q[part]) and torch.equal(alone[1], scale[part])


def test_the_residual_is_the_input():
    x, _, w, dy, ds = inputs(20, 100, torch.float32, torch.float32, torch.float32)
    xl = x.clone().requires_grad_()
    y, s = rms_norm(xl, w, EPS, xl)
    torch.autograd.backward((y, s), (dy, ds))
    full = step(x, x.clone(), w, dy, ds)
    assert torch.equal(y, full[0]) and torch.equal(s, full[1]) and torch.equal(xl.grad, full[2] + full[3])


def test_no_rows_and_absent_gradients():
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    y, s = rms_norm(x, w, EPS, residual=torch.empty(0, 64, device=DEV))
    (y.sum() + s.sum()).backward()
    assert x.grad.shape == x.shape and not w.grad.any()
    q, scale = rms_norm_int8(x.detach(), w.detach())
    assert q.shape == (0, 64) and scale.shape == (0,)
    x, r, w, dy, ds = inputs(6, 64, torch.float32, torch.float32, torch.float32)
    full = step(x, r, w, dy, ds)
    # only the new residual reaches a loss; only y does; a frozen weight; frozen rows
    xl, rl = x.clone().requires_grad_(), r.clone().requires_grad_()
    rms_norm(xl, w, EPS, rl)[1].backward(ds)
    assert torch.equal(xl.grad, ds) and torch.equal(rl.grad, ds)
    xl, rl = x.clone().requires_grad_(), r.clone().requires_grad_()
    rms_norm(xl, w, EPS, rl)[0].backward(dy)
    check_backward(x, r, w, dy, None, full[1], xl.grad, rl.grad, None)
    wl = w.clone().requires_grad_()
    rms_norm(x, wl, EPS, r)[0].backward(dy)
    check_backward(x, r, w, dy, None, full[1], None, None, wl.grad)


def test_gradients_have_tensors_of_their_own():
    """The two gradients of one sum are equal; as leaves' gradients they must not share memory."""
    x, r, w, dy, ds = inputs(9, 200, torch.bfloat16, torch.bfloat16, torch.bfloat16)
    _, _, dx, dr, _ = step(x, r, w, dy, ds)
    assert torch.equal(dx, dr) and dx.data_ptr() != dr.data_ptr()
    # inside a network the two are not leaves
    a, b = (t.clone().requires_grad_() for t in (x, r))
    y, s = rms_norm(a * 1.0, w, EPS, b * 1.0)
    torch.autograd.backward((y, s), (dy, ds))
    assert torch.equal(a.grad, dx) and torch.equal(b.grad, dr) and a.grad.data_ptr() != b.grad.data_ptr()


@pytest.mark.parametrize("residual", [False, True])
def test_python_function_gives_the_same(residual):
    from triton_helpers_amd.layers.rms_norm.kernel import _rms_norm

    x, r, w, dy, ds = inputs(33, 300, torch.bfloat16, torch.bfloat16 if residual else None, torch.float32)
    want = step(x, r, w, dy, ds)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    rl = r.clone().requires_grad_() if residual else None
    out = _rms_norm.apply(xl, wl, EPS, rl)
    torch.autograd.backward(out, (dy, ds) if residual else dy)
    assert torch.equal((out[0] if residual else out), want[0]) and torch.equal(xl.grad, want[2]) and torch.equal(wl.grad, want[4])
    assert not residual or (torch.equal(out[1], want[1]) and torch.equal(rl.grad, want[3]))


def test_the_same_bits_every_time_and_on_another_stream():
    x, r, w, dy, ds = inputs(5000, 1500, torch.bfloat16, torch.bfloat16, torch.bfloat16)
    want = step(x, r, w, dy, ds)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x, r, w, dy, ds)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured():
    x, r, w, dy, ds = inputs(130, 1000, torch.float16, torch.float16, torch.float16)
    static = [t.clone() for t in (x, r, w)]
    leaves = [t.requires_grad_() for t in static]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(rms_norm(leaves[0], leaves[2], EPS, leaves[1]), leaves, (dy, ds))
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stream = rms_norm(leaves[0], leaves[2], EPS, leaves[1])
        grads = torch.autograd.grad((y, stream), leaves, (dy, ds))
        with torch.no_grad():
            q, scale = rms_norm_int8(leaves[0], leaves[2])
    for turn in range(3):
        x, r, w, *_ = inputs(130, 1000, torch.float16, torch.float16, torch.float16, seed=20 + turn)
        with torch.no_grad():
            for t, v in zip(static, (x, r, w)):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = step(x, r, w, dy, ds)
        for a, b in zip((y, stream, *grads), want):
            assert torch.equal(a, b)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip((q, scale), rms_norm_int8(x, w)))


def test_module_under_autocast():
    m = RMSNorm(96).to(DEV)
    x = torch.randn(4, 7, 96, device=DEV, dtype=torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, s = m(x, torch.randn(4, 7, 96, device=DEV))
    assert y.dtype == torch.bfloat16 and s.dtype == torch.float32
    (y.float().sum() + s.sum()).backward()
    assert m.weight.grad.dtype == torch.float32


def test_a_changed_input_and_a_second_derivative_are_refused():
    x, _, w, dy, _ = inputs(4, 64, torch.float32, None, torch.float32)
    xl = x.clone().requires_grad_()
    y = rms_norm(xl * 1.0, w)
    g, = torch.autograd.grad(y, xl, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_int8(xl, w)
