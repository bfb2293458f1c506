"""GPU: 8-bit rows and their product against exact integer sums (in 64 bits).

Tolerances, U = 2^-24 half a step of float32: the integer sum becomes float32 (U), the two scales are multiplied (U) and applied (U), the bias is added (U):
4 U of |s t sum| + |b|.  An activation passes that on by its slope (at most 1.13; 2 |z| for relu2, and its own product's U) and adds: silu,
whose exponential is off by 2 U (1 + |z|), (5 + 2 |z|) U of its value; gelu 1.5e-7 |z| (its Phi) and 4 U.  The result's rounding is half a step of its type.
"""
import pytest
import torch

from triton_helpers_amd.layers.int8_linear import Int8Linear, int8_linear, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 1e-38, torch.float32: 1e-38}
ACTS = ["none", "relu", "relu2", "silu", "gelu"]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int32).to(torch.int8)


def case(m, n, k, bias_dtype=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, w = rows8(g, m, k), rows8(g, n, k)
    s = torch.rand(m, generator=g, device=DEV) * 0.02 + 1e-3
    t = (torch.rand(n, generator=g, device=DEV) * 0.02 + 1e-3) * k**-0.5
    b = None if bias_dtype is None else torch.randn(n, generator=g, device=DEV).to(bias_dtype)
    return q, s, w, t, b


def act(z, name):
    return {"none": lambda: z, "relu": lambda: z.clamp_min(0), "relu2": lambda: z.clamp_min(0) ** 2, "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[name]()


def check(y, q, s, w, t, b, name="none"):
    part = (q.double() @ w.double().t()) * s.double()[:, None] * t.double()
    z, mass = part, part.abs()
    if b is not None:
        z, mass = z + b.double(), mass + b.double().abs()
    want = act(z, name)
    err = 4 * U * mass
    if name == "relu2":
        err = err * 2 * z.abs() + err**2 + U * want
    elif name == "silu":
        err = err * 1.13 + (5 + 2 * z.abs()) * U * want.abs()
    elif name == "gelu":
        err = err * 1.13 + 1.5e-7 * z.abs() + 4 * U * want.abs()
    bound = err * (1 + half_step(y.dtype)) + half_step(y.dtype) * want.abs() + TINY[y.dtype]
    assert y.shape == want.shape and torch.isfinite(y).all()
    excess = (y.double() - want).abs() - bound
    assert (excess <= 0).all(), f"{float(excess.max()):.3g} beyond the bound at {int(excess.argmax())} of {tuple(y.shape)}"


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 16), (4, 15), (5, 64), (16, 17), (64, 256), (100, 255), (257, 257), (130, 1000), (513, 96), (128, 4096)])
def test_sizes(m, n, k):
    q, s, w, t, b = case(m, n, k, torch.bfloat16 if n % 2 else None, seed=m * 1000 + n)
    check(int8_linear(q, s, w, t, b), q, s, w, t, b)


@pytest.mark.parametrize("m,n,k", [(1000, 1024, 512), (3000, 4100, 528), (4097, 2050, 4096), (8192, 8192, 64), (2049, 6145, 100), (70, 5000, 8192), (200, 72, 20000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_large(m, n, k, dtype):
    q, s, w, t, b = case(m, n, k, dtype, seed=k)
    check(int8_linear(q, s, w, t, b, dtype=dtype), q, s, w, t, b)


@pytest.mark.parametrize("m,n,k", [(1272, 5069, 12532), (1500, 5000, 16000), (9584, 880, 13746)])
def test_large_tiles_with_split_sums(m, n, k):
    q, s, w, t, b = case(m, n, k, torch.float32, seed=k)
    check(int8_linear(q, s, w, t, b, "silu"), q, s, w, t, b, "silu")


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(7, 90, 300), (150, 90, 300), (150, 136, 6000)])
def test_activations(m, n, k, dtype, name):
    q, s, w, t, b = case(m, n, k, torch.float32, seed=9)
    b = b * 3
    check(int8_linear(q, s, w, t, b, activation=name, dtype=dtype), q, s, w, t, b, name)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_longest_sums(m):
    """131071 products of -128 and -128 stay inside 32 bits."""
    k = 131071
    q, w = torch.full((m, k), -128, dtype=torch.int8, device=DEV), torch.full((20, k), -128, dtype=torch.int8, device=DEV)
    s, t = torch.ones(m, device=DEV), torch.ones(20, device=DEV)
    assert torch.equal(int8_linear(q, s, w, t, dtype=torch.float32), torch.full((m, 20), float(k * 2**14), device=DEV))
    with pytest.raises(AssertionError, match="131071"):
        int8_linear(torch.zeros(m, k + 1, dtype=torch.int8, device=DEV), s, torch.zeros(20, k + 1, dtype=torch.int8, device=DEV), t)


@pytest.mark.parametrize("m", [5, 200, 600])
def test_strides_and_alignment(m):
    """Columns of wider buffers on and off 16-byte boundaries, more dimensions, expanded rows, strided scales."""
    g = torch.Generator(device=DEV).manual_seed(m)
    base, wbase = rows8(g, m, 2000), rows8(g, 300, 1900)
    for k0, width in ((16, 1024), (3, 1024), (0, 777), (5, 48)):
        q, w = base[:, k0 : k0 + width], wbase[:, k0 : k0 + width]
        s, t, b = (torch.rand(i, 2, generator=g, device=DEV)[:, 0] for i in (m, 300, 300))
        t = t * 1e-3
        y = int8_linear(q, s, w, t, b, activation="silu")
        assert torch.equal(y, int8_linear(q.contiguous(), s.contiguous(), w.contiguous(), t.contiguous(), b.contiguous(), activation="silu"))
        check(y, q, s, w, t, b, "silu")
    q = base[:, :512].unflatten(0, (m // 5, 5))
    s = torch.rand(m // 5, 5, generator=g, device=DEV)
    y = int8_linear(q, s, wbase[:, :512], t)
    assert y.shape == (m // 5, 5, 300) and torch.equal(y.flatten(0, 1), int8_linear(base[:, :512], s.flatten(), wbase[:, :512], t))
    one = base[:1, :512].expand(m, 512)
    assert torch.equal(int8_linear(one, s.flatten(), wbase[:, :512].t().contiguous().t(), t), int8_linear(one.contiguous(), s.flatten(), wbase[:, :512], t))
    # a single row as a vector
    assert torch.equal(int8_linear(base[0, :512], s[0, 0], wbase[:, :512], t), int8_linear(base[:1, :512], s[0, :1], wbase[:, :512], t)[0])


def test_offsets_beyond_32_bits():
    g = torch.Generator(device=DEV).manual_seed(1)
    rows, stride, k = 2100, 2**21, 192
    base = torch.empty(rows, stride, dtype=torch.int8, device=DEV)
    q = base[:, 16 : 16 + k]
    q.copy_(rows8(g, rows, k))
    w, s, t = rows8(g, 48, k), torch.rand(rows, device=DEV), torch.rand(48, device=DEV)
    assert torch.equal(int8_linear(q, s, w, t), int8_linear(q.contiguous(), s, w, t))
    few = base[2050:2060, 16 : 16 + k]
    assert torch.equal(int8_linear(few, s[:10], w, t), int8_linear(few.contiguous(), s[:10], w, t))
    weight = base[:, 16 : 16 + k]
    a = rows8(g, 300, k)
    assert torch.equal(int8_linear(a, s[:300], weight, s), int8_linear(a, s[:300], weight.contiguous(), s))
    assert torch.equal(int8_linear(a[:3], s[:3], weight, s), int8_linear(a[:3], s[:3], weight.contiguous(), s))
    del base, q, few, weight
    m, n = 70000, 32768  # more results than 2^31
    q, w = rows8(g, m, 64), rows8(g, n, 64)
    s, t = torch.rand(m, device=DEV), torch.rand(n, device=DEV)
    y = int8_linear(q, s, w, t)
    for at in (0, 65535, 65536, m - 100):
        check(y[at : at + 100], q[at : at + 100], s[at : at + 100], w, t, None)


@pytest.mark.parametrize("m", [3, 100])
def test_rows_without_a_form(m):
    q, s, w, t, _ = case(m, 50, 70)
    s[1], s[2] = float("nan"), 0.0
    y = int8_linear(q, s, w, t)
    assert torch.isnan(y[1]).all() and not y[2].any() and torch.isfinite(y[0]).all()
    for name in ACTS:
        assert torch.isnan(int8_linear(q, s, w, t, activation=name)[1]).all(), name


def test_no_rows():
    q, s, w, t, _ = case(4, 50, 70)
    assert int8_linear(q[:0], s[:0], w, t).shape == (0, 50)
    a, b = quantize_rows(torch.empty(0, 70, device=DEV))
    assert a.shape == (0, 70) and b.shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 7, 8, 9, 500, 512, 513, 2048, 2050, 8192, 8200, 32768, 32770, 50001])
def test_quantize_rows(width, dtype):
    x = torch.randn(21, width, device=DEV).to(dtype)
    x[0] = 0
    q, s = quantize_rows(x)
    a = x.double().abs().amax(-1)
    assert (s.double() - a / 127).abs().max() <= U * a.max() / 127
    # a quotient is off by 2 U of at most 127 when it is rounded
    assert ((s.double()[:, None] * q - x.double()).abs() <= (0.5 + 127 * 4 * U) * s.double()[:, None]).all()
    assert not q[0].any() and s[0] == 0 and int(q[1:].abs().amax(-1).min()) == 127
    x[3, width - 1], x[4, 0], x[5, 0] = float("nan"), float("inf"), -float("inf")
    q, s = quantize_rows(x)
    assert torch.isnan(s[3:6]).all() and not q[3:6].any() and torch.isfinite(s[6:]).all()
    # rows of a wider buffer, off its boundaries
    wide = torch.randn(9, width + 13, device=DEV).to(dtype)
    assert all(torch.equal(a, b) for a, b in zip(quantize_rows(wide[:, 5 : 5 + width]), quantize_rows(wide[:, 5 : 5 + width].contiguous())))


def test_quantize_more_rows_than_one_launch_takes():
    x = torch.randn(2**21 + 9, 8, device=DEV)
    q, s = quantize_rows(x)
    for part in (slice(0, 50), slice(2**21 - 20, x.shape[0])):
        assert all(torch.equal(a, b) for a, b in zip(quantize_rows(x[part]), (q[part], s[part])))


def test_another_stream_and_captured():
    q, s, w, t, b = case(200, 264, 8192, torch.float32)
    few = q[:3].contiguous()
    x = torch.randn(200, 8192, device=DEV)
    want = int8_linear(q, s, w, t, b)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        assert torch.equal(int8_linear(q, s, w, t, b), want)
    torch.cuda.current_stream().wait_stream(st)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed in turn, share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, c = quantize_rows(x)
            outs.append((int8_linear(a, c, w, t, b), int8_linear(few, s[:3], w, t, b)))
        graphs.append(graph)
    for turn in range(3):
        x.normal_()
        few.copy_(rows8(torch.Generator(device=DEV).manual_seed(turn), 3, 8192))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for one, two in outs:
            assert torch.equal(one, int8_linear(*quantize_rows(x), w, t, b)) and torch.equal(two, int8_linear(few, s[:3], w, t, b))


def test_module():
    lin = torch.nn.Linear(300, 70).to(DEV)
    m = Int8Linear.from_linear(lin, activation="gelu")
    x = torch.randn(4, 30, 300, device=DEV).bfloat16()
    y = m(x)
    q, s = quantize_rows(x)
    assert y.dtype == torch.bfloat16 and torch.equal(y, m(q, s))
    check(y.flatten(0, 1), q.flatten(0, 1), s.flatten(), m.weight, m.weight_scale, m.bias, "gelu")
    full = torch.nn.functional.gelu(lin(x.float()))
    assert (y.float() - full).norm() < 0.03 * full.norm()
    again = Int8Linear.from_linear(torch.nn.Linear(300, 70).to(DEV), activation="gelu")
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(x), y)
    half = again.half()
    assert half.weight_scale.dtype == torch.float32 and torch.equal(half.weight_scale, m.weight_scale) and half(x).shape == y.shape


def test_gradients_are_refused():
    q, s, w, t, b = case(4, 50, 70, torch.float32)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_linear(q, s, w, t, b.requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize_rows(torch.randn(3, 4, device=DEV, requires_grad=True))
    with torch.no_grad():
        int8_linear(q, s, w, t, b)
