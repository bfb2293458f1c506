"""GPU: the wide layers at the ends of their types' ranges."""
import pytest
import torch

from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_amd.layers.wide_mlp import WideMLP

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gradients(x, w, dy, name):
    xl, wl = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    checkpointed_linear(xl, wl, None, name).backward(dy)
    return xl.grad, wl.grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(300, 72, 64), (4096, 64, 64), (4096, 136, 256), (13000, 256, 256)])
@pytest.mark.parametrize("name", ["none", "relu", "relu2", "silu", "gelu"])
def test_masked_rows_of_the_lowest_value(m, n, k, dtype, name):
    """Rows that a mask filled with the type's lowest value and whose upstream gradient is zero: they add nothing, exactly as rows of zeros do."""
    g = torch.Generator(device=DEV).manual_seed(k)
    x, w, dy = (torch.randn(*s, generator=g, device=DEV).to(dtype) for s in ((m, k), (n, k), (m, n)))
    masked = torch.tensor([0, 5, 31, 32, m - 1], device=DEV)
    dy[masked] = 0
    x[masked] = 0
    want = gradients(x, w, dy, name)
    x[masked] = torch.finfo(dtype).min
    x[5, 1:] = 1.0  # a single one in its row
    got = gradients(x, w, dy, name)
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0], want[0])
    # values whose gradient is not zero: the 8-bit form of a row of lowest values is the row itself
    x[masked], dy[masked] = 0, 0
    x[7] = torch.finfo(dtype).min
    dy[:] = 0
    dy[7, :3] = 2.0**-10
    dx, dw = gradients(x, w, dy, name)
    if name == "none":
        assert torch.equal(dw[:3].double(), torch.full((3, k), torch.finfo(dtype).min * 2.0**-10, dtype=torch.float64, device=DEV).to(dtype).double())
    else:  # every gate is closed there
        assert not dw.any() and not dx[7].any()
    assert not dw[3:].any()


def test_more_workgroups_than_one_row_of_a_grid_copies():
    """Copies of more than 2^30 pieces of 16 bytes go to a grid of two dimensions, whose last workgroups have nothing to do.  dx alone, from a copied dy; dW, from act(x^) written out.
    Whole numbers, and only the last rows have gradients: exact."""
    m, tail = 2**23 + 3, 45
    for n, k, need in ((1030, 8, "dx"), (8, 1030, "dw")):
        g = torch.Generator(device=DEV).manual_seed(n)
        w = torch.randint(-2, 3, (n, k), generator=g, device=DEV).bfloat16()
        x, dy = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV), torch.zeros(m, n, dtype=torch.bfloat16, device=DEV)
        x[-tail:] = torch.randint(-3, 4, (tail, k), generator=g, device=DEV).bfloat16()
        x[-tail:, 1] = 127
        dy[-tail:] = torch.randint(-2, 3, (tail, n), generator=g, device=DEV).bfloat16()
        (x if need == "dx" else w).requires_grad_()
        y = checkpointed_linear(x, w)
        y.backward(dy)
        if need == "dx":
            want = (dy[-tail:].double() @ w.double()).bfloat16()
            assert torch.equal(x.grad[-tail:], want) and not x.grad[:-tail].any() and w.grad is None
        else:
            assert torch.equal(w.grad, (dy[-tail:].double().t() @ x[-tail:].double()).bfloat16()) and x.grad is None
        assert torch.equal(y[-tail:].detach(), (x[-tail:].detach().double() @ w.detach().double().t()).bfloat16()) and not y[:-tail].any()
        del x, dy, w, y


@pytest.mark.parametrize("dtype,wide", [(torch.float16, False), (torch.float16, True), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, True)])
def test_blocks_in_8_bits_follow_each_other(dtype, wide):
    """The 8-bit forms of a network's blocks, each of its own type, with a residual stream of that type or of float32."""
    torch.manual_seed(0)
    first, second = (WideMLP(72, 136).to(DEV, dtype) for _ in range(2))
    rows = torch.bfloat16 if dtype == torch.float32 else dtype
    x, r = torch.randn(5, 72, device=DEV).to(rows), torch.randn(5, 72, device=DEV).to(torch.float32 if wide else rows)
    out, stream = first.to_int8()(x, r)
    assert out.dtype == rows and stream.dtype == r.dtype
    out, stream = second.to_int8()(out, stream)
    assert out.dtype == rows and stream.dtype == r.dtype and torch.isfinite(out).all()
    want = [m.to_int8(rows) for m in (first, second)]
    want = want[1](*want[0](x, r))
    assert torch.equal(out, want[0]) and torch.equal(stream, want[1])
    assert first.to_int8(torch.float32)(x, r)[0].dtype == torch.float32


@pytest.mark.parametrize("m", [40, 4096])
def test_relu2_at_the_end_of_float16(m):
    """255.875^2 = 65472.0156 rounds to 65472, the last value but one; 256^2 leaves the type, and its row and column show it.  bfloat16 goes on."""
    n, k = 24, 64
    w = torch.full((n, k), 2.0**-10, device=DEV)
    x = torch.zeros(m, k, device=DEV)
    x[1, 3], x[2, 5], x[3] = 255.875, 256.0, -300.0
    dy = torch.zeros(m, n, device=DEV)
    dy[0], dy[1, 0], dy[2, 1] = 1.0, 2.0**-10, 2.0**-10
    xl, wl = x.half().requires_grad_(), w.half().requires_grad_()
    y = checkpointed_linear(xl, wl, None, "relu2")
    y.backward(dy.half())
    assert torch.equal(y[1].double(), torch.full((n,), 65472 / 1024, dtype=torch.float64, device=DEV).half().double())
    assert torch.isinf(y[2]).all() and not y[0].any() and not y[3:].any()
    # the 8-bit row of a single value is that value to float32's rounding (a / 127 * 127): the same 65472
    assert torch.equal(wl.grad[0, 3], torch.tensor(65472 / 1024, device=DEV).half())
    assert torch.isinf(wl.grad[1, 5]) and torch.isnan(wl.grad[2:, 5]).all()
    rest = torch.ones(k, dtype=torch.bool, device=DEV)
    rest[5] = False
    assert torch.isfinite(wl.grad[:, rest]).all() and torch.isfinite(xl.grad).all()
    xl, wl = x.bfloat16().requires_grad_(), w.bfloat16().requires_grad_()
    y = checkpointed_linear(xl, wl, None, "relu2")
    y.backward(dy.bfloat16())
    assert torch.equal(y[2].double(), torch.full((n,), 64.0, dtype=torch.float64, device=DEV)) and torch.isfinite(wl.grad).all()
