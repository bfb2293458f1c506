"""GPU: the wide layers at the ends of their types' ranges."""
import pytest
import torch

from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear

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
