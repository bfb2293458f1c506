"""GPU: the wide layers through the C interface leave everything around their outputs as it was, rows of a wider buffer and memory in front of and
behind it, and give the results of the Python functions there."""
import ctypes

import pytest
import torch

from triton_helpers_amd import _lib
from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_amd.layers.int8_linear import int8_linear, quantize_rows
from triton_helpers_amd.layers.rms_norm import rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
AROUND = 256
MARK = 77


class Guarded:
    """`rows` rows of `width` values, `stride` apart, with marks in between and AROUND values of them on either side."""

    def __init__(self, rows, width, dtype, stride=None):
        self.rows, self.width, self.stride = rows, width, stride or width
        self.all = torch.full((2 * AROUND + rows * self.stride,), MARK, device=DEV, dtype=dtype)
        self.p = self.all.data_ptr() + AROUND * self.all.element_size()

    def values(self):
        body = self.all[AROUND : AROUND + self.rows * self.stride].view(self.rows, self.stride)
        outside = torch.cat([self.all[:AROUND], self.all[AROUND + self.rows * self.stride :], body[:, self.width :].reshape(-1)])
        assert (outside == MARK).all(), "written outside of the output"
        return body[:, : self.width]


def p(t):
    return None if t is None else t.p if isinstance(t, Guarded) else t.data_ptr()


def work(size):
    g = Guarded(1, max(int(size), 1), torch.uint8)  # 256 bytes in front of a 512-byte boundary: on a 16-byte boundary
    return g, p(g) if size else None, int(size)


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def called(rc):
    assert rc == 0, _lib.load().nf_last_error()


@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 100), (70, 777), (33, 1030), (9, 4099), (2, 33001)])
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, _lib.NF_BF16), (torch.float32, _lib.NF_F32)])
def test_norm(m, k, dtype, code):
    lib = _lib.load()
    x, r, dy, ds = (torch.randn(m, k, device=DEV).to(dtype) for _ in range(4))
    w = torch.randn(k, device=DEV).to(dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    y0, s0 = rms_norm(leaves[0], leaves[1], 1e-6, leaves[2])
    torch.autograd.backward((y0, s0), (dy, ds))
    y, s, rstd, dx, dr, dw = (Guarded(m, k, dtype), Guarded(m, k, dtype), Guarded(1, m, torch.float32), Guarded(m, k, dtype), Guarded(m, k, dtype), Guarded(1, k, dtype))
    called(lib.nf_rms_norm_fwd(p(x), k, code, p(r), k, code, p(w), code, p(y), None, p(s), p(rstd), m, k, 1e-6, stream()))
    g, at, size = work(lib.nf_rms_norm_bwd_workspace_bytes(m, k))
    called(lib.nf_rms_norm_bwd(p(dy), k, code, p(ds), k, p(s), k, code, p(rstd), p(w), code, p(dx), p(dr), p(dw), m, k, at, size, stream()))
    q, scale = Guarded(m, k, torch.int8), Guarded(1, m, torch.float32)
    called(lib.nf_quantize_rows(p(x), k, code, p(q), p(scale), None, k, 0, m, k, stream()))
    for a, b in ((y, y0), (s, s0), (dx, leaves[0].grad), (dr, leaves[2].grad), (dw, leaves[1].grad[None]), (q, quantize_rows(x)[0]), (scale, quantize_rows(x)[1][None])):
        assert torch.equal(a.values(), b)
    rstd.values(), g.values()


@pytest.mark.parametrize("m,n,k,stride", [(1, 1, 1, 3), (17, 33, 100, 40), (64, 5, 4097, 5), (65, 129, 100, 131), (200, 72, 20000, 80), (300, 1001, 96, 1008), (1272, 2569, 6266, 2570)])
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, _lib.NF_BF16), (torch.float32, _lib.NF_F32)])
def test_int8_product(m, n, k, stride, dtype, code):
    lib = _lib.load()
    q, w = (torch.randint(-127, 128, (rows, k), device=DEV, dtype=torch.int8) for rows in (m, n))
    s, t = torch.rand(m, device=DEV), torch.rand(n, device=DEV)
    y = Guarded(m, n, dtype, stride)
    g, at, size = work(lib.nf_int8_linear_workspace_bytes(p(q), k, p(w), k, m, n, k))
    called(lib.nf_int8_linear(p(q), k, p(s), p(w), k, p(t), None, 0, p(y), stride, code, m, n, k, 0, at, size, stream()))
    assert torch.equal(y.values(), int8_linear(q, s, w, t, dtype=dtype))
    g.values()


@pytest.mark.parametrize("m,n,k,stride", [(1, 1, 1, 2), (31, 33, 100, 35), (129, 257, 130, 260), (500, 96, 72, 104), (2051, 64, 120, 72), (13001, 256, 248, 264), (1003, 333, 777, 333),
                                          (3000, 1500, 1704, 1512)])
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, _lib.NF_BF16), (torch.float16, _lib.NF_F16)])
def test_checkpointed_linear(m, n, k, stride, dtype, code):
    lib = _lib.load()
    x, w, b, dy = (torch.randn(*shape, device=DEV).to(dtype) for shape in ((m, k), (n, k), (n,), (m, n)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y0 = checkpointed_linear(*leaves, "gelu")
    y0.backward(dy)
    y, q, scale = Guarded(m, n, dtype, stride), Guarded(m, k, torch.int8), Guarded(1, m, torch.float32)
    act = _lib.NF_ACT["gelu"]
    g, at, size = work(lib.nf_linear_keep_fwd_workspace_bytes(p(x), k, p(w), k, m, n, k, act))
    called(lib.nf_linear_keep_fwd(p(x), k, code, p(w), k, p(b), code, p(y), stride, p(q), p(scale), m, n, k, act, at, size, stream()))
    dx, dw, db = Guarded(m, k, dtype), Guarded(n, k, dtype), Guarded(1, n, dtype)
    h, to, size = work(lib.nf_linear_keep_bwd_workspace_bytes(p(dy), n, p(w), k, m, n, k, 1, 1, 1))
    called(lib.nf_linear_keep_bwd(p(dy), n, code, p(q), p(scale), p(w), k, p(dx), p(dw), code, p(db), code, m, n, k, act, to, size, stream()))
    for a, c in ((y, y0), (q, quantize_rows(x)[0]), (scale, quantize_rows(x)[1][None]), (dx, leaves[0].grad), (dw, leaves[1].grad), (db, leaves[2].grad[None])):
        assert torch.equal(a.values(), c)
    g.values(), h.values()
