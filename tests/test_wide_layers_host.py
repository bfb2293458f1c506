"""CPU-only: what the wide layers' entry points and functions refuse, before anything is launched."""
import ctypes

import pytest
import torch

from triton_helpers_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libnf_cdna4.so not built")
BF, F16, F32 = _lib.NF_BF16, _lib.NF_F16, _lib.NF_F32


def refused(rc, code, word):
    message = _lib.load().nf_last_error()
    assert rc == code and word in message, (rc, message)


def test_norm_entry_points():
    lib = _lib.load()
    eps = ctypes.c_float(1e-6)

    def fwd(x=16, xs=64, dt=BF, r=None, rs=64, rdt=BF, w=None, wdt=F32, y=16, rows=4, width=64, eps=eps, h=None):
        return lib.nf_rms_norm_fwd(x, xs, dt, r, rs, rdt, w, wdt, y, None, h, None, rows, width, eps, None)

    refused(fwd(dt=7), -1, b"dtype")
    refused(fwd(rdt=F16), -2, b"residual")
    refused(fwd(rows=-1), -1, b"rows")
    refused(fwd(rows=2**31), -1, b"rows")
    refused(fwd(width=0), -1, b"width")
    refused(fwd(width=2**30 + 1), -1, b"width")
    refused(fwd(eps=ctypes.c_float(-1.0)), -1, b"eps")
    refused(fwd(x=None), -1, b"NULL")
    refused(fwd(xs=63), -1, b"stride")
    refused(fwd(r=16, rs=8), -1, b"stride")
    refused(fwd(h=16), -1, b"residual")
    assert fwd(x=None, y=None, rows=0) == 0

    def bwd(dy=16, dt=BF, h=16, hs=64, hdt=BF, rstd=16, w=16, dw=None, rows=4, width=64, ws=None, n=0):
        return lib.nf_rms_norm_bwd(dy, 64, dt, None, 64, h, hs, hdt, rstd, w, F32, 16, None, dw, rows, width, ws, n, None)

    refused(bwd(hdt=F16), -2, b"residual")
    refused(bwd(dw=16), -1, b"workspace")
    refused(bwd(dw=16, ws=16, n=lib.nf_rms_norm_bwd_workspace_bytes(4, 64) - 1), -1, b"workspace")
    refused(bwd(dw=16, w=None), -1, b"weight")
    refused(bwd(dw=16, rows=0), -1, b"no rows")
    refused(bwd(rstd=None), -1, b"NULL")
    refused(bwd(hs=1), -1, b"stride")
    assert bwd(rows=0) == 0
    assert lib.nf_rms_norm_bwd_workspace_bytes(0, 64) == 0
    # a slot of partial sums for each group of threads: whole workgroups of four waves up to 2048 values, one workgroup above
    assert lib.nf_rms_norm_bwd_workspace_bytes(5, 64) == 8 * 64 * 4
    assert lib.nf_rms_norm_bwd_workspace_bytes(5, 4096) == 5 * 4096 * 4


def test_norm_arguments():
    from triton_helpers_amd.layers.rms_norm import rms_norm, rms_norm_int8

    x = torch.randn(4, 64)
    for f in (rms_norm, rms_norm_int8):
        with pytest.raises(AssertionError, match="GPU"):
            f(x, torch.ones(64))
        with pytest.raises(AssertionError, match="weight"):
            f(x, torch.ones(63))
        with pytest.raises(AssertionError, match="residual"):
            f(x, None, residual=torch.randn(4, 63))
        with pytest.raises(AssertionError, match="residual"):
            f(x, None, residual=torch.randn(4, 64).half())
        with pytest.raises(AssertionError, match="eps"):
            f(x, None, eps=-1.0)
        with pytest.raises(AssertionError, match="last dimension"):
            f(torch.randn(4, 0), None)
        with pytest.raises(NotImplementedError, match="float64"):
            f(x.double(), None)
        with pytest.raises(NotImplementedError, match="weight"):
            f(x, torch.ones(64, dtype=torch.int32))
