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
    refused(fwd(width=2**26 + 1), -1, b"width")
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
    # a slot of partial sums for each workgroup: of four rows' waves up to 2048 values, of one row above
    assert lib.nf_rms_norm_bwd_workspace_bytes(5, 64) == 2 * 64 * 4
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


def test_product_entry_points():
    lib = _lib.load()

    def product(q=16, qs=64, s=16, w=16, ws=64, t=16, y=16, ys=48, ydt=BF, bdt=F32, rows=4, n=48, k=64, act=0, work=None, size=0):
        return lib.nf_int8_linear(q, qs, s, w, ws, t, None, bdt, y, ys, ydt, rows, n, k, act, work, size, None)

    refused(product(ydt=9), -1, b"dtype")
    refused(product(act=5), -1, b"activation")
    refused(product(rows=-1), -1, b"rows")
    refused(product(n=0), -1, b"n=0")
    refused(product(k=0), -1, b"k=0")
    refused(product(n=2**26 + 1, ys=2**27), -1, b"n=")
    refused(product(rows=2**31 - 1, n=2**20, ys=2**20, work=16, size=2**62), -2, b"more tiles")
    refused(product(k=131072, qs=131072, ws=131072), -2, b"131071")
    refused(product(s=None), -1, b"NULL")
    refused(product(qs=63), -1, b"stride")
    refused(product(ws=63), -1, b"stride")
    refused(product(ys=47), -1, b"stride")
    assert product(rows=0, q=None) == 0
    # few rows, and whole pieces in one run of tiles, need nothing; rows off 16-byte boundaries a copy; a split sum its parts
    size = lib.nf_int8_linear_workspace_bytes
    assert size(16, 64, 16, 64, 64, 48, 64) == 0 and size(1, 63, 3, 63, 64, 48, 63) == 0
    assert size(16, 64, 16, 64, 65, 48, 64) == 0
    assert size(1, 64, 16, 64, 65, 48, 64) >= 65 * 64 and size(16, 64, 17, 64, 65, 48, 64) >= 48 * 64
    assert size(16, 63, 16, 64, 65, 48, 63) >= (65 + 48) * 64
    need = size(16, 8192, 16, 8192, 65, 48, 8192)
    assert need >= 2 * 65 * 48 * 4
    refused(product(qs=8192, ws=8192, rows=65, k=8192, work=16, size=need - 1), -1, b"workspace")
    refused(product(qs=8192, ws=8192, rows=65, k=8192, work=24, size=need), -1, b"workspace")

    def quantize(x=16, xs=64, dt=BF, q=16, s=16, h=None, hs=64, act=0, rows=4, width=64):
        return lib.nf_quantize_rows(x, xs, dt, q, s, h, hs, act, rows, width, None)

    refused(quantize(dt=3), -1, b"dtype")
    refused(quantize(act=-1), -1, b"activation")
    refused(quantize(rows=2**31), -1, b"rows")
    refused(quantize(width=0), -1, b"width")
    refused(quantize(h=16, hs=65), -1, b"h_stride")
    refused(quantize(q=None), -1, b"NULL")
    refused(quantize(xs=63), -1, b"stride")
    assert quantize(rows=0) == 0


def test_product_arguments():
    from triton_helpers_amd.layers.int8_linear import int8_linear, quantize_rows

    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    w, t = torch.zeros(48, 64, dtype=torch.int8), torch.ones(48)
    with pytest.raises(AssertionError, match="GPU"):
        int8_linear(q, s, w, t)
    for bad, word in (((q.float(), s, w, t), "q must be int8"), ((q, s.half(), w, t), "scale must be float32"), ((q, s, w[:, :63], t), "w must be"),
                      ((q, s[:3], w, t), "scale must have"), ((q, s, w, t[:3]), "w_scale must be"), ((q, s, w, t, torch.ones(47)), "bias must be"),
                      ((q, s, w, t, None, "tanh"), "activation"), ((q, s, w.int(), t), "w must be int8"), ((q[:, :0], s, w[:, :0], t), "last dimension")):
        with pytest.raises(AssertionError, match=word):
            int8_linear(*bad)
    with pytest.raises(NotImplementedError):
        int8_linear(q, s, w, t, dtype=torch.float64)
    with pytest.raises(NotImplementedError):
        int8_linear(q, s, w, t, torch.ones(48, dtype=torch.float64))
    with pytest.raises(AssertionError, match="GPU"):
        quantize_rows(torch.randn(4, 64))
    with pytest.raises(NotImplementedError, match="int8"):
        quantize_rows(q)
    with pytest.raises(AssertionError, match="last dimension"):
        quantize_rows(torch.randn(4, 0))


def test_keep_entry_points():
    lib = _lib.load()

    def fwd(x=16, xs=64, dt=BF, w=16, ws=64, bdt=F32, y=16, ys=48, q=16, s=16, rows=4, n=48, k=64, act=0, work=None, size=0):
        return lib.nf_linear_keep_fwd(x, xs, dt, w, ws, None, bdt, y, ys, q, s, rows, n, k, act, work, size, None)

    refused(fwd(dt=F32), -2, b"float16 or bfloat16")
    refused(fwd(bdt=5), -1, b"dtype")
    refused(fwd(act=7), -1, b"activation")
    for bad in ({"rows": 2**30}, {"rows": -1}, {"n": 0}, {"k": 0}, {"k": 2**20 + 1}, {"n": 2**20 + 1}, {"k": 2**22}):
        refused(fwd(**bad), -1, b"rows")
    refused(fwd(w=None), -1, b"NULL")
    refused(fwd(s=None), -1, b"NULL")
    refused(fwd(xs=63), -1, b"stride")
    refused(fwd(ws=63), -1, b"stride")
    refused(fwd(ys=47), -1, b"stride")
    refused(fwd(act=1), -1, b"workspace")
    assert fwd(rows=0, x=None) == 0
    size = lib.nf_linear_keep_fwd_workspace_bytes
    assert size(16, 64, 16, 64, 4, 48, 64, 0) == 0
    assert size(16, 64, 16, 64, 4, 48, 64, 1) >= 4 * 64 * 2
    assert size(18, 64, 16, 64, 4, 48, 64, 0) >= 4 * 64 * 2 and size(16, 64, 18, 64, 4, 48, 64, 0) >= 48 * 64 * 2

    def bwd(dy=16, ds=48, dt=BF, q=16, s=16, w=16, ws=64, dx=16, dw=16, wdt=BF, db=16, bdt=F32, rows=4, n=48, k=64, act=0, work=None, size=0):
        return lib.nf_linear_keep_bwd(dy, ds, dt, q, s, w, ws, dx, dw, wdt, db, bdt, rows, n, k, act, work, size, None)

    refused(bwd(dt=F32), -2, b"float16 or bfloat16")
    refused(bwd(wdt=F16), -2, b"weight's gradient")
    refused(bwd(act=-1), -1, b"activation")
    refused(bwd(rows=0), -1, b"rows")
    refused(bwd(dy=None), -1, b"NULL")
    refused(bwd(q=None), -1, b"NULL")
    refused(bwd(q=None, dw=None, act=2), -1, b"NULL")
    refused(bwd(w=None), -1, b"NULL")
    refused(bwd(ds=47), -1, b"stride")
    refused(bwd(ws=1), -1, b"stride")
    assert lib.nf_linear_keep_bwd_workspace_bytes(16, 48, 16, 64, 4, 48, 64, 0, 0, 1) >= 48 * 4
    need = lib.nf_linear_keep_bwd_workspace_bytes(16, 48, 16, 64, 4, 48, 64, 1, 1, 1)
    assert need >= 4 * 64 * 2
    refused(bwd(work=16, size=need - 1), -1, b"workspace")
    refused(bwd(work=8, size=need), -1, b"workspace")
    assert bwd(dx=None, dw=None, db=None) == 0
    # where a workgroup keeps the weights the results want whole pieces
    refused(fwd(rows=4096, y=24), -3, b"boundaries")
    refused(fwd(rows=4096, q=24), -3, b"boundaries")
    refused(fwd(rows=4096, ys=52), -3, b"boundaries")
    big = lib.nf_linear_keep_bwd_workspace_bytes(16, 48, 16, 64, 4096, 48, 64, 1, 1, 1)
    assert big >= 128 * 48 * (64 + 1) * 4
    refused(bwd(rows=4096, dx=24, work=16, size=big), -3, b"boundaries")
    refused(bwd(rows=4096, work=16, size=big - 1), -1, b"workspace")
    refused(bwd(k=2**20 + 8, ws=2**20 + 8, work=16, size=2**62), -1, b"2^20")
    refused(bwd(rows=2**29, k=2**20, ws=2**20, n=264, ds=264, work=16, size=2**62), -2, b"more tiles")


def test_keep_arguments():
    from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear

    x, w, b = torch.randn(4, 64).bfloat16(), torch.randn(48, 64).bfloat16(), torch.randn(48)
    with pytest.raises(AssertionError, match="GPU"):
        checkpointed_linear(x, w, b)
    for bad, word in (((x, w[:, :63], b), "w must be"), ((x, w, b[:3]), "b must be"), ((x, w, b, "tanh"), "activation"), ((x[:, :0], w[:, :0], b), "last dimension")):
        with pytest.raises(AssertionError, match=word):
            checkpointed_linear(*bad)
    for bad in ((x.float(), w.float(), b), (x, w.half(), b), (x, w, b.double())):
        with pytest.raises(NotImplementedError):
            checkpointed_linear(*bad)


def test_alias_package_and_names():
    """The wide layers resolve through ``triton_helpers.layers`` as the others do."""
    import triton_helpers.layers.checkpointed_linear as c
    import triton_helpers.layers.int8_linear as i
    import triton_helpers.layers.rms_norm as r
    import triton_helpers.layers.wide_mlp as w

    from triton_helpers_amd.layers import checkpointed_linear, int8_linear, rms_norm, wide_mlp

    for alias, own in ((c, checkpointed_linear), (i, int8_linear), (r, rms_norm), (w, wide_mlp)):
        assert sorted(alias.__all__) == sorted(own.__all__)
        assert all(getattr(alias, n) is getattr(own, n) for n in own.__all__)
    m = w.WideMLP(96, 384)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "norm.weight": (96,), "up.weight": (384, 96), "up.bias": (384,), "down.weight": (96, 384), "down.bias": (96,)}
    with pytest.raises(AssertionError, match="GPU"):
        m.to_int8()


def test_leaves_on_the_host_with_a_graph_are_refused_as_such():
    """Arguments are checked for their device, whatever else holds them."""
    from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear
    from triton_helpers_amd.layers.rms_norm import rms_norm

    x, w = torch.randn(4, 8).bfloat16().requires_grad_(), torch.ones(8).requires_grad_()
    alive = x.float() * w
    with pytest.raises(AssertionError, match="GPU"):
        rms_norm(x, w)
    with pytest.raises(AssertionError, match="GPU"):
        checkpointed_linear(x, torch.randn(4, 8).bfloat16().requires_grad_(), w[:4])
    del alive
