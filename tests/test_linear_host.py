"""What the mixed-precision linear-layer and gradient-list routines refuse. The checks come before the GPU is
touched, so they run without one; the addresses here are never read."""
import ctypes as C

import pytest

A, B, CC, D, P, S = (0x10000 * i for i in range(1, 7))


def _call(pl, **kw):
    a = dict(dev=0, type=pl.BF16, TransA="T", TransB="N", M=64, N=32, K=16, alpha=1.0, A=A, ldA=16, B=B, ldB=16, beta=1.0,
             Cm=CC, ldC=64, D=D, ldD=64)
    a.update(kw)
    pl.tile_gemm_act(**a)


def _grad(pl, **kw):
    a = dict(dev=0, type=pl.BF16, TransA="T", TransB="N", M=64, N=32, K=16, alpha=1.0, A=A, ldA=16, B=B, ldB=16,
             act=pl.ACT_GELU, pre=P, ldPre=64, dD=D, lddD=64, dA=0x90000, lddA=16, dB=0xA0000, lddB=16, dbias=0xB0000,
             scratch=S, scratch_bytes=1 << 30)
    a.update(kw)
    pl.tile_gemm_act_grad(**a)


def _refused(pl, f, code=None, **kw):
    with pytest.raises(pl.ParaliaError) as e:
        f(pl, **kw)
    assert e.value.code == (pl.ERR_INVALID_ARG if code is None else code), str(e.value)


@pytest.mark.parametrize("kw", [
    dict(type=7), dict(type=-1), dict(TransA="X"), dict(TransB="?"), dict(M=-1), dict(N=-1), dict(K=-1), dict(M=1 << 31),
    dict(K=1 << 40, ldA=1 << 40, ldB=1 << 40), dict(act=5), dict(act=-1), dict(ldA=15), dict(ldB=15), dict(TransA="N", ldA=63), dict(TransB="T", ldB=31),
    dict(ldC=63), dict(ldD=63), dict(pre=P, ldPre=63), dict(A=0), dict(B=0), dict(Cm=0), dict(D=0), dict(A=A + 1),
    dict(D=D + 1), dict(bias=P + 1), dict(Cm=CC + 1), dict(pre=P + 1, ldPre=64), dict(D=A), dict(D=B), dict(pre=D, ldPre=64),
    dict(pre=A, ldPre=64), dict(Cm=D, ldC=72), dict(bias=D), dict(alpha=float("nan")), dict(beta=float("inf")),
])
def test_forward_refusals(pl, kw):
    _refused(pl, _call, **kw)


def test_fp32_is_unsupported(pl):
    _refused(pl, _call, code=pl.ERR_UNSUPPORTED, type=pl.F32)
    _refused(pl, _grad, code=pl.ERR_UNSUPPORTED, type=pl.F32)


@pytest.mark.parametrize("kw", [
    dict(type=9), dict(TransA="Q"), dict(M=-5), dict(act=9), dict(ldA=1), dict(ldPre=63), dict(lddD=63), dict(lddA=15),
    dict(lddB=15), dict(pre=0), dict(dD=0), dict(A=0), dict(B=0), dict(dD=D + 1), dict(dA=A), dict(dB=B), dict(dA=D),
    dict(dbias=P), dict(dA=0xA0000), dict(scratch=0), dict(scratch_bytes=100), dict(scratch=S + 8),
    dict(betaA=float("nan")), dict(alpha=float("inf")),
])
def test_grad_refusals(pl, kw):
    _refused(pl, _grad, **kw)


def test_too_many_rows_or_columns_are_unsupported(pl):
    n = (1 << 30) - 127
    for kw in (dict(M=n, ldC=n, ldD=n), dict(N=n)):
        _refused(pl, _call, code=pl.ERR_UNSUPPORTED, **kw)
    for kw in (dict(M=n, ldPre=n, lddD=n), dict(N=n), dict(K=n, ldA=n, ldB=n, lddA=n, lddB=n)):
        _refused(pl, _grad, code=pl.ERR_UNSUPPORTED, **kw)


def test_what_is_empty_returns_at_once(pl):
    # nothing to compute: no GPU is asked for, no operand looked at
    _call(pl, M=0, A=0, D=0, Cm=0)
    _call(pl, N=0, B=0, D=0, Cm=0)
    _grad(pl, dA=None, dB=None, dbias=None, scratch=0)
    _grad(pl, K=0, ldA=1, ldB=1, dbias=None, scratch=0)


def _list(pl, g, n, ty, out=None, oty=None):
    class L:
        pass
    x = L()
    x.count = len(g)
    x.g, x.n, x.type = (C.c_void_p * len(g))(*g), (C.c_int64 * len(g))(*n), (C.c_int32 * len(g))(*ty)
    x.g_out = None if out is None else (C.c_void_p * len(g))(*out)
    x.out_type = None if oty is None else (C.c_int32 * len(g))(*oty)
    return x


def test_list_refusals(pl):
    def bad(lst, max_norm=1.0, scratch=S, both=True):
        with pytest.raises(pl.ParaliaError) as e:
            pl.tile_grad_clip(0, lst, max_norm, scratch)
        assert e.value.code == pl.ERR_INVALID_ARG
        if both:
            with pytest.raises(pl.ParaliaError) as e:
                pl.tile_grad_scale(0, lst, S, max_norm)
            assert e.value.code == pl.ERR_INVALID_ARG

    f, h, b = pl.F32, pl.F16, pl.BF16
    bad(_list(pl, [A], [8], [3]))                                     # no such type
    bad(_list(pl, [A], [8], [f], [B], [-1]))
    bad(_list(pl, [A], [-1], [f]))
    bad(_list(pl, [0], [8], [f]))
    bad(_list(pl, [A], [8], [f], [0], [f]))
    bad(_list(pl, [A + 2], [8], [f]))                                 # not on an element boundary
    bad(_list(pl, [A + 1], [8], [b]))
    bad(_list(pl, [A], [8], [b], [B + 2], [f]))
    bad(_list(pl, [A, A], [8, 8], [b, b]))                            # the same tensor twice
    bad(_list(pl, [B, A], [8, 0x10000], [b, b]))                      # an overlap, listed backwards
    bad(_list(pl, [A], [8], [b], [A], [f]))                           # widened onto itself
    bad(_list(pl, [A], [8], [f], [A + 4], [f]))                       # shifted by one
    bad(_list(pl, [A, B], [8, 8], [f, f], [B, CC], [f, f]))           # one's output is the other's input
    bad(_list(pl, [A, B], [8, 8], [f, f], [CC, CC + 16], [f, f]))
    ok = _list(pl, [A, B], [8, 8], [f, h])
    bad(ok, max_norm=-1.0)
    bad(ok, max_norm=float("nan"))
    bad(ok, scratch=0, both=False)
    bad(ok, scratch=S + 4, both=False)
    with pytest.raises(pl.ParaliaError):
        pl.tile_grad_scale(0, ok, 0, 1.0)
    with pytest.raises(pl.ParaliaError):
        pl.tile_grad_norm(0, ok, S)                                   # nowhere to put the norm
    with pytest.raises(pl.ParaliaError):
        pl.tile_grad_norm(0, ok, 0, norm=D)
    for kw in (dict(sumsq=D + 4), dict(norm=D + 2)):                  # results not aligned to their types
        for f in (pl.tile_grad_norm, lambda *a, **k: pl.tile_grad_clip(*a[:2], 1.0, *a[2:], **k)):
            with pytest.raises(pl.ParaliaError) as e:
                f(0, ok, S, **kw)
            assert e.value.code == pl.ERR_INVALID_ARG
    for args, kw in (((D + 4, 1.0), {}), ((D, 1.0), dict(norm=D + 2))):
        with pytest.raises(pl.ParaliaError) as e:
            pl.tile_grad_scale(0, ok, *args, **kw)
        assert e.value.code == pl.ERR_INVALID_ARG


def test_tensor_list_checks(pl):
    import torch
    with pytest.raises(pl.ParaliaError):
        pl.TensorList([torch.zeros(4, 4).t()[1:]])
    with pytest.raises(pl.ParaliaError):
        pl.TensorList([torch.zeros(4)])                               # host memory
    class T:
        """Looks like a GPU tensor."""
        def __init__(self, dtype, n):
            self.dtype, self._n = dtype, n
        def is_contiguous(self):
            return True
        def numel(self):
            return self._n
        def data_ptr(self):
            return A
    with pytest.raises(pl.ParaliaError):
        pl.TensorList([T("torch.int32", 3)])
    with pytest.raises(pl.ParaliaError):
        pl.TensorList([T("torch.float32", 3)], [])
    with pytest.raises(pl.ParaliaError):
        pl.TensorList([T("torch.float32", 3)], [T("torch.float32", 4)])
    x = pl.TensorList([T("torch.bfloat16", 3), T("torch.float16", 0)])
    assert list(x.n) == [3, 0] and list(x.type) == [pl.BF16, pl.F16] and x.g_out is None


def test_host_memory_is_refused(pl):
    import numpy as np
    import torch
    for x in (torch.zeros(1024, dtype=torch.bfloat16), np.zeros(1024, dtype=np.float16)):
        _refused(pl, _call, A=x)
        _refused(pl, _call, D=x)
        _refused(pl, _grad, dbias=x)
        with pytest.raises(pl.ParaliaError):
            pl.tile_grad_norm(0, pl.TensorList([]), x, norm=D)


def test_scratch_sizes(pl):
    lst = pl.TensorList([])
    assert pl.tile_grad_norm_scratch_bytes(lst) >= 8
    assert pl.lib().PARALiA_tile_grad_norm_scratch_bytes(5000) >= 5 * 8
    # an operand on 16-byte boundaries is read in place
    assert pl.tile_gemm_act_scratch_bytes(pl.BF16, "T", "N", 64, 32, 16, A, 16, B, 16) == 0
    # the gradient holds dZ
    assert pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", 64, 32, 16, A, 16, B, 16, 0) >= 64 * 32 * 2
