"""What the mixed-precision linear-layer and gradient-list routines accept and refuse, beside test_linear_host.py. The
addresses are never read: every call here is refused, those that pass the checks in question by a GPU that does not
exist."""
import pytest

A, B, CC, D, P, S, DA, DB, DBIAS = (0x100000 * i for i in range(1, 10))
NO_GPU = 99


def _grad(pl, **kw):
    a = dict(dev=NO_GPU, type=pl.BF16, TransA="T", TransB="N", M=64, N=32, K=16, alpha=1.0, A=A, ldA=16, B=B, ldB=16,
             act=pl.ACT_GELU, pre=P, ldPre=64, dD=D, lddD=64, dA=DA, lddA=16, dB=DB, lddB=16, dbias=DBIAS, scratch=S,
             scratch_bytes=4096)
    a.update(kw)
    with pytest.raises(pl.ParaliaError) as e:
        pl.tile_gemm_act_grad(**a)
    return str(e.value)


def _passes(text):
    """Whether a call came as far as its GPU: there is none, or not so many."""
    return "no CUDA device" in text or "out of range" in text


def test_gradient_asks_for_no_scratch_that_it_does_not_touch(pl):
    none = dict(scratch=None, scratch_bytes=0)
    assert "bytes of scratch" in _grad(pl, **none) and _passes(_grad(pl))
    assert _passes(_grad(pl, N=0, B=0, dD=0, pre=0, **none))
    assert _passes(_grad(pl, act=pl.ACT_NONE, pre=0, **none))
    assert _passes(_grad(pl, dA=None, dB=None, **none))
    assert _passes(_grad(pl, alpha=0.0, **none))
    assert "bytes of scratch" in _grad(pl, act=pl.ACT_NONE, dD=D + 2, **none)       # dD has to be copied
    assert "bytes of scratch" in _grad(pl, act=pl.ACT_NONE, A=A + 2, **none)
