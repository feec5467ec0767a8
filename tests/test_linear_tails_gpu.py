"""Activations and their slopes at every value of the 16-bit types, infinities, NaNs and both tails included.

Z is the bias of a product without inner dimension, so it is exact; a slope is the bias gradient of one column with
dD = 1. Tolerances. A smooth activation is computed in FP32 from s = 2^y: y has at most seven roundings of 2^-24
relative (constants included), which 2^y turns into 7 ln(2) 2^-24 |y| < 2^-21 |y|; the special-function unit, the sum
and the products after it add less than 2^-20. Where 1 - g is left of a g near 1 it is off by 2^-23, times the
factor that stands with it. A sigmoid or tail probability below 2^-126 counts as 0: what is lost is at most 2^-126 times
what it is multiplied by, at the place where that happens (90 for silu, 10.2 and 244 for tanh-GELU, 14 for GELU). Then one
rounding to the type, half a subnormal step at least."""
import math
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu

C = math.sqrt(2.0 / math.pi)
LOST = {"gelu": (14.0, 14.0), "gelu_tanh": (10.2, 244.0), "silu": (90.0, 91.0)}     # times 2^-126: value, slope


def _all(dtype):
    import torch
    import linear_defs as d
    return torch.arange(-32768, 32768, device="cuda").to(torch.int16).view(d.DT[dtype])


def _parts(z, act):
    """In 64 bits: act(z), the two terms of act'(z), the factor of g (1 - g) in it, |y|."""
    import torch
    if act == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * p, p, z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi), torch.zeros_like(z), 0.7214 * z * z
    if act == "silu":
        g, f = torch.sigmoid(z), z
        y = 1.4427 * z.abs()
    else:
        g, f = torch.sigmoid(2.0 * C * (z + 0.044715 * z ** 3)), 2.0 * C * z * (1.0 + 3 * 0.044715 * z * z)
        y = 2.3023 * (z.abs() + 0.044715 * z.abs() ** 3)
    one_g = torch.sigmoid(-z) if act == "silu" else torch.sigmoid(-2.0 * C * (z + 0.044715 * z ** 3))
    return z * g, g, f * g * one_g, f.abs().clamp(max=244.0), y


def _check(got, want, tol, z, what):
    import torch
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = int(bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} values off, first at z = {float(z[i])}: got {float(got[i])}, want "
                             f"{float(want[i])} +- {float(tol[i])}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("columns", [1, 136])
def test_every_value(pl, dtype, act, columns):
    import torch
    import linear_defs as d
    z16 = _all(dtype)
    M, ty, dt = z16.numel(), (pl.BF16 if dtype == "bf16" else pl.F16), z16.dtype
    D = torch.zeros(columns, M, dtype=dt, device="cuda")
    pl.tile_gemm_act(0, ty, "T", "N", M, columns, 0, 1.0, None, 1, None, 1, 0.0, None, M, D, M, bias=z16,
                     act=d.ACTS.index(act))
    torch.cuda.synchronize()
    pl.tile_status(0)
    assert bool((D.view(torch.int16) == D[0].view(torch.int16)).all())
    z, out = z16.double(), D[0]
    assert bool(torch.isnan(out[torch.isnan(z)]).all())
    assert bool((out[torch.isposinf(z)] == float("inf")).all()) and bool((out[torch.isneginf(z)] == 0.0).all())
    f = torch.isfinite(z)
    z, out = z[f], out[f]
    want, _, _, _, y = _parts(z, act)
    u, step = d.half_step(dt), torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    tol = (u + (1 + u) * (2.0 ** -20 + 2.0 ** -21 * y.clamp(max=130.0))) * want.abs() + LOST[act][0] * 2.0 ** -126 + step / 2
    _check(out, want, tol, z, act)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("offset", [0, 1])
def test_every_slope(pl, dtype, act, offset):
    import torch
    import linear_defs as d
    z16 = _all(dtype)
    M, ty, dt = z16.numel(), (pl.BF16 if dtype == "bf16" else pl.F16), z16.dtype
    pre = torch.zeros(M + 8, dtype=dt, device="cuda")[offset:offset + M]
    pre.copy_(z16)
    dD, out = torch.ones(M, dtype=dt, device="cuda"), torch.zeros(M, dtype=dt, device="cuda")
    n = pl.tile_gemm_act_grad_scratch_bytes(ty, "T", "N", M, 1, 1, None, 1, None, 1, d.ACTS.index(act))
    s = torch.empty(n, dtype=torch.uint8, device="cuda")
    pl.tile_gemm_act_grad(0, ty, "T", "N", M, 1, 1, 1.0, None, 1, None, 1, d.ACTS.index(act), pre, M, dD, M, dbias=out,
                          scratch=s, scratch_bytes=n)
    torch.cuda.synchronize()
    pl.tile_status(0)
    z = z16.double()
    assert bool(torch.isnan(out[torch.isnan(z)]).all())
    assert bool((out[torch.isposinf(z)] == 1.0).all()) and bool((out[torch.isneginf(z)] == 0.0).all())
    f = torch.isfinite(z)
    z, out = z[f], out[f]
    _, a, b, factor, y = _parts(z, act)
    b = torch.where(torch.isnan(b), torch.zeros_like(b), b)          # infinity times 0 far out
    u, step = d.half_step(dt), torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    e = (2.0 ** -20 + 2.0 ** -21 * y.clamp(max=130.0)) * (a.abs() + b.abs()) + (z > 0) * factor * 2.0 ** -22
    tol = u * (a + b).abs() + (1 + u) * e + LOST[act][1] * 2.0 ** -126 + step / 2
    _check(out, a + b, tol, z, act + " slope")
