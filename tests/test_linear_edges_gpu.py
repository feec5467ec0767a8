"""Calls of the linear layer beside its main ones: rows that end inside a 16-byte group of an aligned column, a bias off
the grid, no rows, no inner dimension. Whole numbers are held exactly (test_gemm_act_gpu.py), NaN stands around every
matrix."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu

TRANS = [("N", "N"), ("T", "N"), ("N", "T"), ("T", "T")]


def _mods():
    import linear_defs
    import test_gemm_act_gpu
    return linear_defs, test_gemm_act_gpu


@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("cut", [1, 3, 7])
@pytest.mark.parametrize("dims", [(136, 1848, 72), (136, 664, 728), (144, 624, 568), (4848, 136, 272), (72, 1032, 5144),
                                  (1112, 1544, 200)])
def test_rows_that_end_inside_a_group(pl, ta, tb, cut, dims):
    # columns of D start on 16-byte boundaries and end `cut` elements before the next one
    d, t = _mods()
    M, N, K = (x - cut for x in dims)
    t._forward(pl, d, "bf16", ta, tb, M, N, K, pad=cut, ints=True, bias=True, beta=1.0, pre=True)
    t._forward(pl, d, "fp16", ta, tb, M, N, K, pad=cut, ints=True, act="relu", beta=1.0, alias=True)
    t._grad(pl, d, "bf16", ta, tb, M, N, K, pad=cut, ints=True, act="relu", betas=(1.0, 0.0, 1.0))


@pytest.mark.parametrize("dims", [(520, 776, 320), (264, 3, 1032)])
@pytest.mark.parametrize("at", [1, 3, 4])
def test_bias_off_the_grid(pl, dims, at):
    # the same bits as with the bias on it, where sums are exact
    import torch
    M, N, K = dims
    g = torch.Generator(device="cuda").manual_seed(5)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g, device="cuda").to(torch.bfloat16)
    A, B, C, bias = whole(M, K), whole(N, K), whole(N, M), whole(M)
    room = torch.full((M + 16,), float("nan"), dtype=torch.bfloat16, device="cuda")
    room[at:at + M] = bias
    out = []
    for b in (bias, room[at:]):
        D, P = torch.zeros_like(C), torch.zeros_like(C)
        pl.tile_gemm_act(0, pl.BF16, "T", "N", M, N, K, 1.0, A, K, B, K, 1.0, C, M, D, M, bias=b, act=pl.ACT_RELU, pre=P,
                         ldPre=M)
        out.append((D, P))
    torch.cuda.synchronize()
    pl.tile_status(0)
    want = B.float() @ A.float().T + bias.float()
    assert torch.equal(out[0][1], want.to(torch.bfloat16)) and torch.equal(out[1][1], out[0][1])
    assert torch.equal(out[1][0], out[0][0])


@pytest.mark.parametrize("beta", [0.0, 0.5])
@pytest.mark.parametrize("tb", ["N", "T"])
def test_gradient_without_rows(pl, beta, tb):
    # M = 0: dB is beta times what was there, nothing else is touched
    import torch
    d, _ = _mods()
    N, K = 33, 40
    shape = (K, N) if tb == "N" else (N, K)
    dB = d.Mat(*shape, torch.float16, 5).set(torch.full(shape, 3.0 if beta else float("nan")))
    pl.tile_gemm_act_grad(0, pl.F16, "N", tb, 0, N, K, 1.0, None, 1, None, shape[0], pl.ACT_SILU, None, 1, None, 1,
                          dB=dB.addr, lddB=dB.ld, betaB=beta)
    torch.cuda.synchronize()
    pl.tile_status(0)
    assert bool((dB.t == 3.0 * beta).all()) and dB.outside_untouched()


def test_gradient_without_inner_dimension(pl):
    # K = 0: dA and dB are empty, the bias gradient is not
    import torch
    M, N = 40, 24
    pre = torch.ones(N, M, dtype=torch.bfloat16, device="cuda")
    dD = torch.full((N, M), 0.5, dtype=torch.bfloat16, device="cuda")
    db = torch.full((M,), float("nan"), dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.bfloat16, device="cuda")
    pl.tile_gemm_act_grad(0, pl.BF16, "T", "N", M, N, 0, 1.0, none, 1, none, 1, pl.ACT_RELU, pre, M, dD, M, dA=none, lddA=1,
                          dB=none, lddB=1, dbias=db)
    torch.cuda.synchronize()
    pl.tile_status(0)
    assert bool((db == N / 2).all())


@pytest.mark.parametrize("cut", [1, 3, 7])
@pytest.mark.parametrize("dims", [(8, 2000, 128), (8, 15000, 136), (16, 300, 2000), (72, 4440, 64), (2056, 40, 64)])
def test_few_rows_that_end_inside_a_group(pl, cut, dims):
    # no whole group of eight rows, or a last one by itself in a tile; the outer products of the gradient likewise
    d, t = _mods()
    M, N, K = dims[0] - cut, dims[1], dims[2]
    for act in ("none", "relu"):
        t._forward(pl, d, "bf16", "T", "N", M, N, K, pad=cut, ints=True, act=act, bias=True, beta=1.0, pre=True)
    t._grad(pl, d, "fp16", "N", "T", M, N, K, pad=cut, ints=True, act="relu", betas=(1.0, 1.0, 1.0))
    t._grad(pl, d, "bf16", "T", "N", M, N, K - cut, pad=cut, ints=True)
