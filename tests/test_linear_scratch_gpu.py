"""The scratch of the linear layer's gradient: a call asks for what it touches, so sizes and forms that touch none
run without any, and less scratch than the size function names changes no result."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu


def _defs():
    import linear_defs
    return linear_defs


@pytest.mark.parametrize("beta", [0.0, 1.0, 0.5])
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("offset", [0, 1])
def test_empty_batch_takes_what_the_size_function_names(pl, beta, act, offset):
    # N = 0: dA and dbias are beta times what was there (halves of whole numbers: exact in BF16)
    import torch
    d = _defs()
    M, K, a = 40, 24, d.ACTS.index(act)
    g = torch.Generator(device="cuda").manual_seed(1)
    A = d.Mat(K, M, torch.bfloat16, 0, offset).set(d.rand(g, K, M))
    dA = d.Mat(K, M, torch.bfloat16, 3, offset).set(torch.randint(-9, 10, (K, M), generator=g, device="cuda").float())
    db = torch.randint(-9, 10, (M,), generator=g, device="cuda").to(torch.bfloat16)
    n = pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", M, 0, K, A.addr, A.ld, None, K, a)
    assert offset or n == 0
    want_a, want_b = beta * dA.m, beta * db.double()
    if beta == 0.0:
        dA.t.fill_(float("nan")), db.fill_(float("nan"))
    pl.tile_gemm_act_grad(0, pl.BF16, "T", "N", M, 0, K, 1.0, A.addr, A.ld, None, K, a, None, M, None, M, dA=dA.addr,
                          lddA=dA.ld, dbias=db, betaA=beta, betaBias=beta, scratch=None, scratch_bytes=0)
    torch.cuda.synchronize()
    pl.tile_status(0)
    assert torch.equal(dA.m, want_a) and torch.equal(db.double(), want_b)
    assert dA.outside_untouched()


def _operands(d, dtype, M, N, K, seed=2):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = d.DT[dtype]
    r = lambda rows, cols, k: d.Mat(rows, cols, dt).set(d.rand(g, rows, cols, k))
    return r(K, M, K ** -0.5), r(K, N, 1.0), r(M, N, 1.5), r(M, N, 0.25)


def _grad(pl, A, B, P, G, M, N, K, a, scratch, size, alpha=1.0, which=("dA", "dB", "dbias"), beta=0.0, old=2.0):
    import torch
    out = {"dA": torch.full_like(A.t.T.contiguous(), old), "dB": torch.full_like(B.t.T.contiguous(), old),
           "dbias": torch.full((M,), old, dtype=A.dt, device="cuda")}
    arg = {k: (out[k] if k in which else None) for k in out}
    pl.tile_gemm_act_grad(0, pl.BF16, "T", "N", M, N, K, alpha, A.addr, A.ld, B.addr, B.ld, a, P.addr, P.ld, G.addr, G.ld,
                          dA=arg["dA"], lddA=K, dB=arg["dB"], lddB=K, dbias=arg["dbias"], betaA=beta, betaB=beta,
                          betaBias=beta, scratch=scratch, scratch_bytes=size)
    torch.cuda.synchronize()
    pl.tile_status(0)
    return out


@pytest.mark.parametrize("dims", [(264, 200, 136), (2056, 4096, 4096)])
def test_no_activation_needs_no_scratch_on_the_grid(pl, dims):
    # the larger one has dD between 32-byte sectors, where a copy pays if there is room: the same bits
    import torch
    d = _defs()
    M, N, K = dims
    A, B, P, G = _operands(d, "bf16", *dims)
    n = pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", M, N, K, A.addr, A.ld, B.addr, B.ld, pl.ACT_NONE)
    s = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    want = _grad(pl, A, B, P, G, M, N, K, pl.ACT_NONE, s, n)
    got = _grad(pl, A, B, P, G, M, N, K, pl.ACT_NONE, None, 0)
    for k in want:
        assert bool(torch.isfinite(want[k].float()).all()) and torch.equal(want[k], got[k]), k


def test_what_makes_no_product_needs_no_scratch(pl):
    import torch
    d = _defs()
    M, N, K = 203, 155, 77        # operands off the 16-byte grid
    A, B, P, G = _operands(d, "bf16", M, N, K)
    a = d.ACTS.index("silu")
    n = pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", M, N, K, A.addr, A.ld, B.addr, B.ld, a)
    s = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    want = _grad(pl, A, B, P, G, M, N, K, a, s, n)
    got = _grad(pl, A, B, P, G, M, N, K, a, None, 0, which=("dbias",))
    assert torch.equal(want["dbias"], got["dbias"])
    got = _grad(pl, A, B, P, G, M, N, K, a, None, 0, alpha=0.0, which=("dA", "dB"), beta=0.5)
    assert bool((got["dA"] == 1.0).all()) and bool((got["dB"] == 1.0).all())
    with pytest.raises(pl.ParaliaError):
        _grad(pl, A, B, P, G, M, N, K, a, None, 0)
    with pytest.raises(pl.ParaliaError):        # a byte short of dZ and both copies
        _grad(pl, A, B, P, G, M, N, K, a, s, n - 1)
