"""The mixed-precision linear layer (PARALiA_tile_gemm_act and its gradient) on the GPU against the
definitions in 64 bits. Tolerances count roundings (linear_defs.py)."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu

TRANS = [("N", "N"), ("T", "N"), ("N", "T"), ("T", "T")]


def _defs():
    import linear_defs
    return linear_defs


def _stored(flag, rows, cols):
    return (cols, rows) if flag in "Tt" else (rows, cols)


def _ty(pl, dtype):
    return pl.BF16 if dtype == "bf16" else pl.F16


def _scratch(n):
    import torch
    return torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")


def _forward(pl, d, dtype, ta, tb, M, N, K, act="none", alpha=1.0, beta=0.0, bias=False, pre=False, pad=0, offset=0,
             alias=False, ints=False, seed=0, stream=0, values=None):
    import torch
    dt = d.DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def fill(r, c, scale):
        if ints:
            return torch.randint(-2, 3, (r, c), generator=g, device="cuda").float()
        return d.rand(g, r, c, scale)

    A = d.Mat(*_stored(ta, M, K), dt, pad, offset).set(fill(*_stored(ta, M, K), max(K, 1) ** -0.5))
    B = d.Mat(*_stored(tb, K, N), dt, pad, offset).set(fill(*_stored(tb, K, N), 1.0))
    C = d.Mat(M, N, dt, pad, offset).set(fill(M, N, 1.0)) if beta else None
    D = C if alias else d.Mat(M, N, dt, pad, offset)
    P = d.Mat(M, N, dt, pad, offset) if pre else None
    bi = fill(M, 1, 0.3).reshape(-1).to(dt) if bias else None
    c0 = C.m if C is not None else None
    n = pl.tile_gemm_act_scratch_bytes(_ty(pl, dtype), ta, tb, M, N, K, A.addr, A.ld, B.addr, B.ld)
    s = _scratch(n)
    pl.tile_gemm_act(0, _ty(pl, dtype), ta, tb, M, N, K, alpha, A.addr, A.ld, B.addr, B.ld, beta,
                     C.addr if C is not None else None, C.ld if C is not None else 0, D.addr, D.ld, bias=bi,
                     act=d.ACTS.index(act), pre=P.addr if P is not None else None, ldPre=P.ld if P is not None else 0,
                     scratch=s, scratch_bytes=n, stream=stream)
    torch.cuda.synchronize()
    pl.tile_status(0)
    want, z, tol, ztol = d.forward_want(A.m, B.m, ta, tb, alpha, bi, act, beta, c0, dt)
    if ints and act in ("none", "relu"):
        # every sum is a whole number below 2^24: FP32 holds it, and one rounding is left
        tol, ztol = d.half_step(dt) * want.abs(), d.half_step(dt) * z.abs()
    d.check(D.t, want, tol, "D")
    assert D.outside_untouched()
    if P is not None:
        d.check(P.t, z, ztol, "pre")
        assert P.outside_untouched()
    return D


SIZES = [(1, 1, 1), (1, 1, 64), (8, 1, 8), (128, 1, 64), (129, 3, 65), (64, 130, 200), (256, 256, 64), (257, 255, 129),
         (1000, 17, 333), (384, 640, 512), (33, 1025, 40), (2048, 64, 1024), (2, 300, 2), (300, 2, 1000), (520, 33, 4096),
         (1, 2000, 128), (2000, 1, 128), (1280, 1536, 192)]


@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("dims", SIZES)
def test_whole_numbers_are_exact(pl, ta, tb, dims):
    # small whole numbers: any wrong index, dropped or repeated term shows as a whole step
    _forward(pl, _defs(), "bf16", ta, tb, *dims, ints=True, bias=True, beta=1.0, pre=True)
    _forward(pl, _defs(), "fp16", ta, tb, *dims, ints=True, act="relu")


@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 0), (8, 8), (3, 1), (7, 4), (0, 1)])
@pytest.mark.parametrize("dims", [(72, 40, 56), (200, 136, 264), (513, 5, 129), (640, 520, 72)])
def test_strides_and_addresses(pl, ta, tb, pad, offset, dims):
    _forward(pl, _defs(), "bf16", ta, tb, *dims, pad=pad, offset=offset, ints=True, bias=True, beta=1.0, pre=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dims", [(96, 1, 200), (700, 40, 300), (520, 776, 320)])
def test_activations(pl, dtype, act, dims):
    _forward(pl, _defs(), dtype, "T", "N", *dims, act=act, bias=True, beta=0.5, alpha=1.5, pre=True)
    _forward(pl, _defs(), dtype, "N", "T", *dims, act=act, seed=3)


def test_residual_in_place(pl):
    _forward(pl, _defs(), "bf16", "T", "N", 264, 200, 136, act="silu", beta=1.0, alias=True)
    _forward(pl, _defs(), "fp16", "T", "N", 264, 2, 2000, act="none", beta=1.0, alias=True, bias=True)


@pytest.mark.parametrize("dims", [(4096, 1, 16384), (4096, 4096, 4096), (8192, 100, 2048), (1237, 2011, 3001)])
def test_large(pl, dims):
    _forward(pl, _defs(), "bf16", "T", "N", *dims, act="gelu_tanh", bias=True, beta=1.0, pre=True)


@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_empty_product(pl, act):
    # no inner dimension, or a factor of 0: A and B are not read
    import torch
    d = _defs()
    M, N = 70, 9
    bias = torch.randn(M, device="cuda").bfloat16()
    C = d.Mat(M, N, torch.bfloat16).set(torch.randn(M, N))
    D = d.Mat(M, N, torch.bfloat16)
    nan = torch.full((M * 64,), float("nan"), dtype=torch.bfloat16, device="cuda")
    for alpha, K, a, b in ((1.0, 0, None, None), (0.0, 16, nan, nan), (0.0, 16, None, None)):
        D.t.fill_(float("nan"))
        pl.tile_gemm_act(0, pl.BF16, "N", "N", M, N, K, alpha, a, M, b, max(K, 1), 2.0, C.addr, C.ld, D.addr, D.ld,
                         bias=bias, act=d.ACTS.index(act))
        torch.cuda.synchronize()
        v = d.act(bias.double()[:, None].expand(M, N), act)
        want = v + 2.0 * C.m
        d.check(D.t, want, d.half_step(torch.bfloat16) * want.abs() + 2.0 ** -17 * (v.abs() + (2 * C.m).abs()), "D")


def test_beta_zero_ignores_c_and_empty_shapes(pl):
    import torch
    d = _defs()
    A = d.Mat(16, 16, torch.float16).set(torch.eye(16))
    B = d.Mat(16, 8, torch.float16).set(torch.ones(16, 8))
    C = d.Mat(16, 8, torch.float16)     # all NaN
    D = d.Mat(16, 8, torch.float16)
    pl.tile_gemm_act(0, pl.F16, "N", "N", 16, 8, 16, 1.0, A.addr, A.ld, B.addr, B.ld, 0.0, C.addr, C.ld, D.addr, D.ld)
    torch.cuda.synchronize()
    assert bool((D.t == 1.0).all())
    before = D.buf.clone()
    pl.tile_gemm_act(0, pl.F16, "N", "N", 0, 8, 16, 1.0, A.addr, A.ld, B.addr, B.ld, 0.0, None, 1, D.addr, D.ld)
    pl.tile_gemm_act(0, pl.F16, "N", "N", 16, 0, 16, 1.0, A.addr, A.ld, B.addr, B.ld, 0.0, None, 1, D.addr, D.ld)
    torch.cuda.synchronize()
    assert torch.equal(before.view(torch.int16), D.buf.view(torch.int16))


def test_infinities_and_nans_stay_where_they_are(pl):
    # a row of A with an infinity or a NaN reaches its row of D and no other
    import torch
    d = _defs()
    for M, N, K in ((200, 3, 100), (300, 200, 100)):
        A = d.Mat(K, M, torch.bfloat16).set(torch.ones(K, M))
        B = d.Mat(K, N, torch.bfloat16).set(torch.ones(K, N))
        A.t[5, 7] = float("inf")
        A.t[50, 150] = float("nan")
        A.t[0, 9] = float("-inf")
        for act, low in (("none", float("-inf")), ("relu", 0.0), ("gelu", 0.0), ("gelu_tanh", 0.0), ("silu", 0.0)):
            D = d.Mat(M, N, torch.bfloat16)
            n = pl.tile_gemm_act_scratch_bytes(pl.BF16, "T", "N", M, N, K, A.addr, A.ld, B.addr, B.ld)
            pl.tile_gemm_act(0, pl.BF16, "T", "N", M, N, K, 1.0, A.addr, A.ld, B.addr, B.ld, 0.0, None, 1, D.addr, D.ld,
                             act=d.ACTS.index(act), scratch=_scratch(n), scratch_bytes=n)
            torch.cuda.synchronize()
            assert bool(torch.isposinf(D.t[7]).all()), act
            assert bool(torch.isnan(D.t[150]).all()), act
            assert bool((D.t[9].float() == low).all()) or bool((D.t[9].float().abs() < 1e-20).all()) and low == 0.0, act
            rest = torch.ones(M, dtype=torch.bool)
            rest[[7, 150, 9]] = False
            assert bool((D.t[rest.cuda()].float() == 100.0).all()), act


def test_streams_graphs_and_repeats(pl):
    """Two captured graphs with scratch of their own, replayed on their streams after new inputs."""
    import torch
    d = _defs()
    pl.fill_f32(torch.zeros(1, device="cuda"), 1, 0, 0, 0)      # sets the GPU up
    cases = []
    for i, (M, N, K, off) in enumerate(((300, 257, 190, 0), (1000, 3, 515, 1))):
        g = torch.Generator(device="cuda").manual_seed(i)
        A = d.Mat(K, M, torch.bfloat16, offset=off)
        B = d.Mat(K, N, torch.bfloat16, offset=off)
        D = d.Mat(M, N, torch.bfloat16)
        n = pl.tile_gemm_act_scratch_bytes(pl.BF16, "T", "N", M, N, K, A.addr, A.ld, B.addr, B.ld)
        s = _scratch(n)
        st = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        A.t.zero_(), B.t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            pl.tile_gemm_act(0, pl.BF16, "T", "N", M, N, K, 1.0, A.addr, A.ld, B.addr, B.ld, 0.0, None, 1, D.addr, D.ld,
                             act=pl.ACT_SILU, scratch=s, scratch_bytes=n, stream=st.cuda_stream)
        cases.append((M, N, K, A, B, D, s, st, graph, g))
    for rep in range(3):
        for M, N, K, A, B, D, s, st, graph, g in cases:
            A.set(d.rand(g, K, M, K ** -0.5)), B.set(d.rand(g, K, N))
        torch.cuda.synchronize()
        for c in cases:
            with torch.cuda.stream(c[7]):
                c[8].replay()
        torch.cuda.synchronize()
        for M, N, K, A, B, D, *_ in cases:
            want, _, tol, _ = d.forward_want(A.m, B.m, "T", "N", 1.0, None, "silu", 0.0, None, torch.bfloat16)
            d.check(D.t, want, tol, "D")
    pl.tile_status(0)


def test_same_bits_every_time(pl):
    import torch
    d = _defs()
    for dims in ((4096, 5, 8192), (700, 900, 1100)):
        a = _forward(pl, d, "bf16", "T", "N", *dims, seed=9)
        b = _forward(pl, d, "bf16", "T", "N", *dims, seed=9)
        assert torch.equal(a.t, b.t)


# ------------------------------------------------------------------ gradient
def _grad(pl, d, dtype, ta, tb, M, N, K, act="none", alpha=1.0, betas=(0.0, 0.0, 0.0), pad=0, offset=0,
          which=("dA", "dB", "dbias"), seed=0, ints=False):
    import torch
    dt = d.DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def fill(r, c, scale):
        if ints:
            return torch.randint(-2, 3, (r, c), generator=g, device="cuda").float()
        return d.rand(g, r, c, scale)

    sa, sb = _stored(ta, M, K), _stored(tb, K, N)
    A = d.Mat(*sa, dt, pad, offset).set(fill(*sa, max(K, 1) ** -0.5))
    B = d.Mat(*sb, dt, pad, offset).set(fill(*sb, 1.0))
    P = d.Mat(M, N, dt, pad, offset).set(fill(M, N, 1.5))
    G = d.Mat(M, N, dt, pad, offset).set(fill(M, N, 0.25))
    old = {"dA": fill(*sa, 1.0), "dB": fill(*sb, 1.0), "dbias": fill(M, 1, 1.0)}
    out = {"dA": d.Mat(*sa, dt, pad, offset).set(old["dA"]), "dB": d.Mat(*sb, dt, pad, offset).set(old["dB"]),
           "dbias": d.Mat(M, 1, dt).set(old["dbias"])}
    a = d.ACTS.index(act)
    n = pl.tile_gemm_act_grad_scratch_bytes(_ty(pl, dtype), ta, tb, M, N, K, A.addr, A.ld, B.addr, B.ld, a)
    s = _scratch(n)
    s.fill_(255)   # what scratch holds before the call does not matter
    arg = {k: (out[k].addr if k in which else None) for k in out}
    pl.tile_gemm_act_grad(0, _ty(pl, dtype), ta, tb, M, N, K, alpha, A.addr, A.ld, B.addr, B.ld, a, P.addr, P.ld, G.addr,
                          G.ld, dA=arg["dA"], lddA=out["dA"].ld, dB=arg["dB"], lddB=out["dB"].ld, dbias=arg["dbias"],
                          betaA=betas[0], betaB=betas[1], betaBias=betas[2], scratch=s, scratch_bytes=n)
    torch.cuda.synchronize()
    pl.tile_status(0)
    want = d.grad_want(A.m, B.m, ta, tb, alpha, act, P.m, G.m, dt)
    u = d.half_step(dt)
    for i, k in enumerate(("dA", "dB", "dbias")):
        before = old[k].to(dt).double()
        if k not in which:
            assert torch.equal(out[k].m, before), k
            continue
        v, tol = want[k]
        if k == "dbias":
            v, tol = v[:, None], tol[:, None]
        if ints and act in ("none", "relu"):
            tol = u * v.abs()
        if betas[i]:
            tol = tol + (u + 2.0 ** -22) * ((betas[i] * before).abs() + v.abs())
            v = v + betas[i] * before
        d.check(out[k].t, v, tol, k)
        assert out[k].outside_untouched(), k


@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("dims", [(1, 1, 1), (8, 1, 16), (65, 33, 129), (256, 128, 64), (300, 7, 520), (5, 700, 40),
                                  (640, 513, 257), (1024, 300, 1100)])
def test_grad_whole_numbers_are_exact(pl, ta, tb, dims):
    _grad(pl, _defs(), "bf16", ta, tb, *dims, ints=True)
    _grad(pl, _defs(), "fp16", ta, tb, *dims, ints=True, act="relu")


@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
@pytest.mark.parametrize("dims", [(4096, 8, 1024), (2050, 1, 4098), (4100, 100, 1100)])
def test_grad_of_few_columns(pl, ta, tb, dims, pad, offset):
    # one product with hardly any k, one with much: a launch each
    _grad(pl, _defs(), "bf16", ta, tb, *dims, act="relu", betas=(1.0, 0.0, 0.0), pad=pad, offset=offset, ints=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_grad_activations(pl, dtype, act, ta, tb):
    _grad(pl, _defs(), dtype, ta, tb, 264, 200, 136, act=act, alpha=0.75)


@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 8), (3, 1), (0, 1)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_grad_strides_accumulation_and_parts(pl, pad, offset, act):
    d = _defs()
    _grad(pl, d, "bf16", "T", "N", 203, 155, 77, act=act, pad=pad, offset=offset, betas=(1.0, 0.5, 1.0))
    for which in (("dA",), ("dB",), ("dbias",), ("dA", "dbias")):
        _grad(pl, d, "bf16", "T", "N", 203, 155, 77, act=act, pad=pad, offset=offset, which=which)


def test_grad_empty(pl):
    # no columns: the gradients of A and of the bias are 0, not what was there
    import torch
    d = _defs()
    A, B = d.Mat(16, 24, torch.bfloat16).set(torch.ones(16, 24)), d.Mat(16, 1, torch.bfloat16)
    dA, db = d.Mat(16, 24, torch.bfloat16), torch.full((24,), 7.0, dtype=torch.bfloat16, device="cuda")
    n = pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", 24, 0, 16, A.addr, 16, B.addr, 16, pl.ACT_GELU)
    pl.tile_gemm_act_grad(0, pl.BF16, "T", "N", 24, 0, 16, 1.0, A.addr, 16, B.addr, 16, pl.ACT_GELU, None, 24, None, 24,
                          dA=dA.addr, lddA=dA.ld, dbias=db, scratch=_scratch(n), scratch_bytes=n)
    torch.cuda.synchronize()
    assert bool((dA.t == 0).all()) and bool((db == 0).all())


def test_grad_closed_places_of_relu(pl):
    # an infinite or NaN dD where relu is closed does not reach the gradients
    import torch
    d = _defs()
    M, N, K = 40, 24, 32
    A, B = d.Mat(K, M, torch.bfloat16).set(torch.ones(K, M)), d.Mat(K, N, torch.bfloat16).set(torch.ones(K, N))
    P, G = d.Mat(M, N, torch.bfloat16).set(torch.ones(M, N)), d.Mat(M, N, torch.bfloat16).set(torch.ones(M, N))
    P.t[3, :] = -1.0
    G.t[3, 4], G.t[3, 5] = float("inf"), float("nan")
    dA, dB, db = d.Mat(K, M, torch.bfloat16), d.Mat(K, N, torch.bfloat16), d.Mat(M, 1, torch.bfloat16)
    n = pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", M, N, K, A.addr, A.ld, B.addr, B.ld, pl.ACT_RELU)
    pl.tile_gemm_act_grad(0, pl.BF16, "T", "N", M, N, K, 1.0, A.addr, A.ld, B.addr, B.ld, pl.ACT_RELU, P.addr, P.ld,
                          G.addr, G.ld, dA=dA.addr, lddA=dA.ld, dB=dB.addr, lddB=dB.ld, dbias=db.addr,
                          scratch=_scratch(n), scratch_bytes=n)
    torch.cuda.synchronize()
    want = torch.full((M,), float(N), device="cuda")
    want[3] = 0.0
    assert torch.equal(db.t[:, 0].float(), want)
    assert torch.equal(dA.t.float(), want[None, :].expand(K, M))
    assert bool((dB.t.float() == M - 1).all())


@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
def test_grad_against_differences(pl, act):
    """Central differences of the loss sum(D . G) in 64 bits. The operands are sixteenths and eighths of small
    whole numbers, so that FP16 holds Z exactly and the kept pre-activation is the Z of the formula."""
    import torch
    d = _defs()
    M, N, K = 24, 10, 16
    g = torch.Generator(device="cuda").manual_seed(4)

    def whole(r, c, q):
        return torch.randint(-4, 5, (r, c), generator=g, device="cuda").float() / q

    A, B, G = (d.Mat(*s, torch.float16).set(whole(*s, q)) for s, q in (((K, M), 16), ((K, N), 8), ((M, N), 4)))
    bias = whole(M, 1, 8).reshape(-1).half()
    D, P = d.Mat(M, N, torch.float16), d.Mat(M, N, torch.float16)
    a = d.ACTS.index(act)
    pl.tile_gemm_act(0, pl.F16, "T", "N", M, N, K, 1.0, A.addr, A.ld, B.addr, B.ld, 0.0, None, 1, D.addr, D.ld, bias=bias,
                     act=a, pre=P.addr, ldPre=P.ld)
    out = {"dA": d.Mat(K, M, torch.float16), "dB": d.Mat(K, N, torch.float16), "dbias": d.Mat(M, 1, torch.float16)}
    n = pl.tile_gemm_act_grad_scratch_bytes(pl.F16, "T", "N", M, N, K, A.addr, A.ld, B.addr, B.ld, a)
    pl.tile_gemm_act_grad(0, pl.F16, "T", "N", M, N, K, 1.0, A.addr, A.ld, B.addr, B.ld, a, P.addr, P.ld, G.addr, G.ld,
                          dA=out["dA"].addr, lddA=K, dB=out["dB"].addr, lddB=K, dbias=out["dbias"].addr,
                          scratch=_scratch(n), scratch_bytes=n)
    torch.cuda.synchronize()
    z = A.m.T @ B.m + bias.double()[:, None]
    assert torch.equal(P.m, z)
    _, tol = {}, d.grad_want(A.m, B.m, "T", "N", 1.0, act, P.m, G.m, torch.float16)

    def loss(x, y, b):
        return float((d.act(x.T @ y + b, act) * G.m).sum())

    h = 2.0 ** -12
    base = {"dA": A.m, "dB": B.m, "dbias": bias.double()[:, None]}
    for key, i, j in (("dA", 0, 0), ("dA", 7, 23), ("dA", 15, 11), ("dB", 3, 9), ("dB", 15, 0), ("dbias", 5, 0),
                      ("dbias", 23, 0)):
        side = []
        for sign in (1.0, -1.0):
            x = {k: v.clone() for k, v in base.items()}
            x[key][i, j] += sign * h
            side.append(loss(x["dA"], x["dB"], x["dbias"]))
        diff = (side[0] - side[1]) / (2 * h)
        t = tol[key][1]
        t = float(t[i] if t.dim() == 1 else t[i, j])
        # the differences' own error: h^2/6 times a third derivative (below 3 in sum here) and rounding
        assert abs(float(out[key].t[i, j]) - diff) <= t + h * h * 16 + 1e-9, (key, i, j)


def test_offsets_beyond_32_bits(pl):
    # D has 4.6e9 entries; the last columns, rows and a few in between are looked at
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    M, N, K = 65544, 70001, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    A = torch.randint(-2, 3, (M, K), generator=g, device="cuda").to(torch.bfloat16)     # K x M, transposed
    B = torch.randint(-2, 3, (N, K), generator=g, device="cuda").to(torch.bfloat16)     # K x N
    D = torch.full((N, M), float("nan"), dtype=torch.bfloat16, device="cuda")
    pl.tile_gemm_act(0, pl.BF16, "T", "N", M, N, K, 1.0, A, K, B, K, 0.0, None, M, D, M)
    torch.cuda.synchronize()
    pl.tile_status(0)
    cols = torch.tensor([0, 1, 255, 256, 32767, 32768, 40000, 65535, 65536, N - 2, N - 1], device="cuda")
    want = (B[cols].float() @ A.float().T).to(torch.bfloat16)
    assert torch.equal(D[cols], want)
    assert bool(torch.isfinite(D[:, M - 1].float()).all()) and bool(torch.isfinite(D[:, 0].float()).all())
    rows = torch.tensor([0, 127, 128, 30001, M - 1], device="cuda")
    assert torch.equal(D[:, rows], (B.float() @ A[rows].float().T).to(torch.bfloat16))


@pytest.mark.parametrize("ta,tb", TRANS)
def test_copies_that_pay(pl, ta, tb):
    # columns between 32-byte sectors: copied where scratch is given, read in place where it is not; the same bits
    import torch
    M, N, K = 4104, 4120, 2056
    g = torch.Generator(device="cuda").manual_seed(11)
    (ra, ca), (rb, cb) = _stored(ta, M, K), _stored(tb, K, N)
    A, B = (torch.randint(-2, 3, (c, r), generator=g, device="cuda").to(torch.bfloat16) for r, c in ((ra, ca), (rb, cb)))
    n = pl.tile_gemm_act_scratch_bytes(pl.BF16, ta, tb, M, N, K, A, ra, B, rb)
    assert n > 0
    want = (B.T if tb == "T" else B).float() @ (A if ta == "N" else A.T).float()
    out = []
    for scratch, size in ((_scratch(n), n), (None, 0), (_scratch(64), 64)):
        D = torch.zeros(N, M, dtype=torch.bfloat16, device="cuda")
        pl.tile_gemm_act(0, pl.BF16, ta, tb, M, N, K, 1.0, A, ra, B, rb, 0.0, None, M, D, M, scratch=scratch,
                         scratch_bytes=size)
        out.append(D)
    torch.cuda.synchronize()
    pl.tile_status(0)
    assert all(torch.equal(D, want.to(torch.bfloat16)) for D in out)
    _grad(pl, _defs(), "bf16", ta, tb, M, N, K, act="none", alpha=0.5, ints=True)


@pytest.mark.parametrize("N", [1, 40])
def test_leading_dimensions_of_single_columns(pl, N):
    # a single column may have any leading dimension, a wide gap between columns is jumped over
    import torch
    d = _defs()
    M, K = 264, 72
    g = torch.Generator(device="cuda").manual_seed(8)
    ld = 1 << 40 if N == 1 else 100_000
    A = torch.randint(-2, 3, (M, K), generator=g, device="cuda").to(torch.bfloat16)
    B = torch.randint(-2, 3, (N, K), generator=g, device="cuda").to(torch.bfloat16)
    D = torch.zeros((N - 1) * (ld if N > 1 else 0) + M, dtype=torch.bfloat16, device="cuda")
    P = torch.zeros_like(D)
    pl.tile_gemm_act(0, pl.BF16, "T", "N", M, N, K, 1.0, A, K, B, ld if N == 1 else K, 0.0, None, ld, D, ld, pre=P, ldPre=ld)
    torch.cuda.synchronize()
    want = (B.float() @ A.float().T).to(torch.bfloat16)
    for buf in (D, P):
        got = buf[:M].reshape(1, M) if N == 1 else torch.as_strided(buf, (N, M), (ld, 1))
        assert torch.equal(got, want)
