"""The linear-layer and gradient-list routines used together: a training step of a two-layer block (forward, gradient,
clipping), eagerly and as a captured graph, and chains of calls on one stream whose results depend on each call seeing
what the one before it wrote. Every stage is held to the definitions in 64 bits of what went into it on the device."""
import math
import sys
import threading
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))

pytestmark = pytest.mark.gpu


class Block:
    """h = gelu_tanh(W1 x + b1), y = W2 h + b2 + x. Weights are stored as [out, in], activations as [tokens, features]."""

    def __init__(self, pl, d, tokens, width, hidden, dtype, seed=0, stream=0):
        import torch
        self.pl, self.d, self.T, self.W, self.H, self.stream = pl, d, tokens, width, hidden, stream
        self.dt, self.ty = d.DT[dtype], (pl.BF16 if dtype == "bf16" else pl.F16)
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s, k=1.0: (torch.randn(*s, generator=g, device="cuda") * k).to(self.dt)
        e = lambda *s: torch.full(s, float("nan"), dtype=self.dt, device="cuda")
        T, W, H = tokens, width, hidden
        self.x, self.dy = r(T, W), r(T, W, k=0.1)
        self.w1, self.b1, self.w2, self.b2 = r(H, W, k=W ** -0.5), r(H, k=0.1), r(W, H, k=H ** -0.5), r(W, k=0.1)
        self.pre, self.h, self.y = e(T, H), e(T, H), e(T, W)
        self.dw1, self.db1, self.dw2, self.db2, self.dh, self.dx = e(H, W), e(H), e(W, H), e(W), e(T, H), e(T, W)
        need = [pl.tile_gemm_act_scratch_bytes(self.ty, "T", "N", H, T, W, self.w1, W, self.x, W),
                pl.tile_gemm_act_scratch_bytes(self.ty, "T", "N", W, T, H, self.w2, H, self.h, H),
                pl.tile_gemm_act_grad_scratch_bytes(self.ty, "T", "N", H, T, W, self.w1, W, self.x, W, pl.ACT_GELU_TANH),
                pl.tile_gemm_act_grad_scratch_bytes(self.ty, "T", "N", W, T, H, self.w2, H, self.h, H, pl.ACT_NONE)]
        self.n = max(need)
        self.scratch = torch.empty(max(self.n, 16), dtype=torch.uint8, device="cuda")
        self.grads = pl.TensorList([self.dw1, self.db1, self.dw2, self.db2])
        self.list_scratch = torch.empty(pl.tile_grad_norm_scratch_bytes(self.grads), dtype=torch.uint8, device="cuda")
        self.norm = torch.zeros(1, device="cuda")

    def step(self, max_norm):
        pl, T, W, H = self.pl, self.T, self.W, self.H
        kw = dict(scratch=self.scratch, scratch_bytes=self.n, stream=self.stream)
        pl.tile_gemm_act(0, self.ty, "T", "N", H, T, W, 1.0, self.w1, W, self.x, W, 0.0, None, H, self.h, H, bias=self.b1,
                         act=pl.ACT_GELU_TANH, pre=self.pre, ldPre=H, **kw)
        pl.tile_gemm_act(0, self.ty, "T", "N", W, T, H, 1.0, self.w2, H, self.h, H, 1.0, self.x, W, self.y, W,
                         bias=self.b2, **kw)
        pl.tile_gemm_act_grad(0, self.ty, "T", "N", W, T, H, 1.0, self.w2, H, self.h, H, pl.ACT_NONE, None, W, self.dy, W,
                              dA=self.dw2, lddA=H, dB=self.dh, lddB=H, dbias=self.db2, **kw)
        pl.tile_gemm_act_grad(0, self.ty, "T", "N", H, T, W, 1.0, self.w1, W, self.x, W, pl.ACT_GELU_TANH, self.pre, H,
                              self.dh, H, dA=self.dw1, lddA=W, dB=self.dx, lddB=W, dbias=self.db1, **kw)
        self.raw = None
        if max_norm is not None:
            pl.tile_grad_clip(0, self.grads, max_norm, self.list_scratch, norm=self.norm, stream=self.stream)

    def check(self, max_norm):
        """Against the definitions, stage by stage; with `max_norm` the gradients are the clipped ones."""
        d, dt = self.d, self.dt
        # matrices as the definitions have them: columns are tokens
        x, h, pre, y, dy, dh, dx = (t.double().T for t in (self.x, self.h, self.pre, self.y, self.dy, self.dh, self.dx))
        w1, w2 = self.w1.double(), self.w2.double()
        D, Z, tol, ztol = d.forward_want(w1, x, "N", "N", 1.0, self.b1, "gelu_tanh", 0.0, None, dt)
        d.check(h, D, tol, "h")
        d.check(pre, Z, ztol, "pre")
        D, _, tol, _ = d.forward_want(w2, h, "N", "N", 1.0, self.b2, "none", 1.0, x, dt)
        d.check(y, D, tol, "y")
        g2 = d.grad_want(w2, h, "N", "N", 1.0, "none", None, dy, dt)
        g1 = d.grad_want(w1, x, "N", "N", 1.0, "gelu_tanh", pre, dh, dt)
        d.check(dh, *g2["dB"], "dh")
        d.check(dx, *g1["dB"], "dx")
        want = {"dw1": g1["dA"], "db1": g1["dbias"], "dw2": g2["dA"], "db2": g2["dbias"]}
        k = 1.0
        if max_norm is not None:
            # the norm is that of the rounded gradients: off by what they are off, at most
            norm = math.sqrt(sum(float((v ** 2).sum()) for v, _ in want.values()))
            off = math.sqrt(sum(float((t ** 2).sum()) for _, t in want.values()))
            assert abs(float(self.norm) - norm) <= off + 2.0 ** -20 * norm
            k = min(1.0, max_norm / float(self.norm))
        u = d.half_step(dt)
        for key, (v, t) in want.items():
            t2 = k * t + (u + 2.0 ** -20) * (k * v.abs() + k * t) + d.tiny(dt) if k < 1.0 else t
            d.check(getattr(self, key), k * v, t2, key)


SHAPES = [(1, 64, 128), (7, 72, 264), (130, 256, 1024), (257, 203, 515), (1000, 512, 2048)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_training_step(pl, dtype, shape):
    import torch
    import linear_defs as d
    b = Block(pl, d, *shape, dtype)
    for max_norm in (None, 1e9, 0.01):
        b.step(max_norm)
        torch.cuda.synchronize()
        pl.tile_status(0)
        b.check(max_norm)


def test_captured_step_follows_new_inputs(pl):
    import torch
    import linear_defs as d
    pl.fill_f32(torch.zeros(1, device="cuda"), 1, 0, 0, 0)      # sets the GPU up
    st = torch.cuda.Stream()
    b = Block(pl, d, 130, 200, 515, "bf16", stream=st.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        b.step(0.02)
    for seed in (5, 6):
        other = Block(pl, d, 130, 200, 515, "bf16", seed=seed)
        for name in ("x", "dy", "w1", "b1", "w2", "b2"):
            getattr(b, name).copy_(getattr(other, name))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        pl.tile_status(0)
        b.check(0.02)
        # the same bits as eager calls on the same inputs
        other.step(0.02)
        torch.cuda.synchronize()
        for name in ("y", "dx", "dw1", "db1", "dw2", "db2", "norm"):
            assert torch.equal(getattr(b, name), getattr(other, name)), name


@pytest.mark.parametrize("shape", [(512, 3), (515, 40), (512, 700)])
@pytest.mark.parametrize("how", ["eager", "graph", "mixed"])
def test_each_call_sees_what_the_last_one_wrote(pl, shape, how):
    """A chain of products, each of the one before it. With every call followed by a synchronisation the chain
    cannot go wrong; without, it has the same bits."""
    import torch
    n, cols = shape
    links = 40
    g = torch.Generator(device="cuda").manual_seed(1)
    w = [(torch.randn(n, n, generator=g, device="cuda") * n ** -0.5).bfloat16() for _ in range(4)]
    x0 = torch.randn(cols, n, generator=g, device="cuda").bfloat16()
    st = torch.cuda.Stream()
    need = pl.tile_gemm_act_scratch_bytes(pl.BF16, "T", "N", n, cols, n, w[0], n, x0, n)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")   # one for the whole chain

    def chain(bufs, sync):
        for i in range(links):
            a, b = bufs[i % 2], bufs[(i + 1) % 2]
            pl.tile_gemm_act(0, pl.BF16, "T", "N", n, cols, n, 1.0, w[i % 4], n, a, n, 0.5, a, n, b, n,
                             act=pl.ACT_SILU if i % 3 else pl.ACT_NONE, scratch=scratch, scratch_bytes=need,
                             stream=st.cuda_stream)
            if how == "mixed":
                b.mul_(1.0625)      # another library's kernel between two of ours
            if sync:
                torch.cuda.synchronize()

    out = []
    for sync in (True, False):
        bufs = [x0.clone(), torch.zeros_like(x0)]
        torch.cuda.synchronize()
        if how == "graph" and not sync:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                chain(bufs, False)
            bufs[0].copy_(x0)
            torch.cuda.synchronize()
            graph.replay()
        else:
            with torch.cuda.stream(st):
                chain(bufs, sync)
        torch.cuda.synchronize()
        pl.tile_status(0)
        out.append(bufs[links % 2].clone())
    assert bool(torch.isfinite(out[0].float()).all())
    assert torch.equal(out[0], out[1])


def test_calls_from_two_threads(pl):
    """Two host threads, a stream and scratch each, at the same time: the bits of one after the other."""
    import torch
    import linear_defs as d
    streams = [torch.cuda.Stream() for _ in range(2)]
    blocks = [Block(pl, d, 200 + 37 * i, 264, 520, "bf16", seed=i, stream=streams[i].cuda_stream) for i in range(2)]
    torch.cuda.synchronize()
    for b in blocks:
        b.step(0.05)
        torch.cuda.synchronize()
    names = ("y", "dx", "dw1", "db1", "dw2", "db2", "norm")
    want = [{k: getattr(b, k).clone() for k in names} for b in blocks]
    errors = []

    def work(b):
        try:
            for _ in range(30):
                b.step(0.05)
        except Exception as ex:     # noqa: BLE001
            errors.append(ex)

    threads = [threading.Thread(target=work, args=(b,)) for b in blocks]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    pl.tile_status(0)
    for b, w in zip(blocks, want):
        for k in names:
            assert torch.equal(getattr(b, k), w[k]), k


def test_norm_over_two_lists_then_scale(pl):
    """Gradients held by two owners: the squared norms are added, each owner scales its own."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    lists = [[torch.randn(n, generator=g, device="cuda").bfloat16() for n in sizes] for sizes in ((1000, 7), (4099, 30000, 2))]
    before = [[t.clone() for t in l] for l in lists]
    tl = [pl.TensorList(l) for l in lists]
    sums = torch.zeros(2, dtype=torch.float64, device="cuda")
    scratch = torch.empty(max(pl.tile_grad_norm_scratch_bytes(t) for t in tl), dtype=torch.uint8, device="cuda")
    for i, t in enumerate(tl):
        pl.tile_grad_norm(0, t, scratch, sumsq=sums[i:])
    total = sums.sum().reshape(1)
    norm = torch.zeros(1, device="cuda")
    for t in tl:
        pl.tile_grad_scale(0, t, total, 2.5, norm=norm)
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for l in before for t in l))
    assert abs(float(norm) - want) <= 2.0 ** -21 * want
    for l, b in zip(lists, before):
        for t, o in zip(l, b):
            v = o.double() * (2.5 / want)
            assert bool(((t.double() - v).abs() <= (2.0 ** -8 + 2.0 ** -20) * v.abs()).all())


FRESH = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
import __graft_entry__ as e
pl = e.load_package()
pl.lib()

def ops(stream, M):
    N, K = 260, 203
    bf = dict(device="cuda", dtype=torch.bfloat16)
    A, B, D, P = torch.randn(M, K, **bf), torch.randn(N, K, **bf), torch.zeros(N, M, **bf), torch.zeros(N, M, **bf)
    dA, dB, db = torch.zeros_like(A), torch.zeros_like(B), torch.zeros(M, **bf)
    n = max(pl.tile_gemm_act_scratch_bytes(pl.BF16, "T", "N", M, N, K, A, K, B, K),
            pl.tile_gemm_act_grad_scratch_bytes(pl.BF16, "T", "N", M, N, K, A, K, B, K, pl.ACT_GELU))
    s = torch.empty(n, device="cuda", dtype=torch.uint8)
    lst = pl.TensorList([dA, dB, db])
    ls = torch.empty(pl.tile_grad_norm_scratch_bytes(lst), device="cuda", dtype=torch.uint8)
    norm = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    def f():
        kw = dict(scratch=s, scratch_bytes=n, stream=stream)
        pl.tile_gemm_act(0, pl.BF16, "T", "N", M, N, K, 1.0, A, K, B, K, 0.0, None, M, D, M, act=pl.ACT_GELU, pre=P,
                         ldPre=M, **kw)
        pl.tile_gemm_act_grad(0, pl.BF16, "T", "N", M, N, K, 1.0, A, K, B, K, pl.ACT_GELU, P, M, D, M, dA=dA, lddA=K,
                              dB=dB, lddB=K, dbias=db, **kw)
        pl.tile_grad_clip(0, lst, 0.5, ls, norm=norm, stream=stream)
    return f, (D, dA, dB, db, norm)

st = torch.cuda.Stream()
f, out = ops(st.cuda_stream, 515)
# a first call inside a capture is refused and the capture goes on
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=st):
    try:
        f()
        raise SystemExit("the first call was not refused")
    except pl.ParaliaError as ex:
        assert ex.code == pl.ERR_UNSUPPORTED, ex
    out[0].add_(1)
graph.replay()
torch.cuda.synchronize()
pl.fill_f32(torch.zeros(1, device="cuda"), 1, 0, 0, 0)
# set up, but none of these kernels has run: their first launches are captured
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=st):
    f()
graph.replay()
torch.cuda.synchronize()
pl.tile_status(0)
got = [t.clone() for t in out]
f()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, out)) and float(out[4]) > 0
# after a shutdown the library starts again
pl.finalize()
f()
torch.cuda.synchronize()
pl.tile_status(0)
assert all(torch.equal(a, b) for a, b in zip(got, out))
print("fresh ok")
"""


def test_first_calls_of_a_process():
    """In a process of its own: a first call inside a capture, first launches inside a capture, and a shutdown."""
    import subprocess
    root = str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", FRESH, root], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "fresh ok" in r.stdout, r.stdout + r.stderr
