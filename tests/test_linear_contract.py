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
    return "no CUDA device" in text or f"GPU id {NO_GPU}" in text


def test_gradient_asks_for_no_scratch_that_it_does_not_touch(pl):
    none = dict(scratch=None, scratch_bytes=0)
    assert "bytes of scratch" in _grad(pl, **none) and _passes(_grad(pl))
    assert _passes(_grad(pl, N=0, B=0, dD=0, pre=0, **none))
    assert _passes(_grad(pl, act=pl.ACT_NONE, pre=0, **none))
    assert _passes(_grad(pl, dA=None, dB=None, **none))
    assert _passes(_grad(pl, alpha=0.0, **none))
    assert "bytes of scratch" in _grad(pl, act=pl.ACT_NONE, dD=D + 2, **none)       # dD has to be copied
    assert "bytes of scratch" in _grad(pl, act=pl.ACT_NONE, A=A + 2, **none)


class Tensor:
    """Looks like a GPU tensor at `address`."""

    def __init__(self, address, gpu=0, dtype="torch.uint8", numel=1 << 12, element_size=1):
        self.address, self.gpu, self.dtype, self.n, self.size, self.is_cuda = address, gpu, dtype, numel, element_size, True

    def data_ptr(self):
        return self.address

    def get_device(self):
        return self.gpu

    def numel(self):
        return self.n

    def element_size(self):
        return self.size

    @property
    def nbytes(self):
        return self.n * self.size

    def is_contiguous(self):
        return True


def _forward(pl, **kw):
    a = dict(dev=NO_GPU, type=pl.BF16, TransA="T", TransB="N", M=64, N=32, K=16, alpha=1.0, A=A, ldA=16, B=B, ldB=16,
             beta=1.0, Cm=CC, ldC=64, D=D, ldD=64, bias=DBIAS, pre=P, ldPre=64, scratch=S, scratch_bytes=4096)
    a.update(kw)
    with pytest.raises(pl.ParaliaError) as e:
        pl.tile_gemm_act(**a)
    return str(e.value)


def _lists(pl, lst, dev=NO_GPU, scratch=S, sumsq=D, norm=P):
    """What the three list routines say."""
    out = []
    for f in (lambda: pl.tile_grad_norm(dev, lst, scratch, norm=norm, sumsq=sumsq),
              lambda: pl.tile_grad_clip(dev, lst, 1.0, scratch, norm=norm, sumsq=sumsq),
              lambda: pl.tile_grad_scale(dev, lst, sumsq, 1.0, norm=norm)):
        with pytest.raises(pl.ParaliaError) as e:
            f()
        out.append(str(e.value))
    return out


def test_tensors_of_another_gpu_are_refused(pl):
    here, other = Tensor(A, NO_GPU), Tensor(A, 1)
    assert _passes(_forward(pl)) and _passes(_grad(pl))
    for name in ("A", "B", "Cm", "D", "bias", "pre", "scratch"):
        at = {"A": A, "B": B, "Cm": CC, "D": D, "bias": DBIAS, "pre": P, "scratch": S}[name]
        assert _passes(_forward(pl, **{name: Tensor(at, NO_GPU)})), name
        assert "is on GPU 1" in _forward(pl, **{name: Tensor(at, 1)}), name
    for name in ("A", "B", "pre", "dD", "dA", "dB", "dbias", "scratch"):
        assert "is on GPU 1" in _grad(pl, **{name: other}), name
    f32 = lambda address, gpu: Tensor(address, gpu, "torch.float32", 64, 4)
    lst = pl.TensorList([f32(A, 1), f32(B, 1)])
    assert all("is on GPU 1" in t for t in _lists(pl, lst))
    lst = pl.TensorList([f32(A, NO_GPU)], [f32(B, NO_GPU)])
    assert all(_passes(t) for t in _lists(pl, lst))
    f64 = Tensor(D, 1, "torch.float64", 1, 8)
    assert all("is on GPU 1" in t for t in _lists(pl, lst, sumsq=f64))
    assert all("is on GPU 1" in t for t in _lists(pl, lst, norm=f32(P, 1)))
    assert all("is on GPU 1" in t for t in _lists(pl, lst, scratch=Tensor(S, 1))[:2])
    for lists in (([f32(A, 0), f32(B, 1)],), ([f32(A, 0)], [f32(B, 1)])):
        with pytest.raises(pl.ParaliaError):
            pl.TensorList(*lists)
    assert _passes(_forward(pl, A=here))


def test_scratch_smaller_than_said_is_refused(pl):
    scratch = lambda numel, size=1: Tensor(S, NO_GPU, "torch.uint8", numel, size)
    for f in (_forward, _grad):
        assert _passes(f(pl, scratch=scratch(4096), scratch_bytes=4096))
        assert _passes(f(pl, scratch=scratch(1024, 4), scratch_bytes=4096))
        assert "scratch holds 4095 bytes" in f(pl, scratch=scratch(4095), scratch_bytes=4096)
    lst = pl.TensorList([Tensor(A, NO_GPU, "torch.float32", 64, 4)])
    n = pl.tile_grad_norm_scratch_bytes(lst)
    assert all(_passes(t) for t in _lists(pl, lst, scratch=scratch(n)))
    norm, clip, scale = _lists(pl, lst, scratch=scratch(n - 8))
    assert "scratch holds" in norm and "scratch holds" in clip and _passes(scale)


def test_scalars_of_another_type_are_refused(pl):
    lst = pl.TensorList([Tensor(A, NO_GPU, "torch.float32", 64, 4)])
    scalar = lambda address, dtype, size, numel=1: Tensor(address, NO_GPU, "torch." + dtype, numel, size)
    assert all(_passes(t) for t in _lists(pl, lst, sumsq=scalar(D, "float64", 8), norm=scalar(P, "float32", 4, 3)))
    for norm in (scalar(P, "float64", 8), scalar(P, "bfloat16", 2), scalar(P, "int32", 4), scalar(0, "float32", 4, 0)):
        assert all("where a float32 is" in t for t in _lists(pl, lst, norm=norm))
    for sumsq in (scalar(D, "float32", 4, 2), scalar(D, "int64", 8), scalar(0, "float64", 8, 0)):
        assert all("where a float64 is" in t for t in _lists(pl, lst, sumsq=sumsq))


SHARES = "may share memory"


@pytest.mark.parametrize("kw,refused", [
    # the last byte of one is the first of the other, and one element further none is shared
    (dict(D=A + 2 * 64 * 16 - 2), True), (dict(D=A + 2 * 64 * 16), False),
    (dict(A=D + 2 * 64 * 32 - 2), True), (dict(A=D + 2 * 64 * 32), False),
    (dict(B=D + 100), True), (dict(Cm=D + 2), True), (dict(Cm=D), False), (dict(Cm=D, ldC=72), True),
    (dict(Cm=D, N=1, ldC=72), False), (dict(bias=D + 126), True), (dict(bias=D + 2 * 64 * 32), False),
    (dict(pre=D + 2 * 64 * 32 - 2), True), (dict(pre=D + 2 * 64 * 32), False), (dict(pre=CC + 64), True),
    (dict(beta=0.0, Cm=D + 2), False),                                      # C is not read
    # one parent of 200 rows: D, pre and C in rows of their own
    (dict(D=D, ldD=200, pre=D + 128, ldPre=200, Cm=D + 256, ldC=200), False),
    (dict(D=D, ldD=200, pre=D + 126, ldPre=200), True), (dict(D=D + 128, ldD=200, pre=D, ldPre=200), False),
    (dict(D=D + 128, ldD=200, pre=D + 2, ldPre=200), True),
    # columns of the parent taken apart: rows 136 to 199 of a column, rows 0 to 63 of the next
    (dict(D=D + 272, ldD=200, pre=D + 400, ldPre=200), False), (dict(D=D + 272, ldD=200, pre=D + 398, ldPre=200), True),
    # two strides in one range: D has bytes 0 to 127 of every 800; pre at 400 k + 128, + 272 (up to 400 and 800), + 336 (736
    # to 863), at 402 k + 128 (never beyond 718 of 800) and at 434 k + 128 (698 to 825 for k = 5)
    (dict(D=D, ldD=400, pre=D + 128, ldPre=200), False), (dict(D=D, ldD=400, pre=D + 272, ldPre=200), False),
    (dict(D=D, ldD=400, pre=D + 336, ldPre=200), True), (dict(D=D, ldD=400, pre=D + 128, ldPre=201), False),
    (dict(D=D, ldD=400, pre=D + 128, ldPre=217), True), (dict(pre=D, ldPre=400, D=D + 128, ldD=217), True),
    # scratch: columns of A off the grid, 64 of 16 elements, copied
    (dict(A=A + 2, scratch=D + 2 * 64 * 32 - 16), True), (dict(A=A + 2, scratch=D + 2 * 64 * 32), False),
    (dict(A=A + 2, scratch=D - 2048), False), (dict(A=A + 2, scratch=D - 2032), True), (dict(scratch=D), False),
])
def test_outputs_that_overlap_operands(pl, kw, refused):
    text = _forward(pl, **kw)
    assert (SHARES in text) if refused else _passes(text), text


@pytest.mark.parametrize("kw,refused", [
    (dict(dA=A + 2 * 64 * 16 - 2), True), (dict(dA=A + 2 * 64 * 16), False), (dict(dB=DA + 32), True),
    (dict(dB=DA + 2 * 64 * 16), False), (dict(dbias=DA + 2), True), (dict(dbias=DB + 2 * 16 * 32 - 2), True),
    (dict(dbias=D + 4000), True), (dict(dbias=P + 4000), True), (dict(dA=P - 2), True),
    (dict(dA=P - 2, act=0), False), (dict(dA=P, act=0), False),            # without an activation pre is not read
    (dict(dA=DA, lddA=32, dB=DA + 32, lddB=32), False),                    # side by side in one parent
    (dict(dA=S + 4096), False), (dict(dA=S + 4094), True), (dict(dD=S + 64), True), (dict(act=0, dD=S), False),
    (dict(dbias=S, dA=None, dB=None), False),                              # nothing of the scratch is touched
])
def test_gradients_that_overlap(pl, kw, refused):
    text = _grad(pl, **kw)
    assert (SHARES in text) if refused else _passes(text), text


def test_overlaps_of_random_matrices(pl):
    """Three matrices in a range of 700 elements, their elements counted one by one."""
    import random
    rng = random.Random(6)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        M, N = rng.randint(1, 12), rng.randint(1, 12)
        m = [(rng.randrange(0, 700), M + rng.choice((0, 0, rng.randrange(60)))) for _ in range(3)]
        cells = [{at + i + j * ld for j in range(N) for i in range(M)} for at, ld in m]
        d, p, c = cells
        in_place = m[0] == m[2] or N == 1 and m[0][0] == m[2][0]
        shared = bool(d & p or p & c or (d & c and not in_place))
        text = _forward(pl, M=M, N=N, A=A, B=B, bias=0, scratch=0, scratch_bytes=0, D=D + 2 * m[0][0], ldD=m[0][1],
                        pre=D + 2 * m[1][0], ldPre=m[1][1], Cm=D + 2 * m[2][0], ldC=m[2][1])
        assert (SHARES in text) == shared and _passes(text) != shared, (M, N, m, text)
        seen[shared] += 1
    assert min(seen.values()) > 300


def test_results_and_scratch_of_lists_stand_apart(pl):
    f32 = lambda address, numel=64: Tensor(address, NO_GPU, "torch.float32", numel, 4)
    lists = [pl.TensorList([f32(A), f32(B)]), pl.TensorList([f32(A), f32(CC, 0), f32(B)], [f32(DA), f32(CC, 0), f32(DB)])]
    text = "share memory with nothing"
    for k, lst in enumerate(lists):
        n = pl.tile_grad_norm_scratch_bytes(lst)
        assert all(_passes(t) for t in _lists(pl, lst))
        # norm inside sumsq, in either half: blocks that read the sum would see the norm
        for norm in (D, D + 4):
            assert all(text in t for t in _lists(pl, lst, norm=norm))
        assert all(_passes(t) for t in _lists(pl, lst, norm=D + 8)) and all(_passes(t) for t in _lists(pl, lst, norm=D - 4))
        # a result in the scratch or behind it
        for sumsq, bad in ((S, True), (S + n - 8, True), (S + n, False), (S - 8, False)):
            got = _lists(pl, lst, sumsq=sumsq)
            assert [text in t for t in got] == [bad, bad, False] and _passes(got[2])
        # over a tensor, in its last element and behind it
        for norm, bad in ((A, True), (B + 252, True), (B + 256, False), (A - 4, False)):
            assert all((text in t) == bad and _passes(t) != bad for t in _lists(pl, lst, norm=norm)), (k, norm)
        for sumsq, bad in ((A + 248, True), (A + 256, False)):
            assert all((text in t) == bad for t in _lists(pl, lst, sumsq=sumsq)), (k, sumsq)
        for scratch, bad in ((B + 248, True), (B + 256, False), (A - n + 8, True), (A - n, False)):
            assert [text in t for t in _lists(pl, lst, scratch=scratch)] == [bad, bad, False], (k, scratch)
    for at, bad in ((DA + 252, True), (DB + 256, False)):     # an output: not where only the tensors are read
        assert [text in t for t in _lists(pl, lists[1], norm=at)] == [False, bad, bad], at
