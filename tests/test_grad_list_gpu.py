"""Global gradient norm, clipping and scaling of tensor lists on the GPU against the definitions in 64 bits.

Tolerances: the sum of squares is carried in FP64 but for groups of eight 16-bit elements, whose squares
are exact in FP32 and whose sum has seven roundings of 2^-24 at most: 2^-21 relative. The norm then has half
of that and one rounding to FP32: 2^-22 + 2^-24. A scaled element has the factor's error (the norm's and a
rounding, below 2^-21), a product's rounding 2^-24 and its rounding to its own type."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu


def _types():
    import torch
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _half_step(dt):
    import torch
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    import torch
    return 2.0 ** -25 if dt == torch.float16 else 2.0 ** -134 if dt == torch.bfloat16 else 2.0 ** -150


def _list(sizes, dts, seed, scale=1e-2, offset=0):
    """Views of one NaN-filled buffer per type, at odd places."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    out, guards = [], []
    for i, n in enumerate(sizes):
        dt = dts[i % len(dts)]
        buf = torch.full((n + 32,), float("nan"), dtype=dt, device="cuda")
        at = (offset * (i + 1)) % 16
        v = buf[at:at + n]
        v.copy_(torch.randn(n, generator=g, device="cuda") * scale)
        out.append(v)
        guards.append((buf, at, n))
    return out, guards


def _intact(guards):
    import torch
    return all(bool(torch.isnan(b[:at]).all()) and bool(torch.isnan(b[at + n:]).all()) for b, at, n in guards)


def _norm(tensors):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in tensors))


def _scratch(pl, lst):
    import torch
    s = torch.empty(pl.tile_grad_norm_scratch_bytes(lst), dtype=torch.uint8, device="cuda")
    s.fill_(255)
    return s


SIZES = {
    "one": [1], "two": [0, 3, 0], "seven": [7, 8, 9, 1, 16, 15, 17], "edges": [4095, 4096, 4097, 4103, 4104, 8191],
    "mixed": [100_003, 5, 1, 4096, 70_000, 31], "large": [9_000_001, 17, 3_000_000],
    "many": [37 + i % 11 for i in range(1003)], "more": [9] * 2501,
}


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("types", [("fp32",), ("bf16",), ("fp16",), ("bf16", "fp32", "fp16")])
@pytest.mark.parametrize("offset", [0, 1, 5])
def test_norm_and_clip(pl, name, types, offset):
    import torch
    dts = [_types()[t] for t in types]
    g, guards = _list(SIZES[name], dts, seed=len(name), offset=offset)
    lst = pl.TensorList(g)
    s = _scratch(pl, lst)
    norm = torch.full((1,), -1.0, device="cuda")
    sumsq = torch.full((1,), -1.0, dtype=torch.float64, device="cuda")
    pl.tile_grad_norm(0, lst, s, norm=norm, sumsq=sumsq)
    want = _norm(g)
    assert abs(float(sumsq) - want ** 2) <= 2.0 ** -21 * want ** 2
    assert abs(float(norm) - want) <= (2.0 ** -22 + 2.0 ** -24) * want + 1e-45
    before = [t.clone() for t in g]
    # to other tensors, of other types, and from a norm in device memory
    for limit in (want * 0.3, want * 2.0):
        k = min(1.0, limit / want) if want else 1.0
        odt = [_types()[t] for t in ("bf16", "fp32", "fp16")]
        o, oguards = _list(SIZES[name], odt, seed=1, offset=offset + 1)
        for how in ("clip", "scale"):
            for t in o:
                t.fill_(float("nan"))
            l2 = pl.TensorList(g, o)
            norm.fill_(-1.0)
            if how == "clip":
                pl.tile_grad_clip(0, l2, limit, s, norm=norm)
            else:
                pl.tile_grad_scale(0, l2, sumsq, limit, norm=norm)
            assert abs(float(norm) - want) <= (2.0 ** -22 + 2.0 ** -24) * want
            for x, y in zip(g, o):
                v = x.double() * k
                tol = (_half_step(y.dtype) * (1 + 2.0 ** -20) + (2.0 ** -21 + 2.0 ** -23 if k < 1 else 0.0)) * v.abs() + _tiny(y.dtype)
                assert bool(((y.double() - v).abs() <= tol).all())
            assert _intact(oguards)
        assert all(torch.equal(a, b) for a, b in zip(before, g))
    # in place
    pl.tile_grad_clip(0, lst, want * 2.0, s)
    assert all(torch.equal(a, b) for a, b in zip(before, g))
    pl.tile_grad_clip(0, lst, want * 0.3, s, sumsq=sumsq)
    assert abs(float(sumsq) - want ** 2) <= 2.0 ** -21 * want ** 2
    for x, y in zip(before, g):
        v = x.double() * 0.3
        tol = (_half_step(y.dtype) * (1 + 2.0 ** -20) + 2.0 ** -21 + 2.0 ** -23) * v.abs() + _tiny(y.dtype)
        assert bool(((y.double() - v).abs() <= tol).all())
    assert _intact(guards)


def test_empty_list_and_zeros(pl):
    import torch
    norm = torch.full((1,), -1.0, device="cuda")
    for g in ([], [torch.empty(0, device="cuda")], [torch.zeros(1000, device="cuda").bfloat16(), -torch.zeros(77, device="cuda")]):
        lst = pl.TensorList(g)
        s = _scratch(pl, lst)
        norm.fill_(-1.0)
        pl.tile_grad_norm(0, lst, s, norm=norm)
        assert float(norm) == 0.0
        norm.fill_(-1.0)
        pl.tile_grad_clip(0, lst, 0.0, s, norm=norm)
        assert float(norm) == 0.0
        assert all(bool((t == 0).all()) for t in g)


@pytest.mark.parametrize("dtype,value", [("fp32", 3e38), ("fp32", 1e-42), ("bf16", 2e38), ("bf16", 1e-38), ("bf16", 1e-20),
                                         ("fp16", 60000.0), ("fp16", 6e-8)])
def test_ends_of_the_range(pl, dtype, value):
    # squares of these leave FP32; the sum is FP64's
    import torch
    dt = _types()[dtype]
    g = [torch.full((n,), value, device="cuda").to(dt) for n in (1001, 8, 3)]
    lst = pl.TensorList(g)
    s = _scratch(pl, lst)
    norm = torch.zeros(1, device="cuda")
    sumsq = torch.zeros(1, dtype=torch.float64, device="cuda")
    pl.tile_grad_norm(0, lst, s, norm=norm, sumsq=sumsq)
    want = _norm(g)
    assert abs(float(sumsq) - want * want) <= 2.0 ** -21 * want * want
    if want < 3.4e38:
        assert abs(float(norm) - want) <= 2.0 ** -21 * want + 1e-45
    else:
        assert math.isinf(float(norm))
    # a finite norm above FP32's range still clips by the right factor
    pl.tile_grad_clip(0, lst, 1.0, s)
    k = min(1.0, 1.0 / want)
    for t in g:
        v = value if dtype == "fp32" else float(torch.tensor(value).to(dt))
        assert abs(float(t[0]) - v * k) <= (_half_step(dt) * 1.01 + 2.0 ** -20) * abs(v * k) + 2 * _tiny(dt) + (
            2.0 ** -24 if dtype == "fp16" else 0.0)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_norm_that_is_not_finite_clips_nothing(pl, bad, dtype):
    import torch
    g, _ = _list([5000, 3], [_types()[dtype]], seed=2)
    g[0][4321] = bad
    before = [t.clone() for t in g]
    lst = pl.TensorList(g)
    norm = torch.zeros(1, device="cuda")
    pl.tile_grad_clip(0, lst, 1e-3, _scratch(pl, lst), norm=norm)
    assert not math.isfinite(float(norm))
    ints = {4: torch.int32, 2: torch.int16}[g[0].element_size()]
    assert all(torch.equal(a.view(ints), b.view(ints)) for a, b in zip(before, g))


def test_same_bits_every_time_and_graph(pl):
    import torch
    rng = random.Random(1)
    sizes = [rng.randint(1, 200_000) for _ in range(300)]
    g, _ = _list(sizes, [_types()["bf16"], _types()["fp32"]], seed=3, offset=1)
    lst = pl.TensorList(g)
    s = _scratch(pl, lst)
    sums = []
    for _ in range(3):
        q = torch.zeros(1, dtype=torch.float64, device="cuda")
        pl.tile_grad_norm(0, lst, s, sumsq=q)
        sums.append(float(q))
    assert len(set(sums)) == 1
    # captured, replayed on other values
    norm = torch.zeros(1, device="cuda")
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        pl.tile_grad_clip(0, lst, 1.0, s, norm=norm, stream=st.cuda_stream)
    for k in (1.0, 3.0):
        for t in g:
            t.normal_(0.0, k)
        want, first = _norm(g), g[0][:100].clone()
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - want) <= 2.0 ** -21 * want
        v = first.double() / want
        assert bool(((g[0][:100].double() - v).abs() <= 2.0 ** -7 * v.abs() + 1e-30).all())


def test_norm_of_a_shared_tensor_counts_it_twice(pl):
    import torch
    t = torch.full((1000,), 2.0, device="cuda")
    norm = torch.zeros(1, device="cuda")
    lst = pl.TensorList([t, t])
    pl.tile_grad_norm(0, lst, _scratch(pl, lst), norm=norm)
    assert abs(float(norm) - math.sqrt(8000.0)) <= 2.0 ** -22 * 90
    with pytest.raises(pl.ParaliaError):
        pl.tile_grad_clip(0, lst, 1.0, _scratch(pl, lst))


def test_offsets_beyond_32_bits(pl):
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    n = (1 << 32) + 4099
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[-1], t[1 << 31], t[0] = 3.0, 4.0, 12.0
    lst = pl.TensorList([t])
    norm = torch.zeros(1, device="cuda")
    s = _scratch(pl, lst)
    pl.tile_grad_norm(0, lst, s, norm=norm)
    assert float(norm) == 13.0
    pl.tile_grad_clip(0, lst, 6.5, s)
    assert float(t[-1]) == 1.5 and float(t[1 << 31]) == 2.0 and float(t[0]) == 6.0
