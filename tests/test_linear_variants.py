"""Every variant of the mixed-precision product that the choice can pick, on shapes that make it pick it.

A variant is (rows on columns, columns of a tile, CTAs of a tile, CTAs that share its k). The tables hold the smallest
ragged shape found for each: ONE for a launch of one product, TWO for both products of a gradient in one launch. On the
CPU the choice itself is compiled and asked, for the tables and for drawn shapes, so that a variant without a shape is
noticed; on the GPU every shape is held to whole numbers, which any wrong index moves by a whole step."""
import math
import random
import subprocess
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))

TRANS = [("N", "N"), ("T", "N"), ("N", "T"), ("T", "T")]
# variant, whether results lie on the 16-byte grid, M x N x K
ONE = [
    ((0, 16, 1, 1), 0, (67, 83, 71)), ((0, 16, 1, 2), 0, (137, 519, 343)), ((0, 16, 1, 4), 0, (67, 67, 209)),
    ((0, 16, 1, 8), 1, (72, 72, 456)), ((0, 32, 1, 1), 0, (73, 4879, 67)), ((0, 32, 1, 2), 0, (155, 1159, 679)),
    ((0, 32, 1, 4), 0, (133, 637, 653)), ((0, 32, 1, 8), 0, (69, 601, 1307)), ((0, 48, 1, 1), 0, (145, 4937, 71)),
    ((0, 48, 1, 2), 0, (67, 3479, 1019)), ((0, 48, 1, 4), 0, (69, 2491, 735)), ((0, 48, 1, 8), 0, (141, 587, 1393)),
    ((0, 64, 1, 1), 0, (67, 14701, 71)), ((0, 64, 1, 2), 0, (77, 4425, 1131)), ((0, 64, 1, 4), 0, (73, 3793, 1175)),
    ((0, 64, 1, 8), 0, (129, 867, 3145)), ((0, 128, 1, 1), 0, (135, 16893, 325)),
    ((0, 128, 1, 2), 0, (131, 3525, 2691)), ((0, 128, 1, 4), 0, (137, 1599, 4957)),
    ((0, 128, 1, 8), 0, (129, 797, 9453)), ((0, 256, 2, 1), 0, (397, 14759, 71)), ((1, 64, 1, 1), 1, (136, 1848, 72)),
    ((1, 64, 1, 2), 1, (2184, 136, 808)), ((1, 64, 1, 4), 1, (136, 664, 728)), ((1, 64, 1, 8), 1, (144, 624, 568)),
    ((1, 128, 1, 1), 1, (4848, 136, 272)), ((1, 128, 1, 2), 1, (72, 5328, 1744)),
    ((1, 128, 1, 4), 1, (80, 2344, 2968)), ((1, 128, 1, 8), 1, (72, 1032, 5144)),
    ((1, 256, 2, 1), 1, (14512, 136, 72)),
]
# variant, grid, TransA, TransB, M x N x K of the forward product
TWO = [
    ((0, 16, 1, 1), 0, "N", "N", (67, 67, 69)), ((0, 16, 1, 2), 0, "T", "T", (71, 323, 71)),
    ((0, 16, 1, 4), 0, "T", "N", (199, 217, 71)), ((0, 16, 1, 8), 1, "N", "T", (456, 472, 24)),
    ((0, 32, 1, 1), 0, "N", "T", (77, 73, 2713)), ((0, 32, 1, 2), 0, "T", "N", (2349, 69, 67)),
    ((0, 32, 1, 4), 0, "T", "T", (1105, 197, 67)), ((0, 32, 1, 8), 1, "N", "N", (2008, 456, 24)),
    ((0, 48, 1, 1), 0, "N", "T", (73, 81, 4947)), ((0, 48, 1, 2), 0, "N", "N", (71, 2561, 129)),
    ((0, 48, 1, 4), 0, "T", "N", (1011, 203, 129)), ((0, 48, 1, 8), 0, "N", "N", (1329, 817, 25)),
    ((0, 64, 1, 1), 0, "N", "T", (69, 71, 7305)), ((0, 64, 1, 2), 0, "T", "T", (4017, 67, 133)),
    ((0, 64, 1, 4), 0, "T", "N", (195, 1539, 133)), ((0, 64, 1, 8), 0, "T", "T", (503, 3023, 25)),
    ((0, 128, 1, 1), 0, "N", "T", (257, 129, 10595)), ((0, 128, 1, 2), 0, "T", "N", (2937, 1769, 143)),
    ((0, 256, 2, 1), 0, "N", "T", (135, 153, 14319)), ((1, 64, 1, 1), 1, "N", "T", (72, 80, 1968)),
    ((1, 64, 1, 2), 1, "N", "N", (72, 2280, 152)), ((1, 64, 1, 4), 1, "T", "N", (520, 712, 72)),
    ((1, 64, 1, 8), 1, "T", "T", (856, 464, 72)), ((1, 128, 1, 1), 1, "T", "T", (136, 72, 11488)),
    ((1, 128, 1, 2), 1, "T", "N", (1784, 1568, 144)), ((1, 256, 2, 1), 1, "N", "T", (72, 136, 8480)),
]


def _products(ta, tb, M, N, K):
    """The two products of a gradient, that with more k first."""
    db = (K, N, M) if tb == "N" else (N, K, M)
    da = (M, K, N) if ta == "N" else (K, M, N)
    return [da, db] if da[2] > db[2] else [db, da]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    """choose([(products, grid)]) -> [[(products of the launch, variant), ...]]"""
    exe = tmp_path_factory.mktemp("plans") / "linear_plans"
    src = Path(__file__).resolve().parent / "cpp" / "linear_plans.cpp"
    r = subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-I/usr/local/cuda/include", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def ask(calls):
        text = "\n".join(f"{len(ps)} {grid} " + " ".join("%d %d %d" % p for p in ps) for ps, grid in calls)
        lines = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(lines) == len(calls)
        out = []
        for line in lines:
            v = [int(x) for x in line.split()]
            out.append([(v[i], tuple(v[i + 1:i + 5])) for i in range(0, len(v), 5)])
        return out
    return ask


def test_tables_hold_the_variants_they_say(choose):
    assert choose([([dims], grid) for _, grid, dims in ONE]) == [[(1, v)] for v, _, _ in ONE]
    assert choose([(_products(ta, tb, *dims), grid) for _, grid, ta, tb, dims in TWO]) == [[(2, v)] for v, *_ in TWO]
    for _, grid, *_, dims in ONE + TWO:
        assert not grid or all(d % 8 == 0 for d in dims)


def test_no_other_variant_is_picked(choose):
    rng = random.Random(12)
    size = lambda: int(round(math.exp(rng.uniform(0.0, math.log(20000)))))
    calls = []
    for _ in range(60000):
        dims, grid = (size(), size(), size()), rng.randint(0, 1)
        calls.append(([dims] if rng.random() < 0.5 else _products(*rng.choice(TRANS), *dims), grid))
    seen = {launch for launches in choose(calls) for launch in launches}
    known = {(1, v) for v, *_ in ONE} | {(2, v) for v, *_ in TWO}
    assert seen <= known, seen - known


@pytest.mark.gpu
@pytest.mark.parametrize("variant,grid,dims", ONE)
def test_one_product(pl, variant, grid, dims):
    import linear_defs as d
    import test_gemm_act_gpu as t
    for ta, tb in TRANS:
        t._forward(pl, d, "bf16", ta, tb, *dims, offset=1 - grid, ints=True, bias=True, beta=1.0, pre=True)
        t._forward(pl, d, "fp16", ta, tb, *dims, offset=1 - grid, ints=True, act="relu", beta=1.0, alias=True)
    t._forward(pl, d, "bf16", "T", "N", *dims, offset=1 - grid, act="silu", bias=True, pre=True)


@pytest.mark.gpu
@pytest.mark.parametrize("variant,grid,ta,tb,dims", TWO)
def test_both_products_of_a_gradient(pl, variant, grid, ta, tb, dims):
    import linear_defs as d
    import test_gemm_act_gpu as t
    t._grad(pl, d, "bf16", ta, tb, *dims, offset=1 - grid, ints=True)
    t._grad(pl, d, "fp16", ta, tb, *dims, offset=1 - grid, ints=True, act="relu", betas=(1.0, 1.0, 1.0))
    t._grad(pl, d, "bf16", ta, tb, *dims, offset=1 - grid, act="gelu", alpha=0.75)
