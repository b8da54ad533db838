"""Attention of drafted trees, decode steps with weight sums, cache eviction,
beam selection and state reordering against plain 64-bit forms.

Tolerances.  u = 2^-24 is the largest relative error of one fp32 rounding.  A
sum of n rounded terms is off by at most LAM sqrt(n) u times the sum of their
magnitudes but for a probability below 2 exp(-LAM^2 / 2) (Higham and Mary's
probabilistic rounding analysis); LAM = 8.  Products of fp32 values split into
fp16 pairs keep 22 bits of each factor and drop one product: 3 * 2^-22 = 12 u; a
tensor-core sum that is cut instead of rounded is off by 2 u an addition: one
per 16 columns and product, so C = 3 hd / 16 of them in a score (24 is taken
for the smaller heads too), at most 12 in a tile's output.  So a score is off by
  ds = (LAM sqrt(hd) + 12 + 2 C + 2) u * scale * sum |q k|,
a weight by the factor 1 + 2 ds (its numerator and its sum), the exponentials
(2 + |x|) u each with |x| <= 40 where the weight counts, and an output by
  (2 max ds + (LAM sqrt(n) + 12 + 2 * 12 + 42) u) * sum_j p_j |v_j|.
"""
import ctypes

import numpy as np
import pytest

from gncx_b200 import core

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U, LAM = 2.0**-24, 8.0
INVALID, UNALIGNED, UNREACHABLE, CAPACITY = 1, 2, 6, 8


def P(t):
    return None if t is None else t.data_ptr()


def ok(lib, status):
    if status:
        core.check(lib)
    assert status == 0


@pytest.fixture(autouse=True)
def _clean(gpu):
    gpu.gncx_set_synchronous(1)
    yield
    torch.cuda.synchronize()
    gpu.gncx_clear_error()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def attend(q, k, v, scale):
    """q [hd], k and v [n, hd] -> (output, its tolerance, weights, their relative tolerance), all in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    n, hd = k.shape
    s = (k @ q) * scale
    ds = (LAM * hd**0.5 + 14 + 2 * max(24, 3 * ((hd + 15) // 16))) * U * abs(scale) * float((k.abs() @ q.abs()).max())
    p = torch.softmax(s, 0)
    rel = 2 * ds + (LAM * n**0.5 + 78) * U
    return p @ v, rel * (p @ v.abs()) + 1e-30, p, rel


# ---------------------------------------------------------------- tree
def make_tree(kind, n, seed):
    r = np.random.default_rng(seed)
    if kind == "chain":
        return np.arange(n) - 1
    if kind == "star":
        return np.full(n, -1)
    return np.array([-1] + [int(r.integers(-1, i)) for i in range(1, n)])


def tree_path(up, i):
    path = [i]
    while up[path[0]] >= 0:
        path.insert(0, int(up[path[0]]))
    return path


def tree_seen(up, i, pos0, window):
    """Cache rows that node i sees."""
    path = tree_path(up, i)
    pos = pos0 + len(path) - 1
    first = max(0, pos - window + 1) if window > 0 else 0
    return list(range(min(first, pos0), pos0)) + [pos0 + a for d, a in enumerate(path) if pos0 + d >= first]


def run_tree(lib, q, k, v, up, pos0, scale, window, ws=None, out=None):
    n, nh, hd = q.shape
    if out is None:
        out = torch.full_like(q, float("nan"))
    parents = torch.tensor(np.asarray(up), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ok(lib, lib.gncx_attention_tree(P(q), P(k), P(v), P(parents), pos0, n, nh, k.shape[1], hd, scale, window, P(out), P(ws),
                                    ws.numel() if ws is not None else 0))
    torch.cuda.synchronize()
    return out


def check_tree(out, q, k, v, up, pos0, scale, window, nodes=None):
    n, nh, hd = q.shape
    group = nh // k.shape[1]
    for i in range(n) if nodes is None else nodes:
        rows = torch.tensor(tree_seen(up, i, pos0, window), device="cuda")
        ks, vs = k[rows], v[rows]
        for h in range(nh):
            ref, tol, _, _ = attend(q[i, h], ks[:, h // group], vs[:, h // group], scale)
            err = (out[i, h].double() - ref).abs()
            assert bool((err <= tol).all()), (i, h, float((err / tol).max()))


TREES = [(1, 1, 4, 0, 1, 0), (4, 2, 64, 0, 1, 0), (4, 2, 64, 1, 1, 0), (4, 4, 64, 0, 9, 0), (8, 1, 128, 31, 7, 0),
         (6, 2, 96, 5, 40, 0), (16, 8, 128, 511, 5, 0), (32, 8, 128, 1000, 33, 0), (16, 8, 64, 257, 64, 0), (8, 4, 256, 300, 9, 0),
         (3, 1, 80, 129, 17, 0), (5, 5, 20, 70, 30, 0), (12, 1, 128, 200, 11, 0), (40, 2, 64, 130, 6, 0),
         (4, 2, 64, 500, 20, 1), (4, 2, 64, 500, 20, 7), (4, 2, 128, 500, 20, 33), (16, 4, 64, 3001, 25, 1024),
         (8, 8, 128, 63, 90, 100), (4, 1, 128, 100, 20, 4000), (2, 2, 128, 640, 1, 64), (2, 2, 128, 640, 1, 65),
         (24, 8, 128, 4099, 43, 0), (64, 8, 64, 700, 48, 0)]


@pytest.mark.parametrize("nh,nkv,hd,pos0,n,window", TREES)
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_tree(gpu, nh, nkv, hd, pos0, n, window, kind):
    rows = pos0 + n
    q, k, v = randn(1, n, nh, hd) * 2, randn(2, rows + 3, nkv, hd), randn(3, rows + 3, nkv, hd)
    k[rows:], v[rows:] = float("nan"), float("nan")  # rows behind the drafted ones
    lo = max(0, pos0 - window + 1) if window else 0
    k[:min(lo, pos0)], v[:min(lo, pos0)] = float("nan"), float("inf")  # rows that no window reaches
    up = make_tree(kind, n, pos0 + n)
    keep = k.clone(), v.clone()
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window)
    nodes = sorted({0, 1, n // 2, n - 2, n - 1, *range(0, n, 7)} & set(range(n)))
    check_tree(out, q, k, v, up, pos0, hd**-0.5, window, nodes)
    assert torch.equal(k.view(torch.int32), keep[0].view(torch.int32)) and torch.equal(v.view(torch.int32), keep[1].view(torch.int32))


@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_tree_of_1024(gpu, kind):
    n, pos0 = 1024, 77
    q, k, v = randn(4, n, 2, 32), randn(5, pos0 + n, 1, 32), randn(6, pos0 + n, 1, 32)
    up = make_tree(kind, n, 9)
    for window in (0, 50):
        out = run_tree(gpu, q, k, v, up, pos0, 0.2, window)
        check_tree(out, q, k, v, up, pos0, 0.2, window, [0, 1, 31, 32, 511, 1023])


def test_tree_long(gpu):
    """Heavy rows at the ends of a long cache, where a lost row would show."""
    nh, nkv, hd, pos0, n = 32, 8, 128, 33001, 64
    q, k, v = randn(7, n, nh, hd), randn(8, pos0 + n, nkv, hd), randn(9, pos0 + n, nkv, hd)
    for row in (0, 1, 8191, 16384, pos0 - 2, pos0 - 1):
        k[row] *= 8
    up = make_tree("random", n, 3)
    check_tree(run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0), q, k, v, up, pos0, hd**-0.5, 0, [0, 13, 40, 63])


@pytest.mark.parametrize("qs,ks,vs", [(1e-3, 1e-6, 1e-20), (1e4, 1e-3, 1e20), (1e-18, 1e18, 1e30), (1.0, 1.0, 1e-30)])
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_scales(gpu, qs, ks, vs, hd):
    """Values far from 1, and rows of very different size next to each other."""
    nh, nkv, pos0, n = 8, 2, 700, 24
    q, k, v = randn(10, n, nh, hd) * qs, randn(11, pos0 + n, nkv, hd) * ks, randn(12, pos0 + n, nkv, hd) * vs
    k *= 2.0 ** torch.randint(-20, 3, (pos0 + n, nkv, 1), device="cuda", generator=gen(13))
    v *= 2.0 ** torch.randint(-20, 1, (pos0 + n, nkv, 1), device="cuda", generator=gen(14))
    up = make_tree("random", n, 5)
    check_tree(run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0), q, k, v, up, pos0, hd**-0.5, 0, [0, 5, 23])


@pytest.mark.parametrize("hd", [64, 96, 128])
def test_tree_peaked_softmax(gpu, hd):
    """Scores far apart: all weight on few rows, in any split."""
    nh, nkv, pos0, n = 8, 2, 3000, 17
    q, k, v = randn(15, n, nh, hd) * 6, randn(16, pos0 + n, nkv, hd) * 3, randn(17, pos0 + n, nkv, hd)
    up = make_tree("random", n, 6)
    check_tree(run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0), q, k, v, up, pos0, hd**-0.5, 0)


# Several tiles of 64 rows per CTA and at most 128 query rows (148 SMs), where two
# lanes share the rows: whole and odd numbers of tiles, a last split of one row,
# the largest such group, one beyond it.
LANES = [(32, 32, 64, 1700, 9), (32, 32, 128, 1999, 11), (64, 32, 96, 3333, 40), (30, 30, 80, 2700, 3), (148, 148, 64, 450, 5),
         (148, 148, 128, 385, 2), (148, 148, 128, 400, 1), (20, 10, 128, 4993, 7), (64, 16, 128, 5000, 32), (64, 16, 128, 5000, 33),
         (8, 1, 128, 70001, 16)]


@pytest.mark.parametrize("nh,nkv,hd,pos0,n", LANES)
@pytest.mark.parametrize("size", [1.0, 5.0])
def test_tree_lanes(gpu, nh, nkv, hd, pos0, n, size):
    rows = pos0 + n
    q, k, v = randn(40, n, nh, hd) * size, randn(41, rows + 3, nkv, hd), randn(42, rows + 3, nkv, hd)
    k[rows:], v[rows:] = float("nan"), float("nan")
    for row in (0, 63, 64, 127, 128, 200, pos0 - 1):  # heavy rows on both sides of the tiles' borders
        k[row] *= 4
    up = make_tree("random", n, 11)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    heads = sorted({0, nh // 2, nh - 1})
    for i in sorted({0, n // 2, n - 1}):
        rs = torch.tensor(tree_seen(up, i, pos0, 0), device="cuda")
        for h in heads:
            g = h // (nh // nkv)
            ref, tol, _, _ = attend(q[i, h], k[rs][:, g], v[rs][:, g], hd**-0.5)
            assert bool(((out[i, h].double() - ref).abs() <= tol).all()), (i, h)
    assert bool(out.isfinite().all())
    assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0))


@pytest.mark.parametrize("row", [3, 70, 388, 1750, 1799])
def test_tree_lanes_infinite_and_nan_rows_show(gpu, row):
    nh, nkv, hd, pos0, n = 32, 32, 128, 1800, 6
    q, k, v = randn(43, n, nh, hd), randn(44, pos0 + n, nkv, hd), randn(45, pos0 + n, nkv, hd)
    v[row, 4, 9], k[row, 7, 2] = float("-inf"), float("nan")
    out = run_tree(gpu, q, k, v, make_tree("random", n, 12), pos0, hd**-0.5, 0)
    assert bool((out[:, 4, 9] == float("-inf")).all()) and bool(out[:, 7].isnan().all())
    out[:, 4, 9], out[:, 7] = 0, 0
    assert bool(out.isfinite().all())


# Head sizes above 128: tiles of 32 rows, 128 query rows at a time.
WIDE = [(1, 1, 256, 1, 1, 0), (1, 1, 256, 31, 1, 0), (2, 1, 256, 32, 3, 0), (2, 1, 256, 33, 3, 0), (4, 2, 144, 200, 9, 0), (8, 4, 256, 1000, 31, 0),
        (8, 2, 160, 777, 33, 0), (16, 4, 256, 2500, 32, 0), (4, 1, 192, 1537, 64, 0), (12, 4, 240, 5000, 11, 0), (148, 148, 256, 230, 3, 0),
        (74, 74, 256, 417, 2, 0), (4, 1, 256, 5000, 20, 700), (8, 2, 208, 300, 90, 33), (16, 4, 256, 9001, 64, 0)]


@pytest.mark.parametrize("nh,nkv,hd,pos0,n,window", WIDE)
@pytest.mark.parametrize("size", [1.0, 5.0])
def test_tree_wide(gpu, nh, nkv, hd, pos0, n, window, size):
    rows = pos0 + n
    q, k, v = randn(52, n, nh, hd) * size, randn(53, rows + 3, nkv, hd), randn(54, rows + 3, nkv, hd)
    k[rows:], v[rows:] = float("nan"), float("nan")
    lo = max(0, pos0 - window + 1) if window else 0
    k[:min(lo, pos0)], v[:min(lo, pos0)] = float("nan"), float("inf")
    for row in {min(lo, pos0 - 1), pos0 // 2, pos0 - 1}:
        k[row] *= 3
    up = make_tree("random", n, 13)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window)
    assert bool(out.isfinite().all())
    for i in sorted({0, n // 2, n - 1}):
        rs = torch.tensor(tree_seen(up, i, pos0, window), device="cuda")
        for h in sorted({0, nh // 2, nh - 1}):
            g = h // (nh // nkv)
            ref, tol, _, _ = attend(q[i, h], k[rs][:, g], v[rs][:, g], hd**-0.5)
            err = (out[i, h].double() - ref).abs()
            assert bool((err <= tol).all()), (i, h, float((err / tol).max()))
    assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window))


@pytest.mark.parametrize("qs,ks,vs", [(1e-3, 1e-6, 1e-20), (1e4, 1e-3, 1e20), (1e-18, 1e18, 1e30), (1.0, 1.0, 1e-30)])
def test_tree_wide_scales(gpu, qs, ks, vs):
    nh, nkv, hd, pos0, n = 8, 2, 256, 700, 24
    q, k, v = randn(55, n, nh, hd) * qs, randn(56, pos0 + n, nkv, hd) * ks, randn(57, pos0 + n, nkv, hd) * vs
    k *= 2.0 ** torch.randint(-20, 3, (pos0 + n, nkv, 1), device="cuda", generator=gen(58))
    v *= 2.0 ** torch.randint(-20, 1, (pos0 + n, nkv, 1), device="cuda", generator=gen(59))
    up = make_tree("random", n, 5)
    check_tree(run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0), q, k, v, up, pos0, hd**-0.5, 0, [0, 5, 23])


@pytest.mark.parametrize("row", [0, 45, 1290, 1301])
@pytest.mark.parametrize("col", [9, 128, 255])
def test_tree_wide_infinite_and_nan_rows_show(gpu, row, col):
    nh, nkv, hd, pos0, n = 16, 16, 256, 1302, 6
    q, k, v = randn(60, n, nh, hd), randn(61, pos0 + n, nkv, hd), randn(62, pos0 + n, nkv, hd)
    v[row, 4, col], k[row, 7, col] = float("inf"), float("nan")
    out = run_tree(gpu, q, k, v, make_tree("random", n, 14), pos0, hd**-0.5, 0)
    assert bool((out[:, 4, col] == float("inf")).all()) and bool(out[:, 7].isnan().all())
    out[:, 4, col], out[:, 7] = 0, 0
    assert bool(out.isfinite().all())


# Few query rows and a short cache, one launch of clusters: on both sides of its limits
# of query rows (8 and 16 per cluster, 15 clusters), nodes (64) and cache rows.
FEW = [(1, 1, 128, 0, 1, 0), (1, 1, 128, 0, 64, 0), (1, 1, 128, 0, 65, 0), (2, 1, 64, 3, 60, 5), (16, 8, 128, 764, 4, 0), (16, 8, 128, 765, 4, 0),
       (16, 8, 128, 379, 5, 0), (16, 8, 128, 380, 5, 0), (16, 8, 128, 300, 8, 0), (16, 8, 128, 300, 9, 0), (4, 4, 256, 250, 6, 0),
       (4, 4, 256, 251, 6, 0), (15, 15, 128, 200, 8, 0), (16, 16, 128, 200, 8, 0), (24, 8, 128, 5000, 2, 200), (8, 1, 20, 90, 14, 0),
       (12, 4, 252, 200, 2, 90), (3, 1, 36, 7, 5, 2), (4, 2, 128, 600, 4, 1), (5, 1, 64, 40, 24, 0)]


@pytest.mark.parametrize("nh,nkv,hd,pos0,n,window", FEW)
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_tree_few(gpu, nh, nkv, hd, pos0, n, window, kind):
    rows = pos0 + n
    q, k, v = randn(63, n, nh, hd) * 2, randn(64, rows + 3, nkv, hd), randn(65, rows + 3, nkv, hd)
    k[rows:], v[rows:] = float("nan"), float("nan")
    lo = max(0, pos0 - window + 1) if window else 0
    k[:min(lo, pos0)], v[:min(lo, pos0)] = float("nan"), float("inf")
    up = make_tree(kind, n, pos0 + n + 1)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window)
    check_tree(out, q, k, v, up, pos0, hd**-0.5, window)
    assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("pos0,n", [(40, 7), (0, 16), (300, 8)])
def test_tree_few_other_branches_do_not_leak(gpu, bad, pos0, n):
    nh, nkv, hd = 4, 4, 64
    q, k, v = randn(66, n, nh, hd), randn(67, pos0 + n, nkv, hd), randn(68, pos0 + n, nkv, hd)
    up = make_tree("random", n, 7)
    k[pos0 + 3], v[pos0 + 3] = bad, bad
    clean = [i for i in range(n) if 3 not in tree_path(up, i)]
    assert 1 < len(clean) < n
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    check_tree(out, q, k, v, up, pos0, hd**-0.5, 0, clean)
    assert not bool(out[3].isfinite().any())


def test_tree_few_bad_parents_are_an_error(gpu):
    q, k, v = randn(69, 4, 2, 64), randn(70, 24, 2, 64), randn(71, 24, 2, 64)
    out = torch.zeros_like(q)
    for up in ([-1, 1, 0, 0], [-1, 0, 3, 0], [-1, 0, -2, 0], [5, 0, 0, 0], [-1, 0, 0, 2**31 - 1]):
        parents = torch.tensor(up, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        st = gpu.gncx_attention_tree(P(q), P(k), P(v), P(parents), 20, 4, 2, 2, 64, 0.1, 0, P(out), None, 0)
        assert st == INVALID and gpu.gncx_last_error() == INVALID, up
        gpu.gncx_clear_error()
    ok(gpu, gpu.gncx_sync())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_tree_other_branches_do_not_leak(gpu, bad):
    nh, nkv, hd, pos0, n = 8, 2, 128, 300, 40
    q, k, v = randn(18, n, nh, hd), randn(19, pos0 + n, nkv, hd), randn(20, pos0 + n, nkv, hd)
    up = make_tree("random", n, 7)
    up[3] = 1
    k[pos0 + 3], v[pos0 + 3] = bad, bad
    clean = [i for i in range(n) if 3 not in tree_path(up, i)]
    assert 5 < len(clean) < n
    check_tree(run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0), q, k, v, up, pos0, hd**-0.5, 0, clean)


@pytest.mark.parametrize("hd", [64, 128])
def test_tree_infinite_and_nan_rows_show(gpu, hd):
    """A NaN in a seen row reaches the outputs of its KV head, and no other head's."""
    nh, nkv, pos0, n = 4, 2, 400, 8
    q, k, v = randn(21, n, nh, hd), randn(22, pos0 + n, nkv, hd), randn(23, pos0 + n, nkv, hd)
    k[250, 0, 5] = float("nan")
    up = make_tree("random", n, 8)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    assert bool(out[:, :2].isnan().all())
    v2 = v.clone()
    v2[100, 1, 7] = float("inf")
    k[250, 0, 5] = 0
    out2 = run_tree(gpu, q, k, v2, up, pos0, hd**-0.5, 0)
    assert bool((out2[:, 2:, 7] == float("inf")).all()) and bool(out2[:, :2].isfinite().all())
    assert bool(out[:, 2:].isfinite().all()) and bool(out2[:, 2:, :7].isfinite().all()) and bool(out2[:, 2:, 8:].isfinite().all())


@pytest.mark.parametrize("nh,nkv,hd,pos0,n,window", [(16, 8, 128, 700, 12, 0), (8, 2, 64, 300, 30, 40)])
def test_tree_chain_is_sequential_decoding(gpu, nh, nkv, hd, pos0, n, window):
    q, k, v = randn(24, n, nh, hd), randn(25, pos0 + n, nkv, hd), randn(26, pos0 + n, nkv, hd)
    out = run_tree(gpu, q, k, v, make_tree("chain", n, 0), pos0, hd**-0.5, window)
    for i in range(n):
        y = torch.empty(nh, hd, device="cuda")
        torch.cuda.synchronize()
        gpu.gncx_mqa_attention_step_ext(P(q[i].contiguous()), None, None, P(k), P(v), pos0 + i, nh, nkv, hd, hd**-0.5, window, 0, P(y))
        core.check(gpu)
        assert float((out[i] - y).abs().max()) <= 1e-5 * float(y.abs().max())


def test_tree_is_deterministic(gpu):
    n, pos0 = 33, 5001
    q, k, v = randn(27, n, 16, 128), randn(28, pos0 + n, 4, 128), randn(29, pos0 + n, 4, 128)
    up = make_tree("random", n, 10)
    first = run_tree(gpu, q, k, v, up, pos0, 0.1, 0)
    for _ in range(3):
        assert torch.equal(first, run_tree(gpu, q, k, v, up, pos0, 0.1, 0))


def test_tree_bad_parents_are_an_error(gpu):
    q, k, v = randn(30, 4, 4, 64), randn(31, 104, 2, 64), randn(32, 104, 2, 64)
    out = torch.zeros_like(q)
    for up in ([-1, 1, 0, 0], [-1, 0, 3, 0], [-1, 0, -2, 0], [5, 0, 0, 0], [-1, 0, 0, 2**31 - 1]):
        parents = torch.tensor(up, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        st = gpu.gncx_attention_tree(P(q), P(k), P(v), P(parents), 100, 4, 4, 2, 64, 0.1, 0, P(out), None, 0)
        assert st == INVALID and gpu.gncx_last_error() == INVALID, up
        gpu.gncx_clear_error()
    ok(gpu, gpu.gncx_sync())


def test_tree_workspace(gpu):
    n, pos0, nh, nkv, hd = 9, 3000, 8, 2, 128
    need = gpu.gncx_attention_tree_workspace(pos0, n, nh, nkv, hd, 0)
    sizes = [gpu.gncx_attention_tree_workspace(p, n, nh, nkv, hd, 0) for p in range(0, 6000, 37)]
    assert sizes == sorted(sizes)
    q, k, v = randn(33, n, nh, hd), randn(34, pos0 + n, nkv, hd), randn(35, pos0 + n, nkv, hd)
    up = make_tree("random", n, 1)
    guard = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    out = run_tree(gpu, q, k, v, up, pos0, 0.1, 0, ws=guard[:need])
    assert bool((guard[need:] == 0xA5).all())
    assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, 0.1, 0))
    parents = torch.tensor(up, dtype=torch.int32, device="cuda")
    before = out.clone()
    args = (P(q), P(k), P(v), P(parents), pos0, n, nh, nkv, hd, 0.1, 0, P(out))
    assert gpu.gncx_attention_tree(*args, P(guard), need - 1) == CAPACITY
    assert gpu.gncx_attention_tree(*args, P(guard) + 8, need) == UNALIGNED
    host = (ctypes.c_float * 4096)()
    assert gpu.gncx_attention_tree(P(q) + 4, *args[1:], None, 0) == UNALIGNED
    assert gpu.gncx_attention_tree(None, *args[1:], None, 0) == INVALID
    assert gpu.gncx_attention_tree(*args[:3], (ctypes.addressof(host) + 15) & ~15, *args[4:], None, 0) == UNREACHABLE
    torch.cuda.synchronize()
    assert torch.equal(out, before)


# ---------------------------------------------------------------- decode step with weight sums
def run_step(lib, q, k_new, v_new, k, v, pos, token_pos, scale, write, weight, positions, ws=None):
    nh, hd = q.shape
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    ok(lib, lib.gncx_mqa_attention_step_weights(P(q), P(k_new), P(v_new), P(k), P(v), pos, token_pos, nh, k.shape[1], hd, scale,
                                                write, P(out), P(weight), P(positions), weight.shape[1], P(ws),
                                                ws.numel() if ws is not None else 0))
    torch.cuda.synchronize()
    return out


STEPS = [(1, 1, 4, 0), (4, 2, 64, 0), (4, 2, 64, 1), (4, 4, 128, 30), (4, 4, 128, 31), (4, 4, 128, 32), (6, 2, 96, 33), (8, 1, 256, 100),
         (16, 8, 128, 511), (32, 8, 128, 1000), (3, 1, 80, 1023), (12, 4, 64, 1024), (10, 2, 128, 1025), (7, 7, 20, 2500),
         (40, 2, 64, 300), (32, 8, 128, 20011), (24, 1, 128, 4100),
         # the last of one launch, the first of two; groups of 1 to 5 heads
         (4, 2, 64, 4095), (4, 2, 64, 4096), (8, 4, 128, 2047), (8, 4, 128, 2048), (4, 1, 256, 511), (4, 1, 256, 512), (3, 1, 96, 2729),
         (3, 1, 96, 2730), (5, 1, 64, 500), (2, 2, 4, 4095), (6, 3, 60, 7), (8, 2, 128, 8)]


@pytest.mark.parametrize("nh,nkv,hd,pos", STEPS)
@pytest.mark.parametrize("write", [0, 1])
def test_step_weights(gpu, nh, nkv, hd, pos, write):
    stride = pos + 4
    q, k, v = randn(40, nh, hd) * 2, randn(41, pos + 3, nkv, hd), randn(42, pos + 3, nkv, hd)
    k_new, v_new = randn(43, nkv, hd), randn(44, nkv, hd)
    k[pos + 1:], v[pos + 1:] = float("nan"), float("nan")
    if write:  # what an evicted row left there
        k[pos], v[pos] = float("nan"), float("inf")
    weight = torch.rand(nkv, stride, device="cuda", generator=gen(45))
    positions = torch.arange(stride, dtype=torch.int32, device="cuda").repeat(nkv, 1) * 3
    if write:
        weight[:, pos] = float("nan")
    w0, p0, k0, v0 = weight.clone(), positions.clone(), k.clone(), v.clone()
    out = run_step(gpu, q, k_new if write else None, v_new if write else None, k, v, pos, 10**6, hd**-0.5, write, weight, positions)
    if write:
        k0[pos], v0[pos], p0[:, pos] = k_new, v_new, 10**6
        w0[:, pos] = 0
    assert torch.equal(k.view(torch.int32), k0.view(torch.int32)) and torch.equal(v.view(torch.int32), v0.view(torch.int32))
    assert torch.equal(positions, p0)
    assert torch.equal(weight[:, pos + 1:], w0[:, pos + 1:])
    group = nh // nkv
    for c in range(nkv):
        add, tol_w = torch.zeros(pos + 1, dtype=torch.float64, device="cuda"), 0.0
        for h in range(c * group, (c + 1) * group):
            ref, tol, p, rel = attend(q[h], k0[:pos + 1, c], v0[:pos + 1, c], hd**-0.5)
            err = (out[h].double() - ref).abs()
            assert bool((err <= tol).all()), (h, float((err / tol).max()))
            add += p
            tol_w = max(tol_w, rel)
        ref_w = w0[c, :pos + 1].double() + add
        err = (weight[c, :pos + 1].double() - ref_w).abs()
        assert bool((err <= (tol_w + (group + 1) * U) * add + U * ref_w + 1e-38).all()), c


@pytest.mark.parametrize("rows", [(0, 401), (31, 62), (100, 300), (17, 18), (400, 401)])
def test_step_weights_nan_rows_show(gpu, rows):
    """A NaN among a KV head's scores makes its weights and outputs NaN, also where it fills a whole range of rows."""
    nh, nkv, hd, pos = 4, 2, 64, 400
    q, k, v = randn(49, nh, hd), randn(50, pos + 1, nkv, hd), randn(51, pos + 1, nkv, hd)
    k[rows[0]:rows[1], 0, 5] = float("nan")
    weight = torch.ones(nkv, pos + 1, device="cuda")
    out = run_step(gpu, q, None, None, k, v, pos, pos, hd**-0.5, 0, weight, None)
    assert bool(out[:2].isnan().all()) and bool(weight[0].isnan().all())
    assert bool(out[2:].isfinite().all()) and bool(weight[1].isfinite().all())


def test_step_weights_without_positions_and_own_workspace(gpu):
    nh, nkv, hd, pos = 8, 4, 128, 777
    q, k, v = randn(46, nh, hd), randn(47, pos + 1, nkv, hd), randn(48, pos + 1, nkv, hd)
    need = gpu.gncx_mqa_attention_step_weights_workspace(pos, nh, nkv, hd)
    sizes = [gpu.gncx_mqa_attention_step_weights_workspace(p, nh, nkv, hd) for p in range(0, 9000, 41)]
    assert sizes == sorted(sizes)
    guard = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    w1, w2 = torch.zeros(nkv, pos + 1, device="cuda"), torch.zeros(nkv, pos + 1, device="cuda")
    y1 = run_step(gpu, q, None, None, k, v, pos, pos, 0.1, 0, w1, None, ws=guard[:need])
    y2 = run_step(gpu, q, None, None, k, v, pos, pos, 0.1, 0, w2, None)
    assert torch.equal(y1, y2) and torch.equal(w1, w2) and bool((guard[need:] == 0xA5).all())
    assert abs(float(w1.double().sum()) - nh) <= nh * 1e-5
    y = torch.empty_like(q)
    args = (P(q), None, None, P(k), P(v), pos, pos, nh, nkv, hd, 0.1)
    assert gpu.gncx_mqa_attention_step_weights(*args, 0, P(y), P(w1), None, pos + 1, P(guard), need - 1) == CAPACITY
    assert gpu.gncx_mqa_attention_step_weights(*args, 1, P(y), P(w1), None, pos + 1, None, 0) == INVALID
    assert gpu.gncx_mqa_attention_step_weights(*args, 0, P(y), None, None, pos + 1, None, 0) == INVALID
    assert gpu.gncx_mqa_attention_step_weights(*args, 0, P(y) + 8, P(w1), None, pos + 1, None, 0) == UNALIGNED


# ---------------------------------------------------------------- eviction
def evict_ref(k, v, w, pos, n_rows, keep, recent):
    """In place on copies; returns (k, v, weights, positions) of the first `keep` rows."""
    k, v = k.cpu().clone(), v.cpu().clone()
    w, pos = w.cpu().numpy(), None if pos is None else pos.cpu().numpy()
    wo, po = np.empty((w.shape[0], keep), np.float32), np.zeros((w.shape[0], keep), np.int32)
    for h in range(w.shape[0]):
        late = pos[h, :n_rows] >= recent if pos is not None else np.zeros(n_rows, bool)
        x = np.where(np.isnan(w[h, :n_rows]), -np.inf, w[h, :n_rows].astype(np.float64))
        order = sorted(range(n_rows), key=lambda i: (not late[i], bool(np.isnan(w[h, i])) and not late[i], 0.0 if late[i] else -x[i], i))
        stay = np.zeros(n_rows, bool)
        stay[order[:keep]] = True
        to = np.flatnonzero(~stay[:keep])
        frm = keep + np.flatnonzero(stay[keep:])
        src = np.arange(keep)
        src[to] = frm
        wo[h] = w[h, src]
        if pos is not None:
            po[h] = pos[h, src]
        k[:keep, h], v[:keep, h] = k[torch.from_numpy(src), h], v[torch.from_numpy(src), h]
    return k, v, wo, po


def run_evict(lib, k, v, w, pos, n_rows, keep, recent, w_out=None, p_out=None, ws=None):
    nkv, hd = k.shape[1:]
    if w_out is None:
        w_out = torch.full((nkv, keep), float("nan"), device="cuda")
        p_out = None if pos is None else torch.full((nkv, keep), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ok(lib, lib.gncx_kv_evict(P(k), P(v), P(w), P(pos), w.shape[1], n_rows, keep, recent, nkv, hd, P(w_out), P(p_out),
                              w_out.shape[1], P(ws), ws.numel() if ws is not None else 0))
    torch.cuda.synchronize()
    return w_out, p_out


def evict_weights(kind, nkv, n, seed):
    w = torch.rand(nkv, n, device="cuda", generator=gen(seed))
    if kind == "equal":
        w = torch.full_like(w, 0.25)
    if kind == "few":
        w = (w * 5).floor()
    if kind == "odd":
        w = w - 0.5
        at = torch.randint(0, 7, (nkv, n), device="cuda", generator=gen(seed + 1))
        for i, x in enumerate((float("nan"), float("inf"), float("-inf"), 0.0, -0.0)):
            w[at == i] = x
    if kind == "spread":
        w = w.pow(8) * 40
    return w


EVICTS = [(1, 4, 1, 1), (1, 4, 2, 1), (2, 64, 33, 32), (2, 64, 64, 33), (3, 80, 100, 7), (8, 128, 1000, 999), (4, 128, 1025, 512),
          (2, 256, 5000, 1234), (8, 64, 4097, 4096), (1, 128, 40000, 100), (2, 20, 70001, 35001), (5, 12, 31, 31), (1, 300, 96, 48),
          (1, 4, 8192, 5000), (2, 4, 8193, 8192), (1, 4, 140001, 70000), (1, 4, 140001, 140000)]


@pytest.mark.parametrize("nkv,hd,n,keep", EVICTS)
@pytest.mark.parametrize("kind", ["spread", "equal", "few", "odd"])
def test_evict(gpu, nkv, hd, n, keep, kind):
    k, v = randn(50, n + 2, nkv, hd), randn(51, n + 2, nkv, hd)
    w = evict_weights(kind, nkv, n + 5, 52)
    pos = torch.stack([torch.randperm(n + 5, device="cuda", generator=gen(53 + h)) for h in range(nkv)]).int()
    for recent in (n + 5, n + 5 - max(1, keep // 3), 0):  # none, some, all protected
        kk, vv, w0 = k.clone(), v.clone(), w.clone()
        rk, rv, rw, rp = evict_ref(k, v, w, pos, n, keep, recent)
        w_out, p_out = run_evict(gpu, kk, vv, w, pos, n, keep, recent)
        assert torch.equal(kk.cpu(), rk) and torch.equal(vv.cpu(), rv)
        assert np.array_equal(w_out.cpu().numpy(), rw, equal_nan=True) and np.array_equal(p_out.cpu().numpy(), rp)
        assert torch.equal(w.view(torch.int32), w0.view(torch.int32))


def test_evict_in_place_and_without_positions(gpu):
    nkv, hd, n, keep = 4, 64, 3000, 777
    k, v, w = randn(54, n, nkv, hd), randn(55, n, nkv, hd), evict_weights("spread", nkv, n, 56)
    rk, rv, rw, _ = evict_ref(k, v, w, None, n, keep, 0)
    tail = w[:, keep:].clone()
    need = gpu.gncx_kv_evict_workspace(n, keep, nkv)
    guard = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    run_evict(gpu, k, v, w, None, n, keep, 0, w_out=w, ws=guard[:need])
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)
    assert np.array_equal(w[:, :keep].cpu().numpy(), rw) and torch.equal(w[:, keep:], tail)
    assert bool((guard[need:] == 0xA5).all())
    assert gpu.gncx_kv_evict(P(k), P(v), P(w), None, n, n, keep, 0, nkv, hd, P(w), None, n, P(guard), need - 1) == CAPACITY
    assert gpu.gncx_kv_evict(P(k), P(v) + 4, P(w), None, n, n, keep, 0, nkv, hd, P(w), None, n, None, 0) == UNALIGNED


def test_evict_to_nothing_is_no_work(gpu):
    k = randn(57, 8, 1, 4)
    w = torch.rand(1, 8, device="cuda")
    k0 = k.clone()
    w_out = torch.zeros(1, 1, device="cuda")
    torch.cuda.synchronize()
    ok(gpu, gpu.gncx_kv_evict(P(k), P(k), P(w), None, 8, 8, 0, 0, 1, 4, P(w_out), None, 1, None, 0))
    assert torch.equal(k, k0)


# ---------------------------------------------------------------- beams
def beam_ref(x, s, fin, eos, n):
    x, s = x.cpu().double().numpy(), s.cpu().double().numpy()
    fin = np.zeros(len(s), bool) if fin is None else fin.cpu().numpy() != 0
    cand = []
    for b in range(len(s)):
        if fin[b]:
            if s[b] > -np.inf:
                cand.append((-s[b], b, 0.0, eos))
            continue
        with np.errstate(all="ignore"):
            m = np.max(x[b])
            lse = m + np.log(np.sum(np.exp(x[b] - m))) if np.isfinite(m) else (np.nan if not m == -np.inf else -np.inf)
            top = np.lexsort((np.arange(x.shape[1]), -x[b]))[:n]
            for t in top:
                c = s[b] + (x[b, t] - lse)
                if c > -np.inf:
                    cand.append((-c, b, -x[b, t], int(t)))
    cand.sort()
    out = [(-c, b, t, int(fin[b] or t == eos)) for c, b, _, t in cand[:n]]
    out += [(-np.inf, -1, -1, 0)] * (n - len(out))
    return [np.array(z) for z in zip(*out)]


def run_beam(lib, x, s, fin, eos, n, ws=None, outs=None):
    if outs is None:
        outs = (torch.full((n,), float("nan"), device="cuda"), *(torch.full((n,), -9, dtype=torch.int32, device="cuda") for _ in range(3)))
    torch.cuda.synchronize()
    ok(lib, lib.gncx_beam_select(P(x), P(s), P(fin), x.shape[0], x.shape[1], eos, n, *(P(o) for o in outs), P(ws),
                                 ws.numel() if ws is not None else 0))
    torch.cuda.synchronize()
    return outs


def check_beam(got, ref):
    score, parent, token, ended = (t.cpu().numpy() for t in got)
    assert np.array_equal(parent, ref[1]) and np.array_equal(token, ref[2]) and np.array_equal(ended, ref[3])
    some = np.isfinite(ref[0])
    assert np.array_equal(np.isfinite(score), some)
    # one rounding to fp32, and the 64-bit sums' own
    assert np.all(np.abs(score[some] - ref[0][some]) <= (U + 1e-12) * np.abs(ref[0][some]) + 1e-12)


BEAMS = [(1, 1, 1), (1, 5, 9), (3, 7, 40), (1, 151936, 1), (4, 151936, 8), (2, 4095, 16), (2, 4096, 16), (2, 4097, 16),
         (5, 8193, 10), (16, 32000, 32), (64, 151936, 128), (7, 50257, 256), (256, 1000, 256), (1, 300001, 256), (3, 262144, 200),
         # few lists, of which several threads read each
         (1, 4096, 256), (2, 300, 256), (5, 4000, 129), (1, 200, 256), (3, 1000, 200), (16, 4000, 32), (31, 900, 33), (7, 3106, 7), (9, 5000, 255)]


@pytest.mark.parametrize("b,vocab,n", BEAMS)
def test_beam(gpu, b, vocab, n):
    x, s = randn(60 + b, b, vocab) * 3, -torch.rand(b, device="cuda", generator=gen(61)) * 3
    check_beam(run_beam(gpu, x, s, None, -1, n), beam_ref(x, s, None, -1, n))
    fin = (torch.rand(b, device="cuda", generator=gen(62)) < 0.4).int() * 5
    eos = vocab // 2
    check_beam(run_beam(gpu, x, s, fin, eos, n), beam_ref(x, s, fin, eos, n))
    if b > 1:  # the first step: one live beam
        s[1:] = float("-inf")
        check_beam(run_beam(gpu, x, s, None, -1, n), beam_ref(x, s, None, -1, n))


@pytest.mark.parametrize("ended", ["none", "all", "all but one", "first half", "every third", "the last"])
@pytest.mark.parametrize("b,vocab,n", [(29, 40001, 58), (64, 9001, 128), (100, 17000, 200), (149, 8200, 256), (256, 4097, 256), (256, 30000, 7)])
def test_beam_ended_beams_leave_their_share(gpu, b, vocab, n, ended):
    """Many beams: the vocabulary is divided by the number of those that have not ended."""
    x, s = randn(65, b, vocab) * 2, -torch.rand(b, device="cuda", generator=gen(66)) * 4
    i = torch.arange(b, device="cuda")
    fin = {"none": i < 0, "all": i >= 0, "all but one": i != b // 2, "first half": i < b // 2, "every third": i % 3 == 0, "the last": i == b - 1}[ended]
    fin = fin.int()
    s[b // 3] = float("-inf")
    check_beam(run_beam(gpu, x, s, fin, 11, n), beam_ref(x, s, fin, 11, n))


@pytest.mark.parametrize("kind", ["equal", "few", "rising", "falling", "masked", "one", "huge", "zeros", "tiny"])
@pytest.mark.parametrize("b,vocab,n", [(3, 20000, 64), (1, 9000, 256), (2, 70001, 5)])
def test_beam_hard_logits(gpu, kind, b, vocab, n):
    x = randn(63, b, vocab)
    if kind == "equal":
        x[:] = 0.5
    if kind == "few":
        x = x.round()
    if kind == "rising":
        x = torch.arange(vocab, device="cuda").float().repeat(b, 1) * 1e-3
    if kind == "falling":
        x = torch.arange(vocab, 0, -1, device="cuda").float().repeat(b, 1) * 1e-3
    if kind == "masked":
        x[:, torch.rand(vocab, device="cuda", generator=gen(64)) < 0.99] = float("-inf")
    if kind == "one":
        x[:] = float("-inf")
        x[:, vocab - 1] = 2.0
    if kind == "huge":
        x *= 1e30
    if kind == "zeros":
        x = torch.where(x > 0, 0.0, -0.0)
    if kind == "tiny":
        x *= 1e-30
    x = x.contiguous()
    s = -torch.arange(b, device="cuda").float() * 0.125
    check_beam(run_beam(gpu, x, s, None, 3, n), beam_ref(x, s, None, 3, n))


def test_beam_without_candidates(gpu):
    x = randn(65, 4, 5000)
    x[0, 17] = float("nan")
    x[1, 4999] = float("inf")
    x[2] = float("-inf")
    s = torch.tensor([0.0, 0.0, 0.0, -1.0], device="cuda")
    check_beam(run_beam(gpu, x, s, None, -1, 8), beam_ref(x, s, None, -1, 8))
    got = run_beam(gpu, x[:3].contiguous(), s[:3].contiguous(), None, -1, 8)
    assert bool((got[1] == -1).all()) and bool((got[0] == float("-inf")).all()) and bool((got[3] == 0).all())
    s[3] = float("nan")
    assert bool((run_beam(gpu, x, s, None, -1, 8)[1] == -1).all())
    fin = torch.ones(4, dtype=torch.int32, device="cuda")  # all ended: one candidate each
    s = torch.tensor([-3.0, -1.0, float("-inf"), -1.0], device="cuda")
    got = run_beam(gpu, x, s, fin, 7, 6)
    assert got[1].tolist() == [1, 3, 0, -1, -1, -1] and got[2].tolist() == [7, 7, 7, -1, -1, -1]


def test_beam_in_place_and_own_workspace(gpu):
    b, vocab, n = 6, 32003, 6
    x, s = randn(66, b, vocab) * 2, -torch.rand(b, device="cuda", generator=gen(67))
    fin = torch.tensor([0, 1, 0, 0, 1, 0], dtype=torch.int32, device="cuda")
    ref = beam_ref(x, s, fin, 9, n)
    need = gpu.gncx_beam_select_workspace(b, vocab, n)
    guard = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    ints = torch.empty(2, n, dtype=torch.int32, device="cuda")
    check_beam(run_beam(gpu, x, s, fin, 9, n, ws=guard[:need], outs=(s, ints[0], ints[1], fin)), ref)
    assert bool((guard[need:] == 0xA5).all())
    args = (P(x), P(s), P(fin), b, vocab, 9, n, P(s), P(ints), P(ints), None)
    assert gpu.gncx_beam_select(*args, P(guard), need - 1) == CAPACITY
    assert gpu.gncx_beam_select(P(x) + 2, *args[1:], None, 0) == UNALIGNED


# ---------------------------------------------------------------- reordering
@pytest.mark.parametrize("slots", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 100, 256])
@pytest.mark.parametrize("words", [1, 3, 4, 260, 1024, 5003])
def test_reorder(gpu, slots, words):
    states = 3
    r = np.random.default_rng(slots * 7 + words)
    x = randn(70, states, slots, words)
    kinds = [r.integers(0, slots, slots), r.permutation(slots), np.roll(np.arange(slots), 1), np.zeros(slots, int),
             np.where(r.random(slots) < 0.5, -1, r.integers(0, slots, slots)), np.arange(slots), np.full(slots, -1)]
    for idx in kinds:
        y, index = x.clone(), torch.tensor(idx, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        ok(gpu, gpu.gncx_state_reorder(P(y), states, slots * words * 4, slots, words * 4, words * 4, P(index)))
        torch.cuda.synchronize()
        src = torch.tensor(np.where(idx < 0, np.arange(slots), idx), device="cuda")
        assert torch.equal(y, x[:, src])


@pytest.mark.parametrize("slots", [22, 23, 24, 25, 45, 46, 47, 48, 49, 93, 94, 95, 96, 97])
@pytest.mark.parametrize("words", [1024, 1023])
def test_reorder_shared_memory_near_48_kb(gpu, slots, words):
    """Slots whose columns and the kernel's own variables together cross what a launch gets without asking."""
    idx = np.roll(np.arange(slots), 5)
    x = randn(72, 2, slots, words)
    y, index = x.clone(), torch.tensor(idx, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ok(gpu, gpu.gncx_state_reorder(P(y), 2, slots * words * 4, slots, words * 4, words * 4, P(index)))
    torch.cuda.synchronize()
    assert torch.equal(y, x[:, torch.tensor(idx, device="cuda")])


@pytest.mark.parametrize("hd", [88, 92, 96, 100])
def test_tree_shared_memory_near_48_kb(gpu, hd):
    nh, nkv, pos0, n = 30, 10, 9, 5
    q, k, v = randn(73, n, nh, hd), randn(74, pos0 + n, nkv, hd), randn(75, pos0 + n, nkv, hd)
    up = make_tree("random", n, 1)
    check_tree(run_tree(gpu, q, k, v, up, pos0, 0.1, 0), q, k, v, up, pos0, 0.1, 0)


def test_reorder_strides(gpu):
    """Part of each slot, slots innermost, and a start off 16 bytes."""
    idx = torch.tensor([2, 0, 0, -1, 1], dtype=torch.int32, device="cuda")
    src = torch.tensor([2, 0, 0, 3, 1], device="cuda")
    x = randn(71, 4, 5, 24)
    y = x.clone()
    torch.cuda.synchronize()
    ok(gpu, gpu.gncx_state_reorder(P(y) + 4 * 4, 4, 5 * 96, 5, 96, 40, P(idx)))  # words 4 .. 13
    ref = x.clone()
    ref[:, :, 4:14] = x[:, src, 4:14]
    assert torch.equal(y, ref)
    y = x.clone()
    torch.cuda.synchronize()
    ok(gpu, gpu.gncx_state_reorder(P(y) + 4, 4, 5 * 96, 5, 96, 48, P(idx)))
    ref = x.clone()
    ref[:, :, 1:13] = x[:, src, 1:13]
    assert torch.equal(y, ref)
    x = randn(72, 5, 7, 8)  # slot outermost: 7 states of 8 words inside it
    y = x.clone()
    torch.cuda.synchronize()
    ok(gpu, gpu.gncx_state_reorder(P(y), 7, 32, 5, 7 * 32, 32, P(idx)))
    assert torch.equal(y, x[src])
    y = x.clone()
    torch.cuda.synchronize()
    assert gpu.gncx_state_reorder(P(y), 7, 28, 5, 100, 32, P(idx)) == INVALID
    gpu.gncx_clear_error()
    assert gpu.gncx_state_reorder(P(y) + 2, 7, 32, 5, 7 * 32, 32, P(idx)) == UNALIGNED
    gpu.gncx_clear_error()
    ok(gpu, gpu.gncx_state_reorder(None, 0, 32, 5, 32, 32, None))
    assert torch.equal(y, x)


def test_reorder_bad_index_is_an_error(gpu):
    x = randn(73, 1, 4, 64)
    y = x.clone()
    idx = torch.tensor([1, 4, -2, 0], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert gpu.gncx_state_reorder(P(y), 1, 1024, 4, 256, 256, P(idx)) == INVALID
    gpu.gncx_clear_error()
    assert torch.equal(y, x[:, torch.tensor([1, 1, 2, 0], device="cuda")])
    gpu.gncx_set_synchronous(0)  # stream-ordered: the next gncx_sync reports it
    ok(gpu, gpu.gncx_state_reorder(P(y), 1, 1024, 4, 256, 256, P(idx)))
    assert gpu.gncx_sync() == INVALID
    gpu.gncx_clear_error()
    ok(gpu, gpu.gncx_sync())


# ---------------------------------------------------------------- offsets past 32 bits
def test_offsets_past_32_bits(gpu):
    """Caches of more than 2^31 elements: the last rows are the ones used."""
    nh, nkv, hd, n, window = 8, 8, 128, 4, 48
    pos0 = 2**31 // (nkv * hd) + 100
    k = torch.zeros(pos0 + n, nkv, hd, device="cuda")
    v = torch.zeros(pos0 + n, nkv, hd, device="cuda")
    k[-200:], v[-200:] = randn(80, 200, nkv, hd), randn(81, 200, nkv, hd)
    q = randn(82, n, nh, hd)
    up = make_tree("chain", n, 0)
    check_tree(run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window), q, k, v, up, pos0, hd**-0.5, window)
    # zero keys get equal scores; a heavy row at the end gets what is left
    pos = pos0 + n - 1
    weight = torch.zeros(nkv, pos + 1, device="cuda")
    k[-200:-1] = 0
    k[-1] = 0
    v[-200:] = 0
    v[-1] = 1.0
    q1 = torch.ones(nh, hd, device="cuda")
    k[-1] = 14.0 / hd  # score 14 against 0
    y = run_step(gpu, q1, None, None, k, v, pos, pos, 1.0, 0, weight, None)
    p_last = float(np.exp(14.0) / (np.exp(14.0) + pos))
    assert float((y - p_last).abs().max()) <= 1e-4 * p_last and float((weight[:, -1] - p_last).abs().max()) <= 1e-4 * p_last
    # the last rows are the heaviest: they move to the front
    keep = 64
    w_out, _ = run_evict(gpu, k, v, weight + torch.arange(pos + 1, device="cuda") * 1e-6, None, pos + 1, keep, 0)
    assert torch.equal(v[keep - 1], torch.ones(nkv, hd, device="cuda")) and bool((v[:keep - 1] == 0).all())
    x = k.view(-1)[: 2**31 + 4096].view(torch.int32)
    half = (x.numel() // 2) // 4 * 4
    a, b = x[:half].clone(), x[half:2 * half].clone()
    idx = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ok(gpu, gpu.gncx_state_reorder(P(x), 1, 8 * half, 2, 4 * half, 4 * half, P(idx)))
    assert torch.equal(x[:half], b) and torch.equal(x[half:2 * half], a)


# ---------------------------------------------------------------- graphs, streams
def test_captured_and_replayed(gpu):
    """All calls in one graph, replayed on new inputs; another graph with its own workspaces at the same time."""
    nh, nkv, hd, pos0, n, beams, vocab = 8, 2, 64, 900, 12, 4, 9000
    lib = gpu

    class Set:
        def __init__(self, seed):
            self.q, self.k, self.v = randn(seed, n, nh, hd), randn(seed + 1, pos0 + n, nkv, hd), randn(seed + 2, pos0 + n, nkv, hd)
            self.up = torch.tensor(make_tree("random", n, seed), dtype=torch.int32, device="cuda")
            self.out = torch.zeros_like(self.q)
            self.y = torch.zeros(nh, hd, device="cuda")
            self.w = torch.zeros(nkv, pos0 + n, device="cuda")
            self.wo = torch.zeros(nkv, 500, device="cuda")
            self.x, self.s = randn(seed + 3, beams, vocab), torch.zeros(beams, device="cuda")
            self.so = torch.zeros(beams, device="cuda")
            self.io = torch.zeros(2, beams, dtype=torch.int32, device="cuda")
            self.state = randn(seed + 4, 2, beams, 96)
            size = lambda b: torch.empty(b, dtype=torch.uint8, device="cuda")  # noqa: E731
            self.ws = [size(lib.gncx_attention_tree_workspace(pos0, n, nh, nkv, hd, 0)),
                       size(lib.gncx_mqa_attention_step_weights_workspace(pos0, nh, nkv, hd)),
                       size(lib.gncx_kv_evict_workspace(pos0, 500, nkv)), size(lib.gncx_beam_select_workspace(beams, vocab, beams))]

        def call(self, own=True):
            ws = [(P(w), w.numel()) if own else (None, 0) for w in self.ws]
            st = [lib.gncx_attention_tree(P(self.q), P(self.k), P(self.v), P(self.up), pos0, n, nh, nkv, hd, 0.125, 0, P(self.out), *ws[0]),
                  lib.gncx_mqa_attention_step_weights(P(self.q), None, None, P(self.k), P(self.v), pos0, pos0, nh, nkv, hd, 0.125, 0,
                                                      P(self.y), P(self.w), None, pos0 + n, *ws[1]),
                  lib.gncx_kv_evict(P(self.k), P(self.v), P(self.w), None, pos0 + n, pos0, 500, 0, nkv, hd, P(self.wo), None, 500, *ws[2]),
                  lib.gncx_beam_select(P(self.x), P(self.s), None, beams, vocab, 1, beams, P(self.so), P(self.io), P(self.io[1]), None, *ws[3]),
                  lib.gncx_state_reorder(P(self.state), 2, beams * 384, beams, 384, 384, P(self.io))]
            return st

        def fill(self, other):
            for name in ("q", "k", "v", "up", "x", "s", "state", "w"):
                getattr(self, name).copy_(getattr(other, name))

        def results(self):
            return [t.clone() for t in (self.out, self.y, self.w, self.wo, self.so, self.io, self.state, self.k, self.v)]

    home = torch.cuda.current_stream()
    a, b = Set(90), Set(95)
    wants = []
    for s in (Set(100), Set(105)):
        keep = Set(0)
        keep.fill(s)
        assert keep.call() == [0] * 5
        torch.cuda.synchronize()
        wants.append((s, keep.results()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    try:
        # refused while capturing: in synchronous mode, and without a workspace of the caller's
        lib.gncx_set_synchronous(0)
        for st, s in zip(streams, (a, b)):
            lib.gncx_set_stream(ctypes.c_void_p(st.cuda_stream))
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=st):
                assert s.call(own=False)[:4] == [INVALID] * 4
                lib.gncx_set_synchronous(1)
                assert s.call() == [INVALID] * 5
                lib.gncx_set_synchronous(0)
                lib.gncx_clear_error()
            del g
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                assert s.call() == [0] * 5
            graphs.append(g)
        # the library's own workspace grows in between: the graphs do not use it
        lib.gncx_set_stream(ctypes.c_void_p(home.cuda_stream))
        big = randn(99, 40, 32, 128), randn(98, 9040, 8, 128)
        run_tree(lib, big[0], big[1], big[1], make_tree("star", 40, 0), 9000, 0.1, 0)
        for x, y in ((0, 1), (1, 0), (0, 0)):
            a.fill(wants[x][0])
            b.fill(wants[y][0])
            torch.cuda.synchronize()
            for g, st in zip(graphs, streams):  # both at once
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for s, i in ((a, x), (b, y)):
                for got, want in zip(s.results(), wants[i][1]):
                    assert torch.equal(got, want)
    finally:
        lib.gncx_set_stream(ctypes.c_void_p(home.cuda_stream))
        lib.gncx_set_synchronous(1)


def test_captured_small_and_wide_forms(gpu):
    """The forms for few rows, one evicted row, head size 256 and ended beams, replayed with other parents, rows and beams."""
    lib, home = gpu, torch.cuda.current_stream()
    q, k, v = randn(110, 5, 8, 64), randn(111, 205, 4, 64), randn(112, 205, 4, 64)
    qw, kw, vw = randn(113, 20, 8, 256), randn(114, 1220, 2, 256), randn(115, 1220, 2, 256)
    up, upw = (torch.zeros(i, dtype=torch.int32, device="cuda") for i in (5, 20))
    out, outw = torch.zeros_like(q), torch.zeros_like(qw)
    x, fin = randn(116, 40, 9000), torch.zeros(40, dtype=torch.int32, device="cuda")
    s, so, io = torch.zeros(40, device="cuda"), torch.zeros(80, device="cuda"), torch.zeros(3, 80, dtype=torch.int32, device="cuda")
    w, pos = torch.zeros(4, 205, device="cuda"), torch.zeros(4, 205, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    wa, step = (P(ws), ws.numel()), torch.zeros(8, 64, device="cuda")

    def call():
        assert lib.gncx_attention_tree(P(q), P(k), P(v), P(up), 200, 5, 8, 4, 64, 0.1, 0, P(out), *wa) == 0
        assert lib.gncx_attention_tree(P(qw), P(kw), P(vw), P(upw), 1200, 20, 8, 2, 256, 0.06, 0, P(outw), *wa) == 0
        assert lib.gncx_beam_select(P(x), P(s), P(fin), 40, 9000, 3, 80, P(so), P(io), P(io[1]), P(io[2]), *wa) == 0
        assert lib.gncx_mqa_attention_step_weights(P(q), P(k), P(v), P(k), P(v), 204, 7, 8, 4, 64, 0.1, 0, P(step), P(w), P(pos), 205, *wa) == 0
        assert lib.gncx_kv_evict(P(k), P(v), P(w), P(pos), 205, 205, 204, 9, 4, 64, P(w), P(pos), 205, *wa) == 0

    def fill(seed):
        r = np.random.default_rng(seed)
        for t, n in ((up, 5), (upw, 20)):
            t.copy_(torch.tensor(make_tree("random", n, seed), dtype=torch.int32))
        fin.copy_(torch.tensor(r.integers(0, 2, 40), dtype=torch.int32))
        pos.copy_(torch.tensor(r.integers(0, 12, (4, 205)), dtype=torch.int32))
        for i, t in enumerate((q, k, v, qw, kw, vw, x, w)):
            t.copy_(randn(1000 * seed + i, *t.shape))

    outs = (out, outw, so, io, step, w, pos, k, v)
    wants = []
    for seed in (1, 2, 3):
        fill(seed)
        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        wants.append([t.clone() for t in outs])
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        lib.gncx_set_synchronous(0)
        lib.gncx_set_stream(ctypes.c_void_p(stream.cuda_stream))
        with torch.cuda.graph(g, stream=stream):
            call()
        for seed in (3, 1, 2, 1):
            fill(seed)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            torch.cuda.synchronize()
            for got, want in zip(outs, wants[seed - 1]):
                assert torch.equal(got, want)
    finally:
        lib.gncx_set_stream(ctypes.c_void_p(home.cuda_stream))
        lib.gncx_set_synchronous(1)


def test_stream_ordered_calls_in_a_row(gpu):
    """Stream-ordered, the library's workspace, on a stream of the caller's: each call waits for the one before."""
    home = torch.cuda.current_stream()
    s = torch.cuda.Stream()
    q, k, v = randn(110, 20, 8, 128), randn(111, 2020, 4, 128), randn(112, 2020, 4, 128)
    up = torch.tensor(make_tree("random", 20, 2), dtype=torch.int32, device="cuda")
    x, sc = randn(113, 8, 30000), torch.zeros(8, device="cuda")
    want_tree = run_tree(gpu, q, k, v, up.cpu().numpy(), 2000, 0.1, 0)
    want_beam = [t.clone() for t in run_beam(gpu, x, sc, None, -1, 16)]
    out = [torch.zeros_like(q) for _ in range(10)]
    so, io = torch.zeros(10, 16, device="cuda"), torch.zeros(10, 2, 16, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    try:
        gpu.gncx_set_synchronous(0)
        gpu.gncx_set_stream(ctypes.c_void_p(s.cuda_stream))
        for i in range(10):
            ok(gpu, gpu.gncx_attention_tree(P(q), P(k), P(v), P(up), 2000, 20, 8, 4, 128, 0.1, 0, P(out[i]), None, 0))
            ok(gpu, gpu.gncx_beam_select(P(x), P(sc), None, 8, 30000, -1, 16, P(so[i]), P(io[i, 0]), P(io[i, 1]), None, None, 0))
        ok(gpu, gpu.gncx_sync())
    finally:
        gpu.gncx_set_stream(ctypes.c_void_p(home.cuda_stream))
        gpu.gncx_set_synchronous(1)
    for i in range(10):
        assert torch.equal(out[i], want_tree) and torch.equal(so[i], want_beam[0])
        assert torch.equal(io[i, 0], want_beam[1]) and torch.equal(io[i, 1], want_beam[2])


def test_stream_ordered_mode_set_before_the_first_call():
    """gncx_set_synchronous(0) as a process's first call holds: a call after it does not wait, and can be captured."""
    import subprocess
    import sys
    from conftest import ROOT
    code = """
import ctypes, torch
from gncx_b200 import core
lib = core.load()
lib.gncx_set_synchronous(0)
s = torch.cuda.Stream()
lib.gncx_set_stream(ctypes.c_void_p(s.cuda_stream))
x = torch.arange(8, device="cuda").float().view(2, 4)
i = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    st = lib.gncx_state_reorder(x.data_ptr(), 1, 32, 2, 16, 16, i.data_ptr())
assert st == 0, lib.gncx_last_error_message()
g.replay()
torch.cuda.synchronize()
assert x.tolist() == [[4, 5, 6, 7], [0, 1, 2, 3]], x
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


# ---------------------------------------------------------------- runs as they would be used
def test_speculative_decoding_run(gpu):
    """Draft a tree, verify it, accept a path, go on: outputs and caches of plain sequential decoding."""
    nh, nkv, hd, layers, rows = 8, 4, 64, 3, 400
    r = np.random.default_rng(4)
    k, v = torch.zeros(layers, rows, nkv, hd, device="cuda"), torch.zeros(layers, rows, nkv, hd, device="cuda")
    pos = 100
    k[:, :pos], v[:, :pos] = randn(120, layers, pos, nkv, hd), randn(121, layers, pos, nkv, hd)
    ks, vs = k.clone(), v.clone()  # the sequential decoder's
    for step in range(6):
        n = int(r.integers(1, 30))
        up = make_tree("random", n, step)
        qn = randn(130 + step, layers, n, nh, hd)
        kn, vn = randn(140 + step, layers, n, nkv, hd), randn(150 + step, layers, n, nkv, hd)
        k[:, pos:pos + n], v[:, pos:pos + n] = kn, vn
        outs = [run_tree(gpu, qn[i].contiguous(), k[i], v[i], up, pos, hd**-0.5, 0) for i in range(layers)]
        path = tree_path(up, int(r.integers(0, n)))
        index = torch.full((n,), -1, dtype=torch.int32)
        index[:len(path)] = torch.tensor(path, dtype=torch.int32)
        index = index.cuda()
        torch.cuda.synchronize()
        row = nkv * hd * 4
        for c in (k, v):
            ok(gpu, gpu.gncx_state_reorder(P(c) + pos * row, layers, rows * row, n, row, row, P(index)))
        for node in path:
            for i in range(layers):
                y = torch.empty(nh, hd, device="cuda")
                torch.cuda.synchronize()
                gpu.gncx_mqa_attention_step_ext(P(qn[i, node].contiguous()), P(kn[i, node].contiguous()), P(vn[i, node].contiguous()),
                                                P(ks[i]), P(vs[i]), pos, nh, nkv, hd, hd**-0.5, 0, 1, P(y))
                core.check(gpu)
                assert float((outs[i][node] - y).abs().max()) <= 1e-5 * float(y.abs().max())
            pos += 1
        torch.cuda.synchronize()
        assert torch.equal(k[:, :pos], ks[:, :pos]) and torch.equal(v[:, :pos], vs[:, :pos])


def test_beam_search_run(gpu):
    """Beam search over a small table model with per-beam caches, against the same search on the host."""
    beams, vocab, steps, width, eos = 4, 300, 12, 32, 5
    table = randn(160, vocab, vocab) * 2
    rows = randn(161, vocab, width)  # the "cache row" of a token
    state = torch.zeros(2, beams, steps, width, device="cuda")
    scores = torch.tensor([0.0] + [float("-inf")] * (beams - 1), device="cuda")
    fin, tokens = torch.zeros(beams, dtype=torch.int32, device="cuda"), torch.full((beams,), 1, dtype=torch.int32, device="cuda")
    parents = torch.zeros(beams, dtype=torch.int32, device="cuda")
    host = [(0.0, [1], False)]  # score, tokens, ended
    lp = torch.log_softmax(table.double(), 1).cpu().numpy()
    for t in range(steps):
        state[:, :, t] = rows[tokens.long()]
        logits = table[tokens.long()].contiguous()
        torch.cuda.synchronize()
        ok(gpu, gpu.gncx_beam_select(P(logits), P(scores), P(fin), beams, vocab, eos, beams, P(scores), P(parents), P(tokens), P(fin), None, 0))
        ok(gpu, gpu.gncx_state_reorder(P(state), 2, beams * steps * width * 4, beams, steps * width * 4, (t + 1) * width * 4, P(parents)))
        cand = []
        for s, seq, ended in host:
            if ended:
                cand.append((s, seq + [eos], True))
            else:
                cand += [(s + lp[seq[-1], w], seq + [w], w == eos) for w in range(vocab)]
        cand.sort(key=lambda c: -c[0])
        host = cand[:beams]
        torch.cuda.synchronize()
        assert tokens.tolist() == [seq[-1] for _, seq, _ in host] and fin.tolist() == [int(e) for _, _, e in host]
        assert np.allclose(scores.cpu().numpy(), [s for s, _, _ in host], rtol=1e-5)
        for i, (_, seq, _) in enumerate(host):
            want = rows[torch.tensor(seq[:-1], device="cuda")]
            assert torch.equal(state[0, i, :t + 1], want) and torch.equal(state[1, i, :t + 1], want)


def test_bounded_cache_run(gpu):
    """Decoding with a budget: the cache keeps the newest rows and the heaviest others."""
    nh, nkv, hd, budget, newest = 4, 2, 64, 40, 8
    k, v = torch.zeros(budget + 1, nkv, hd, device="cuda"), torch.zeros(budget + 1, nkv, hd, device="cuda")
    w, pos = torch.zeros(nkv, budget + 1, device="cuda"), torch.zeros(nkv, budget + 1, dtype=torch.int32, device="cuda")
    all_k, all_v = randn(170, 150, nkv, hd), randn(171, 150, nkv, hd)
    used = 0
    for t in range(150):
        q = randn(200 + t, nh, hd) * 2
        held, w0, u0 = pos.clone(), w.clone(), used
        y = run_step(gpu, q, all_k[t].contiguous(), all_v[t].contiguous(), k, v, used, t, hd**-0.5, 1, w, pos)
        used += 1
        for h in range(nh):
            c = h // 2
            rows = torch.cat([held[c, :u0].long(), torch.tensor([t], device="cuda")])
            ref, tol, p, _ = attend(q[h], all_k[rows, c], all_v[rows, c], hd**-0.5)
            assert bool(((y[h].double() - ref).abs() <= tol).all())
        assert float((w[:, :used].double().sum() - w0[:, :u0].double().sum() - nh).abs()) < 1e-4
        if used > budget:
            order_w, order_p = w.clone(), pos.clone()
            _, _, rw, rp = evict_ref(k, v, order_w, order_p, used, budget, t + 1 - newest)
            ok(gpu, gpu.gncx_kv_evict(P(k), P(v), P(w), P(pos), budget + 1, used, budget, t + 1 - newest, nkv, hd, P(w), P(pos),
                                      budget + 1, None, 0))
            used = budget
            assert np.array_equal(w[:, :budget].cpu().numpy(), rw) and np.array_equal(pos[:, :budget].cpu().numpy(), rp)
        for c in range(nkv):  # every row is the one its position says, the newest are there
            at = pos[c, :used].long()
            assert torch.equal(k[:used, c], all_k[at, c]) and torch.equal(v[:used, c], all_v[at, c])
            assert set(range(max(0, t + 1 - newest), t + 1)) <= set(at.tolist())
