"""Operators for several candidates and bounded caches over more of what their
documentation allows: long caches, values of very different size, rows that are
all protected, forms that other tests pass by.  Tolerances as derived in
test_candidates_gpu.py."""
import numpy as np
import pytest

from test_candidates_gpu import (EVICTS, INVALID, P, _clean, attend, check_tree, evict_weights, gen, make_tree, ok, randn,  # noqa: F401
                                 run_evict, run_tree, tree_path, tree_seen)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---------------------------------------------------------------- tree
@pytest.mark.parametrize("nh,nkv,pos0,n", [(8, 4, 30001, 64), (2, 1, 3000, 200), (148, 148, 1500, 1)])
def test_tree_wide_many_tiles(gpu, nh, nkv, pos0, n):
    """Head size 256, up to 47 tiles of 32 rows per CTA: the halves of the output go through the same barriers each time."""
    hd = 256
    q, k, v = randn(1, n, nh, hd), randn(2, pos0 + n, nkv, hd), randn(3, pos0 + n, nkv, hd)
    up = make_tree("random", n, 21)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    for i in sorted({0, n - 1}):
        rows = torch.tensor(tree_seen(up, i, pos0, 0), device="cuda")
        for h in sorted({0, nh - 1}):
            g = h // (nh // nkv)
            ref, tol, _, _ = attend(q[i, h], k[rows][:, g], v[rows][:, g], hd**-0.5)
            assert bool(((out[i, h].double() - ref).abs() <= tol).all()), (i, h)
    for _ in range(10):
        assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0))


# ---------------------------------------------------------------- eviction
def stays(w, pos, n_rows, keep, recent):
    """The rows that stay, as documented: protected ones first, then by weight (NaN least), then the lowest row."""
    w = w[:n_rows].cpu().double().numpy()
    late = np.zeros(n_rows, bool) if pos is None else pos[:n_rows].cpu().numpy() >= recent
    nan = np.isnan(w)
    order = np.lexsort((np.arange(n_rows), -np.where(nan, 0.0, w), nan, ~late))
    stay = np.zeros(n_rows, bool)
    stay[order[:keep]] = True
    return stay


def check_evict(gpu, w, pos, n, keep, recent, in_place=False, hd=4):
    nkv = w.shape[0]
    k, v = randn(30, n, nkv, hd), randn(31, n, nkv, hd)
    src = []
    for h in range(nkv):
        stay = stays(w[h], pos[h], n, keep, recent)
        s = np.arange(n)
        s[np.flatnonzero(~stay[:keep])] = keep + np.flatnonzero(stay[keep:])
        src.append(torch.from_numpy(s).cuda())
    want = [torch.stack([t[src[h], h] for h in range(nkv)], 1) for t in (k, v)]
    want_w = torch.stack([w[h][src[h][:keep]] for h in range(nkv)])
    want_p = torch.stack([pos[h][src[h][:keep]] for h in range(nkv)])
    w, pos = w.clone(), pos.clone()
    w_out, p_out = run_evict(gpu, k, v, w, pos, n, keep, recent, *((w, pos) if in_place else ()))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert torch.equal(w_out[:, :keep].view(torch.int32), want_w.view(torch.int32)) and torch.equal(p_out[:, :keep], want_p)


@pytest.mark.parametrize("nkv,hd,n,keep", EVICTS)
@pytest.mark.parametrize("kind", ["spread", "equal", "few", "odd"])
def test_evict_in_documented_order(gpu, nkv, hd, n, keep, kind):
    w = evict_weights(kind, nkv, n + 5, 52)
    pos = torch.stack([torch.randperm(n + 5, device="cuda", generator=gen(53 + h)) for h in range(nkv)]).int()
    for recent in (n + 5, n + 5 - max(1, keep // 3), 0):  # none, some, all protected
        check_evict(gpu, w, pos, n, keep, recent, hd=hd)


# rows and rows that stay: one row, one CTA, clusters, and more rows than those take
PROTECTED = [(2, 1), (1000, 999), (4097, 4096), (60001, 60000), (40, 9), (4000, 1500), (8000, 3000), (20000, 700), (50000, 20000), (120000, 31000),
             (140001, 40000), (140001, 140000)]


@pytest.mark.parametrize("n,keep", PROTECTED)
@pytest.mark.parametrize("kind", ["spread", "few", "odd"])
def test_evict_ranks_protected_rows_by_weight(gpu, n, keep, kind):
    """As many protected rows as stay, one more, twice as many, all: they are ranked by weight."""
    nkv = 2
    w = evict_weights(kind, nkv, n, 32)
    pos = torch.stack([torch.randperm(n, device="cuda", generator=gen(33 + h)) for h in range(nkv)]).int()
    for protected in sorted({keep, min(keep + 1, n), min(2 * keep, n), n}):
        check_evict(gpu, w, pos, n, keep, n - protected)
        check_evict(gpu, w, pos, n, keep, n - protected, in_place=True)


def test_evict_five_protected_rows(gpu):
    w = torch.tensor([[5.0, 1.0, 9.0, 2.0, 7.0]], device="cuda")
    pos = torch.tensor([[4, 0, 2, 1, 3]], dtype=torch.int32, device="cuda")
    k = torch.arange(20, device="cuda").float().view(5, 1, 4)
    v = -k
    w_out, p_out = run_evict(gpu, k, v, w, pos, 5, 2, 0)
    assert w_out.tolist() == [[9.0, 7.0]] and p_out.tolist() == [[2, 3]]
    assert k[:2, 0, 0].tolist() == [8.0, 16.0] and v[:2, 0, 0].tolist() == [-8.0, -16.0]


def test_evict_one_of_protected_rows_keeps_the_new_token(gpu):
    """A cache whose rows are all recent loses the least weight, not the row written last."""
    n = 65
    w = torch.rand(3, n, device="cuda", generator=gen(34)) + 1
    w[0, 11], w[1, n - 1], w[2, 0] = 0.5, 0.5, float("nan")
    pos = torch.arange(n, dtype=torch.int32, device="cuda").repeat(3, 1)
    check_evict(gpu, w, pos, n, n - 1, 0)
    w_out, p_out = run_evict(gpu, randn(35, n, 3, 4), randn(36, n, 3, 4), w, pos, n, n - 1, 0)
    assert p_out[0, 11] == n - 1 and p_out[1].tolist() == list(range(n - 1)) and p_out[2, 0] == n - 1


# ---------------------------------------------------------------- values of very different size
U, LAM = 2.0**-24, 8.0


def attend_rows(q, k, v, scale):
    """q [hd], k and v [n, hd] -> (output, its tolerance) in 64 bits, with each row's own error instead of the largest.

    A score is off by ds_j = (LAM sqrt(hd) + 14 + 2 C) u scale sum |q k_j| (the terms of test_candidates_gpu.py), its
    weight by that and the exponential's (2 + |x_j|) u, x_j its distance from the maximum in powers of two, and the sum
    of the weights by the weights' errors and its own rounding: D.  Each term p_j v_j of an output is off by its weight's
    error, D, the pairs' 12 u and the output's sum, (LAM sqrt(n) + 24) u.  What the pairs cut, half a step of the lo
    part, 2^-25: as rows are scaled to a largest value in [2^3, 2^15), 2^-28 of max |k_j| or max |v_j| an element; and as
    the largest weight times V in a row's scale is scaled to at least 2^13, 2^-25 2^15 / (2^13 2^3) = 2^-26 of the
    largest p_j max |v_j| for a row's weight (for hardly more than half of the rows, at random: LAM sqrt(n / 4))."""
    q, k, v = q.double(), k.double(), v.double()
    n, hd = k.shape
    s = (k @ q) * scale
    c = LAM * hd**0.5 + 14 + 2 * max(24, 3 * ((hd + 15) // 16))
    p = torch.softmax(s, 0)
    ds = abs(scale) * (c * U * (k.abs() @ q.abs()) + 2.0**-28 * q.abs().sum() * k.abs().amax(1))
    r = ds + (2 + (s.max() - s) / np.log(2.0)) * U
    off = r + (p * r).sum() + (2 * LAM * n**0.5 + 36) * U
    pv = p * v.abs().amax(1)
    cut = 2.0**-28 * pv.sum() + 2.0**-27 * (LAM * n**0.5 + 8) * pv.max()
    return p @ v, (p * off) @ v.abs() + cut + 1e-36


def check_rows(out, q, k, v, up, pos0, scale, window, nodes, heads):
    group = q.shape[1] // k.shape[1]
    worst = 0.0
    for i in nodes:
        rows = torch.tensor(tree_seen(up, i, pos0, window), device="cuda")
        for h in heads:
            ref, tol = attend_rows(q[i, h], k[rows][:, h // group], v[rows][:, h // group], scale)
            err = (out[i, h].double() - ref).abs()
            worst = max(worst, float((err / tol).max()))
            assert bool((err <= tol).all()), (i, h, float((err / tol).max()), float((err / ref.abs().clamp_min(1e-30)).max()))
    return worst


# Forms of the tensor-core kernel: one lane, two lanes, lanes on alternating tiles, and columns above 128; on the CUDA
# cores: few query rows, other head sizes.
FORMS = {"one lane": (8, 2, 128, 700, 24), "one lane of 64": (8, 2, 64, 700, 24), "two lanes": (32, 4, 128, 900, 20), "two lanes of 64": (32, 4, 64, 900, 20),
         "alternating": (32, 32, 128, 1800, 6), "alternating, of 64": (32, 32, 64, 1800, 6), "wide": (16, 4, 256, 700, 24), "wide, many tiles": (148, 148, 256, 400, 2),
         "one launch": (8, 2, 128, 300, 3), "columns of 36": (8, 2, 36, 900, 30), "columns of 252": (8, 2, 252, 900, 30)}


def uneven(seed, n, nh, nkv, hd, pos0):
    """Scores within about a unit of each other, except where `bias` (one column of K) lowers them."""
    q, k, v = randn(seed, n, nh, hd) * 0.1, randn(seed + 1, pos0 + n, nkv, hd) * 0.1, randn(seed + 2, pos0 + n, nkv, hd)
    q[..., 0], k[..., 0] = 1.0, 0.0
    return q, k, v


# the row of another size: in the same chunk of 8 rows (or 4), the same tile, another tile, the first, the last
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("r", [6, 13, 17, 20, 24, 30, 36, 60, 100])
def test_tree_rows_without_weight_do_not_blur_v(gpu, form, r):
    """Rows that get next to no weight have V 2^r larger than the rows that get it all."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(40, n, nh, nkv, hd, pos0)
    large = torch.zeros(pos0 + n, dtype=torch.bool, device="cuda")
    for row in (0, 5, 70, 130, 200, 201, 202, 203, 204, 205, 206, 207, 290, pos0 - 1):
        large[row] = True
    v[large] *= 2.0**r
    k[large, :, 0] = -(r * 0.75 + 40) / 1.0  # a weight of e^-(..): its product with V is small too
    up = make_tree("random", n, 41)
    out = run_tree(gpu, q, k, v, up, pos0, 1.0, 0)
    check_rows(out, q, k, v, up, pos0, 1.0, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("r", [6, 13, 20, 30, 40, 60])
def test_tree_small_weights_of_large_v(gpu, form, r):
    """Rows with weights of about 2^-r whose V is 2^(r + 3) larger make up the output."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(50, n, nh, nkv, hd, pos0)
    light = torch.zeros(pos0 + n, dtype=torch.bool, device="cuda")
    light[64:192] = True
    light[200:230:3] = True
    v[light] *= 2.0 ** (r + 3)
    k[light, :, 0] = -r * 0.6931
    up = make_tree("random", n, 51)
    out = run_tree(gpu, q, k, v, up, pos0, 1.0, 0)
    check_rows(out, q, k, v, up, pos0, 1.0, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [0.0, 1e-30, 2.0**-20])
def test_tree_weight_on_rows_of_little_v(gpu, form, size):
    """A row takes nearly all weight and has a V of zero or next to it: the others' 2^-30 make the output."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(60, n, nh, nkv, hd, pos0)
    sink = torch.zeros(pos0 + n, dtype=torch.bool, device="cuda")
    sink[3] = sink[131] = True
    v[sink] *= size
    k[sink, :, 0] = 20.8
    up = make_tree("random", n, 61)
    out = run_tree(gpu, q, k, v, up, pos0, 1.0, 0)
    check_rows(out, q, k, v, up, pos0, 1.0, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lowest,highest", [(-100, 100), (-30, 30), (-6, 6)])
def test_tree_v_rows_of_any_size(gpu, form, lowest, highest):
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(70, n, nh, nkv, hd, pos0)
    v *= 2.0 ** torch.randint(lowest, highest + 1, (pos0 + n, nkv, 1), device="cuda", generator=gen(73))
    k[..., 0] = torch.rand(pos0 + n, nkv, device="cuda", generator=gen(74)) * -30
    up = make_tree("random", n, 71)
    out = run_tree(gpu, q, k, v, up, pos0, 1.0, 0)
    check_rows(out, q, k, v, up, pos0, 1.0, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("share", [0.3, 0.9, 0.99])
def test_tree_sparse_v(gpu, form, share):
    """Many zeros in V, so that some threads see none but small values of a row that is not small (or is zero)."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(80, n, nh, nkv, hd, pos0)
    v[torch.rand(v.shape, device="cuda", generator=gen(83)) < share] = 0
    up = make_tree("random", n, 81)
    out = run_tree(gpu, q, k, v, up, pos0, 1.0, 0)
    check_rows(out, q, k, v, up, pos0, 1.0, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))
    for _ in range(20):
        assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, 1.0, 0))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("r", [6, 13, 18, 22, 26, 30, 40])
def test_tree_large_rows_do_not_blur_k(gpu, form, r):
    """Rows of K 2^r larger than their neighbours, which get no weight: the others' scores keep their bits."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(90, n, nh, nkv, hd, pos0)
    large = torch.arange(pos0 + n, device="cuda") % 8 == 3
    large[96:104] = True
    k[large] = 0
    k[large, :, 0] = -(2.0**r) * 0.4  # q's first column is 1: a score of -2^r and lower
    k[large, :, 1] = 2.0**r * 0.2
    q[..., 1] = 0.25
    up = make_tree("random", n, 91)
    for row in (11, 99):
        k[row, :, 0] = -(2.0**5)
        k[row, :, 1] = 0
    out = run_tree(gpu, q, k, v, up, pos0, 1.0, 0)
    check_rows(out, q, k, v, up, pos0, 1.0, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lowest,highest", [(-60, 0), (-20, 2), (-6, 3)])
def test_tree_k_and_v_rows_of_any_size(gpu, form, lowest, highest):
    """Rows of K and V of any size next to each other; each row's own sum |q k| bounds its score's error."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = randn(95, n, nh, hd), randn(96, pos0 + n, nkv, hd), randn(97, pos0 + n, nkv, hd)
    k *= 2.0 ** torch.randint(lowest, highest + 1, (pos0 + n, nkv, 1), device="cuda", generator=gen(98))
    v *= 2.0 ** torch.randint(3 * lowest // 2, highest + 1, (pos0 + n, nkv, 1), device="cuda", generator=gen(99))
    up = make_tree("random", n, 93)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    check_rows(out, q, k, v, up, pos0, hd**-0.5, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("share", [0.3, 0.9, 0.99])
def test_tree_sparse_k(gpu, form, share):
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = randn(100, n, nh, hd), randn(101, pos0 + n, nkv, hd), randn(102, pos0 + n, nkv, hd)
    k[torch.rand(k.shape, device="cuda", generator=gen(103)) < share] = 0
    up = make_tree("random", n, 94)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    check_rows(out, q, k, v, up, pos0, hd**-0.5, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))
    for _ in range(20):
        assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e12, 1e20, -1e9])
def test_tree_scores_of_any_size(gpu, form, size):
    """One row's score is far above the others', all of them beyond what fp32 resolves to one: its V comes out.

    With one weight of 1, off by 2^-22 as a pair and a few roundings, the output is off by 8 u; and by what the pairs cut
    of V: a row's largest value is at least 2^3 in its scale (else it has a scale of its own), half a step of the lo part
    is 2^-25, so 2^-28 of the row's largest value."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = uneven(110, n, nh, nkv, hd, pos0)
    row = 137
    k[row, :, 0] = 8.0
    out = run_tree(gpu, q * size, k * (1 if size > 0 else -1), v, make_tree("random", n, 111), pos0, 1.0, 0)
    want = v[row].repeat_interleave(nh // nkv, 0).expand_as(out)
    assert bool(((out - want).abs() <= 8 * U * want.abs() + 2.0**-28 * want.abs().amax(-1, keepdim=True)).all())
    # and small ones with a large scale, or V of any size
    k *= 1e-3
    v *= 2.0 ** torch.randint(-30, 30, (pos0 + n, nkv, 1), device="cuda", generator=gen(112))
    out = run_tree(gpu, q, k, v, make_tree("random", n, 111), pos0, float(abs(size)) * 1e3, 0)
    want = v[row].repeat_interleave(nh // nkv, 0).expand_as(out)
    assert bool(((out - want).abs() <= 8 * U * want.abs() + 2.0**-28 * want.abs().amax(-1, keepdim=True)).all())


# ---------------------------------------------------------------- reordering
def test_reorder_one_slot_looks_at_its_index(gpu):
    x = randn(120, 3, 1, 64)
    y = x.clone()
    for i in (1, 5, -2, 2**31 - 1, -(2**31)):
        index = torch.tensor([i], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        assert gpu.gncx_state_reorder(P(y), 3, 256, 1, 256, 256, P(index)) == INVALID, i
        gpu.gncx_clear_error()
    for i in (0, -1):
        index = torch.tensor([i], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        ok(gpu, gpu.gncx_state_reorder(P(y), 3, 256, 1, 256, 256, P(index)))
        ok(gpu, gpu.gncx_state_reorder(P(y), 3, 0, 1, 0, 256, P(index)))  # strides that no second slot or state uses
    torch.cuda.synchronize()
    assert torch.equal(x, y)
    assert gpu.gncx_state_reorder(P(y), 3, 256, 1, 256, 256, None) == INVALID


# ---------------------------------------------------------------- forms that smaller shapes pass by
def one_launch(nh, nkv, pos0, n, hd, window):
    """Whether few query rows over a short cache go to the form of one launch (148 SMs)."""
    rows, fit = n * nh // nkv, 15 // nkv
    seen = pos0 + n - (max(0, pos0 - window + 1) if window else 0)
    if n > 64:
        return False
    return seen <= (256 if hd > 128 else 768) if rows <= 8 * fit else rows <= 16 * fit and hd <= 128 and seen <= 384


# Head sizes that are no multiple of 16: on the CUDA cores, with splits and records of their own.
OTHER = [(2, 1, 4, 1000, 3, 0), (5, 5, 20, 900, 30, 0), (4, 2, 36, 300, 70, 50), (3, 3, 60, 64, 100, 0), (8, 4, 100, 1000, 9, 0), (6, 3, 132, 2000, 40, 0),
         (12, 4, 136, 8192, 16, 0), (4, 1, 252, 1500, 70, 300), (148, 148, 20, 33, 65, 0), (8, 1, 100, 31, 200, 0), (2, 2, 132, 5001, 2, 4096),
         (16, 2, 252, 32, 65, 7), (1, 1, 12, 70001, 1, 0)]


@pytest.mark.parametrize("nh,nkv,hd,pos0,n,window", OTHER)
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_tree_other_head_sizes(gpu, nh, nkv, hd, pos0, n, window, kind):
    assert hd % 16 and not one_launch(nh, nkv, pos0, n, hd, window)
    rows = pos0 + n
    q, k, v = randn(130, n, nh, hd) * 2, randn(131, rows + 3, nkv, hd), randn(132, rows + 3, nkv, hd)
    k[rows:], v[rows:] = float("nan"), float("nan")
    lo = max(0, pos0 - window + 1) if window else 0
    k[:min(lo, pos0)], v[:min(lo, pos0)] = float("nan"), float("inf")
    up = make_tree(kind, n, pos0 + n + 2)
    keep = k.clone(), v.clone()
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window)
    group = nh // nkv
    for i in sorted({0, n // 2, n - 1}):
        seen = torch.tensor(tree_seen(up, i, pos0, window), device="cuda")
        for h in sorted({0, nh // 2, nh - 1}):
            ref, tol, _, _ = attend(q[i, h], k[seen][:, h // group], v[seen][:, h // group], hd**-0.5)
            assert bool(((out[i, h].double() - ref).abs() <= tol).all()), (i, h)
    assert bool(out.isfinite().all())
    assert torch.equal(out, run_tree(gpu, q, k, v, up, pos0, hd**-0.5, window))
    assert torch.equal(k.view(torch.int32), keep[0].view(torch.int32)) and torch.equal(v.view(torch.int32), keep[1].view(torch.int32))


@pytest.mark.parametrize("form", FORMS)
def test_tree_infinite_and_nan_rows_show_in_each_form(gpu, form):
    """A NaN in a seen row reaches the outputs of its KV head, an infinity of V its column, and no other head's."""
    nh, nkv, hd, pos0, n = FORMS[form]
    group, up = nh // nkv, make_tree("random", n, 141)
    for row in (0, 70, pos0 - 1):
        q, k, v = randn(140, n, nh, hd), randn(141, pos0 + n, nkv, hd), randn(142, pos0 + n, nkv, hd)
        k[row, 0, 5], v[row, 1, 7], v[row, 1, hd - 1] = float("nan"), float("inf"), float("-inf")
        out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0).view(n, nkv, group, hd)
        assert bool(out[:, 0].isnan().all())
        assert bool((out[:, 1, :, 7] == float("inf")).all()) and bool((out[:, 1, :, hd - 1] == float("-inf")).all())
        out[:, 0], out[:, 1, :, 7], out[:, 1, :, hd - 1] = 0, 0, 0
        assert bool(out.isfinite().all())
        v[row, 1] = float("nan")  # all of a row of V
        out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0).view(n, nkv, group, hd)
        assert bool(out[:, 1].isnan().all()) and bool(out[:, 2:].isfinite().all())


@pytest.mark.parametrize("form", [f for f in FORMS if f != "one launch"])
def test_tree_bad_parents_are_an_error_in_each_form(gpu, form):
    nh, nkv, hd, pos0, n = FORMS[form]
    pos0, n = max(pos0, 2000 // nkv), 4
    assert not one_launch(nh, nkv, pos0, n, hd, 0)
    q, k, v = randn(150, n, nh, hd), randn(151, pos0 + n, nkv, hd), randn(152, pos0 + n, nkv, hd)
    out = torch.zeros_like(q)
    for up in ([-1, 1, 0, 0], [-1, 0, 3, 0], [-1, 0, -2, 0], [5, 0, 0, 0], [-1, 0, 0, 2**31 - 1]):
        parents = torch.tensor(up, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        st = gpu.gncx_attention_tree(P(q), P(k), P(v), P(parents), pos0, n, nh, nkv, hd, 0.1, 0, P(out), None, 0)
        assert st == INVALID and gpu.gncx_last_error() == INVALID, up
        gpu.gncx_clear_error()
    ok(gpu, gpu.gncx_sync())
    up = make_tree("random", n, 153)
    check_tree(run_tree(gpu, q, k, v, up, pos0, 0.1, 0), q, k, v, up, pos0, 0.1, 0, [0, 3])


@pytest.mark.parametrize("form", FORMS)
def test_tree_other_branches_do_not_leak_in_each_form(gpu, form):
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = randn(160, n, nh, hd), randn(161, pos0 + n, nkv, hd), randn(162, pos0 + n, nkv, hd)
    up = make_tree("random", n, 163)
    k[pos0 + n - 1], v[pos0 + n - 1] = float("nan"), float("inf")  # no other node's ancestor
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    check_tree(out, q, k, v, up, pos0, hd**-0.5, 0, sorted({0, (n - 1) // 2, max(0, n - 2)}))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["growing", "shrinking", "zeros first", "zeros last", "all zeros"])
def test_tree_sizes_that_change_along_the_cache(gpu, form, kind):
    """K and V whose size at the start of a CTA's rows says little about the others'."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = randn(170, n, nh, hd), randn(171, pos0 + n, nkv, hd), randn(172, pos0 + n, nkv, hd)
    at = torch.linspace(-14, 14, pos0 + n, device="cuda")[:, None, None]
    if kind in ("growing", "shrinking"):
        size = 2.0 ** (at if kind == "growing" else -at)
        k, v = k * size * 2.0**-12, v * size
    rows = torch.arange(pos0 + n, device="cuda")
    none = {"zeros first": rows % 100 < 70, "zeros last": rows % 100 >= 30, "all zeros": rows >= 0}.get(kind, rows < 0)
    k[none], v[none] = 0, 0
    up = make_tree("random", n, 173)
    out = run_tree(gpu, q, k, v, up, pos0, hd**-0.5, 0)
    check_rows(out, q, k, v, up, pos0, hd**-0.5, 0, sorted({0, n // 2, n - 1}), sorted({0, nh // 2, nh - 1}))


@pytest.mark.parametrize("form", FORMS)
def test_tree_infinite_v_among_rows_of_other_sizes(gpu, form):
    """Infinities in small, large and ordinary rows of V, one of each sign in a row and both in a column."""
    nh, nkv, hd, pos0, n = FORMS[form]
    q, k, v = randn(180, n, nh, hd), randn(181, pos0 + n, nkv, hd), randn(182, pos0 + n, nkv, hd)
    v[7], v[90], v[201] = v[7] * 1e-9, v[90] * 1e9, v[201] * 0
    inf = float("inf")
    v[7, 0, 3], v[7, 0, 4], v[90, 0, 5], v[90, 0, hd - 1], v[201, 0, 0], v[150, 0, 6], v[151, 0, 6] = inf, -inf, -inf, inf, inf, inf, -inf
    out = run_tree(gpu, q, k, v, make_tree("random", n, 183), pos0, hd**-0.5, 0).view(n, nkv, nh // nkv, hd)[:, 0]
    for col, want in ((3, inf), (4, -inf), (5, -inf), (hd - 1, inf), (0, inf)):
        assert bool((out[..., col] == want).all()), col
    assert bool(out[..., 6].isnan().all())
    cols = [c for c in range(hd) if c not in (0, 3, 4, 5, 6, hd - 1)]
    assert bool(out[..., cols].isfinite().all())
