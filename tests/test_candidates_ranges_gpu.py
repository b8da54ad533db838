"""Operators for several candidates and bounded caches over more of what their
documentation allows: long caches, values of very different size, rows that are
all protected, forms that other tests pass by.  Tolerances as derived in
test_candidates_gpu.py."""
import numpy as np
import pytest

from test_candidates_gpu import (EVICTS, _clean, attend, check_tree, evict_weights, gen, make_tree, randn, run_evict, run_tree,  # noqa: F401
                                 tree_seen)

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
