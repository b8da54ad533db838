"""Operators for several candidates and bounded caches over more of what their
documentation allows: long caches, values of very different size, rows that are
all protected, forms that other tests pass by.  Tolerances as derived in
test_candidates_gpu.py."""
import numpy as np
import pytest

from test_candidates_gpu import _clean, attend, check_tree, make_tree, randn, run_tree, tree_seen  # noqa: F401

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
