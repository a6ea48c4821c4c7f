"""Attention over the INT8 cache by the 2-norm of every row of every head (the bar is derived in attention_model):
ordinary histories, sinks, outlying value scales, value scales of keys that a row does not see."""
import math

import numpy as np
import pytest
import torch

import attention_model as A
from test_gpu_serving import DEV, Cache, H, KvRows, T, as_int64, ints, random_tree, starts_of

from qwenasr_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    from qwenasr_b200 import build
    build.build()
    assert torch.cuda.is_available()


SHAPES = [  # counts, positions, n_kv, group, hd, tree
    ([1, 1, 1], [4, 127, 1700], 2, 2, 128, False),   # single tokens
    ([1, 1], [300, 0], 3, 1, 64, False),             # two heads of 64 share a tile, an odd one
    ([1], [900], 1, 5, 128, False),
    ([3, 2], [130, 0], 2, 1, 128, True),             # blocks of 4, 8, 16 and 32 rows
    ([3, 4], [1, 600], 1, 2, 128, True),
    ([6], [250], 2, 2, 128, True),
    ([31, 7], [1000, 120], 2, 2, 128, True),
    ([29], [333], 3, 1, 64, True),
    ([130], [0], 1, 2, 128, False),                  # prompt chunks
    ([40, 70], [88, 250], 2, 1, 64, False),
]


@pytest.mark.parametrize("counts,positions,n_kv,group,hd,tree", SHAPES)
@pytest.mark.parametrize("kind", ["plain", "peaked", "sink1", "sink2", "sink6", "last3", "last6", "last9", "outlier2",
                                  "outlier3"])
@pytest.mark.parametrize("max_keys", [0, 1])         # split over a cluster as the cache allows, or not at all
def test_rows_by_norm(kind, counts, positions, n_kv, group, hd, tree, max_keys):
    rng = np.random.default_rng(sum(positions) + hd + len(kind))
    n_heads, total = n_kv * group, sum(counts)
    c = Cache(rng, len(counts), 1, 2100, n_kv, hd)
    q = np.empty((total, n_heads, hd), np.float32)
    masks = [w for r in counts for w in random_tree(rng, r)] if tree else None  # no token but itself sees the last
    starts = starts_of(counts)
    for i, (r, p) in enumerate(zip(counts, positions)):
        for kv in range(n_kv):
            cut = slice(kv * hd, (kv + 1) * hd)
            q0, *rest = A.history(rng, kind, p + r, hd)
            c.k[i, 0, :p + r, cut], c.ks[i, 0, :p + r, kv], c.v[i, 0, :p + r, cut], c.vs[i, 0, :p + r, kv] = rest
            at = q[starts[i]:starts[i + 1], kv * group:(kv + 1) * group]
            at[:] = q0 * (1 + 0.1 * rng.standard_normal(at.shape))
    rows = KvRows(ints(starts), ints(positions), n_rows=total, max_rows=max(counts), max_keys=max_keys)
    out, scale = torch.empty(total, n_heads * hd, device=DEV), 1 / math.sqrt(hd)
    K.tree_attention_int8(out, T(q.reshape(total, -1)), c.up(), 0, rows, n_heads, scale, as_int64(masks) if tree else None)
    got = H(out).reshape(total, n_heads, hd).astype(np.float64)
    for i, (r, p) in enumerate(zip(counts, positions)):
        for t in range(r):
            row = starts[i] + t
            see = np.ones(p + r, bool)
            see[p:] = [masks[row] >> j & 1 if tree else j <= t for j in range(r)]
            for h in range(n_heads):
                kv = h // group
                cut = slice(kv * hd, (kv + 1) * hd)
                o, bar = A.exact(q[row, h], c.k[i, 0, :p + r, cut], c.ks[i, 0, :p + r, kv], c.v[i, 0, :p + r, cut],
                                 c.vs[i, 0, :p + r, kv], scale, see)
                err = np.linalg.norm(got[row, h] - o)
                assert err <= bar, (i, t, h, err / bar, err / np.linalg.norm(o))
