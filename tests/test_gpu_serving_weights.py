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


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [0, 10, 20, 24, 26, 29, 32, 40, 70])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_every_size(power, hd, sign):
    """One key's score is far from the others', at 2^power: beyond 2^24 f32 holds the scores' own differences coarsely,
    and the result is that key's value row to the bits that a product keeps (2^-22 of it, and 4 roundings), whatever
    the value scales are; with equal scores it is the mean."""
    rng = np.random.default_rng(power)
    n, n_kv, group = 300, 2, 9                        # 18 rows a kv head: a block of 32
    c = Cache(rng, 1, 1, 400, n_kv, hd)
    c.fill(rng, 0, 0, n)
    win, s = 170, hd ** -0.5
    c.k[0, 0, :n] = 1 if sign > 0 else 3              # the winner's score: 2^power * 3, or -2^power among -3 * 2^power
    c.k[0, 0, win] = 3 if sign > 0 else 1
    c.ks[0, 0, :n] = np.float32(sign * 2.0 ** power / (hd * s))
    c.vs[0, 0, :n] *= np.exp2(rng.integers(-9, 10, (n, n_kv))).astype(np.float32)
    c.vs[0, 0, win] = [3.7, 0.02]
    q = np.ones((1, n_kv * group * hd), np.float32)
    out = torch.empty(1, n_kv * group * hd, device=DEV)
    for max_keys in (0, 1):
        rows = KvRows(ints([0, 1]), ints([n - 1]), n_rows=1, max_rows=1, max_keys=max_keys)
        K.tree_attention_int8(out, T(q), c.up(), 0, rows, n_kv * group, s)
        got = H(out).reshape(n_kv, group, hd).astype(np.float64)
        for kv in range(n_kv):
            cut = slice(kv * hd, (kv + 1) * hd)
            o, bar = A.exact(q[0, :hd], c.k[0, 0, :n, cut], c.ks[0, 0, :n, kv], c.v[0, 0, :n, cut], c.vs[0, 0, :n, kv],
                             s, np.ones(n, bool))
            if power >= 10:                           # the others weigh e^-2048 or nothing
                o = c.v[0, 0, win, cut] * np.float64(c.vs[0, 0, win, kv])
                bar = (2.0 ** -22 + 4 * 2.0 ** -24) * np.linalg.norm(o)
            assert (np.linalg.norm(got[kv] - o, axis=1) <= bar).all(), (power, np.linalg.norm(got[kv] - o, axis=1) / bar)


@pytest.mark.parametrize("power", [-90, -40, 40, 105])
@pytest.mark.parametrize("hd,group", [(128, 2), (128, 20), (64, 1), (64, 9)])
def test_values_of_every_size(power, hd, group):
    """All value scales at 2^power: the result scales with them, to the bar of ordinary values."""
    rng = np.random.default_rng(hd + group)
    n = 700
    c = Cache(rng, 1, 1, 900, 2, hd)
    q = np.empty((2, group, hd), np.float32)
    for kv in range(2):
        cut = slice(kv * hd, (kv + 1) * hd)
        q0, c.k[0, 0, :n, cut], c.ks[0, 0, :n, kv], c.v[0, 0, :n, cut], c.vs[0, 0, :n, kv] = A.history(rng, "plain", n, hd)
        q[kv] = q0 * (1 + 0.1 * rng.standard_normal((group, hd)))
    c.vs[0, 0, :n] *= np.float32(2.0 ** power)
    out = torch.empty(1, 2 * group * hd, device=DEV)
    rows = KvRows(ints([0, 1]), ints([n - 1]), n_rows=1, max_rows=1)
    K.tree_attention_int8(out, T(q.reshape(1, -1)), c.up(), 0, rows, 2 * group, hd ** -0.5)
    got = H(out).reshape(2, group, hd).astype(np.float64)
    for kv in range(2):
        cut = slice(kv * hd, (kv + 1) * hd)
        for h in range(group):
            o, bar = A.exact(q[kv, h], c.k[0, 0, :n, cut], c.ks[0, 0, :n, kv], c.v[0, 0, :n, cut], c.vs[0, 0, :n, kv],
                             hd ** -0.5, np.ones(n, bool))
            assert np.linalg.norm(got[kv, h] - o) <= bar
