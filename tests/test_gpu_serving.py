"""The serving operators on the GPU against plain 64-bit implementations:
quantised KV append and read-back, attention over the INT8 cache (single
tokens, trees, chunks), token picks under rules.

Bars.  Codes, read-back and picked logits are fixed sequences of f32 roundings
and are compared bit for bit.  Attention: with
  dS  = scale * max|q| * 2^-22 * max_j sum_d |k_jd|  (q to 23 bits of its row's
        maximum, half a step)  + 8 * 2^-24 * max|S|  (the f32 steps from the sum
        to the exponent's argument),
a weight is off by a factor e^(2 dS) * (1 + 2^-21) (the exponential) and by 2^-23 of
the largest weight of its 128-key tile (23 bits, half a step and the largest's own
rounding); every f32 sum of n terms of one sign by n * 2^-24.  All of it multiplies values of at most vmax, so
|out - exact| <= vmax * (4 dS + 2^-20 + 128 * 2^-23 + (n / 128 + 128) * 2^-24).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from qwenasr_b200 import kernels as K  # noqa: E402
from qwenasr_b200 import synthetic  # noqa: E402
from qwenasr_b200.kvcache import KvCacheInt8, KvRows  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _lib():
    from qwenasr_b200 import build
    build.build()
    assert torch.cuda.is_available()


def T(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def ints(a):
    return torch.tensor(list(a), dtype=torch.int32, device=DEV)


def H(t):
    torch.cuda.synchronize()
    return t.detach().cpu().numpy()


def starts_of(counts):
    return [0] + [int(x) for x in np.cumsum(counts)]


def quantize(x, hd):
    """Rows [n, n_kv * hd] -> codes, scales [n, n_kv] by the quantiser rule of the model files."""
    q, s = synthetic.quantize_np(x.reshape(-1, hd))
    return q.reshape(x.shape), s.reshape(x.shape[0], -1)


class Cache:
    """A cache on the device and its host copy, filled with garbage (any codes, NaN scales)."""

    def __init__(self, rng, slots, layers, max_seq, n_kv, hd):
        self.n_kv, self.hd, self.d = n_kv, hd, n_kv * hd
        shape = (slots, layers, max_seq)
        self.k, self.v = (rng.integers(-128, 128, shape + (self.d,)).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (np.full(shape + (n_kv,), np.nan, np.float32) for _ in range(2))

    def fill(self, rng, slot, layer, n, size=1.0):
        for c, s in ((self.k, self.ks), (self.v, self.vs)):
            x = (rng.standard_normal((n, self.d)) * size).astype(np.float32)
            c[slot, layer, :n], s[slot, layer, :n] = quantize(x, self.hd) if n else (c[slot, layer, :0], s[slot, layer, :0])

    def up(self):
        self.dev = KvCacheInt8(T(self.k), T(self.v), T(self.ks), T(self.vs))
        return self.dev


# ------------------------------------------------------------ append, read --
@pytest.mark.parametrize("counts,positions,n_kv,hd,pad", [
    ([1], [0], 8, 128, 0),
    ([1, 1, 1], [5, 0, 39], 8, 128, 0),
    ([3, 0, 7, 1], [0, 4, 33, 39], 1, 128, 2),   # an empty sequence, rows behind the last one
    ([0, 0], [0, 40], 2, 64, 3),
    ([5, 9], [31, 2], 3, 64, 1),                  # an odd number of half-warp heads
    ([40], [0], 5, 128, 0),                       # a whole slot
    ([2] * 70, [7] * 70, 2, 64, 5),               # more sequences than two ballots take
])
def test_append_and_read(counts, positions, n_kv, hd, pad):
    rng = np.random.default_rng(sum(counts) + n_kv)
    n, layers, max_seq, layer = len(counts), 3, 40, 1
    c = Cache(rng, n + 1, layers, max_seq, n_kv, hd)
    dev = c.up()
    slots = rng.permutation(n + 1)[:n]
    total = sum(counts)
    x = [(rng.standard_normal((total + pad, n_kv * hd)) * np.exp(rng.normal(0, 3, (total + pad, 1)))).astype(np.float32)
         for _ in range(2)]
    flag = ints([0])
    rows = KvRows(ints(starts_of(counts)), ints(positions), ints(slots), n_rows=total + pad, max_rows=max(counts),
                  bad_flag=flag)
    K.kv_append_int8(dev, layer, rows, T(x[0]), T(x[1]))
    back = [torch.full((total + pad, n_kv * hd), 7.0, device=DEV) for _ in range(2)]
    K.kv_read_int8(back[0], back[1], dev, layer, rows)
    want = [a.copy() for a in (c.k, c.v, c.ks, c.vs)]
    ref = [np.full((total + pad, n_kv * hd), 7.0, np.float32) for _ in range(2)]
    for i, (cnt, pos, sl) in enumerate(zip(counts, positions, slots)):
        r0 = starts_of(counts)[i]
        for w in range(2):
            if cnt:
                q, s = quantize(x[w][r0:r0 + cnt], hd)
                want[w][sl, layer, pos:pos + cnt], want[w + 2][sl, layer, pos:pos + cnt] = q, s
                ref[w][r0:r0 + cnt] = (q.reshape(cnt, n_kv, hd).astype(np.float32) * s[..., None]).reshape(cnt, -1)
    for got, w in zip((dev.k, dev.v, dev.k_scales, dev.v_scales), want):
        assert np.array_equal(H(got), w, equal_nan=w.dtype == np.float32)
    for got, w in zip(back, ref):
        assert np.array_equal(H(got), w)
    assert H(flag)[0] == 0


def test_append_matches_the_row_quantiser():
    """The codes of a head are those of qasr_quantize_f32_to_int8 on that head row."""
    rng = np.random.default_rng(4)
    x = T((rng.standard_normal((37, 8 * 128)) * 3).astype(np.float32))
    cache = KvCacheInt8.zeros(1, 1, 64, 8, 128)
    rows = KvRows(ints([0, 37]), ints([11]), n_rows=37, max_rows=37)
    K.kv_append_int8(cache, 0, rows, x, x)
    q, s = torch.empty(37 * 8, 128, dtype=torch.int8, device=DEV), torch.empty(37 * 8, device=DEV)
    K.quantize_f32_to_int8(x, 37 * 8, 128, q, s)
    assert torch.equal(cache.k[0, 0, 11:48].view(-1, 128), q) and torch.equal(cache.v[0, 0, 11:48].view(-1, 128), q)
    assert torch.equal(cache.k_scales[0, 0, 11:48].flatten(), s)


def test_append_extremes():
    """Zero rows, tiny rows, the largest values, NaN and infinities: each head on its own."""
    x = np.zeros((8, 2 * 64), np.float32)
    x[1, :64] = 2.0 ** -125                 # 127 / absmax overflows: stored as zeros
    x[1, 64:] = 2.0 ** -118
    x[2, :] = np.float32(3.4e38)
    x[2, 5] = -np.float32(3.4e38)
    x[3, 3], x[3, 70] = np.nan, 1.0
    x[4, 3], x[4, 70] = np.inf, -2.0
    x[5, 3], x[5, 70] = -np.inf, np.nan
    x[6, :64] = np.linspace(-1, 1, 64)      # codes at halves and at both ends
    x[6, 64:] = 1.0
    x[7, 0] = 127.0
    x[7, 1:64] = np.arange(63) + 0.5        # scale 1: halves go away from zero
    cache = KvCacheInt8.zeros(1, 1, 8, 2, 64)
    rows = KvRows(ints([0, 8]), ints([0]), n_rows=8, max_rows=8)
    K.kv_append_int8(cache, 0, rows, T(x), T(-x))
    k, v, ks, vs = (H(t)[0, 0] for t in (cache.k, cache.v, cache.k_scales, cache.v_scales))
    assert not k[0].any() and not ks[0].any() and not k[1, :64].any() and ks[1, 0] == 0
    assert (k[1, 64:] == 127).all() and ks[1, 1] == np.float32(2.0 ** -118) / np.float32(127)
    assert k[2, 5] == -127 and k[2, 6] == 127 and v[2, 5] == 127 and np.isfinite(ks[2]).all()
    assert np.isnan(ks[3, 0]) and ks[3, 1] == np.float32(1) / np.float32(127) and k[3, 70] == 127
    assert np.isnan(ks[4, 0]) and v[4, 70] == 127 and np.isfinite(vs[4, 1])
    assert np.isnan(ks[5]).all() and np.isnan(vs[5]).all()
    q, s = quantize(x[6:], 64)
    assert np.array_equal(k[6:], q) and np.array_equal(ks[6:], s)
    assert (k[7, 1:64] == np.arange(63) + 1).all() and (v[7, 1:64] == -(np.arange(63) + 1)).all()


def test_append_picks_source_rows():
    rng = np.random.default_rng(8)
    x, y = (rng.standard_normal((20, 128)).astype(np.float32) for _ in range(2))
    cache, flag = KvCacheInt8.zeros(2, 1, 16, 1, 128), ints([0])
    rows = KvRows(ints([0, 3, 5]), ints([2, 0]), n_rows=6, max_rows=3, bad_flag=flag)
    K.kv_append_int8(cache, 0, rows, T(x), T(y), ints([7, 7, 19, 0, 12, 99]))  # row 5 belongs to nobody
    q, s = quantize(x[[7, 7, 19]], 128)
    assert np.array_equal(H(cache.k)[0, 0, 2:5], q) and np.array_equal(H(cache.k_scales)[0, 0, 2:5], s)
    q, s = quantize(y[[0, 12]], 128)
    assert np.array_equal(H(cache.v)[1, 0, :2], q) and H(flag)[0] == 0
    before = H(cache.k).copy()
    K.kv_append_int8(cache, 0, rows, T(x), T(y), ints([20, -1, 3, 1, 1, 0]))  # two source rows that do not exist
    after = H(cache.k)
    assert H(flag)[0] == 1 and np.array_equal(after[0, 0, 2:4], before[0, 0, 2:4])
    assert np.array_equal(after[0, 0, 4], quantize(x[[3]], 128)[0][0])


BAD = [  # (row_starts, positions, slots, max_rows): sequence 1 of three does not fit
    ([0, 2, 4, 6], [0, 15, 0], [0, 1, 2], 2),     # past the cache
    ([0, 2, 4, 6], [0, -1, 0], [0, 1, 2], 2),
    ([0, 2, 4, 6], [0, 3, 0], [0, 3, 2], 2),      # no such slot
    ([0, 2, 4, 6], [0, 3, 0], [0, -1, 2], 2),
    ([0, 1, 5, 6], [0, 3, 0], [0, 1, 2], 2),      # longer than max_rows
    ([0, 2, 4, 6], [0, 2147483647, 0], [0, 1, 2], 2),
]


@pytest.mark.parametrize("starts,positions,slots,max_rows", BAD)
def test_bad_sequences_are_left_out(starts, positions, slots, max_rows):
    rng = np.random.default_rng(2)
    c = Cache(rng, 3, 2, 16, 2, 64)
    for sl in range(3):
        c.fill(rng, sl, 1, 16)
    dev, flag = c.up(), ints([0])
    rows = KvRows(ints(starts), ints(positions), ints(slots), n_rows=6, max_rows=max_rows, bad_flag=flag)
    x = rng.standard_normal((6, 128)).astype(np.float32)
    bad = slice(starts[1], starts[2])
    out, back = torch.full((6, 256), 9.0, device=DEV), torch.full((6, 128), 9.0, device=DEV)
    K.tree_attention_int8(out, T(rng.standard_normal((6, 256)).astype(np.float32)), dev, 1, rows, 4, 0.125)
    assert H(flag)[0] == 1
    assert (H(out)[bad] == 9).all() and (H(out)[:starts[1]] != 9).all() and (H(out)[starts[2]:] != 9).all()
    flag.zero_()
    K.kv_read_int8(back, None, dev, 1, rows)
    assert H(flag)[0] == 1 and (H(back)[bad] == 9).all() and (H(back)[starts[2]:] != 9).all()
    flag.zero_()
    K.kv_append_int8(dev, 1, rows, T(x), T(x))
    k = H(dev.k)
    assert H(flag)[0] == 1 and np.array_equal(k[1], c.k[1]) and np.array_equal(k[:, 0], c.k[:, 0])
    assert np.array_equal(k[0, 1, positions[0]], quantize(x[:1], 64)[0][0])


def test_starts_in_disorder_and_outside():
    """Starts that fall or point outside the packed rows touch nothing they should not."""
    rng = np.random.default_rng(3)
    c = Cache(rng, 3, 1, 16, 1, 64)
    for sl in range(3):
        c.fill(rng, sl, 0, 16)
    dev = c.up()
    for starts in ([0, 4, 2, 6], [-3, 2, 4, 6], [0, 2, 4, 2147483647], [5, 3, 1, 0], [0, 2, 4, -2147483648]):
        flag = ints([0])
        rows = KvRows(ints(starts), ints([0, 0, 0]), None, n_rows=6, max_rows=4, bad_flag=flag)
        out = torch.full((7, 64), 9.0, device=DEV)
        K.tree_attention_int8(out[:6], T(rng.standard_normal((6, 64)).astype(np.float32)), dev, 0, rows, 1, 0.125)
        K.kv_read_int8(out[:6], None, dev, 0, rows)
        K.kv_append_int8(dev, 0, rows, torch.zeros(6, 64, device=DEV), torch.zeros(6, 64, device=DEV))
        assert H(flag)[0] == 1 and (H(out)[6] == 9).all()


# --------------------------------------------------------------- attention --
def random_tree(rng, n):
    up = []
    for t in range(n):
        parent = -1 if t == 0 else int(rng.integers(max(0, t - 5), t))
        up.append((up[parent] if t else 0) | 1 << t)
    return up


def as_int64(words):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device=DEV)


def attend_exact(c, layer, q, counts, positions, slots, masks, n_heads, scale):
    """(out, bound) in 64 bits; rows of no sequence are None."""
    out, bar = np.full(q.shape, np.nan), np.zeros((q.shape[0], 1))
    g, hd = n_heads // c.n_kv, c.hd
    for i, (n, p, sl) in enumerate(zip(counts, positions, slots)):
        r0 = starts_of(counts)[i]
        for h in range(n_heads):
            kv = h // g
            cut = slice(kv * hd, (kv + 1) * hd)
            k = c.k[sl, layer, :p + n, cut].astype(np.float64) * c.ks[sl, layer, :p + n, kv, None].astype(np.float64)
            v = c.v[sl, layer, :p + n, cut].astype(np.float64) * c.vs[sl, layer, :p + n, kv, None].astype(np.float64)
            for t in range(n):
                see = np.ones(p + n, bool)
                see[p:] = [(masks[r0 + t] >> j & 1) == 1 if masks else j <= t for j in range(n)]
                x = q[r0 + t, h * hd:(h + 1) * hd].astype(np.float64)
                o = np.zeros(hd)
                if see.any():
                    s = scale * (k[see] @ x)
                    w = np.exp(s - s.max())
                    o = w @ v[see] / w.sum()
                    ds = scale * np.abs(x).max() * 2.0 ** -22 * np.abs(k[see]).sum(1).max() + 2.0 ** -21 * np.abs(s).max()
                    tol = 4 * ds + 2.0 ** -20 + 2.0 ** -16 + (len(s) / 128 + 128) * 2.0 ** -24
                    bar[r0 + t] = max(bar[r0 + t, 0], np.abs(v[see]).max() * tol)
                out[r0 + t, h * hd:(h + 1) * hd] = o
    return out, bar


def check_attend(rng, counts, positions, n_kv, group, hd, tree, size=1.0, pad=1, layers=2, masks=None, max_seq=None,
                 max_keys=0):
    n, total, n_heads = len(counts), sum(counts), n_kv * group
    max_seq = max_seq or max(p + r for p, r in zip(positions, counts)) + 3
    c = Cache(rng, n + 1, layers, max_seq, n_kv, hd)
    slots = [int(x) for x in rng.permutation(n + 1)[:n]]
    for sl, p, r in zip(slots, positions, counts):
        c.fill(rng, sl, layers - 1, p + r)
    q = (rng.standard_normal((total + pad, n_heads * hd)) * size).astype(np.float32)
    if tree and masks is None:
        masks = [w for r in counts for w in random_tree(rng, r)]
    scale = 1.0 / math.sqrt(hd)
    flag = ints([0])
    rows = KvRows(ints(starts_of(counts)), ints(positions), ints(slots), n_rows=total + pad, max_rows=max(counts),
                  max_keys=max_keys, bad_flag=flag)
    out = torch.full((total + pad, n_heads * hd), 5.0, device=DEV)
    dev_masks = as_int64(masks + [(1 << 64) - 1] * pad) if tree else None
    K.tree_attention_int8(out, T(q), c.up(), layers - 1, rows, n_heads, scale, dev_masks)
    got = H(out)
    ref, bar = attend_exact(c, layers - 1, q, counts, positions, slots, masks if tree else None, n_heads, scale)
    assert H(flag)[0] == 0
    assert (got[total:] == 5).all()
    err = np.abs(got[:total] - ref[:total])
    assert (err <= bar[:total]).all(), (err.max(), bar[:total].max(), np.argwhere(err > bar[:total])[:4])


@pytest.mark.parametrize("counts,positions,n_kv,group,hd", [
    ([1], [0], 8, 2, 128),                                  # a first token: one key
    ([1, 1, 1], [1, 126, 127], 2, 2, 128),                  # around the end of a 128-key tile
    ([1, 1, 1, 1], [128, 255, 256, 2000], 1, 1, 128),
    ([1] * 5, [3, 900, 0, 511, 40], 3, 1, 64),              # head_dim 64, an odd number of kv heads
    ([1, 0, 1], [700, 20, 30], 4, 7, 128),                  # an empty sequence, seven heads a group
    ([1, 1], [300, 5], 1, 64, 64),                          # the largest group
    ([1, 1], [300, 5], 2, 33, 128),
    ([1], [5000], 1, 4, 128),                               # many tiles for one head
])
def test_decode_steps(counts, positions, n_kv, group, hd):
    check_attend(np.random.default_rng(sum(positions) + hd), counts, positions, n_kv, group, hd, tree=False)


@pytest.mark.parametrize("counts,positions,n_kv,group,hd", [
    ([2], [0], 1, 1, 128),
    ([7, 31, 1], [120, 0, 1000], 2, 2, 128),
    ([64, 3], [60, 127], 2, 2, 128),                        # bit 63; a tree over a tile's end
    ([64, 64], [0, 65], 1, 1, 64),
    ([13, 0, 29], [500, 9, 77], 3, 3, 64),
    ([64], [333], 1, 16, 128),                              # 1024 query rows for one kv head
])
def test_trees(counts, positions, n_kv, group, hd):
    check_attend(np.random.default_rng(sum(positions) + hd), counts, positions, n_kv, group, hd, tree=True)


@pytest.mark.parametrize("counts,positions,n_kv,group,hd", [
    ([130], [0], 2, 2, 128),                                # a prompt from nothing
    ([65, 200, 1], [129, 0, 300], 1, 2, 128),               # chunks over a history
    ([97], [31], 3, 1, 64),
    ([40, 7], [88, 250], 1, 5, 64),
])
def test_chunks(counts, positions, n_kv, group, hd):
    check_attend(np.random.default_rng(sum(positions) + hd), counts, positions, n_kv, group, hd, tree=False)


@pytest.mark.parametrize("max_keys", [1, 300, 2100, 1 << 30])
def test_max_keys_is_a_hint(max_keys):
    """A bound that is far off changes how the work is split, not what comes out."""
    rng = np.random.default_rng(max_keys % 1000)
    check_attend(rng, [1, 1, 1], [2000, 0, 777], 2, 2, 128, tree=False, max_keys=max_keys, max_seq=4100)
    check_attend(rng, [31], [1900], 1, 2, 64, tree=True, max_keys=max_keys)


@pytest.mark.parametrize("counts,group,hd,tree", [
    ([1, 1], 2, 128, False), ([1], 4, 64, False), ([4], 2, 128, True), ([7], 2, 128, True), ([5], 3, 64, True),
    ([16], 2, 128, True), ([40], 1, 64, True), ([33], 2, 128, False),
])
def test_many_tiles_per_cta(counts, group, hd, tree):
    """With the hint at one key nothing is split: a dozen tiles and more go through one CTA's ring."""
    rng = np.random.default_rng(group * hd + sum(counts))
    check_attend(rng, counts, [1500 + 130 * i for i in range(len(counts))], 2, group, hd, tree=tree, max_keys=1)


def test_full_cache():
    check_attend(np.random.default_rng(1), [2, 1], [126, 127], 2, 2, 128, tree=False, max_seq=128, pad=0)


@pytest.mark.parametrize("size", [0.0, 1e-30, 40.0, 1e4])
def test_query_sizes(size):
    """Flat and very peaked softmaxes: a zero query averages, a large one picks."""
    check_attend(np.random.default_rng(5), [1, 4], [600, 129], 2, 2, 128, tree=False, size=size)


def test_masks_that_leave_nothing():
    """Rows that see no key are zero; a token need not see itself; bits beyond the tree mean nothing."""
    rng = np.random.default_rng(6)
    masks = [0, 0b10, 0b101 | 1 << 40, 0, (1 << 64) - 1, 0b1]
    check_attend(rng, [3, 3], [0, 0], 2, 2, 128, tree=True, masks=list(masks))
    check_attend(rng, [3, 3], [0, 200], 1, 3, 64, tree=True, masks=list(masks))


def test_nan_stays_where_it_is_seen():
    """A tree row whose scales are NaN or infinite reaches the tokens that see it and no other; so does a
    query of NaN or infinity."""
    rng = np.random.default_rng(7)
    n, p, n_kv, hd = 6, 130, 2, 128
    c = Cache(rng, 1, 1, 200, n_kv, hd)
    c.fill(rng, 0, 0, p + n)
    masks = [0b1, 0b11, 0b101, 0b1101, 0b11011, 0b100001]
    clean = Cache(rng, 1, 1, 200, n_kv, hd)
    for a in ("k", "v", "ks", "vs"):
        setattr(clean, a, getattr(c, a).copy())
    c.vs[0, 0, p + 2] = np.inf      # seen by tokens 2 and 3
    c.ks[0, 0, p + 4, 1] = np.nan   # seen by token 4, second kv head
    c.vs[0, 0, p + 5, 0] = np.nan   # seen by token 5, first kv head
    q = rng.standard_normal((n, 4 * hd)).astype(np.float32)
    q[1, 3 * hd + 5] = np.nan       # token 1, head 3
    q[0, 7] = np.inf                # token 0, head 0
    rows = KvRows(ints([0, n]), ints([p]), n_rows=n, max_rows=n)
    out = torch.empty(n, 4 * hd, device=DEV)
    K.tree_attention_int8(out, T(q), c.up(), 0, rows, 4, 0.1, as_int64(masks))
    got = H(out).reshape(n, 4, hd)
    bad = np.zeros((n, 4), bool)
    bad[2:4] = True
    bad[4, 2:], bad[5, :2], bad[1, 3], bad[0, 0] = True, True, True, True
    assert not np.isfinite(got[bad]).any()
    q2 = np.where(np.isfinite(q), q, 0).astype(np.float32)
    ref, bar = attend_exact(clean, 0, q2, [n], [p], [0], masks, 4, 0.1)
    ref = ref.reshape(n, 4, hd)
    assert (np.abs(got - ref)[~bad] <= bar.max()).all()


def test_value_scales_of_every_size():
    """Value rows from tiny to huge in one history: the error is measured against the largest one."""
    rng = np.random.default_rng(9)
    c = Cache(rng, 1, 1, 400, 1, 128)
    c.fill(rng, 0, 0, 390)
    c.vs[0, 0, :390] *= np.exp2(rng.integers(-60, 60, (390, 1))).astype(np.float32)
    c.vs[0, 0, 100:130] = 0
    q = rng.standard_normal((1, 256)).astype(np.float32)
    rows = KvRows(ints([0, 1]), ints([389]), n_rows=1, max_rows=1)
    out = torch.empty(1, 256, device=DEV)
    K.tree_attention_int8(out, T(q), c.up(), 0, rows, 2, 0.0884)
    ref, bar = attend_exact(c, 0, q, [1], [389], [0], None, 2, 0.0884)
    assert (np.abs(H(out) - ref) <= bar).all()


def test_long_cache_offsets():
    """Slots beyond 2^32 bytes of codes and rows near the end of a 1.1-million-row slot."""
    n_kv, hd, max_seq, slots = 16, 128, 1_100_000, 2
    cache = KvCacheInt8.zeros(slots, 1, max_seq, n_kv, hd)
    assert cache.k.numel() > 1 << 32
    rng = np.random.default_rng(10)
    n, p = 5, max_seq - 300
    x, y = (rng.standard_normal((300, n_kv * hd)).astype(np.float32) for _ in range(2))
    K.kv_append_int8(cache, 0, KvRows(ints([0, 300]), ints([p]), ints([1]), n_rows=300, max_rows=300), T(x), T(y))
    (kq, ks), (vq, vs) = quantize(x, hd), quantize(y, hd)
    assert np.array_equal(H(cache.k[1, 0, p:]), kq) and np.array_equal(H(cache.v_scales[1, 0, p:]), vs)
    back = torch.empty(n, n_kv * hd, device=DEV)
    K.kv_read_int8(None, back, cache, 0, KvRows(ints([0, n]), ints([max_seq - n]), ints([1]), n_rows=n, max_rows=n))
    assert np.array_equal(H(back), (vq[-n:].reshape(n, n_kv, hd).astype(np.float32) * vs[-n:, :, None]).reshape(n, -1))
    # all rows but the last 300 are zeros: equal scores 0 and values 0
    q = (rng.standard_normal((1, n_kv * hd)) * 12).astype(np.float32)
    out = torch.empty(1, n_kv * hd, device=DEV)
    K.tree_attention_int8(out, T(q), cache, 0, KvRows(ints([0, 1]), ints([max_seq - 1]), ints([1]), n_rows=1,
                                                      max_rows=1), n_kv, 0.0884)
    got = H(out).reshape(n_kv, hd)
    for h in range(n_kv):
        cut = slice(h * hd, (h + 1) * hd)
        k = kq[:, cut].astype(np.float64) * ks[:, h, None]
        s = 0.0884 * (k @ q[0, cut].astype(np.float64))
        mx = max(s.max(), 0)
        w = np.exp(s - mx)
        ref = w @ (vq[:, cut].astype(np.float64) * vs[:, h, None]) / (w.sum() + (max_seq - 300) * np.exp(-mx))
        ds = 0.0884 * np.abs(q[0, cut]).max() * 2.0 ** -22 * np.abs(k).sum(1).max() + 2.0 ** -21 * np.abs(s).max()
        tol = 4 * ds + 2.0 ** -20 + 2.0 ** -16 + (max_seq / 128 + 128) * 2.0 ** -24
        assert (np.abs(got[h] - ref) <= np.abs(y).max() * tol).all()


def test_another_stream_and_repeat():
    """The same call twice and on a side stream gives the same bits (no atomics in any order)."""
    rng = np.random.default_rng(11)
    c = Cache(rng, 4, 1, 700, 2, 128)
    for sl in range(4):
        c.fill(rng, sl, 0, 700)
    dev = c.up()
    q = T(rng.standard_normal((4, 512)).astype(np.float32))
    rows = KvRows(ints([0, 1, 2, 3, 4]), ints([699, 3, 128, 400]), n_rows=4, max_rows=1)
    outs = [torch.empty(4, 512, device=DEV) for _ in range(3)]
    K.tree_attention_int8(outs[0], q, dev, 0, rows, 4, 0.1)
    K.tree_attention_int8(outs[1], q, dev, 0, rows, 4, 0.1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.tree_attention_int8(outs[2], q, dev, 0, rows, 4, 0.1)
    s.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_graphs_follow_positions():
    """Two captured steps (append + attention) over one cache, replayed with positions and rows changed in
    place, alone and on two streams at once, equal the eager calls."""
    rng = np.random.default_rng(12)
    n_kv, hd, n_heads = 2, 128, 4
    c = Cache(rng, 4, 1, 400, n_kv, hd)
    for sl in range(4):
        c.fill(rng, sl, 0, 400)
    dev = c.up()
    graphs, parts = [], []
    for slots in ([0, 1], [2, 3]):
        s = torch.cuda.Stream()
        pos = ints([100, 10])
        kn, vn = torch.zeros(2, n_kv * hd, device=DEV), torch.zeros(2, n_kv * hd, device=DEV)
        q, out = torch.zeros(2, n_heads * hd, device=DEV), torch.zeros(2, n_heads * hd, device=DEV)
        rows = KvRows(ints([0, 1, 2]), pos, ints(slots), n_rows=2, max_rows=1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            K.kv_append_int8(dev, 0, rows, kn, vn)
            K.tree_attention_int8(out, q, dev, 0, rows, n_heads, 0.1)
        graphs.append((g, s))
        parts.append((pos, kn, vn, q, out, rows))
    for step in range(3):
        for i, (pos, kn, vn, q, out, rows) in enumerate(parts):
            pos.copy_(ints([130 * step + 5 + i, 399 - step]))
            for t in (kn, vn, q):
                t.copy_(T(rng.standard_normal(t.shape).astype(np.float32)))
        torch.cuda.synchronize()
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        replayed = [p[4].clone() for p in parts]
        for i, (pos, kn, vn, q, out, rows) in enumerate(parts):
            K.kv_append_int8(dev, 0, rows, kn, vn)
            K.tree_attention_int8(out, q, dev, 0, rows, n_heads, 0.1)
            torch.cuda.synchronize()
            assert torch.equal(out, replayed[i])


def test_first_calls_under_capture():
    """A process whose very first calls of every operator are captured into a graph."""
    code = '''
import torch
from qwenasr_b200 import kernels as K
from qwenasr_b200.kvcache import KvCacheInt8, KvRows
i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
cache = KvCacheInt8.zeros(1, 1, 300, 2, 128)
rows = KvRows(i32([0, 3]), i32([0]), n_rows=3, max_rows=3)
k, v, q = torch.randn(3, 256, device="cuda"), torch.randn(3, 256, device="cuda"), torch.randn(3, 512, device="cuda")
out, back, ids, logits = torch.empty_like(q), torch.empty_like(k), i32([7, 7, 7]), torch.randn(3, 1000, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    K.kv_append_int8(cache, 0, rows, k, v)
    K.kv_read_int8(back, None, cache, 0, rows)
    K.tree_attention_int8(out, q, cache, 0, rows, 4, 0.1)
    K.logits_pick(ids, None, logits, 3, 1000)
g.replay()
torch.cuda.synchronize()
assert ids.tolist() == logits.argmax(1).tolist()
assert (back - k).abs().max() <= k.abs().max() / 127 and torch.isfinite(out).all()
g2, o2 = out.clone(), out.zero_()
K.tree_attention_int8(out, q, cache, 0, rows, 4, 0.1)
assert torch.equal(out, g2)
print("captured")
'''
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_two_host_threads():
    """Calls from two threads on two streams at once, over one cache: each gets what it gets alone."""
    import threading
    rng = np.random.default_rng(14)
    c = Cache(rng, 2, 1, 600, 2, 128)
    for sl in range(2):
        c.fill(rng, sl, 0, 600)
    dev = c.up()
    work = []
    for sl in range(2):
        q = T(rng.standard_normal((40, 512)).astype(np.float32))
        rows = KvRows(ints([0, 40]), ints([500 + sl]), ints([sl]), n_rows=40, max_rows=40)
        logits = T(rng.standard_normal((3, 5000)).astype(np.float32))
        work.append((q, rows, torch.empty_like(q), logits, ints([0, 0, 0]), torch.cuda.Stream()))
    alone = []
    for q, rows, out, logits, ids, _ in work:
        K.tree_attention_int8(out, q, dev, 0, rows, 4, 0.1)
        K.logits_pick(ids, None, logits, 3, 5000)
        alone.append((out.clone(), ids.clone()))
        out.zero_()
        ids.zero_()
    torch.cuda.synchronize()
    failed = []

    def run(i):
        q, rows, out, logits, ids, s = work[i]
        try:
            with torch.cuda.stream(s):
                for _ in range(50):
                    K.tree_attention_int8(out, q, dev, 0, rows, 4, 0.1)
                    K.logits_pick(ids, None, logits, 3, 5000)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for (q, rows, out, logits, ids, s), (o, n) in zip(work, alone):
        assert torch.equal(out, o) and torch.equal(ids, n)


def test_wrong_device_and_shapes_raise():
    cache = KvCacheInt8.zeros(1, 1, 8, 1, 64)
    rows = KvRows(ints([0, 1]), ints([0]), n_rows=1, max_rows=1)
    x = torch.zeros(1, 64, device=DEV)
    with pytest.raises(ValueError):
        K.kv_append_int8(cache, 0, rows, x.cpu(), x)
    with pytest.raises(ValueError):
        K.kv_append_int8(cache, 0, rows, x.half(), x)
    with pytest.raises(ValueError):
        K.tree_attention_int8(torch.empty(1, 32, device=DEV), x, cache, 0, rows, 1, 0.1)
    with pytest.raises(ValueError):
        K.tree_attention_int8(torch.empty(1, 64, device=DEV), x, cache, 0, rows, 1, 0.1, ints([1]))
    with pytest.raises(ValueError):
        KvCacheInt8(cache.k, cache.v, cache.k_scales, cache.v_scales[:, :, :4])
    with pytest.raises(ValueError):
        KvRows(ints([0, 1]), ints([]), n_rows=1, max_rows=1)
    with pytest.raises(ValueError):
        K.logits_pick(ints([0]), None, torch.zeros(1, 8, device=DEV), 1, 9)


# -------------------------------------------------------------------- pick --
def pick_ref(x, hist, rep, pres, freq, bias, allow):
    """The rules row by row in f32, rounding by rounding; (ids, values)."""
    y, ids = x.copy(), []
    V = x.shape[1]
    for m in range(x.shape[0]):
        tok, n = np.unique(np.asarray(hist[m], np.int64), return_counts=True) if hist is not None else ([], [])
        for t, c in zip(tok, n):
            if not 0 <= t < V:
                continue
            l = y[m, t]
            l = l / rep[m] if l > 0 else l * rep[m]
            y[m, t] = l - (pres[m] + freq[m] * np.float32(c))
        if bias is not None:
            for t, b in dict(bias[m]).items():  # the last entry for a token
                if 0 <= t < V:
                    y[m, t] = y[m, t] + np.float32(b)
        ok = np.ones(V, bool) if allow is None else allow[m]
        y[m, ~ok] = -np.inf
        may = ok & ~np.isnan(y[m])
        ids.append(-1 if not may.any() else int(np.flatnonzero(may & (y[m] == y[m][may].max()))[0]))
    return np.array(ids, np.int32), y


def pack(lists):
    return ints([v for row in lists for v in row]), ints(starts_of([len(r) for r in lists]))


def mask_words(allow, V):
    bits = np.zeros((allow.shape[0], (V + 31) // 32 * 32), np.uint64)
    bits[:, :V] = allow
    w = (bits.reshape(allow.shape[0], -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
    return torch.from_numpy(w.view(np.int32)).to(DEV)


def run_pick(x, hist=None, rep=None, pres=None, freq=None, bias=None, allow=None, in_place=False, want_out=True):
    M, V = x.shape
    kw = {}
    if hist is not None:
        kw["history"], kw["history_starts"] = pack(hist)
        kw.update(repetition=T(rep), presence=T(pres), frequency=T(freq))
    if bias is not None:
        kw["bias_ids"], kw["bias_starts"] = pack([[t for t, _ in r] for r in bias])
        kw["bias_values"] = T(np.array([b for r in bias for _, b in r], np.float32))
    if allow is not None:
        kw["allow_mask"] = mask_words(allow, V)
    flag, ids, logits = ints([0]), ints([-7] * M), T(x)
    out = logits if in_place else torch.empty_like(logits) if want_out else None
    K.logits_pick(ids, out, logits, M, V, bad_flag=flag, **kw)
    return H(ids), (H(out) if out is not None else None), int(H(flag)[0])


@pytest.mark.parametrize("M,V,n_hist,n_bias,masked", [
    (1, 151936, 120, 0, False), (3, 151936, 700, 30, True), (5, 1000, 50, 7, True), (2, 1, 3, 1, True),
    (4, 33, 10, 3, True), (9, 4099, 2000, 64, False), (65, 2048, 0, 0, True), (1, 70001, 1, 5, True),
    (2, 31, 0, 4, False),
    (70, 40000, 900, 9, True), (70, 40001, 600, 9, True),   # two CTAs a row, two tiles each
    (260, 21000, 40, 3, False),                              # one CTA a row, three tiles
    (2, 400000, 3000, 40, True), (1, 350001, 30, 0, False),  # more than 16 tiles: several per CTA
    (257, 20000, 14000, 6, False),                           # most of the vocabulary listed
    (300, 270000, 5, 3, False),                              # one CTA a row, 27 tiles
])
def test_pick(M, V, n_hist, n_bias, masked):
    rng = np.random.default_rng(M * V)
    x = (rng.standard_normal((M, V)) * 3).astype(np.float32)
    x[0, :min(V, 5)] = [0.0, -0.0, 0.0, np.float32(1e-42), -np.float32(1e-42)][:min(V, 5)]
    hist = [list(rng.integers(0, V, n_hist * (m + 1) // M)) for m in range(M)] if n_hist else None
    rep = (1 + rng.random(M)).astype(np.float32)
    pres, freq = rng.random(M).astype(np.float32), (rng.random(M) * 0.3).astype(np.float32)
    bias = [[(int(t), float(b)) for t, b in zip(rng.integers(0, V, n_bias), rng.normal(0, 4, n_bias))]
            for _ in range(M)] if n_bias else None  # small vocabularies repeat tokens
    allow = rng.random((M, V)) < rng.random((M, 1)) if masked else None
    ref_ids, ref = pick_ref(x, hist, rep, pres, freq, bias, allow)
    for kw in ({}, {"in_place": True}, {"want_out": False}):
        ids, out, flag = run_pick(x, hist, rep, pres, freq, bias, allow, **kw)
        assert flag == 0 and np.array_equal(ids, ref_ids), kw
        assert out is None or np.array_equal(out, ref)


def test_pick_ties_nan_and_infinities():
    x = np.zeros((9, 300), np.float32)
    x[0, [17, 200]] = 5                      # the first of equal ones
    x[1, 3], x[1, 250] = -0.0, 0.0           # all zeros: index 0
    x[2, :] = -np.inf                        # allowed, if hopeless: index 0
    x[3, :] = np.nan                         # nothing to pick
    x[4, :] = np.nan
    x[4, 99] = -np.inf                       # the only value
    x[5, 0], x[5, 7], x[5, 8] = np.nan, np.inf, np.inf
    x[6, 12] = 3.0                           # masked below
    x[7, :] = -1.0                           # nothing allowed below
    x[8, 299] = 1.0
    allow = np.ones((9, 300), bool)
    allow[6, 12] = False
    allow[7] = False
    ids, out, _ = run_pick(x, allow=allow)
    assert ids.tolist() == [17, 0, 0, -1, 99, 7, 0, -1, 299]
    ref = x.copy()
    ref[~allow] = -np.inf
    assert np.array_equal(out, ref, equal_nan=True)
    ids, _, _ = run_pick(x[:6])
    assert ids.tolist() == [17, 0, 0, -1, 99, 7]


def test_pick_bad_entries():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 500)).astype(np.float32)
    one, zero = np.ones(2, np.float32), np.zeros(2, np.float32)
    big = np.full(2, 2.0, np.float32)
    ids, out, flag = run_pick(x, [[3, 500, -1, 3], [4]], big, one, one, [[(-5, 9.0), (2, 1.0)], [(500, 3.0)]])
    ref_ids, ref = pick_ref(x, [[3, 500, -1, 3], [4]], big, one, one, [[(-5, 9.0), (2, 1.0)], [(500, 3.0)]], None)
    assert flag == 1 and np.array_equal(ids, ref_ids) and np.array_equal(out, ref)
    # starts that do not fit their list: that row goes without it
    logits, got, ids, flag = T(x), torch.empty(2, 500, device=DEV), ints([0, 0]), ints([0])
    K.logits_pick(ids, got, logits, 2, 500, history=ints([1, 2, 3]), history_starts=ints([0, 3, 9]),
                  repetition=T(big), presence=T(zero), frequency=T(zero), bad_flag=flag)
    ref_ids, ref = pick_ref(x, [[1, 2, 3], []], big, zero, zero, None, None)
    assert H(flag)[0] == 1 and np.array_equal(H(ids), ref_ids) and np.array_equal(H(got), ref)


def test_pick_penalties_default_to_nothing():
    x = np.random.default_rng(2).standard_normal((2, 640)).astype(np.float32)
    h, s = pack([[1, 2, 2], [5]])
    out = torch.empty(2, 640, device=DEV)
    K.logits_pick(None, out, T(x), 2, 640, history=h, history_starts=s)
    assert np.array_equal(H(out), x)
    K.logits_pick(None, out, T(x), 2, 640, history=h, history_starts=s, frequency=T(np.array([1, 2], np.float32)))
    x[0, 1] -= 1
    x[0, 2] -= 2
    x[1, 5] -= 2
    assert np.array_equal(H(out), x)


def test_pick_unaligned_rows_in_a_graph():
    """Logits that start off a 16-byte boundary, captured and replayed with the history changed in place."""
    rng = np.random.default_rng(3)
    buf = T(rng.standard_normal(2 * 1000 + 1).astype(np.float32))
    logits = buf[1:].view(2, 1000)
    hist, starts, rep = ints([1, 2, 3, 4]), ints([0, 2, 4]), T(np.array([1.5, 2.0], np.float32))
    ids, out = ints([0, 0]), torch.empty(2, 1000, device=DEV)
    kw = dict(history=hist, history_starts=starts, repetition=rep)
    K.logits_pick(ids, out, logits, 2, 1000, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.logits_pick(ids, out, logits, 2, 1000, **kw)
    top = logits.argmax(1).tolist()
    hist.copy_(ints([top[0], 8, top[1], top[1]]))
    g.replay()
    zero = np.zeros(2, np.float32)
    ref_ids, ref = pick_ref(H(logits), [[top[0], 8], [top[1], top[1]]], H(rep), zero, zero, None, None)
    assert np.array_equal(H(ids), ref_ids) and np.array_equal(H(out), ref)


# ---------------------------------------------------------- all of them --
def test_speculative_decoding_follows_greedy_decoding():
    """A small decoder layer stack over the INT8 cache: a prompt chunk, then drafted trees that are verified
    and committed (append + attention, picks under rules, accepted rows appended again) give the tokens that
    one-token steps give, and the cache ends with the same codes."""
    rng = np.random.default_rng(21)
    L, n_heads, n_kv, hd, vocab, hidden = 2, 4, 2, 128, 512, 256
    qd, kd = n_heads * hd, n_kv * hd
    eps = 1e-6

    def w8(n, k):
        q, s = synthetic.quantize_np((rng.standard_normal((n, k)) * 0.05).astype(np.float32))
        return T(q), T(s)

    layers = [dict(wq=w8(qd, hidden), wk=w8(kd, hidden), wv=w8(kd, hidden), wo=w8(hidden, qd)) for _ in range(L)]
    head, embed = w8(vocab, hidden), T(rng.standard_normal((vocab, hidden)).astype(np.float32))
    ones, qk = torch.ones(hidden, device=DEV), torch.ones(hd, device=DEV)

    def forward(cache, tokens, places, rows, mask):
        """Logits of packed tokens at rotary places; their K/V rows go to the cache.  Returns (logits, [k, v] per layer)."""
        n = len(tokens)
        x = torch.empty(n, hidden, device=DEV)
        K.embed_gather(x, embed, ints(tokens), n, hidden, vocab)
        cos, sin = torch.empty(n, hd, device=DEV), torch.empty(n, hd, device=DEV)
        K.compute_rope_neox(cos, sin, ints(places), n, hd, 1e6)
        kept = []
        for i, w in enumerate(layers):
            xn = torch.empty_like(x)
            K.rms_norm(xn, x, ones, n, hidden, eps)
            q, k, v = (torch.empty(n, d, device=DEV) for d in (qd, kd, kd))
            for r in range(n):  # row by row: the matvec path whatever the number of tokens
                for dst, name, d in ((q, "wq", qd), (k, "wk", kd), (v, "wv", kd)):
                    K.linear_nobias_int8(dst[r], xn[r], *w[name], 1, hidden, d)
            K.rms_norm_per_head(q, qk, n, n_heads, hd, eps)
            K.rms_norm_per_head(k, qk, n, n_kv, hd, eps)
            K.apply_rope_neox(q, cos, sin, n, n_heads, hd)
            K.apply_rope_neox(k, cos, sin, n, n_kv, hd)
            K.kv_append_int8(cache, i, rows, k, v)
            a = torch.empty(n, qd, device=DEV)
            K.tree_attention_int8(a, q, cache, i, rows, n_heads, 1 / math.sqrt(hd), mask)
            for r in range(n):
                K.int8_matvec_residual(x[r], a[r], *w["wo"], 1, qd, hidden)
            kept.append((k, v))
        logits = torch.empty(n, vocab, device=DEV)
        xn = torch.empty_like(x)
        K.rms_norm(xn, x, ones, n, hidden, eps)
        for r in range(n):
            K.linear_nobias_int8(logits[r], xn[r], *head, 1, hidden, vocab)
        return logits, kept

    def pick(logits, seen):
        n = logits.shape[0]
        ids = ints([0] * n)
        h, s = pack(seen)
        K.logits_pick(ids, None, logits, n, vocab, history=h, history_starts=s, repetition=T(np.full(n, 1.3, np.float32)))
        return H(ids).tolist()

    prompt, steps = [int(t) for t in rng.integers(0, vocab, 130)], 12

    def start():
        cache = KvCacheInt8.zeros(1, L, 200, n_kv, hd)
        n = len(prompt)
        logits, _ = forward(cache, prompt, range(n), KvRows(ints([0, n]), ints([0]), n_rows=n, max_rows=n), None)
        return cache, pick(logits[-1:], [prompt])

    # one token a step
    cache1, tokens = start()
    while len(tokens) < steps:
        p = len(prompt) + len(tokens) - 1
        logits, _ = forward(cache1, tokens[-1:], [p], KvRows(ints([0, 1]), ints([p]), n_rows=1, max_rows=1), None)
        tokens += pick(logits, [prompt + tokens])

    # trees: a root, the right continuation somewhere among wrong ones
    cache2, got = start()
    assert got == tokens[:1]
    while len(got) < steps:
        p, at = len(prompt) + len(got) - 1, len(got) - 1
        right = tokens[at + 1:at + 3]
        wrong = [(t + 1) % vocab for t in right]
        #        0 root, 1 wrong, 2 right, 3 below wrong, 4 below right (wrong), 5 below right (right)
        draft = [got[-1], wrong[0] if wrong else 0, right[0] if right else 1, 9, wrong[1] if len(wrong) > 1 else 2,
                 right[1] if len(right) > 1 else 3]
        parent = [-1, 0, 0, 1, 2, 2]
        up, depth = [], []
        for t, pa in enumerate(parent):
            up.append((up[pa] if t else 0) | 1 << t)
            depth.append(depth[pa] + 1 if t else 0)
        n = len(draft)
        logits, kept = forward(cache2, draft, [p + d for d in depth], KvRows(ints([0, n]), ints([p]), n_rows=n, max_rows=n),
                               as_int64(up))
        path_to = [[draft[j] for j in range(n) if up[t] >> j & 1] for t in range(n)]
        ids = pick(logits, [prompt + got[:-1] + path for path in path_to])
        node, path, new = 0, [0], [ids[0]]
        while True:
            nxt = [j for j in range(n) if parent[j] == node and draft[j] == ids[node]]
            if not nxt:
                break
            node = nxt[0]
            path.append(node)
            new.append(ids[node])
        m = len(path)
        rows = KvRows(ints([0, m]), ints([p]), n_rows=m, max_rows=m)
        for i, (k, v) in enumerate(kept):
            K.kv_append_int8(cache2, i, rows, k, v, ints(path))
        got += new
    assert got[:steps] == tokens
    # the caches agree: the same codes but where the two ways' roundings fall on either side of a half
    n = len(prompt) + steps - 1
    for a, b, s in ((cache1.k, cache2.k, cache1.k_scales), (cache1.v, cache2.v, cache1.v_scales)):
        d = (a[0, :, :n].short() - b[0, :, :n].short()).abs()
        assert int(d.max()) <= 1 and float((d > 0).float().mean()) < 1e-3
