"""The serving operators at their edges: scales that are no numbers, empty batches and lists, the variant of long calls,
starts in disorder, rows written just before, penalties over two histories."""
import numpy as np
import pytest
import torch

from test_gpu_serving import (Cache, DEV, H, KvCacheInt8, KvRows, T, as_int64, attend_exact, ints, mask_words, pack,
                              pick_ref, quantize, starts_of)

from qwenasr_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    from qwenasr_b200 import build
    build.build()
    assert torch.cuda.is_available()


# ----------------------------------------------------------- key scales --
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hd", [64, 128])
def test_key_scale_that_is_no_number(bad, hd):
    """It makes NaN of the rows that see it, whatever the sign of q k, and of no other."""
    rng = np.random.default_rng(hd)
    n, p, n_kv, at = 4, 130, 3, 132                     # token 2's own row, seen by tokens 2 and 3
    c = Cache(rng, 1, 1, 200, n_kv, hd)
    c.fill(rng, 0, 0, p + n)
    c.k[0, 0, at] = 1
    masks = [0b1, 0b11, 0b100, 0b1100]
    q = rng.standard_normal((n, 2 * n_kv * hd)).astype(np.float32)
    q = np.abs(q) * np.where(np.arange(2 * n_kv) % 2, -1, 1).repeat(hd).astype(np.float32)  # both signs in each group
    ref, bar = attend_exact(c, 0, q, [n], [p], [0], masks, 2 * n_kv, 0.1)
    c.ks[0, 0, at, 1] = bad                             # one kv head: query heads 2 and 3
    out = torch.empty(n, 2 * n_kv * hd, device=DEV)
    rows = KvRows(ints([0, n]), ints([p]), n_rows=n, max_rows=n)
    K.tree_attention_int8(out, T(q), c.up(), 0, rows, 2 * n_kv, 0.1, as_int64(masks))
    got, ref = H(out).reshape(n, 2 * n_kv, hd), ref.reshape(n, 2 * n_kv, hd)
    hit = np.zeros((n, 2 * n_kv), bool)
    hit[2:, 2:4] = True
    assert np.isnan(got[hit]).all()
    assert (np.abs(got - ref) <= bar[:, :, None])[~hit].all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_the_only_key_has_no_number_for_a_scale(bad):
    cache = KvCacheInt8.zeros(1, 1, 8, 1, 128)
    cache.k.fill_(1)
    cache.v.fill_(1)
    cache.v_scales.fill_(1)
    cache.k_scales.fill_(bad)
    q = torch.ones(2, 128, device=DEV)
    q[1] = -1
    out = torch.zeros(1, 256, device=DEV)
    K.tree_attention_int8(out, q.view(1, 256), cache, 0, KvRows(ints([0, 1]), ints([0]), n_rows=1, max_rows=1), 2, 0.1)
    assert np.isnan(H(out)).all()


# ---------------------------------------------------------------- empty --
def test_empty_batches():
    """No rows at all: empty tensors, which have no address, are as good as any."""
    cache = KvCacheInt8.zeros(1, 1, 8, 2, 64)
    none = torch.empty(0, 128, device=DEV)
    for starts in ([0], [0, 0, 0]):
        rows = KvRows(ints(starts), ints([0] * (len(starts) - 1)), n_rows=0, max_rows=0)
        K.kv_append_int8(cache, 0, rows, none, none)
        K.kv_append_int8(cache, 0, rows, none, none, ints([]))
        K.kv_read_int8(none, none, cache, 0, rows)
        K.kv_read_int8(None, none, cache, 0, rows)
        K.tree_attention_int8(none, torch.empty(0, 128, device=DEV), cache, 0, rows, 2, 0.1)
        K.tree_attention_int8(none, none, cache, 0, rows, 2, 0.1, torch.empty(0, dtype=torch.int64, device=DEV))
    K.logits_pick(ints([]), torch.empty(0, 50, device=DEV), torch.empty(0, 50, device=DEV), 0, 50)
    K.logits_pick(ints([]), None, torch.empty(0, 50, device=DEV), 0, 50, history=ints([]), history_starts=ints([0]),
                  repetition=torch.empty(0, device=DEV))
    assert not H(cache.k).any() and not H(cache.k_scales).any()


def test_no_history_yet():
    """A batch's first picks: no token has appeared, the penalties apply to nothing; no biases either."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 700)).astype(np.float32)
    two, one = T(np.full(3, 2, np.float32)), T(np.ones(3, np.float32))
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    for kw in (dict(repetition=two), dict(repetition=two, presence=one, frequency=one), {},
               dict(bias_ids=none, bias_values=torch.empty(0, device=DEV), bias_starts=ints([0, 0, 0, 0]))):
        ids, out, flag = ints([-7] * 3), torch.empty(3, 700, device=DEV), ints([0])
        K.logits_pick(ids, out, T(x), 3, 700, history=none, history_starts=ints([0, 0, 0, 0]), bad_flag=flag, **kw)
        assert np.array_equal(H(ids), x.argmax(1)) and np.array_equal(H(out), x) and H(flag)[0] == 0
    # starts beyond the empty list are flagged, as with any other list
    K.logits_pick(ids, out, T(x), 3, 700, history=none, history_starts=ints([0, 0, 1, 1]), repetition=two, bad_flag=flag)
    assert np.array_equal(H(ids), x.argmax(1)) and np.array_equal(H(out), x) and H(flag)[0] == 1
    # one row of three has a history
    hist, starts = pack([[], [5, 6, 5], []])
    K.logits_pick(ids, out, T(x), 3, 700, history=hist, history_starts=starts, repetition=two, presence=one, frequency=one)
    f = np.float32
    ref_ids, ref = pick_ref(x, [[], [5, 6, 5], []], np.full(3, 2, f), np.ones(3, f), np.ones(3, f), None, None)
    assert np.array_equal(H(ids), ref_ids) and np.array_equal(H(out), ref)


# ---------------------------------------------------- long calls, bit by bit --
def pieces(n_kv, hd):
    return -(-n_kv * hd // 128)


@pytest.mark.parametrize("n_kv,hd", [(5, 128), (8, 128), (9, 64), (11, 64), (1, 128), (7, 64)])
@pytest.mark.parametrize("beyond", [-1, 0, 1, 700])  # rows around the one where calls go four pieces a warp
@pytest.mark.parametrize("gather", [False, True])
def test_long_calls(n_kv, hd, beyond, gather):
    rng = np.random.default_rng(n_kv * hd + beyond + 1)
    total, pad, d = -(-8192 // pieces(n_kv, hd)) + beyond, 3, n_kv * hd
    counts = [total // 3, 0, total - total // 3 - 5, 5]
    max_seq, layer = max(counts) + 9, 1
    cache = KvCacheInt8.zeros(4, 2, max_seq, n_kv, hd)
    n_src = total + (50 if gather else pad)
    k, v = ((rng.standard_normal((n_src, d)) * np.exp(rng.normal(0, 2, (n_src, 1)))).astype(np.float32) for _ in range(2))
    src = rng.permutation(n_src)[:total] if gather else np.arange(total)
    k[src[7], :hd] = np.nan                              # a head without a scale; the row's others keep theirs
    k[src[8]], v[src[8], -hd:] = 0, 0
    slots, positions = [2, 0, 3, 1], [1, 4, 9, 0]
    rows = KvRows(ints(starts_of(counts)), ints(positions), ints(slots), n_rows=total + pad, max_rows=max(counts),
                  bad_flag=(flag := ints([0])))
    K.kv_append_int8(cache, layer, rows, T(k), T(v), ints(list(src) + [10 ** 9] * pad) if gather else None)
    back = [torch.full((total + pad, d), 7.0, device=DEV) for _ in range(4)]
    K.kv_read_int8(back[0], back[1], cache, layer, rows)
    K.kv_read_int8(back[2], None, cache, layer, rows)
    K.kv_read_int8(None, back[3], cache, layer, rows)
    assert H(flag)[0] == 0
    for x, code, scale, outs in ((k, cache.k, cache.k_scales, back[::2]), (v, cache.v, cache.v_scales, back[1::2])):
        lost = np.isnan(x[src])
        q, s = quantize(np.where(lost, 0, x[src]), hd)
        s[lost.reshape(total, n_kv, hd).any(2)] = np.nan
        want_c, want_s = np.zeros(code.shape, np.int8), np.zeros(scale.shape, np.float32)
        for i, (n, p, sl) in enumerate(zip(counts, positions, slots)):
            r0 = starts_of(counts)[i]
            want_c[sl, layer, p:p + n], want_s[sl, layer, p:p + n] = q[r0:r0 + n], s[r0:r0 + n]
        assert np.array_equal(H(code), want_c) and np.array_equal(H(scale), want_s, equal_nan=True)
        ref = (q.reshape(total, n_kv, hd).astype(np.float32) * s[..., None]).reshape(total, d)
        for o in outs:
            assert np.array_equal(H(o)[:total], ref, equal_nan=True) and (H(o)[total:] == 7).all()


# ------------------------------------------------------------- disorder --
@pytest.mark.parametrize("starts,positions,fits", [
    ([0, 50, 2, 4], [3, 0, 5], [2]),                     # a start outside leaves out the two sequences that it bounds
    ([0, 2147483647, 2, 4, 6], [3, 0, 5, 1], [2, 3]),
    ([0, 2, -9, 2, 4], [3, 0, 0, 5], [0, 3]),
    ([0] + [2 * i + 2 for i in range(40)] + [200, 82, 84], [1] * 43, [*range(40), 42]),  # over a second ballot's lanes
])
def test_a_bad_start_leaves_the_others_in(starts, positions, fits):
    """Every operator takes the same sequences: append and read-back write what attention attends for."""
    rng = np.random.default_rng(len(starts))
    n, n_rows, d = len(starts) - 1, max(s for s in starts if s < 100) + 2, 128
    c = Cache(rng, n, 1, 16, 1, d)
    for sl in range(n):
        c.fill(rng, sl, 0, 16)
    dev, flag = c.up(), ints([0])
    rows = KvRows(ints(starts), ints(positions), None, n_rows=n_rows, max_rows=4, bad_flag=flag)
    mine = np.zeros(n_rows, bool)
    for m in fits:
        mine[starts[m]:starts[m + 1]] = True
    x = rng.standard_normal((n_rows, d)).astype(np.float32)
    K.kv_append_int8(dev, 0, rows, T(x), T(x))
    assert H(flag)[0] == 1
    want = c.k.copy()
    for m in fits:
        r = starts[m + 1] - starts[m]
        want[m, 0, positions[m]:positions[m] + r] = quantize(x[starts[m]:starts[m + 1]], d)[0]
    assert np.array_equal(H(dev.k), want)
    outs = [torch.full((n_rows, d), 9.0, device=DEV) for _ in range(2)]
    K.kv_read_int8(outs[0], None, dev, 0, rows)
    K.tree_attention_int8(outs[1], T(x), dev, 0, rows, 1, 0.1)
    for o in outs:
        assert np.array_equal((H(o) != 9).any(1), mine)


# ---------------------------------------------------------------- order --
def test_rows_written_just_before():
    """Steps back to back, on two streams over one cache: each append's rows and scales, neighbours of those that the
    attention before has read, are what the next attention sees (as with a wait after every call)."""
    steps, d = 150, 128
    rng = np.random.default_rng(3)
    new = T(rng.standard_normal((2, steps, 3, 1, d)).astype(np.float32))
    outs = []
    for wait in (True, False):
        cache, streams = KvCacheInt8.zeros(2, 1, 400, 1, d), [torch.cuda.Stream() for _ in range(2)]
        out, pos = torch.zeros(2, steps, 1, d, device=DEV), [ints([0]) for _ in range(2)]
        k, v = torch.empty(2, 1, d, device=DEV), torch.empty(2, 1, d, device=DEV)
        rows = [KvRows(ints([0, 1]), pos[i], ints([i]), n_rows=1, max_rows=1, max_keys=400) for i in range(2)]
        torch.cuda.synchronize()
        for t in range(steps):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    pos[i].fill_(t)
                    k[i].copy_(new[i, t, 0])
                    v[i].copy_(new[i, t, 1])
                    K.kv_append_int8(cache, 0, rows[i], k[i], v[i])
                    if wait:
                        torch.cuda.synchronize()
                    K.tree_attention_int8(out[i, t], new[i, t, 2], cache, 0, rows[i], 1, 0.1)
                    if wait:
                        torch.cuda.synchronize()
        torch.cuda.synchronize()
        outs.append(H(out))
    assert np.array_equal(outs[0], outs[1]) and (outs[0] != 0).any(-1).all()


# --------------------------------------------------------- two histories --
def test_penalties_over_two_histories():
    """Repetition over prompt and output, presence and frequency over the output alone: two calls, the second in
    place, give what the rule says for both lists."""
    rng = np.random.default_rng(4)
    M, V = 3, 900
    x = (rng.standard_normal((M, V)) * 3).astype(np.float32)
    prompt = [list(rng.integers(0, V, 60)) for _ in range(M)]
    output = [[], list(rng.integers(0, V, 5)), list(rng.integers(0, 9, 40))]
    rep, pres, freq = (rng.random(M).astype(np.float32) + b for b in (np.float32(1), np.float32(0), np.float32(0)))
    one, zero = np.ones(M, np.float32), np.zeros(M, np.float32)
    allow = rng.random((M, V)) < 0.7
    _, mid = pick_ref(x, [p + o for p, o in zip(prompt, output)], rep, zero, zero, None, None)
    ref_ids, ref = pick_ref(mid, output, one, pres, freq, None, allow)
    ids, out = ints([-7] * M), torch.empty(M, V, device=DEV)
    h, s = pack([p + o for p, o in zip(prompt, output)])
    K.logits_pick(None, out, T(x), M, V, history=h, history_starts=s, repetition=T(rep))
    h, s = pack(output)
    K.logits_pick(ids, out, out, M, V, history=h, history_starts=s, presence=T(pres), frequency=T(freq),
                  allow_mask=mask_words(allow, V))
    assert np.array_equal(H(ids), ref_ids) and np.array_equal(H(out), ref)
