"""The serving operators at their edges: scales that are no numbers, empty batches and lists."""
import numpy as np
import pytest
import torch

from test_gpu_serving import (Cache, DEV, H, KvCacheInt8, KvRows, T, as_int64, attend_exact, ints, pack, pick_ref)

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
