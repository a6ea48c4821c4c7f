"""Refusals of the serving operators (INT8 KV cache, attention over it, token
picks) that need no GPU: every bad argument gives a status and a message
before anything is launched, and the Python face raises on bad tensors."""
import ctypes as C

import pytest
import torch

from qwenasr_b200 import _lib
from qwenasr_b200.kvcache import KvCacheInt8, KvRows

P = C.c_void_p(256)  # an aligned address that is never dereferenced
ODD = C.c_void_p(264)


@pytest.fixture(scope="module")
def lib():
    from qwenasr_b200 import build
    build.build()
    return _lib.load()


def cache(**kw):
    d = dict(k=256, v=256, k_scales=256, v_scales=256, n_slots=2, n_layers=3, max_seq=64, n_kv_heads=8, head_dim=128)
    d.update(kw)
    return C.byref(_lib.KvInt8(*d.values()))


def rows(**kw):
    d = dict(row_starts=256, positions=256, slots=None, n_seqs=2, n_rows=4, max_rows=2, max_keys=0, bad_flag=None)
    d.update(kw)
    return C.byref(_lib.KvRows(*d.values()))


BAD_CACHE = [
    (dict(k=None), _lib.QASR_ERR_INVALID), (dict(v_scales=None), _lib.QASR_ERR_INVALID),
    (dict(k=264), _lib.QASR_ERR_INVALID), (dict(v=257), _lib.QASR_ERR_INVALID),
    (dict(k_scales=258), _lib.QASR_ERR_INVALID), (dict(n_slots=0), _lib.QASR_ERR_INVALID),
    (dict(max_seq=-1), _lib.QASR_ERR_INVALID), (dict(n_kv_heads=0), _lib.QASR_ERR_INVALID),
    (dict(n_layers=1), _lib.QASR_ERR_INVALID),  # layer 1 does not exist
    (dict(head_dim=96), _lib.QASR_ERR_UNSUPPORTED), (dict(n_kv_heads=257), _lib.QASR_ERR_UNSUPPORTED),
    (dict(n_slots=1 << 16, max_seq=1 << 16), _lib.QASR_ERR_UNSUPPORTED),
]
BAD_ROWS = [dict(row_starts=None), dict(positions=None), dict(n_seqs=-1), dict(n_rows=-1), dict(max_rows=-2)]


def calls(lib, c, r):
    yield "qasr_kv_append_int8", lib.qasr_kv_append_int8(c, 1, r, P, P, None, 4, None)
    yield "qasr_kv_read_int8", lib.qasr_kv_read_int8(P, P, c, 1, r, None)
    yield "qasr_tree_attention_int8", lib.qasr_tree_attention_int8(P, C.c_void_p(512), c, 1, r, None, 16, 0.1, None)


@pytest.mark.parametrize("kw,code", BAD_CACHE)
def test_bad_cache(lib, kw, code):
    for name, rc in calls(lib, cache(**kw), rows()):
        assert rc == code, name
        assert name in _lib.last_error()


@pytest.mark.parametrize("kw", BAD_ROWS)
def test_bad_rows(lib, kw):
    for name, rc in calls(lib, cache(), rows(**kw)):
        assert rc == _lib.QASR_ERR_INVALID, name
        assert name in _lib.last_error()


def test_too_many_rows(lib):
    for name, rc in calls(lib, cache(), rows(n_rows=1 << 29)):
        assert rc == _lib.QASR_ERR_UNSUPPORTED, name


@pytest.mark.parametrize("layer", [-1, 3])
def test_bad_layer(lib, layer):
    assert lib.qasr_kv_append_int8(cache(), layer, rows(), P, P, None, 4, None) == _lib.QASR_ERR_INVALID
    assert "layer" in _lib.last_error()


def test_null_structs(lib):
    assert lib.qasr_kv_append_int8(None, 0, rows(), P, P, None, 4, None) == _lib.QASR_ERR_INVALID
    assert lib.qasr_kv_read_int8(P, P, cache(), 0, None, None) == _lib.QASR_ERR_INVALID
    assert lib.qasr_logits_pick(P, None, P, None, 1, 100, None) == _lib.QASR_ERR_INVALID


def test_append_and_read_refusals(lib):
    bad = _lib.QASR_ERR_INVALID
    assert lib.qasr_kv_append_int8(cache(), 0, rows(), None, P, None, 4, None) == bad
    assert lib.qasr_kv_append_int8(cache(), 0, rows(), P, ODD, None, 4, None) == bad
    assert lib.qasr_kv_append_int8(cache(), 0, rows(), P, P, None, 3, None) == bad  # fewer source rows than rows
    assert "n_src = 3" in _lib.last_error()
    assert lib.qasr_kv_read_int8(None, None, cache(), 0, rows(), None) == bad
    assert lib.qasr_kv_read_int8(ODD, P, cache(), 0, rows(), None) == bad


def test_attention_refusals(lib):
    def attend(out=P, q=C.c_void_p(512), r=None, mask=None, heads=16):
        return lib.qasr_tree_attention_int8(out, q, cache(), 0, r or rows(), mask, heads, 0.1, None)

    assert attend(out=None) == _lib.QASR_ERR_INVALID
    assert attend(q=P) == _lib.QASR_ERR_INVALID  # in place
    assert attend(out=ODD) == _lib.QASR_ERR_INVALID
    assert attend(mask=C.c_void_p(260)) == _lib.QASR_ERR_INVALID
    assert attend(heads=12) == _lib.QASR_ERR_INVALID
    assert attend(heads=0) == _lib.QASR_ERR_INVALID
    assert attend(heads=8 * 65) == _lib.QASR_ERR_UNSUPPORTED
    assert attend(r=rows(max_rows=65), mask=P) == _lib.QASR_ERR_UNSUPPORTED
    assert "64 rows" in _lib.last_error()
    assert attend(r=rows(n_seqs=70000)) == _lib.QASR_ERR_UNSUPPORTED
    assert attend(r=rows(max_rows=1 << 30, n_rows=1 << 27)) == _lib.QASR_ERR_UNSUPPORTED
    assert "query rows" in _lib.last_error()


def test_pick_refusals(lib):
    def pick(ids=P, out=None, logits=P, M=2, vocab=100, **kw):
        return lib.qasr_logits_pick(ids, out, logits, C.byref(_lib.PickRules(**kw)), M, vocab, None)

    bad = _lib.QASR_ERR_INVALID
    assert pick(ids=None) == bad
    assert pick(logits=None) == bad
    assert pick(M=-1) == bad
    assert pick(vocab=0) == bad
    assert pick(history=256, n_history=3) == bad  # no starts
    assert pick(history=256, history_starts=256, n_history=-1) == bad
    assert pick(bias_ids=256, bias_starts=256, n_bias=2) == bad  # no values
    assert pick(repetition=256) == bad  # penalties without a history
    assert pick(M=70000) == _lib.QASR_ERR_UNSUPPORTED
    assert pick(vocab=(1 << 30) + 1) == _lib.QASR_ERR_UNSUPPORTED
    assert "qasr_logits_pick" in _lib.last_error()


def test_nothing_to_do_launches_nothing(lib):
    """Empty batches return before any device work (there is no device here)."""
    for r in (rows(n_seqs=0, row_starts=None, positions=None), rows(n_rows=0)):
        for name, rc in calls(lib, cache(), r):
            assert rc == _lib.QASR_OK, name
    assert lib.qasr_tree_attention_int8(P, C.c_void_p(512), cache(), 1, rows(max_rows=0), None, 16, 0.1, None) == 0
    assert lib.qasr_logits_pick(P, None, P, C.byref(_lib.PickRules()), 0, 100, None) == _lib.QASR_OK


def test_python_faces_refuse_host_tensors():
    c8, f = torch.zeros(1, 1, 4, 128, dtype=torch.int8), torch.zeros(1, 1, 4, 1)
    with pytest.raises(ValueError, match="CUDA"):
        KvCacheInt8(c8, c8, f, f)
    with pytest.raises(ValueError, match="CUDA"):
        KvRows(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), n_rows=1, max_rows=1)
    from qwenasr_b200 import kernels as K
    with pytest.raises(ValueError, match="CUDA"):
        K.logits_pick(None, None, torch.zeros(1, 8), 1, 8)


def test_empty_operands_have_no_address(lib):
    """What an empty tensor hands over, a null pointer, is no error in an empty call."""
    for r in (rows(n_seqs=0, row_starts=None, positions=None), rows(n_rows=0)):
        assert lib.qasr_kv_append_int8(cache(), 1, r, None, None, None, 0, None) == _lib.QASR_OK
        assert lib.qasr_kv_read_int8(None, None, cache(), 1, r, None) == _lib.QASR_OK
        assert lib.qasr_tree_attention_int8(None, None, cache(), 1, r, None, 16, 0.1, None) == _lib.QASR_OK
    rules = _lib.PickRules(history_starts=256, repetition=256, bias_starts=256)
    assert lib.qasr_logits_pick(None, None, None, C.byref(rules), 0, 100, None) == _lib.QASR_OK


def test_penalties_of_an_empty_history_pass_the_checks(lib):
    """They get as far as the limit of rows, as those of any history do."""
    def pick(**kw):
        return lib.qasr_logits_pick(P, None, P, C.byref(_lib.PickRules(**kw)), 70000, 100, None)

    assert pick(history_starts=256, repetition=256, presence=256, frequency=256) == _lib.QASR_ERR_UNSUPPORTED
    assert pick(bias_starts=256) == _lib.QASR_ERR_UNSUPPORTED
    assert pick(history_starts=256, n_history=2, repetition=256) == _lib.QASR_ERR_INVALID  # entries without a list
    assert pick(repetition=256) == _lib.QASR_ERR_INVALID
