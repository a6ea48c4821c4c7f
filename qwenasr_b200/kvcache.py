"""The INT8 KV cache and the rows of a call: what the serving operators of
qwenasr_b200.kernels (kv_append_int8, kv_read_int8, tree_attention_int8) work
on.  Host objects only: they check shapes once and hold the C structs, so that
a step over many layers pays for neither again.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib


def _tensor(t, dtype, device, name, numel=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA tensor of {dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if numel is not None and t.numel() < numel:
        raise ValueError(f"{name} has {t.numel()} elements, needs {numel}")
    return t


class KvCacheInt8:
    """Codes k, v int8 [n_slots, n_layers, max_seq, n_kv_heads * head_dim] and
    scales f32 [n_slots, n_layers, max_seq, n_kv_heads] (qasr_kv_int8): the
    one-byte counterpart of KvCache (crates/qwen-asr/src/decoder.rs:130-202).
    The tensors are the caller's and stay alive with this object."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        _tensor(k, torch.int8, None, "k")
        self.device = k.device
        _tensor(v, torch.int8, self.device, "v")
        _tensor(k_scales, torch.float32, self.device, "k_scales")
        _tensor(v_scales, torch.float32, self.device, "v_scales")
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"k and v must be [slots, layers, max_seq, kv_dim] alike, got {tuple(k.shape)}, "
                             f"{tuple(v.shape)}")
        n_kv = k_scales.shape[-1] if k_scales.dim() == 4 else 0
        if k_scales.shape != v_scales.shape or k_scales.shape[:-1] != k.shape[:-1] or not n_kv or k.shape[3] % n_kv:
            raise ValueError(f"scales must be [slots, layers, max_seq, n_kv_heads] of the codes, got "
                             f"{tuple(k_scales.shape)}, {tuple(v_scales.shape)}")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.n_slots, self.n_layers, self.max_seq, self.kv_dim = k.shape
        self.n_kv_heads, self.head_dim = n_kv, self.kv_dim // n_kv
        self.c = _lib.KvInt8(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), self.n_slots,
                             self.n_layers, self.max_seq, n_kv, self.head_dim)
        self.ref, self.dev = C.byref(self.c), k.get_device()

    @classmethod
    def zeros(cls, n_slots: int, n_layers: int, max_seq: int, n_kv_heads: int, head_dim: int, device="cuda:0"):
        shape = (n_slots, n_layers, max_seq)
        codes = [torch.zeros(*shape, n_kv_heads * head_dim, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(*shape, n_kv_heads, device=device) for _ in range(2)]
        return cls(*codes, *scales)


class KvRows:
    """The packed rows of a call (qasr_kv_rows): sequence m owns rows
    row_starts[m] .. row_starts[m+1]-1, which stand at cache rows positions[m] ..
    of slot slots[m] (slots None: slot m).  int32 device tensors, read when the
    kernels run: they may be changed in place between calls or graph replays.
    n_rows: rows of the packed buffers; max_rows: a bound on one sequence's
    rows; max_keys: a bound on one sequence's cache rows, by which attention
    splits its work (0: the cache's max_seq; results agree to rounding); bad_flag: int32 [1], set when a
    sequence does not fit."""

    def __init__(self, row_starts: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor | None = None, *,
                 n_rows: int, max_rows: int, max_keys: int = 0, bad_flag: torch.Tensor | None = None):
        n = row_starts.numel() - 1 if isinstance(row_starts, torch.Tensor) else -1
        if n < 0:
            raise ValueError("row_starts must be a tensor of n_seqs + 1 entries")
        _tensor(row_starts, torch.int32, None, "row_starts")
        self.device = row_starts.device
        _tensor(positions, torch.int32, self.device, "positions", n)
        if slots is not None:
            _tensor(slots, torch.int32, self.device, "slots", n)
        if bad_flag is not None:
            _tensor(bad_flag, torch.int32, self.device, "bad_flag", 1)
        self.row_starts, self.positions, self.slots, self.bad_flag = row_starts, positions, slots, bad_flag
        self.n_seqs, self.n_rows, self.max_rows, self.max_keys = n, int(n_rows), int(max_rows), int(max_keys)
        self.c = _lib.KvRows(row_starts.data_ptr(), positions.data_ptr(), None if slots is None else slots.data_ptr(),
                             n, self.n_rows, self.max_rows, self.max_keys, None if bad_flag is None else bad_flag.data_ptr())
        self.ref, self.dev = C.byref(self.c), row_starts.get_device()
