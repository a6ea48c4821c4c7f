// kv_int8.cuh -- the INT8 KV cache as the kernels see it: argument checks on
// the host, sequence lookups on the device.
#pragma once
#include "common.cuh"

namespace qasr {

// Returns QASR_OK or an error with a message naming `fn`.
int kv_int8_check(const char *fn, const qasr_kv_int8 *c, int layer, const qasr_kv_rows *r);

// One sequence of a call, its entries checked: packed rows row0 .. row0+n-1 at
// cache rows pos .. of `slot`.  n = 0 for a sequence that does not fit.
struct KvSeq {
  int row0, n, pos, slot;
  bool ok;
};

QASR_DEV KvSeq kv_seq(const qasr_kv_rows &r, const qasr_kv_int8 &c, int m) {
  KvSeq s;
  s.row0 = r.row_starts[m];
  const int end = r.row_starts[m + 1];
  s.pos = r.positions[m];
  s.slot = r.slots ? r.slots[m] : m;
  // in 64 bits: the entries may be anything
  const long long n = (long long)end - s.row0;
  s.ok = s.row0 >= 0 && n >= 0 && end <= r.n_rows && n <= r.max_rows && s.pos >= 0 && s.pos + n <= c.max_seq &&
         s.slot >= 0 && s.slot < c.n_slots;
  s.n = s.ok ? (int)n : 0;
  if (!s.ok) s.row0 = s.pos = s.slot = 0;
  return s;
}

// Whole warp: the sequence that owns packed row `row`, or -1.  Counts the
// starts at or below the row, 32 at a time; entries in disorder give a
// sequence that does not hold the row, which kv_seq's caller checks.
QASR_DEV int kv_seq_of_row(const qasr_kv_rows &r, int row, int lane) {
  int m = -1;
  for (int base = 0; base < r.n_seqs; base += 32) {
    const int i = base + lane;
    m += __popc(__ballot_sync(0xffffffffu, i < r.n_seqs && r.row_starts[i] <= row));
  }
  return m;
}

// One warp of a launch: every sequence's entries, *bad_flag if one does not fit.
QASR_DEV void kv_flag_bad(const qasr_kv_rows &r, const qasr_kv_int8 &c, int lane) {
  if (!r.bad_flag) return;
  for (int m = lane; m < r.n_seqs; m += 32)
    if (!kv_seq(r, c, m).ok) atomicMax(r.bad_flag, 1);
}

// Row (slot, layer, pos) of the cache, as an index of n_kv_heads scales.
QASR_DEV size_t kv_row(const qasr_kv_int8 &c, int slot, int layer, int pos) {
  return ((size_t)slot * c.n_layers + layer) * c.max_seq + pos;
}

}  // namespace qasr
