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

// The raw entries of sequence m, checked.
QASR_DEV KvSeq kv_seq_checked(const qasr_kv_rows &r, const qasr_kv_int8 &c, int start, int end, int pos, int slot) {
  KvSeq s{start, 0, pos, slot, false};
  const long long n = (long long)end - start;  // in 64 bits: the entries may be anything
  s.ok = start >= 0 && n >= 0 && end <= r.n_rows && n <= r.max_rows && pos >= 0 && pos + n <= c.max_seq && slot >= 0 &&
         slot < c.n_slots;
  if (s.ok)
    s.n = (int)n;
  else
    s.row0 = s.pos = s.slot = 0;
  return s;
}

QASR_DEV KvSeq kv_seq(const qasr_kv_rows &r, const qasr_kv_int8 &c, int m) {
  return kv_seq_checked(r, c, r.row_starts[m], r.row_starts[m + 1], r.positions[m], r.slots ? r.slots[m] : m);
}

// Whole warp: where packed row `row` stands in the cache; ok = false for a row
// behind the last sequence or of one that does not fit.  Each lane takes the
// entries of one sequence, checks them and sees whether they hold the row, so
// that a bad start leaves out the sequences that it bounds and no others, as in
// attention.  (Of sequences that overlap, which no good starts do, the first.)
struct KvPlace {
  bool ok;
  int slot, pos;
};
QASR_DEV KvPlace kv_place(const qasr_kv_rows &r, const qasr_kv_int8 &c, int row, int lane) {
  for (int base = 0; base < r.n_seqs; base += 32) {
    const int i = base + lane;
    const bool in = i < r.n_seqs;
    const int start = in ? r.row_starts[i] : 0, end = in ? r.row_starts[i + 1] : 0, pos = in ? r.positions[i] : 0;
    const int slot = in && r.slots ? r.slots[i] : i;
    const KvSeq s = kv_seq_checked(r, c, start, end, pos, slot);  // not in: without rows
    const uint32_t hit = __ballot_sync(0xffffffffu, row >= s.row0 && row - s.row0 < s.n);
    if (hit) {
      const int own = __ffs(hit) - 1;
      return KvPlace{true, __shfl_sync(0xffffffffu, s.slot, own),
                     __shfl_sync(0xffffffffu, s.pos - s.row0, own) + row};
    }
  }
  return KvPlace{false, 0, 0};
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
