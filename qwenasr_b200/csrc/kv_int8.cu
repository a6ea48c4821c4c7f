// kv_int8.cu -- writing and reading back the INT8 KV cache.
//
// A head row x (64 or 128 values) is stored as codes round(x * (127 / a)), a =
// max|x|, halves away from zero, and the scale a / 127: the rule of
// qasr_quantize_f32_to_int8 (crates/qwen-asr/src/quantize.rs:633-662) applied
// per head, in the same f32 steps, so the codes are bit-identical to it.
// Reading back is code * scale, one rounding.
#include "kv_int8.cuh"

namespace qasr {

int kv_int8_check(const char *fn, const qasr_kv_int8 *c, int layer, const qasr_kv_rows *r) {
  if (!c || !r || !c->k || !c->v || !c->k_scales || !c->v_scales) {
    set_error("%s: null cache or rows", fn);
    return QASR_ERR_INVALID;
  }
  if (c->n_slots <= 0 || c->n_layers <= 0 || c->max_seq <= 0 || c->n_kv_heads <= 0 || layer < 0 ||
      layer >= c->n_layers) {
    set_error("%s: bad cache shape (%d slots, %d layers, max_seq %d, %d kv heads) or layer %d", fn, c->n_slots,
              c->n_layers, c->max_seq, c->n_kv_heads, layer);
    return QASR_ERR_INVALID;
  }
  if (c->head_dim != 64 && c->head_dim != 128) {
    set_error("%s: head_dim %d unsupported (64 or 128)", fn, c->head_dim);
    return QASR_ERR_UNSUPPORTED;
  }
  if (c->n_kv_heads > 256) {
    set_error("%s: %d kv heads unsupported (at most 256)", fn, c->n_kv_heads);
    return QASR_ERR_UNSUPPORTED;
  }
  // cache rows are addressed by 32-bit tile coordinates
  if ((double)c->n_slots * c->n_layers * c->max_seq > 2147483000.0) {
    set_error("%s: more than 2^31 cache rows (%d x %d x %d)", fn, c->n_slots, c->n_layers, c->max_seq);
    return QASR_ERR_UNSUPPORTED;
  }
  if ((reinterpret_cast<uintptr_t>(c->k) & 15) || (reinterpret_cast<uintptr_t>(c->v) & 15) ||
      (reinterpret_cast<uintptr_t>(c->k_scales) & 3) || (reinterpret_cast<uintptr_t>(c->v_scales) & 3)) {
    set_error("%s: cache codes must be 16-byte aligned, scales 4-byte aligned", fn);
    return QASR_ERR_INVALID;
  }
  if ((double)r->n_rows * c->n_kv_heads > 2147483000.0) {  // warps of an append or read are numbered in 32 bits
    set_error("%s: too many rows (%d of %d heads)", fn, r->n_rows, c->n_kv_heads);
    return QASR_ERR_UNSUPPORTED;
  }
  if (r->n_seqs < 0 || r->n_rows < 0 || r->max_rows < 0 || (r->n_seqs && (!r->row_starts || !r->positions))) {
    set_error("%s: bad rows (%d sequences, %d rows, at most %d each) or null row_starts / positions", fn, r->n_seqs,
              r->n_rows, r->max_rows);
    return QASR_ERR_INVALID;
  }
  return QASR_OK;
}

// Four values times inv = 127 / a, rounded halves away from zero, as bytes.
// Adding 1/2 and then 2^23, both toward zero, leaves the rounded magnitude in
// the low bits: no sum here is pushed up to the next integer.  a * inv is at
// most 127 and two roundings, so 127 needs no clamp.
QASR_DEV uint32_t codes4(float4 x, float inv) {
  const float v[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = __fmul_rn(v[i], inv);
    const int m = __float_as_int(__fadd_rz(__fadd_rz(fabsf(t), 0.5f), 8388608.0f)) & 0xff;
    const int sign = __float_as_int(t) >> 31;
    c[i] = (uint32_t)((m ^ sign) - sign);
  }
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// The sources are plain pointers, here and in attention: what the kernel before writes, while this one's blocks are
// resident already, must not go the way of read-only data.
// Columns of a cache row go in pieces of 128 (one or two heads).  A warp takes
// `per` pieces of one row, K and V; kPieces of each are in flight together.
constexpr int kKvThreads = 128, kKvWarps = kKvThreads / 32;  // 32,640 rows: 58 us, 60 with 256 threads, 68 with 512
template <int HD, int kPieces>
__global__ void __launch_bounds__(kKvThreads)
kv_append_int8_kernel(const qasr_kv_int8 c, int layer, const qasr_kv_rows r, const float *k_new, const float *v_new,
                      const int32_t *src_rows, int n_src, int pieces, int per) {
  constexpr int LPH = HD / 4, HPP = 128 / HD;  // lanes per head, heads per piece
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * kKvWarps + (threadIdx.x >> 5), groups = (unsigned)(pieces + per - 1) / per;
  pdl_wait();  // first: what starts as a dependent of this kernel finds all kernels before it done
  pdl_launch_dependents();
  if (item == 0) kv_flag_bad(r, c, lane);
  const unsigned row = item / groups;
  if (row >= (unsigned)r.n_rows) return;
  // The source row does not wait for the look-up of its place: both round trips run side by side.
  const int src = src_rows ? src_rows[row] : (int)row;
  const bool have = src >= 0 && src < n_src;
  const size_t kv_dim = (size_t)c.n_kv_heads * HD;
  const int p0 = (int)(item % groups) * per, p1 = min(p0 + per, pieces);
  float4 x[kPieces][2];
  auto load = [&](int p) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const size_t col = (size_t)(p + i) * 128 + 4 * lane;
      const bool in = have && p + i < p1 && col < kv_dim;  // an odd number of 64-wide heads ends in half a piece
      x[i][0] = in ? *reinterpret_cast<const float4 *>(k_new + src * kv_dim + col) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[i][1] = in ? *reinterpret_cast<const float4 *>(v_new + src * kv_dim + col) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  load(p0);
  const KvPlace at = kv_place(r, c, (int)row, lane);
  if (!at.ok) return;
  if (!have) {
    if (lane == 0 && r.bad_flag) atomicMax(r.bad_flag, 1);
    return;
  }
  const size_t cr = kv_row(c, at.slot, layer, at.pos);
  for (int p = p0; p < p1; p += kPieces) {
    if (p > p0) load(p);
    // Largest magnitudes, as bits (ordered like the values, NaN above infinity).  Lane e keeps those of head e of
    // the warp's (piece, K or V, head of the piece): both divisions run once for all of them.
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 2 * kPieces * HPP; ++e) {
      constexpr uint32_t kAbs = 0x7fffffffu;
      const float4 v = x[e / HPP / 2][e / HPP % 2];
      const uint32_t b = max(max(__float_as_uint(v.x) & kAbs, __float_as_uint(v.y) & kAbs),
                             max(__float_as_uint(v.z) & kAbs, __float_as_uint(v.w) & kAbs));
      const uint32_t t = __reduce_max_sync(0xffffffffu, HPP == 1 || lane / LPH == e % HPP ? b : 0u);
      if (lane == e) top = t;
    }
    const bool odd = top >= 0x7f800000u, tiny = top < 0x04000000u;  // no number; below 2^-119
    const float a = __uint_as_float(odd || tiny ? 0x3f800000u : top);
    const float inv = odd || tiny ? 0.0f : __fdiv_rn(127.0f, a);
    const float scale = odd ? __uint_as_float(0x7fc00000u) : tiny ? 0.0f : __fdiv_rn(a, 127.0f);
    const int piece = p + lane / (2 * HPP), head = piece * HPP + lane % HPP;
    if (lane < 2 * kPieces * HPP && piece < p1 && head < c.n_kv_heads)
      (lane / HPP % 2 ? c.v_scales : c.k_scales)[cr * c.n_kv_heads + head] = scale;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const size_t col = (size_t)(p + i) * 128 + 4 * lane;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const float f = __shfl_sync(0xffffffffu, inv, (2 * i + kv) * HPP + (HPP == 1 ? 0 : lane / LPH));
        const uint32_t w = f == 0.0f ? 0u : codes4(x[i][kv], f);
        if (p + i < p1 && col < kv_dim) *reinterpret_cast<uint32_t *>((kv ? c.v : c.k) + cr * kv_dim + col) = w;
      }
    }
  }
}

QASR_DEV float4 dequantize4(uint32_t w, float s) {
  float f[4];
  i8x4_to_f32(w, f);
  return make_float4(__fmul_rn(f[0], s), __fmul_rn(f[1], s), __fmul_rn(f[2], s), __fmul_rn(f[3], s));
}

// A long call writes four bytes for each that it reads: evict-first, so that
// the codes stay in L2 (3232 rows 9.0 -> 7.6 us).
template <bool LONG>
QASR_DEV void put4(float *to, float4 v) {
  if constexpr (LONG)
    __stcs(reinterpret_cast<float4 *>(to), v);
  else
    *reinterpret_cast<float4 *>(to) = v;
}

// As the append: one warp per `per` pieces of a row.
template <int HD, int kPieces>
__global__ void __launch_bounds__(kKvThreads)
kv_read_int8_kernel(float *__restrict__ k_out, float *__restrict__ v_out, const qasr_kv_int8 c, int layer,
                    const qasr_kv_rows r, int pieces, int per) {
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * kKvWarps + (threadIdx.x >> 5), groups = (unsigned)(pieces + per - 1) / per;
  pdl_wait();
  pdl_launch_dependents();
  if (item == 0) kv_flag_bad(r, c, lane);
  const unsigned row = item / groups;
  if (row >= (unsigned)r.n_rows) return;
  const KvPlace at = kv_place(r, c, (int)row, lane);
  if (!at.ok) return;
  const size_t kv_dim = (size_t)c.n_kv_heads * HD, cr = kv_row(c, at.slot, layer, at.pos);
  const int p0 = (int)(item % groups) * per, p1 = min(p0 + per, pieces);
  for (int p = p0; p < p1; p += kPieces) {
    uint32_t w[2][kPieces];
    float s[2][kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const size_t col = (size_t)(p + i) * 128 + 4 * lane, head = cr * c.n_kv_heads + col / HD;
      const bool in = p + i < p1 && col < kv_dim;
      w[0][i] = in && k_out ? *reinterpret_cast<const uint32_t *>(c.k + cr * kv_dim + col) : 0u;
      w[1][i] = in && v_out ? *reinterpret_cast<const uint32_t *>(c.v + cr * kv_dim + col) : 0u;
      s[0][i] = in && k_out ? c.k_scales[head] : 0.0f;
      s[1][i] = in && v_out ? c.v_scales[head] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const size_t col = (size_t)(p + i) * 128 + 4 * lane;
      if (p + i >= p1 || col >= kv_dim) break;
      if (k_out) put4<(kPieces > 1)>(k_out + row * kv_dim + col, dequantize4(w[0][i], s[0][i]));
      if (v_out) put4<(kPieces > 1)>(v_out + row * kv_dim + col, dequantize4(w[1][i], s[1][i]));
    }
  }
}

}  // namespace qasr

using namespace qasr;
static inline cudaStream_t S(void *s) { return reinterpret_cast<cudaStream_t>(s); }
static inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kDeep = 4;

// Small calls are bound by latency: one piece a warp (64 pieces, append and
// read-back 3.9 us against 5.1 with four; 4408 pieces read in 3.1 against 3.5).
// From 8192 pieces on four, which quarters the look-ups and keeps 2 to 4 KB per
// warp in flight (25,856 pieces, both calls, 17.3 against 22.0 us; 261,120 read
// in 58 against 80 us, 5.8 TB/s; two or eight a warp 62 and 66 us).
struct KvLaunch {
  int pieces, per;
  unsigned grid;
  bool deep;
  KvLaunch(const qasr_kv_int8 &c, const qasr_kv_rows &r) {
    pieces = ceil_div(c.n_kv_heads, 128 / c.head_dim);
    deep = (long)r.n_rows * pieces >= 8192;
    per = deep ? kDeep : 1;
    grid = (unsigned)ceil_div((long)r.n_rows * ceil_div(pieces, per), kKvWarps);
  }
};

extern "C" int qasr_kv_append_int8(const qasr_kv_int8 *cache, int layer, const qasr_kv_rows *rows, const float *k_new,
                                   const float *v_new, const int32_t *src_rows, int n_src, void *stream) {
  if (int rc = kv_int8_check("qasr_kv_append_int8", cache, layer, rows)) return rc;
  if (rows->n_seqs == 0 || rows->n_rows == 0) return QASR_OK;  // empty operands have no address
  if (!k_new || !v_new || !al16(k_new) || !al16(v_new) || n_src < 0 || (!src_rows && n_src < rows->n_rows)) {
    set_error("qasr_kv_append_int8: k_new and v_new must be 16-byte aligned and hold n_rows = %d rows (n_src = %d) "
              "unless src_rows picks them", rows->n_rows, n_src);
    return QASR_ERR_INVALID;
  }
  const KvLaunch l(*cache, *rows);
  const auto kernel = cache->head_dim == 128
                          ? (l.deep ? kv_append_int8_kernel<128, kDeep> : kv_append_int8_kernel<128, 1>)
                          : (l.deep ? kv_append_int8_kernel<64, kDeep> : kv_append_int8_kernel<64, 1>);
  const cudaError_t e = launch_pdl(kernel, l.grid, kKvThreads, 0, S(stream), *cache, layer, *rows, k_new, v_new, src_rows, n_src,
                                   l.pieces, l.per);
  return cuda_status(e, "qasr_kv_append_int8");
}

extern "C" int qasr_kv_read_int8(float *k_out, float *v_out, const qasr_kv_int8 *cache, int layer,
                                 const qasr_kv_rows *rows, void *stream) {
  if (int rc = kv_int8_check("qasr_kv_read_int8", cache, layer, rows)) return rc;
  if (rows->n_seqs == 0 || rows->n_rows == 0) return QASR_OK;
  if ((!k_out && !v_out) || !al16(k_out) || !al16(v_out)) {
    set_error("qasr_kv_read_int8: k_out or v_out must be given, 16-byte aligned");
    return QASR_ERR_INVALID;
  }
  const KvLaunch l(*cache, *rows);
  const auto kernel = cache->head_dim == 128 ? (l.deep ? kv_read_int8_kernel<128, kDeep> : kv_read_int8_kernel<128, 1>)
                                             : (l.deep ? kv_read_int8_kernel<64, kDeep> : kv_read_int8_kernel<64, 1>);
  const cudaError_t e =
      launch_pdl(kernel, l.grid, kKvThreads, 0, S(stream), k_out, v_out, *cache, layer, *rows, l.pieces, l.per);
  return cuda_status(e, "qasr_kv_read_int8");
}
