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
  if (r->n_seqs < 0 || r->n_rows < 0 || r->max_rows < 0 || (r->n_seqs && (!r->row_starts || !r->positions))) {
    set_error("%s: bad rows (%d sequences, %d rows, at most %d each) or null row_starts / positions", fn, r->n_seqs,
              r->n_rows, r->max_rows);
    return QASR_ERR_INVALID;
  }
  return QASR_OK;
}

// Lanes per head: each lane holds four values.
template <int HD>
QASR_DEV uint32_t head_max(uint32_t bits) {
#pragma unroll
  for (int o = HD / 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  return bits;
}

// Four values of a head row -> their codes; *scale = the head's scale.
// Magnitudes are compared as their bits (ordered like the values, NaN above
// infinity), so one maximum finds both the scale and a NaN or infinity.
template <int HD>
QASR_DEV uint32_t quantize4(float4 x, float *scale) {
  constexpr uint32_t kAbs = 0x7fffffffu, kInf = 0x7f800000u, kTiny = 0x04000000u;  // 2^-119
  const uint32_t top = head_max<HD>(max(max(__float_as_uint(x.x) & kAbs, __float_as_uint(x.y) & kAbs),
                                        max(__float_as_uint(x.z) & kAbs, __float_as_uint(x.w) & kAbs)));
  const float a = __uint_as_float(top);
  if (top >= kInf || top < kTiny) {
    *scale = top >= kInf ? __uint_as_float(0x7fc00000u) : 0.0f;
    return 0u;
  }
  *scale = __fdiv_rn(a, 127.0f);
  const float inv = __fdiv_rn(127.0f, a);
  const float v[4] = {x.x, x.y, x.z, x.w};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = fminf(fmaxf(roundf(__fmul_rn(v[i], inv)), -128.0f), 127.0f);
    w |= ((uint32_t)(int)c & 0xffu) << (8 * i);
  }
  return w;
}

// One warp per (packed row, 128 / HD heads).
template <int HD>
__global__ void __launch_bounds__(256)
kv_append_int8_kernel(const qasr_kv_int8 c, int layer, const qasr_kv_rows r, const float *__restrict__ k_new,
                      const float *__restrict__ v_new, const int32_t *__restrict__ src_rows, int n_src) {
  constexpr int HPW = 128 / HD, LPH = HD / 4;
  const int lane = threadIdx.x & 31;
  const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int groups = (c.n_kv_heads + HPW - 1) / HPW;
  pdl_launch_dependents();
  pdl_wait();
  if (item == 0) kv_flag_bad(r, c, lane);
  if (item >= (long)r.n_rows * groups) return;
  const int row = (int)(item / groups), head = (int)(item % groups) * HPW + lane / LPH;
  const int m = kv_seq_of_row(r, row, lane);
  if (m < 0) return;
  const KvSeq s = kv_seq(r, c, m);
  if (row < s.row0 || row - s.row0 >= s.n) return;  // behind the last sequence, or a bad one
  const int src = src_rows ? src_rows[row] : row;
  if (src < 0 || src >= n_src) {
    if (lane == 0 && r.bad_flag) atomicMax(r.bad_flag, 1);
    return;
  }
  const bool live = head < c.n_kv_heads;  // an odd head count leaves half a warp idle
  const size_t kv_dim = (size_t)c.n_kv_heads * HD;
  const size_t at = (size_t)src * kv_dim + (size_t)head * HD + lane % LPH * 4;
  float4 kx = make_float4(0.f, 0.f, 0.f, 0.f), vx = kx;
  if (live) {
    kx = *reinterpret_cast<const float4 *>(k_new + at);
    vx = *reinterpret_cast<const float4 *>(v_new + at);
  }
  float ks, vs;
  const uint32_t kc = quantize4<HD>(kx, &ks), vc = quantize4<HD>(vx, &vs);
  if (!live) return;
  const size_t cr = kv_row(c, s.slot, layer, s.pos + (row - s.row0));
  const size_t dst = cr * kv_dim + (size_t)head * HD + lane % LPH * 4;
  *reinterpret_cast<uint32_t *>(c.k + dst) = kc;
  *reinterpret_cast<uint32_t *>(c.v + dst) = vc;
  if (lane % LPH == 0) {
    c.k_scales[cr * c.n_kv_heads + head] = ks;
    c.v_scales[cr * c.n_kv_heads + head] = vs;
  }
}

QASR_DEV float4 dequantize4(uint32_t w, float s) {
  float f[4];
  i8x4_to_f32(w, f);
  return make_float4(__fmul_rn(f[0], s), __fmul_rn(f[1], s), __fmul_rn(f[2], s), __fmul_rn(f[3], s));
}

// One warp per (packed row, 128 / HD heads), as the append.
template <int HD>
__global__ void __launch_bounds__(256)
kv_read_int8_kernel(float *__restrict__ k_out, float *__restrict__ v_out, const qasr_kv_int8 c, int layer,
                    const qasr_kv_rows r) {
  constexpr int HPW = 128 / HD, LPH = HD / 4;
  const int lane = threadIdx.x & 31;
  const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int groups = (c.n_kv_heads + HPW - 1) / HPW;
  pdl_launch_dependents();
  pdl_wait();
  if (item == 0) kv_flag_bad(r, c, lane);
  if (item >= (long)r.n_rows * groups) return;
  const int row = (int)(item / groups), head = (int)(item % groups) * HPW + lane / LPH;
  const int m = kv_seq_of_row(r, row, lane);
  if (m < 0) return;
  const KvSeq s = kv_seq(r, c, m);
  if (row < s.row0 || row - s.row0 >= s.n || head >= c.n_kv_heads) return;
  const size_t kv_dim = (size_t)c.n_kv_heads * HD, col = (size_t)head * HD + lane % LPH * 4;
  const size_t cr = kv_row(c, s.slot, layer, s.pos + (row - s.row0));
  if (k_out)
    *reinterpret_cast<float4 *>(k_out + row * kv_dim + col) =
        dequantize4(*reinterpret_cast<const uint32_t *>(c.k + cr * kv_dim + col), c.k_scales[cr * c.n_kv_heads + head]);
  if (v_out)
    *reinterpret_cast<float4 *>(v_out + row * kv_dim + col) =
        dequantize4(*reinterpret_cast<const uint32_t *>(c.v + cr * kv_dim + col), c.v_scales[cr * c.n_kv_heads + head]);
}

}  // namespace qasr

using namespace qasr;
static inline cudaStream_t S(void *s) { return reinterpret_cast<cudaStream_t>(s); }
static inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

extern "C" int qasr_kv_append_int8(const qasr_kv_int8 *cache, int layer, const qasr_kv_rows *rows, const float *k_new,
                                   const float *v_new, const int32_t *src_rows, int n_src, void *stream) {
  if (int rc = kv_int8_check("qasr_kv_append_int8", cache, layer, rows)) return rc;
  if (!k_new || !v_new || !al16(k_new) || !al16(v_new) || n_src < 0 || (!src_rows && n_src < rows->n_rows)) {
    set_error("qasr_kv_append_int8: k_new and v_new must be 16-byte aligned and hold n_rows = %d rows (n_src = %d) "
              "unless src_rows picks them", rows->n_rows, n_src);
    return QASR_ERR_INVALID;
  }
  if (rows->n_seqs == 0 || rows->n_rows == 0) return QASR_OK;
  const int hpw = 128 / cache->head_dim;
  const unsigned grid = (unsigned)ceil_div((long)rows->n_rows * ceil_div(cache->n_kv_heads, hpw), 8);
  cudaError_t e;
  if (cache->head_dim == 128)
    e = launch_pdl(kv_append_int8_kernel<128>, grid, 256, 0, S(stream), *cache, layer, *rows, k_new, v_new, src_rows, n_src);
  else
    e = launch_pdl(kv_append_int8_kernel<64>, grid, 256, 0, S(stream), *cache, layer, *rows, k_new, v_new, src_rows, n_src);
  return cuda_status(e, "qasr_kv_append_int8");
}

extern "C" int qasr_kv_read_int8(float *k_out, float *v_out, const qasr_kv_int8 *cache, int layer,
                                 const qasr_kv_rows *rows, void *stream) {
  if (int rc = kv_int8_check("qasr_kv_read_int8", cache, layer, rows)) return rc;
  if ((!k_out && !v_out) || !al16(k_out) || !al16(v_out)) {
    set_error("qasr_kv_read_int8: k_out or v_out must be given, 16-byte aligned");
    return QASR_ERR_INVALID;
  }
  if (rows->n_seqs == 0 || rows->n_rows == 0) return QASR_OK;
  const int hpw = 128 / cache->head_dim;
  const unsigned grid = (unsigned)ceil_div((long)rows->n_rows * ceil_div(cache->n_kv_heads, hpw), 8);
  cudaError_t e;
  if (cache->head_dim == 128)
    e = launch_pdl(kv_read_int8_kernel<128>, grid, 256, 0, S(stream), k_out, v_out, *cache, layer, *rows);
  else
    e = launch_pdl(kv_read_int8_kernel<64>, grid, 256, 0, S(stream), k_out, v_out, *cache, layer, *rows);
  return cuda_status(e, "qasr_kv_read_int8");
}
