// tree_attention.cu -- attention of one or several tokens per sequence over
// the INT8 KV cache: decode steps, drafted trees, prompt chunks.
//
// With codes c and scales s of a cache row j, query t of a head:
//   S_tj = scale * sum_d q_td kc_jd * ks_j
//   out_t = sum_j e^(S_tj - max_j S_tj) * vs_j * vc_j / sum_j e^(S_tj - max_j S_tj)
// over the rows j that t sees; nothing visible gives zero.
#include "kv_int8.cuh"

namespace qasr {

struct TreeAttnParams {
  float *out;
  const float *q;
  qasr_kv_int8 c;
  qasr_kv_rows r;
  const uint64_t *tree_mask;
  int layer, n_heads;
  float scale;
};

// Cache rows below the sequence's first token are past; row pos + j is token
// j's, visible by the mask or, without one, to the tokens from j on.
QASR_DEV bool tree_visible(int place, int t, int n, bool tree, uint64_t mask) {
  if (place < 0) return true;
  if (place >= n) return false;
  return tree ? (mask >> place & 1) != 0 : place <= t;
}

// One warp per (sequence, query head, token): 32 keys a round, one per lane
// for the scores, HD / 32 output values per lane.
template <int HD>
__global__ void __launch_bounds__(128) tree_attention_kernel(const TreeAttnParams p) {
  __shared__ __align__(16) float sq[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = blockIdx.z, h = blockIdx.y, t = blockIdx.x * 4 + warp;
  if (blockIdx.x == 0 && h == 0 && m == 0 && warp == 0) kv_flag_bad(p.r, p.c, lane);
  const KvSeq s = kv_seq(p.r, p.c, m);
  if (t >= s.n) return;
  const int kvh = h / (p.n_heads / p.c.n_kv_heads);
  const size_t row = s.row0 + t, kv_dim = (size_t)p.c.n_kv_heads * HD;
  const float *q = p.q + (row * p.n_heads + h) * HD;
  for (int d = lane; d < HD; d += 32) sq[warp][d] = q[d];
  __syncwarp();
  const uint64_t mask = p.tree_mask ? p.tree_mask[row] : 0;
  const size_t base = kv_row(p.c, s.slot, p.layer, 0);
  const int len = s.pos + s.n;
  float mx = -INFINITY, l = 0.0f, o[HD / 32] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    float sc = -INFINITY, vs = 0.0f;
    if (j < len && tree_visible(j - s.pos, t, s.n, p.tree_mask != nullptr, mask)) {
      const uint32_t *k = reinterpret_cast<const uint32_t *>(p.c.k + (base + j) * kv_dim + (size_t)kvh * HD);
      float a = 0.0f;
      for (int d = 0; d < HD / 4; ++d) {
        float f[4];
        i8x4_to_f32(k[d], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) a = fmaf(sq[warp][4 * d + e], f[e], a);
      }
      sc = a * p.c.k_scales[(base + j) * p.c.n_kv_heads + kvh] * p.scale;
      vs = p.c.v_scales[(base + j) * p.c.n_kv_heads + kvh];
    }
    const bool nan = __any_sync(0xffffffffu, sc != sc);
    const float mn = nan ? __uint_as_float(0x7fc00000u) : fmaxf(mx, warp_max(sc));
    if (mn == -INFINITY) continue;
    const float corr = mx == -INFINITY ? 0.0f : expf(mx - mn);
    const float pj = sc == -INFINITY ? 0.0f : expf(sc - mn);
    mx = mn;
    l = l * corr + warp_sum(pj);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) o[e] *= corr;
    const float w = sc == -INFINITY ? 0.0f : pj * vs;
    for (int i = 0; i < min(32, len - j0); ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const int8_t *v = p.c.v + (base + j0 + i) * kv_dim + (size_t)kvh * HD;
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) o[e] = fmaf(wi, (float)v[lane + 32 * e], o[e]);
    }
  }
  float *out = p.out + (row * p.n_heads + h) * HD;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) out[lane + 32 * e] = l == 0.0f ? 0.0f : o[e] / l;
}

}  // namespace qasr

using namespace qasr;

extern "C" int qasr_tree_attention_int8(float *out, const float *q, const qasr_kv_int8 *cache, int layer,
                                        const qasr_kv_rows *rows, const uint64_t *tree_mask, int n_heads, float scale,
                                        void *stream) {
  if (int rc = kv_int8_check("qasr_tree_attention_int8", cache, layer, rows)) return rc;
  if (!out || !q || out == q || (reinterpret_cast<uintptr_t>(out) & 15) || (reinterpret_cast<uintptr_t>(q) & 15) ||
      (reinterpret_cast<uintptr_t>(tree_mask) & 7)) {
    set_error("qasr_tree_attention_int8: q and out must be distinct and 16-byte aligned, tree_mask 8-byte aligned");
    return QASR_ERR_INVALID;
  }
  if (n_heads <= 0 || n_heads % cache->n_kv_heads) {
    set_error("qasr_tree_attention_int8: n_heads %d is not a multiple of %d kv heads", n_heads, cache->n_kv_heads);
    return QASR_ERR_INVALID;
  }
  if (n_heads / cache->n_kv_heads > 64) {
    set_error("qasr_tree_attention_int8: %d query heads per kv head unsupported (at most 64)",
              n_heads / cache->n_kv_heads);
    return QASR_ERR_UNSUPPORTED;
  }
  if (tree_mask && rows->max_rows > 64) {
    set_error("qasr_tree_attention_int8: a tree mask covers at most 64 rows per sequence (max_rows %d)",
              rows->max_rows);
    return QASR_ERR_UNSUPPORTED;
  }
  if (rows->n_seqs > 65535) {
    set_error("qasr_tree_attention_int8: at most 65535 sequences (%d)", rows->n_seqs);
    return QASR_ERR_UNSUPPORTED;
  }
  if (rows->n_seqs == 0 || rows->n_rows == 0 || rows->max_rows == 0) return QASR_OK;
  const TreeAttnParams p{out, q, *cache, *rows, tree_mask, layer, n_heads, scale};
  const dim3 grid((unsigned)ceil_div(rows->max_rows, 4), (unsigned)n_heads, (unsigned)rows->n_seqs);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (cache->head_dim == 128)
    tree_attention_kernel<128><<<grid, 128, 0, st>>>(p);
  else
    tree_attention_kernel<64><<<grid, 128, 0, st>>>(p);
  return launch_status("qasr_tree_attention_int8");
}
