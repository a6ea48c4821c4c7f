// logits_pick.cu -- token picks under rules: penalties for tokens that
// appeared, additive biases, a mask of allowed tokens, first-max argmax.
//
// Per row and token with value l and c occurrences in the row's history:
//   c > 0: l > 0 ? l / repetition : l * repetition, minus (presence + frequency * c)
//   then plus its bias, then -inf unless allowed;
// the pick is the lowest index of the largest allowed value (strict '>', the
// rule of crates/qwen-asr/src/decoder.rs:942-947), NaN aside.
#include "common.cuh"
#include "tcgen05.cuh"

namespace qasr {

constexpr int kPickThreads = 512;
constexpr int kPickQuads = 5;  // 4-token groups a thread holds of a tile, all in flight before the lists are read
constexpr int kPickTile = kPickThreads * kPickQuads * 4;  // 10,240 tokens: a 16th of the published vocabulary fits
constexpr int kPickCluster = 16;

struct PickParams {
  int32_t *ids;
  float *out;         // may equal `in`
  const float *in;
  qasr_pick_rules r;
  int vocab, chunk;   // tokens per CTA of the row's cluster, a multiple of 32
  int table;          // tokens of a table in shared memory: min(chunk, kPickTile), a multiple of 32
};

// The entries of row m of a packed list; an empty range where they do not fit.
QASR_DEV void pick_list(const int32_t *starts, int n, int m, int32_t *bad, int &a, int &b) {
  a = starts[m];
  b = starts[m + 1];
  if (a < 0 || b < a || b > n) {
    if (bad) atomicMax(bad, 1);
    a = b = 0;
  }
}

// One cluster per row; each CTA takes `chunk` tokens in tiles of kPickTile
// (one, up to 163,840 tokens).  HBM-bound by design: a thread's logits and mask
// bits of the tile are requested first, and while they are on their way the
// row's lists, few against its tokens, are read by every CTA, which keeps what
// falls into its tile: counts by integer atomics (no order), the bias as the
// largest list index (the last entry for a token).  A thread touches the tables
// and its running maximum once per four tokens; tokens with an entry are rare.
// VEC: rows start on 16-byte boundaries; a quad is four neighbours, loaded as
// one.  Otherwise its elements lie kPickThreads apart, each load coalesced.
template <bool VEC>
__global__ void __launch_bounds__(kPickThreads, 2) logits_pick_kernel(const PickParams p) {
  extern __shared__ __align__(16) uint32_t s_table[];  // counts, then bias entries (index + 1)
  __shared__ unsigned long long s_warp[kPickThreads / 32], s_rank[kPickCluster];
  pdl_launch_dependents();
  pdl_wait();
  cluster_arrive_all();  // every CTA of the cluster has started before one writes to another
  const int rank = (int)cluster_ctarank(), m = blockIdx.y, V = p.vocab;
  const qasr_pick_rules &r = p.r;
  const float *x = p.in + (size_t)m * V;
  float *y = p.out ? p.out + (size_t)m * V : nullptr;
  const uint32_t *mask = r.allow_mask ? r.allow_mask + (size_t)m * ((V + 31) / 32) : nullptr;
  const int c0 = (int)min((long)rank * p.chunk, (long)V), c1 = (int)min((long)c0 + p.chunk, (long)V);
  uint32_t *s_count = s_table, *s_bias = s_table + (r.history ? p.table : 0);
  int h0 = 0, h1 = 0, b0 = 0, b1 = 0;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  float best = -INFINITY;
  int at = -1, any = -1;  // the best value's token; the first allowed number, should all be -infinity

  for (int t0 = c0; t0 < c1; t0 += kPickTile) {
    const int t1 = min(t0 + kPickTile, c1);
    auto token = [&](int k, int e) {
      return VEC ? t0 + (k * kPickThreads + (int)threadIdx.x) * 4 + e
                 : t0 + (k * 4 + e) * kPickThreads + (int)threadIdx.x;
    };
    float v[kPickQuads][4];
    uint32_t ok[kPickQuads];
#pragma unroll
    for (int k = 0; k < kPickQuads; ++k) {
      if constexpr (VEC) {
        const int t = token(k, 0);
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        ok[k] = 0;
        if (t < t1) {  // a row is a multiple of four: the whole quad is in
          q = *reinterpret_cast<const float4 *>(x + t);
          ok[k] = mask ? mask[t >> 5] : ~0u;
        }
        v[k][0] = q.x, v[k][1] = q.y, v[k][2] = q.z, v[k][3] = q.w;
      } else {
        ok[k] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = token(k, e);
          v[k][e] = t < t1 ? x[t] : 0.0f;
          if (t < t1 && (!mask || (mask[t >> 5] >> (t & 31) & 1))) ok[k] |= 1u << e;
        }
      }
    }
    if (t0 == c0) {
      if (r.history) pick_list(r.history_starts, r.n_history, m, r.bad_flag, h0, h1);
      if (r.bias_ids) pick_list(r.bias_starts, r.n_bias, m, r.bad_flag, b0, b1);
      if (r.repetition) rep = r.repetition[m];
      if (r.presence) pres = r.presence[m];
      if (r.frequency) freq = r.frequency[m];
    }
    const bool counted = h1 > h0, biased = b1 > b0;
    if (counted || biased) {
      __syncthreads();  // the previous tile's tables are read
      const int words = (r.history ? p.table : 0) + (r.bias_ids ? p.table : 0);
      for (int i = 4 * threadIdx.x; i < words; i += 4 * kPickThreads)
        *reinterpret_cast<uint4 *>(s_table + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
      for (int i = h0 + threadIdx.x; i < h1; i += kPickThreads) {
        const int t = r.history[i];
        if (t >= t0 && t < t1) atomicAdd(&s_count[t - t0], 1u);
        if ((t < 0 || t >= V) && r.bad_flag) atomicMax(r.bad_flag, 1);
      }
      for (int i = b0 + threadIdx.x; i < b1; i += kPickThreads) {
        const int t = r.bias_ids[i];
        if (t >= t0 && t < t1) atomicMax(&s_bias[t - t0], (uint32_t)(i - b0 + 1));
        if ((t < 0 || t >= V) && r.bad_flag) atomicMax(r.bad_flag, 1);
      }
      __syncthreads();
    }
    auto entries = [&](const uint32_t *table, int k, uint32_t (&n)[4]) {  // of a quad; true if there are any
      if constexpr (VEC) {
        const int t = token(k, 0);
        const uint4 q = t < t1 ? *reinterpret_cast<const uint4 *>(table + (t - t0)) : make_uint4(0, 0, 0, 0);
        n[0] = q.x, n[1] = q.y, n[2] = q.z, n[3] = q.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) n[e] = token(k, e) < t1 ? table[token(k, e) - t0] : 0;
      }
      return (n[0] | n[1] | n[2] | n[3]) != 0;
    };
#pragma unroll
    for (int k = 0; k < kPickQuads; ++k) {
      const uint32_t bits = VEC ? ok[k] >> (token(k, 0) & 31) & 15u : ok[k];
      uint32_t n[4];
      if (counted && entries(s_count, k, n)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n[e]) {
            const float l = v[k][e] > 0.0f ? __fdiv_rn(v[k][e], rep) : __fmul_rn(v[k][e], rep);
            v[k][e] = __fsub_rn(l, __fadd_rn(pres, __fmul_rn(freq, (float)n[e])));
          }
      }
      if (biased && entries(s_bias, k, n)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n[e]) v[k][e] = __fadd_rn(v[k][e], r.bias_values[b0 + n[e] - 1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = bits >> e & 1 ? v[k][e] : -INFINITY;
      // fmaxf leaves NaN out
      if (fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3])) > best) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v[k][e] > best) best = v[k][e], at = token(k, e);
      }
      if (any < 0 && bits) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (any < 0 && (bits >> e & 1) && v[k][e] == v[k][e]) any = token(k, e);
      }
      if (y) {
        if constexpr (VEC) {
          if (token(k, 0) < t1)
            *reinterpret_cast<float4 *>(y + token(k, 0)) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (token(k, e) < t1) y[token(k, e)] = v[k][e];
        }
      }
    }
  }
  // one order for the CTA and the cluster: the larger value, then the lower token; 0 where there is none.
  // -0 + 0 = +0: the two zeros are one value.
  unsigned long long key = at >= 0    ? argmax_key(__fadd_rn(best, 0.0f), (uint32_t)at)
                           : any >= 0 ? argmax_key(-INFINITY, (uint32_t)any)
                                      : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = key;
  __syncthreads();
  cluster_wait_all();
  if (threadIdx.x < 32) {
    key = threadIdx.x < kPickThreads / 32 ? s_warp[threadIdx.x] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if (threadIdx.x == 0)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_map(smem_u32(&s_rank[rank]), 0)), "l"(key)
                   : "memory");
  }
  __syncwarp();
  cluster_sync_all();
  if (rank == 0 && threadIdx.x == 0 && p.ids) {
    key = 0;
    for (int c = 0; c < (int)gridDim.x; ++c) key = max(key, s_rank[c]);
    p.ids[m] = key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
  }
}

}  // namespace qasr

using namespace qasr;

extern "C" int qasr_logits_pick(int32_t *ids, float *logits_out, const float *logits, const qasr_pick_rules *rules,
                                int M, int vocab, void *stream) {
  if (!logits || (!ids && !logits_out) || !rules || M < 0 || vocab <= 0) {
    set_error("qasr_logits_pick: invalid arguments (null logits or rules, no output, M=%d, vocab=%d)", M, vocab);
    return QASR_ERR_INVALID;
  }
  const qasr_pick_rules &r = *rules;
  if ((r.history && (!r.history_starts || r.n_history < 0)) ||
      (r.bias_ids && (!r.bias_values || !r.bias_starts || r.n_bias < 0))) {
    set_error("qasr_logits_pick: history needs history_starts, bias_ids need bias_values and bias_starts");
    return QASR_ERR_INVALID;
  }
  if (!r.history && (r.repetition || r.presence || r.frequency)) {
    set_error("qasr_logits_pick: penalties need a history");
    return QASR_ERR_INVALID;
  }
  if (M > 65535 || vocab > (1 << 30)) {
    set_error("qasr_logits_pick: at most 65535 rows and 2^30 tokens (M=%d, vocab=%d)", M, vocab);
    return QASR_ERR_UNSUPPORTED;
  }
  if (M == 0) return QASR_OK;
  PickParams p{ids, logits_out, logits, r, vocab, 0, 0};
  p.chunk = ceil_div(ceil_div(vocab, kPickCluster), 32) * 32;
  p.table = p.chunk < kPickTile ? p.chunk : kPickTile;
  const size_t smem = (size_t)p.table * 4 * ((r.history ? 1 : 0) + (r.bias_ids ? 1 : 0));
  const bool vec = vocab % 4 == 0 && !((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(logits_out)) & 15);
  auto kernel = vec ? logits_pick_kernel<true> : logits_pick_kernel<false>;
  static bool attr_done[64][2] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return QASR_ERR_INVALID;
  if (!attr_done[dev][vec]) {
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                         "qasr_logits_pick: cluster size opt-in");
    if (!rc)
      rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickTile * 8),
                       "qasr_logits_pick: shared memory opt-in");
    if (rc) return rc;
    attr_done[dev][vec] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kPickCluster, (unsigned)M);
  cfg.blockDim = dim3(kPickThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kPickCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p), "qasr_logits_pick");
}
