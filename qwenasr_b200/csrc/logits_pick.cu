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
constexpr int kPickTile = 4096;  // tokens per pass: their counts and bias entries stand in shared memory
constexpr int kPickCluster = 16;

struct PickParams {
  int32_t *ids;
  float *out;         // may equal `in`
  const float *in;
  qasr_pick_rules r;
  int vocab, chunk;   // tokens per CTA of the row's cluster, a multiple of 32
  bool vec;           // rows start on 16-byte boundaries
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

// One cluster per row; each CTA takes `chunk` tokens in tiles of kPickTile.
// The row's lists are few against its tokens: every CTA reads them once per
// tile and keeps what falls into the tile, counts by integer atomics (no
// order), the bias as the largest list index (the last entry for a token).
__global__ void __launch_bounds__(kPickThreads) logits_pick_kernel(const PickParams p) {
  __shared__ __align__(16) uint32_t s_count[kPickTile], s_bias[kPickTile];
  __shared__ unsigned long long s_warp[kPickThreads / 32], s_rank[kPickCluster];
  pdl_launch_dependents();
  pdl_wait();
  cluster_arrive_all();  // every CTA of the cluster has started before one writes to another
  const int rank = (int)cluster_ctarank(), m = blockIdx.y, V = p.vocab;
  const qasr_pick_rules &r = p.r;
  int h0 = 0, h1 = 0, b0 = 0, b1 = 0;
  if (r.history) pick_list(r.history_starts, r.n_history, m, r.bad_flag, h0, h1);
  if (r.bias_ids) pick_list(r.bias_starts, r.n_bias, m, r.bad_flag, b0, b1);
  const bool touched = h1 > h0 || b1 > b0;
  const float rep = r.repetition ? r.repetition[m] : 1.0f, pres = r.presence ? r.presence[m] : 0.0f,
              freq = r.frequency ? r.frequency[m] : 0.0f;
  const float *x = p.in + (size_t)m * V;
  float *y = p.out ? p.out + (size_t)m * V : nullptr;
  const uint32_t *mask = r.allow_mask ? r.allow_mask + (size_t)m * ((V + 31) / 32) : nullptr;
  const int c0 = (int)min((long)rank * p.chunk, (long)V), c1 = (int)min((long)c0 + p.chunk, (long)V);
  unsigned long long best = 0;  // 0: nothing yet (every key of a value is larger)

  auto value = [&](float l, int t, int t0) {
    if (touched) {
      if (const uint32_t n = s_count[t - t0]) {
        l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
        l = __fsub_rn(l, __fadd_rn(pres, __fmul_rn(freq, (float)n)));
      }
      if (const uint32_t e = s_bias[t - t0]) l = __fadd_rn(l, r.bias_values[b0 + e - 1]);
    }
    return l;
  };
  auto take = [&](float l, int t, bool allowed) {
    // -0 + 0 = +0: the two zeros are one value
    if (allowed && l == l) best = max(best, argmax_key(__fadd_rn(l, 0.0f), (uint32_t)t));
  };

  for (int t0 = c0; t0 < c1; t0 += kPickTile) {
    const int t1 = min(t0 + kPickTile, c1);
    if (touched) {
      __syncthreads();  // the previous tile's tables are read
      for (int i = threadIdx.x; i < kPickTile; i += kPickThreads) s_count[i] = s_bias[i] = 0;
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
    if (p.vec) {
      for (int t = t0 + 4 * threadIdx.x; t < t1; t += 4 * kPickThreads) {
        float4 l = *reinterpret_cast<const float4 *>(x + t);
        const uint32_t ok = mask ? mask[t >> 5] >> (t & 31) : 15u;
        float *e = &l.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = value(e[i], t + i, t0);
          if (!(ok >> i & 1)) e[i] = -INFINITY;
          take(e[i], t + i, ok >> i & 1);
        }
        if (y) *reinterpret_cast<float4 *>(y + t) = l;
      }
    } else {
      for (int t = t0 + threadIdx.x; t < t1; t += kPickThreads) {
        const bool ok = !mask || (mask[t >> 5] >> (t & 31) & 1);
        const float l = ok ? value(x[t], t, t0) : -INFINITY;
        take(l, t, ok);
        if (y) y[t] = l;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = best;
  __syncthreads();
  cluster_wait_all();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPickThreads / 32; ++w) best = max(best, s_warp[w]);
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_map(smem_u32(&s_rank[rank]), 0)), "l"(best)
                 : "memory");
  }
  cluster_sync_all();
  if (rank == 0 && threadIdx.x == 0 && p.ids) {
    best = 0;
    for (int c = 0; c < (int)gridDim.x; ++c) best = max(best, s_rank[c]);
    p.ids[m] = best ? (int32_t)(0xffffffffu - (uint32_t)best) : -1;
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
  PickParams p{ids, logits_out, logits, r, vocab, 0, false};
  p.chunk = ceil_div(ceil_div(vocab, kPickCluster), 32) * 32;
  p.vec = vocab % 4 == 0 && !((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(logits_out)) & 15);
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return QASR_ERR_INVALID;
  if (!attr_done[dev]) {
    if (int rc = cuda_status(cudaFuncSetAttribute(logits_pick_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                             "qasr_logits_pick: cluster size opt-in"))
      return rc;
    attr_done[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kPickCluster, (unsigned)M);
  cfg.blockDim = dim3(kPickThreads);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kPickCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, logits_pick_kernel, p), "qasr_logits_pick");
}
