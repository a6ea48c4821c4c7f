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
constexpr int kPickMaxCluster = 16;

struct PickParams {
  int32_t *ids;
  float *out;         // may equal `in`
  const float *in;
  qasr_pick_rules r;
  int vocab, chunk;   // tokens per CTA of the row's cluster, a multiple of 32
  int table;          // tokens of a table in shared memory: min(chunk, kPickTile), a multiple of 32
};

// A row's range of a packed list of n entries: empty, and flagged, if it does not fit.
QASR_DEV void pick_fit(int n, int &a, int &b, int32_t *bad) {
  if (a < 0 || b < a || b > n) {
    if (bad) atomicMax(bad, 1);
    a = b = 0;
  }
}

// One cluster per row; each CTA takes `chunk` tokens in tiles of kPickTile
// (one, for 16 CTAs and up to 163,840 tokens).  HBM-bound by design: a thread's
// logits and mask bits of the tile are requested first, and while they are on
// their way the row's lists, few against its tokens, are read by every CTA, which keeps what
// falls into its tile: a bit per token that has an entry at all, counts by integer
// atomics (no order), the bias as the largest list index (the last entry for a
// token).  The tables are cleared at the listed tokens only.  Tokens with an
// entry are rare: a thread looks at one word of bits per four tokens, and only
// maxima are kept on the way; the token is looked up by the few threads that
// hold the CTA's maximum.  Every CTA sends its best to rank 0 with a store that
// counts on a barrier there and leaves: nobody waits for its own output.
// Measured (B200, 151,936 tokens): one row with a history of 120 4.1 us (launch
// and two round trips), 8 rows 4.9, 64 rows with every rule 23.2 us, 3.4 TB/s
// (loads, instructions and stores of four tiles one after the other; 18 us
// without mask and bias).
// VEC: rows start on 16-byte boundaries; a quad is four neighbours, loaded as
// one.  Otherwise its elements lie kPickThreads apart, each load coalesced (no
// rules, 8 rows 3.9 and 4.5 us, 64 rows 14.6 and 16.4).
// MASK: the rules have a mask of allowed tokens.
template <bool VEC, bool MASK>
__global__ void __launch_bounds__(kPickThreads, 2) logits_pick_kernel(const PickParams p) {
  constexpr int T = kPickThreads, kWarps = T / 32;
  extern __shared__ __align__(16) uint32_t s_table[];  // counts, then bias entries (index + 1)
  __shared__ uint32_t s_bits[kPickTile / 32];          // tokens of the tile with an entry
  __shared__ unsigned long long s_warp[kWarps], s_rank[kPickMaxCluster];
  __shared__ uint64_t s_bar;
  __shared__ float s_top[kWarps];
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&s_bar, 1);
    mbar_fence_init();
    mbar_arrive_expect_tx(&s_bar, gridDim.x * 8);  // rank 0's: the keys of all ranks
  }
  for (int i = tid; i < kPickTile / 32; i += T) s_bits[i] = 0;
  __syncthreads();
  cluster_arrive_all();  // waited for before a key is sent: rank 0's barrier is ready
  pdl_wait();  // first: what starts as a dependent of this kernel finds all kernels before it done
  pdl_launch_dependents();
  const int rank = (int)cluster_ctarank(), m = blockIdx.y, V = p.vocab;
  const qasr_pick_rules &r = p.r;
  const float *x = p.in + (size_t)m * V;
  float *y = p.out ? p.out + (size_t)m * V : nullptr;
  const uint32_t *mask = MASK ? r.allow_mask + (size_t)m * ((V + 31) / 32) : nullptr;
  const int c0 = (int)min((long)rank * p.chunk, (long)V), c1 = (int)min((long)c0 + p.chunk, (long)V);
  uint32_t *s_count = s_table, *s_bias = s_table + (r.history ? p.table : 0);
  int h0 = 0, h1 = 0, b0 = 0, b1 = 0, first_h = 0, first_b = 0;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  // the best value, its token, and the first allowed number should all be -infinity (tokens are looked up late)
  float best = -INFINITY;
  int at = -1, any = -1;
  constexpr int kNone = 0x7fffffff;

  for (int t0 = c0; t0 < c1; t0 += kPickTile) {
    const int n = min(kPickTile, c1 - t0);  // tokens of the tile
    auto place = [&](int k, int e) { return VEC ? k * 4 * T + 4 * tid + e : (k * 4 + e) * T + tid; };
    float v[kPickQuads][4];
    uint32_t ok[kPickQuads];  // VEC: the mask word of the quad; else the quad's bits
#pragma unroll
    for (int k = 0; k < kPickQuads; ++k) {
      if constexpr (VEC) {  // rows, chunks and tiles are multiples of four: a quad is in or out
        float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        ok[k] = 0;
        if (place(k, 0) < n) {
          q = *reinterpret_cast<const float4 *>(x + t0 + place(k, 0));
          if (MASK) ok[k] = mask[(t0 >> 5) + (k * 4 * T >> 5) + (tid >> 3)];
        }
        v[k][0] = q.x, v[k][1] = q.y, v[k][2] = q.z, v[k][3] = q.w;
      } else {
        ok[k] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = place(k, e);
          v[k][e] = i < n ? x[t0 + i] : -INFINITY;
          if (MASK && i < n) ok[k] |= (mask[(t0 + i) >> 5] >> ((t0 + i) & 31) & 1) << e;
        }
      }
    }
    if (t0 == c0) {
      if (r.history) h0 = r.history_starts[m], h1 = r.history_starts[m + 1];
      if (r.bias_ids) b0 = r.bias_starts[m], b1 = r.bias_starts[m + 1];
      if (r.repetition) rep = r.repetition[m];
      if (r.presence) pres = r.presence[m];
      if (r.frequency) freq = r.frequency[m];
      pick_fit(r.n_history, h0, h1, r.bad_flag);
      pick_fit(r.n_bias, b0, b1, r.bad_flag);
      // the first entries of both lists, most often all of them: one round trip, kept for the later tiles
      if (h0 + tid < h1) first_h = r.history[h0 + tid];
      if (b0 + tid < b1) first_b = r.bias_ids[b0 + tid];
    }
    const bool listed = h1 > h0 || b1 > b0;
    if (listed) {
      auto each = [&](auto &&history, auto &&bias) {
        for (int i = h0 + tid; i < h1; i += T) history(i == h0 + tid ? first_h : r.history[i]);
        for (int i = b0 + tid; i < b1; i += T) bias(i == b0 + tid ? first_b : r.bias_ids[i], i - b0 + 1);
      };
      if (t0 > c0) {
        __syncthreads();  // the previous tile's bits are read
        for (int i = tid; i < kPickTile / 32; i += T) s_bits[i] = 0;
      }
      each(
          [&](int t) {
            if ((unsigned)(t - t0) < (unsigned)n) {
              s_count[t - t0] = 0;
              if (r.bias_ids) s_bias[t - t0] = 0;
            }
            if ((unsigned)t >= (unsigned)V && r.bad_flag) atomicMax(r.bad_flag, 1);
          },
          [&](int t, int) {
            if ((unsigned)(t - t0) < (unsigned)n) {
              if (r.history) s_count[t - t0] = 0;
              s_bias[t - t0] = 0;
            }
            if ((unsigned)t >= (unsigned)V && r.bad_flag) atomicMax(r.bad_flag, 1);
          });
      __syncthreads();
      each(
          [&](int t) {
            if ((unsigned)(t - t0) < (unsigned)n) {
              atomicAdd(&s_count[t - t0], 1u);
              atomicOr(&s_bits[(t - t0) >> 5], 1u << ((t - t0) & 31));
            }
          },
          [&](int t, int entry) {
            if ((unsigned)(t - t0) < (unsigned)n) {
              atomicMax(&s_bias[t - t0], (uint32_t)entry);
              atomicOr(&s_bits[(t - t0) >> 5], 1u << ((t - t0) & 31));
            }
          });
      __syncthreads();
    }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kPickQuads; ++k) {
      if (listed) {
        uint32_t hit = 0;
        if constexpr (VEC)
          hit = s_bits[(k * 4 * T >> 5) + (tid >> 3)] >> (4 * tid & 31) & 15u;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) hit |= (s_bits[place(k, e) >> 5] >> (place(k, e) & 31) & 1) << e;
        while (hit) {  // one at a time: seldom more in a warp's 128 tokens
          const int e = __ffs(hit) - 1, i = place(k, 0) + (VEC ? e : e * T);
          hit &= hit - 1;
          float l = e == 0 ? v[k][0] : e == 1 ? v[k][1] : e == 2 ? v[k][2] : v[k][3];
          if (const uint32_t c = r.history ? s_count[i] : 0) {
            l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
            l = __fsub_rn(l, __fadd_rn(pres, __fmul_rn(freq, (float)c)));
          }
          if (const uint32_t c = r.bias_ids ? s_bias[i] : 0) l = __fadd_rn(l, r.bias_values[b0 + c - 1]);
#pragma unroll
          for (int f = 0; f < 4; ++f) v[k][f] = e == f ? l : v[k][f];
        }
      }
      if constexpr (MASK) {
        if constexpr (VEC) ok[k] = ok[k] >> (4 * tid & 31) & 15u;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = ok[k] >> e & 1 ? v[k][e] : -INFINITY;
      }
      top = fmaxf(top, fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3])));  // leaves NaN out
      if (y) {
        if constexpr (VEC) {
          if (place(k, 0) < n)
            *reinterpret_cast<float4 *>(y + t0 + place(k, 0)) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (place(k, e) < n) y[t0 + place(k, e)] = v[k][e];
        }
      }
    }
    // The tile's best token.  With one tile per CTA only the threads that hold the CTA's maximum look for it.
    bool look = top > best;
    if (c1 - c0 <= kPickTile) {
      const float w = warp_max(top);
      if (lane == 0) s_top[tid >> 5] = w;
      __syncthreads();
      const float c = warp_max(s_top[lane % kWarps]);
      look = look && top == c;
      if (c > -INFINITY) any = kNone;  // some value is larger: the first number does not matter
    }
    if (look) {
      best = top;
      at = kNone;
#pragma unroll
      for (int k = 0; k < kPickQuads; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) at = v[k][e] == top ? min(at, t0 + place(k, e)) : at;
    }
    if (any < 0 && best == -INFINITY) {
      int f = kNone;
#pragma unroll
      for (int k = 0; k < kPickQuads; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (place(k, e) < n && (!MASK || (ok[k] >> e & 1)) && v[k][e] == v[k][e]) f = min(f, t0 + place(k, e));
      any = f == kNone ? -1 : f;
    }
  }
  if (any == kNone) any = -1;
  // one order for the CTA and the cluster: the larger value, then the lower token; 0 where there is none.
  // -0 + 0 = +0: the two zeros are one value.
  unsigned long long key = at >= 0    ? argmax_key(__fadd_rn(best, 0.0f), (uint32_t)at)
                           : any >= 0 ? argmax_key(-INFINITY, (uint32_t)any)
                                      : 0ull;
  if (__any_sync(0xffffffffu, key != 0)) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  }
  if (lane == 0) s_warp[tid >> 5] = key;
  __syncthreads();
  cluster_wait_all();
  if (tid < 32) {
    key = s_warp[lane % kWarps];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if (tid == 0)
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u64 [%0], %1, [%2];" ::"r"(
                       cluster_map(smem_u32(&s_rank[rank]), 0)),
                   "l"(key), "r"(cluster_map(smem_u32(&s_bar), 0))
                   : "memory");
    if (rank == 0) {
      bool done = __all_sync(0xffffffffu, mbar_wait_cluster(&s_bar, 0));
      if (!done) {
        // The others may yet send: this CTA must not leave before.  They wait for nothing and leave after it, and the
        // cluster's barrier, which counts the threads that are left, then completes with this warp's arrival; what
        // they sent lands soon after.  (The whole warp: a lane that has left the branch may wait for the others.)
        cluster_arrive_all();
        cluster_wait_all();
        done = __all_sync(0xffffffffu, mbar_wait_cluster(&s_bar, 0));
      }
      if (tid == 0) {
        key = 0;
        for (int c = 0; c < (int)gridDim.x; ++c) key = max(key, *reinterpret_cast<volatile unsigned long long *>(&s_rank[c]));
        if (!done && r.bad_flag) atomicMax(r.bad_flag, -QASR_ERR_TIMEOUT);
        if (p.ids) p.ids[m] = done && key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
      }
    }
  }
}

}  // namespace qasr

using namespace qasr;

extern "C" int qasr_logits_pick(int32_t *ids, float *logits_out, const float *logits, const qasr_pick_rules *rules,
                                int M, int vocab, void *stream) {
  if (!rules || M < 0 || vocab <= 0) {
    set_error("qasr_logits_pick: invalid arguments (null rules, M=%d, vocab=%d)", M, vocab);
    return QASR_ERR_INVALID;
  }
  if (M == 0) return QASR_OK;  // before the pointers are looked at: an empty tensor has none
  if (!logits || (!ids && !logits_out)) {
    set_error("qasr_logits_pick: null logits or no output");
    return QASR_ERR_INVALID;
  }
  qasr_pick_rules r = *rules;
  // An empty list has no address of its own: it goes by any other, of which nothing is read (every row's range of it
  // is empty or flagged).
  if (!r.history && r.n_history == 0) r.history = r.history_starts;
  if (!r.bias_ids && r.n_bias == 0) r.bias_ids = r.bias_starts;
  if (r.bias_ids && !r.bias_values && r.n_bias == 0) r.bias_values = reinterpret_cast<const float *>(r.bias_starts);
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
  PickParams p{ids, logits_out, logits, r, vocab, 0, 0};
  // CTAs per row: as many as 16, one tile each, while all CTAs run at once (two on an SM; clusters of 16 leave part
  // of a GPC's SMs idle).  Vocabulary 151,936, us with 16 / 8 / 4 CTAs a row: 1 row 4.0 / 5.4 / 8.6, 8 rows 4.9 /
  // 6.0 / 8.8, 32 rows 15.9 / 11.3 / 18.9, 64 rows with every rule 33.4 / 25.7 / 23.9.
  int C = kPickMaxCluster;
  while (C > 1 && (long)M * C > 256) C /= 2;
  p.chunk = ceil_div(ceil_div(vocab, C), 32) * 32;
  p.table = p.chunk < kPickTile ? p.chunk : kPickTile;
  const size_t smem = (size_t)p.table * 4 * ((r.history ? 1 : 0) + (r.bias_ids ? 1 : 0));
  const bool vec = vocab % 4 == 0 && !((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(logits_out)) & 15);
  const bool mask = r.allow_mask != nullptr;
  const auto kernel = vec ? (mask ? logits_pick_kernel<true, true> : logits_pick_kernel<true, false>)
                          : (mask ? logits_pick_kernel<false, true> : logits_pick_kernel<false, false>);
  static bool attr_done[64][2][2] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return QASR_ERR_INVALID;
  if (!attr_done[dev][vec][mask]) {
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                         "qasr_logits_pick: cluster size opt-in");
    if (!rc)
      rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickTile * 8),
                       "qasr_logits_pick: shared memory opt-in");
    if (rc) return rc;
    attr_done[dev][vec][mask] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)C, (unsigned)M);
  cfg.blockDim = dim3(kPickThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p), "qasr_logits_pick");
}
