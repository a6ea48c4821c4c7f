// tree_attention.cu -- attention of one or several tokens per sequence over
// the INT8 KV cache: decode steps, drafted trees, prompt chunks.
//
// With codes c and scales s of a cache row j, query t of a head:
//   S_tj = scale * sum_d q_td kc_jd * ks_j
//   out_t = sum_j e^(S_tj - max_j S_tj) * vs_j * vc_j / sum_j e^(S_tj - max_j S_tj)
// over the rows j that t sees; nothing visible gives zero.
//
// Both products run on the tensor cores (tcgen05, kind::i8) on the codes as
// they lie in the cache, exactly in 32-bit integers:
//  * a query row is scaled by a power of two 2^(23-E) (2^E bounds its largest
//    magnitude; 2^(22-E) where that would pass three digits), rounded to an
//    integer and split into three signed base-256 digits.  S^T [keys x 3 digit
//    planes of the rows] = K codes [128 keys x 128] * digits^T; the rounding of q
//    is half a step of 2^(E-23).  (With one bit less, as in the INT8 projections, it
//    is most of the outputs' error: 4.3e-7 of their norm and not 3.1e-7 at
//    head_dim 64.)
//  * a product e^S_tj * vs_j over the largest one that the row sees in the tile
//    lies in [0, 1]; 2^22.998 times it, rounded, are three unsigned digits (the
//    low bytes of the float 2^23 + that), off by at most 2^-23.9 of the largest
//    product.  Many products of the tile's largest size add up to an error of
//    some 2^-22 of their sum, about that of f32 sums.  The reference is the row's
//    own and the product's: with the largest weight and the largest scale, each
//    for itself, a sink (much weight, small values) or the scale of a key that
//    the row does not see would take the bits of all others.  O^T [128 values x
//    digit planes] = V codes^T * digits, with V read as it lies (M-major) and the
//    digits written by the thread that owns the key (N-major): nothing is
//    transposed or converted on the way.
// Digit sums are recombined in f32 (one rounding below the value's own) and
// accumulated over the tiles in f32 with the usual running maximum and sum.
//
// Keys sit on the M side (128 TMEM lanes, one thread each), rows on the N
// side: one query row then costs 16 columns instead of a 128-row tile, which
// is what a decode step needs, and the work per key grows with the rows that
// are there.  Two kv heads of 64 values share one 128-wide tile: the digits of
// a row are zero in the other head's half, and its half of O is dropped.
//
// A cluster of C CTAs shares one (sequence, kv head, block of NR rows): each
// takes a run of 128-key tiles, the partial states are pushed to the CTA that
// finishes a row over distributed shared memory, so a call needs no
// workspace, no atomics and no second launch.
//
// Measured (B200, 16 query heads over 8 kv heads of 128, calls replayed back to
// back): 32 sequences x 1 token over 8000 keys 87 us, 541 MB, 0.95 of the copy
// rate (HBM-bound); over 250 .. 8000 keys 47.4 us; one sequence over 545 keys 5.1 us
// (the chain of one tile), 8 over 1001 keys 6.5 us; 8 trees of 31 tokens 16.6 us
// (256 CTAs in one wave: the longest history's five tiles in one CTA, where the
// mean is 2.75, and the set-up and exchange around them); prompts of 4 x 404 tokens
// 24.3 us (728 CTAs with work in 2.5 waves, two tiles each on average; all
// instructions together, 75 per query row and key, are 12 us of issue).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "kv_int8.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace qasr {

// Three planes of 4 consecutive columns of this warp's 32 TMEM lanes, at
// columns 0, stride and 2 * stride of taddr.
QASR_DEV void tmem_ld_planes(uint32_t taddr, uint32_t stride, uint32_t (&d)[3][4]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%12];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%4, %5, %6, %7}, [%13];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%8, %9, %10, %11}, [%14];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(d[0][0]), "=r"(d[0][1]), "=r"(d[0][2]), "=r"(d[0][3]), "=r"(d[1][0]), "=r"(d[1][1]),
        "=r"(d[1][2]), "=r"(d[1][3]), "=r"(d[2][0]), "=r"(d[2][1]), "=r"(d[2][2]), "=r"(d[2][3])
      : "r"(taddr), "r"(taddr + stride), "r"(taddr + 2 * stride)
      : "memory");
}

// Three planes of 8 consecutive columns of this warp's 32 TMEM lanes, at
// columns 0, stride and 2 * stride of taddr.
QASR_DEV void tmem_ld_planes(uint32_t taddr, uint32_t stride, uint32_t (&d)[3][8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%24];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%25];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16, %17, %18, %19, %20, %21, %22, %23}, [%26];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(d[0][0]), "=r"(d[0][1]), "=r"(d[0][2]), "=r"(d[0][3]), "=r"(d[0][4]), "=r"(d[0][5]),
        "=r"(d[0][6]), "=r"(d[0][7]), "=r"(d[1][0]), "=r"(d[1][1]), "=r"(d[1][2]), "=r"(d[1][3]),
        "=r"(d[1][4]), "=r"(d[1][5]), "=r"(d[1][6]), "=r"(d[1][7]), "=r"(d[2][0]), "=r"(d[2][1]),
        "=r"(d[2][2]), "=r"(d[2][3]), "=r"(d[2][4]), "=r"(d[2][5]), "=r"(d[2][6]), "=r"(d[2][7])
      : "r"(taddr), "r"(taddr + stride), "r"(taddr + 2 * stride)
      : "memory");
}

// Three planes of 16 consecutive columns of this warp's 32 TMEM lanes, at
// columns 0, stride and 2 * stride of taddr.
QASR_DEV void tmem_ld_planes(uint32_t taddr, uint32_t stride, uint32_t (&d)[3][16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%48];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%49];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47}, [%50];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(d[0][0]), "=r"(d[0][1]), "=r"(d[0][2]), "=r"(d[0][3]), "=r"(d[0][4]), "=r"(d[0][5]),
        "=r"(d[0][6]), "=r"(d[0][7]), "=r"(d[0][8]), "=r"(d[0][9]), "=r"(d[0][10]), "=r"(d[0][11]),
        "=r"(d[0][12]), "=r"(d[0][13]), "=r"(d[0][14]), "=r"(d[0][15]), "=r"(d[1][0]), "=r"(d[1][1]),
        "=r"(d[1][2]), "=r"(d[1][3]), "=r"(d[1][4]), "=r"(d[1][5]), "=r"(d[1][6]), "=r"(d[1][7]),
        "=r"(d[1][8]), "=r"(d[1][9]), "=r"(d[1][10]), "=r"(d[1][11]), "=r"(d[1][12]), "=r"(d[1][13]),
        "=r"(d[1][14]), "=r"(d[1][15]), "=r"(d[2][0]), "=r"(d[2][1]), "=r"(d[2][2]), "=r"(d[2][3]),
        "=r"(d[2][4]), "=r"(d[2][5]), "=r"(d[2][6]), "=r"(d[2][7]), "=r"(d[2][8]), "=r"(d[2][9]),
        "=r"(d[2][10]), "=r"(d[2][11]), "=r"(d[2][12]), "=r"(d[2][13]), "=r"(d[2][14]), "=r"(d[2][15])
      : "r"(taddr), "r"(taddr + stride), "r"(taddr + 2 * stride)
      : "memory");
}

// Two f32 in one register pair, two of a step at a time.
using F2 = unsigned long long;
QASR_DEV F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
QASR_DEV float f2_lo(F2 a) { return __uint_as_float((uint32_t)a); }
QASR_DEV float f2_hi(F2 a) { return __uint_as_float((uint32_t)(a >> 32)); }
QASR_DEV F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
QASR_DEV F2 f2_add_up(F2 a, F2 b) {  // rounded up
  F2 r;
  asm("add.rp.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
QASR_DEV F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
QASR_DEV F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

constexpr int kTaKeys = 128;             // keys of a tile: TMEM lanes of S^T
constexpr int kTaTile = kTaKeys * 128;   // bytes of a K (or V) tile
constexpr int kTaMaxCluster = 16;
constexpr float kTaMagic = 8388608.0f;   // 2^23: its low three bytes are zero

// Rows of a block: NR query rows, their digit planes side by side (plane d at
// column d * NR), N columns for the tensor cores (a multiple of 16).
template <int NR>
struct TaShape {
  static_assert(NR == 4 || NR == 8 || NR == 16 || NR == 32, "rows of a block");
  static constexpr int kN = NR == 4 ? 16 : NR == 8 ? 32 : 3 * NR;
  static constexpr int kTmem = NR == 32 ? 256 : NR == 16 ? 128 : NR == 8 ? 64 : 32;  // S and O, a power of two
  // K and V tiles in flight, with two CTAs on an SM: three where shared memory has room (32 histories of 250 ..
  // 8000 keys 47.8 us, 59.3 with two)
  static constexpr int kStages = NR == 4 ? 3 : 2;
  // softmax warpgroups, each owning R rows of every tile: two halve the chain of instructions from one product to
  // the next (prompt chunks 29.6 us, 33.8 with one group of 32 rows a thread)
  static constexpr int kGroups = NR == 32 ? 2 : 1;
  static constexpr int kR = NR / kGroups;
  static constexpr int kWarps = 4 * kGroups, kThreads = 32 * kWarps + 64;  // and the MMA and the TMA warp
  static constexpr int kQBytes = kN * 128, kPBytes = kN * 128;
};

struct TreeAttnParams {
  CUtensorMap tm_k, tm_v;  // codes as [cache rows, kv_dim], box 128 rows x 128 bytes, 128-byte swizzle
  float *out;
  const float *q;
  qasr_kv_int8 c;
  qasr_kv_rows r;
  const uint64_t *tree_mask;
  int layer, n_heads;
  int group, width;  // query heads per kv head; query rows of one token in a block (group x heads per tile)
  int cshift;        // log2 of the cluster size
  float scale;
};

template <int NR>
struct TaSmem {
  using Sh = TaShape<NR>;
  alignas(1024) unsigned char ring[Sh::kStages][2][kTaTile];  // K, V
  alignas(1024) unsigned char q[Sh::kQBytes];  // digits, K-major, 128-byte swizzle
  alignas(1024) unsigned char p[Sh::kPBytes];  // digits, N-major, no swizzle
  // partial states pushed by the cluster: entry r / C * C + c is CTA c's of row r, one of the rows r % C = rank
  static constexpr int kRecv = NR < kTaMaxCluster ? kTaMaxCluster : NR;
  float recv[kRecv][128], recv_m[kRecv], recv_l[kRecv];
  // per tile (two in flight), warp and pair of rows: minus the running maximum, units per weight, the factor of the
  // sums before the tile, what a unit of O counts
  alignas(16) F2 rowc[2][Sh::kWarps][Sh::kR / 2][4];
  // per tile and warp: the rows' largest scores, then their largest products of weight and value scale (log 2)
  alignas(16) float wmax[2][Sh::kWarps][2 * Sh::kR];
  alignas(16) float qf[NR];  // 2^(E-22) * scale * log2(e)
  float lsum[4][NR], mrun[NR];
  uint32_t mask[2][NR];
  int tok[NR];            // the row's token, -1 for none
  long long at[NR];       // element of q and out where value column 0 of the row's tile falls
  uint64_t full_k[3], full_v[3], empty[3], sfull, sfree, pready, ofull, qready, done;
  uint32_t tmem, hi;
  int abort;
};

// Descriptor of the digits P: N-major without swizzle, 16 columns x 8 keys per
// 128-byte core matrix, the next 8 keys 128 bytes on, the next 16 columns
// 2048 bytes on (128 keys).
QASR_DEV uint64_t ta_desc_p(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(2048 >> 4) << 32 |
         (uint64_t)1 << 46;
}

// kind::i8, S32 sums; A signed, B signed (S) or unsigned (O), both K-major (S)
// or both M/N-major (O).
constexpr uint32_t ta_idesc_s(int N) { return umma_idesc_s8(128, N); }
constexpr uint32_t ta_idesc_o(int N) {
  return (2u << 4) | (1u << 7) | (1u << 15) | (1u << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

QASR_DEV float ta_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
QASR_DEV float ta_lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
QASR_DEV float ta_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
QASR_DEV float ta_warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
QASR_DEV void ta_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
QASR_DEV void ta_store_remote(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Bounded wait that also gives up once another role has.
template <int NR>
QASR_DEV bool ta_wait(TaSmem<NR> &sm, uint64_t *bar, unsigned parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*reinterpret_cast<volatile int *>(&sm.abort)) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      atomicExch(&sm.abort, 1);
      return false;
    }
  }
  return true;
}

// Digits of four q values at bytes b .. b+3 of digit row n = r, r + NR, r + 2 NR.
template <int NR>
QASR_DEV void ta_put_digits(unsigned char *q, int r, int b, float4 v, float qm) {
  // a power of two: the products are exact, but for what is far below a half
  int X[4] = {__float2int_rn(__fmul_rn(v.x, qm)), __float2int_rn(__fmul_rn(v.y, qm)),
              __float2int_rn(__fmul_rn(v.z, qm)), __float2int_rn(__fmul_rn(v.w, qm))};
#pragma unroll
  for (int d = 2; d >= 0; --d) {  // balanced: -128 .. 127, the carry goes up
    const uint32_t w =
        __byte_perm(__byte_perm(X[0], X[1], 0x0040), __byte_perm(X[2], X[3], 0x0040), 0x5410);
    const int n = d * NR + r;
    *reinterpret_cast<uint32_t *>(q + n * 128 + (((b >> 4) ^ (n & 7)) << 4) + (b & 15)) = w;
#pragma unroll
    for (int i = 0; i < 4; ++i) X[i] = (int)((unsigned)X[i] + 128u) >> 8;
  }
}

// HD: head_dim; HPB = 128 / HD kv heads share a tile.  Grid: (C x head blocks,
// row blocks, sequences), clusters of C along x; the last rows, which see the
// most keys, come first.
template <int HD, int NR>
__global__ void __launch_bounds__(TaShape<NR>::kThreads, 2)
tree_attention_kernel(const __grid_constant__ TreeAttnParams p) {
  using Sh = TaShape<NR>;
  constexpr int HPB = 128 / HD, N = Sh::kN, ST = Sh::kStages, R = Sh::kR;
  constexpr int kMmaWarp = Sh::kWarps, kTmaWarp = Sh::kWarps + 1;
  extern __shared__ unsigned char smem_raw[];
  TaSmem<NR> &sm = *reinterpret_cast<TaSmem<NR> *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = 1 << p.cshift, rank = blockIdx.x & (C - 1), hb = blockIdx.x >> p.cshift, m = blockIdx.z;
  const int G = p.group, W = p.width;
  // what does not depend on the kernel before: barriers, tensor memory
  if (warp == kTmaWarp && lane == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sm.full_k[i], 1);
      mbar_init(&sm.full_v[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.sfull, 1);
    mbar_init(&sm.sfree, Sh::kWarps);
    mbar_init(&sm.pready, Sh::kWarps);
    mbar_init(&sm.ofull, 1);
    mbar_init(&sm.qready, 1);
    mbar_init(&sm.done, 1);
    sm.abort = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) tmem_alloc(&sm.tmem, Sh::kTmem);
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem, tmem_o = tmem + N;
  pdl_wait();  // first: what starts as a dependent of this kernel finds all kernels before it done
  pdl_launch_dependents();

  const KvSeq s = kv_seq(p.r, p.c, m);
  const int v0 = (int)(gridDim.y - 1 - blockIdx.y) * NR, rows = min(NR, s.n * W - v0);  // the block's rows v0 .. of s.n * W
  const bool first = blockIdx.x == 0 && blockIdx.y == 0 && m == 0;
  if (rows <= 0) {  // the whole cluster
    if (first && warp == 0) kv_flag_bad(p.r, p.c, lane);
    if (warp == kMmaWarp) tmem_dealloc(tmem, Sh::kTmem);
    return;
  }
  const bool tree = p.tree_mask != nullptr;
  const int len = s.pos + (tree ? s.n : (v0 + rows - 1) / W + 1);  // keys any row may see
  const unsigned tiles = (unsigned)(len + kTaKeys - 1) / kTaKeys;
  // below 2^25 tiles: times a rank still fits
  const int i0 = (int)(tiles * rank >> p.cshift), n = (int)(tiles * (rank + 1) >> p.cshift) - i0;
  if (C > 1) cluster_arrive_all();  // waited for before the first remote store: every CTA has started

  // thread = value column (acc2), key (l2), two rows each; lane = row (m_run)
  F2 acc2[R / 2], l2[R / 2];
  float m_run = -INFINITY;
#pragma unroll
  for (int r = 0; r < R / 2; ++r) acc2[r] = l2[r] = 0ull;
  const int col = tid & 127, wg = warp >> 2;  // softmax warps: key / value column, first row wg * R

  if (warp == kTmaWarp) {
    // ---------------------------------------------------------------- TMA
    if (lane == 0) {
      const int row = (int)kv_row(p.c, s.slot, p.layer, 0);
      int i = 0;
      for (; i < n; ++i) {
        const int st = i % ST, y = row + (i0 + i) * kTaKeys;
        if (i >= ST && !ta_wait(sm, &sm.empty[st], (unsigned)((i / ST - 1) & 1))) break;
        mbar_arrive_expect_tx(&sm.full_k[st], kTaTile);
        tma_load_2d_u8(sm.ring[st][0], &p.tm_k, hb * 128, y, &sm.full_k[st]);
        mbar_arrive_expect_tx(&sm.full_v[st], kTaTile);
        tma_load_2d_u8(sm.ring[st][1], &p.tm_v, hb * 128, y, &sm.full_v[st]);
      }
      // copies that nobody waited for (after a timeout) land before the CTA leaves
      for (int k = max(0, i - ST); k < i; ++k) {
        mbar_wait(&sm.full_k[k % ST], (unsigned)((k / ST) & 1));
        mbar_wait(&sm.full_v[k % ST], (unsigned)((k / ST) & 1));
      }
    }
    __syncwarp();
    if (first) kv_flag_bad(p.r, p.c, lane);
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA
    if (lane == 0 && n > 0) {
      const uint32_t qa = smem_u32(sm.q), pa = smem_u32(sm.p);
      auto scores = [&](int i) {
        const int st = i % ST;
        if (!ta_wait(sm, &sm.full_k[st], (unsigned)((i / ST) & 1))) return false;
        tc_fence_after();
        const uint32_t ka = smem_u32(sm.ring[st][0]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_s8(tmem, umma_desc_sw128(ka + 32 * k), umma_desc_sw128(qa + 32 * k), ta_idesc_s(N), k > 0);
        umma_commit(&sm.sfull);
        return true;
      };
      bool ok = ta_wait(sm, &sm.qready, 0) && scores(0);
      for (int i = 0; ok && i < n; ++i) {
        const int st = i % ST;
        if (i + 1 < n) ok = ta_wait(sm, &sm.sfree, (unsigned)(i & 1)) && scores(i + 1);
        ok = ok && ta_wait(sm, &sm.full_v[st], (unsigned)((i / ST) & 1)) && ta_wait(sm, &sm.pready, (unsigned)(i & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_u32(sm.ring[st][1]);
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 32 keys a step: four 8-key groups of 1024 (V) and 128 (P) bytes
          umma_s8(tmem_o, umma_desc_sw128(va + 4096 * k), ta_desc_p(pa + 512 * k), ta_idesc_o(N), k > 0);
        umma_commit(&sm.empty[st]);
        umma_commit(&sm.ofull);
      }
      // All products end before TMEM is freed, also where another role has given up and waits for none of them
      // (otherwise the softmax warps wait for the last one meanwhile).
      umma_commit(&sm.done);
      mbar_wait(&sm.done, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax
    // lane r: row r's token, place in q and out, and half of the tile (pairs of heads)
    const int v = v0 + lane, t = lane < rows ? v / W : -1, h = v - t * W;
    const uint32_t hi = HPB == 2 ? __ballot_sync(0xffffffffu, lane < rows && h >= G) : 0;  // bit r: the second head
    const bool live = t >= 0 && hb * W + h < p.n_heads;
    const long long at = live ? ((long long)(s.row0 + t) * p.n_heads + hb * W + h - (HPB == 2 && h >= G)) * HD : -1;
    constexpr int kQ = NR / Sh::kWarps;
    float4 x4[kQ];
#pragma unroll
    for (int k = 0; k < kQ; ++k) {  // warp w converts rows w, w + warps, ..: all their loads in flight
      const int r = warp + Sh::kWarps * k, b = 4 * lane, b0 = HPB == 2 && (hi >> r & 1) ? HD : 0;
      const long long a = __shfl_sync(0xffffffffu, at, r);
      x4[k] = a >= 0 && b >= b0 && b < b0 + HD ? *reinterpret_cast<const float4 *>(p.q + a + b)
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const uint64_t mask = warp == 0 && t >= 0 && tree ? p.tree_mask[s.row0 + t] : 0;
#pragma unroll
    for (int k = 0; k < kQ; ++k) {
      const float4 x = x4[k];
      constexpr uint32_t kAbs = 0x7fffffffu;
      const uint32_t top = __reduce_max_sync(
          0xffffffffu, max(max(__float_as_uint(x.x) & kAbs, __float_as_uint(x.y) & kAbs),
                           max(__float_as_uint(x.z) & kAbs, __float_as_uint(x.w) & kAbs)));
      // 2^e above the largest magnitude; a row below 2^-100 loses bits.  The largest integer of three signed digits
      // is 127 (65536 + 256 + 1): 2^23 units to 2^e, but 2^22 for the half per cent of magnitudes that would round
      // above it.  NaN or an infinity (all exponent bits) makes the row's factor, and so its scores, NaN.
      const int r = warp + Sh::kWarps * k, e = max((int)(top >> 23) - 126, -100);
      const int up = 23 - e - ((top & 0x7fffffu) > 0x7efefeu);
      ta_put_digits<NR>(sm.q, r, 4 * lane, x, __int_as_float((127 + up) << 23));
      if (lane == 0) {
        const float f = __fmul_rn(__int_as_float((127 - up) << 23), __fmul_rn(p.scale, 1.44269504088896341f));
        sm.qf[r] = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : f;
      }
    }
    if (warp == 0 && lane < NR) {
      sm.mask[0][lane] = (uint32_t)mask;
      sm.mask[1][lane] = (uint32_t)(mask >> 32);
      sm.tok[lane] = t;
      sm.at[lane] = at;
      if (lane == 0) sm.hi = hi;
    }
    for (int b = 3 * NR * 128 + 4 * tid; b < Sh::kQBytes; b += 512) *reinterpret_cast<uint32_t *>(sm.q + b) = 0;
    fence_proxy_async();
    named_bar(1, 32 * Sh::kWarps);
    if (tid == 0) ta_arrive(&sm.qready);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21, my_s = tmem + lanes + wg * R, my_o = tmem_o + lanes + wg * R;
    const uint32_t my_hi = hi >> (wg * R);  // bit r: the group's row r is of the pair's second head
    const int *tok = sm.tok + wg * R;
    const float *qf = sm.qf + wg * R;
    float nks[HPB], nvs[HPB];  // scales of this thread's key of the next tile
    int next = i0 * kTaKeys + col;
    const size_t srow = (kv_row(p.c, s.slot, p.layer, 0) + next) * p.c.n_kv_heads + hb * HPB;
    const float *ksp = p.c.k_scales + srow, *vsp = p.c.v_scales + srow;
    const bool two = hb * HPB + 1 < p.c.n_kv_heads;
    auto load_scales = [&](bool more) {
#pragma unroll
      for (int u = 0; u < HPB; ++u) {
        const bool in = more && next < len && (u == 0 || two);
        nks[u] = in ? ksp[u] : 0.0f;  // no read-only loads: the append before may have written them since the launch
        nvs[u] = in ? vsp[u] : 0.0f;
      }
      next += kTaKeys;
      ksp += (size_t)kTaKeys * p.c.n_kv_heads;
      vsp += (size_t)kTaKeys * p.c.n_kv_heads;
    };
    // acc = acc * old + O * coef for the tile whose constants are in rowc[b]
    auto fold = [&](int b) {
      uint32_t d[3][R];
      tmem_ld_planes(my_o, NR, d);
#pragma unroll
      for (int r = 0; r < R; r += 2) {
        const ulonglong2 c = *reinterpret_cast<const ulonglong2 *>(&sm.rowc[b][warp][r / 2][2]);
        const F2 o =
            f2_fma(f2((float)(int)d[2][r], (float)(int)d[2][r + 1]), f2(65536.0f, 65536.0f),
                   f2((float)((int)d[1][r] * 256 + (int)d[0][r]), (float)((int)d[1][r + 1] * 256 + (int)d[0][r + 1])));
        acc2[r / 2] = f2_fma(acc2[r / 2], c.x, f2_mul(o, c.y));
      }
    };
    // After a timeout (sm.abort) every wait returns at once and the loop runs on: a group's warps must meet at
    // the same number of barriers.  The results are thrown away.
    load_scales(n > 0);
    for (int i = 0; i < n; ++i) {
      const int buf = i & 1, j = (i0 + i) * kTaKeys + col;
      float ks[HPB], vs[HPB];
#pragma unroll
      for (int u = 0; u < HPB; ++u) {
        ks[u] = fmaf(nks[u], 0.0f, nks[u]);  // an infinity becomes NaN: a score of -infinity would count as hidden
        vs[u] = nvs[u];
      }
      load_scales(i + 1 < n);
      ta_wait(sm, &sm.sfull, (unsigned)(i & 1));
      __syncwarp();
      tc_fence_after();
      float x[R];  // scores in units of log 2
      {
        uint32_t d[3][R];
        tmem_ld_planes(my_s, NR, d);
#pragma unroll
        for (int r = 0; r < R; r += 2) {
          const F2 k = f2(HPB == 2 && (my_hi >> r & 1) ? ks[HPB - 1] : ks[0],
                          HPB == 2 && (my_hi >> (r + 1) & 1) ? ks[HPB - 1] : ks[0]);
          const F2 sum =
              f2_fma(f2((float)(int)d[0][r], (float)(int)d[0][r + 1]), f2(65536.0f, 65536.0f),
                     f2((float)((int)d[1][r] * 256 + (int)d[2][r]), (float)((int)d[1][r + 1] * 256 + (int)d[2][r + 1])));
          const F2 x2 = f2_mul(sum, f2_mul(*reinterpret_cast<const F2 *>(qf + r), k));
          x[r] = f2_lo(x2);
          x[r + 1] = f2_hi(x2);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) ta_arrive(&sm.sfree);
      const int place = j - s.pos;  // >= 0: the row of one of the sequence's own tokens
      if ((i0 + i + 1) * kTaKeys > s.pos) {
        if (tree) {
          const uint32_t *seen = sm.mask[place >> 5 & 1] + wg * R;
          const uint32_t past = place < 0, own = place < s.n;  // bits: visible anyway, in the tree at all
          const int bit = place & 31;
#pragma unroll
          for (int r = 0; r < R; ++r) x[r] = (past | (seen[r] >> bit & own)) ? x[r] : -INFINITY;
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) x[r] = place <= tok[r] ? x[r] : -INFINITY;
        }
      }
      // a value scale that is no number in [0, 2^125) counts as NaN, for the rows that see it
      bool odd[HPB];
      float lvs[HPB];
#pragma unroll
      for (int u = 0; u < HPB; ++u) {
        odd[u] = !(vs[u] >= 0.0f && vs[u] < 4.2535296e37f);
        if (odd[u]) vs[u] = 0.0f;
        lvs[u] = ta_lg2(vs[u]);
      }
      // Of two heads' values the one of row r.  The bits pass through a register that the compiler knows nothing of,
      // or it keeps the choice of all rows at hand and spills 80 bytes for it (32 rows: 28.7 us against 26.4).
      uint32_t second = my_hi;
      if constexpr (HPB == 2) asm volatile("" : "+r"(second));
      auto of_row = [&](const float(&a)[HPB], int r) { return HPB == 2 && (second >> r & 1) ? a[HPB - 1] : a[0]; };
#pragma unroll
      for (int r = 0; r < R; r += 4) {  // the warp's maxima; products' logarithms rounded up: none passes its maximum
        const F2 a = f2_add_up(f2(x[r], x[r + 1]), f2(of_row(lvs, r), of_row(lvs, r + 1)));
        const F2 b = f2_add_up(f2(x[r + 2], x[r + 3]), f2(of_row(lvs, r + 2), of_row(lvs, r + 3)));
        const float4 s4 =
            make_float4(ta_warp_max(x[r]), ta_warp_max(x[r + 1]), ta_warp_max(x[r + 2]), ta_warp_max(x[r + 3]));
        const float4 u4 =
            make_float4(ta_warp_max(f2_lo(a)), ta_warp_max(f2_hi(a)), ta_warp_max(f2_lo(b)), ta_warp_max(f2_hi(b)));
        if (lane == 0) {
          *reinterpret_cast<float4 *>(&sm.wmax[buf][warp][r]) = s4;
          *reinterpret_cast<float4 *>(&sm.wmax[buf][warp][R + r]) = u4;
        }
      }
      named_bar(2 + wg, 128);
      const int w0 = 4 * wg;  // the group's warps
      auto over_warps = [&](int e) {
        return fmaxf(fmaxf(sm.wmax[buf][w0][e], sm.wmax[buf][w0 + 1][e]),
                     fmaxf(sm.wmax[buf][w0 + 2][e], sm.wmax[buf][w0 + 3][e]));
      };
      // A product's integer is 2^(x - base) * vs * units, at most 2^23: 2^22.998 leaves room for the errors of the
      // logarithms and exponentials (below 2^-13 in all) and for the roundings.  What a unit counts is the reciprocal
      // of `units`, to an ulp or two that scales the whole tile's share.
      const float most = lane < 2 * R ? over_warps(lane) : 0.0f;
      float umax = __shfl_down_sync(0xffffffffu, most, R);
      const float top = fmaxf(m_run, most), base = lane >= R || top == -INFINITY ? 0.0f : top;
      float *c = reinterpret_cast<float *>(sm.rowc[buf][warp][lane / 2 % (R / 2)]) + lane % 2;
      if (lane < R) c[0] = -base;
      umax = __fsub_rn(umax, base);
      // Where scores are so large that a product's logarithm, rounded up, says little, the logarithms are taken again,
      // less the base.  All warps of the group have the same bases: they all come here, or none.
      if (__any_sync(0xffffffffu, fabsf(base) >= 65536.0f)) {
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; r += 2) {
          const F2 from = f2_add(f2(x[r], x[r + 1]), sm.rowc[buf][warp][r / 2][0]);
          const F2 y = f2_add_up(from, f2(of_row(lvs, r), of_row(lvs, r + 1)));
          const float2 u2 = make_float2(ta_warp_max(f2_lo(y)), ta_warp_max(f2_hi(y)));
          if (lane == 0) *reinterpret_cast<float2 *>(&sm.wmax[buf][warp][R + r]) = u2;
        }
        named_bar(2 + wg, 128);
        if (lane < R) umax = over_warps(R + lane);
      }
      if (lane < R) {
        // a tile whose products are all below 2^-100 of the row's largest weight loses bits
        const float units = ta_ex2(__fadd_rn(fminf(-umax, 100.0f), 22.998f));
        c[2] = units;
        c[4] = m_run == -INFINITY ? 0.0f : ta_ex2(__fsub_rn(m_run, base));
        c[6] = ta_rcp(units);
        m_run = top;
      }
      __syncwarp();
      bool any_odd = odd[0];
      if constexpr (HPB == 2) any_odd |= odd[HPB - 1];
      if (__any_sync(0xffffffffu, any_odd)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (x[r] != -INFINITY && (HPB == 2 && (my_hi >> r & 1) ? odd[HPB - 1] : odd[0]))
            l2[r / 2] |= 0x7fc00000ull << (r % 2 * 32);  // a quiet NaN whatever it was
      }
      if (i > 0) {  // the previous tile's O; its digits in sm.p are free after it
        ta_wait(sm, &sm.ofull, (unsigned)((i - 1) & 1));
        __syncwarp();
        tc_fence_after();
        fold(buf ^ 1);
      }
      constexpr int kWords = R == 16 ? 12 : N / 4;  // of this thread's key: three planes of R bytes, then unused columns
      uint32_t w[kWords];
#pragma unroll
      for (int r = 3 * R / 4; r < kWords; ++r) w[r] = 0;
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += 4) {
        uint32_t f[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int r = r0 + e;
          const ulonglong2 c = *reinterpret_cast<const ulonglong2 *>(&sm.rowc[buf][warp][r / 2][0]);
          const F2 old = sm.rowc[buf][warp][r / 2][2];
          const F2 y = f2_add(f2(x[r], x[r + 1]), c.x);
          const F2 pr = f2(ta_ex2(f2_lo(y)), ta_ex2(f2_hi(y)));
          l2[r / 2] = f2_fma(l2[r / 2], old, pr);
          const F2 w2 = f2_fma(f2_mul(pr, f2(of_row(vs, r), of_row(vs, r + 1))), c.y, f2(kTaMagic, kTaMagic));
          f[e] = (uint32_t)w2;
          f[e + 1] = (uint32_t)(w2 >> 32);
        }
        // bytes 0, 1 and 2 of the four rows
        const uint32_t a = __byte_perm(f[0], f[1], 0x5140), b = __byte_perm(f[2], f[3], 0x5140);
        w[r0 / 4] = __byte_perm(a, b, 0x5410);
        w[R / 4 + r0 / 4] = __byte_perm(a, b, 0x7632);
        w[R / 2 + r0 / 4] = __byte_perm(__byte_perm(f[0], f[1], 0x0062), __byte_perm(f[2], f[3], 0x0062), 0x5410);
      }
#pragma unroll
      for (int g = 0; g < kWords / 4; ++g)  // 16 columns of the key: a whole plane of the group where R is 16
        *reinterpret_cast<uint4 *>(sm.p + (g * Sh::kGroups + wg) * 2048 + col * 16) =
            make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
      fence_proxy_async();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) ta_arrive(&sm.pready);
    }
    if (n > 0) {
      ta_wait(sm, &sm.ofull, (unsigned)((n - 1) & 1));
      __syncwarp();
      tc_fence_after();
      fold((n - 1) & 1);
    }
    tc_fence_before();
    // sums over the keys
    float l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) l[r] = r % 2 ? f2_hi(l2[r / 2]) : f2_lo(l2[r / 2]);
    sm.lsum[warp & 3][wg * R + reduce_index<R>(lane)] = warp_reduce_scatter<R>(l);
    if (lane < R && (warp & 3) == 0) sm.mrun[wg * R + lane] = m_run;
  }
  __syncwarp();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmem);  // before the cluster waits: a CTA that waits for TMEM never waits for this one
  }
  const bool failed = sm.abort != 0;
  if (failed && tid == 0 && p.r.bad_flag) atomicMax(p.r.bad_flag, -QASR_ERR_TIMEOUT);
  float part_l = 0.0f;  // lane = row
  if (lane < NR)
    part_l = failed ? __uint_as_float(0x7fc00000u)
                    : __fadd_rn(__fadd_rn(sm.lsum[0][lane], sm.lsum[1][lane]),
                                __fadd_rn(sm.lsum[2][lane], sm.lsum[3][lane]));
  if (C == 1) {
    if (warp < Sh::kWarps) {
      const float inv = part_l == 0.0f ? 0.0f : __frcp_rn(part_l);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = wg * R + i;
        const float f = __shfl_sync(0xffffffffu, inv, r);
        const long long at = sm.at[r];
        const bool mine = HPB == 1 || (col >= HD) == (sm.hi >> r & 1);
        if (at >= 0 && mine) p.out[at + col] = __fmul_rn(i % 2 ? f2_hi(acc2[i / 2]) : f2_lo(acc2[i / 2]), f);
      }
    }
    return;
  }

  // Row r is finished by CTA r % C; partial states go there.
  cluster_wait_all();
  const int below = C - 1;
  if (warp < Sh::kWarps) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = wg * R + i;
      if (r < rows)
        ta_store_remote(cluster_map(smem_u32(&sm.recv[(r & ~below) + rank][col]), r & below),
                        i % 2 ? f2_hi(acc2[i / 2]) : f2_lo(acc2[i / 2]));
    }
    if (warp == 0 && lane < rows) {
      const int e = (lane & ~below) + rank;
      ta_store_remote(cluster_map(smem_u32(&sm.recv_m[e]), lane & below), sm.mrun[lane]);
      ta_store_remote(cluster_map(smem_u32(&sm.recv_l[e]), lane & below), part_l);
    }
  }
  __syncwarp();
  cluster_sync_all();
  // one warp per row: lane c has part c's maximum and sum, then four columns of the output
  for (int r = rank + warp * C; r < rows; r += C * (Sh::kThreads / 32)) {
    const int e0 = r & ~below;
    const float mc = lane < C ? sm.recv_m[e0 + lane] : -INFINITY, lc = lane < C ? sm.recv_l[e0 + lane] : 0.0f;
    const float top = warp_max(mc);
    // a part that saw nothing has sum 0 (NaN if it failed or saw a NaN) and counts as nothing
    const float fc = mc == -INFINITY ? 0.0f : ta_ex2(__fsub_rn(mc, top));
    const float sum = warp_sum(mc == -INFINITY ? lc : __fmul_rn(lc, fc));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < C; ++c) {
      const float f = __shfl_sync(0xffffffffu, fc, c);
      const float4 a = *reinterpret_cast<const float4 *>(&sm.recv[e0 + c][4 * lane]);
      o.x = fmaf(a.x, f, o.x);
      o.y = fmaf(a.y, f, o.y);
      o.z = fmaf(a.z, f, o.z);
      o.w = fmaf(a.w, f, o.w);
    }
    const float inv = sum == 0.0f ? 0.0f : __frcp_rn(sum);
    const long long at = sm.at[r];
    const bool mine = HPB == 1 || (4 * lane >= HD) == (sm.hi >> r & 1);
    if (at >= 0 && mine)
      *reinterpret_cast<float4 *>(p.out + at + 4 * lane) =
          make_float4(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv), __fmul_rn(o.z, inv), __fmul_rn(o.w, inv));
  }
}

// Query rows of one kv head (or pair) of the longest sequence.
static long longest_rows(const TreeAttnParams &p) { return (long)std::min(p.r.max_rows, p.r.n_rows) * p.width; }

template <int HD, int NR>
static int tree_attention_launch(TreeAttnParams p, cudaStream_t st) {
  constexpr int HPB = 128 / HD;
  const size_t smem = sizeof(TaSmem<NR>) + 1024;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return QASR_ERR_INVALID;
  if (!attr_done[dev]) {
    int rc = cuda_status(cudaFuncSetAttribute(tree_attention_kernel<HD, NR>,
                                              cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                         "qasr_tree_attention_int8: shared memory opt-in");
    if (!rc)
      rc = cuda_status(cudaFuncSetAttribute(tree_attention_kernel<HD, NR>,
                                            cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                       "qasr_tree_attention_int8: cluster size opt-in");
    if (rc) return rc;
    attr_done[dev] = true;
  }
  const int heads = ceil_div(p.c.n_kv_heads, HPB);
  const long row_blocks = (longest_rows(p) + NR - 1) / NR;  // at most 65,535
  // CTAs per block of rows.  A CTA costs 3 to 4 us beside its tiles, so no more than 256 of them in all (over 1000
  // rows, 32 blocks take 5.9 us with 8 each and 14.1 with 16; 64 blocks 6.5 with 4, 11.3 with 8), but up to 512 where
  // long histories (32 tiles) may differ in length and the longest would set the time: 256 blocks over 250 .. 8000 rows
  // take 47 us with two each and 62 with one (all 8000: 87 and 81); 128 blocks 30 with four and 36 with two (50 and
  // 44).  Sixteen of a cluster find room on few SMs of a GPC at a time: only for 8 blocks (2000 rows: 5.6 us, 5.7 with
  // 8; 16 blocks 9.4 and 5.5).  These are single tokens; blocks of 32 rows go by the same limits.  Without a bound
  // from the host the tiles are the cache's capacity, and short histories in a large cache get CTAs without work.
  const int keys = p.r.max_keys > 0 ? std::min(p.r.max_keys, p.c.max_seq) : p.c.max_seq;
  const int tiles = ceil_div(keys, kTaKeys);
  const long blocks = (long)heads * row_blocks * p.r.n_seqs;
  const int most = blocks <= 8 && tiles >= 16 ? 16 : 8;
  p.cshift = 0;
  for (int C = 2; C <= most && C < 2 * tiles && blocks * C <= (C <= 4 && tiles >= 32 ? 512 : 256); C *= 2) ++p.cshift;
  const int C = 1 << p.cshift;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(C * heads), (unsigned)row_blocks, (unsigned)p.r.n_seqs);
  cfg.blockDim = dim3(TaShape<NR>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, tree_attention_kernel<HD, NR>, p), "qasr_tree_attention_int8");
}

// The smallest block that takes a head's query rows, at most 32.  The work of a tile goes by the block's rows, used
// or not, but two blocks read the keys twice: one sequence a kv head's 2 rows over 1000 keys, us with blocks of 4 /
// 8 / 16 / 32: 5.0 / 5.3 / 5.9 / 6.3; 8 sequences of 4 rows 6.7 / 7.1 / 7.9 / 9.5; of 8 rows 8.4 / 7.1 / 7.9 / 9.6; of 16
// rows (trees of 8) 10.3 / 9.1 / 8.0 / 10.1; of 32 rows 19.8 / 12.4 / 10.7 / 10.4.
template <int HD>
static int tree_attention_rows(const TreeAttnParams &p, cudaStream_t st) {
  const long rows = longest_rows(p);
  if (rows <= 4) return tree_attention_launch<HD, 4>(p, st);
  if (rows <= 8) return tree_attention_launch<HD, 8>(p, st);
  if (rows <= 16) return tree_attention_launch<HD, 16>(p, st);
  return tree_attention_launch<HD, 32>(p, st);
}

// Codes as a [cache rows, kv_dim] byte matrix.
static int kv_codes_map(CUtensorMap *tm, const int8_t *codes, const qasr_kv_int8 &c) {
  const auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
  if (!encode) {
    set_error("qasr_tree_attention_int8: cuTensorMapEncodeTiled unavailable");
    return QASR_ERR_CUDA;
  }
  const cuuint64_t kv_dim = (cuuint64_t)c.n_kv_heads * c.head_dim;
  const cuuint64_t dims[2] = {kv_dim, (cuuint64_t)c.n_slots * c.n_layers * c.max_seq};
  const cuuint64_t strides[1] = {kv_dim};
  const cuuint32_t box[2] = {128, kTaKeys};
  const cuuint32_t estr[2] = {1, 1};
  const auto run = [&] {
    return encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(codes), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = run();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {  // this host thread has made no runtime call that binds the device's context
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = run();
  }
  if (r != CUDA_SUCCESS) {
    set_error("qasr_tree_attention_int8: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return QASR_ERR_CUDA;
  }
  return QASR_OK;
}

}  // namespace qasr

using namespace qasr;

extern "C" int qasr_tree_attention_int8(float *out, const float *q, const qasr_kv_int8 *cache, int layer,
                                        const qasr_kv_rows *rows, const uint64_t *tree_mask, int n_heads, float scale,
                                        void *stream) {
  if (int rc = kv_int8_check("qasr_tree_attention_int8", cache, layer, rows)) return rc;
  if (rows->n_seqs == 0 || rows->n_rows == 0 || rows->max_rows == 0) return QASR_OK;  // empty operands have no address
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
  TreeAttnParams p{};
  p.r = *rows;
  p.group = n_heads / cache->n_kv_heads;
  p.width = p.group * (128 / cache->head_dim);
  if (longest_rows(p) > 32l * 65535) {
    set_error("qasr_tree_attention_int8: too many query rows per sequence (max_rows %d)", rows->max_rows);
    return QASR_ERR_UNSUPPORTED;
  }
  if (int rc = kv_codes_map(&p.tm_k, cache->k, *cache)) return rc;
  if (int rc = kv_codes_map(&p.tm_v, cache->v, *cache)) return rc;
  p.out = out;
  p.q = q;
  p.c = *cache;
  p.tree_mask = tree_mask;
  p.layer = layer;
  p.n_heads = n_heads;
  p.scale = scale;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return cache->head_dim == 128 ? tree_attention_rows<128>(p, st) : tree_attention_rows<64>(p, st);
}
