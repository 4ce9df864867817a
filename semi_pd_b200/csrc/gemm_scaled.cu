// Products whose epilogue works on the accumulator as it comes out of TMEM, in two families of tiles on CTA PAIRS:
//
//   int8_scaled_mm    C[m][n] = s_a[m] s_b[n] sum_k a[m][k] b[n][k] + bias[n]     8-bit integers, exact sums in 32-bit integers
//   linear_logprobs   lse[m] = log sum_v exp l[m][v], logprob[m] = l[m][target[m]] - lse[m],  l = x w^T (8-bit: with both scales),
//                     without l ever reaching memory: a tile leaves (maximum, sum of exponentials) per token, a second kernel joins
//                     the tiles of a token
//
// 8-bit operands take tcgen05.mma kind::i8, whose instruction covers 32 bytes of K as kind::f16's does, at the same rate: a k-block
// is 128 bytes of a row in either, and one pipeline serves both.
//
// Tokens on N (few_tokens_kernel): D[256 weight rows x n tokens] = W A^T, n a multiple of 32 up to 256.  A cluster of 2 S CTAs has one
// tile, pair s the k-blocks [s kb / S, (s + 1) kb / S); pairs leave their sums in their own idle ring, and after a cluster barrier each
// adds all of them for its share of the tokens.  Sums of integers have no order, so nothing depends on S.  Two such CTAs share an SM
// (their rings together 200 KB in flight): one's start and end run under the other's stream.
// Tokens on M (many_tokens_kernel): 256 tokens x 256 columns, persistent, two accumulators: a tile's epilogue runs under the next
// tile's MMAs.
#include <cuda.h>
#include <atomic>

#include "common.cuh"
#include "pair.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace spd {

enum GemmKind { kInt8 = 0, kKindBf16 = 1, kKindF16 = 2 };
enum GemmEnd { kScaled = 0, kLogprob = 1 };

constexpr int kGsBlock = 128;                   // bytes of K in a k-block
constexpr int kGsHalf = 128 * kGsBlock;         // 128 rows of one operand
constexpr int kGsMaxSmem = 232448;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Instruction descriptor: sums in 32-bit integers of signed 8-bit operands, or in fp32 of 16-bit ones; both operands K-major.
template <int kKind>
__device__ __forceinline__ constexpr uint32_t gs_idesc(uint32_t M, uint32_t N) {
  return (kKind == kInt8 ? (2u << 4) | (1u << 7) | (1u << 10) : kKind == kKindBf16 ? (1u << 4) | (1u << 7) | (1u << 10) : 1u << 4) |
         ((N >> 3) << 17) | ((M >> 4) << 24);
}
template <int kKind>
__device__ __forceinline__ void gs_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kKind == kInt8)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    umma_ss_2cta(d, a, b, idesc, accumulate);
}
template <int kKind>
__device__ __forceinline__ float gs_value(uint32_t r) {
  return kKind == kInt8 ? static_cast<float>(static_cast<int>(r)) : __uint_as_float(r);
}

// All threads of the cluster are here; nothing that they wrote is meant to be seen.  (With release semantics the barrier waits for
// every store to global memory that is still on its way: 0.3 us of a short product.)
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

struct ScaledParams {
  void* out;           // kScaled: [m_rows, n_cols]
  int64_t ldc;
  const void* bias;    // [n_cols] or null
  const float* sa;     // a token's scale (8-bit operands)
  const float* sb;     // a weight row's
  float2* part;        // kLogprob: [tiles][m_rows] (maximum, sum of exponentials over it)
  float* hit;          // [m_rows]: the target's logit
  const int64_t* target;
  int n_cols, m_rows;
  int kblocks;
  int tok_tiles, n;    // tokens on N: token tiles, MMA columns of each
  int accs;            // accumulators that take k-blocks in turn (16-bit operands)
  int stages, slot;
  int to_l2;           // k-blocks of weights behind the ring's that a CTA asks into L2
  int x_tiles, y_tiles, panel;             // tokens on M
  uint64_t by_panel, by_width, by_last;    // reciprocals of a panel's tiles, of its width and the last one's (see quotient)
  int early;           // the weights are older than the kernel before this one: the first of them are fetched before it has ended
  unsigned* wait_expired;
};

// (maximum, sum of 2^((v - maximum) log2 e)) of values taken in, in fp32.  An infinite maximum counts as 0: a sum over nothing but
// -inf stays 0, one with +inf becomes inf, and NaN stays NaN, as in the formula.
struct LogSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ static float base(float m) { return fabsf(m) == INFINITY ? 0.f : m * kLog2e; }
  __device__ __forceinline__ void join(float m2, float s2) {
    const float t = fmaxf(m, m2), b = base(t);
    s = (s == 0.f ? 0.f : s * fast_exp2(base(m) - b)) + (s2 == 0.f ? 0.f : s2 * fast_exp2(base(m2) - b));
    m = t;
  }
};

// ------------------------------------------------------------------------------------------------
// tokens on N
// ------------------------------------------------------------------------------------------------
constexpr int kFewThreads = 192;  // warps 0-3: epilogue, 4: TMA, 5: MMA and TMEM
constexpr int kFewStages = 12;    // at most
constexpr int kFewFixed = 1024 + 256 + 2048;  // alignment, barriers, a scale and a target for each token
constexpr int kMaxSplit = 4;

// TMEM columns of a CTA, 256 at most: CTAs with tokens on N take at least half of the SM's shared memory (kHalfSmem), CTAs with tokens
// on M, which take all columns, all of it.  So whatever of these are on an SM together never wait for one another's columns: a CTA
// that did, while its peer holds another SM's, could close a circle of waits.
__host__ __device__ constexpr int few_columns(int cols) { return cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : 256; }

__device__ __forceinline__ int4 ld_cluster_s32x4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// The maximum (kMax) or sum over the warp's 32 lanes of 32 values each: lane t gets that of value t.
template <bool kMax>
__device__ __forceinline__ float warp_reduce_32(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const float keep = up ? v[j + o] : v[j], send = up ? v[j] : v[j + o];
      const float got = __shfl_xor_sync(0xffffffffu, send, o);
      v[j] = kMax ? fmaxf(keep, got) : keep + got;
    }
  }
  return v[0];
}

template <int kKind, int kEnd, typename T>
__global__ void __launch_bounds__(kFewThreads, 2)
few_tokens_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmO,
                  const ScaledParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.stages * p.slot);  // [stages]  (the leaders' are the live ones)
  uint64_t* empty = full + kFewStages;
  uint64_t* tfull = empty + kFewStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* tok_scale = reinterpret_cast<float*>(smem + p.stages * p.slot + 256);  // [256]
  int* tok_target = reinterpret_cast<int*>(tok_scale + 256);                    // [256]: row of this CTA, or none
  float2* share = reinterpret_cast<float2*>(smem);                              // [4][256], when the ring is idle

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank(), rank = crank & 1, leader = crank & ~1u;
  const int S = static_cast<int>(cluster_nctarank() >> 1), s = static_cast<int>(crank >> 1);
  const int tile = blockIdx.x / (2 * S), wt = tile / p.tok_tiles, tt = tile - wt * p.tok_tiles;
  const int kb0 = s * p.kblocks / S, kb1 = (s + 1) * p.kblocks / S;
  const int accs = kKind == kInt8 ? 1 : p.accs, half = p.n >> 1, tmem_cols = few_columns(p.n * accs);
  const int tok_base = tt * p.n, tokens = min(p.n, p.m_rows - tok_base);
  const int row_base = wt * 256 + static_cast<int>(rank) * 128;

  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmA);
    *dead = 0;
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(tfull, 1);
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc_2cta(tmem_slot, tmem_cols);
    tmem_relinquish_2cta();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the pair's barriers exist before any cross-CTA signal
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  griddep_launch_dependents();

  if (warp == 4) {
    if (elect_one()) {
      const uint32_t lead_full0 = map_to_rank(smem_u32(full), leader);
      const uint32_t bytes = 2 * (kGsHalf + half * kGsBlock);
      auto load_w = [&](int stage, int kb) {
        tma_load_2d_2cta(smem + stage * p.slot, &tmW, lead_full0 + stage * 8, kb * (kGsBlock / 2), row_base,
                         p.tok_tiles > 1 ? kEvictNormal : kEvictFirst);
      };
      const int ahead = min(p.stages, kb1 - kb0);
      if (!p.early) griddep_wait();
      for (int i = 0; i < ahead; ++i) {
        if (rank == 0) mbar_expect_tx(&full[i], bytes);
        load_w(i, kb0 + i);
      }
      const int asked = row_base < p.n_cols ? min(kb1, kb0 + ahead + p.to_l2) : 0;
      for (int kb = kb0 + ahead; kb < asked; ++kb) tma_prefetch_2d(&tmW, kb * (kGsBlock / 2), row_base);
      if (p.early) griddep_wait();
      int stage = 0, phase = 0;
      const int a_row = tok_base + static_cast<int>(rank) * half;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb - kb0 >= ahead) {
          mbar_wait_bounded(&empty[stage], phase ^ 1, dead);
          if (rank == 0) mbar_expect_tx(&full[stage], bytes);
          load_w(stage, kb);
        }
        tma_load_2d_2cta(smem + stage * p.slot + kGsHalf, &tmA, lead_full0 + stage * 8, kb * (kGsBlock / 2), a_row, kEvictLast);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    griddep_wait();  // (the tokens come behind it; a bounded wait for them starts there)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = gs_idesc<kKind>(256, p.n);
      const uint16_t both = static_cast<uint16_t>(0b11 << leader);
      int stage = 0, phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait_bounded(&full[stage], phase, dead);
        tc_fence_after_sync();
        const uint32_t wa = smem_u32(smem + stage * p.slot), aa = wa + kGsHalf;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          gs_mma<kKind>(tmem + ((kb - kb0) & (accs - 1)) * p.n, umma_desc_sw128(wa + k * 32, 16, 1024),
                        umma_desc_sw128(aa + k * 32, 16, 1024), idesc, (kb - kb0 >= accs || k > 0) ? 1u : 0u);
        umma_commit_2cta_mc(&empty[stage], both);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      umma_commit_2cta_mc(tfull, both);
    }
    __syncwarp();
  }
  if (warp < 4) {
    griddep_wait();  // the tokens' scales and what is written from here on
    const int row = warp * 32 + lane;
    const int64_t col = row_base + row;
    const bool have = col < p.n_cols;
    const float sb = kKind == kInt8 && have ? p.sb[col] : 1.f;
    float bias = 0.f;
    if constexpr (kEnd == kScaled) {
      if (p.bias && have) bias = to_f32<T>(reinterpret_cast<const T*>(p.bias)[col]);
    }
    for (int t = threadIdx.x; t < p.n; t += 128) {
      tok_scale[t] = kKind == kInt8 && t < tokens ? p.sa[tok_base + t] : 1.f;
      if constexpr (kEnd == kLogprob) {
        const int64_t at = t < tokens ? p.target[tok_base + t] : -1;
        tok_target[t] = at >= row_base && at < min(row_base + 128, p.n_cols) ? static_cast<int>(at - row_base) : -1;
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    mbar_wait_bounded(tfull, 0, dead);  // every MMA of the pair is done: both rings are idle
    tc_fence_after_sync();
    const uint32_t taddr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
#pragma unroll 1
    for (int c = 0; c < tokens; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(taddr + c, r);
      tmem_ld_wait();
      float sa[32];  // read before the first store: a load between two stores to shared memory waits for its turn, 1 us a chunk
      auto scales = [&]() {
#pragma unroll
        for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(sa + j) = *reinterpret_cast<const float4*>(tok_scale + c + j);
      };
      if constexpr (kEnd == kScaled) {
        if (S > 1) {
          uint32_t* part = reinterpret_cast<uint32_t*>(smem) + row;
#pragma unroll
          for (int j = 0; j < 32; ++j) part[(c + j) * 128] = r[j];
        } else {
          // 64 columns of 32 tokens as the copy's box has them: 16 bytes i of token j at i ^ (j & 7).  Every 32 tokens leave by TMA
          // while the next are scaled: against stores when all are there, 777 x 5000 x 1360 11.1 -> 10.7 us, 700 x 4096 x 256
          // 6.2 -> 5.7, 1500 x 4096 x 4096 20.6 -> 20.2; 2 x 24632 x 144 3.6 -> 3.7.
          uint8_t* box = smem + c * 256 + (warp >> 1) * 4096;
          const int at = (row & 63) * 2;
          scales();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            *reinterpret_cast<T*>(box + j * 128 + (at ^ ((j & 7) * 16))) = from_f32<T>(fmaf(gs_value<kKind>(r[j]) * sa[j], sb, bias));
          fence_proxy_async_smem();
          asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp >> 1)) : "memory");
          if ((warp & 1) == 0 && lane == 0 && col < p.n_cols) {
            tma_store_2d(&tmO, box, static_cast<int>(col), tok_base + c);
            bulk_commit_group();
          }
        }
      } else {
        float v[32], e[32];
        if constexpr (kKind == kInt8) {
          scales();
        } else {
          for (int a = 1; a < accs; ++a) {
            uint32_t more[32];
            tmem_ld_32x32b_x32(taddr + a * p.n + c, more);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(more[j]));
          }
        }
        int hit[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) *reinterpret_cast<int4*>(hit + j) = *reinterpret_cast<const int4*>(tok_target + c + j);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          v[j] = kKind == kInt8 ? gs_value<kKind>(r[j]) * sa[j] * sb : __uint_as_float(r[j]);
          if (hit[j] == row) p.hit[tok_base + c + j] = v[j];
          if (!have) v[j] = -INFINITY;
          e[j] = v[j];
        }
        const float top = warp_reduce_32<true>(e, lane);  // of token c + lane
        const float base = LogSum::base(top);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = fast_exp2(fmaf(v[j], kLog2e, -__shfl_sync(0xffffffffu, base, j)));
        const float sum = warp_reduce_32<false>(v, lane);
        share[warp * 256 + c + lane] = make_float2(top, sum);
      }
    }
    tc_fence_before_sync();
    if constexpr (kEnd == kScaled) {
      if (S == 1 && lane == 0) bulk_wait_group0();
    } else {
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int t = threadIdx.x; t < tokens; t += 128) {
        LogSum all;
#pragma unroll
        for (int w = 0; w < 4; ++w) all.join(share[w * 256 + t].x, share[w * 256 + t].y);
        p.part[static_cast<int64_t>(wt * 2 + rank) * p.m_rows + tok_base + t] = make_float2(all.m, all.s);
      }
    }
  }
  if (kEnd == kScaled && S > 1) {
    if (warp >= 4) griddep_wait();  // they write C too
    __syncwarp();
    cluster_sync_all();  // all pairs' sums are in place
    const int tok0 = s * p.n / S, tok1 = min((s + 1) * p.n / S, tokens);
    const uint32_t base = smem_u32(smem);
    uint32_t src[kMaxSplit];
#pragma unroll
    for (int i = 0; i < kMaxSplit; ++i) src[i] = map_to_rank(base, (i < S ? i : 0) * 2 + rank);
    const int col = row_base + lane * 4;
    if (col < p.n_cols) {
      const float4 sb = make_float4(p.sb[col], p.sb[col + 1], p.sb[col + 2], p.sb[col + 3]);
      float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.bias) {
        const T* b = reinterpret_cast<const T*>(p.bias) + col;
        bias = make_float4(to_f32<T>(b[0]), to_f32<T>(b[1]), to_f32<T>(b[2]), to_f32<T>(b[3]));
      }
#pragma unroll 4
      for (int t = tok0 + warp; t < tok1; t += kFewThreads / 32) {
        int4 f[kMaxSplit];
#pragma unroll
        for (int i = 0; i < kMaxSplit; ++i)
          if (i < S) f[i] = ld_cluster_s32x4(src[i] + (t * 128 + lane * 4) * 4);
        int4 v = f[0];
#pragma unroll
        for (int i = 1; i < kMaxSplit; ++i)
          if (i < S) {
            v.x += f[i].x;
            v.y += f[i].y;
            v.z += f[i].z;
            v.w += f[i].w;
          }
        const float sa = tok_scale[t];
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + static_cast<int64_t>(tok_base + t) * p.ldc + col) =
            make_uint2(pack2<T>(fmaf(static_cast<float>(v.x) * sa, sb.x, bias.x), fmaf(static_cast<float>(v.y) * sa, sb.y, bias.y)),
                       pack2<T>(fmaf(static_cast<float>(v.z) * sa, sb.z, bias.z), fmaf(static_cast<float>(v.w) * sa, sb.w, bias.w)));
      }
    }
  }

  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (*dead) {
    wait_drain();
    if (threadIdx.x == 0) wait_report(p.wait_expired);
  }
  cluster_sync_relaxed();  // nobody leaves while a peer may still read its shared memory or signal its barriers
  if (warp == 5) tmem_dealloc_2cta(tmem, tmem_cols);
}

// ------------------------------------------------------------------------------------------------
// tokens on M
// ------------------------------------------------------------------------------------------------
constexpr int kManyThreads = 256;  // warp 0: TMA, 1: MMA, 2: TMEM, 4-7: epilogue
constexpr int kManyStages = 6;
constexpr int kManyRing = kManyStages * 2 * kGsHalf;
constexpr int kManyStage = 32 * 128;  // 64 columns of a warp's 32 rows
constexpr int kManySmem = kManyRing + 4 * kManyStage + 2 * 256 * 8 + 256 + 1024;
static_assert(kManySmem <= kGsMaxSmem, "shared memory of a CTA");  // (a launch asks for kGsMaxSmem: see few_columns)

// n / d of non-negative n, d < 2^31 for a reciprocal ceil(2^64 / d), exact (it is less than 1 too large, and n d < 2^64); 0 stands for
// 2^64.  The compiler's division took an epilogue warp 150 clk, four of them a tile.
__host__ inline uint64_t reciprocal(int d) { return ~uint64_t{0} / d + 1; }
__device__ __forceinline__ int quotient(int n, uint64_t reciprocal) {
  return reciprocal ? static_cast<int>(__umul64hi(static_cast<uint64_t>(n), reciprocal)) : n;
}

__device__ __forceinline__ void many_tile(const ScaledParams& p, int tile, int& xt, int& yt) {
  const int pn = quotient(tile, p.by_panel), r = tile - pn * p.x_tiles * p.panel;
  const int y0 = pn * p.panel, whole = y0 + p.panel <= p.y_tiles, q = whole ? p.panel : p.y_tiles - y0;
  xt = quotient(r, whole ? p.by_width : p.by_last);
  yt = y0 + r - xt * q;
}

// One thread of each CTA: its 128 token rows and 128 weight rows of every k-block; the leader's barrier counts both CTAs' bytes.
__device__ __forceinline__ void many_load(const CUtensorMap& tmA, const CUtensorMap& tmW, const ScaledParams& p, uint8_t* smem,
                                          uint64_t* full, uint64_t* empty, uint32_t rank, int pair, int npairs, volatile int* dead) {
  int stage = 0, phase = 0;
  const uint32_t lead_full0 = map_to_rank(smem_u32(full), 0);
  for (int tile = pair; tile < p.x_tiles * p.y_tiles; tile += npairs) {
    int xt, yt;
    many_tile(p, tile, xt, yt);
    const int a_row = xt * 256 + static_cast<int>(rank) * 128, w_row = yt * 256 + static_cast<int>(rank) * 128;
    for (int kb = 0; kb < p.kblocks; ++kb) {
      mbar_wait_bounded(&empty[stage], phase ^ 1, dead);
      if (rank == 0) mbar_expect_tx(&full[stage], 4 * kGsHalf);
      uint8_t* slot = smem + stage * 2 * kGsHalf;
      tma_load_2d_2cta(slot, &tmA, lead_full0 + stage * 8, kb * (kGsBlock / 2), a_row, kEvictNormal);
      tma_load_2d_2cta(slot + kGsHalf, &tmW, lead_full0 + stage * 8, kb * (kGsBlock / 2), w_row, kEvictNormal);
      if (++stage == kManyStages) { stage = 0; phase ^= 1; }
    }
  }
}

// One thread of the leader: the MMAs of every tile, `chunk` k-blocks into either accumulator in turn.
template <int kKind>
__device__ __forceinline__ void many_multiply(const ScaledParams& p, uint8_t* smem, uint64_t* full, uint64_t* empty, uint64_t* tfull,
                                              uint64_t* tempty, uint32_t tmem, int pair, int npairs, int chunk, volatile int* dead) {
  constexpr uint32_t idesc = gs_idesc<kKind>(256, 256);
  int stage = 0, phase = 0, n = 0;
  for (int tile = pair; tile < p.x_tiles * p.y_tiles; tile += npairs)
    for (int kb0 = 0; kb0 < p.kblocks; kb0 += chunk, ++n) {
      const int as = n & 1, kb1 = min(kb0 + chunk, p.kblocks);
      mbar_wait_bounded(&tempty[as], ((n >> 1) & 1) ^ 1, dead);  // both CTAs have drained this accumulator
      tc_fence_after_sync();
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait_bounded(&full[stage], phase, dead);
        tc_fence_after_sync();
        const uint32_t aa = smem_u32(smem + stage * 2 * kGsHalf), wa = aa + kGsHalf;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          gs_mma<kKind>(tmem + as * 256, umma_desc_sw128(aa + k * 32, 16, 1024), umma_desc_sw128(wa + k * 32, 16, 1024), idesc,
                        (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit_2cta_mc(&empty[stage], 0b11);
        if (++stage == kManyStages) { stage = 0; phase ^= 1; }
      }
      umma_commit_2cta_mc(&tfull[as], 0b11);
    }
}

template <typename T>
__global__ void __launch_bounds__(kManyThreads, 1)
many_tokens_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ CUtensorMap tmO, const ScaledParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sOut = smem + kManyRing;                                          // kManyStage per epilogue warp
  float2* cols = reinterpret_cast<float2*>(sOut + 4 * kManyStage);           // [2][256] (scale, bias) of a tile's columns
  uint64_t* full = reinterpret_cast<uint64_t*>(cols + 512);                  // [stages]  (the leader's are the live ones)
  uint64_t* empty = full + kManyStages;                                      // [stages]
  uint64_t* tfull = empty + kManyStages;                                     // [2]
  uint64_t* tempty = tfull + 2;                                              // [2]       (the leader's)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1, num_tiles = p.x_tiles * p.y_tiles;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    *dead = 0;
  }
  if (warp == 1 && lane == 0) {
    for (int i = 0; i < kManyStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 8);
    }
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc_2cta(tmem_slot, 512);
    tmem_relinquish_2cta();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA signal
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();

  if (warp == 0) {
    if (elect_one()) many_load(tmA, tmW, p, smem, full, empty, rank, pair, npairs, dead);
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) many_multiply<kInt8>(p, smem, full, empty, tfull, tempty, tmem, pair, npairs, p.kblocks, dead);
  } else if (warp >= 4) {
    const int q = warp & 3, et = threadIdx.x - 128;
    uint8_t* stage = sOut + q * kManyStage;
    const uint32_t lead_tempty0 = map_to_rank(smem_u32(tempty), 0);
    // An epilogue shorter than this bounds products of few k-blocks (256 x 256 results: 9000 clk a tile at first, five k-blocks of
    // MMAs take 2700).  So: a tile's scales and biases are fetched a tile ahead (1000 clk; the bias as it is in memory, to convert
    // it would wait for it), the accumulator is given back by an arrival that does not wait for the stores (a releasing one: 1700),
    // and the results leave by TMA, a warp's 64 columns while it works on the next.  8000 x 4096 x 256 34.5 -> 25.6 us,
    // 8192 x 4096 x 1024 40.7 -> 31.2, 6061 x 14984 x 528 104 -> 83 (of which 20 for the stores; to fill such an output takes 49),
    // 4099 x 6144 x 4096 68.3 -> 67.5.  Not taken: eight warps (25.1, 30.6, 84, 67.7); integers to fp32 by halves for every second
    // value, for the conversions' rate of 16 a clk (28.5, 33.6, 86).
    float sb[2], sa = 1.f;
    T bias[2];
    auto fetch = [&](int tile) {
      int xt, yt;
      many_tile(p, tile, xt, yt);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = yt * 256 + et + i * 128;
        const bool in = c < p.n_cols;
        sb[i] = in ? p.sb[c] : 0.f;
        bias[i] = in && p.bias ? reinterpret_cast<const T*>(p.bias)[c] : from_f32<T>(0.f);
      }
      const int64_t m = static_cast<int64_t>(xt) * 256 + rank * 128 + q * 32 + lane;
      sa = m < p.m_rows ? p.sa[m] : 1.f;
    };
    if (pair < num_tiles) fetch(pair);
    int n = 0;
    for (int tile = pair; tile < num_tiles; tile += npairs, ++n) {
      int xt, yt;
      many_tile(p, tile, xt, yt);
      const int as = n & 1, n0 = yt * 256, columns = min(256, p.n_cols - n0);
      const int64_t m0 = static_cast<int64_t>(xt) * 256 + rank * 128 + q * 32;
      const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.m_rows - m0));
      const float2* col = cols + as * 256;
      const float row_scale = sa;
#pragma unroll
      for (int i = 0; i < 2; ++i) cols[as * 256 + et + i * 128] = make_float2(sb[i], to_f32<T>(bias[i]));
      // (one barrier a tile: a warp that is a tile ahead writes the other half, and cannot get two ahead)
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (tile + npairs < num_tiles) fetch(tile + npairs);
      mbar_wait_bounded(&tfull[as], (n >> 1) & 1, dead);
      tc_fence_after_sync();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + as * 256;
      auto values = [&](int c, const uint32_t (&r)[32], uint4 (&out)[4]) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float4 f = *reinterpret_cast<const float4*>(col + c + j);
          v[j] = fmaf(gs_value<kInt8>(r[j]) * row_scale, f.x, f.y);
          v[j + 1] = fmaf(gs_value<kInt8>(r[j + 1]) * row_scale, f.z, f.w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          out[i] = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                              pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
      };
#pragma unroll 1
      for (int c = 0; c < columns; c += 64) {
        uint32_t r0[32], r1[32];
        uint4 o[2][4];
        tmem_ld_32x32b_x32(taddr + c, r0);
        tmem_ld_32x32b_x32(taddr + c + 32, r1);
        tmem_ld_wait();
        values(c, r0, o[0]);
        values(c + 32, r1, o[1]);
        if (c + 64 >= columns) tc_fence_before_sync();
        if (lane == 0) bulk_wait_group_read0();  // the copy of the last 64 columns has read them
        __syncwarp();
        if (c + 64 >= columns && lane == 0) mbar_arrive_remote_relaxed(lead_tempty0 + as * 8);  // the accumulator is free
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) * 16)) = o[i >> 2][i & 3];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && rows > 0) {
          tma_store_2d(&tmO, stage, n0 + c, static_cast<int>(m0));
          bulk_commit_group();
        }
      }
    }
    if (lane == 0) bulk_wait_group0();
  }

  __syncwarp();  // the warps of the elected lanes come together before the barriers, which count whole warps
  griddep_launch_dependents();
  tc_fence_before_sync();
  __syncthreads();
  if (*dead) {
    wait_drain();
    if (threadIdx.x == 0) wait_report(p.wait_expired);
  }
  cluster_sync_relaxed();  // the peer may still read this CTA's shared memory / signal its barriers
  if (warp == 2) tmem_dealloc_2cta(tmem, 512);
}

// Log-probabilities with tokens on M: 256 tokens x 256 vocabulary rows.  Eight warps take the accumulator, a lane with a token, its
// 128 columns of one half kept in registers as fp32.  The tensor cores cut what does not fit behind the sum of 16-bit products, always
// towards zero, and a long row adds that up (K = 4096: 1.1e-6 of the result); so a sum is taken out of TMEM after every 16 k-blocks and
// added up in registers, while the other accumulator takes the next ones: a tenth of the error, no time (16 k-blocks take the MMAs
// 8192 clk, taking 128 columns out 400).  8-bit sums are exact and come out once.
constexpr int kLogThreads = 320;  // warp 0: TMA, 1: MMA and TMEM, 2-9: epilogue
constexpr int kLogChunk = 16;     // k-blocks
static_assert(kManyRing + 2 * 256 * 4 + 256 + 1024 <= kGsMaxSmem, "shared memory of a CTA");

template <int kKind>
__global__ void __launch_bounds__(kLogThreads, 1)
many_logprobs_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const ScaledParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* cols = reinterpret_cast<float*>(smem + kManyRing);         // [2][256] scales of a tile's vocabulary rows
  uint64_t* full = reinterpret_cast<uint64_t*>(cols + 512);         // [stages]  (the leader's are the live ones)
  uint64_t* empty = full + kManyStages;                             // [stages]
  uint64_t* tfull = empty + kManyStages;                            // [2]
  uint64_t* tempty = tfull + 2;                                     // [2]       (the leader's)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1, num_tiles = p.x_tiles * p.y_tiles;
  const int chunk = kKind == kInt8 ? p.kblocks : kLogChunk;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    *dead = 0;
    for (int i = 0; i < kManyStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 16);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_2cta(tmem_slot, 512);
    tmem_relinquish_2cta();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA signal
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();

  if (warp == 0) {
    if (elect_one()) many_load(tmA, tmW, p, smem, full, empty, rank, pair, npairs, dead);
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) many_multiply<kKind>(p, smem, full, empty, tfull, tempty, tmem, pair, npairs, chunk, dead);
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2, et = threadIdx.x - 64;
    const uint32_t lead_tempty0 = map_to_rank(smem_u32(tempty), 0);
    int n = 0, turn = 0;
    for (int tile = pair; tile < num_tiles; tile += npairs, turn ^= 1) {
      int xt, yt;
      many_tile(p, tile, xt, yt);
      const int n0 = yt * 256 + half * 128;
      const int64_t m0 = static_cast<int64_t>(xt) * 256 + rank * 128 + q * 32;
      const bool have = m0 + lane < p.m_rows;
      const float* col = cols + turn * 256 + half * 128;
      float sa = 1.f;
      if constexpr (kKind == kInt8) {
        cols[turn * 256 + et] = yt * 256 + et < p.n_cols ? p.sb[yt * 256 + et] : 0.f;
        // (one barrier a tile: a warp that is a tile ahead writes the other half, and cannot get two ahead)
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (have) sa = p.sa[m0 + lane];
      }
      const int64_t target = have ? p.target[m0 + lane] - n0 : -1;
      float v[128];
      for (int kb0 = 0; kb0 < p.kblocks; kb0 += chunk, ++n) {
        const int as = n & 1;
        mbar_wait_bounded(&tfull[as], (n >> 1) & 1, dead);
        tc_fence_after_sync();
        const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + as * 256 + half * 128;
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(taddr + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) v[c + j] = kb0 == 0 ? gs_value<kKind>(r[j]) : v[c + j] + gs_value<kKind>(r[j]);
        }
        tc_fence_before_sync();
        __syncwarp();
        // (a releasing arrival would wait for the last tile's stores: 4000 x 50272 x 768, 8 bits 176 us instead of 153)
        if (lane == 0) mbar_arrive_remote_relaxed(lead_tempty0 + as * 8);
      }
      const int valid = p.n_cols - n0;
      if constexpr (kKind == kInt8) {
#pragma unroll
        for (int j = 0; j < 128; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(col + j);
          v[j] = v[j] * sa * f.x;
          v[j + 1] = v[j + 1] * sa * f.y;
          v[j + 2] = v[j + 2] * sa * f.z;
          v[j + 3] = v[j + 3] * sa * f.w;
        }
      }
      if (target >= 0 && target < 128 && target < valid) {
#pragma unroll
        for (int j = 0; j < 128; ++j)
          if (target == j) p.hit[m0 + lane] = v[j];
      }
      if (valid < 128) {
#pragma unroll
        for (int j = 0; j < 128; ++j)
          if (j >= valid) v[j] = -INFINITY;
      }
      float top[4] = {v[0], v[1], v[2], v[3]}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 4; j < 128; ++j) top[j & 3] = fmaxf(top[j & 3], v[j]);
      top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      const float base = LogSum::base(top[0]);
#pragma unroll
      for (int j = 0; j < 128; ++j) sum[j & 3] += fast_exp2(fmaf(v[j], kLog2e, -base));
      if (have) p.part[static_cast<int64_t>(yt * 2 + half) * p.m_rows + m0 + lane] = make_float2(top[0], (sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
  }

  __syncwarp();  // the warps of the elected lanes come together before the barriers, which count whole warps
  griddep_launch_dependents();
  tc_fence_before_sync();
  __syncthreads();
  if (*dead) {
    wait_drain();
    if (threadIdx.x == 0) wait_report(p.wait_expired);
  }
  cluster_sync_relaxed();  // the peer may still read this CTA's shared memory / signal its barriers
  if (warp == 1) tmem_dealloc_2cta(tmem, 512);
}

// ------------------------------------------------------------------------------------------------
// the tiles of a token joined
// ------------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 256;

// `width` tokens of a CTA beside one another (1, 2 or 4: 32 bytes of every tile), kJoinThreads / width shares of the tiles for each.
// Bound by the latency of its loads, so a share is short and takes four tiles at a time (32 tokens, 1002 parts: 30 us with 8 shares a
// token).
__global__ void __launch_bounds__(kJoinThreads)
logprob_join_kernel(float* logprobs, float* lse, const float2* part, const float* hit, const int64_t* target, int tokens, int tiles, int vocab, int width) {
  __shared__ float2 sums[kJoinThreads];
  griddep_launch_dependents();
  griddep_wait();
  const int t = blockIdx.x * width + (threadIdx.x & (width - 1)), shares = kJoinThreads / width;
  LogSum all;
  if (t < tokens)
    for (int i = threadIdx.x / width; i < tiles; i += 4 * shares) {
      float2 f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = i + j * shares < tiles ? __ldcg(part + static_cast<int64_t>(i + j * shares) * tokens + t) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) all.join(f[j].x, f[j].y);
    }
  sums[threadIdx.x] = make_float2(all.m, all.s);
  for (int o = shares >> 1; o > 0; o >>= 1) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < o * width) {
      const float2 f = sums[threadIdx.x + o * width];
      all.join(f.x, f.y);
      sums[threadIdx.x] = make_float2(all.m, all.s);
    }
  }
  if (static_cast<int>(threadIdx.x) < width && t < tokens) {
    const float z = (LogSum::base(all.m) + log2f(all.s)) * kLn2;
    const int64_t at = target[t];
    lse[t] = z;
    logprobs[t] = at >= 0 && at < vocab ? __ldcg(hit + t) - z : 0.f;
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
// the kernel's limit of shared memory, once on every device
template <typename K>
static int allow_smem(K kern, std::atomic<uint64_t>& done) {
  int dev = 0;
  SPD_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    SPD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGsMaxSmem));
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  return 0;
}

template <typename K, typename... Args>
static int launch_pairs(K kern, std::atomic<uint64_t>& done, int ctas, int cluster, int threads, int smem, cudaStream_t stream,
                        const Args&... args) {
  if (int rc = allow_smem(kern, done)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  SPD_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  return 0;
}

// How a product is cut: token tiles and pairs of a tile for tokens on N, or tiles of 256 x 256 (tok_tiles 0).
struct ScaledPlan {
  int tok_tiles, split, smem;
};
constexpr int kHalfSmem = 113 * 1024;  // of a CTA that shares its SM with another

// Weights that a call with one tile of tokens asks into L2 behind what its rings hold, while it waits for the tokens and for the kernel
// before it: memory does not pause there.  us, without / 8, 16, 24 MB: 1 x 28672 x 4096 21.4 / 21.1, 20.7, 20.4; 1 x 4096 x 4096 5.8 / 5.5,
// 5.4, 5.5; 16 x 5120 x 5120 7.7 / 7.5, 7.3, 7.2; 40 x 4096 x 14336 14.4 / 14.3, 14.1, 14.3 (64 MB: 15.2); behind a kernel that leaves nothing
// to overlap 64 x 28672 x 4096 23.2 / 22.6, 21.9, 21.8, 1 x 8192 x 3584 9.8 / 9.9, 10.2, 10.2.  With several tiles of tokens it costs time:
// 256 x 6144 x 4096 10.8 / 11.5; so it does in a part of the SMs, which memory does not bound: a decode step of Llama-3-8B, 32 requests
// on 72 SMs 4.22 / 4.33 ms (on all of them 2.95 / 2.95).  Single lines asked for by the epilogue's warps: 21.1 instead of 20.7.
constexpr int kAheadInL2 = 16 << 20;

// Shared memory for the ring of a CTA with tokens on N: `slots` of what it takes for n tokens
static int few_slots(int n, int smem) {
  const int slots = (smem - kFewFixed) / (kGsHalf + n / 2 * kGsBlock);
  return slots < kFewStages ? slots : kFewStages;
}

// Clusters of `ctas` CTAs, one CTA an SM, that run at once as the driver says of a stream, and how many of them to reckon with
// (gemm_pair_split.cu): a partition's SMs stand on the chip as they do, which their number does not tell.
int clusters_found(int ctas, int sms, cudaStream_t stream);
int cluster_room(int ctas, int found, int sms);

// Clusters of 2 S CTAs that run at once, one CTA an SM or two.  The driver counts one CTA an SM, whatever a CTA takes of it, so two an SM are
// twice that at least; a cluster of 6 or 8 CTAs finds room where one of half as many fits, unless the SMs stand in small groups, which the
// two counts tell by being far apart.  Clusters of 4, 6, 8 with two CTAs an SM that ran at once (CTAs noted when they began) / twice the
// driver's count / its count for half the CTAs: whole B200 71, 45, 33 / 66, 44, 30 / 74, 45, 33; 76 SMs 33, 21, 15 / 30, 18, 12 / 38, 21, 15;
// 72 36, 19, 18 / 36, 18, 18 / 36, 18, 18; 108 50, 30, 23 / 46, 26, 20 / 54, 30, 23; 52 18, 12, 9 / 18, 12, 6 / 26, 12, 9; 36 10, 4, 3 / 10, 4, 2 /
// 18, 6, 5.  One too many is a second round: 20 tiles of 6 CTAs, 16 x 5120 x 5120 on 72 SMs, 14.2 us, of 4 CTAs 9.1; 36 of 4 CTAs,
// 256 x 2304 x 8192 on 76, 22.2, 36 of 2 CTAs 15.8.  One too few costs less: 20 of 6, 64 x 5120 x 5120 on 76, 10.2, of 2 11.0.
struct Clusters {
  int sms;
  cudaStream_t stream;
  const int* found;  // the driver's answers for 1 - 8 CTAs where a caller has them, or null
  int at_once[kMaxSplit + 1][2];
  bool asked[kMaxSplit + 1][2];  // the others are as many as there are SMs for

  Clusters(int sms, cudaStream_t stream, const int* found) : sms(sms), stream(stream), found(found) {
    const bool whole = sms >= device_sm_count_cached();
    for (int S = 1; S <= kMaxSplit; ++S)
      for (int half = 0; half < 2; ++half) {
        at_once[S][half] = half ? sms / S : sms / (2 * S);
        asked[S][half] = S == 1;
        if (S > 1 && (found || whole)) ask(S, half);
      }
  }
  // (1 us of host time in a partition for each answer of the driver's)
  void ask(int S, int half) {
    at_once[S][half] = room(2 * S) * (half ? 2 : 1);
    if (half && S > 2) {
      const int more = room(S);
      if (more > at_once[S][half] && 4 * more <= 5 * at_once[S][half]) at_once[S][half] = more;
    }
    asked[S][half] = true;
  }
  int room(int ctas) const { return cluster_room(ctas, found ? found[ctas - 1] : clusters_found(ctas, sms, stream), sms); }
};

// Every form's time in us as fitted to 264 products (1 - 2000 tokens; 22 weights of 1024 x 2048 to 28672 x 4096, K from 144 to 14336),
// weights out of memory, in a row of such calls; the form chosen took 1.013 times the fastest one's time in the mean, 1.12 at most.
// Tokens on N, all tiles at once: a k-block of 128 bytes takes a pair 0.15 to 0.24 (half the ring: 1.65 times that), two pairs on an
// SM 0.09 to 0.29 each; the weights 8.6 GB/ms, and two thirds of that again for every further tile of tokens that reads them.  Where the
// next call's CTAs fit beside this one's, what their rings hold is on its way before this one ends: 0.4 of that share.  Then the
// epilogue, the pairs' sums, and what CTAs and tiles cost each other.  Tokens on M: 0.29 a k-block and 1 a tile, 2.8 at least, and the
// weights of a single row of tiles at 5.3 GB/ms.
// More tiles than run at once, one of tokens: 57344 x 8192 of 1 token 74 us (tokens on M 111), of 160 87 (104), 128256 x 4096 of 1 80 (131),
// of 100 94 (97), of 256 125 (105).
//
// By the driver's counts, and not by the share of the whole device's that a partition has ("one fewer" of 6 and 8 CTAs), us before / now:
// 76 SMs 16 x 4096 x 4096 13.5 / 7.5, 64 x 4096 x 14336 29.2 / 16.2, 256 x 1024 x 8192 20.3 / 10.3; 72 256 x 2304 x 8192 15.8 / 13.0;
// 108 1 x 3584 x 8192 14.8 / 8.5; 36 64 x 3584 x 8192 24.0 / 15.2; whole 640 x 2304 x 14336 22.5 / 20.3.  Of 284 products (5 partitions) none
// takes 4 % longer.
static ScaledPlan fastest_plan(int64_t M, int64_t N, int kblocks, const Clusters& clusters) {
  const int sms = clusters.sms;
  const int64_t w_tiles = (N + 255) / 256, waves = ((M + 255) / 256 * w_tiles + sms / 2 - 1) / (sms / 2);
  ScaledPlan plan{0, 1, 0};
  const double tile = 0.288 * kblocks + 1;
  double best = 6.4 + static_cast<double>(waves) * (tile > 2.8 ? tile : 2.8);
  const double pass = 128e-6 / 7.7 * static_cast<double>(N) * kblocks;
  if (M <= 256 && best < 6.4 + 1.45 * pass) best = 6.4 + 1.45 * pass;
  const int64_t units = (M + 31) / 32, fewest = (units + 7) / 8;
  for (int64_t t = fewest; t <= units && t <= fewest + 12 && (t == 1 || t * w_tiles <= sms); ++t) {
    const int n = static_cast<int>(32 * ((units + t - 1) / t));
    const double part = n / 256.0, weights = pass * (0.9 + 0.67 * static_cast<double>(t - 1));
    for (int S = 1; S <= kMaxSplit && (S == 1 || kblocks >= 4 * S); ++S)
      for (int smem : {kGsMaxSmem, kHalfSmem}) {
        const bool half = smem == kHalfSmem;
        const int slots = few_slots(n, smem);
        const int64_t ctas = t * w_tiles * 2 * S;
        const int64_t at_once = clusters.at_once[S][half];
        const bool several = t * w_tiles > at_once;
        if (several && (t > 1 || S > 1 || !half)) continue;
        if (slots * (kGsHalf + n / 2 * kGsBlock) < n * (S > 1 ? 512 : 256)) continue;
        const bool two = half && ctas > sms;
        const double kb = static_cast<double>(kblocks) / S, alone = kb * (0.15 + 0.085 * part) * (half ? 1.65 : 1),
                     shared = kb * (0.09 + 0.2 * part) * (two ? 2 : 1);
        double us = alone > shared ? alone : shared;
        if (us < weights) us = weights;
        if (ctas <= (half ? sms : sms / 2)) us *= 1 - 0.4 * (slots < kb ? slots / kb : 1);
        us += 2.7 + 2.7 * part * (two && S == 1 ? 0.9 : 1) + (S > 1 ? 0.3 + 3.7 * part : 0) + 0.25 * static_cast<double>(ctas) / sms +
              (t > 1 ? 0.3 : 0);
        if (several) {
          us = static_cast<double>((w_tiles + at_once - 1) / at_once) * (1.2 * shared + 2.7 + 5.3 * part);
          if (us < 1.22 * pass + 4) us = 1.22 * pass + 4;
        }
        if (us < best) {
          best = us;
          plan = ScaledPlan{static_cast<int>(t), S, smem};
        }
      }
  }
  return plan;
}

// The fastest of the forms that fit: the driver is asked only about those that would be it.
static ScaledPlan product_plan(int64_t M, int64_t N, int kblocks, Clusters clusters) {
  for (;;) {
    const ScaledPlan plan = fastest_plan(M, N, kblocks, clusters);
    const int half = plan.smem == kHalfSmem;
    if (clusters.asked[plan.split][half]) return plan;
    clusters.ask(plan.split, half);
  }
}

// 16-bit operands with tokens on N: k-blocks go to up to 8 accumulators in turn, as many as half of TMEM holds (see many_logprobs_kernel)
static int few_accumulators(int n, int kblocks) {
  int accs = 8;
  while (accs > 1 && (accs * n > 256 || accs > kblocks)) accs /= 2;
  return accs;
}

// The same for log-probabilities, whose epilogue with tokens on N is the longer one (it goes across lanes), and whose tiles take more
// than one wave: 144 calls (1 - 800 tokens; 128256 x 4096, 102400 x 2048, 32000 x 4096, 50272 x 768, 8192 x 2048, 1000 x 1024; 16 and 8 bits),
// 1.01 times the fastest form's time in the mean, 1.13 at most.
// Sums of 16-bit products stay with tokens on M where more than 32 k-blocks would come together in one accumulator: they are that much
// less exact (64 in one 1.4e-6 of the result, 32 7e-7, 16 4e-7).
static ScaledPlan logprob_plan(int64_t M, int64_t N, int kblocks, int sms, bool int8) {
  const int64_t w_tiles = (N + 255) / 256, pairs = sms / 2, waves = ((M + 255) / 256 * w_tiles + pairs - 1) / pairs;
  const double bytes = 128e-6 * static_cast<double>(N) * kblocks;
  ScaledPlan plan{0, 1, 0};
  double best = 8.8 + static_cast<double>(waves) * (0.337 * kblocks + 1.65);
  const int64_t units = (M + 31) / 32, fewest = (units + 7) / 8;
  for (int64_t t = fewest; t <= units && t <= fewest + 12; ++t) {
    const int n = static_cast<int>(32 * ((units + t - 1) / t));
    if (!int8 && kblocks > 32 * few_accumulators(n, kblocks)) continue;
    const double part = n / 256.0, tiles = static_cast<double>(t * w_tiles);
    const double one = 0.4 + (tiles > pairs ? kblocks * (0.308 + 0.316 * part) + 17.9 * part : kblocks * (0.131 + 0.694 * part));
    double us = tiles > 2 * pairs ? one * tiles / static_cast<double>(2 * pairs) : one;
    us = 6.2 + (us > bytes / 6.84 ? us : bytes / 6.84);
    if (us < best) {
      best = us;
      plan = ScaledPlan{static_cast<int>(t), 1, kHalfSmem};
    }
  }
  return plan;
}

// ring slots for tokens on N; the sums (of one pair: the results) have to fit the ring
static int few_ring(ScaledParams& p, const ScaledPlan& plan) {
  p.slot = kGsHalf + p.n / 2 * kGsBlock;
  const int fit = few_slots(p.n, plan.smem), most = (p.kblocks + plan.split - 1) / plan.split;
  const int sums = (p.n * (plan.split > 1 ? 512 : 256) + p.slot - 1) / p.slot;
  p.stages = fit;
  if (p.stages > most) p.stages = most < sums ? sums : most;
  SPD_REQUIRE(p.stages >= 1 && p.stages >= sums && p.stages <= fit, SPD_E_SHAPE, "a ring of %d slots for %d", fit, sums);
  return 0;
}

template <int kKind, int kEnd, typename T>
static int scaled_product(const void* a, const void* w, int64_t M, int64_t N, int64_t kbytes, int64_t a_stride, int64_t w_stride,
                          ScaledParams p, const ScaledPlan& plan, int sms, cudaStream_t stream) {
  // rows as 16-bit elements: the copies move bytes
  CUtensorMap ta, tw;
  SPD_REQUIRE((M + 31) / 32 * ((N + 255) / 256) <= (1 << 28), SPD_E_SHAPE, "%lld x %lld are too many tiles for one call", (long long)M,
              (long long)N);
  p.n_cols = static_cast<int>(N);
  p.m_rows = static_cast<int>(M);
  p.kblocks = static_cast<int>((kbytes + kGsBlock - 1) / kGsBlock);
  if (int rc = wait_flag(&p.wait_expired)) return rc;
  p.tok_tiles = plan.tok_tiles;
  if (plan.tok_tiles > 0) {
    p.n = static_cast<int>(32 * (((M + 31) / 32 + plan.tok_tiles - 1) / plan.tok_tiles));
    if (int rc = few_ring(p, plan)) return rc;
    if (int rc = make_tmap_2d_sw128(&tw, w, N, kbytes / 2, w_stride / 2, 128, kGsBlock / 2)) return rc;
    if (int rc = make_tmap_2d_sw128(&ta, a, M, kbytes / 2, a_stride / 2, p.n / 2, kGsBlock / 2)) return rc;
    CUtensorMap to = tw;  // (results of one pair leave by TMA)
    if (kEnd == kScaled && plan.split == 1)
      if (int rc = make_tmap_2d_sw128(&to, p.out, M, N, p.ldc, 32, 64)) return rc;
    p.accs = kKind == kInt8 ? 1 : few_accumulators(p.n, p.kblocks);
    const int need = p.stages * p.slot + kFewFixed, smem = need > kHalfSmem ? need : kHalfSmem;
    static std::atomic<uint64_t> done{0};
    const int ctas = static_cast<int>((N + 255) / 256) * plan.tok_tiles * 2 * plan.split;
    p.to_l2 = kEnd == kScaled && plan.tok_tiles == 1 && sms >= device_sm_count_cached() ? kAheadInL2 / kGsHalf / ctas : 0;
    return launch_pairs(few_tokens_kernel<kKind, kEnd, T>, done, ctas, 2 * plan.split, kFewThreads, smem, stream,
                        tw, ta, to, p);
  }
  if (int rc = make_tmap_2d_sw128(&tw, w, N, kbytes / 2, w_stride / 2, 128, kGsBlock / 2)) return rc;
  if (int rc = make_tmap_2d_sw128(&ta, a, M, kbytes / 2, a_stride / 2, 128, kGsBlock / 2)) return rc;
  p.x_tiles = static_cast<int>((M + 255) / 256);
  p.y_tiles = static_cast<int>((N + 255) / 256);
  // weight tiles of a rasterisation panel: as many as stay in L2 beside what else passes (gemm.cu)
  const int64_t q = (40ll << 20) / (256 * kbytes);
  p.panel = static_cast<int>(q < 1 ? 1 : q < p.y_tiles ? q : p.y_tiles);
  p.by_panel = reciprocal(p.x_tiles * p.panel);
  p.by_width = reciprocal(p.panel);
  p.by_last = p.y_tiles % p.panel ? reciprocal(p.y_tiles % p.panel) : p.by_width;
  const int64_t tiles = static_cast<int64_t>(p.x_tiles) * p.y_tiles;
  const int pairs = static_cast<int>(tiles < sms / 2 ? tiles : sms / 2);
  static std::atomic<uint64_t> done{0};
  if constexpr (kEnd == kScaled) {
    CUtensorMap to;
    if (int rc = make_tmap_2d_sw128(&to, p.out, M, N, p.ldc, 32, 64)) return rc;
    return launch_pairs(many_tokens_kernel<T>, done, 2 * pairs, 2, kManyThreads, kGsMaxSmem, stream, ta, tw, to, p);
  } else return launch_pairs(many_logprobs_kernel<kKind>, done, 2 * pairs, 2, kLogThreads, kGsMaxSmem, stream, ta, tw, p);
}

static int budget(int sm_budget) {
  const int sms = sm_budget > 0 ? sm_budget : device_sm_count_cached();
  return sms < 2 ? 2 : sms;
}

}  // namespace spd

using namespace spd;

extern "C" {

int spd_int8_scaled_mm(void* out, const int8_t* a, const int8_t* b, const float* scales_a, const float* scales_b, const void* bias,
                       int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldc, int dtype, int older_w, int sm_budget,
                       spd_stream_t stream) {
  SPD_REQUIRE(M >= 0 && N > 0 && K > 0 && M <= 0x7fffff00 && N <= 0x7fffff00, SPD_E_BADARG, "spd_int8_scaled_mm: bad sizes");
  SPD_REQUIRE(K < 131072, SPD_E_SHAPE, "spd_int8_scaled_mm: sums of 131072 products and more may not fit 32 bits");  // (-128)^2 2^17 = 2^31
  SPD_REQUIRE(dtype == SPD_BF16 || dtype == SPD_F16, SPD_E_BADARG, "spd_int8_scaled_mm: bad dtype %d", dtype);
  SPD_REQUIRE(K % 16 == 0 && N % 8 == 0 && lda % 16 == 0 && ldb % 16 == 0 && ldc % 8 == 0, SPD_E_ALIGN,
              "spd_int8_scaled_mm: K, lda and ldb must be multiples of 16, N and ldc of 8");
  SPD_REQUIRE(lda >= K && ldb >= K && ldc >= N, SPD_E_BADARG, "spd_int8_scaled_mm: leading dimension too small");
  if (M == 0) return 0;
  SPD_REQUIRE(out && a && b && scales_a && scales_b, SPD_E_BADARG, "spd_int8_scaled_mm: null pointer");
  SPD_REQUIRE(aligned16(out) && aligned16(a) && aligned16(b), SPD_E_ALIGN, "spd_int8_scaled_mm: pointers must be 16-byte aligned");
  ScaledParams p{};
  p.out = out;
  p.ldc = ldc;
  p.bias = bias;
  p.sa = scales_a;
  p.sb = scales_b;
  p.early = older_w;
  const int sms = budget(sm_budget);
  const ScaledPlan plan = product_plan(M, N, static_cast<int>((K + kGsBlock - 1) / kGsBlock), {sms, as_stream(stream), nullptr});
  SPD_DISPATCH_DTYPE(dtype, { return (scaled_product<kInt8, kScaled, T>(a, b, M, N, K, lda, ldb, p, plan, sms, as_stream(stream))); });
}

int spd_int8_scaled_mm_tiles(int64_t M, int64_t N, int64_t K, int sm_budget, const int* clusters, int* split, int* ctas_per_sm) {
  SPD_REQUIRE(M > 0 && N > 0 && K > 0 && M <= 0x7fffff00 && N <= 0x7fffff00 && K < 131072 && split && ctas_per_sm, SPD_E_BADARG,
              "spd_int8_scaled_mm_tiles: bad arguments");
  const int sms = budget(sm_budget);
  const ScaledPlan plan = product_plan(M, N, static_cast<int>((K + kGsBlock - 1) / kGsBlock), {sms, nullptr, clusters});
  *split = plan.split;
  *ctas_per_sm = plan.tok_tiles > 0 && plan.smem == kHalfSmem ? 2 : 1;
  return plan.tok_tiles;
}

int64_t spd_linear_logprobs_workspace_bytes(int64_t M, int64_t V) {
  if (M < 0 || V <= 0) return SPD_E_BADARG;
  return M * ((V + 255) / 256 * 16 + 4);  // two parts of every 256 vocabulary rows, the target's logit
}

int spd_linear_logprobs(float* logprobs, float* lse, const void* x, const void* w, const float* scales_x, const float* scales_w,
                        const int64_t* targets, int64_t M, int64_t V, int64_t K, int64_t ldx, int64_t ldw, int dtype, int older_w,
                        void* workspace, int64_t workspace_bytes, int sm_budget, spd_stream_t stream) {
  SPD_REQUIRE(M >= 0 && V > 0 && K > 0 && M <= 0x7fffff00 && V <= 0x7fffff00, SPD_E_BADARG, "spd_linear_logprobs: bad sizes");
  SPD_REQUIRE(dtype == SPD_BF16 || dtype == SPD_F16 || dtype == SPD_I8, SPD_E_BADARG, "spd_linear_logprobs: bad dtype %d", dtype);
  const int size = dtype == SPD_I8 ? 1 : 2;
  SPD_REQUIRE(dtype != SPD_I8 || K < 131072, SPD_E_SHAPE, "spd_linear_logprobs: sums of 131072 products and more may not fit 32 bits");
  SPD_REQUIRE(K * size % 16 == 0 && ldx * size % 16 == 0 && ldw * size % 16 == 0, SPD_E_ALIGN,
              "spd_linear_logprobs: rows must be multiples of 16 bytes");
  SPD_REQUIRE(ldx >= K && ldw >= K, SPD_E_BADARG, "spd_linear_logprobs: leading dimension too small");
  if (M == 0) return 0;
  SPD_REQUIRE(logprobs && lse && x && w && targets && workspace, SPD_E_BADARG, "spd_linear_logprobs: null pointer");
  SPD_REQUIRE((dtype == SPD_I8) == (scales_x != nullptr) && (dtype == SPD_I8) == (scales_w != nullptr), SPD_E_BADARG,
              "spd_linear_logprobs: 8-bit operands and no others have scales");
  SPD_REQUIRE(aligned16(x) && aligned16(w) && aligned16(workspace), SPD_E_ALIGN, "spd_linear_logprobs: pointers must be 16-byte aligned");
  SPD_REQUIRE(workspace_bytes >= spd_linear_logprobs_workspace_bytes(M, V), SPD_E_WORKSPACE, "spd_linear_logprobs: workspace too small");
  const int sms = budget(sm_budget);
  ScaledParams p{};
  p.sa = scales_x;
  p.sb = scales_w;
  p.target = targets;
  p.part = reinterpret_cast<float2*>(workspace);
  p.early = older_w;
  const int64_t kbytes = K * size;
  const ScaledPlan plan = logprob_plan(M, V, static_cast<int>((kbytes + kGsBlock - 1) / kGsBlock), sms, dtype == SPD_I8);
  const int tiles = static_cast<int>((V + 255) / 256) * 2;
  p.hit = reinterpret_cast<float*>(p.part + tiles * M);
  cudaStream_t st = as_stream(stream);
  int rc;
  if (dtype == SPD_I8) rc = scaled_product<kInt8, kLogprob, __nv_bfloat16>(x, w, M, V, kbytes, ldx, ldw, p, plan, sms, st);
  else if (dtype == SPD_BF16) rc = scaled_product<kKindBf16, kLogprob, __nv_bfloat16>(x, w, M, V, kbytes, 2 * ldx, 2 * ldw, p, plan, sms, st);
  else rc = scaled_product<kKindF16, kLogprob, __half>(x, w, M, V, kbytes, 2 * ldx, 2 * ldw, p, plan, sms, st);
  if (rc) return rc;
  int width = 1;
  while (width < 4 && width < M) width *= 2;
  SPD_CUDA(launch(logprob_join_kernel, dim3(static_cast<unsigned>((M + width - 1) / width)), dim3(kJoinThreads), 0, st, pdl_enabled(), logprobs,
                  lse, p.part, p.hit, targets, static_cast<int>(M), tiles, static_cast<int>(V), width));
  return 0;
}

}  // extern "C"
