// Decode attention for requests that continue the same tokens (spd_attn_decode_shared): the shared keys.
//
// out = sum_p 2^(s_p) v_p / sum_p 2^(s_p) over a request's keys is joined from two ranges of keys: the ones that its group
// shares (here) and its own (attn_decode.cu), each with its maximum m, sum l and unnormalised output O.  Read by every
// member, the shared keys cost members x their bytes; here a tile of 128 keys is read once for up to 256 query rows (members x
// query heads of a kv head), which makes the decode step a matrix product: from about 250 rows it is bound by the tensor
// cores, with fewer by the stream of K and V.
//
// Every CTA takes an equal range of the list of (group, kv head, pair of query tiles, key tile) units (shared_groups.cuh).
//   warps 0-3 / 4-7  softmax of query tile 0 / 1: one thread per query row; P goes back into the TMEM columns of its S
//   warp 8, warp 9   K / V loader: a ring of four 128 x 128 tiles, K_j V_j K_{j+1} ..., by TMA where a tile's slots are
//                    consecutive, gathered row by row elsewhere
//   warp 10, warp 11 MMA issuer of query tile 0 / 1
// A key tile is taken in two halves of 64 keys, so that a warpgroup's softmax of one half runs beside the MMAs of the other.
// Sums, maxima and outputs are fp32 up to the join; P is rounded to the type of the keys, as the tensor cores take it, and l
// sums the rounded P, so that the rounding of a P that outweighs the others cancels.  The reference maximum is raised when a
// score passes it by 2^8 (O is then rescaled in TMEM), so a P is at most 2^8.
// Every mbarrier wait is bounded (see mbar_wait_bounded, spd_wait_status).
#include <cuda.h>

#include "common.cuh"
#include "prefill_tiles.cuh"
#include "ptx.cuh"
#include "shared_groups.cuh"
#include "tmap.cuh"

namespace spd {

constexpr int kSpThreads = 384;
constexpr int kSpM = 128;    // query rows per warpgroup
constexpr int kSpU = 64;     // keys of a softmax / MMA unit
constexpr int kSpD = 128;    // head size
constexpr int kSpTileBytes = 128 * 128 * 2;
constexpr int kSpSlots = 4;
constexpr int kSpStage = 8 * 2048;  // per softmax warp: 32 rows x 16 fp32 columns of an output on their way to memory
constexpr int kSpBars = 512;
constexpr int kSpSmem = kSpTileBytes * (2 + kSpSlots) + kSpStage + kSpBars + static_cast<int>(sizeof(SharedPlan)) + kShGroups * 4 + 1024;
static_assert(kSpSmem <= 232448, "shared memory of one block");
constexpr float kSpRescale = 8.f;  // exponent of 2 that a score may pass the reference maximum by

struct SharedParams {
  const void *k_pool, *v_pool;
  const int32_t* req_to_token;
  const int64_t *req_pool_indices, *seq_lens;
  int batch, Hq, Hk, group;
  int64_t rtt_stride;
  float scale_log2;
  int use_tma;
  SharedGroups sg;
  unsigned* wait_expired;
};

struct SpItem {
  int g, hk, b0;     // group, kv head, batch row of the first member
  int rows0, rows1;  // query rows of the two tiles
  int tile0, n;      // first key tile of this CTA and how many
};
struct SpWalk {
  int u, end, g;
  __device__ __forceinline__ bool next(const SharedParams& p, const SharedPlan& pl, SpItem& it) {
    while (u < end) {
      while (pl.unit0[g + 1] <= u) ++g;
      const int per_item = pl.tiles[g] + kShItemUnits, local = u - pl.unit0[g], item = local / per_item, at = local - item * per_item;
      const int len = min(end - u, per_item - at);
      u += len;
      const int t0 = max(0, at - kShItemUnits), t1 = at + len - kShItemUnits;
      if (t1 <= t0) continue;
      const int count = pl.count[g], pairs = sh_pairs(count, p.sg.mpt), pair = item % pairs;
      const int left = count - pair * 2 * p.sg.mpt;
      it.g = g;
      it.hk = item / pairs;
      it.b0 = pl.start[g] + pair * 2 * p.sg.mpt;
      it.rows0 = min(p.sg.mpt, left) * p.group;
      it.rows1 = min(p.sg.mpt, max(0, left - p.sg.mpt)) * p.group;
      it.tile0 = t0;
      it.n = t1 - t0;
      return true;
    }
    return false;
  }
};

// byte offset of (row, 16-byte chunk) inside a tile of two [128 rows x 128 B] blocks with the 128-byte swizzle
__device__ __forceinline__ uint32_t sp_tile_off(int row, int chunk16) {
  return (chunk16 >> 3) * 16384 + row * 128 + (((chunk16 & 7) ^ (row & 7)) << 4);
}

template <typename T>
__global__ void __launch_bounds__(kSpThreads, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ SharedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                      // 2 tiles
  uint8_t* sKV = smem + 2 * kSpTileBytes;  // ring: position 2t = K of tile t, 2t + 1 = V of tile t
  uint8_t* sO = smem + (2 + kSpSlots) * kSpTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sO + kSpStage);
  uint64_t* q_full = bars;                  // 2
  uint64_t* kv_full = bars + 2;             // kSpSlots
  uint64_t* kv_empty = kv_full + kSpSlots;  // kSpSlots
  uint64_t* s_full = kv_empty + kSpSlots;   // 4: [tile][half]
  uint64_t* p_full = s_full + 4;            // 4
  uint64_t* pv_done = p_full + 4;           // 4
  uint64_t* o_free = pv_done + 4;           // 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SharedPlan& pl = *reinterpret_cast<SharedPlan*>(reinterpret_cast<uint8_t*>(bars) + kSpBars);
  int* lead = reinterpret_cast<int*>(&pl + 1);  // per group: a member whose page-table row is in use

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (warp == 10) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 1);
      for (int i = 0; i < kSpSlots; ++i) {
        mbar_init(&kv_full[i], 32);
        mbar_init(&kv_empty[i], 2);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 4);
        mbar_init(&pv_done[i], 1);
      }
      for (int i = 0; i < 2; ++i) mbar_init(&o_free[i], 4);
      *dead = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 11 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // query rows that no box reaches (128 is no multiple of 3, 5, 6 or 7 heads) are zeros
  for (int i = threadIdx.x; i < 2 * kSpTileBytes / 16; i += kSpThreads) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  for (int i = threadIdx.x; i < kShGroups; i += kSpThreads) lead[i] = INT_MAX;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_S = tmem_base;        // 2 x (64 + 64) columns; P of a half in the first 32 of its S
  const uint32_t tmem_O = tmem_base + 256;  // 2 x 128 columns

  griddep_wait();
  // The kernel behind this one reads what the kernels before it wrote, and waits for this one before it joins: its CTAs may
  // start as the SMs become free.
  griddep_launch_dependents();
  sh_plan<kSpThreads>(p.sg, p.seq_lens, p.batch, p.Hk, pl, [&](int b, int, int g) {
    if (g >= 0) atomicMin(&lead[g], b);
  });
  SpWalk walk;
  {
    const int total = pl.unit0[p.sg.groups], per = sh_per_cta(total, p.sg.grid);
    walk.u = min(total, per * static_cast<int>(blockIdx.x));
    walk.end = min(total, walk.u + per);
    int lo = 0, hi = p.sg.groups - 1;  // the last group whose units do not begin behind the range's start
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pl.unit0[mid] <= walk.u) lo = mid; else hi = mid - 1;
    }
    walk.g = lo;
  }
  SpItem it;
  bool have = walk.next(p, pl, it);

  if (warp >= 10) {
    // ===================== MMA issuer of query tile 0 (warp 10) / 1 (warp 11) =====================
    const bool leader = elect_one();
    const int w = warp - 10;
    constexpr uint32_t idesc_qk = umma_idesc<T>(kSpM, kSpU, 0, 0);  // A, B K-major
    constexpr uint32_t idesc_pv = umma_idesc<T>(kSpM, kSpD, 0, 1);  // A = P (TMEM), B = V MN-major
    const uint64_t qd = umma_desc_sw128(smem_u32(sQ + w * kSpTileBytes), 16, 1024);
    const uint64_t kd0 = umma_desc_sw128(smem_u32(sKV), 16, 1024);
    const uint64_t vd0 = umma_desc_sw128(smem_u32(sKV), 16384, 1024);
    const uint32_t qk_hi = static_cast<uint32_t>(qd >> 32), v_hi = static_cast<uint32_t>(vd0 >> 32);
    const uint32_t q_bytes = static_cast<uint32_t>(p.sg.mpt * p.group) * 256;
    uint32_t t_base = 0;  // tiles of all items before
    uint32_t pq = 0;      // PV units issued
    uint32_t eq = 0;      // items of the tile
    bool q_ahead = false;
    auto load_q = [&](const SpItem& i) {
      if (leader) {
        mbar_expect_tx(&q_full[w], q_bytes);
        tma_load_3d(sQ + w * kSpTileBytes, &tmQ, &q_full[w], 0, i.hk * p.group, i.b0 + w * p.sg.mpt, kEvictNormal);
        tma_load_3d(sQ + w * kSpTileBytes + 16384, &tmQ, &q_full[w], 64, i.hk * p.group, i.b0 + w * p.sg.mpt, kEvictNormal);
      }
      __syncwarp();
    };
    while (have) {
      SpItem nx;
      const bool more = walk.next(p, pl, nx);
      const int n = it.n, nt = (w == 0 ? it.rows0 : it.rows1) > 0 ? n : 0;
      if (nt > 0) {
        if (!q_ahead) load_q(it);
        q_ahead = false;
        mbar_wait_bounded(&q_full[w], eq & 1, dead);
      }
      // S(j, h): P(j - 1, h), which these columns held, has been consumed by PV(j - 1, h), issued earlier by this thread
      auto issue_s = [&](int j, int h) {
        const uint32_t pos = 2 * (t_base + j);
        mbar_wait_bounded(&kv_full[pos % kSpSlots], (pos / kSpSlots) & 1, dead);
        if (h == 0) fence_proxy_async_smem();
        tc_fence_after_sync();
        uint32_t qa = static_cast<uint32_t>(qd);
        uint32_t ka = static_cast<uint32_t>(kd0) + (pos % kSpSlots) * (kSpTileBytes / 16) + h * (kSpU * 128 / 16);
#pragma unroll 1
        for (int k = 0; k < kSpD / 16; ++k) {
          umma_ss_if(leader, tmem_S + w * 128 + h * kSpU, qa, ka, qk_hi, idesc_qk, k);
          const uint32_t step = k == 3 ? (16384 - 96) / 16 : 2;
          qa += step;
          ka += step;
        }
        umma_commit_if(leader, &s_full[w * 2 + h]);
      };
      // a ring slot is released by both issuers; one whose tile has no rows waits for the copy first, to keep to the phases
      auto release_k = [&](int j) {
        const uint32_t pos = 2 * (t_base + j);
        if (nt == 0) mbar_wait_bounded(&kv_full[pos % kSpSlots], (pos / kSpSlots) & 1, dead);
        umma_commit_if(leader, &kv_empty[pos % kSpSlots]);
      };
      if (nt > 0) {
        issue_s(0, 0);
        issue_s(0, 1);
      }
      release_k(0);
      for (int j = 0; j < n; ++j) {
        const uint32_t vpos = 2 * (t_base + j) + 1;
        if (nt > 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (j == n - 1 && h == 0 && more && (w == 0 ? nx.rows0 : nx.rows1) > 0) {
              // the item's last S is under way: once it is complete, Q's memory is free for the next item
              mbar_wait_bounded(&s_full[w * 2 + 1], (pq >> 1) & 1, dead);
              load_q(nx);
              q_ahead = true;
            }
            mbar_wait_bounded(&p_full[w * 2 + h], (pq >> 1) & 1, dead);
            mbar_wait_bounded(&kv_full[vpos % kSpSlots], (vpos / kSpSlots) & 1, dead);
            if (h == 0) fence_proxy_async_smem();
            if (j == 0 && h == 0) mbar_wait_bounded(&o_free[w], (eq & 1) ^ 1, dead);  // the previous item's O has been read
            tc_fence_after_sync();
            uint32_t va = static_cast<uint32_t>(vd0) + (vpos % kSpSlots) * (kSpTileBytes / 16) + h * (kSpU * 128 / 16);
            uint32_t pa = tmem_S + w * 128 + h * kSpU;
            uint32_t acc = (j > 0 || h > 0) ? 1u : 0u;
#pragma unroll 1
            for (int k = 0; k < kSpU / 16; ++k) {
              umma_ts_if(leader, tmem_O + w * kSpD, pa, va, v_hi, idesc_pv, acc);
              pa += 8;
              va += 2048 / 16;
              acc = 1;
            }
            umma_commit_if(leader, &pv_done[w * 2 + h]);
            ++pq;
            if (j + 1 < n) issue_s(j + 1, h);
          }
        } else {
          mbar_wait_bounded(&kv_full[vpos % kSpSlots], (vpos / kSpSlots) & 1, dead);
        }
        umma_commit_if(leader, &kv_empty[vpos % kSpSlots]);
        if (j + 1 < n) release_k(j + 1);
      }
      if (nt > 0) ++eq;
      t_base += n;
      it = nx;
      have = more;
    }
  } else if (warp >= 8) {
    // ===================== K loader (warp 8) / V loader (warp 9) =====================
    const int is_v = warp == 9 ? 1 : 0;
    const int chunk = lane & 15, rsub = lane >> 4;
    const T* pool = reinterpret_cast<const T*>(is_v ? p.v_pool : p.k_pool);
    const CUtensorMap* tmap = is_v ? &tmV : &tmK;
    const int64_t row_elems = static_cast<int64_t>(p.Hk) * kSpD;
    // page-table lookups run one tile ahead of the copies, four rows a lane
    const int32_t* rtt = nullptr;
    auto begin = [&]() { rtt = p.req_to_token + p.req_pool_indices[lead[it.g]] * p.rtt_stride + it.tile0 * kShTile + lane; };
    int slot[4], j = 0;
    auto lookup = [&](int* s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = __ldg(rtt + j * kShTile + i * 32);
    };
    if (have) {
      begin();
      lookup(slot);
    }
    for (uint32_t pos = is_v; have; pos += 2) {
      const int hk = it.hk;
      if (++j == it.n) {
        j = 0;
        have = walk.next(p, pl, it);
        if (have) begin();
      }
      int next[4];
      if (have) lookup(next);
      const int base = __shfl_sync(0xffffffffu, slot[0], 0);
      bool contig = p.use_tma && base > 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) contig &= slot[i] == base + i * 32 + lane;
      contig = __all_sync(0xffffffffu, contig);
      const int st = pos % kSpSlots;
      mbar_wait_bounded(&kv_empty[st], ((pos / kSpSlots) & 1) ^ 1, dead);
      if (contig) {
        if (lane == 0) {
          uint8_t* dst = sKV + st * kSpTileBytes;
          fence_proxy_async_smem();  // the slot may last have been written by the gather path
          mbar_expect_tx_noarrive(&kv_full[st], kSpTileBytes);
          tma_load_2d(dst, tmap, &kv_full[st], hk * kSpD, base, kEvictNormal);
          tma_load_2d(dst + 16384, tmap, &kv_full[st], hk * kSpD + 64, base, kEvictNormal);
        }
        __syncwarp();
        mbar_arrive(&kv_full[st]);
      } else {
        const uint32_t dst = smem_u32(sKV + st * kSpTileBytes);
        const T* col = pool + static_cast<int64_t>(hk) * kSpD + chunk * 8;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const int row = i * 2 + rsub;
          const int64_t s = __shfl_sync(0xffffffffu, slot[i >> 4], row & 31);
          cp_async16(dst + sp_tile_off(row, chunk), col + s * row_elems, true);
        }
        cp_async_mbar_arrive_noinc(&kv_full[st]);  // when this lane's copies have landed
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) slot[i] = next[i];
    }
  } else {
    // ===================== softmax (one thread per query row) =====================
    const int w = warp >> 2, row = threadIdx.x & 127, row0 = row & ~31;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_S + lane_base + w * 128, to = tmem_O + lane_base + w * kSpD;
    const float scale = p.scale_log2, ahead = kSpRescale / scale;
    uint8_t* stage = sO + warp * 2048;
    // where this thread's pieces of an output go, by batch row: its own row's (m, l), and the rows 8 i + lane / 4 of its warp
    const int ml_at = row / p.group * p.Hq + row % p.group;
    int o_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row0 + i * 8 + (lane >> 2);
      o_at[i] = (r / p.group * p.Hq + r % p.group) * kSpD + (lane & 3) * 4;
    }
    uint32_t u = 0;  // units of the tile (all items)
    while (have) {
      const int rows = w == 0 ? it.rows0 : it.rows1;
      if (rows == 0) {
        have = walk.next(p, pl, it);
        continue;
      }
      const bool active = row0 < rows;  // (of this warp: the others only keep the barriers' count)
      float m = -INFINITY, l = 0.f;     // the reference maximum (raw scores) and sum folded into O
      const uint32_t u0 = u, u1 = u + 2 * it.n;
      for (; u < u1; ++u) {
        const int h = u & 1;
        mbar_wait_bounded(&s_full[w * 2 + h], (u >> 1) & 1, dead);
        if (active) {
          tc_fence_after_sync();
          uint32_t ra[32], rb[32], pk[32];
          const float mx = softmax_load_max<false, false>(ts + h * kSpU, ra, rb, 0, 0, 0);
          const bool raise = __any_sync(0xffffffffu, mx > m + ahead);
          float alpha = 1.f;
          if (raise) {
            const float up = fmaxf(m, mx);
            alpha = m == -INFINITY ? 0.f : fast_exp2((m - up) * scale);
            l *= alpha;
            m = up;
          }
          l += softmax_unit<T>(ra, rb, pk, scale, m == -INFINITY ? 0.f : m * scale);
          tmem_st_32x32b_x32(ts + h * kSpU, pk);
          if (raise && u > u0) {
            // O stands still once the PV of the unit before is complete (those before it are: S of this unit was issued after
            // them)
            mbar_wait_bounded(&pv_done[w * 2 + ((u - 1) & 1)], ((u - 1) >> 1) & 1, dead);
            tc_fence_after_sync();
            rescale_row128(to, alpha);
          }
          tmem_st_wait();
          tc_fence_before_sync();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w * 2 + h]);
      }
      // the item's part: O through shared memory, 64 bytes of a row at a time (a thread per row would touch 32 lines a store)
      const bool first = it.tile0 == 0;
      const int64_t at = first ? static_cast<int64_t>(it.b0 + w * p.sg.mpt) * p.Hq + it.hk * p.group
                               : (static_cast<int64_t>(blockIdx.x) * 2 + w) * kSpM;
      if (active) {
        mbar_wait_bounded(&pv_done[w * 2 + 1], ((u - 1) >> 1) & 1, dead);
        tc_fence_after_sync();
        float* o = (first ? p.sg.o_first : p.sg.o_next) + at * kSpD;
#pragma unroll 1
        for (int c = 0; c < kSpD; c += 16) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(to + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = i * 8 + (lane >> 2);
            if (row0 + rr < rows)
              *reinterpret_cast<uint4*>(o + (first ? o_at[i] : (row0 + rr) * kSpD + (lane & 3) * 4) + c) =
                  *reinterpret_cast<const uint4*>(stage + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
          }
          __syncwarp();
        }
        if (row < rows)
          reinterpret_cast<float2*>(first ? p.sg.ml_first : p.sg.ml_next)[at + (first ? ml_at : row)] = make_float2(m * scale, l);
        tc_fence_before_sync();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&o_free[w]);
      have = walk.next(p, pl, it);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*dead) {
    wait_drain();
    if (threadIdx.x == 0) wait_report(p.wait_expired);
  }
  if (warp == 10) tmem_dealloc(tmem_base, 512);
}

int attn_decode_own(void* out, const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
                    const int64_t* req_pool_indices, const int64_t* seq_lens, int64_t batch, int num_q_heads, int num_kv_heads,
                    int head_dim, int64_t q_stride, int64_t out_stride, int64_t req_to_token_stride, float sm_scale, int dtype,
                    void* workspace, int64_t workspace_bytes, const SharedGroups& sg, unsigned* wait_expired, int sm_budget,
                    cudaStream_t stream);  // attn_decode.cu
int check_attn_args(const char* fn, const void* out, const void* q, const void* k_pool, const void* v_pool, const void* rtt,
                    const void* rpi, int Hq, int Hk, int D, int64_t q_stride, int64_t out_stride);

// The workspace: attn_decode's own scratch (what it asks for a batch that does not fill the SMs holds the parts of every CTA
// too), the parts by batch row, those by CTA.
static int64_t own_bytes(int64_t batch, int num_q_heads, int num_kv_heads) {
  const int64_t rows = device_sm_count_cached() / num_kv_heads + 2;
  return spd_attn_decode_workspace_bytes(batch < rows ? batch : rows, num_q_heads, kSpD) / 16 * 16;
}
static int64_t part_bytes(int64_t batch, int num_q_heads) {
  return ((batch < kShRows ? batch : kShRows) * num_q_heads + static_cast<int64_t>(device_sm_count_cached()) * 2 * kSpM) * (kSpD + 2) * 4;
}

}  // namespace spd

using namespace spd;

extern "C" {

int64_t spd_attn_decode_shared_workspace_bytes(int64_t max_batch, int num_q_heads, int num_kv_heads, int head_dim) {
  if (max_batch < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim != kSpD) return 0;
  return own_bytes(max_batch, num_q_heads, num_kv_heads) + part_bytes(max_batch, num_q_heads);
}

int spd_attn_decode_shared(void* out, const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
                           const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* group_indptr,
                           const int64_t* shared_lens, int64_t batch, int64_t num_groups, int64_t max_shared_len,
                           int num_q_heads, int num_kv_heads, int head_dim, int64_t q_stride, int64_t out_stride,
                           int64_t req_to_token_stride, float sm_scale, int dtype, void* workspace, int64_t workspace_bytes,
                           int sm_budget, spd_stream_t stream) {
  if (int rc = check_attn_args("spd_attn_decode_shared", out, q, k_pool, v_pool, req_to_token, req_pool_indices, num_q_heads,
                               num_kv_heads, head_dim, q_stride, out_stride))
    return rc;
  SPD_REQUIRE(seq_lens && batch >= 0 && num_groups >= 0 && max_shared_len >= 0 && (num_groups == 0 || (group_indptr && shared_lens)),
              SPD_E_BADARG, "spd_attn_decode_shared: bad lengths or groups");
  SPD_REQUIRE(head_dim == kSpD, SPD_E_SHAPE, "spd_attn_decode_shared: head_dim must be 128 (got %d)", head_dim);
  if (batch == 0) return 0;
  const int64_t need = spd_attn_decode_shared_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim);
  SPD_REQUIRE(workspace && workspace_bytes >= need, SPD_E_WORKSPACE, "spd_attn_decode_shared: workspace too small (%lld bytes)",
              (long long)workspace_bytes);
  const int device_sms = device_sm_count_cached();
  const int sms = sm_budget > 0 && sm_budget < device_sms ? sm_budget : device_sms;
  // Every request reads its own pages where nothing can be shared, where a plan would not hold the batch, and where the scale
  // is not positive (the maximum of raw scores serves the scaled ones only there).
  if (batch < 2 || batch > kShRows || num_groups < 1 || num_groups > kShGroups || max_shared_len < kShTile || !(sm_scale > 0.f))
    return spd_attn_decode_paged_own(out, q, k_pool, v_pool, req_to_token, req_pool_indices, seq_lens, batch, num_q_heads,
                                     num_kv_heads, head_dim, q_stride, out_stride, req_to_token_stride, sm_scale, dtype, workspace,
                                     workspace_bytes, sm_budget, stream);
  SharedParams p{};
  if (int rc = wait_flag(&p.wait_expired)) return rc;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.req_to_token = req_to_token;
  p.req_pool_indices = req_pool_indices;
  p.seq_lens = seq_lens;
  p.batch = static_cast<int>(batch);
  p.Hq = num_q_heads;
  p.Hk = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.rtt_stride = req_to_token_stride;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  static const bool tma_on = []() { const char* e = getenv("SPD_ATTN_TMA"); return !(e && e[0] == '0'); }();
  p.use_tma = tma_on ? 1 : 0;
  p.sg.indptr = group_indptr;
  p.sg.lens = shared_lens;
  p.sg.groups = static_cast<int>(num_groups);
  p.sg.mpt = kSpM / p.group;
  p.sg.grid = sms;
  const int64_t own = own_bytes(batch, num_q_heads, num_kv_heads);
  p.sg.o_first = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + own);
  p.sg.o_next = p.sg.o_first + batch * num_q_heads * kSpD;
  p.sg.ml_first = p.sg.o_next + static_cast<int64_t>(sms) * 2 * kSpM * kSpD;
  p.sg.ml_next = p.sg.ml_first + batch * num_q_heads * 2;
  CUtensorMap tq, tk, tv;
  {
    // q as [batch][heads][128]: a box of mpt members and a kv head's query heads is a tile of mpt x group rows
    const uint64_t dims[3] = {kSpD, static_cast<uint64_t>(num_q_heads), static_cast<uint64_t>(batch)};
    const uint64_t strides[2] = {kSpD, static_cast<uint64_t>(q_stride)};
    const uint32_t box[3] = {64, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.sg.mpt)};
    if (int rc = make_tmap_sw128(&tq, q, 3, dims, strides, box)) return rc;
  }
  const uint64_t row_elems = static_cast<uint64_t>(num_kv_heads) * kSpD;
  if (int rc = get_tmap(&tk, k_pool, 1ull << 31, row_elems, row_elems, kShTile)) return rc;
  if (int rc = get_tmap(&tv, v_pool, 1ull << 31, row_elems, row_elems, kShTile)) return rc;
  SPD_DISPATCH_DTYPE(dtype, {
    auto kern = attn_shared_kernel<T>;
    static bool configured = false;
    if (!configured) {
      SPD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpSmem));
      configured = true;
    }
    SPD_CUDA(launch(kern, dim3(sms), dim3(kSpThreads), kSpSmem, as_stream(stream), pdl_enabled(), tq, tk, tv, p));
  });
  return attn_decode_own(out, q, k_pool, v_pool, req_to_token, req_pool_indices, seq_lens, batch, num_q_heads, num_kv_heads,
                         head_dim, q_stride, out_stride, req_to_token_stride, sm_scale, dtype, workspace, own, p.sg,
                         p.wait_expired, sm_budget, as_stream(stream));
}

}  // extern "C"
