// Decode attention for requests that continue the same tokens (spd_attn_decode_shared).
//
// A request's out = sum_p 2^(s_p) v_p / sum_p 2^(s_p) over its keys is joined from two ranges: the keys that its group shares and its
// own ones, each with its maximum m, sum l and unnormalised output O.  Read by every member, the shared keys cost members
// x their bytes; here a tile of 128 of them is read once for up to 256 query rows (members x query heads of a kv head), which
// makes the step a matrix product: from about 250 rows it is bound by the tensor cores and the exponentials, with fewer, and
// over a request's own keys, by the stream of K and V.
//
// Shared are whole tiles: as many as a group's shared slots and its shortest member (of those that are not empty) have.  What is
// left of them is read with each member's own tokens, from its own page-table row, so the split never shows in the result, and
// no query of the shared part needs a mask.
//
// ONE list of work: items (group, kv head, pair of query tiles) over the shared keys, then items (request, kv head) over the own
// ones, each with its key tiles one after another.  Tiles and items count what they cost, and every CTA takes an equal range
// of the list, so CTAs at the tensor cores' limit run beside CTAs at the memory's.  An item's sums are kept per CTA
// ("parts"): by batch row where the CTA has the item's first tile, else in a place of the CTA's own, since of all its items
// only the first can have begun earlier.  A second kernel joins them.
// (As two kernels, the shared keys' and attn_decode.cu's for the own ones: 64 requests of 130 own tokens behind 8192 shared
// ones, 32 / 8 heads, 48.6 us; each of them starts for 5 us without using the memory.)
//
//   warps 0-3 / 4-7  softmax of query tile 0 / 1: one thread per query row; P goes back into the TMEM columns of its S
//   warp 8, warp 9   K / V loader: a ring of four 128 x 128 tiles, K_j V_j K_{j+1} ..., by TMA where a tile's slots are
//                    consecutive, gathered row by row elsewhere
//   warp 10, warp 11 MMA issuer of query tile 0 / 1
// A key tile is taken in two halves of 64 keys, so that a warpgroup's softmax of one half runs beside the MMAs of the other.  Items
// over own keys have the query heads of one kv head as their only rows (the tensor cores wait for the keys anyhow) and
// go to the two warpgroups in turn, so that the softmax of one runs beside the other's.
// Sums, maxima and outputs are fp32 up to the join; P is rounded to the type of the keys, as the tensor cores take it, and l
// sums the rounded P, so that the rounding of a P that outweighs the others cancels.  The reference maximum is raised when a
// score passes it by 2^8 (O is then rescaled in TMEM), so a P is at most 2^8.
// Every mbarrier wait is bounded (see mbar_wait_bounded, spd_wait_status).
#include <cuda.h>
#include <limits.h>

#include "common.cuh"
#include "prefill_tiles.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace spd {

constexpr int kSpThreads = 384;
constexpr int kSpM = 128;    // query rows per warpgroup
constexpr int kSpTile = 128; // keys of a tile
constexpr int kSpU = 64;     // keys of a softmax / MMA unit
constexpr int kSpD = 128;    // head size
constexpr int kSpTileBytes = 128 * 128 * 2;
constexpr int kSpSlots = 4;
constexpr int kSpRows = 1024;    // batch rows that a plan holds
constexpr int kSpGroups = 256;   // groups
constexpr int kSpMaxTiles = 65535;
constexpr int kSpOwnQ = 4;       // buffers for the queries of items over own keys: [8 rows x 64 columns] twice
constexpr int kSpStage = 8 * 2048;  // per softmax warp: 32 rows x 16 fp32 columns of an output on their way to memory
constexpr int kSpBars = 256;
constexpr float kSpRescale = 8.f;  // exponent of 2 that a score may pass the reference maximum by
// what the list's entries cost: a key tile for two query tiles, for one; an item's start and end
constexpr int kCostPair = 3, kCostTile = 2, kCostShared = 4, kCostOwn = 1;
constexpr int kCostMin = 4;  // of a CTA

struct SharedParams {
  const void *k_pool, *v_pool;
  const int32_t* req_to_token;
  const int64_t *req_pool_indices, *seq_lens;
  const int32_t* group_indptr;  // [groups + 1]
  const int64_t* shared_lens;   // [groups]
  int batch, Hq, Hk, group;     // group: query heads of a kv head
  int groups, mpt;              // mpt: members of a query tile, 128 / group
  int64_t rtt_stride;
  float scale_log2;
  int use_tma;
  // parts.  o: fp32 rows of 128, before the division by l; ml: m (exponent of 2), l
  float *o_first, *ml_first;  // [2: shared, own][batch][query heads]
  float *o_next, *ml_next;    // [grid][2 tiles][128]
  int2* notes;                // [2: shared, own][batch][kv heads]: the CTA of the first part; parts (0: none) | row there << 16
  unsigned* wait_expired;
};

struct SharedPlan {  // in shared memory
  int len[kSpRows];          // a request's own tokens
  uint16_t skip[kSpRows];    // its shared tiles
  int unit0[kSpGroups + 1];  // cost of the groups before
  int req[kSpGroups];        // page-table row of a member that is not empty
  uint16_t start[kSpGroups], count[kSpGroups], tiles[kSpGroups];
  int sums[16];
  int own_row, own_head, own_at, own_req;  // where this CTA's range begins among the own keys
};
constexpr int kSpSmem = kSpTileBytes * (2 + kSpSlots) + kSpOwnQ * 2048 + kSpStage + kSpBars + static_cast<int>(sizeof(SharedPlan)) + 1024;
static_assert(kSpSmem <= 232448, "shared memory of one block");

__device__ __forceinline__ int sp_pairs(int count, int mpt) { return count <= mpt ? 1 : (count + 2 * mpt - 1) / (2 * mpt); }
// cost of a key tile in an item over shared keys
__device__ __forceinline__ int sp_cost(int count, int mpt) { return count <= mpt ? kCostTile : kCostPair; }
__device__ __forceinline__ int sp_tiles(int len) { return (len + kSpTile - 1) / kSpTile; }
__device__ __forceinline__ int sp_own_cost(int len) { return len > 0 ? kCostOwn + kCostTile * sp_tiles(len) : 0; }

struct SpRange {
  int begin, end;  // this CTA's part of the list
  int shared;      // cost of all items over shared keys, which come first
  int per;
  __device__ __forceinline__ bool own() const { return begin < end && end > shared; }  // reaches into the items over own keys
};

// sum over the threads before this one, and over all (into sums, by warp); a barrier inside
__device__ __forceinline__ int sp_scan(int v, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSpThreads / 32; ++w) {
    const int x = sums[w];
    before += w < warp ? x : 0;
    total += x;
  }
  return before + incl - v;
}

// The plan, by all threads of the CTA, from the groups' offsets and the lengths.
__device__ __forceinline__ SpRange sp_plan(const SharedParams& p, SharedPlan& pl) {
  static_assert(kSpThreads >= kSpGroups && kSpThreads / 32 <= 16, "a thread per group");
  constexpr int kPer = (kSpRows + kSpThreads - 1) / kSpThreads;
  const int g = threadIdx.x;
  // thread t reads rows [b0, b1); everything that the plan reads is requested at once
  const int per_thread = (p.batch + kSpThreads - 1) / kSpThreads, b0 = min(p.batch, g * per_thread), rows = min(p.batch, b0 + per_thread) - b0;
  int L[kPer], req[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    L[i] = i < rows ? static_cast<int>(max(0ll, min(static_cast<long long>(p.seq_lens[b0 + i]), static_cast<long long>(INT_MAX - kSpTile)))) : 0;
    req[i] = i < rows ? static_cast<int>(p.req_pool_indices[b0 + i]) : 0;
  }
  int shared = 0, count = 0;
  if (g < p.groups) {
    const int s = min(max(p.group_indptr[g], 0), p.batch), e = min(max(p.group_indptr[g + 1], s), p.batch);
    shared = static_cast<int>(max(0ll, min(static_cast<long long>(p.shared_lens[g]), static_cast<long long>(kSpMaxTiles) * kSpTile)));
    count = e - s;
    pl.start[g] = static_cast<uint16_t>(s);
    pl.count[g] = static_cast<uint16_t>(count);
    pl.unit0[g] = INT_MAX;  // for now: the shortest member
    pl.req[g] = INT_MAX;    // for now: the first member that is not empty
  }
  __syncthreads();
  int at[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = b0 + i;
    at[i] = -1;
    if (i < rows && L[i] > 0) {
      int lo = 0, hi = p.groups - 1;  // the last group that does not start behind the row
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pl.start[mid] <= b) lo = mid; else hi = mid - 1;
      }
      while (lo > 0 && pl.count[lo] == 0) --lo;  // groups of no rows start where the next one does
      if (b >= pl.start[lo] && b < pl.start[lo] + pl.count[lo]) {
        at[i] = lo;
        atomicMin(&pl.unit0[lo], L[i]);
        atomicMin(&pl.req[lo], b);
      }
    }
  }
  __syncthreads();
  int cost = 0, tiles = 0;
  if (g < p.groups) {
    const int least = pl.unit0[g];
    tiles = count >= 2 && least != INT_MAX ? min(shared, least) / kSpTile : 0;
    pl.tiles[g] = static_cast<uint16_t>(tiles);
    cost = tiles > 0 ? p.Hk * sp_pairs(count, p.mpt) * (kCostShared + tiles * sp_cost(count, p.mpt)) : 0;
  }
  int first[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) first[i] = at[i] >= 0 ? pl.req[at[i]] : -1;
  SpRange r;
  const int before = sp_scan(cost, pl.sums, r.shared);  // (its barrier: tiles are there, req has been read)
  if (g < p.groups) pl.unit0[g] = before;
  if (g == 0) pl.unit0[p.groups] = r.shared;
  int own = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (i >= rows) break;
    if (first[i] == b0 + i) pl.req[at[i]] = req[i];
    const int skip = at[i] >= 0 ? pl.tiles[at[i]] : 0;
    L[i] -= skip * kSpTile;
    pl.len[b0 + i] = L[i];
    pl.skip[b0 + i] = static_cast<uint16_t>(skip);
    own += sp_own_cost(L[i]) * p.Hk;
  }
  __syncthreads();  // sums have been read
  int all_own;
  const int own_before = sp_scan(own, pl.sums, all_own);
  const int total = r.shared + all_own;
  r.per = max(kCostMin, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  r.begin = min(total, r.per * static_cast<int>(blockIdx.x));
  r.end = min(total, r.begin + r.per);
  // where the range begins among the own items: found by the thread whose rows it is in
  int rem = max(r.begin, r.shared) - r.shared - own_before;
  if (r.own() && rem >= 0 && rem < own) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = i < rows ? sp_own_cost(L[i]) : 0;
      if (rem >= 0 && rem < c * p.Hk) {
        pl.own_row = b0 + i;
        pl.own_head = rem / c;
        pl.own_at = rem % c;
        pl.own_req = req[i];
      }
      rem -= c * p.Hk;
    }
  }
  __syncthreads();
  // rows without a shared or without an own part: the join looks at their notes too
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    for (int hk = threadIdx.x; hk < p.Hk; hk += kSpThreads) {
      if (pl.skip[b] == 0) p.notes[b * p.Hk + hk] = make_int2(0, 0);
      if (pl.len[b] == 0) p.notes[(p.batch + b) * p.Hk + hk] = make_int2(0, 0);
    }
  return r;
}

struct SpItem {
  bool own;
  int b0, hk;        // batch row of the first member, or of the request; kv head
  int req;           // page-table row
  int rows0, rows1;  // query rows of the two tiles
  int skip, keys;    // own: tiles before its first key; keys that the item's tiles hold
  int tile0, n;      // first key tile of this CTA and how many
  int buf;           // own: buffer of the queries
  int c0, parts;     // CTA of the first part and number of parts
};

// The items of this CTA, one after another; every role walks for itself.
struct SpWalk {
  int u, g;                // position in the list, group
  int row, head, owns;     // own items: the next one, and how many were before it here
  int64_t req;             // its page-table row, read when the row before is begun
  int64_t req_next;
  __device__ __forceinline__ void init(const SharedParams& p, const SharedPlan& pl, const SpRange& r) {
    u = r.begin;
    int lo = 0, hi = p.groups - 1;  // the last group whose items do not begin behind the range's start
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pl.unit0[mid] <= u) lo = mid; else hi = mid - 1;
    }
    g = lo;
    owns = 0;
    row = head = 0;
    req = req_next = 0;
    if (r.own()) {
      row = pl.own_row;
      head = pl.own_head;
      req = pl.own_req;
      req_next = row + 1 < p.batch ? p.req_pool_indices[row + 1] : 0;
    }
  }
  // tiles [t0, t1) of an item whose first tile stands at s0, `cost` each, that begin in [u, end)
  __device__ __forceinline__ bool cut(const SpRange& r, int s0, int cost, int n, SpItem& it) {
    it.tile0 = min(n, max(0, (u - s0 + cost - 1) / cost));
    it.n = min(n, max(0, (r.end - s0 + cost - 1) / cost)) - it.tile0;
    it.c0 = s0 / r.per;
    it.parts = (s0 + (n - 1) * cost) / r.per - it.c0 + 1;
    u = min(r.end, s0 + n * cost);
    return it.n > 0;
  }
  __device__ __forceinline__ bool next(const SharedParams& p, const SharedPlan& pl, const SpRange& r, SpItem& it) {
    while (u < min(r.end, r.shared)) {
      while (pl.unit0[g + 1] <= u) ++g;
      const int count = pl.count[g], tiles = pl.tiles[g], cost = sp_cost(count, p.mpt), per_item = kCostShared + tiles * cost;
      const int item = (u - pl.unit0[g]) / per_item, pairs = sp_pairs(count, p.mpt), pair = item % pairs;
      const int left = count - pair * 2 * p.mpt;
      it.own = false;
      it.hk = item / pairs;
      it.b0 = pl.start[g] + pair * 2 * p.mpt;
      it.req = pl.req[g];
      it.rows0 = min(p.mpt, left) * p.group;
      it.rows1 = min(p.mpt, max(0, left - p.mpt)) * p.group;
      it.skip = 0;
      it.keys = tiles * kSpTile;
      it.buf = 0;
      if (cut(r, pl.unit0[g] + item * per_item + kCostShared, cost, tiles, it)) return true;
    }
    while (u < r.end) {
      const int len = pl.len[row], n = sp_tiles(len);
      it.own = true;
      it.hk = head;
      it.b0 = row;
      it.req = static_cast<int>(req);
      it.skip = pl.skip[row];
      it.keys = len;
      bool some = false;
      if (len > 0) {
        // (the list's position of the item: known for the first one here, the others follow it)
        const int s0 = (owns == 0 && u == max(r.begin, r.shared) && row == pl.own_row && head == pl.own_head ? u - pl.own_at : u) + kCostOwn;
        some = cut(r, s0, kCostTile, n, it);
      }
      if (++head == p.Hk || len == 0) {
        head = 0;
        ++row;
        req = req_next;
        req_next = row + 1 < p.batch ? p.req_pool_indices[row + 1] : 0;
      }
      if (some) {
        it.rows0 = owns & 1 ? 0 : p.group;
        it.rows1 = owns & 1 ? p.group : 0;
        it.buf = owns % kSpOwnQ;
        ++owns;
        return true;
      }
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
attn_shared_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1,
                   const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ SharedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                      // 2 tiles
  uint8_t* sKV = smem + 2 * kSpTileBytes;  // ring: position 2t = K of tile t, 2t + 1 = V of tile t
  // queries of items over own keys: 8 rows of a tile whose other rows are whatever lies behind them, and never looked at
  uint8_t* sOwnQ = smem + (2 + kSpSlots) * kSpTileBytes;
  uint8_t* sO = sOwnQ + kSpOwnQ * 2048;
  static_assert(kSpStage + kSpBars + sizeof(SharedPlan) >= 16384, "the rows behind the last queries are shared memory too");
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
    tma_prefetch_desc(&tmQ1);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  griddep_launch_dependents();
  griddep_wait();
  tc_fence_before_sync();
  const SpRange range = sp_plan(p, pl);  // (its barriers also stand between the set-up above and what follows)
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_S = tmem_base;        // 2 x (64 + 64) columns; P of a half in the first 32 of its S
  const uint32_t tmem_O = tmem_base + 256;  // 2 x 128 columns
  SpWalk walk;
  walk.init(p, pl, range);
  SpItem it;
  bool have = walk.next(p, pl, range, it);

  if (warp >= 10) {
    // ===================== MMA issuer of query tile 0 (warp 10) / 1 (warp 11) =====================
    const bool leader = elect_one();
    const int w = warp - 10;
    constexpr uint32_t idesc_qk = umma_idesc<T>(kSpM, kSpU, 0, 0);  // A, B K-major
    constexpr uint32_t idesc_pv = umma_idesc<T>(kSpM, kSpD, 0, 1);  // A = P (TMEM), B = V MN-major
    const uint64_t qd = umma_desc_sw128(smem_u32(sQ + w * kSpTileBytes), 16, 1024);
    const uint32_t own_q = static_cast<uint32_t>(umma_desc_sw128(smem_u32(sOwnQ), 16, 1024));
    const uint64_t kd0 = umma_desc_sw128(smem_u32(sKV), 16, 1024);
    const uint64_t vd0 = umma_desc_sw128(smem_u32(sKV), 16384, 1024);
    const uint32_t qk_hi = static_cast<uint32_t>(qd >> 32), v_hi = static_cast<uint32_t>(vd0 >> 32);
    const uint32_t q_bytes = static_cast<uint32_t>(p.mpt * p.group) * 256;
    uint32_t t_base = 0;  // tiles of all items before
    uint32_t pq = 0;      // PV units issued
    uint32_t eq = 0;      // items of the tile
    uint32_t qq = 0;      // of them, items over shared keys
    bool q_ahead = false;
    auto load_q = [&](const SpItem& i) {
      if (leader) {
        mbar_expect_tx(&q_full[w], q_bytes);
        tma_load_3d(sQ + w * kSpTileBytes, &tmQ, &q_full[w], 0, i.hk * p.group, i.b0 + w * p.mpt, kEvictNormal);
        tma_load_3d(sQ + w * kSpTileBytes + 16384, &tmQ, &q_full[w], 64, i.hk * p.group, i.b0 + w * p.mpt, kEvictNormal);
      }
      __syncwarp();
    };
    while (have) {
      SpItem nx;
      const bool more = walk.next(p, pl, range, nx);
      const int n = it.n, nt = (w == 0 ? it.rows0 : it.rows1) > 0 ? n : 0;
      if (nt > 0 && !it.own) {
        if (!q_ahead) load_q(it);
        q_ahead = false;
        mbar_wait_bounded(&q_full[w], qq & 1, dead);
        ++qq;
      }
      // S(j, h): P(j - 1, h), which these columns held, has been consumed by PV(j - 1, h), issued earlier by this thread.
      // (The queries of an item over own keys arrive with its first K tile here.)
      const uint32_t q_lo = it.own ? own_q + it.buf * (2048 / 16) : static_cast<uint32_t>(qd);
      const uint32_t q_step = it.own ? (1024 - 96) / 16 : (16384 - 96) / 16;
      auto issue_s = [&](int j, int h) {
        const uint32_t pos = 2 * (t_base + j);
        mbar_wait_bounded(&kv_full[pos % kSpSlots], (pos / kSpSlots) & 1, dead);
        if (h == 0) fence_proxy_async_smem();
        tc_fence_after_sync();
        uint32_t qa = q_lo;
        uint32_t ka = static_cast<uint32_t>(kd0) + (pos % kSpSlots) * (kSpTileBytes / 16) + h * (kSpU * 128 / 16);
#pragma unroll 1
        for (int k = 0; k < kSpD / 16; ++k) {
          umma_ss_if(leader, tmem_S + w * 128 + h * kSpU, qa, ka, qk_hi, idesc_qk, k);
          qa += k == 3 ? q_step : 2;
          ka += k == 3 ? (16384 - 96) / 16 : 2;
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
            if (j == n - 1 && h == 0 && more && !nx.own && (w == 0 ? nx.rows0 : nx.rows1) > 0) {
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
    // ===================== K loader (warp 8, and queries of items over own keys) / V loader (warp 9) =====================
    const int is_v = warp == 9 ? 1 : 0;
    const int chunk = lane & 15, rsub = lane >> 4;
    const T* pool = reinterpret_cast<const T*>(is_v ? p.v_pool : p.k_pool);
    const CUtensorMap* tmap = is_v ? &tmV : &tmK;
    const int64_t row_elems = static_cast<int64_t>(p.Hk) * kSpD;
    // Page-table lookups run one tile ahead of the copies, four rows a lane; -1: behind the item's last key.
    const int32_t* rtt = nullptr;  // the lane's entry of the next tile's first row
    int slot[4], j = 0, left = 0;  // left: keys from that tile on
    auto begin = [&]() {
      rtt = p.req_to_token + it.req * p.rtt_stride + static_cast<int64_t>(it.skip + it.tile0) * kSpTile + lane;
      left = it.keys - it.tile0 * kSpTile;
      j = 0;
    };
    auto lookup = [&](int* s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = lane + i * 32 < left ? rtt[i * 32] : -1;
      rtt += kSpTile;
      left -= kSpTile;
    };
    if (have) {
      begin();
      lookup(slot);
    }
    for (uint32_t pos = is_v; have; pos += 2) {
      const int hk = it.hk;
      const bool first = j == 0;
      const int q_buf = !is_v && it.own && first ? it.buf : -1, q_row = it.b0;
      if (++j == it.n) {
        have = walk.next(p, pl, range, it);
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
      if (lane == 0 && q_buf >= 0) {
        // Four items ago this buffer held the queries of an item whose tiles are all older than the one that this slot held
        // before: its MMAs have finished.
        mbar_expect_tx_noarrive(&kv_full[st], p.group * 256);
        tma_load_3d(sOwnQ + q_buf * 2048, &tmQ1, &kv_full[st], 0, hk * p.group, q_row, kEvictNormal);
        tma_load_3d(sOwnQ + q_buf * 2048 + 1024, &tmQ1, &kv_full[st], 64, hk * p.group, q_row, kEvictNormal);
      }
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
        __syncwarp();
        const uint32_t dst = smem_u32(sKV + st * kSpTileBytes);
        const T* col = pool + static_cast<int64_t>(hk) * kSpD + chunk * 8;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const int row = i * 2 + rsub;
          const int64_t s = __shfl_sync(0xffffffffu, slot[i >> 4], row & 31);
          cp_async16(dst + sp_tile_off(row, chunk), col + (s >= 0 ? s : 0) * row_elems, s >= 0);
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
    for (; have; have = walk.next(p, pl, range, it)) {
      const int rows = w == 0 ? it.rows0 : it.rows1;
      if (rows == 0) continue;
      const bool active = row0 < rows;  // (of this warp: the others only keep the barriers' count)
      float m = -INFINITY, l = 0.f;     // the reference maximum (raw scores) and sum folded into O
      int key0 = it.tile0 * kSpTile;    // of the unit
      const uint32_t u0 = u, u1 = u + 2 * it.n;
      for (; u < u1; ++u, key0 += kSpU) {
        const int h = u & 1;
        mbar_wait_bounded(&s_full[w * 2 + h], (u >> 1) & 1, dead);
        if (active) {
          tc_fence_after_sync();
          uint32_t ra[32], rb[32], pk[32];
          const float mx = key0 + kSpU > it.keys ? softmax_load_max<true, false>(ts + h * kSpU, ra, rb, key0, it.keys - 1, 0)
                                                 : softmax_load_max<false, false>(ts + h * kSpU, ra, rb, 0, 0, 0);
          const bool raise = __any_sync(0xffffffffu, mx > m + ahead && row < rows);
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
      if (active) {
        const bool first = it.tile0 == 0;
        const int64_t set = it.own ? static_cast<int64_t>(p.batch) * p.Hq : 0;
        const int64_t at = first ? set + static_cast<int64_t>(it.b0 + (it.own ? 0 : w * p.mpt)) * p.Hq + it.hk * p.group
                                 : (static_cast<int64_t>(blockIdx.x) * 2 + w) * kSpM;
        mbar_wait_bounded(&pv_done[w * 2 + 1], ((u - 1) >> 1) & 1, dead);
        tc_fence_after_sync();
        float* o = (first ? p.o_first : p.o_next) + at * kSpD;
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
          reinterpret_cast<float2*>(first ? p.ml_first : p.ml_next)[at + (first ? ml_at : row)] = make_float2(m * scale, l);
        // where the join finds the parts: of a CTA behind the first one, the item is its first, so an own one is in tile 0 there
        if (first && row < rows && row % p.group == 0) {
          const int b = it.b0 + (it.own ? 0 : w * p.mpt + row / p.group);
          if (it.own || pl.skip[b] > 0)  // (an empty request in the middle of a group takes no part)
            p.notes[((it.own ? p.batch : 0) + b) * p.Hk + it.hk] = make_int2(it.c0, it.parts | (it.own ? 0 : w * kSpM + row) << 16);
        }
        tc_fence_before_sync();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&o_free[w]);
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

// out = the join of a query head's parts, over the shared and over the own keys.  A warp per row of the output, four columns a
// lane; a lane looks at one part's (m, l).  Latency bounds it, so a row's loads are requested before the first is waited for.
constexpr int kSjWarps = 8;
constexpr int kSjParts = 8;  // of a row at a time
template <typename T>
__global__ void __launch_bounds__(kSjWarps * 32)
attn_shared_join_kernel(T* __restrict__ out, int64_t out_stride, const __grid_constant__ SharedParams p, int rows) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kSjWarps + (threadIdx.x >> 5);
  griddep_launch_dependents();
  griddep_wait();
  if (row >= rows) return;
  const int b = row / p.Hq, h = row - b * p.Hq, hk = h / p.group;
  const int2 ns = __ldcg(p.notes + b * p.Hk + hk), no = __ldcg(p.notes + (p.batch + b) * p.Hk + hk);
  const int shared = ns.y & 0xffff, parts = shared + (no.y & 0xffff);
  // the i-th part's row among those by batch row (its first) or by CTA
  auto place = [&](int i, bool& first) {
    const bool own = i >= shared;
    const int2 n = own ? no : ns;
    const int k = own ? i - shared : i;
    first = k == 0;
    return first ? static_cast<int64_t>(own ? rows : 0) + row
                 : (static_cast<int64_t>(n.x) + k) * 2 * kSpM + (n.y >> 16) + (h - hk * p.group);
  };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, den = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const int mine = i0 + lane, here = min(32, parts - i0);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (mine < parts) {
      bool first;
      const int64_t at = place(mine, first);
      ml = __ldcg(reinterpret_cast<const float2*>(first ? p.ml_first : p.ml_next) + at);
    }
    float wt = 0.f;
    for (int j0 = 0; j0 < here; j0 += kSjParts) {
      float4 v[kSjParts];
#pragma unroll
      for (int k = 0; k < kSjParts; ++k)
        if (j0 + k < here) {
          bool first;
          const int64_t at = place(i0 + j0 + k, first);
          v[k] = __ldcg(reinterpret_cast<const float4*>((first ? p.o_first : p.o_next) + at * kSpD) + lane);
        }
      if (j0 == 0) {
        const float top = fmaxf(M, warp_max(ml.y > 0.f ? ml.x : -INFINITY));
        const float keep = den > 0.f ? fast_exp2(M - top) : 0.f;
        wt = ml.y > 0.f ? fast_exp2(ml.x - top) : 0.f;
        den = den * keep + warp_sum(wt * ml.y);
        acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
        M = top;
      }
#pragma unroll
      for (int k = 0; k < kSjParts; ++k)
        if (j0 + k < here) {
          const float f = __shfl_sync(0xffffffffu, wt, j0 + k);
          acc.x = fmaf(f, v[k].x, acc.x);
          acc.y = fmaf(f, v[k].y, acc.y);
          acc.z = fmaf(f, v[k].z, acc.z);
          acc.w = fmaf(f, v[k].w, acc.w);
        }
    }
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  *reinterpret_cast<uint2*>(out + b * out_stride + static_cast<int64_t>(h) * kSpD + lane * 4) =
      make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
}

int check_attn_args(const char* fn, const void* out, const void* q, const void* k_pool, const void* v_pool, const void* rtt,
                    const void* rpi, int Hq, int Hk, int D, int64_t q_stride, int64_t out_stride);

// The workspace: attn_decode's, for the calls that it serves; or the parts by batch row, those by CTA, the notes.
static int64_t decode_bytes(int64_t batch, int num_q_heads, int num_kv_heads) {
  const int64_t rows = device_sm_count_cached() / num_kv_heads + 2;  // (as many as it asks for a larger batch too)
  return spd_attn_decode_workspace_bytes(batch < rows ? batch : rows, num_q_heads, kSpD) / 16 * 16;
}
static int64_t part_bytes(int64_t batch, int num_q_heads, int num_kv_heads) {
  const int64_t b = batch < kSpRows ? batch : kSpRows;
  return (2 * b * num_q_heads + static_cast<int64_t>(device_sm_count_cached()) * 2 * kSpM) * (kSpD + 2) * 4 + 2 * b * num_kv_heads * 8;
}

}  // namespace spd

using namespace spd;

extern "C" {

int64_t spd_attn_decode_shared_workspace_bytes(int64_t max_batch, int num_q_heads, int num_kv_heads, int head_dim) {
  if (max_batch < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim != kSpD) return 0;
  // (one behind the other: a call of the one kind leaves the counters of the other at zero)
  return decode_bytes(max_batch, num_q_heads, num_kv_heads) + part_bytes(max_batch, num_q_heads, num_kv_heads);
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
  if (batch < 2 || batch > kSpRows || num_groups < 1 || num_groups > kSpGroups || max_shared_len < kSpTile || !(sm_scale > 0.f))
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
  p.group_indptr = group_indptr;
  p.shared_lens = shared_lens;
  p.groups = static_cast<int>(num_groups);
  p.mpt = kSpM / p.group;
  const int64_t rows = batch * num_q_heads;
  p.o_first = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_bytes(batch, num_q_heads, num_kv_heads));
  p.o_next = p.o_first + 2 * rows * kSpD;
  p.ml_first = p.o_next + static_cast<int64_t>(sms) * 2 * kSpM * kSpD;
  p.ml_next = p.ml_first + 2 * rows * 2;
  p.notes = reinterpret_cast<int2*>(p.ml_next + static_cast<int64_t>(sms) * 2 * kSpM * 2);
  // q as [batch][heads][128]: a box of mpt members and a kv head's query heads is a tile of mpt x group rows
  CUtensorMap tq, tq1, tk, tv;
  const uint64_t dims[3] = {kSpD, static_cast<uint64_t>(num_q_heads), static_cast<uint64_t>(batch)};
  const uint64_t strides[2] = {kSpD, static_cast<uint64_t>(q_stride)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.mpt)}, box1[3] = {64, box[1], 1};
  if (int rc = make_tmap_sw128(&tq, q, 3, dims, strides, box)) return rc;
  if (int rc = make_tmap_sw128(&tq1, q, 3, dims, strides, box1)) return rc;
  const uint64_t row_elems = static_cast<uint64_t>(num_kv_heads) * kSpD;
  if (int rc = get_tmap(&tk, k_pool, 1ull << 31, row_elems, row_elems, kSpTile)) return rc;
  if (int rc = get_tmap(&tv, v_pool, 1ull << 31, row_elems, row_elems, kSpTile)) return rc;
  SPD_DISPATCH_DTYPE(dtype, {
    auto kern = attn_shared_kernel<T>;
    static bool configured = false;
    if (!configured) {
      SPD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpSmem));
      configured = true;
    }
    SPD_CUDA(launch(kern, dim3(sms), dim3(kSpThreads), kSpSmem, as_stream(stream), pdl_enabled(), tq, tq1, tk, tv, p));
    SPD_CUDA(launch(attn_shared_join_kernel<T>, dim3(static_cast<unsigned>((rows + kSjWarps - 1) / kSjWarps)), dim3(kSjWarps * 32), 0,
                    as_stream(stream), pdl_enabled(), static_cast<T*>(out), out_stride, p, static_cast<int>(rows)));
  });
  return 0;
}

}  // extern "C"
