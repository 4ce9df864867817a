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
// ones, each with its key tiles one after another.  Tiles and items count what they cost, and every CTA takes a range of the
// list that costs the same, so CTAs at the tensor cores' limit run beside CTAs at the memory's.  An item's sums are kept per CTA
// ("parts"): by batch row where the CTA has the item's first tile, else in a place of the CTA's own, since of all its items
// only the first can have begun earlier.  A second kernel joins them.
// (As two kernels, the shared keys' and attn_decode.cu's for the own ones: 64 requests of 130 own tokens behind 8192 shared
// ones, 32 / 8 heads, 48.6 us, and 31.7 so; each kernel starts for 5 us without using the memory.)
//
//   warps 0-3 / 4-7  softmax of query tile 0 / 1: one thread per query row; P goes back into the TMEM columns of its S
//   warp 8, warp 9   K / V loader: a ring of four 128 x 128 tiles, K_j V_j K_{j+1} ..., by TMA (single rows where a
//                    tile's slots are not consecutive); over own keys both, for warpgroup 0 / 1
//   warp 10, warp 11 MMA issuer of query tile 0 / 1
// Over shared keys a tile is taken in two halves of 64 keys, so that a warpgroup's softmax of one half runs beside the MMAs of
// the other.  An item over own keys has the few query heads of one kv head as its rows; it is computed the other way round,
// S^T = K Q^T and O^T = V^T P^T, with a thread per key and P^T in shared memory, as in attn_decode.cu.  (With queries in the
// rows there too, one warp did all the exponentials: 160 requests of 132 own tokens, 32 / 32 heads, 276 us, and 81 now.)
// The items go to the two warpgroups in turn, and each has a loader, an issuer and a ring of three tiles to itself (its half of
// the ring above and the memory of its query tile): with one ring for both, an item waited for the one before in every role
// (229 us).
// Sums, maxima and outputs are fp32 up to the join; P is rounded to the type of the keys, as the tensor cores take it, and l
// sums the rounded P, so that the rounding of a P that outweighs the others cancels.  The reference maximum is raised when a
// score passes it by 2^8 (O is then rescaled in TMEM), so a P is at most 2^8.
// Every mbarrier wait is bounded (see mbar_wait_bounded, spd_wait_status).
// Measured, both kernels, caches cold: 64 requests of 130 own tokens behind 8192, 32 / 8 heads, 33 us (68.5 MB: 10.4 at the rate
// of a copy); 8 groups of 6, 134 behind 2944, 40 / 8 heads, 39 us (114 MB: 17.4); 160 of 132 behind 1408, 32 / 32 heads, 82 us
// (370 MB: 56); 256 of 300 behind 32768, 64 / 8 heads, 328 - 412 us as the power cap has it (277 GFLOP: 0.67 - 0.85 PFLOP/s).
// Start, the parts' way to memory and the join are 10 of the 33 us.
// The roles run side by side, so their code together competes for the instruction cache: long waits are out of the way, and
// loops are not unrolled where that gains nothing.  (With the waits unrolled in place the kernel had 217 KB; 48 requests of 134
// own tokens in 8 groups took 46.3 us, with 126 KB 38.9; 256 query rows by 32768 keys 369 and 337.  The MMAs over own keys
// unrolled: 352.)
#include <cuda.h>
#include <float.h>
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
constexpr int kSpMaxGroup = 8;
constexpr int kSpN = 16;         // own keys: columns of an MMA (>= kSpMaxGroup)
constexpr int kSpOwnSlots = 3;   // tiles of a warpgroup's ring over own keys
constexpr int kSpSmall = 2048;   // own keys: [8 rows x 128] of queries or P^T, in two blocks with the 128-byte swizzle
// per softmax warp: 32 rows x 16 fp32 columns of an output on their way to memory; or per warpgroup: two buffers of P^T, two of
// queries
constexpr int kSpStage = 8 * 2048;
static_assert(kSpStage == 2 * 4 * kSpSmall, "one memory for both");
constexpr int kSpBars = 256;
constexpr int kSpRed = 2 * 2 * kSpMaxGroup * 4 * 4;  // per warpgroup, twice: the maxima or sums of 4 warps for every head
constexpr float kSpRescale = 8.f;  // exponent of 2 that a score may pass the reference maximum by
// What the list's entries cost, in about 570 clk: a key tile for two query tiles, for one, over own keys (a tile of few keys is
// bound by the chain of its steps, not by its bytes); an item's start and end.
constexpr int kCostPair = 7, kCostOne = 4, kCostOwnTile = 4, kCostOwnLeast = 3, kCostShared = 24, kCostOwn = 1;
// of a range that begins among shared items for two query tiles (256 rows of output to keep).  64 requests behind 8192 tokens,
// 130 of their own, 32 / 8 heads: 33.3 us with 0, 32.2 with 16, 31.7 with 20; 160 behind 1408, 32 / 32: 84.7, 83.2, 81.1.  For
// items of one query tile 0 and 16 take 38.6 and 41.2 (8 groups of 6).  Half a mean range at most: where there is little to do,
// few such parts are written at once (128 requests behind 128 tokens, 8 / 1 heads: 16.6 with 0, 22.5 with 20).
constexpr int kCostPart = 20;
constexpr int kCostMin = 7;    // of a range, and one more

struct SharedParams {
  const int32_t* req_to_token;
  const int64_t *req_pool_indices, *seq_lens;
  const int32_t* group_indptr;  // [groups + 1]
  const int64_t* shared_lens;   // [groups]
  int batch, Hq, Hk, group;     // group: query heads of a kv head
  int groups, mpt;              // mpt: members of a query tile, 128 / group
  int64_t rtt_stride;
  float scale_log2;
  // parts.  o: fp32 rows of 128, before the division by l; ml: m (exponent of 2), l
  float *o_first, *ml_first;  // [3: shared, own, shared keys of warpgroup 1 in a split item][batch][query heads]
  float *o_next, *ml_next;    // [grid][2 warpgroups][128]
  // [2: shared, own][batch][kv heads]: the CTA of the first part; CTAs with parts (0: none) | split << 15 | row there << 16
  int2* notes;
  unsigned* wait_expired;
};

struct SharedPlan {  // in shared memory
  int len[kSpRows];          // a request's own tokens
  uint16_t skip[kSpRows];    // its shared tiles
  int unit0[kSpGroups + 1];  // cost of the groups before
  int req[kSpGroups];        // page-table row of a member that is not empty
  int least[kSpGroups], lead[kSpGroups];
  uint16_t start[kSpGroups], count[kSpGroups], tiles[kSpGroups];
  int2 sums[kSpThreads / 32];
  int own_row, own_head, own_at, own_req;  // where this CTA's range begins among the own keys
};
constexpr int kSpSmem = kSpTileBytes * (2 + kSpSlots) + kSpStage + kSpBars + kSpRed + static_cast<int>(sizeof(SharedPlan)) + 1024;
static_assert(kSpSmem <= 232448, "shared memory of one block");

__device__ __forceinline__ int sp_pairs(int count, int mpt) { return count <= mpt ? 1 : (count + 2 * mpt - 1) / (2 * mpt); }
// cost of a key tile in an item over shared keys
__device__ __forceinline__ int sp_cost(int count, int mpt) { return count <= mpt ? kCostOne : kCostPair; }
__device__ __forceinline__ int sp_tiles(int len) { return (len + kSpTile - 1) / kSpTile; }
// of an item over own keys
__device__ __forceinline__ int sp_own_cost(int len) {
  return len > 0 ? kCostOwn + kCostOwnTile * ((len - 1) / kSpTile) + max(kCostOwnLeast, ((len - 1) % kSpTile) * kCostOwnTile / kSpTile + 1)
                 : 0;
}

struct SpRange {
  int begin, end;  // this CTA's part of the list
  int shared;      // cost of all items over shared keys, which come first
  int per, per_shared, shared_ctas;  // length of a range: the first shared_ctas ones, which begin among the shared items; others
  __device__ __forceinline__ bool own() const { return begin < end && end > shared; }  // reaches into the items over own keys
  __device__ __forceinline__ int start(int cta) const { return min(cta, shared_ctas) * per_shared + max(0, cta - shared_ctas) * per; }
  __device__ __forceinline__ int cta(int u) const {
    const int first = shared_ctas * per_shared;
    return u < first ? u / per_shared : shared_ctas + (u - first) / per;
  }
  // Every CTA costs the same: a range among the shared items also `part` for a part's beginning and end.  With n ranges of x over
  // A of them, (N - n) of x + part over the rest, n x = A:  N x^2 + (N part - total) x = A part.
  __device__ __forceinline__ void divide(int total, int ctas, int part) {
    const float N = ctas, b = N * part - total;
    const float x = part > 0 ? (sqrtf(b * b + 4.f * N * part * shared) - b) / (2.f * N) : total / N;
    per_shared = max(kCostMin, static_cast<int>(x));
    do {  // (rounding, and shared items that leave the last of their ranges partly empty)
      ++per_shared;
      per = per_shared + part;
      shared_ctas = (shared + per_shared - 1) / per_shared;
    } while (shared_ctas > ctas || start(ctas) < total);
    begin = min(total, start(blockIdx.x));
    end = min(total, start(blockIdx.x + 1));
  }
};

// The plan, by all threads of the CTA, from the groups' offsets and the lengths.  It stands before the CTA's first load, so it
// asks for all that it reads at once and has few barriers.
__device__ __forceinline__ SpRange sp_plan(const SharedParams& p, SharedPlan& pl) {
  static_assert(kSpThreads >= kSpGroups, "a thread per group");
  constexpr int kPer = (kSpRows + kSpThreads - 1) / kSpThreads, kWarps = kSpThreads / 32;
  const int g = threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // thread t reads rows [b0, b0 + rows)
  const int per_thread = (p.batch + kSpThreads - 1) / kSpThreads, b0 = min(p.batch, g * per_thread), rows = min(p.batch, b0 + per_thread) - b0;
  int L[kPer], req[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    L[i] = i < rows ? static_cast<int>(max(0ll, min(static_cast<long long>(p.seq_lens[b0 + i]), static_cast<long long>(INT_MAX - kSpTile)))) : 0;
    req[i] = i < rows ? static_cast<int>(p.req_pool_indices[b0 + i]) : 0;
  }
  if (g < p.groups) {
    const int s = min(max(p.group_indptr[g], 0), p.batch), e = min(max(p.group_indptr[g + 1], s), p.batch);
    pl.start[g] = static_cast<uint16_t>(s);
    pl.count[g] = static_cast<uint16_t>(e - s);
    // the tiles that its slots allow; the shortest member, and the first that is not empty
    pl.tiles[g] = static_cast<uint16_t>(max(0ll, min(static_cast<long long>(p.shared_lens[g]) / kSpTile, static_cast<long long>(kSpMaxTiles))));
    pl.least[g] = INT_MAX;
    pl.lead[g] = INT_MAX;
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
      if (pl.count[lo] >= 2 && b >= pl.start[lo] && b < pl.start[lo] + pl.count[lo]) {
        at[i] = lo;
        atomicMin(&pl.least[lo], L[i]);
        atomicMin(&pl.lead[lo], b);
      }
    }
  }
  __syncthreads();
  auto tiles_of = [&](int group) {
    const int least = pl.least[group];
    return least == INT_MAX ? 0 : min(static_cast<int>(pl.tiles[group]), least / kSpTile);
  };
  // costs: of this thread's group, of its rows' own keys
  int cost = 0, own = 0;
  if (g < p.groups) {
    const int tiles = tiles_of(g), count = pl.count[g];
    cost = tiles > 0 ? p.Hk * sp_pairs(count, p.mpt) * (kCostShared + tiles * sp_cost(count, p.mpt)) : 0;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < rows) {
      const int skip = at[i] >= 0 ? tiles_of(at[i]) : 0;
      if (skip > 0 && pl.lead[at[i]] == b0 + i) pl.req[at[i]] = req[i];
      L[i] -= skip * kSpTile;
      pl.len[b0 + i] = L[i];
      pl.skip[b0 + i] = static_cast<uint16_t>(skip);
      own += sp_own_cost(L[i]) * p.Hk;
    }
  int incl = cost, own_incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o), y = __shfl_up_sync(0xffffffffu, own_incl, o);
    if (lane >= o) {
      incl += x;
      own_incl += y;
    }
  }
  if (lane == 31) pl.sums[warp] = make_int2(incl, own_incl);
  const bool pairs = __syncthreads_or(cost > 0 && pl.count[g] > p.mpt);
  SpRange r;
  r.shared = 0;
  int before = incl - cost, own_before = own_incl - own, all_own = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int2 x = pl.sums[w];
    if (w < warp) {
      before += x.x;
      own_before += x.y;
    }
    r.shared += x.x;
    all_own += x.y;
  }
  if (g < p.groups) {
    pl.unit0[g] = before;
    pl.tiles[g] = static_cast<uint16_t>(tiles_of(g));  // (who reads the tiles as they were has passed the barrier)
  }
  if (g == 0) pl.unit0[p.groups] = r.shared;
  const int total = r.shared + all_own;
  r.divide(total, gridDim.x, pairs ? min(kCostPart, total / (2 * static_cast<int>(gridDim.x))) : 0);
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
  return r;
}

struct SpItem {
  int b0, hk;        // batch row of the first member, or of the request; kv head
  int req;           // page-table row
  // Shared keys: query rows of the two tiles.  Where there is one tile only, the item is split: both warpgroups have it, with
  // every second key tile each (the ring's slots 2 w and 2 w + 1), and leave a part each.
  int rows0, rows1;
  int keys;          // keys that the item's tiles hold
  int s0, tiles;     // the list's position of its first tile; tiles
  int cost;          // of each
  int tile0, n;      // first key tile of this CTA and how many
  // tiles that begin in [u, end)
  __device__ __forceinline__ bool cut(int u, int end) {
    tile0 = min(tiles, max(0, (u - s0 + cost - 1) / cost));
    n = min(tiles, max(0, (end - s0 + cost - 1) / cost)) - tile0;
    return n > 0;
  }
  __device__ __forceinline__ bool split() const { return rows1 == 0; }
  __device__ __forceinline__ int rows(int w) const { return w == 0 || split() ? rows0 : rows1; }
  __device__ __forceinline__ int member0(int w, int mpt) const { return split() ? b0 : b0 + w * mpt; }
  // warpgroup w's tiles of this CTA are first, first + step, ..., `count` of them; base: tiles of the items before
  __device__ __forceinline__ void share(int w, uint32_t base, int& first, int& step, int& count) const {
    first = split() ? static_cast<int>((base ^ w) & 1) : 0;
    step = split() ? 2 : 1;
    count = (n - first + step - 1) / step;
  }
  // for the join, see SharedParams; by the CTA that has the item's first tile
  __device__ __forceinline__ int2 note(const SpRange& r, bool halves, int row) const {
    const int c0 = blockIdx.x, last = s0 + (tiles - 1) * cost;
    return make_int2(c0, (last < r.end ? 1 : r.cta(last) - c0 + 1) | (halves ? 1 << 15 : 0) | row << 16);
  }
};

// This CTA's items over shared keys, one after another; every role walks for itself.
struct SpWalk {
  int u, end, g;  // position in the list, end of the range there, group
  __device__ __forceinline__ SpWalk(const SharedParams& p, const SharedPlan& pl, const SpRange& r) : u(r.begin), end(min(r.end, r.shared)) {
    int lo = 0, hi = p.groups - 1;  // the last group whose items do not begin behind the range's start
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pl.unit0[mid] <= u) lo = mid; else hi = mid - 1;
    }
    g = lo;
  }
  __device__ __forceinline__ bool next(const SharedParams& p, const SharedPlan& pl, SpItem& it) {
    while (u < end) {
      while (pl.unit0[g + 1] <= u) ++g;
      const int count = pl.count[g], pairs = sp_pairs(count, p.mpt);
      it.tiles = pl.tiles[g];
      it.cost = sp_cost(count, p.mpt);
      const int per_item = kCostShared + it.tiles * it.cost, item = (u - pl.unit0[g]) / per_item;
      it.hk = item / pairs;
      const int pair = item - it.hk * pairs, left = count - pair * 2 * p.mpt;
      it.b0 = pl.start[g] + pair * 2 * p.mpt;
      it.req = pl.req[g];
      it.rows0 = min(p.mpt, left) * p.group;
      it.rows1 = min(p.mpt, max(0, left - p.mpt)) * p.group;
      it.keys = it.tiles * kSpTile;
      it.s0 = pl.unit0[g] + item * per_item + kCostShared;
      const bool some = it.cut(u, end);
      u = min(end, it.s0 + it.tiles * it.cost);
      if (some) return true;
    }
    return false;
  }
};

// This CTA's items over own keys: every second one, warpgroup w's.  A step is on the way of every role of the CTA, so what the
// heads of a request share is looked up once for all of them.
struct SpOwnWalk {
  int u, end, row, head, turn;
  int keys, tiles, cost;  // of the row's items
  int64_t req, req_next;  // page-table row of the row here and of the one behind it, read ahead
  __device__ __forceinline__ SpOwnWalk(const SharedParams& p, const SharedPlan& pl, const SpRange& r, int w)
      : u(0), end(0), row(0), head(0), turn(w), keys(0), tiles(0), cost(0), req(0), req_next(0) {
    if (r.own()) {
      row = pl.own_row;
      head = pl.own_head;
      u = max(r.begin, r.shared) - pl.own_at;  // of the item; its tiles before the range are cut off below
      end = r.end;
      req = pl.own_req;
      req_next = row + 1 < p.batch ? p.req_pool_indices[row + 1] : 0;
      enter(pl);
    }
  }
  __device__ __forceinline__ void enter(const SharedPlan& pl) {
    keys = pl.len[row];
    tiles = sp_tiles(keys);
    cost = sp_own_cost(keys);
  }
  __device__ __forceinline__ bool next(const SharedParams& p, const SharedPlan& pl, const SpRange& r, SpItem& it) {
    while (u < end) {
      while (keys <= 0 || head == p.Hk) {  // (the list goes on, so there is a row with keys)
        head = 0;
        ++row;
        req = req_next;
        req_next = row + 1 < p.batch ? p.req_pool_indices[row + 1] : 0;
        enter(pl);
      }
      const int s0 = u + kCostOwn, begin = max(r.begin, r.shared);
      const int tile0 = s0 >= begin ? 0 : min(tiles, (begin - s0 + kCostOwnTile - 1) / kCostOwnTile);
      const int n = (end - s0 >= tiles * kCostOwnTile ? tiles : min(tiles, max(0, (end - s0 + kCostOwnTile - 1) / kCostOwnTile))) - tile0;
      u += cost;
      const int hk = head++;
      if (n > 0 && (turn++ & 1) == 0) {
        it.b0 = row;
        it.hk = hk;
        it.req = static_cast<int>(req);
        it.keys = keys;
        it.s0 = s0;
        it.tiles = tiles;
        it.cost = kCostOwnTile;
        it.tile0 = tile0;
        it.n = n;
        return true;
      }
    }
    return false;
  }
};

// mbar_wait_bounded, out of the way but for the first try
__device__ __noinline__ void sp_wait_long(uint64_t* bar, uint32_t parity, volatile int* dead) {
#pragma unroll 1
  for (int i = 0; i < kMbarWaitTries; ++i) {
    if (mbar_try_wait(bar, parity)) return;
    if (*dead) return;
  }
  *dead = 1;
}
__device__ __forceinline__ void sp_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  if (!mbar_try_wait(bar, parity)) sp_wait_long(bar, parity, dead);
}
// of an element of P^T: row (query head), key
__device__ __forceinline__ uint32_t sp_p_off(int row, int key) {
  const int chunk = key >> 3;
  return (chunk >> 3) * 1024 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4) + (key & 7) * 2;
}
// barrier of a warpgroup's 128 threads
__device__ __forceinline__ void sp_bar(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
// the two rounded values of a word as fp32.  (bf16 by hand: through the conversion of a pair, a unit's 64 exponentials and
// sums took 1590 clk, so 716.)
template <typename T>
__device__ __forceinline__ float2 sp_unpack(uint32_t w) {
  if constexpr (umma_fmt<T>::v == 1) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return unpack2<T>(w);
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {  // NaN where all are
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// One row's 64 scores of a unit: p = exp2(s * scale - m_off), rounded and packed into pk; the sum of the rounded p.
template <typename T>
__device__ __forceinline__ float sp_softmax_unit(const uint32_t* ra, const uint32_t* rb, uint32_t* pk, float scale, float m_off) {
  const uint64_t scale2 = pack_f32x2(scale, scale), neg_m2 = pack_f32x2(-m_off, -m_off);
#pragma unroll
  for (int i = 0; i < 64; i += 2) {
    const uint32_t* r = i < 32 ? ra + i : rb + i - 32;
    float x0, x1;
    unpack_f32x2(ffma2(pack_f32x2(__uint_as_float(r[0]), __uint_as_float(r[1])), scale2, neg_m2), x0, x1);
    pk[i >> 1] = pack2<T>(fast_exp2(x0), fast_exp2(x1));
  }
  uint64_t sum[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float2 f = sp_unpack<T>(pk[i]);
    sum[i & 1] = fadd2(sum[i & 1], pack_f32x2(f.x, f.y));
  }
  float a, b, c, d;
  unpack_f32x2(sum[0], a, b);
  unpack_f32x2(sum[1], c, d);
  return (a + b) + (c + d);
}
// largest value of the warp (not NaN, unless all are)
__device__ __forceinline__ float sp_warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
struct SpBoxes {
  CUtensorMap rows[5];  // of the keys or values: boxes of 128, 64, 32, 16 rows and one row, by 64 columns
};
template <typename T>
__global__ void __launch_bounds__(kSpThreads, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1,
                   const __grid_constant__ SpBoxes tmK, const __grid_constant__ SpBoxes tmV,
                   const __grid_constant__ SharedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                      // 2 tiles
  uint8_t* sKV = smem + 2 * kSpTileBytes;  // ring: position 2t = K of tile t, 2t + 1 = V of tile t
  uint8_t* sO = smem + (2 + kSpSlots) * kSpTileBytes;
  // own keys: the 8 rows of queries or of P^T are half of an operand whose other 8 are whatever lies behind them, and never
  // looked at
  auto own_p = [&](int w, int i) { return sO + (w * 4 + i) * kSpSmall; };
  auto own_q = [&](int w, int i) { return sO + (w * 4 + 2 + i) * kSpSmall; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(sO + kSpStage);
  uint64_t* q_full = bars;                  // 2
  uint64_t* kv_full = bars + 2;             // kSpSlots, and the query tiles' memory as slots over own keys
  uint64_t* kv_empty = kv_full + kSpSlots + 2;
  uint64_t* s_full = kv_empty + kSpSlots + 2;  // 4: [tile][half]
  uint64_t* p_full = s_full + 4;            // 4
  uint64_t* pv_done = p_full + 4;           // 4
  uint64_t* o_free = pv_done + 4;           // 2
  uint64_t* stage_free = o_free + 2;        // 2: the warpgroup is through with the shared keys
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stage_free + 2);
  static_assert((4 + 2 * (kSpSlots + 2) + 12 + 4) * 8 <= kSpBars, "barriers");
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_red = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + kSpBars);
  SharedPlan& pl = *reinterpret_cast<SharedPlan*>(reinterpret_cast<uint8_t*>(s_red) + kSpRed);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (warp == 10) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 1);
      for (int i = 0; i < kSpSlots + 2; ++i) {
        mbar_init(&kv_full[i], 1);
        mbar_init(&kv_empty[i], 2);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 4);
        mbar_init(&pv_done[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&o_free[i], 4);
        mbar_init(&stage_free[i], 4);
      }
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
    tma_prefetch_desc(&tmK.rows[0]);
    tma_prefetch_desc(&tmV.rows[0]);
  }
  griddep_launch_dependents();
  griddep_wait();
  tc_fence_before_sync();
  const SpRange range = sp_plan(p, pl);  // (its barriers also stand between the set-up above and what follows)
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_S = tmem_base;        // 2 x (64 + 64) columns; P of a half in the first 32 of its S
  const uint32_t tmem_O = tmem_base + 256;  // 2 x 128 columns
  // Shared keys: tile t of the CTA is in the ring's places 2 t (K) and 2 t + 1 (V), of kSpSlots.  Own keys: tile t of warpgroup
  // w is in the places 2 t and 2 t + 1 of a ring of three, the slots 2 w and 2 w + 1 of the other ring, whose uses go on
  // counting, and the memory of the warpgroup's query tile, which is free when its last S over shared keys is complete.
  struct OwnSlot {
    int bar, tile;  // barriers; memory, in tiles from the queries' on
    uint32_t full, empty;  // parities to wait for
  };
  auto own_slot = [](int w, uint32_t place, uint32_t shared_tiles) {
    const uint32_t use = place / kSpOwnSlots, c = place - use * kSpOwnSlots, before = (shared_tiles + 1 - w) / 2;
    if (c == 2) return OwnSlot{kSpSlots + w, w, use & 1, use & 1};
    return OwnSlot{2 * w + static_cast<int>(c), 2 + 2 * w + static_cast<int>(c), (before + use) & 1, ((before + use) & 1) ^ 1};
  };
  SpWalk walk(p, pl, range);
  SpItem it;
  uint32_t t_base = 0;  // tiles of all items before

  if (warp >= 10) {
    // ===================== MMA issuer of query tile 0 (warp 10) / 1 (warp 11) =====================
    const bool leader = elect_one();
    const int w = warp - 10;
    constexpr uint32_t idesc_qk = umma_idesc<T>(kSpM, kSpU, 0, 0);     // A, B K-major
    constexpr uint32_t idesc_pv = umma_idesc<T>(kSpM, kSpD, 0, 1);     // A = P (TMEM), B = V MN-major
    constexpr uint32_t idesc_st = umma_idesc<T>(kSpTile, kSpN, 0, 0);  // own keys: A = K (K-major), B = Q (K-major)
    constexpr uint32_t idesc_ot = umma_idesc<T>(kSpD, kSpN, 1, 0);     // A = V (MN-major), B = P^T (K-major)
    const uint64_t qd = umma_desc_sw128(smem_u32(sQ + w * kSpTileBytes), 16, 1024);
    const uint64_t kd0 = umma_desc_sw128(smem_u32(sKV), 16, 1024);
    const uint64_t vd0 = umma_desc_sw128(smem_u32(sKV), 16384, 1024);
    const uint32_t qk_hi = static_cast<uint32_t>(qd >> 32), v_hi = static_cast<uint32_t>(vd0 >> 32);
    const uint32_t q_bytes = static_cast<uint32_t>(p.mpt * p.group) * 256;
    uint32_t pq = 0;  // PV units issued: two per tile of shared keys, one per tile of own ones
    uint32_t eq = 0;  // items of the tile
    bool q_ahead = false;
    auto load_q = [&](const SpItem& i) {
      if (leader) {
        mbar_expect_tx(&q_full[w], q_bytes);
        const int b = i.member0(w, p.mpt);
        tma_load_3d(sQ + w * kSpTileBytes, &tmQ, &q_full[w], 0, i.hk * p.group, b, kEvictNormal);
        tma_load_3d(sQ + w * kSpTileBytes + 16384, &tmQ, &q_full[w], 64, i.hk * p.group, b, kEvictNormal);
      }
      __syncwarp();
    };
    auto wait_kv = [&](uint32_t pos) { sp_wait(&kv_full[pos % kSpSlots], (pos / kSpSlots) & 1, dead); };
    bool have = walk.next(p, pl, it);
    while (have) {
      SpItem nx;
      const bool more = walk.next(p, pl, nx);
      int first, step, count, nx_first, nx_step = 0, nx_count = 0;
      it.share(w, t_base, first, step, count);
      if (more) nx.share(w, t_base + it.n, nx_first, nx_step, nx_count);
      if (count > 0) {
        if (!q_ahead) load_q(it);
        q_ahead = false;
        sp_wait(&q_full[w], eq & 1, dead);
      }
      // S(j, h): the P which these columns held has been consumed by the PV of this tile's predecessor here, issued earlier by
      // this thread
      auto issue_s = [&](int j, int h) {
        const uint32_t pos = 2 * (t_base + j);
        if (h == 0) wait_kv(pos);
        tc_fence_after_sync();
        uint32_t qa = static_cast<uint32_t>(qd);
        uint32_t ka = static_cast<uint32_t>(kd0) + (pos % kSpSlots) * (kSpTileBytes / 16) + h * (kSpU * 128 / 16);
#pragma unroll
        for (int k = 0; k < kSpD / 16; ++k) {
          umma_ss_if(leader, tmem_S + w * 128 + h * kSpU, qa, ka, qk_hi, idesc_qk, k);
          const uint32_t step = k == 3 ? (16384 - 96) / 16 : 2;
          qa += step;
          ka += step;
        }
        umma_commit_if(leader, &s_full[w * 2 + h]);
      };
      // a ring slot gets an arrival from either issuer, or both from the only one that reads it
      auto release = [&](uint32_t pos) {
        umma_commit_if(leader, &kv_empty[pos % kSpSlots]);
        if (step == 2) umma_commit_if(leader, &kv_empty[pos % kSpSlots]);
      };
      if (count > 0) {
        issue_s(first, 0);
        issue_s(first, 1);
        release(2 * (t_base + first));
      }
      for (int i = 0; i < count; ++i) {
        const int j = first + i * step;
        const uint32_t vpos = 2 * (t_base + j) + 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (i == count - 1 && h == 0 && nx_count > 0) {
            // the item's last S is under way: once it is complete, Q's memory is free for the next item
            sp_wait(&s_full[w * 2 + 1], (pq >> 1) & 1, dead);
            load_q(nx);
            q_ahead = true;
          }
          sp_wait(&p_full[w * 2 + h], (pq >> 1) & 1, dead);
          if (h == 0) wait_kv(vpos);
          if (i == 0 && h == 0) sp_wait(&o_free[w], (eq & 1) ^ 1, dead);  // the previous item's O has been read
          tc_fence_after_sync();
          uint32_t va = static_cast<uint32_t>(vd0) + (vpos % kSpSlots) * (kSpTileBytes / 16) + h * (kSpU * 128 / 16);
          uint32_t pa = tmem_S + w * 128 + h * kSpU;
          uint32_t acc = (i > 0 || h > 0) ? 1u : 0u;
#pragma unroll
          for (int k = 0; k < kSpU / 16; ++k) {
            umma_ts_if(leader, tmem_O + w * kSpD, pa, va, v_hi, idesc_pv, acc);
            pa += 8;
            va += 2048 / 16;
            acc = 1;
          }
          umma_commit_if(leader, &pv_done[w * 2 + h]);
          ++pq;
          if (i + 1 < count) issue_s(j + step, h);
        }
        release(vpos);
        if (i + 1 < count) release(2 * (t_base + j + step));
      }
      // A split item's other tiles have not been seen here, and a parity tells a phase from the one before only: an item for
      // both begins when both issuers have waited for all tiles before it.
      if (step == 2 && more && nx_step == 1) asm volatile("bar.sync 3, 64;" ::: "memory");
      if (count > 0) ++eq;
      t_base += it.n;
      it = nx;
      have = more;
    }
    umma_commit_if(leader, &kv_empty[kSpSlots + w]);  // (twice: an arrival for either issuer)
    umma_commit_if(leader, &kv_empty[kSpSlots + w]);
    // ---- own keys: S^T = K Q^T runs a tile ahead of O^T += V^T P^T, across items ----
    const uint32_t k_lo = static_cast<uint32_t>(umma_desc_sw128(smem_u32(smem), 16, 1024));
    const uint32_t v_lo = static_cast<uint32_t>(umma_desc_sw128(smem_u32(smem), 16384, 1024));
    const uint32_t q_lo = static_cast<uint32_t>(umma_desc_sw128(smem_u32(own_q(w, 0)), 16, 1024));
    const uint32_t p_lo = static_cast<uint32_t>(umma_desc_sw128(smem_u32(own_p(w, 0)), 16, 1024));
    SpOwnWalk own(p, pl, range, w), own_s = own;
    SpItem is;
    uint32_t ks = 0, vs = 0, pu = pq;  // tiles of S and of PV; S units issued
    int js = 0, qs = 0;                // S: tile of the item, buffer of its queries
    bool more_s = own_s.next(p, pl, range, is);
    auto issue_s = [&]() {  // into the buffer of the unit before the last, whose P has been waited for
      const OwnSlot at = own_slot(w, 2 * ks, t_base);
      const uint32_t h = pu & 1;
      sp_wait(&kv_full[at.bar], at.full, dead);  // (Q arrives with the item's first tile here)
      tc_fence_after_sync();
      uint32_t ka = k_lo + at.tile * (kSpTileBytes / 16), qa = q_lo + qs * (kSpSmall / 16);
#pragma unroll 1
      for (int k = 0; k < kSpD / 16; ++k) {
        umma_ss_if(leader, tmem_S + w * 128 + h * kSpU, ka, qa, qk_hi, idesc_st, k);
        ka += k == 3 ? (16384 - 96) / 16 : 2;
        qa += k == 3 ? (1024 - 96) / 16 : 2;
      }
      umma_commit_if(leader, &kv_empty[at.bar]);
      umma_commit_if(leader, &kv_empty[at.bar]);
      umma_commit_if(leader, &s_full[w * 2 + h]);
      ++pu;
      ++ks;
      if (++js == is.n) {
        js = 0;
        qs ^= 1;
        more_s = own_s.next(p, pl, range, is);
      }
    };
    if (more_s) issue_s();
    while (own.next(p, pl, range, it)) {
      for (int j = 0; j < it.n; ++j, ++vs) {
        // the next S goes first, unless its K is still on the way
        bool later = false;
        if (more_s) {
          const OwnSlot at = own_slot(w, 2 * ks, t_base);
          later = !__any_sync(0xffffffffu, mbar_test(&kv_full[at.bar], at.full));
          if (!later) issue_s();
        }
        const OwnSlot at = own_slot(w, 2 * vs + 1, t_base);
        const uint32_t h = pq & 1;
        sp_wait(&p_full[w * 2 + h], (pq >> 1) & 1, dead);
        sp_wait(&kv_full[at.bar], at.full, dead);
        const int valid = min(kSpTile, it.keys - (it.tile0 + j) * kSpTile), steps = (valid + 15) / 16;  // of 16 keys
        if (valid & 15) {  // V rows that the last step takes in and nobody asked for: their P is 0, they may be anything
          uint8_t* rows = smem + at.tile * kSpTileBytes + (lane >> 3 & 1) * 16384 + (lane & 7) * 16;
          for (int r = valid + (lane >> 4); r < steps * 16; r += 2) *reinterpret_cast<uint4*>(rows + r * 128) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (j == 0) sp_wait(&o_free[w], (eq & 1) ^ 1, dead);  // the previous item's O has been read
        tc_fence_after_sync();
        uint32_t va = v_lo + at.tile * (kSpTileBytes / 16), pa = p_lo + h * (kSpSmall / 16);
#pragma unroll 1
        for (int k = 0; k < steps; ++k) {
          umma_ss_if(leader, tmem_O + w * kSpD, va, pa, qk_hi, idesc_ot, j + k);
          va += 2048 / 16;
          pa += k == 3 ? (1024 - 96) / 16 : 2;
        }
        umma_commit_if(leader, &kv_empty[at.bar]);
        umma_commit_if(leader, &kv_empty[at.bar]);
        umma_commit_if(leader, &pv_done[w * 2 + h]);
        ++pq;
        if (later) issue_s();
      }
      ++eq;
    }
  } else if (warp >= 8) {
    // ===================== loaders =====================
    const int lw = warp - 8;
    // a tile's slots, rows 4 lane .. 4 lane + 3, from its first row's entry on; -1: behind the item's last key
    auto lookup = [&](const int32_t* rtt, int left, int* s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = lane * 4 + i < left ? rtt[lane * 4 + i] : -1;
    };
    // A tile into the memory at `tile`; its barrier gets one arrival beside the bytes.  Consecutive slots: as few boxes as make
    // up its rows, in steps of 16; else boxes of 16 rows where those are consecutive; others four rows an instruction.
    // (Scattered rows by 16-byte cp.async took a warp 4500 clk a tile.  A TMA instruction takes it about 100: with boxes of 16
    // rows wherever a tile was not full, and an arrival of every lane, 160 requests of 132 own tokens, 32 / 32 heads, took
    // 93 us.)  What stands behind an item's last key in a box belongs to others, or lies past the pool and reads as zeros: the
    // scores of such K rows are not looked at, such V rows are cleared before the MMA.
    auto load = [&](const SpBoxes& tm, int bar, int tile, int hk, const int* slot, int valid) {
      uint8_t* dst = smem + tile * kSpTileBytes;
      const int base = __shfl_sync(0xffffffffu, slot[0], 0), base16 = __shfl_sync(0xffffffffu, slot[0], lane & ~3);
      bool all = true, some = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool behind = lane * 4 + i >= valid;
        all &= behind || slot[i] == base + lane * 4 + i;
        some &= behind || slot[i] == base16 + (lane & 3) * 4 + i;
      }
      all = __all_sync(0xffffffffu, all);
      const int pieces = (valid + 15) / 16, col = hk * kSpD;  // of 16 rows
      if (lane == 0) mbar_expect_tx(&kv_full[bar], pieces * 16 * 256);
      __syncwarp();
      if (all) {
        // lanes 2 b and 2 b + 1: the box of 128 >> b rows, if it is one of those that make up the pieces, behind the larger ones
        const int half = lane & 1, b = lane >> 1, size = 8 >> b;
        if (b < 4 && (pieces & size)) {
          const int row = (pieces & ~(2 * size - 1)) * 16;
          tma_load_2d(dst + half * 16384 + row * 128, &tm.rows[b], &kv_full[bar], col + half * 64, base + row, kEvictNormal);
        }
      } else {
        some = (__ballot_sync(0xffffffffu, some) >> (lane & ~3) & 15) == 15;
        if (lane >> 2 < pieces) {
          if (some) {
            if ((lane & 3) < 2)
              tma_load_2d(dst + (lane & 1) * 16384 + (lane >> 2) * 2048, &tm.rows[3], &kv_full[bar], col + (lane & 1) * 64, base16,
                          kEvictNormal);
          } else {
#pragma unroll
            for (int half = 0; half < 2; ++half)
              tma_gather4_2d(smem_u32(dst + half * 16384 + lane * 512), &tm.rows[4], &kv_full[bar], col + half * 64, slot[0], slot[1],
                             slot[2], slot[3], kEvictNormal);
          }
        }
      }
    };
    // ---- shared keys: K by warp 8, V by warp 9; lookups run one tile ahead of the copies ----
    int slot[4], next[4];
    auto entry = [&](int skip, int j) {
      return p.req_to_token + it.req * p.rtt_stride + static_cast<int64_t>(skip + it.tile0 + j) * kSpTile;
    };
    bool have = walk.next(p, pl, it);
    if (have) lookup(entry(0, 0), kSpTile, slot);
    for (int j = 0; have; ++t_base) {
      const int hk = it.hk;
      if (++j == it.n) {
        have = walk.next(p, pl, it);
        j = 0;
      }
      if (have) lookup(entry(0, j), kSpTile, next);
      const uint32_t pos = 2 * t_base + lw;
      sp_wait(&kv_empty[pos % kSpSlots], ((pos / kSpSlots) & 1) ^ 1, dead);
      load(lw ? tmV : tmK, pos % kSpSlots, 2 + pos % kSpSlots, hk, slot, kSpTile);
#pragma unroll
      for (int i = 0; i < 4; ++i) slot[i] = next[i];
    }
    // ---- own keys: warpgroup lw's, with the queries ----
    SpOwnWalk own(p, pl, range, lw);
    uint32_t place = 0;
    int q_buf = 0, b = 0, valid = 0, hk = 0, j = 0;
    bool first = false, more = true;
    have = false;
    it.n = 0;
#pragma unroll 1
    while (more) {
      if (j == it.n) {
        more = own.next(p, pl, range, it);
        j = 0;
      }
      const int left = it.keys - (it.tile0 + j) * kSpTile;
      if (more) lookup(entry(pl.skip[it.b0], j), left, next);
      // the queries' buffers are memory that the warpgroup's outputs over shared keys pass through
      if (!have) sp_wait(&stage_free[lw], 0, dead);
#pragma unroll 1
      for (int is_v = 0; have && is_v < 2; ++is_v, ++place) {
        const OwnSlot at = own_slot(lw, place, t_base);
        sp_wait(&kv_empty[at.bar], at.empty, dead);
        if (is_v == 0 && first) {
          // The buffer's last queries were those of the item before the last one, whose tiles are no younger than the V tile
          // that this slot held: its MMAs have finished.
          if (lane == 0) {
            mbar_expect_tx_noarrive(&kv_full[at.bar], p.group * 256);
            tma_load_3d(own_q(lw, q_buf), &tmQ1, &kv_full[at.bar], 0, hk * p.group, b, kEvictNormal);
            tma_load_3d(own_q(lw, q_buf) + 1024, &tmQ1, &kv_full[at.bar], 64, hk * p.group, b, kEvictNormal);
          }
          __syncwarp();
          q_buf ^= 1;
        }
        load(is_v ? tmV : tmK, at.bar, at.tile, hk, slot, valid);
      }
      have = more;
      hk = it.hk;
      b = it.b0;
      first = j == 0;
      valid = min(kSpTile, left);
      ++j;
#pragma unroll
      for (int i = 0; i < 4; ++i) slot[i] = next[i];
    }
  } else {
    // ===================== softmax =====================
    // Rows without a shared or without an own part: the join looks at their notes too.  (The first scores are a while off.)
#pragma unroll 1
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
#pragma unroll 1
      for (int hk = threadIdx.x; hk < p.Hk; hk += 2 * kSpM) {
        if (pl.skip[b] == 0) p.notes[b * p.Hk + hk] = make_int2(0, 0);
        if (pl.len[b] == 0) p.notes[(p.batch + b) * p.Hk + hk] = make_int2(0, 0);
      }
    const int w = warp >> 2, row = threadIdx.x & 127, row0 = row & ~31;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_S + lane_base + w * 128, to = tmem_O + lane_base + w * kSpD;
    const float scale = p.scale_log2, ahead = kSpRescale / scale;
    uint32_t u = 0;  // units of the tile (all items)
    {
      // ---- shared keys: a thread per query row ----
      uint8_t* stage = sO + warp * 2048;
      // where this thread's pieces of an output go, by batch row: its own row's (m, l), and the rows 8 i + lane / 4 of its warp
      const int member = row / p.group, ml_at = member * p.Hq + row - member * p.group;
      int o_at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row0 + i * 8 + (lane >> 2), m = r / p.group;
        o_at[i] = (m * p.Hq + r - m * p.group) * kSpD + (lane & 3) * 4;
      }
      for (; walk.next(p, pl, it); t_base += it.n) {
        int first_tile, step, count;
        it.share(w, t_base, first_tile, step, count);
        const int rows = it.rows(w);
        const bool active = row0 < rows;  // (of this warp: the others only keep the barriers' count)
        float m = -INFINITY, l = 0.f;     // the reference maximum (raw scores) and sum folded into O
        const uint32_t u0 = u, u1 = u + 2 * count;
        for (; u < u1; ++u) {
          const int h = u & 1;
          sp_wait(&s_full[w * 2 + h], (u >> 1) & 1, dead);
          if (active) {
            tc_fence_after_sync();
            uint32_t ra[32], rb[32], pk[32];
            tmem_ld_32x32b_x32(ts + h * kSpU, ra);
            tmem_ld_32x32b_x32(ts + h * kSpU + 32, rb);
            tmem_ld_wait();
            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              m0 = fmax3(m0, __uint_as_float(ra[i]), __uint_as_float(ra[i + 1]));
              m1 = fmax3(m1, __uint_as_float(rb[i]), __uint_as_float(rb[i + 1]));
            }
            const float mx = fmaxf(m0, m1);
            // The reference maximum is raised before the exponentials, where a score passes it by 2^8 (rarely but for the first
            // unit); O is rescaled when the PV of the unit before is complete
            const bool raise = __any_sync(0xffffffffu, mx > m + ahead && row < rows);
            float alpha = 1.f;
            if (raise) {
              const float up = fmaxf(m, mx);
              alpha = m == -INFINITY ? 0.f : fast_exp2((m - up) * scale);
              l *= alpha;
              m = up;
            }
            l += sp_softmax_unit<T>(ra, rb, pk, scale, m == -INFINITY ? 0.f : m * scale);
            tmem_st_32x32b_x32(ts + h * kSpU, pk);
            if (raise && u > u0) {
              // O stands still once the PV of the unit before is complete (those before it are: S of this unit was issued
              // after them)
              sp_wait(&pv_done[w * 2 + ((u - 1) & 1)], ((u - 1) >> 1) & 1, dead);
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
          const int b0 = it.member0(w, p.mpt);
          const int64_t at = first ? static_cast<int64_t>((it.split() && w == 1 ? 2 * p.batch : 0) + b0) * p.Hq + it.hk * p.group
                                   : (static_cast<int64_t>(blockIdx.x) * 2 + w) * kSpM;
          if (count > 0) {
            sp_wait(&pv_done[w * 2 + 1], ((u - 1) >> 1) & 1, dead);
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
          }
          if (row < rows)
            reinterpret_cast<float2*>(first ? p.ml_first : p.ml_next)[at + (first ? ml_at : row)] = make_float2(m * scale, l);
          // (an empty request in the middle of a group takes no part; without a tile the part is one of sum 0)
          const int b = b0 + member;
          if (first && row < rows && row == member * p.group && pl.skip[b] > 0 && (w == 0 || !it.split()))
            p.notes[b * p.Hk + it.hk] = it.note(range, it.split(), w * kSpM + row);
          tc_fence_before_sync();
          __syncwarp();
        }
        if (lane == 0 && count > 0) mbar_arrive(&o_free[w]);
      }
      fence_proxy_async_smem();  // queries are copied into the staging memory
      __syncwarp();
      if (lane == 0) mbar_arrive(&stage_free[w]);
    }
    // ---- own keys: a thread per key of a tile, then per column of the output ----
    const int G = p.group;
    // what the four warps find, [head][warp]; of the tiles alternately, so that one barrier stands between writing and reading
    float4* red = reinterpret_cast<float4*>(s_red) + w * 2 * kSpMaxGroup;
    auto put = [&](uint32_t buf, int g, float v) {
      if (lane == 0) reinterpret_cast<float*>(red + (buf & 1) * kSpMaxGroup + g)[warp & 3] = v;
    };
    uint32_t rounds = 0;  // of them
    SpOwnWalk own(p, pl, range, w);
    while (own.next(p, pl, range, it)) {
      float m_ref[kSpMaxGroup], l_thr[kSpMaxGroup];
#pragma unroll
      for (int g = 0; g < kSpMaxGroup; ++g) {
        m_ref[g] = -FLT_MAX;  // as long as all scores are -inf, which weigh nothing: -inf - -inf is not -inf
        l_thr[g] = 0.f;
      }
      for (int j = 0; j < it.n; ++j, ++u) {
        const int h = u & 1;
        sp_wait(&s_full[w * 2 + h], (u >> 1) & 1, dead);
        tc_fence_after_sync();
        uint32_t r[16];
        tmem_ld_32x32b_x16(ts + h * kSpU, r);
        tmem_ld_wait();
        const bool valid = (it.tile0 + j) * kSpTile + row < it.keys;
        float s[kSpMaxGroup];
#pragma unroll
        for (int g = 0; g < kSpMaxGroup; ++g)
          if (g < G) {
            s[g] = valid ? __uint_as_float(r[g]) * scale : -INFINITY;
            put(rounds, g, sp_warp_max(s[g]));
          }
        sp_bar(1 + w);
        float alpha[kSpMaxGroup];
        bool raise = false;  // the same in all threads
#pragma unroll
        for (int g = 0; g < kSpMaxGroup; ++g) {
          alpha[g] = 1.f;
          if (g < G) {
            const float4 x = red[(rounds & 1) * kSpMaxGroup + g];
            const float mx = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
            if (mx > m_ref[g] + kSpRescale) {
              alpha[g] = fast_exp2(m_ref[g] - mx);
              l_thr[g] *= alpha[g];
              m_ref[g] = mx;
              raise = true;
            }
          }
        }
        ++rounds;
        if (raise && j > 0) {
          sp_wait(&pv_done[w * 2 + ((u - 1) & 1)], ((u - 1) >> 1) & 1, dead);  // O stands still
          tc_fence_after_sync();
          uint32_t o[16];
          tmem_ld_32x32b_x16(to, o);
          tmem_ld_wait();
#pragma unroll
          for (int g = 0; g < kSpMaxGroup; ++g) o[g] = __float_as_uint(__uint_as_float(o[g]) * alpha[g]);
          tmem_st_32x32b_x16(to, o);
          tmem_st_wait();
        }
        // the P buffer's last reader is the PV of the unit before the last
        if (u >= 2) sp_wait(&pv_done[w * 2 + h], ((u - 2) >> 1) & 1, dead);
        uint8_t* pdst = own_p(w, h);
#pragma unroll
        for (int g = 0; g < kSpMaxGroup; ++g)
          if (g < G) {
            const T pt = from_f32<T>(fast_exp2(s[g] - m_ref[g]));
            l_thr[g] += to_f32<T>(pt);
            *reinterpret_cast<T*>(pdst + sp_p_off(g, row)) = pt;
          }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w * 2 + h]);
      }
#pragma unroll
      for (int g = 0; g < kSpMaxGroup; ++g)
        if (g < G) put(rounds, g, warp_sum(l_thr[g]));
      sp_bar(1 + w);
      const bool first = it.tile0 == 0;
      const int64_t at = first ? static_cast<int64_t>(p.batch + it.b0) * p.Hq + it.hk * G
                               : (static_cast<int64_t>(blockIdx.x) * 2 + w) * kSpM;
      if (row == 0) {
        float2* ml = reinterpret_cast<float2*>(first ? p.ml_first : p.ml_next) + at;
#pragma unroll
        for (int g = 0; g < kSpMaxGroup; ++g)
          if (g < G) {
            const float4 x = red[(rounds & 1) * kSpMaxGroup + g];
            ml[g] = make_float2(m_ref[g], (x.x + x.y) + (x.z + x.w));
          }
        // behind the CTA of the first part an item is its CTA's first, so it is warpgroup 0's there
        if (first) p.notes[(p.batch + it.b0) * p.Hk + it.hk] = it.note(range, false, 0);
      }
      ++rounds;
      sp_wait(&pv_done[w * 2 + ((u - 1) & 1)], ((u - 1) >> 1) & 1, dead);
      tc_fence_after_sync();
      uint32_t r[16];
      tmem_ld_32x32b_x16(to, r);
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[w]);
      float* o = (first ? p.o_first : p.o_next) + at * kSpD + row;
#pragma unroll
      for (int g = 0; g < kSpMaxGroup; ++g)
        if (g < G) o[g * kSpD] = __uint_as_float(r[g]);
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
// A part of sum 0 has scores of -inf only, or no tile at all, and takes no part; a sum that is not a number does.  0 / 0 where
// no part is left, 0 where there was none.
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
  const int halves = ns.y >> 15 & 1, shared = (ns.y & 0x7fff) << halves, parts = shared + (no.y & 0x7fff);
  // the i-th part's row among those by batch row (its first) or by CTA
  auto place = [&](int i, bool& first) {
    const bool own = i >= shared;
    const int2 n = own ? no : ns;
    const int k = own ? i - shared : i >> halves, second = own ? 0 : i & halves;
    first = k == 0;
    return first ? static_cast<int64_t>(own ? 1 : 2 * second) * rows + row
                 : (static_cast<int64_t>(n.x) + k) * 2 * kSpM + second * kSpM + (n.y >> 16) + (h - hk * p.group);
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
        const float top = fmaxf(M, warp_max(ml.y != 0.f ? ml.x : -INFINITY));
        const float keep = den != 0.f ? fast_exp2(M - top) : 0.f;
        wt = ml.y != 0.f ? fast_exp2(ml.x - top) : -1.f;
        den = den * keep + warp_sum(ml.y != 0.f ? wt * ml.y : 0.f);
        acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
        M = top;
      }
#pragma unroll
      for (int k = 0; k < kSjParts; ++k)
        if (j0 + k < here) {
          const float f = __shfl_sync(0xffffffffu, wt, j0 + k);
          if (!(f < 0.f)) {  // (a part of sum 0 may have no columns)
            acc.x = fmaf(f, v[k].x, acc.x);
            acc.y = fmaf(f, v[k].y, acc.y);
            acc.z = fmaf(f, v[k].z, acc.z);
            acc.w = fmaf(f, v[k].w, acc.w);
          }
        }
    }
  }
  const float inv = parts > 0 ? 1.f / den : 0.f;
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
  return (3 * b * num_q_heads + static_cast<int64_t>(device_sm_count_cached()) * 2 * kSpM) * (kSpD + 2) * 4 + 2 * b * num_kv_heads * 8;
}

// Whether reading the shared keys once is the faster way, from what the host knows.
struct SharedTokens {
  int64_t group, member;  // that the groups share; that their members would read of them one by one
  int64_t own, longest;   // that every request reads by itself either way; of the longest request
};
// The weights fit 325 shapes of equal groups measured both ways (2 to 256 requests in 1 to 32 groups, 128 to 16384 shared tokens,
// 64 own, bf16, four head layouts): the choice takes 0.5% longer than the better way on average, 24% at worst.  A tile of 128
// shared keys costs an SM 1.2 here and each member 0.7 there (mostly from L2); requests that there are cut over many SMs cost 0.4
// per part and query head in their merge; the longer start, the join and the shorter ranges cost 6 here, and 0.0008 per request
// and kv head.  A tile of own keys beyond the 64 costs 0.25 more here, 1.46 there.  There, items that are not cut (attn_decode.cu
// has the rule) wait for the longest one, 0.7 a tile; here the list is cut evenly.
// 620 batches of unequal groups beside up to 400 requests of no group (2 to 100 members, 128 to 32768 shared tokens, own ones of 1
// to 16000, seven head layouts): 0.9% longer than the better way on average, 74% at worst (57 requests on 2 kv heads, one of 13176 tokens).
// us by request / shared.  32 / 8 heads, one group: 64 members of 256 tokens 18.8 / 18.9, 512: 24.1 / 21.3, 1024: 33.8 / 22.0,
// 16384: 388 / 41.5; 8 of 1024: 14.3 / 15.5, 4096: 25.1 / 22.7, 16384: 57.0 / 31.2; 4 of 4096: 21.6 / 22.0.  Groups of two: 8
// of 4096: 46.3 / 39.8, of 16384: 164 / 100; 32 of 2048: 62.3 / 67.9, of 4096: 161 / 107.  16 / 2 heads, 2 of 512: 17.6 / 15.1,
// of 4096: 53.1 / 24.6.  32 / 32 heads, 16 of 256: 17.7 / 17.6, of 1024: 32.3 / 21.3.  64 of 8192 beside n requests of 500 tokens,
// 32 / 8 heads: n = 0 184 / 39, 64: 197 / 64, 100: 209 / 78, 400: 305 / 188; 16 of 8192 beside 100: 86 / 78; 8 of 4096 beside 100
// of 2000: 143 / 170; 126 of 128 and 2 of 16384: 113 / 57.
static double shared_saves(int64_t batch, const SharedTokens& t, int num_q_heads, int num_kv_heads, int sms) {
  const double pairs = static_cast<double>(batch) * num_kv_heads, per_sm = static_cast<double>(num_kv_heads) / kSpTile / sms;
  double there = per_sm * 0.7 * t.member;
  if (pairs < sms) {
    const double parts = sms / pairs < t.longest / 256. ? sms / pairs : t.longest / 256.;
    there += 0.4 * (num_q_heads / num_kv_heads) * parts;
  } else {
    const double units = pairs + static_cast<double>(num_kv_heads) * (t.member + t.own) / kSpTile;
    const double rounds = static_cast<double>((static_cast<int64_t>(pairs) + sms - 1) / sms);
    const double chain = 0.7 * t.longest / kSpTile - per_sm * 1.46 * t.own;
    if ((rounds / pairs - 1. / sms) * units < 18. && chain > there) there = chain;
  }
  const double own = static_cast<double>(t.own) - 64. * batch;
  return there - per_sm * (1.2 * t.group + (own > 0. ? 0.25 * own : 0.)) - (6.0 + 0.0008 * pairs * 148 / sms);
}

}  // namespace spd

using namespace spd;

extern "C" {

int64_t spd_attn_decode_shared_workspace_bytes(int64_t max_batch, int num_q_heads, int num_kv_heads, int head_dim) {
  if (max_batch < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim != kSpD) return 0;
  // (one behind the other: a call of the one kind leaves the counters of the other at zero)
  return decode_bytes(max_batch, num_q_heads, num_kv_heads) + part_bytes(max_batch, num_q_heads, num_kv_heads);
}

int spd_attn_decode_shared_saves_tokens(int64_t batch, int64_t num_groups, int64_t group_tokens, int64_t member_tokens,
                                        int64_t own_tokens, int64_t longest, int num_q_heads, int num_kv_heads, int head_dim,
                                        int sm_budget) {
  if (batch < 2 || batch > kSpRows || num_groups < 1 || num_groups > kSpGroups || group_tokens < kSpTile || member_tokens < group_tokens ||
      num_kv_heads < 1 || num_q_heads < num_kv_heads || head_dim != kSpD)
    return 0;
  const int device_sms = device_sm_count_cached();
  const double us = shared_saves(batch, SharedTokens{group_tokens, member_tokens, own_tokens, longest}, num_q_heads, num_kv_heads,
                                 sm_budget > 0 && sm_budget < device_sms ? sm_budget : device_sms);
  return us <= 0. ? 0 : us >= 1e9 ? 1000000000 : static_cast<int>(us) + 1;
}

// as if all requests were in groups of one size that share max_shared_len tokens, with 64 of their own
int spd_attn_decode_shared_saves(int64_t batch, int64_t num_groups, int64_t max_shared_len, int num_q_heads, int num_kv_heads,
                                 int head_dim, int sm_budget) {
  if (batch < 2 || batch > kSpRows || num_groups < 1 || num_groups > batch || max_shared_len < kSpTile) return 0;
  const int64_t most = max_shared_len < (1ll << 40) ? max_shared_len : 1ll << 40;
  return spd_attn_decode_shared_saves_tokens(batch, num_groups, num_groups * most, batch * most, 64 * batch, most, num_q_heads,
                                             num_kv_heads, head_dim, sm_budget);
}

int spd_attn_decode_shared_pays(int64_t batch, int64_t num_groups, int64_t max_shared_len, int num_q_heads, int num_kv_heads,
                                int head_dim, int sm_budget) {
  return spd_attn_decode_shared_saves(batch, num_groups, max_shared_len, num_q_heads, num_kv_heads, head_dim, sm_budget) > 0;
}

}  // extern "C"

static int attn_decode_shared(void* out, const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
                              const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* group_indptr,
                              const int64_t* shared_lens, int64_t batch, int64_t num_groups, bool pays, int64_t pool_slots,
                              int num_q_heads, int num_kv_heads, int head_dim, int64_t q_stride, int64_t out_stride,
                              int64_t req_to_token_stride, float sm_scale, int dtype, void* workspace, int64_t workspace_bytes,
                              int sm_budget, spd_stream_t stream) {
  if (int rc = check_attn_args("spd_attn_decode_shared", out, q, k_pool, v_pool, req_to_token, req_pool_indices, num_q_heads,
                               num_kv_heads, head_dim, q_stride, out_stride))
    return rc;
  SPD_REQUIRE(seq_lens && batch >= 0 && num_groups >= 0 && pool_slots > 0 && pool_slots < (1ll << 31) &&
                  (num_groups == 0 || (group_indptr && shared_lens)),
              SPD_E_BADARG, "spd_attn_decode_shared: bad lengths or groups");
  SPD_REQUIRE(head_dim == kSpD, SPD_E_SHAPE, "spd_attn_decode_shared: head_dim must be 128 (got %d)", head_dim);
  if (batch == 0) return 0;
  const int64_t need = spd_attn_decode_shared_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim);
  SPD_REQUIRE(workspace && workspace_bytes >= need, SPD_E_WORKSPACE, "spd_attn_decode_shared: workspace too small (%lld bytes)",
              (long long)workspace_bytes);
  SPD_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, SPD_E_ALIGN, "spd_attn_decode_shared: workspace must be 16-B aligned");
  const int device_sms = device_sm_count_cached();
  const int sms = sm_budget > 0 && sm_budget < device_sms ? sm_budget : device_sms;
  // What the list can cost at most: no request has more tokens than its row of the page table has entries.
  const int64_t most = batch * num_kv_heads * (kCostOwnTile * (req_to_token_stride / kSpTile + 1) + kCostShared + kCostOwn);
  // Every request reads its own pages where nothing can be shared or it does not pay, where a plan would not hold the batch or
  // its 32-bit costs the list, and where the scale is not positive (the maximum of raw scores serves the scaled ones only there).
  if (!(sm_scale > 0.f) || most > INT_MAX / 2 || !pays)
    return spd_attn_decode_paged_own(out, q, k_pool, v_pool, req_to_token, req_pool_indices, seq_lens, batch, num_q_heads,
                                     num_kv_heads, head_dim, q_stride, out_stride, req_to_token_stride, sm_scale, dtype, workspace,
                                     workspace_bytes, sm_budget, stream);
  SharedParams p{};
  if (int rc = wait_flag(&p.wait_expired)) return rc;
  p.req_to_token = req_to_token;
  p.req_pool_indices = req_pool_indices;
  p.seq_lens = seq_lens;
  p.batch = static_cast<int>(batch);
  p.Hq = num_q_heads;
  p.Hk = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.rtt_stride = req_to_token_stride;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.group_indptr = group_indptr;
  p.shared_lens = shared_lens;
  p.groups = static_cast<int>(num_groups);
  p.mpt = kSpM / p.group;
  const int64_t rows = batch * num_q_heads;
  p.o_first = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_bytes(batch, num_q_heads, num_kv_heads));
  p.o_next = p.o_first + 3 * rows * kSpD;
  p.ml_first = p.o_next + static_cast<int64_t>(sms) * 2 * kSpM * kSpD;
  p.ml_next = p.ml_first + 3 * rows * 2;
  p.notes = reinterpret_cast<int2*>(p.ml_next + static_cast<int64_t>(sms) * 2 * kSpM * 2);
  // q as [batch][heads][128]: a box of mpt members and a kv head's query heads is a tile of mpt x group rows
  CUtensorMap tq, tq1;
  SpBoxes tk, tv;
  const uint64_t dims[3] = {kSpD, static_cast<uint64_t>(num_q_heads), static_cast<uint64_t>(batch)};
  const uint64_t strides[2] = {kSpD, static_cast<uint64_t>(q_stride)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.mpt)}, box1[3] = {64, box[1], 1};
  if (int rc = make_tmap_sw128(&tq, q, 3, dims, strides, box)) return rc;
  if (int rc = make_tmap_sw128(&tq1, q, 3, dims, strides, box1)) return rc;
  const uint64_t row_elems = static_cast<uint64_t>(num_kv_heads) * kSpD, slots = static_cast<uint64_t>(pool_slots);
  constexpr int kBoxes[5] = {128, 64, 32, 16, 1};
  for (int i = 0; i < 5; ++i) {
    if (int rc = get_tmap(&tk.rows[i], k_pool, slots, row_elems, row_elems, kBoxes[i])) return rc;
    if (int rc = get_tmap(&tv.rows[i], v_pool, slots, row_elems, row_elems, kBoxes[i])) return rc;
  }
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

extern "C" {

int spd_attn_decode_shared(void* out, const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
                           const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* group_indptr,
                           const int64_t* shared_lens, int64_t batch, int64_t num_groups, int64_t max_shared_len,
                           int64_t pool_slots, int num_q_heads, int num_kv_heads, int head_dim, int64_t q_stride, int64_t out_stride,
                           int64_t req_to_token_stride, float sm_scale, int dtype, void* workspace, int64_t workspace_bytes,
                           int sm_budget, spd_stream_t stream) {
  SPD_REQUIRE(max_shared_len >= 0, SPD_E_BADARG, "spd_attn_decode_shared: bad max_shared_len");
  return attn_decode_shared(out, q, k_pool, v_pool, req_to_token, req_pool_indices, seq_lens, group_indptr, shared_lens, batch, num_groups,
                            spd_attn_decode_shared_pays(batch, num_groups, max_shared_len, num_q_heads, num_kv_heads, head_dim, sm_budget),
                            pool_slots, num_q_heads, num_kv_heads, head_dim, q_stride, out_stride, req_to_token_stride, sm_scale, dtype,
                            workspace, workspace_bytes, sm_budget, stream);
}

int spd_attn_decode_shared_tokens(void* out, const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
                                  const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* group_indptr,
                                  const int64_t* shared_lens, int64_t batch, int64_t num_groups, int64_t group_tokens,
                                  int64_t member_tokens, int64_t own_tokens, int64_t longest, int64_t pool_slots, int num_q_heads,
                                  int num_kv_heads, int head_dim, int64_t q_stride, int64_t out_stride, int64_t req_to_token_stride, float sm_scale, int dtype,
                                  void* workspace, int64_t workspace_bytes, int sm_budget, spd_stream_t stream) {
  SPD_REQUIRE(group_tokens >= 0 && member_tokens >= 0 && own_tokens >= 0 && longest >= 0, SPD_E_BADARG, "spd_attn_decode_shared: bad token counts");
  return attn_decode_shared(out, q, k_pool, v_pool, req_to_token, req_pool_indices, seq_lens, group_indptr, shared_lens, batch, num_groups,
                            spd_attn_decode_shared_saves_tokens(batch, num_groups, group_tokens, member_tokens, own_tokens, longest,
                                                                num_q_heads, num_kv_heads, head_dim, sm_budget) > 0,
                            pool_slots, num_q_heads, num_kv_heads, head_dim, q_stride, out_stride, req_to_token_stride, sm_scale, dtype,
                            workspace, workspace_bytes, sm_budget, stream);
}

}  // extern "C"
