// Groups of requests that continue the same tokens: what both kernels of spd_attn_decode_shared derive, each CTA for itself,
// from the groups' row offsets and the lengths.  attn_shared.cu attends to the shared keys, a whole group at once;
// attn_decode.cu to every request's own ones, and joins the two.
//
// A group shares whole tiles of 128 keys: as many as its shared slots and its shortest member (of those that are not empty)
// have.  What is left of them is read with each member's own tokens, from its own page-table row, so the split never shows in
// the result, and no query of the shared part needs a mask.
//
// The shared part's work: per group, kv head and pair of query tiles (128 rows each: `mpt` members times the query heads of a
// kv head) an item of kShItemUnits + tiles units; the list of all units is cut into equal ranges for `grid` CTAs.  An item's
// sums are kept per CTA ("parts"): by batch row where the CTA has the item's first tile, else in a place of the CTA's own, since
// of all its items only the first can have begun earlier.
#pragma once
#include <limits.h>
#include <stdint.h>

#include "ptx.cuh"

namespace spd {

constexpr int kShTile = 128;
constexpr int kShRows = 1024;    // batch rows that a plan holds
constexpr int kShGroups = 256;   // groups
constexpr int kShMaxTiles = 65535;
constexpr int kShItemUnits = 1;  // what an item's start and end cost, in tiles
constexpr int kShMinUnits = 2;

struct SharedGroups {
  const int32_t* indptr;  // [groups + 1]
  const int64_t* lens;    // [groups]
  int groups, mpt, grid;
  // o: fp32 rows of 128, before the division by l; ml: m (exponent of 2), l
  float *o_first, *ml_first;  // [batch][query heads]
  float *o_next, *ml_next;    // [grid][2 tiles][128]
};

struct SharedPlan {  // in shared memory
  int unit0[kShGroups + 1];  // units of the groups before
  uint16_t start[kShGroups], count[kShGroups], tiles[kShGroups];
  int sums[kShGroups / 32];
};

__device__ __forceinline__ int sh_pairs(int count, int mpt) { return count <= mpt ? 1 : (count + 2 * mpt - 1) / (2 * mpt); }
__device__ __forceinline__ int sh_per_cta(int total, int grid) { return max(kShMinUnits, (total + grid - 1) / grid); }

// The plan, by all threads of the CTA.  row(b, length, group or -1) is called once per batch row, by one thread, before the
// tiles are known.
template <int kThreads, typename Row>
__device__ __forceinline__ void sh_plan(const SharedGroups& sg, const int64_t* seq_lens, int batch, int Hk, SharedPlan& pl, Row row) {
  static_assert(kThreads >= kShGroups, "a thread per group");
  constexpr int kPer = (kShRows + kThreads - 1) / kThreads;
  const int g = threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int L[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x + i * kThreads;
    L[i] = b < batch ? static_cast<int>(__ldcg(reinterpret_cast<const long long*>(seq_lens) + b)) : 0;
  }
  int shared = 0, count = 0;
  if (g < sg.groups) {
    const int s = min(max(__ldcg(sg.indptr + g), 0), batch), e = min(max(__ldcg(sg.indptr + g + 1), s), batch);
    const long long n = __ldcg(reinterpret_cast<const long long*>(sg.lens) + g);
    shared = static_cast<int>(max(0ll, min(n, static_cast<long long>(kShMaxTiles) * kShTile)));
    count = e - s;
    pl.start[g] = static_cast<uint16_t>(s);
    pl.count[g] = static_cast<uint16_t>(count);
    pl.unit0[g] = INT_MAX;  // for now: the shortest member
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x + i * kThreads;
    if (b >= batch) break;
    int at = -1;
    if (L[i] > 0) {  // the last group that does not start behind the row
      int lo = 0, hi = sg.groups - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pl.start[mid] <= b) lo = mid; else hi = mid - 1;
      }
      // (groups of no rows start where the next one does: an empty one found here has the row's group before it)
      while (lo > 0 && pl.count[lo] == 0 && pl.start[lo - 1] <= b) --lo;
      if (b >= pl.start[lo] && b < pl.start[lo] + pl.count[lo]) {
        at = lo;
        atomicMin(&pl.unit0[lo], L[i]);
      }
    }
    row(b, L[i], at);
  }
  __syncthreads();
  int units = 0;
  if (g < sg.groups) {
    const int least = pl.unit0[g], tiles = count >= 2 && least != INT_MAX ? min(shared, least) / kShTile : 0;
    pl.tiles[g] = static_cast<uint16_t>(tiles);
    units = tiles > 0 ? Hk * sh_pairs(count, sg.mpt) * (tiles + kShItemUnits) : 0;
  }
  int incl = units;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31 && warp < kShGroups / 32) pl.sums[warp] = incl;
  __syncthreads();
  if (g < sg.groups) {
    int before = 0;
    for (int w = 0; w < warp; ++w) before += pl.sums[w];
    pl.unit0[g] = before + incl - units;
    if (g == sg.groups - 1) pl.unit0[sg.groups] = before + incl;
  }
  __syncthreads();
}

}  // namespace spd
