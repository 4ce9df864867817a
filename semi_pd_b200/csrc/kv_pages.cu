// Rows of the cache that move between slots, in all layers' pools at once: copying, forking and compacting requests.
// The pools are "planes" of equally long rows, one row per slot; a request's tokens are its entries of req_to_token.
//
// Nothing is computed: a call moves 2 x rows x bytes of a token and should take what those bytes take.  A block owns a few
// rows of one plane: their slots are looked up once, in parallel, into shared memory, and its threads then walk the rows'
// 16-byte pieces as one list, kKvUnroll of them loaded before the first is stored.  Rows of more than kKvPart bytes (a request's
// recurrent state is one row) are taken in parts, each as a plane of its own, so that they too are spread over the SMs (one
// request's states of 2 MB in 24 layers, 101 MB: 16.2 us, 6.2 TB/s).
// Measured: 12001 latent rows in 27 layers (747 MB) copied in 118 us, 6.3 TB/s; 16 requests' fp32 rows compacted (1.89 GB) in 292,
// 6.5; 8 parents with 16 children each forked (568 MB, nearly all of it written) in 104 - 110, 5.2.  A plain copy has 6.56.
#include "common.cuh"
#include "prefill_tiles.cuh"
#include "ptx.cuh"

namespace spd {

constexpr int kKvThreads = 256;
constexpr int kKvRows = 64;    // rows of a block at most
constexpr int kKvUnroll = 4;
constexpr int kKvSets = 64;
constexpr int kKvPart = 32768;       // bytes of a row that a block takes at most, a multiple of any piece
constexpr int64_t kKvRow = 1 << 30;  // of a row
// Children of a fork whose rows a block stores after loading them once: those of one parent and length, which stand together
// in the lists, up to a multiple of kKvKin.  They are the fastest index of the grid, so that the next block of the parent finds
// its rows in L2.  us with 1 / 2 / 4: 8 parents of 16 children, 567 MB at least, 138 / 104 / 107; 64 parents of one child
// 145 / 134 / 165; one child, 16 MB, 7.2 / 7.1 / 7.7.  With the children slowest and 1: 165 (8 parents of 16).
constexpr int kKvKin = 2;

struct KvSet {
  char* base;
  int64_t stride;     // bytes between planes
  int64_t rows;       // slots
  int64_t row_bytes;
  int first;          // planes of the sets before
  int parts;          // planes that a buffer's rows are taken in
  uint32_t pieces_m, pieces_s;  // division by the pieces of a row, or of a part
};
struct KvPlanes {
  int sets, planes;   // (parts count as planes)
  KvSet set[kKvSets];
};

// A block's place in its call: rows [chunk x rows of a block, ...), plane (the last one: the page table), child of a fork.
struct KvPlace {
  int64_t chunk;
  int plane, child, chunks;
};
// where the rows of a call lie
struct KvCopyRows {
  static constexpr bool kChildren = false, kParts = true;
  const int64_t *src, *dst;
  int64_t n;
};
struct KvForkRows {
  static constexpr bool kChildren = true, kParts = false;  // (tokens' rows are short, and the parts cost 8 of 106 us)
  const int64_t *parents, *children, *lens, *tail;
  int32_t* table;
  int64_t stride, requests, width;
  int run_len, n;
};
struct KvCompactRows {
  static constexpr bool kChildren = false, kParts = true;
  const int64_t *src, *dst, *keep, *indptr, *loc;
  int32_t* table;
  int64_t stride, requests, width, n, total;
};

// a child that has a page-table row to become a copy in
__device__ __forceinline__ bool kv_child(const KvForkRows& r, int64_t child, int64_t parent) {
  return child >= 0 && child < r.requests && child != parent;
}
// the last request whose first row is not behind row j
__device__ __forceinline__ int64_t kv_request(const int64_t* indptr, int64_t n, int64_t j) {
  int64_t lo = 0, hi = n - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (indptr[mid] <= j) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// rows [first, first + count) of this block -> (source, destination) slots; a row with a slot of -1 stays as it is
__device__ __forceinline__ int kv_rows(const KvCopyRows& r, const KvPlace& at, int, int per_block, int64_t* src, int64_t* dst) {
  const int64_t first = at.chunk * per_block;
  const int count = static_cast<int>(min(static_cast<int64_t>(per_block), r.n - first));
  for (int i = threadIdx.x; i < count; i += kKvThreads) {
    src[i] = r.src[first + i];
    dst[i] = r.dst[first + i];
  }
  return count;
}
// (kin children of one parent and length from at.child on: dst[k x kKvRows + i])
__device__ __forceinline__ int kv_rows(const KvForkRows& r, const KvPlace& at, int kin, int per_block, int64_t* src, int64_t* dst) {
  const int64_t parent = r.parents[at.child], len = r.lens[at.child];
  int64_t tail[kKvKin];  // (read before anything is stored: a store keeps the loads behind it waiting)
#pragma unroll
  for (int k = 0; k < kKvKin; ++k) tail[k] = at.child + k < r.n ? r.tail[at.child + k] : -1;
  if (parent < 0 || parent >= r.requests || len < 0 || len > r.width) return 0;
  const int64_t full = len / r.run_len * r.run_len, first = at.chunk * per_block;
  const int count = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(per_block), len - full - first)));
  for (int i = threadIdx.x; i < count; i += kKvThreads) {
    bool out[kKvKin];  // a child without a page-table row: beside the load of the entry and by these threads only (all: 4 of 106 us)
#pragma unroll
    for (int k = 0; k < kKvKin; ++k) out[k] = k < kin && !kv_child(r, r.children[at.child + k], parent);
    src[i] = r.table[parent * r.stride + full + first + i];
#pragma unroll
    for (int k = 0; k < kKvKin; ++k)
      if (k < kin) dst[k * kKvRows + i] = out[k] ? -1 : tail[k] + first + i;
  }
  return count;
}
__device__ __forceinline__ int kv_rows(const KvCompactRows& r, const KvPlace& at, int, int per_block, int64_t* src, int64_t* dst) {
  const int64_t first = at.chunk * per_block;
  const int count = static_cast<int>(min(static_cast<int64_t>(per_block), r.total - first));
  for (int i = threadIdx.x; i < count; i += kKvThreads) {
    const int64_t j = first + i, request = r.src[kv_request(r.indptr, r.n, j)], pos = r.keep[j];
    const bool ok = request >= 0 && request < r.requests && pos >= 0 && pos < r.width;
    src[i] = ok ? r.table[request * r.stride + pos] : -1;
    dst[i] = r.loc[j];
  }
  return count;
}

// the page table's part of a call
__device__ __forceinline__ void kv_table(const KvCopyRows&, const KvPlace&) {}
__device__ __forceinline__ void kv_table(const KvForkRows& r, const KvPlace& at) {
  const int64_t parent = r.parents[at.child], child = r.children[at.child], len = r.lens[at.child], tail = r.tail[at.child];
  if (parent < 0 || parent >= r.requests || !kv_child(r, child, parent) || len < 0 || len > r.width) return;
  const int64_t full = len / r.run_len * r.run_len;
  const int32_t* from = r.table + parent * r.stride;
  int32_t* to = r.table + child * r.stride;
  for (int64_t i = at.chunk * kKvThreads + threadIdx.x; i < len; i += static_cast<int64_t>(at.chunks) * kKvThreads)
    to[i] = i < full ? from[i] : static_cast<int32_t>(tail + i - full);
}
__device__ __forceinline__ void kv_table(const KvCompactRows& r, const KvPlace& at) {
  for (int64_t j = at.chunk * kKvThreads + threadIdx.x; j < r.total; j += static_cast<int64_t>(at.chunks) * kKvThreads) {
    const int64_t i = kv_request(r.indptr, r.n, j), pos = j - r.indptr[i], request = r.dst[i];
    if (request >= 0 && request < r.requests && pos >= 0 && pos < r.width) r.table[request * r.stride + pos] = static_cast<int32_t>(r.loc[j]);
  }
}

// How many children from this one on the block stores to: those of its parent and length up to a multiple of kKvKin; 0 where an
// earlier child's block does it.
__device__ __forceinline__ int kv_kin(const KvForkRows& r, int child) {
  const int first = child / kKvKin * kKvKin;
  int64_t parent[kKvKin], len[kKvKin];
#pragma unroll
  for (int k = 0; k < kKvKin; ++k) {
    parent[k] = first + k < r.n ? r.parents[first + k] : -1;
    len[k] = first + k < r.n ? r.lens[first + k] : -1;
  }
  int kin = 0;
#pragma unroll
  for (int k = 0; k < kKvKin; ++k) {
    if (first + k >= r.n) break;
    const bool new_run = k == 0 || parent[k] != parent[k - 1] || len[k] != len[k - 1];
    if (first + k == child) {
      if (!new_run) return 0;
      kin = 1;
    } else if (first + k > child) {
      if (new_run) break;
      ++kin;
    }
  }
  return kin;
}
template <typename Rows> __device__ __forceinline__ int kv_kin(const Rows&, int) { return 1; }

// V: the piece that a thread moves at a time, 16 bytes where rows and pointers allow it
template <typename V, typename Rows>
__global__ void __launch_bounds__(kKvThreads) kv_move_kernel(const __grid_constant__ KvPlanes pl, const Rows rows, int per_block) {
  __shared__ int64_t s_src[kKvRows], s_dst[(Rows::kChildren ? kKvKin : 1) * kKvRows];
  griddep_launch_dependents();
  griddep_wait();
  const KvPlace at = Rows::kChildren ? KvPlace{blockIdx.y, static_cast<int>(blockIdx.z), static_cast<int>(blockIdx.x), static_cast<int>(gridDim.y)}
                                     : KvPlace{blockIdx.x, static_cast<int>(blockIdx.y), 0, static_cast<int>(gridDim.x)};
  if (at.plane == pl.planes) {
    kv_table(rows, at);
    return;
  }
  const int kin = kv_kin(rows, at.child);
  if (kin == 0) return;
  const int count = kv_rows(rows, at, kin, per_block, s_src, s_dst);
  if (count <= 0) return;
  int si = 0;
  while (si + 1 < pl.sets && at.plane >= pl.set[si + 1].first) ++si;
  const KvSet& set = pl.set[si];
  int pieces, last;
  char* plane;
  if constexpr (Rows::kParts) {
    const int rel = at.plane - set.first, buffer = set.parts == 1 ? rel : rel / set.parts, part = rel - buffer * set.parts;
    pieces = static_cast<int>((set.parts == 1 ? set.row_bytes : static_cast<int64_t>(kKvPart)) / sizeof(V));
    // (the last part is shorter)
    last = static_cast<int>(min(static_cast<int64_t>(pieces), (set.row_bytes - static_cast<int64_t>(part) * kKvPart) / static_cast<int64_t>(sizeof(V))));
    plane = set.base + buffer * set.stride + static_cast<int64_t>(part) * kKvPart;
  } else {
    pieces = last = static_cast<int>(set.row_bytes / sizeof(V));
    plane = set.base + (at.plane - set.first) * set.stride;
  }
  __syncthreads();
  const int total = count * pieces;
  for (int i0 = threadIdx.x; i0 < total; i0 += kKvThreads * kKvUnroll) {
    V v[kKvUnroll];
    int row[kKvUnroll], piece[kKvUnroll];
#pragma unroll
    for (int k = 0; k < kKvUnroll; ++k) {
      const int i = i0 + k * kKvThreads;
      row[k] = -1;
      if (i < total) {
        const int r = fastdiv(i, set.pieces_m, set.pieces_s);
        const int64_t s = s_src[r];
        piece[k] = i - r * pieces;
        if (s >= 0 && s < set.rows && (!Rows::kParts || piece[k] < last)) {
          row[k] = r;
          const V* from = reinterpret_cast<const V*>(plane + s * set.row_bytes) + piece[k];
          v[k] = Rows::kChildren ? *from : __ldcs(from);  // (a parent's rows are read again)
        }
      }
    }
    for (int c = 0; c < kin; ++c) {
#pragma unroll
      for (int k = 0; k < kKvUnroll; ++k) {
        if (row[k] < 0) continue;
        const int64_t d = s_dst[c * kKvRows + row[k]];
        if (d >= 0 && d < set.rows) *(reinterpret_cast<V*>(plane + d * set.row_bytes) + piece[k]) = v[k];
      }
    }
  }
}

// req_to_token rows of requests that were compacted in place: after the kernel that reads them
__global__ void __launch_bounds__(kKvThreads) kv_table_kernel(const KvCompactRows rows) {
  griddep_launch_dependents();
  griddep_wait();
  kv_table(rows, KvPlace{blockIdx.x, 0, 0, static_cast<int>(gridDim.x)});
}

// The plane sets as the kernel takes them, and the bytes of a piece that suits all of them (0 and an error otherwise).
static int kv_planes(const char* fn, const spd_kv_planes_t* sets, int num_sets, bool parts, KvPlanes& pl, int& piece) {
  SPD_REQUIRE(sets && num_sets > 0 && num_sets <= kKvSets, SPD_E_BADARG, "%s: 1 to %d plane sets (got %d)", fn, kKvSets, num_sets);
  pl.sets = num_sets;
  pl.planes = 0;
  piece = 16;
  for (int i = 0; i < num_sets; ++i) {
    const spd_kv_planes_t& s = sets[i];
    SPD_REQUIRE(s.base && s.planes > 0 && s.rows > 0 && s.row_bytes > 0 && s.plane_stride >= 0, SPD_E_BADARG, "%s: bad plane set", fn);
    SPD_REQUIRE(s.row_bytes % 2 == 0 && s.plane_stride % 2 == 0 && (reinterpret_cast<uintptr_t>(s.base) & 1) == 0, SPD_E_ALIGN,
                "%s: rows of an even number of bytes", fn);
    SPD_REQUIRE(s.row_bytes <= kKvRow, SPD_E_SHAPE, "%s: rows of 1 GB at most", fn);
    const uint64_t bits = reinterpret_cast<uintptr_t>(s.base) | s.row_bytes | s.plane_stride;
    while (bits % piece) piece >>= 1;
    pl.set[i].base = static_cast<char*>(s.base);
    pl.set[i].stride = s.plane_stride;
    pl.set[i].rows = s.rows;
    pl.set[i].row_bytes = s.row_bytes;
    pl.set[i].first = pl.planes;
    pl.set[i].parts = parts ? static_cast<int>((s.row_bytes + kKvPart - 1) / kKvPart) : 1;
    const int64_t planes = pl.planes + static_cast<int64_t>(s.planes) * pl.set[i].parts;
    SPD_REQUIRE(planes < 65535, SPD_E_SHAPE, "%s: too many planes (a row of more than %d bytes counts once for every %d)", fn, kKvPart,
                kKvPart);
    pl.planes = static_cast<int>(planes);
  }
  for (int i = 0; i < num_sets; ++i)
    fastdiv_magic(static_cast<uint32_t>((pl.set[i].parts == 1 ? pl.set[i].row_bytes : kKvPart) / piece), pl.set[i].pieces_m, pl.set[i].pieces_s);
  return 0;
}

// Rows of a block: 32 KB of them, fewer where the call would not give every SM four blocks, and 4 KB at least.
static int kv_rows_per_block(const KvPlanes& pl, int64_t rows) {
  int64_t bytes = 0;
  for (int i = 0; i < pl.sets; ++i) bytes = bytes > pl.set[i].row_bytes ? bytes : pl.set[i].row_bytes;
  if (bytes > kKvPart) bytes = kKvPart;  // (a part; without parts it is one row a block either way)
  int64_t per = (32768 + bytes - 1) / bytes;
  const int64_t spread = rows * pl.planes / (4 * device_sm_count_cached()), least = (4096 + bytes - 1) / bytes;
  if (per > spread) per = spread;
  if (per < least) per = least;
  return static_cast<int>(per < 1 ? 1 : per > kKvRows ? kKvRows : per);
}

template <typename Rows>
static int kv_move(const KvPlanes& pl, int piece, const Rows& rows, int64_t n, int per_block, int64_t children, bool table, cudaStream_t st) {
  const unsigned chunks = static_cast<unsigned>((n + per_block - 1) / per_block), planes = static_cast<unsigned>(pl.planes + (table ? 1 : 0));
  const dim3 grid = Rows::kChildren ? dim3(static_cast<unsigned>(children), chunks, planes) : dim3(chunks, planes);
  SPD_REQUIRE(!Rows::kChildren || chunks < 65536, SPD_E_SHAPE, "spd_kv_fork: runs of too many tokens");
#define SPD_KV_MOVE(V) SPD_CUDA(launch(kv_move_kernel<V, Rows>, grid, dim3(kKvThreads), 0, st, pdl_enabled(), pl, rows, per_block))
  switch (piece) {
    case 16: SPD_KV_MOVE(uint4); break;
    case 8: SPD_KV_MOVE(uint2); break;
    case 4: SPD_KV_MOVE(uint32_t); break;
    default: SPD_KV_MOVE(unsigned short);
  }
#undef SPD_KV_MOVE
  return 0;
}

}  // namespace spd

using namespace spd;

extern "C" {

int spd_kv_copy(const spd_kv_planes_t* sets, int num_sets, const int64_t* src, const int64_t* dst, int64_t n, spd_stream_t stream) {
  KvPlanes pl;
  int piece;
  if (int rc = kv_planes("spd_kv_copy", sets, num_sets, KvCopyRows::kParts, pl, piece)) return rc;
  SPD_REQUIRE(n >= 0 && n < (1ll << 31) && (n == 0 || (src && dst)), SPD_E_BADARG, "spd_kv_copy: bad slots");
  if (n == 0) return 0;
  return kv_move(pl, piece, KvCopyRows{src, dst, n}, n, kv_rows_per_block(pl, n), 1, false, as_stream(stream));
}

int spd_kv_fork(const spd_kv_planes_t* sets, int num_sets, int32_t* req_to_token, int64_t req_to_token_stride, int64_t requests,
                int64_t max_tokens, const int64_t* parents, const int64_t* children, const int64_t* seq_lens, const int64_t* tail_slots,
                int64_t n, int run_len, spd_stream_t stream) {
  KvPlanes pl;
  int piece;
  if (int rc = kv_planes("spd_kv_fork", sets, num_sets, KvForkRows::kParts, pl, piece)) return rc;
  SPD_REQUIRE(req_to_token && n >= 0 && (n == 0 || (parents && children && seq_lens && tail_slots)) && requests > 0 &&
                  max_tokens > 0 && run_len > 0 && req_to_token_stride >= max_tokens,
              SPD_E_BADARG, "spd_kv_fork: bad arguments");
  SPD_REQUIRE(n < 65536, SPD_E_SHAPE, "spd_kv_fork: at most 65535 children (got %lld)", (long long)n);
  if (n == 0) return 0;
  const KvForkRows rows{parents, children, seq_lens, tail_slots, req_to_token, req_to_token_stride, requests, max_tokens, run_len, static_cast<int>(n)};
  return kv_move(pl, piece, rows, run_len - 1 > 0 ? run_len - 1 : 1, kv_rows_per_block(pl, n * run_len / 2), n, true, as_stream(stream));
}

int spd_kv_compact(const spd_kv_planes_t* sets, int num_sets, int32_t* req_to_token, int64_t req_to_token_stride, int64_t requests,
                   int64_t max_tokens, const int64_t* src_requests, const int64_t* dst_requests, const int64_t* keep,
                   const int64_t* keep_indptr, const int64_t* loc, int64_t n, int64_t total, int write_table, spd_stream_t stream) {
  KvPlanes pl;
  int piece;
  if (int rc = kv_planes("spd_kv_compact", sets, num_sets, KvCompactRows::kParts, pl, piece)) return rc;
  SPD_REQUIRE(req_to_token && n >= 0 && total >= 0 && total < (1ll << 31) && requests > 0 && max_tokens > 0 &&
                  req_to_token_stride >= max_tokens && (n == 0 || total == 0 || (src_requests && keep && keep_indptr && loc)),
              SPD_E_BADARG, "spd_kv_compact: bad arguments");
  if (n == 0 || total == 0) return 0;
  KvCompactRows rows{src_requests, dst_requests, keep, keep_indptr, loc, req_to_token, req_to_token_stride, requests, max_tokens, n, total};
  if (int rc = kv_move(pl, piece, rows, total, kv_rows_per_block(pl, total), 1, write_table && dst_requests, as_stream(stream))) return rc;
  if (write_table && !dst_requests) {
    rows.dst = src_requests;
    const int64_t blocks = (total + kKvThreads - 1) / kKvThreads;
    SPD_CUDA(launch(kv_table_kernel, dim3(static_cast<unsigned>(blocks < 1024 ? blocks : 1024)), dim3(kKvThreads), 0, as_stream(stream),
                    pdl_enabled(), rows));
  }
  return 0;
}

}  // extern "C"
