// Activations in 8-bit integers with one scale per token, alone or behind what produces them: RMS norm, the sum with a residual
// and its norm, SiLU(gate) * up.
//
//   s = max(max_k |y_k|, 1e-10) / 127,    q_k = y_k / s rounded to the nearest integer,    y_k ~ s q_k
//
// One CTA has a row and keeps it in registers between the two passes that the formula needs (the maximum, then the quotients), so
// memory sees one read of every input and one byte per output.  With a norm the maximum needs no third pass: y_k = c v_k w_k with
// one c = 1 / rms(v) for the row, so the sum of v^2 and the maximum of |v w| come out of one reduction, and c cancels out of q.
// In the fused forms y stays in 32 bits: it is never rounded to the inputs' 16-bit type in between.
//
// Rounding.  For 16-bit y the result is the exact one, halves away from zero: with X and A the integer significands (at most 11
// bits) of |y| and of the largest, y / s = 127 X 2^-e / A lies on a half or at least 1 / (2 A 2^e) beside it, relative to itself
// at least 1 / (254 X) > 2^-19; the factor 1 + 2^-20 on 127 / max is above the three roundings of 2^-24 in the way and below that
// distance, so it moves halves up and nothing else over a border.  32-bit y has no such distance, and no factor (with it SiLU * mul
// of 7800 rows of 14336 had 194 integers that 64 bits give otherwise, without 23; plain fp32 has 22).
//
// A NaN or an infinity in a row makes its scale NaN or infinite, and with it everything that the row is multiplied into: the
// maximum is taken over the bits of |y|, which order NaN above infinity above numbers.
//
// What bounds it: memory.
#include <atomic>

#include "common.cuh"
#include "ptx.cuh"

namespace spd {

enum QuantForm { kQuantPlain = 0, kQuantNorm = 1, kQuantAddNorm = 2, kQuantSilu = 3 };

struct QuantParams {
  int8_t* q;       // [rows, dim]
  float* scales;   // [rows]
  const void* x;   // [rows, dim] (SiLU: [rows, 2 dim], gate || up)
  void* residual;  // [rows, dim]: becomes x + residual
  const void* w;   // [dim]
  int64_t rows, x_stride;
  int vecs;        // pieces of 8 in a row
  float eps;
};

// Four products rounded to integers of 8 bits, halves to even.  Added to 1.5 * 2^23, whose last place is 1, a float of that size holds
// its integer in two's complement in its lowest byte; the conversion instruction goes at the rate of the exponentials (SiLU * mul of
// 8192 x 14336 in 100 us with it).
__device__ __forceinline__ uint32_t pack_s8(float a, float b, float c, float d, float k) {
  constexpr float kPlace = 12582912.f;
  const uint32_t lo = __byte_perm(__float_as_uint(fmaf(a, k, kPlace)), __float_as_uint(fmaf(b, k, kPlace)), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(fmaf(c, k, kPlace)), __float_as_uint(fmaf(d, k, kPlace)), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// max(top, |y|) that lets NaN through
__device__ __forceinline__ float max_abs(float top, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(y)));
  return r;
}

// g / (1 + e^-g).  The exponential is good to (2 + 1.2 |g|) 2^-23, for its argument is rounded at g log2 e; 1 + e^-g has that error only
// for negative g, and there g e^g falls faster than the error grows: next to the row's maximum it is below 2^-22.  With expf: as many
// integers that 64 bits give otherwise, and 8192 x 14336 in 109 us instead of 95.
__device__ __forceinline__ float silu_flushed(float g) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(-1.4426950408889634f * g)));
  return g * r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = unpack2<T>(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

// y of one piece of 8, from x and what stands beside it (the residual, or up); *sum: x + residual for memory
template <typename T, int kForm>
__device__ __forceinline__ void quant_piece(const uint4& x, const uint4& beside, const uint4& w, float (&y)[8], float& ss, float& top,
                                            uint4* sum) {
  unpack8<T>(x, y);
  float f[8];
  if constexpr (kForm == kQuantAddNorm) {
    unpack8<T>(beside, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] += f[j];
    // the new residual is rounded, what the norm sees is not
    *sum = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
  }
  if constexpr (kForm == kQuantNorm || kForm == kQuantAddNorm) {
    unpack8<T>(w, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(y[j], y[j], ss);
      y[j] *= f[j];
    }
  }
  if constexpr (kForm == kQuantSilu) {
    unpack8<T>(beside, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = silu_flushed(y[j]) * f[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max_abs(top, y[j]);
}

// The factor on y (before the norm's own) and the row's scale, from the row's maximum and sum of squares
template <int kForm>
__device__ __forceinline__ float quant_factor(uint32_t top, float ss, const QuantParams& p, float& scale) {
  constexpr bool kHasNorm = kForm == kQuantNorm || kForm == kQuantAddNorm;
  const float c = kHasNorm ? rsqrtf(ss / static_cast<float>(p.vecs * 8) + p.eps) : 1.f;
  float most = __uint_as_float(top) * c;
  most = most < 1e-10f ? 1e-10f : most;  // (NaN stays)
  scale = __fdiv_rn(most, 127.f);
  return __fdiv_rn(127.f, most) * (kHasNorm ? c : kForm == kQuantPlain ? 1.f + 0x1p-20f : 1.f);
}

__device__ __forceinline__ uint2 quant_pack(const float (&y)[8], float k) {
  return make_uint2(pack_s8(y[0], y[1], y[2], y[3], k), pack_s8(y[4], y[5], y[6], y[7], k));
}

// x as it is stays packed until it is multiplied: its maximum is taken over pairs of 16 bits, and 32 registers a thread leave room for
// 64 warps an SM.  us: 5001 x 8192 28.0 -> 19.5 (floor 18.8), 8192 x 4096 19.1 -> 15.5 with 4 pieces a thread (2: 16.5).
template <int kForm, int kThreads, int kVecs>
constexpr int quant_ctas() {  // of an SM
  return kThreads == 1024 ? 1 : (kForm == kQuantPlain || kVecs == 1 ? 2048 : kVecs == 2 ? 1536 : 1024) / kThreads;
}
template <typename T, int kForm, int kThreads, int kVecs>
__global__ void __launch_bounds__(kThreads, (quant_ctas<kForm, kThreads, kVecs>())) quant_int8_kernel(const QuantParams p) {
  constexpr bool kHasNorm = kForm == kQuantNorm || kForm == kQuantAddNorm;
  constexpr int kWarps = kThreads / 32;
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  griddep_launch_dependents();
  griddep_wait();
  const int64_t row = blockIdx.x;
  const uint4* x = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.x) + row * p.x_stride);
  uint4* r = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.residual) + row * p.x_stride);
  float y[kForm == kQuantPlain ? 1 : kVecs][8];
  uint4 raw[kForm == kQuantPlain ? kVecs : 1];
  float ss = 0.f, most = 0.f;
  uint32_t top = 0;
  if constexpr (kForm == kQuantPlain) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * kThreads;
      raw[i] = v < p.vecs ? x[v] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      constexpr uint32_t kAbs = 0x7fff7fffu;
      top = __vmaxu2(top, __vmaxu2(__vmaxu2(raw[i].x & kAbs, raw[i].y & kAbs), __vmaxu2(raw[i].z & kAbs, raw[i].w & kAbs)));
    }
    const float2 f = unpack2<T>(__vmaxu2(top, top >> 16) & 0xffffu);
    top = __float_as_uint(f.x);
  } else {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * kThreads;
      if (v < p.vecs) {
        uint4 beside{}, w{}, sum;
        if constexpr (kForm == kQuantAddNorm) beside = r[v];
        if constexpr (kForm == kQuantSilu) beside = x[p.vecs + v];
        if constexpr (kHasNorm) w = reinterpret_cast<const uint4*>(p.w)[v];
        quant_piece<T, kForm>(x[v], beside, w, y[i], ss, most, &sum);
        if constexpr (kForm == kQuantAddNorm) r[v] = sum;
      }
    }
    top = __float_as_uint(most);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (kHasNorm) ss = warp_sum(ss);
  if (lane == 0) {
    tops[warp] = top;
    if constexpr (kHasNorm) sums[warp] = ss;
  }
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < kWarps ? tops[lane] : 0u);
  if constexpr (kHasNorm) ss = warp_sum(lane < kWarps ? sums[lane] : 0.f);
  float scale;
  const float k = quant_factor<kForm>(top, ss, p, scale);
  if (threadIdx.x == 0) p.scales[row] = scale;
  uint2* q = reinterpret_cast<uint2*>(p.q) + row * p.vecs;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = threadIdx.x + i * kThreads;
    if (v < p.vecs) {
      if constexpr (kForm == kQuantPlain) {
        float f[8];
        unpack8<T>(raw[i], f);
        q[v] = quant_pack(f, k);
      } else {
        q[v] = quant_pack(y[i], k);
      }
    }
  }
}

// Many rows of 32-bit values: a CTA takes rows one after another, and while a row is worked on the next one is on its way into shared
// memory.  A thread copies and reads its own pieces, so only the row's reduction needs a barrier (in turn in two places, one a row).
// us, a CTA a row / this: SiLU, 8192 x 14336 125 / 97 (floor 90), 1300 x 14336 22.5 / 18.3 (14.2); residual and norm, 4099 x 4096
// 19.6 / 18.3 (18.0).  Results are the same bits: the sums are over the same pieces in the same order.
template <typename T, int kForm, int kThreads, int kVecs>
__global__ void __launch_bounds__(kThreads) quant_int8_rows_kernel(const QuantParams p) {
  constexpr bool kHasNorm = kForm == kQuantNorm || kForm == kQuantAddNorm;
  constexpr int kIn = kForm == kQuantNorm ? 1 : 2, kWarps = kThreads / 32;
  extern __shared__ uint4 ahead[];  // [2][kIn][kVecs][kThreads]
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[2][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch_dependents();
  griddep_wait();
  auto place = [&](int turn, int in, int i) { return ahead + ((turn * kIn + in) * kVecs + i) * kThreads + threadIdx.x; };
  auto row_of = [&](int64_t row, int in) -> uint4* {
    if (kForm == kQuantAddNorm && in == 1) return reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.residual) + row * p.x_stride);
    return const_cast<uint4*>(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.x) + row * p.x_stride)) +
           (kForm == kQuantSilu ? in * p.vecs : 0);
  };
  auto fetch = [&](int64_t row, int turn) {
    if (row < p.rows) {
#pragma unroll
      for (int in = 0; in < kIn; ++in) {
        const uint4* src = row_of(row, in);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int v = threadIdx.x + i * kThreads;
          if (v < p.vecs) cp_async16(smem_u32(place(turn, in, i)), src + v, true);
        }
      }
    }
    cp_async_commit();
  };
  fetch(blockIdx.x, 0);
  uint4 w[kHasNorm ? kVecs : 1];
  if constexpr (kHasNorm) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * kThreads;
      if (v < p.vecs) w[i] = reinterpret_cast<const uint4*>(p.w)[v];
    }
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    fetch(row + gridDim.x, turn ^ 1);
    cp_async_wait<1>();
    float y[kVecs][8];
    float ss = 0.f, most = 0.f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * kThreads;
      if (v < p.vecs) {
        uint4 beside{}, sum;
        if constexpr (kIn == 2) beside = *place(turn, 1, i);
        quant_piece<T, kForm>(*place(turn, 0, i), beside, w[kHasNorm ? i : 0], y[i], ss, most, &sum);
        if constexpr (kForm == kQuantAddNorm) row_of(row, 1)[v] = sum;
      }
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if constexpr (kHasNorm) ss = warp_sum(ss);
    if (lane == 0) {
      tops[turn][warp] = top;
      if constexpr (kHasNorm) sums[turn][warp] = ss;
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < kWarps ? tops[turn][lane] : 0u);
    if constexpr (kHasNorm) ss = warp_sum(lane < kWarps ? sums[turn][lane] : 0.f);
    float scale;
    const float k = quant_factor<kForm>(top, ss, p, scale);
    if (threadIdx.x == 0) p.scales[row] = scale;
    uint2* q = reinterpret_cast<uint2*>(p.q) + row * p.vecs;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * kThreads;
      if (v < p.vecs) q[v] = quant_pack(y[i], k);
    }
  }
}

// CTAs of a kernel that run on an SM at once, asked once for every device (kKern: kernels of one type keep apart)
template <auto kKern>
static int resident_ctas(int threads, int smem, int* out) {
  static std::atomic<int> known[64];
  int dev = 0;
  SPD_CUDA(cudaGetDevice(&dev));
  int n = known[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    SPD_CUDA(cudaFuncSetAttribute(kKern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    SPD_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kKern, threads, smem));
    known[dev & 63].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return 0;
}

template <typename T, int kForm, int kThreads, int kVecs>
static int launch_quant_sized(const QuantParams& p, int sms, cudaStream_t stream) {
  constexpr int kSmem = 2 * (kForm == kQuantNorm ? 1 : 2) * kVecs * kThreads * 16;
  if constexpr (kForm != kQuantPlain && kSmem <= 220 * 1024) {
    constexpr auto kern = quant_int8_rows_kernel<T, kForm, kThreads, kVecs>;
    int per = 0;
    if (int rc = resident_ctas<kern>(kThreads, kSmem, &per)) return rc;
    const int64_t ctas = static_cast<int64_t>(per) * sms;
    if (per > 0 && p.rows > ctas) {  // else every row has a CTA of its own at once
      SPD_CUDA(launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmem, stream, pdl_enabled(), p));
      return 0;
    }
  }
  SPD_CUDA(launch(quant_int8_kernel<T, kForm, kThreads, kVecs>, dim3(static_cast<unsigned>(p.rows)), dim3(kThreads), 0, stream,
                  pdl_enabled(), p));
  return 0;
}

template <typename T, int kForm>
static int launch_quant(const QuantParams& p, int sms, cudaStream_t stream) {
  if (p.vecs <= 128) return launch_quant_sized<T, kForm, 128, 1>(p, sms, stream);
  if constexpr (kForm == kQuantPlain) {
    if (p.vecs <= 512) return launch_quant_sized<T, kForm, 128, 4>(p, sms, stream);
    if (p.vecs <= 1024) return launch_quant_sized<T, kForm, 256, 4>(p, sms, stream);
  } else {
    // 32-bit values: 2 pieces a thread (8192 x 8192 with a residual 77 us, 4 pieces 84; 4099 x 4096 19.5, 4 pieces 21.3)
    if (p.vecs <= 256) return launch_quant_sized<T, kForm, 256, 1>(p, sms, stream);
    if (kForm == kQuantNorm && p.vecs <= 512) return launch_quant_sized<T, kForm, 128, 4>(p, sms, stream);  // 4099 x 4096 10.2, 2 pieces 12.0
    if (p.vecs <= 512) return launch_quant_sized<T, kForm, 256, 2>(p, sms, stream);
    if (p.vecs <= 1024) return launch_quant_sized<T, kForm, 512, 2>(p, sms, stream);
  }
  if (p.vecs <= 2048) return launch_quant_sized<T, kForm, 512, 4>(p, sms, stream);
  return launch_quant_sized<T, kForm, 1024, 4>(p, sms, stream);
}

}  // namespace spd

using namespace spd;

extern "C" int spd_quant_int8(int8_t* q, float* scales, const void* x, void* residual, const void* weight, int64_t rows, int64_t dim,
                              int64_t x_stride, float eps, int silu_mul, int dtype, int sm_budget, spd_stream_t stream) {
  SPD_REQUIRE(rows >= 0 && rows <= 0x7fffffff && dim > 0, SPD_E_BADARG, "spd_quant_int8: bad sizes");
  SPD_REQUIRE(dim <= 32768, SPD_E_SHAPE, "spd_quant_int8: rows of at most 32768");
  SPD_REQUIRE(dim % 16 == 0 && x_stride % 8 == 0, SPD_E_ALIGN, "spd_quant_int8: dim must be a multiple of 16, x_stride of 8");
  SPD_REQUIRE(x_stride >= (silu_mul ? 2 * dim : dim), SPD_E_BADARG, "spd_quant_int8: x_stride too small");
  SPD_REQUIRE(!residual || weight, SPD_E_BADARG, "spd_quant_int8: a residual comes with a norm's weight");
  SPD_REQUIRE(!silu_mul || !weight, SPD_E_BADARG, "spd_quant_int8: a norm or SiLU * mul, not both");
  if (rows == 0) return 0;
  SPD_REQUIRE(q && scales && x, SPD_E_BADARG, "spd_quant_int8: null pointer");
  SPD_REQUIRE(aligned16(q) && aligned16(x) && aligned16(residual) && aligned16(weight), SPD_E_ALIGN,
              "spd_quant_int8: pointers must be 16-byte aligned");
  const QuantParams p{q, scales, x, residual, weight, rows, x_stride, static_cast<int>(dim / 8), eps};
  const int sms = sm_budget > 0 ? sm_budget : device_sm_count_cached();
  cudaStream_t st = as_stream(stream);
  SPD_DISPATCH_DTYPE(dtype, {
    if (silu_mul) return launch_quant<T, kQuantSilu>(p, sms, st);
    if (residual) return launch_quant<T, kQuantAddNorm>(p, sms, st);
    if (weight) return launch_quant<T, kQuantNorm>(p, sms, st);
    return launch_quant<T, kQuantPlain>(p, sms, st);
  });
}
