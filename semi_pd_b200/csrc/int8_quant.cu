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
// distance, so it moves halves up and nothing else over a border.
//
// A NaN or an infinity in a row makes its scale NaN or infinite, and with it everything that the row is multiplied into: the
// maximum is taken over the bits of |y|, which order NaN above infinity above numbers.
//
// What bounds it: memory.
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
  int64_t x_stride;
  int vecs;        // pieces of 8 in a row
  float eps;
};

__device__ __forceinline__ uint32_t pack_s8(float a, float b, float c, float d) {
  uint32_t hi, lo;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(lo) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(hi));
  return lo;
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

template <typename T, int kForm, int kThreads, int kVecs>
__global__ void __launch_bounds__(kThreads) quant_int8_kernel(const QuantParams p) {
  constexpr bool kHasNorm = kForm == kQuantNorm || kForm == kQuantAddNorm;
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  griddep_launch_dependents();
  griddep_wait();
  const int64_t row = blockIdx.x;
  const uint4* x = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.x) + row * p.x_stride);
  float y[kVecs][8];
  float ss = 0.f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = threadIdx.x + i * kThreads;
    if (v < p.vecs) {
      unpack8<T>(x[v], y[i]);
      if constexpr (kForm == kQuantAddNorm) {
        uint4* r = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.residual) + row * p.x_stride) + v;
        float f[8];
        unpack8<T>(*r, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[i][j] += f[j];
        *r = make_uint4(pack2<T>(y[i][0], y[i][1]), pack2<T>(y[i][2], y[i][3]), pack2<T>(y[i][4], y[i][5]),
                        pack2<T>(y[i][6], y[i][7]));  // the new residual is rounded, what the norm sees is not
      }
      if constexpr (kHasNorm) {
        float f[8];
        unpack8<T>(reinterpret_cast<const uint4*>(p.w)[v], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ss = fmaf(y[i][j], y[i][j], ss);
          y[i][j] *= f[j];
        }
      }
      if constexpr (kForm == kQuantSilu) {
        float f[8];
        unpack8<T>(x[p.vecs + v], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[i][j] = silu_f32(y[i][j]) * f[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(y[i][j]) & 0x7fffffffu);
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kThreads / 32;
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (kHasNorm) ss = warp_sum(ss);
  if (lane == 0) {
    tops[warp] = top;
    if constexpr (kHasNorm) sums[warp] = ss;
  }
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < kWarps ? tops[lane] : 0u);
  float c = 1.f;
  if constexpr (kHasNorm)
    c = rsqrtf(warp_sum(lane < kWarps ? sums[lane] : 0.f) / static_cast<float>(p.vecs * 8) + p.eps);
  float most = __uint_as_float(top) * c;
  most = most < 1e-10f ? 1e-10f : most;  // (NaN stays)
  if (threadIdx.x == 0) p.scales[row] = __fdiv_rn(most, 127.f);
  const float k = __fdiv_rn(127.f, most) * (kHasNorm ? c : 1.f + 0x1p-20f);
  uint2* q = reinterpret_cast<uint2*>(p.q) + row * p.vecs;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = threadIdx.x + i * kThreads;
    if (v < p.vecs)
      q[v] = make_uint2(pack_s8(y[i][0] * k, y[i][1] * k, y[i][2] * k, y[i][3] * k),
                        pack_s8(y[i][4] * k, y[i][5] * k, y[i][6] * k, y[i][7] * k));
  }
}

template <typename T, int kForm>
static int launch_quant(const QuantParams& p, int64_t rows, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(rows));
#define SPD_QUANT(THREADS, VECS)                  \
  if (p.vecs <= THREADS * VECS) {                 \
    SPD_CUDA(launch(quant_int8_kernel<T, kForm, THREADS, VECS>, grid, dim3(THREADS), 0, stream, pdl_enabled(), p)); \
    return 0;                                     \
  }
  SPD_QUANT(128, 1)
  SPD_QUANT(256, 1)
  SPD_QUANT(256, 2)
  SPD_QUANT(256, 4)
  SPD_QUANT(512, 4)
  SPD_QUANT(1024, 4)
#undef SPD_QUANT
  return set_error(SPD_E_SHAPE, "spd_quant_int8: rows of at most 32768");
}

}  // namespace spd

using namespace spd;

extern "C" int spd_quant_int8(int8_t* q, float* scales, const void* x, void* residual, const void* weight, int64_t rows, int64_t dim,
                              int64_t x_stride, float eps, int silu_mul, int dtype, spd_stream_t stream) {
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
  const QuantParams p{q, scales, x, residual, weight, x_stride, static_cast<int>(dim / 8), eps};
  cudaStream_t st = as_stream(stream);
  SPD_DISPATCH_DTYPE(dtype, {
    if (silu_mul) return launch_quant<T, kQuantSilu>(p, rows, st);
    if (residual) return launch_quant<T, kQuantAddNorm>(p, rows, st);
    if (weight) return launch_quant<T, kQuantNorm>(p, rows, st);
    return launch_quant<T, kQuantPlain>(p, rows, st);
  });
}
