// mtr_f8.cuh -- blocks of 128 values to 8-bit floats (e4m3) with one scale each, for
// the kernels of the projection in 8-bit floating point (mtr_lmhead_f8.cu: rows and
// weights into buffers; mtr_lmhead_f8_few.cu: rows into shared memory), and the
// launch of the projection of few rows.
#pragma once

#include "mtr_quant.cuh"

namespace mtr {
namespace f8 {

constexpr int BLOCK = 128;
constexpr float RECIPROCAL = 1.0f / 448.0f;  // of e4m3's largest value

// The projection of few rows: whether it takes them, and its launch.
bool few_rows(int64_t rows, int64_t d, int64_t vocab);
cudaError_t launch_few(const MtrLmHeadF8Args& a, cudaStream_t s);

__device__ __forceinline__ float largest(float v) {
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(v) : "f"(v));
  return v;
}
__device__ __forceinline__ float magnitude(const float (&v)[4]) {
  return max_nan(max_nan(fabsf(v[0]), fabsf(v[1])), max_nan(fabsf(v[2]), fabsf(v[3])));
}
// RNE to e4m3 of the fp32 quotients x / s, held to -448 .. 448 (only blocks below
// 448 2^-140 or so, whose scales keep a few bits, pass that)
__device__ __forceinline__ uint32_t quotients(const float (&x)[4], const i8::Divisor& d) {
  float q[4];
  if (d.divide) {
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __fdiv_rn(x[e], d.s);
  } else {
    const u64 y2 = pk2(d.inv, d.inv), ns2 = pk2(-d.s, -d.s);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const u64 x2 = pk2(x[e], x[e + 1]), q0 = mul2(x2, y2);
      up2(fma2(fma2(q0, ns2, x2), y2, q0), q[e], q[e + 1]);
    }
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(q[1]), "f"(q[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(q[3]), "f"(q[2]));
  return d.zero ? 0u : (uint32_t)lo | (uint32_t)hi << 16;
}
// Values c .. c + 3 of a row of `cols` (0 behind it); VEC: in one load.
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* x, int c, int cols, float (&v)[4]) {
  if (VEC && c + 4 <= cols) {
    if constexpr (sizeof(T) == 4) {
      const float4 w = *reinterpret_cast<const float4*>(x + c);
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(x + c);
      const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to_f(t[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? to_f(x[c + e]) : 0.0f;
  }
}

}  // namespace f8
}  // namespace mtr
