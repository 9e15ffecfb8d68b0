// mtr_quant.cuh -- rows to int8 with one scale each, for the kernels that quantise
// (mtr_lmhead_i8.cu: rows into a buffer; mtr_lmhead_few.cu: rows into shared
// memory), and the launch of the projection of few rows.
#pragma once

#include "mtr_vec.cuh"

namespace mtr {
namespace i8 {

// The projection of few rows (mtr_lmhead_few.cu): whether it takes them, and its launch.
bool few_rows(int64_t rows, int64_t d, int64_t vocab);
cudaError_t launch_few(const MtrLmHeadI8Args& a, cudaStream_t s);

__device__ __forceinline__ float magnitude(const uint4& w, float) {
  return max_nan(max_nan(fabsf(__uint_as_float(w.x)), fabsf(__uint_as_float(w.y))),
                 max_nan(fabsf(__uint_as_float(w.z)), fabsf(__uint_as_float(w.w))));
}
template <typename T>
__device__ __forceinline__ float magnitude(uint4 w, T) {
  w.x &= 0x7fff7fffu;
  w.y &= 0x7fff7fffu;
  w.z &= 0x7fff7fffu;
  w.w &= 0x7fff7fffu;
  return Vec<T>::value(Vec<T>::top(w));
}

// The divisor of a row: q(x) = RNE(RN(x / s)), held to -127 .. 127.  With y =
// RN(1 / s), q0 = RN(x y), r = RN(x - q0 s) (exact) and q1 = RN(q0 + r y), q1 is
// the correctly rounded quotient (Markstein) unless s has an all-ones significand;
// three steps, packed two values at a time.  Those scales, and the ones so
// small that 1 / s or r could leave the normal range, divide instead.  Only
// those can pass 127: a scale of one step of 2^-149 may be rounded down by a
// third, and the row's largest quotient is then 190.
struct Divisor {
  float s, inv;
  bool zero, divide;
};
__device__ __forceinline__ Divisor divisor_of(float top, float reciprocal = 1.0f / 127.0f) {
  Divisor d;
  d.s = top < pos_inf() ? __fmul_rn(top, reciprocal) : __int_as_float(0x7fc00000);
  d.zero = !(d.s > 0.0f);
  d.divide = d.s < 0x1p-90f || (__float_as_uint(d.s) & 0x7fffffu) == 0x7fffffu;
  d.inv = d.zero || d.divide ? 0.0f : __fdiv_rn(1.0f, d.s);
  return d;
}
constexpr float WHOLE = 12582912.0f;  // 1.5 2^23: y + WHOLE holds RNE(y) in its low bits, |y| < 2^22
__device__ __forceinline__ uint32_t quotient(float x, const Divisor& d) {
  return __float_as_uint(__fadd_rn(fminf(fmaxf(__fdiv_rn(x, d.s), -127.0f), 127.0f), WHOLE));
}
template <int N>
__device__ __forceinline__ void quotients(const float (&x)[N], const Divisor& d, uint32_t (&w)[N / 4]) {
  uint32_t b[N];
  if (d.divide) {
#pragma unroll
    for (int e = 0; e < N; ++e) b[e] = quotient(x[e], d);
  } else {
    const u64 y2 = pk2(d.inv, d.inv), ns2 = pk2(-d.s, -d.s), whole2 = pk2(WHOLE, WHOLE);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const u64 x2 = pk2(x[e], x[e + 1]), q0 = mul2(x2, y2), q1 = fma2(fma2(q0, ns2, x2), y2, q0);
      float lo, hi;
      up2(add2(q1, whole2), lo, hi);
      b[e] = __float_as_uint(lo);
      b[e + 1] = __float_as_uint(hi);
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint32_t lo = __byte_perm(b[4 * i], b[4 * i + 1], 0x0040), hi = __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040);
    w[i] = d.zero ? 0u : __byte_perm(lo, hi, 0x5410);
  }
}

// Quantises one row of `cols` values with `per` threads (tid of them, the sub-th
// group of the CTA; a power of two from 32, all of the CTA's warps in step when it
// is more) into q, and returns its scale.  The threads hold the row's first HOLD
// vectors each between the two passes over it (the largest magnitude, the
// quotients); longer rows are read again from L2.  VEC: x allows 16-byte loads
// and q stores of as many quotients; else every value is its own access.
// `between` runs between the passes.
template <typename T, bool VEC, int HOLD, typename F>
__device__ __forceinline__ float quantize_row(const T* x, int cols, int per, int sub, int tid, float* tops, int8_t* q, F between) {
  constexpr int E = VEC ? Vec<T>::E : 1;
  const int vecs = cols / E, behind = vecs * E, rest = cols - behind;
  float top = 0.0f;
  uint4 w[HOLD];
  T one[HOLD];
  if (VEC) {
#pragma unroll
    for (int j = 0; j < HOLD; ++j) {
      w[j] = make_uint4(0u, 0u, 0u, 0u);
      const int i = tid + j * per;
      if (i < vecs) w[j] = reinterpret_cast<const uint4*>(x)[i];
    }
#pragma unroll
    for (int j = 0; j < HOLD; ++j) top = max_nan(top, magnitude(w[j], T()));
    for (int i = tid + HOLD * per; i < vecs; i += per) top = max_nan(top, magnitude(reinterpret_cast<const uint4*>(x)[i], T()));
    if (tid < rest) top = max_nan(top, fabsf(to_f(x[behind + tid])));
  } else {
#pragma unroll
    for (int j = 0; j < HOLD; ++j) {
      const int i = tid + j * per;
      one[j] = i < vecs ? x[i] : from_f<T>(0.0f);
    }
#pragma unroll
    for (int j = 0; j < HOLD; ++j) top = max_nan(top, fabsf(to_f(one[j])));
    for (int i = tid + HOLD * per; i < vecs; i += per) top = max_nan(top, fabsf(to_f(x[i])));
  }
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(top));
  if (per > 32) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int k = 0; k < per / 32; ++k) top = max_nan(top, tops[sub * (per / 32) + k]);
  }
  const Divisor d = divisor_of(top);
  between();
  if constexpr (VEC) {
    auto put = [&](int i, const uint4& v) {
      float f[E];
      uint32_t b[E / 4];
      Vec<T>::unpack(v, f);
      quotients(f, d, b);
      if constexpr (E == 8) reinterpret_cast<uint2*>(q)[i] = make_uint2(b[0], b[1]);
      else reinterpret_cast<uint32_t*>(q)[i] = b[0];
    };
#pragma unroll
    for (int j = 0; j < HOLD; ++j)
      if (tid + j * per < vecs) put(tid + j * per, w[j]);
    for (int i = tid + HOLD * per; i < vecs; i += per) put(i, reinterpret_cast<const uint4*>(x)[i]);
    if (tid < rest) q[behind + tid] = d.zero ? (int8_t)0 : (int8_t)quotient(to_f(x[behind + tid]), d);
  } else {
#pragma unroll
    for (int j = 0; j < HOLD; ++j)
      if (tid + j * per < vecs) q[tid + j * per] = d.zero ? (int8_t)0 : (int8_t)quotient(to_f(one[j]), d);
    for (int i = tid + HOLD * per; i < vecs; i += per) q[i] = d.zero ? (int8_t)0 : (int8_t)quotient(to_f(x[i]), d);
  }
  return d.s;
}

}  // namespace i8
}  // namespace mtr
