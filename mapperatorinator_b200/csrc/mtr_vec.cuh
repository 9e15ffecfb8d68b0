// mtr_vec.cuh -- rows of fp32, bf16 or fp16 values in 16-byte vectors: what the
// kernels that stream such rows share (mtr_logprob.cu, mtr_lmhead_i8.cu).
#pragma once

#include "mtr_common.cuh"

namespace mtr {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// ---------------------------------------------------------------- host side
// A row-strided matrix as bytes: `rows` rows of `width`, `stride` apart.
struct Bytes {
  const void* at;
  int64_t rows, stride, width;
};
inline Bytes bytes_of(const void* at, int64_t rows, int64_t stride, int64_t cols, int64_t es) { return {at, rows, stride * es, cols * es}; }
// Whether two share a byte: their spans overlap, and they do not lie side by side in rows of one width.
inline bool overlap(const Bytes& a, const Bytes& b) {
  const uintptr_t a0 = (uintptr_t)a.at, b0 = (uintptr_t)b.at;
  if (a0 >= b0 + (uintptr_t)((b.rows - 1) * b.stride + b.width) || b0 >= a0 + (uintptr_t)((a.rows - 1) * a.stride + a.width)) return false;
  if (a.stride != b.stride) return true;
  const int64_t off = (int64_t)(b0 - a0) % a.stride, behind = off < 0 ? off + a.stride : off;  // from a row of a to the next of b
  return behind < a.width || behind + b.width > a.stride;
}

// max that gives NaN when an operand is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 16 bytes of a row: E values, their packed maximum, their fp32 values; reach:
// which of them are at least `cut`, value 2 k + h in bit k + 16 h (fp32: value k in
// bit k); count of a sum of `equal`s: how many values equal m.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static constexpr uint32_t FILL = 0xff800000u;  // -inf
  static constexpr float LOWEST = -0x1.fffffep127f;
  typedef float Top;                             // the largest of a vector; NaN when one is
  static __device__ __forceinline__ Top top(const uint4& w) {
    return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ Top larger(Top a, Top b) { return max_nan(a, b); }
  static __device__ __forceinline__ float value(Top t) { return t; }
  static __device__ __forceinline__ Top pattern(float m) { return m; }
  static __device__ __forceinline__ uint32_t equal(const uint4& w, Top m) {
    return (__uint_as_float(w.x) == m) + (__uint_as_float(w.y) == m) + (__uint_as_float(w.z) == m) + (__uint_as_float(w.w) == m);
  }
  static __device__ __forceinline__ uint32_t count(uint32_t equal) { return equal; }
  static __device__ __forceinline__ uint32_t reach(const uint4& w, Top cut) {
    return (__uint_as_float(w.x) >= cut ? 1u : 0u) | (__uint_as_float(w.y) >= cut ? 2u : 0u) |
           (__uint_as_float(w.z) >= cut ? 4u : 0u) | (__uint_as_float(w.w) >= cut ? 8u : 0u);
  }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[E]) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  static constexpr uint32_t FILL = 0xff80ff80u;
  static constexpr float LOWEST = -0x1.fep127f;
  typedef __nv_bfloat162 Top;
  static __device__ __forceinline__ Top pair(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
  static __device__ __forceinline__ Top top(const uint4& w) {
    return __hmax2_nan(__hmax2_nan(pair(w.x), pair(w.y)), __hmax2_nan(pair(w.z), pair(w.w)));
  }
  static __device__ __forceinline__ Top larger(Top a, Top b) { return __hmax2_nan(a, b); }
  static __device__ __forceinline__ float value(Top t) { return max_nan(__low2float(t), __high2float(t)); }
  static __device__ __forceinline__ Top pattern(float m) { return __float2bfloat162_rn(m); }
  static __device__ __forceinline__ uint32_t equal(const uint4& w, Top m) {
    return (__heq2_mask(pair(w.x), m) & 0x10001u) + (__heq2_mask(pair(w.y), m) & 0x10001u) +
           (__heq2_mask(pair(w.z), m) & 0x10001u) + (__heq2_mask(pair(w.w), m) & 0x10001u);
  }
  static __device__ __forceinline__ uint32_t count(uint32_t equal) { return (equal & 0xffffu) + (equal >> 16); }
  static __device__ __forceinline__ uint32_t reach(const uint4& w, Top cut) {
    return (__hge2_mask(pair(w.x), cut) & 0x10001u) | (__hge2_mask(pair(w.y), cut) & 0x20002u) |
           (__hge2_mask(pair(w.z), cut) & 0x40004u) | (__hge2_mask(pair(w.w), cut) & 0x80008u);
  }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[E]) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
};
template <>
struct Vec<__half> {
  static constexpr int E = 8;
  static constexpr uint32_t FILL = 0xfc00fc00u;
  static constexpr float LOWEST = -65504.0f;
  typedef __half2 Top;
  static __device__ __forceinline__ Top pair(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
  static __device__ __forceinline__ Top top(const uint4& w) {
    return __hmax2_nan(__hmax2_nan(pair(w.x), pair(w.y)), __hmax2_nan(pair(w.z), pair(w.w)));
  }
  static __device__ __forceinline__ Top larger(Top a, Top b) { return __hmax2_nan(a, b); }
  static __device__ __forceinline__ float value(Top t) { return max_nan(__low2float(t), __high2float(t)); }
  static __device__ __forceinline__ Top pattern(float m) { return __float2half2_rn(m); }
  static __device__ __forceinline__ uint32_t equal(const uint4& w, Top m) {
    return (__heq2_mask(pair(w.x), m) & 0x10001u) + (__heq2_mask(pair(w.y), m) & 0x10001u) +
           (__heq2_mask(pair(w.z), m) & 0x10001u) + (__heq2_mask(pair(w.w), m) & 0x10001u);
  }
  static __device__ __forceinline__ uint32_t count(uint32_t equal) { return (equal & 0xffffu) + (equal >> 16); }
  static __device__ __forceinline__ uint32_t reach(const uint4& w, Top cut) {
    return (__hge2_mask(pair(w.x), cut) & 0x10001u) | (__hge2_mask(pair(w.y), cut) & 0x20002u) |
           (__hge2_mask(pair(w.z), cut) & 0x40004u) | (__hge2_mask(pair(w.w), cut) & 0x80008u);
  }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[E]) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 g = __half22float2(pair(v[i]));
      f[2 * i] = g.x;
      f[2 * i + 1] = g.y;
    }
  }
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

}  // namespace mtr
