// mtr_lmhead_few.cu -- the 8-bit output projection of few rows (one token of one
// song, or of a few): the same logits to the bit as mtr_lmhead_i8.cu, in one
// launch and without tensor-core tiles, 120 of whose 128 rows would be empty.
//
// Every CTA quantises the rows into shared memory (each CTA reads them again:
// a few KB), then its warps take four vocabulary ids at a time: 16 bytes of each
// id's weights a lane, multiplied with every row's bytes by dp4a (exact int32 sums,
// as the tensor cores') and joined over the warp by one integer redux a sum.  The
// weights are read once: HBM bounds a large vocabulary, launch and two dependent
// trips to memory a small one.
#include "mtr_quant.cuh"

namespace mtr {
namespace i8 {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MOST_ROWS = 8;
// CTAs an SM, for whose registers four trips of a lane's loads are asked for at
// once (2 x 4096 -> 16384: 13.4 us; with 3 CTAs, 15.7; with two trips and 80
// registers, 18.9)
constexpr int CTAS = 2;
constexpr int HELD = 64 * 1024;  // bytes of int8 rows in shared memory at most

struct FewParams {
  const void* x;
  int64_t x_stride;
  const int8_t* weight;
  int64_t w_stride;
  const float* col_scale;
  void* out;
  int64_t out_stride;
  int32_t x_dtype, out_dtype;
  int32_t rows, d, wide;  // wide: d in whole 16 bytes
  int32_t vocab;
  int32_t vec;            // rows of x allow 16-byte loads
};

template <int R, typename T>
__device__ __forceinline__ float hold_rows(const FewParams& p, int8_t* held, float* tops) {
  constexpr int per = THREADS / R;
  const int sub = threadIdx.x / per, tid = threadIdx.x % per;
  const bool live = sub < p.rows;
  const T* x = (const T*)p.x + (live ? sub : 0) * p.x_stride;
  int8_t* q = held + sub * p.wide;
  const int cols = live ? p.d : 0;
  for (int c = cols + tid; c < p.wide; c += per) q[c] = 0;
  return p.vec ? quantize_row<T, true, 4>(x, cols, per, sub, tid, tops, q, [] {})
               : quantize_row<T, false, 4>(x, cols, per, sub, tid, tops, q, [] {});
}

// R: rows, or the next power of two; VB: ids a warp takes at a time
template <int R, int VB>
__global__ void __launch_bounds__(THREADS, CTAS) few_rows_kernel(const FewParams p) {
  extern __shared__ __align__(16) int8_t held[];
  __shared__ float tops[WARPS], row_scale[R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_prior_grid();
  float scale;
  switch (p.x_dtype) {
    case MTR_DTYPE_F32: scale = hold_rows<R, float>(p, held, tops); break;
    case MTR_DTYPE_BF16: scale = hold_rows<R, __nv_bfloat16>(p, held, tops); break;
    default: scale = hold_rows<R, __half>(p, held, tops); break;
  }
  if (threadIdx.x % (THREADS / R) == 0) row_scale[threadIdx.x / (THREADS / R)] = scale;
  __syncthreads();

  const int V = p.vocab, full = p.d / 16, rest = p.d % 16;
  for (int64_t v0 = ((int64_t)blockIdx.x * WARPS + warp) * VB; v0 < V; v0 += (int64_t)gridDim.x * WARPS * VB) {
    const int8_t* w[VB];
#pragma unroll
    for (int k = 0; k < VB; ++k) w[k] = p.weight + min((int64_t)(V - 1), v0 + k) * p.w_stride;
    int acc[R][VB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < VB; ++k) acc[r][k] = 0;
    auto add = [&](const uint4 (&b)[VB], int i) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint4 h = *reinterpret_cast<const uint4*>(held + r * p.wide + i * 16);
#pragma unroll
        for (int k = 0; k < VB; ++k)
          acc[r][k] = __dp4a((int)b[k].w, (int)h.w,
                             __dp4a((int)b[k].z, (int)h.z, __dp4a((int)b[k].y, (int)h.y, __dp4a((int)b[k].x, (int)h.x, acc[r][k]))));
      }
    };
#pragma unroll 4
    for (int i = lane; i < full; i += 32) {
      uint4 b[VB];
#pragma unroll
      for (int k = 0; k < VB; ++k) b[k] = reinterpret_cast<const uint4*>(w[k])[i];
      add(b, i);
    }
    if (rest && lane == full % 32) {  // the last bytes of d; what lies behind them is not read
      uint4 b[VB];
#pragma unroll
      for (int k = 0; k < VB; ++k) {
        uint32_t word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (c < rest) word[c / 4] |= (uint32_t)(uint8_t)w[k][full * 16 + c] << (c % 4 * 8);
        b[k] = make_uint4(word[0], word[1], word[2], word[3]);
      }
      add(b, full);
    }
    __syncwarp();
    // lane r VB + k has the sum of row r and id k
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < VB; ++k) {
        const int sum = __reduce_add_sync(FULL, acc[r][k]);
        if (lane == r * VB + k) mine = sum;
      }
    const int r = lane / VB;
    const int64_t v = v0 + lane % VB;
    if (r < p.rows && v < V) {
      const float f = __fmul_rn(__fmul_rn(__int2float_rn(mine), row_scale[r]), p.col_scale[v]);
      const int64_t at = r * p.out_stride + v;
      switch (p.out_dtype) {
        case MTR_DTYPE_F32: ((float*)p.out)[at] = f; break;
        case MTR_DTYPE_BF16: ((__nv_bfloat16*)p.out)[at] = from_f<__nv_bfloat16>(f); break;
        default: ((__half*)p.out)[at] = from_f<__half>(f); break;
      }
    }
  }
}

template <int R, int VB>
cudaError_t launch_rows(const FewParams& p, cudaStream_t s) {
  auto kern = few_rows_kernel<R, VB>;
  const int dyn = R * p.wide;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() { attr_err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, HELD); });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  const int64_t all = (p.vocab + WARPS * VB - 1) / (WARPS * VB), room = (int64_t)CTAS * device_sms();
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(all < room ? all : room), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = (size_t)dyn;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = launch_attrs(attr, 1, true);
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int R>
cudaError_t launch_ids(const FewParams& p, cudaStream_t s) {
  // four ids share a row's bytes once every warp has some (2 x 768 -> 4096 4 / 1 id: 3.8 / 5.0 us, 2 x 100 -> 1000 2.7 / 2.2)
  return p.vocab >= 2 * WARPS * device_sms() ? launch_rows<R, 4>(p, s) : launch_rows<R, 1>(p, s);
}

}  // namespace

// Where this kernel is the faster one.  What it does for a (row, id) beside the
// products is dear when d is short (vocab R <= 128 d, or a small vocabulary), and
// from 4 rows on its products cost more than the weight's way from HBM (R^2 d
// vocab <= 2^30; R the rows, to a power of two).  us with weights that are not in
// L2, here / there (148 SMs): 2 x 768 -> 4096 3.8 / 6.4, 8 x 768 -> 4096 4.4 /
// 6.6, 8 x 2048 -> 8192 8.0 / 10.2, 2 x 4096 -> 16384 13.4 / 16.7, 2 x 1024 ->
// 65536 15.6 / 16.0, 1 x 4096 -> 131072 76.8 / 85.8; and beyond the bounds
// 2 x 300 -> 65536 17.2 / 11.7, 4 x 768 -> 32768 10.8 / 10.2, 8 x 2048 -> 16384
// 12.5 / 11.8, 8 x 4096 -> 16384 20.9 / 16.7.
bool few_rows(int64_t rows, int64_t d, int64_t vocab) {
  const int64_t r = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
  return rows <= MOST_ROWS && r * ((d + 15) / 16 * 16) <= HELD && (r * vocab <= 128 * d || r * vocab <= 1 << 15) &&
         (r <= 2 || r * r * d * vocab <= 1ll << 30);
}

cudaError_t launch_few(const MtrLmHeadI8Args& a, cudaStream_t s) {
  FewParams p;
  p.x = a.hidden;
  p.x_stride = a.hidden_row_stride;
  p.weight = a.weight;
  p.w_stride = a.weight_row_stride;
  p.col_scale = a.weight_scale;
  p.out = a.logits;
  p.out_stride = a.logits_row_stride;
  p.x_dtype = a.hidden_dtype;
  p.out_dtype = a.logits_dtype;
  p.rows = a.rows;
  p.d = a.d_model;
  p.wide = (a.d_model + 15) / 16 * 16;
  p.vocab = a.vocab;
  const int es = a.hidden_dtype == MTR_DTYPE_F32 ? 4 : 2;
  p.vec = (uintptr_t)a.hidden % 16 == 0 && a.hidden_row_stride * es % 16 == 0;
  if (a.rows <= 1) return launch_ids<1>(p, s);
  if (a.rows <= 2) return launch_ids<2>(p, s);
  return a.rows <= 4 ? launch_ids<4>(p, s) : launch_ids<8>(p, s);
}

}  // namespace i8
}  // namespace mtr
