// mtr_lmhead_i8.cu -- the decoder's output projection in 8-bit integers on the
// sm_100a tensor cores, feeding the fused sampler.
//
// Rows of the hidden states and of the weight are held as int8 with one fp32
// scale each: scale = max|x| RN(1/127), q = round(x / scale), so
//   logits[r, v] = (sum_k q_h[r, k] q_w[v, k]) scale_h[r] scale_w[v].
// The sum is exact: |sum| <= 127 * 128 * d < 2^31 for d <= 131072, and
// tcgen05.mma kind::i8 accumulates in int32 tensor memory.  Rounding happens
// three times, each to fp32 or wider than the result: float(sum) (24 of at most
// 31 bits), the product with scale_h and the one with scale_w; then once more
// to the logits' type.
#include "mtr_tc.cuh"

namespace mtr {
namespace i8 {

using namespace tc;

constexpr int BM = 128;
constexpr int BN = 128;
constexpr int BK = 128;  // int8 elements of one 128-byte swizzled row
constexpr int UK = 32;   // K of one tcgen05.mma kind::i8
constexpr int STAGES = 4;
constexpr uint32_t A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr uint32_t RING_BYTES = STAGES * STAGE_BYTES + 1024;  // + alignment slack
constexpr int QUANT_THREADS = 256;

struct QuantParams {
  const void* x;
  int64_t x_stride;
  int32_t cols;
  int8_t* q;
  int64_t q_stride;
  float* scale;
};

struct ProjParams {
  const float* row_scale;
  const float* col_scale;
  void* out;
  int64_t out_stride;
  int32_t rows;
  int32_t vocab;
  int32_t kblocks;
  uint32_t* err;
};

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

// max that gives NaN when an operand is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// One CTA per row: the largest magnitude, then the quotients.
template <typename T>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_kernel(const QuantParams p) {
  __shared__ float tops[QUANT_THREADS / 32];
  const int tid = threadIdx.x;
  wait_prior_grid();
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.x + row * p.x_stride;
  int8_t* q = p.q + row * p.q_stride;
  float top = 0.0f;
  for (int k = tid; k < p.cols; k += QUANT_THREADS) top = max_nan(top, fabsf(to_f(x[k])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(FULL, top, o));
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
  top = tops[0];
  for (int w = 1; w < QUANT_THREADS / 32; ++w) top = max_nan(top, tops[w]);
  const bool finite = top < pos_inf();
  const float s = finite ? __fmul_rn(top, 1.0f / 127.0f) : __int_as_float(0x7fc00000);
  if (tid == 0) p.scale[row] = s;
  for (int k = tid; k < p.cols; k += QUANT_THREADS)
    q[k] = s > 0.0f ? (int8_t)__float2int_rn(__fdiv_rn(to_f(x[k]), s)) : (int8_t)0;
}

__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}

// Instruction descriptor of kind::i8: int32 accumulator (bits 4-5 = 2), signed A
// and B (bits 7-9, 10-12 = 1), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// One CTA per 128 x 128 tile of logits: one thread loads (TMA, 4-stage ring), one
// issues the products, then all four warps scale and store the accumulator.
template <typename Tout>
__global__ void __launch_bounds__(128, 1)
    lmhead_i8_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                     const ProjParams p) {
  extern __shared__ uint8_t dsm_raw[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t abort_flag;
  __shared__ float col_scale[BN];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * BN, m0 = blockIdx.y * BM;
  const uint32_t raw = smem_u32(dsm_raw);
  uint8_t* ring = dsm_raw + (((raw + 1023u) & ~1023u) - raw);
  auto a_tile = [&](int s) { return ring + (size_t)s * STAGE_BYTES; };
  auto b_tile = [&](int s) { return ring + (size_t)s * STAGE_BYTES + A_BYTES; };

  const int KB = p.kblocks;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"((uint32_t)BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  wait_prior_grid();
  if (n0 + (int)threadIdx.x < p.vocab) col_scale[threadIdx.x] = p.col_scale[n0 + threadIdx.x];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int kb = 0; kb < KB; ++kb) {
      const int s = kb % STAGES;
      if (kb >= STAGES && !mbar_wait(&empty[s], ((kb / STAGES) & 1) ^ 1, WAIT_NS)) {
        abort_flag = 1u;
        if (p.err) atomicOr(p.err, 1u);
        break;
      }
      if (abort_flag) break;
      mbar_expect_tx(&full[s], STAGE_BYTES);
      tma_load_2d(a_tile(s), &map_h, kb * BK, m0, &full[s]);
      tma_load_2d(b_tile(s), &map_w, kb * BK, n0, &full[s]);
      issued = kb + 1;
    }
    // copies still in flight land before the CTA may leave (bounded)
    for (int kb = (issued > STAGES ? issued - STAGES : 0); kb < issued; ++kb)
      mbar_wait(&full[kb % STAGES], (kb / STAGES) & 1, abort_flag ? WAIT_NS : 0ull);
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_i8(BM, BN);
    for (int kb = 0; kb < KB; ++kb) {
      const int s = kb % STAGES;
      if (!mbar_wait(&full[s], (kb / STAGES) & 1, WAIT_NS) || abort_flag) {
        abort_flag = 1u;
        if (p.err) atomicOr(p.err, 2u);
        break;
      }
      tc_fence_after();
      const uint32_t a0 = smem_u32(a_tile(s)), b0 = smem_u32(b_tile(s));
#pragma unroll
      for (int k = 0; k < BK / UK; ++k)
        mma_i8(tmem, sw128_desc(a0 + k * UK), sw128_desc(b0 + k * UK), idesc, (kb | k) != 0 ? 1u : 0u);
      tc_commit(&empty[s]);
    }
    tc_commit(&done);
  }
  __syncwarp();

  bool waited = true;
  if (lane == 0) waited = mbar_wait(&done, 0, WAIT_NS);
  waited = __shfl_sync(FULL, waited, 0) != 0;
  tc_fence_after();
  const bool go = __all_sync(FULL, waited && !abort_flag);
  if (!waited && lane == 0 && p.err) atomicOr(p.err, 4u);
  if (go) {
    const int row = m0 + warp * 32 + lane;
    const float rs = row < p.rows ? p.row_scale[row] : 0.0f;
    Tout* dst = (Tout*)p.out + (int64_t)row * p.out_stride + n0;
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
      uint32_t v[32];
      tmem_ld32(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c, v);
      tmem_wait_ld();
      if (row < p.rows) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (n0 + c + j < p.vocab)
            dst[c + j] = from_f<Tout>(__fmul_rn(__fmul_rn(__int2float_rn((int)v[j]), rs), col_scale[c + j]));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)BN) : "memory");
  }
}

// ---------------------------------------------------------------- host side
// 2-D byte tensor map over a row-major [rows, cols] matrix, box of BK columns x
// box_rows rows, 128-byte swizzle, 0 outside the matrix.
static bool make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t row_stride, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row_stride};
  const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static cudaLaunchConfig_t config(dim3 grid, int threads, size_t dyn, cudaStream_t s, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = dyn;
  cfg.stream = s;
  cfg.numAttrs = launch_attrs(attr, 1, true);
  cfg.attrs = attr;
  return cfg;
}

static cudaError_t launch_quantize(const void* x, int64_t x_stride, int dtype, int rows, int cols, int8_t* q,
                                   int64_t q_stride, float* scale, cudaStream_t s) {
  const QuantParams p{x, x_stride, cols, q, q_stride, scale};
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(dim3((unsigned)rows, 1, 1), QUANT_THREADS, 0, s, attr);
  switch (dtype) {
    case MTR_DTYPE_F32: return cudaLaunchKernelEx(&cfg, quantize_kernel<float>, p);
    case MTR_DTYPE_BF16: return cudaLaunchKernelEx(&cfg, quantize_kernel<__nv_bfloat16>, p);
    default: return cudaLaunchKernelEx(&cfg, quantize_kernel<__half>, p);
  }
}

template <typename Tout>
static cudaError_t launch_proj(const MtrLmHeadI8Args& a, const int8_t* q, int64_t q_stride, const float* row_scale,
                               cudaStream_t s) {
  CUtensorMap mh, mw;
  if (!make_map(&mh, q, a.rows, a.d_model, q_stride, BM) ||
      !make_map(&mw, a.weight, a.vocab, a.d_model, a.weight_row_stride, BN))
    return cudaErrorInvalidValue;
  auto kern = lmhead_i8_kernel<Tout>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() {
    attr_err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RING_BYTES);
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  const ProjParams p{row_scale, a.weight_scale, a.logits, a.logits_row_stride, a.rows, a.vocab, (a.d_model + BK - 1) / BK, a.error_word};
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      config(dim3((unsigned)((a.vocab + BN - 1) / BN), (unsigned)((a.rows + BM - 1) / BM), 1), 128, RING_BYTES, s, attr);
  return cudaLaunchKernelEx(&cfg, kern, mh, mw, p);
}

static int esize(int32_t dtype) { return dtype == MTR_DTYPE_F32 ? 4 : 2; }
static bool dtype_ok(int32_t dtype) { return dtype >= MTR_DTYPE_F32 && dtype <= MTR_DTYPE_F16; }
static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// bytes [p, p + n) and [q, q + m) share one
static bool overlap(const void* p, int64_t n, const void* q, int64_t m) {
  return (uintptr_t)p < (uintptr_t)q + (uintptr_t)m && (uintptr_t)q < (uintptr_t)p + (uintptr_t)n;
}
static int64_t span(int64_t rows, int64_t stride, int64_t cols, int64_t es) { return ((rows - 1) * stride + cols) * es; }

}  // namespace i8
}  // namespace mtr

// ---------------------------------------------------------------- C ABI
using namespace mtr::i8;

int mtr_quantize_rows_validate(const MtrQuantizeArgs* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrQuantizeArgs)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->cols < 1) return MTR_ERR_BAD_SHAPE;
  if (!dtype_ok(a->x_dtype)) return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  if (!a->x || !a->q || !a->scale) return MTR_ERR_NULL_ARG;
  if (a->x_row_stride < a->cols || a->q_row_stride < a->cols) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->x % esize(a->x_dtype) || (uintptr_t)a->scale % 4) return MTR_ERR_ALIGNMENT;
  const int64_t xs = span(a->rows, a->x_row_stride, a->cols, esize(a->x_dtype)), qs = span(a->rows, a->q_row_stride, a->cols, 1);
  if (overlap(a->x, xs, a->q, qs) || overlap(a->x, xs, a->scale, 4ll * a->rows) || overlap(a->q, qs, a->scale, 4ll * a->rows))
    return MTR_ERR_BAD_PARAM;
  return MTR_OK;
}

int mtr_quantize_rows_launch(const MtrQuantizeArgs* a, void* stream) {
  const int v = mtr_quantize_rows_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  const cudaError_t e = launch_quantize(a->x, a->x_row_stride, a->x_dtype, a->rows, a->cols, a->q, a->q_row_stride, a->scale,
                                        (cudaStream_t)stream);
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}

int64_t mtr_lmhead_i8_workspace(int32_t rows, int32_t d_model) {
  if (rows <= 0 || d_model <= 0) return 0;
  return up((int64_t)rows * up(d_model, 16), 256) + 4ll * rows;
}

int mtr_lmhead_i8_validate(const MtrLmHeadI8Args* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrLmHeadI8Args)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->rows > MTR_MAX_I8_ROWS) return MTR_ERR_BAD_SHAPE;
  if (a->d_model < 1 || a->d_model > MTR_MAX_I8_D_MODEL) return MTR_ERR_BAD_SHAPE;
  if (a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
  if (!dtype_ok(a->hidden_dtype) || !dtype_ok(a->logits_dtype)) return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  if (!a->hidden || !a->weight || !a->weight_scale || !a->logits || !a->workspace) return MTR_ERR_NULL_ARG;
  if (a->hidden_row_stride < a->d_model || a->weight_row_stride < a->d_model || a->logits_row_stride < a->vocab)
    return MTR_ERR_BAD_SHAPE;
  const int64_t need = mtr_lmhead_i8_workspace(a->rows, a->d_model);
  if (a->workspace_bytes < need) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->hidden % esize(a->hidden_dtype) || (uintptr_t)a->weight % 16 || a->weight_row_stride % 16 ||
      (uintptr_t)a->weight_scale % 4 || (uintptr_t)a->logits % esize(a->logits_dtype) || (uintptr_t)a->workspace % 256 ||
      (uintptr_t)a->error_word % 4)
    return MTR_ERR_ALIGNMENT;
  const int64_t ls = span(a->rows, a->logits_row_stride, a->vocab, esize(a->logits_dtype));
  const int64_t hs = span(a->rows, a->hidden_row_stride, a->d_model, esize(a->hidden_dtype));
  const int64_t ws = span(a->vocab, a->weight_row_stride, a->d_model, 1);
  if (overlap(a->logits, ls, a->hidden, hs) || overlap(a->logits, ls, a->weight, ws) ||
      overlap(a->logits, ls, a->weight_scale, 4ll * a->vocab) || overlap(a->logits, ls, a->workspace, need) ||
      overlap(a->workspace, need, a->hidden, hs) || overlap(a->workspace, need, a->weight, ws) ||
      overlap(a->workspace, need, a->weight_scale, 4ll * a->vocab))
    return MTR_ERR_BAD_PARAM;
  return MTR_OK;
}

static int lmhead_i8_launch_impl(const MtrLmHeadI8Args* a, cudaStream_t s) {
  int8_t* q = (int8_t*)a->workspace;
  const int64_t q_stride = up(a->d_model, 16);
  float* scale = (float*)(q + up(a->rows * q_stride, 256));
  cudaError_t e = launch_quantize(a->hidden, a->hidden_row_stride, a->hidden_dtype, a->rows, a->d_model, q, q_stride, scale, s);
  if (e == cudaSuccess) {
    switch (a->logits_dtype) {
      case MTR_DTYPE_F32: e = launch_proj<float>(*a, q, q_stride, scale, s); break;
      case MTR_DTYPE_BF16: e = launch_proj<__nv_bfloat16>(*a, q, q_stride, scale, s); break;
      default: e = launch_proj<__half>(*a, q, q_stride, scale, s); break;
    }
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}

int mtr_lmhead_i8_launch(const MtrLmHeadI8Args* a, void* stream) {
  const int v = mtr_lmhead_i8_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  return lmhead_i8_launch_impl(a, (cudaStream_t)stream);
}

int mtr_lmhead_i8_sample_launch(const MtrLmHeadI8Args* lm, const MtrSamplerArgs* sa, void* stream) {
  int v = mtr_lmhead_i8_validate(lm);
  if (v != MTR_OK) return v;
  v = mtr_sampler_validate(sa);
  if (v != MTR_OK) return v;
  // the sampler reads exactly the logits the projection writes
  if (sa->logits != lm->logits || sa->logits_dtype != lm->logits_dtype || sa->logits_row_stride != lm->logits_row_stride ||
      sa->vocab != lm->vocab)
    return MTR_ERR_BAD_PARAM;
  const int64_t second = sa->cfg_second_offset > 0 ? sa->cfg_second_offset : sa->num_rows;
  const int64_t need = sa->cfg_enabled ? second + sa->num_rows : sa->num_rows;
  if (need > lm->rows) return MTR_ERR_BAD_SHAPE;
  if (lm->rows == 0 || sa->num_rows == 0) return MTR_OK;
  v = lmhead_i8_launch_impl(lm, (cudaStream_t)stream);
  if (v != MTR_OK) return v;
  return mtr::sampler_launch(sa, (cudaStream_t)stream, true);
}
