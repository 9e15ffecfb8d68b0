// mtr_logprob.cu -- log probabilities of given tokens, entropy, log-sum-exp and
// top alternatives of each row of logits, and the gradient of all of them.
//
// With x = logits / T, m the largest logit, d_v = (logit_v - m) / T and
// S = sum_v e^(d_v):
//   log p_v = d_v - log S        lse = m / T + log S
//   H       = log S - (sum_v e^(d_v) d_v) / S
// S is held as n + S': n counts the scores equal to the maximum (each adds
// exactly 1) and S' sums the others, so log S = log1p(S' + (n - 1)) keeps its
// relative precision when one score carries nearly all the mass (the log
// probability and the entropy are then the small numbers that matter).  All
// sums are fp32; d is formed as (logit - m) * (log2(e) / T), so that equal
// logits give 0 exactly.  A masked score (-inf) has e^d = 0, and d is clamped
// so that e^d d is 0 as well.
#include "mtr_common.cuh"

namespace mtr {
namespace lp {

constexpr float LN2 = 0x1.62e430p-1f;
constexpr float LOG2E_D = 0x1.715476p+0f;
constexpr int THREADS = 256;

struct FwdParams {
  const void* logits;
  int64_t stride;
  const void* tokens;
  int32_t ids32;
  int32_t rows;
  int32_t vocab;
  int32_t top_n;
  float scale;      // log2(e) / T
  float inv_t;      // 1 / T
  float* logprobs;
  float* entropy;
  float* lse;
  int64_t* top_ids;
  float* top_logprobs;
  float4* stats;
  uint32_t* status;
};

struct GradParams {
  const void* logits;
  int64_t stride;
  const void* tokens;
  int32_t ids32;
  int32_t rows;
  int32_t vocab;
  int32_t top_n;
  float scale;
  float inv_t;
  const float4* stats;
  const int64_t* top_ids;
  const float* g_logprobs;
  const float* g_entropy;
  const float* g_lse;
  const float* g_top;
  void* grad;
  int64_t grad_stride;
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that gives NaN when an operand is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float qnan() { return __int_as_float(0x7fc00000); }

// order of the alternatives: larger logit first, then the lower id; -0 and +0 are equal scores
__device__ __forceinline__ u64 order_key(float x, uint32_t id) {
  uint32_t b = __float_as_uint(x + 0.0f);  // -0 -> +0
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((u64)b << 32) | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(u64 k) {
  uint32_t b = (uint32_t)(k >> 32);
  b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
  return __uint_as_float(b);
}
__device__ __forceinline__ int32_t key_id(u64 k) { return (int32_t)~(uint32_t)k; }

__device__ __forceinline__ int64_t load_id(const void* ids, int32_t ids32, int64_t i) {
  return ids32 ? (int64_t)((const int32_t*)ids)[i] : ((const int64_t*)ids)[i];
}

// What one thread, warp or CTA holds of a row: the largest logit, how many
// logits equal it, and the sums over the others (d in units of log 2).
struct Part {
  float m;   // -inf: nothing but masked scores so far
  float n;   // logits equal to m (0 while m = -inf)
  float s;   // sum of 2^d over the others
  float u;   // sum of 2^d d
};

__device__ __forceinline__ Part empty_part() { return Part{neg_inf(), 0.0f, 0.0f, 0.0f}; }

// The sums of `a` and `b` about the larger maximum: moving a part from m to M
// scales its terms by 2^e, e = (m - M) scale, and adds e to each d.
__device__ __forceinline__ Part join(const Part& a, const Part& b, float scale) {
  const float M = fmaxf(a.m, b.m);
  if (!(M > neg_inf())) return Part{M, 0.0f, a.s + b.s, a.u + b.u};
  Part r{M, 0.0f, 0.0f, 0.0f};
  const Part* both[2] = {&a, &b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Part& p = *both[i];
    if (p.m == M) {
      r.n += p.n;
      r.s += p.s;
      r.u += p.u;
    } else {  // m = -inf: every sum is 0 (or NaN, which stays)
      const float e = fmaxf((p.m - M) * scale, -1000.0f);
      const float f = ex2(e), t = p.n + p.s;
      r.s += t * f;
      r.u += fmaf(t, e, p.u) * f;
    }
  }
  return r;
}

__device__ __forceinline__ Part warp_join(Part p, float scale) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Part q{__shfl_xor_sync(FULL, p.m, o), __shfl_xor_sync(FULL, p.n, o), __shfl_xor_sync(FULL, p.s, o),
                 __shfl_xor_sync(FULL, p.u, o)};
    p = join(p, q, scale);
  }
  return p;
}

// What the sums of a whole row say.  NaN and +inf logits make s NaN: NaN by
// itself, +inf by inf - inf.
struct Row {
  float m, log_s, entropy, lse;
  bool bad, none;
};
__device__ __forceinline__ Row row_of(const Part& p, float inv_t) {
  Row r;
  r.m = p.m;
  r.bad = !(p.s < pos_inf()) || !(p.m < pos_inf());
  r.none = !r.bad && !(p.m > neg_inf());
  if (r.bad) {
    r.log_s = r.entropy = r.lse = qnan();
  } else if (r.none) {
    r.log_s = 0.0f;
    r.entropy = 0.0f;
    r.lse = neg_inf();
  } else {
    const float rest = p.s + (p.n - 1.0f);
    r.log_s = log1pf(rest);
    r.entropy = fmaxf(r.log_s - LN2 * p.u / (1.0f + rest), 0.0f);
    r.lse = fmaf(p.m, inv_t, r.log_s);
  }
  return r;
}
__device__ __forceinline__ float log_prob(float x, const Row& r, float inv_t) {
  if (r.bad) return qnan();
  if (r.none || x == neg_inf()) return neg_inf();
  return (x - r.m) * inv_t - r.log_s;
}

// One CTA per row: the maximum, then the sums, then one argmax over the row
// for each alternative.
template <typename T>
__global__ void __launch_bounds__(THREADS) logprob_kernel(const FwdParams p) {
  __shared__ Part parts[THREADS / 32];
  __shared__ u64 keys[THREADS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wait_prior_grid();
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.logits + row * p.stride;
  const int V = p.vocab;
  Part a = empty_part();
  for (int v = tid; v < V; v += THREADS) a.m = fmaxf(a.m, to_f(x[v]));  // drops NaN
  for (int v = tid; v < V; v += THREADS) {
    const float f = to_f(x[v]);
    if (f == a.m && f > neg_inf() && f < pos_inf()) {
      a.n += 1.0f;
      continue;
    }
    if (f == neg_inf()) continue;
    const float d = max_nan((f - a.m) * p.scale, -1000.0f), e = ex2(d);
    a.s += e;
    a.u = fmaf(e, d, a.u);
  }
  a = warp_join(a, p.scale);
  if (lane == 0) parts[warp] = a;
  __syncthreads();
  a = parts[0];
  for (int w = 1; w < THREADS / 32; ++w) a = join(a, parts[w], p.scale);
  const Row r = row_of(a, p.inv_t);
  if (tid == 0) {
    uint32_t st = r.bad ? MTR_ROW_NONFINITE : r.none ? MTR_ROW_ALL_MASKED : 0u;
    if (p.tokens) {
      const int64_t t = load_id(p.tokens, p.ids32, row);
      if (t >= V) st |= MTR_ROW_BAD_ID;
      if (p.logprobs) p.logprobs[row] = (t < 0 || t >= V) ? 0.0f : log_prob(to_f(x[t]), r, p.inv_t);
    }
    if (p.entropy) p.entropy[row] = r.entropy;
    if (p.lse) p.lse[row] = r.lse;
    if (p.stats) p.stats[row] = make_float4(r.m, r.log_s, r.entropy, 0.0f);
    if (p.status) p.status[row] = st;
  }
  u64 last = ~0ull;
  for (int j = 0; j < p.top_n; ++j) {
    u64 best = 0;
    if (!r.bad && last)
      for (int v = tid; v < V; v += THREADS) {
        const float f = to_f(x[v]);
        const u64 k = f > neg_inf() ? order_key(f, (uint32_t)v) : 0;
        if (k < last && k > best) best = k;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 q = __shfl_xor_sync(FULL, best, o);
      best = q > best ? q : best;
    }
    if (lane == 0) keys[warp] = best;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) best = keys[w] > best ? keys[w] : best;
    __syncthreads();
    if (tid == 0) {
      p.top_ids[row * p.top_n + j] = best ? key_id(best) : -1;
      p.top_logprobs[row * p.top_n + j] = r.bad ? qnan() : best ? log_prob(key_value(best), r, p.inv_t) : neg_inf();
    }
    last = best;
  }
}

// grad_v = [p_v (a + b log2 p_v) + (what is given to v alone)] / T, a row of four coefficients
struct GradRow {
  float m, log2_s, a, b;
  bool bad, none;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) logprob_grad_kernel(const GradParams p) {
  const int tid = threadIdx.x;
  wait_prior_grid();
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.logits + row * p.stride;
  T* g = (T*)p.grad + row * p.grad_stride;
  const int V = p.vocab;
  const float4 st = p.stats[row];
  const int64_t tok = p.tokens ? load_id(p.tokens, p.ids32, row) : -1;
  const bool has = tok >= 0 && tok < V;
  const float gt = has && p.g_logprobs ? p.g_logprobs[row] : 0.0f;
  const float gh = p.g_entropy ? p.g_entropy[row] : 0.0f;
  float even = (p.g_lse ? p.g_lse[row] : 0.0f) - gt - gh * st.z;
  for (int j = 0; j < p.top_n; ++j)
    if (p.top_ids[row * p.top_n + j] >= 0) even -= p.g_top[row * p.top_n + j];
  const bool bad = !(st.y == st.y), none = st.x == neg_inf();
  const float log2_s = st.y * LOG2E_D, slope = -gh * LN2;
  for (int v = tid; v < V; v += THREADS) {
    const float d = max_nan(fmaf(to_f(x[v]) - st.x, p.scale, -log2_s), -1000.0f);
    float r = ex2(d) * fmaf(slope, d, even);
    if (has && v == tok) r += gt;
    for (int j = 0; j < p.top_n; ++j)
      if (p.top_ids[row * p.top_n + j] == v) r += p.g_top[row * p.top_n + j];
    g[v] = from_f<T>(bad ? qnan() : none ? 0.0f : r * p.inv_t);
  }
}

template <typename K, typename P>
static cudaError_t launch(K kern, const P& p, int64_t grid, int threads, cudaStream_t s) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = launch_attrs(attr, 1, true);
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

static int esize(int32_t dtype) { return dtype == MTR_DTYPE_F32 ? 4 : 2; }

// whether two row-strided matrices share a byte
static bool overlap(const void* a, int64_t sa, const void* b, int64_t sb, int64_t rows, int64_t cols, int64_t es) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  const uintptr_t a1 = a0 + (uintptr_t)(((rows - 1) * sa + cols) * es), b1 = b0 + (uintptr_t)(((rows - 1) * sb + cols) * es);
  return a0 < b1 && b0 < a1;
}

template <typename A>
static int check_common(const A* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(A)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
  if (a->logits_dtype < MTR_DTYPE_F32 || a->logits_dtype > MTR_DTYPE_F16) return MTR_ERR_BAD_PARAM;
  if (a->tokens_dtype != MTR_IDS_I64 && a->tokens_dtype != MTR_IDS_I32) return MTR_ERR_BAD_PARAM;
  if (a->top_n < 0 || a->top_n > MTR_MAX_TOP_N) return MTR_ERR_BAD_PARAM;
  if (!(a->temperature > 0.0f) || !(a->temperature < INFINITY) || !(1.4426950408889634f / a->temperature < INFINITY))
    return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  if (!a->logits) return MTR_ERR_NULL_ARG;
  if (a->logits_row_stride < a->vocab) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->logits % esize(a->logits_dtype) || (uintptr_t)a->tokens % (a->tokens_dtype == MTR_IDS_I64 ? 8 : 4))
    return MTR_ERR_ALIGNMENT;
  return MTR_OK;
}

}  // namespace lp
}  // namespace mtr

// ---------------------------------------------------------------- C ABI
using namespace mtr::lp;

int mtr_logprob_validate(const MtrLogprobArgs* a) {
  const int v = check_common(a);
  if (v != MTR_OK || a->rows == 0) return v;
  if (a->out_logprobs && !a->tokens) return MTR_ERR_NULL_ARG;
  if (a->top_n > 0 && (!a->out_top_ids || !a->out_top_logprobs)) return MTR_ERR_NULL_ARG;
  if ((uintptr_t)a->out_logprobs % 4 || (uintptr_t)a->out_entropy % 4 || (uintptr_t)a->out_lse % 4 ||
      (uintptr_t)a->out_top_ids % 8 || (uintptr_t)a->out_top_logprobs % 4 || (uintptr_t)a->out_stats % 16 ||
      (uintptr_t)a->out_status % 4)
    return MTR_ERR_ALIGNMENT;
  return MTR_OK;
}

int mtr_logprob_launch(const MtrLogprobArgs* a, void* stream) {
  const int v = mtr_logprob_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  FwdParams p;
  p.logits = a->logits;
  p.stride = a->logits_row_stride;
  p.tokens = a->tokens;
  p.ids32 = a->tokens_dtype == MTR_IDS_I32;
  p.rows = a->rows;
  p.vocab = a->vocab;
  p.top_n = a->top_n;
  p.scale = (float)(1.4426950408889634 / (double)a->temperature);
  p.inv_t = (float)(1.0 / (double)a->temperature);
  p.logprobs = a->out_logprobs;
  p.entropy = a->out_entropy;
  p.lse = a->out_lse;
  p.top_ids = a->out_top_ids;
  p.top_logprobs = a->out_top_logprobs;
  p.stats = (float4*)a->out_stats;
  p.status = a->out_status;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  switch (a->logits_dtype) {
    case MTR_DTYPE_F32: e = launch(logprob_kernel<float>, p, p.rows, THREADS, s); break;
    case MTR_DTYPE_BF16: e = launch(logprob_kernel<__nv_bfloat16>, p, p.rows, THREADS, s); break;
    default: e = launch(logprob_kernel<__half>, p, p.rows, THREADS, s); break;
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}

int mtr_logprob_grad_validate(const MtrLogprobGradArgs* a) {
  const int v = check_common(a);
  if (v != MTR_OK || a->rows == 0) return v;
  if (!a->stats || !a->grad_logits) return MTR_ERR_NULL_ARG;
  if (a->g_logprobs && !a->tokens) return MTR_ERR_NULL_ARG;
  if (a->top_n > 0 && (!a->top_ids || !a->g_top)) return MTR_ERR_NULL_ARG;
  if (a->grad_row_stride < a->vocab) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->stats % 16 || (uintptr_t)a->top_ids % 8 || (uintptr_t)a->g_logprobs % 4 ||
      (uintptr_t)a->g_entropy % 4 || (uintptr_t)a->g_lse % 4 || (uintptr_t)a->g_top % 4 ||
      (uintptr_t)a->grad_logits % esize(a->logits_dtype))
    return MTR_ERR_ALIGNMENT;
  if (overlap(a->logits, a->logits_row_stride, a->grad_logits, a->grad_row_stride, a->rows, a->vocab, esize(a->logits_dtype)))
    return MTR_ERR_BAD_PARAM;
  return MTR_OK;
}

int mtr_logprob_grad_launch(const MtrLogprobGradArgs* a, void* stream) {
  const int v = mtr_logprob_grad_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  GradParams p;
  p.logits = a->logits;
  p.stride = a->logits_row_stride;
  p.tokens = a->tokens;
  p.ids32 = a->tokens_dtype == MTR_IDS_I32;
  p.rows = a->rows;
  p.vocab = a->vocab;
  p.top_n = a->top_n;
  p.scale = (float)(1.4426950408889634 / (double)a->temperature);
  p.inv_t = (float)(1.0 / (double)a->temperature);
  p.stats = (const float4*)a->stats;
  p.top_ids = a->top_ids;
  p.g_logprobs = a->g_logprobs;
  p.g_entropy = a->g_entropy;
  p.g_lse = a->g_lse;
  p.g_top = a->g_top;
  p.grad = a->grad_logits;
  p.grad_stride = a->grad_row_stride;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  switch (a->logits_dtype) {
    case MTR_DTYPE_F32: e = launch(logprob_grad_kernel<float>, p, p.rows, THREADS, s); break;
    case MTR_DTYPE_BF16: e = launch(logprob_grad_kernel<__nv_bfloat16>, p, p.rows, THREADS, s); break;
    default: e = launch(logprob_grad_kernel<__half>, p, p.rows, THREADS, s); break;
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}
