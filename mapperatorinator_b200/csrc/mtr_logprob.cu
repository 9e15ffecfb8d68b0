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
// sums are fp32.
//
// The forward kernel reads a row once, in 16-byte vectors, and is bound by
// HBM as long as a score costs few instructions: 6.5 TB/s feed an SM 12 bf16
// scores a clock, and its four schedulers issue 128 lanes, so 10 a score are
// all there are.  Per score: unpack (1), the two packed steps of
// t = (x - m) (-log2(e) / T) (2 x 1/2), one unsigned minimum, 2^-t (1), and the
// packed sums of 2^-t and of 2^-t t (2 x 1/2); the maximum is packed too (1/2).
// The minimum does three things at once: t >= 0 compares as an unsigned word,
// so masked scores (t = +inf) and far ones become t = 1000, whose 2^-t is 0
// and whose product with t is 0 as well (inf would give NaN), and a score equal
// to the maximum, whose t is -0 = 0x80000000, becomes 1000 too and so leaves
// the sums: it is counted in n.  NaN is found by the maximum, which keeps it.
#include <stdio.h>
#include <stdlib.h>
#include "mtr_common.cuh"

namespace mtr {
namespace lp {

constexpr float LN2 = 0x1.62e430p-1f;
constexpr float LOG2E_D = 0x1.715476p+0f;

struct FwdParams {
  const void* logits;
  int64_t stride;
  const void* tokens;
  int32_t ids32;
  int32_t rows;
  int32_t vocab;
  int32_t top_n;
  int32_t cluster;  // CTAs of a row
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

// What one lane, warp, CTA or cluster holds of a row: the largest logit, how
// many logits equal it, and the sums over the others.  s is NaN once a logit is
// NaN or +inf.
struct Part {
  float m;   // -inf: nothing but masked scores so far
  float n;   // logits equal to m (0 while m = -inf)
  float s;   // sum of 2^-t over the others
  float u;   // sum of 2^-t t
};

__device__ __forceinline__ Part empty_part() { return Part{neg_inf(), 0.0f, 0.0f, 0.0f}; }

// `p` about a larger maximum M: its terms shrink by 2^-g, g = (M - m) scale, and
// each t grows by g; what equalled m is one of the others now.
__device__ __forceinline__ void move_to(Part& p, float M, float scale) {
  if (p.m > neg_inf()) {
    const float g = fminf((M - p.m) * scale, 1000.0f), f = ex2(-g), t = p.s + p.n;
    p.s = t * f;
    p.u = fmaf(t, g, p.u) * f;
    p.n = 0.0f;
  }
  p.m = M;
}
__device__ __forceinline__ Part join(Part a, Part b, float scale) {
  const float M = fmaxf(a.m, b.m);
  if (a.m < M) move_to(a, M, scale);
  if (b.m < M) move_to(b, M, scale);
  return Part{M, a.n + b.n, a.s + b.s, a.u + b.u};
}
// join of lanes 0 .. width - 1 (a power of two), the same result in each of them
__device__ __forceinline__ Part lanes_join(Part p, int width, float scale) {
  for (int o = 1; o < width; o <<= 1) {
    const Part q{__shfl_xor_sync(FULL, p.m, o), __shfl_xor_sync(FULL, p.n, o), __shfl_xor_sync(FULL, p.s, o),
                 __shfl_xor_sync(FULL, p.u, o)};
    p = join(p, q, scale);
  }
  return p;
}

// What the sums of a whole row say.
struct Row {
  float m, log_s, entropy, lse;
  bool bad, none;
};
__device__ __forceinline__ Row row_of(const Part& p, float inv_t) {
  Row r;
  r.m = p.m;
  r.bad = !(p.s < pos_inf());
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
    r.entropy = r.log_s + LN2 * p.u / (1.0f + rest);
    r.lse = fmaf(p.m, inv_t, r.log_s);
  }
  return r;
}
__device__ __forceinline__ float log_prob(float x, const Row& r, float inv_t) {
  if (r.bad) return qnan();
  if (r.none || x == neg_inf()) return neg_inf();
  return (x - r.m) * inv_t - r.log_s;
}

// 16 bytes of a row's logits.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static constexpr uint32_t FILL = 0xff800000u;  // -inf
  typedef float Top;                             // the largest of a vector; NaN when one is
  static __device__ __forceinline__ Top top(const uint4& w) {
    return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ Top larger(Top a, Top b) { return max_nan(a, b); }
  static __device__ __forceinline__ float value(Top t) { return t; }
  static __device__ __forceinline__ Top pattern(float m) { return m; }
  static __device__ __forceinline__ bool has(Top t, Top m) { return t == m; }
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
  typedef __nv_bfloat162 Top;
  static __device__ __forceinline__ Top pair(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
  static __device__ __forceinline__ Top top(const uint4& w) {
    return __hmax2_nan(__hmax2_nan(pair(w.x), pair(w.y)), __hmax2_nan(pair(w.z), pair(w.w)));
  }
  static __device__ __forceinline__ Top larger(Top a, Top b) { return __hmax2_nan(a, b); }
  static __device__ __forceinline__ float value(Top t) { return max_nan(__low2float(t), __high2float(t)); }
  static __device__ __forceinline__ Top pattern(float m) { return __float2bfloat162_rn(m); }
  static __device__ __forceinline__ bool has(Top t, Top m) { return __heq2_mask(t, m) != 0u; }
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
  typedef __half2 Top;
  static __device__ __forceinline__ Top pair(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
  static __device__ __forceinline__ Top top(const uint4& w) {
    return __hmax2_nan(__hmax2_nan(pair(w.x), pair(w.y)), __hmax2_nan(pair(w.z), pair(w.w)));
  }
  static __device__ __forceinline__ Top larger(Top a, Top b) { return __hmax2_nan(a, b); }
  static __device__ __forceinline__ float value(Top t) { return max_nan(__low2float(t), __high2float(t)); }
  static __device__ __forceinline__ Top pattern(float m) { return __float2half2_rn(m); }
  static __device__ __forceinline__ bool has(Top t, Top m) { return __heq2_mask(t, m) != 0u; }
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

__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
// the lanes' values in descending order (none is NaN)
__device__ __forceinline__ float warp_sort_desc(float v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor_sync(FULL, v, j);
      const bool desc = (lane & k) == 0, low = (lane & j) == 0;
      v = (desc == low) ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

constexpr int MAX_WARPS = 8;
constexpr int MAX_CLUSTER = 8;
constexpr int LIST = 512;  // candidates of a row's alternatives

struct Shared {
  Part part[MAX_WARPS];
  float nth[MAX_WARPS], rth[MAX_WARPS];
  Part cta;         // read by the cluster's other CTAs
  float cta_nth, cta_rth;
  int count;        // candidates listed (may pass LIST: then the list is not complete)
  uint8_t winner[MAX_WARPS][32];
  u64 key[MAX_WARPS];
  u64 list[LIST];
};

// One row per CTA, or per cluster of CTAs, of up to 8 warps.
//
// The row is its 16-byte vectors, dealt to the CTAs in runs and to the threads
// in turn, and up to 2 (E - 1) logits before the first boundary and behind the
// last, which are lanes' single scores of the first warp.  A thread has TV
// vectors in flight; a warp keeps one maximum (one redux for each tile of TV
// vectors), so that its lanes' sums move to a new maximum together and rarely.
//
// Alternatives: with lm the lanes' maxima, any T with at least n logits >= T
// bounds the n largest from below.  Two such T are at hand: the n-th largest lm
// of a warp, the best warp's taken, and the smallest over all warps of the r-th
// largest lm, r n-th part of the warps (n <= r warps).  The larger of the two
// leaves about n to 3 n lanes with lm >= T, whose vectors are read again (from
// L2) for the list of candidates, which are ranked by comparing all pairs.  A
// list that overflows (many equal logits) falls back to one pass for each
// alternative.
template <typename T, int TV>
__global__ void __launch_bounds__(MAX_WARPS * 32, 2) logprob_kernel(const FwdParams p) {
  typedef Vec<T> X;
  constexpr int E = X::E;
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = blockDim.x, warps = threads >> 5;
  const int cs = p.cluster, rank = cs > 1 ? (int)(blockIdx.x % cs) : 0;
  const int64_t row = cs > 1 ? blockIdx.x / cs : blockIdx.x;
  const int V = p.vocab;
  const float scale = p.scale;
  if (tid == 0) sh.count = 0;
  wait_prior_grid();
  const T* x = (const T*)p.logits + row * p.stride;
  // the token and its logit, needed last, are asked for first
  int64_t token = -1;
  float token_x = 0.0f;
  if (tid == 0 && rank == 0 && p.tokens) {
    token = load_id(p.tokens, p.ids32, row);
    if (token >= 0 && token < V) token_x = to_f(x[token]);
  }
  const int off = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int head = min(off ? E - off : 0, V), vecs = (V - head) / E, tail = V - head - vecs * E;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int run = (vecs + cs - 1) / cs, v0 = min(rank * run, vecs), v1 = min(v0 + run, vecs);

  Part a = empty_part();
  float lm = neg_inf();  // the lane's largest logit
  // the single scores: lanes 0 .. head - 1 and 16 .. 16 + tail - 1
  float single = neg_inf();
  int single_id = -1;
  if (warp == 0 && rank == 0) {
    if (lane < head) single_id = lane;
    else if (lane >= 16 && lane < 16 + tail) single_id = V - tail + lane - 16;
    if (single_id >= 0) single = to_f(x[single_id]);
  }
  bool bad = false;
  if (warp == 0 && rank == 0 && head + tail > 0) {
    const float top = warp_max_nan(single);
    bad = !(top < pos_inf());
    if (!bad && top > neg_inf()) {
      a.m = top;
      if (single == top) a.n = 1.0f;
      else if (single > neg_inf()) {
        const float t = fminf((top - single) * scale, 1000.0f);
        a.s = ex2(-t);
        a.u = a.s * t;
      }
      lm = single;
    }
  }
  u64 s2 = 0, u2 = 0;  // pairs of partial sums, added to a.s, a.u when the maximum moves
  for (int t0 = v0; t0 < v1; t0 += threads * TV) {
    uint4 w[TV];
    typename X::Top top[TV];
#pragma unroll
    for (int j = 0; j < TV; ++j) {
      const int i = t0 + j * threads + tid;
      w[j] = i < v1 ? body[i] : make_uint4(X::FILL, X::FILL, X::FILL, X::FILL);
    }
#pragma unroll
    for (int j = 0; j < TV; ++j) top[j] = X::top(w[j]);
    typename X::Top all = top[0];
#pragma unroll
    for (int j = 1; j < TV; ++j) all = X::larger(all, top[j]);
    const float mine = X::value(all), most = warp_max_nan(mine);
    if (!(most < pos_inf())) bad = true;
    lm = fmaxf(lm, mine);
    if (most > a.m) {
      float lo, hi;
      up2(s2, lo, hi);
      a.s += lo + hi;
      up2(u2, lo, hi);
      a.u += lo + hi;
      s2 = u2 = 0;
      move_to(a, most, scale);
    }
    if (bad || !(a.m > neg_inf())) continue;
    if (mine == a.m) {
      const typename X::Top m = X::pattern(a.m);
#pragma unroll
      for (int j = 0; j < TV; ++j)
        if (X::has(top[j], m)) {
          float f[E];
          X::unpack(w[j], f);
#pragma unroll
          for (int e = 0; e < E; ++e) a.n += f[e] == a.m ? 1.0f : 0.0f;
        }
    }
    const float nm = 0.0f - a.m;  // +0 for both zeros, so that equal scores differ by +0
    const u64 nm2 = pk2(nm, nm), ns2 = pk2(-scale, -scale);
#pragma unroll
    for (int j = 0; j < TV; ++j) {
      float f[E];
      X::unpack(w[j], f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float t0f, t1f;
        up2(mul2(add2(pk2(f[e], f[e + 1]), nm2), ns2), t0f, t1f);
        t0f = __uint_as_float(min(__float_as_uint(t0f), 0x447a0000u));  // 1000
        t1f = __uint_as_float(min(__float_as_uint(t1f), 0x447a0000u));
        const u64 e2 = pk2(ex2(-t0f), ex2(-t1f));
        s2 = add2(s2, e2);
        u2 = fma2(e2, pk2(t0f, t1f), u2);
      }
    }
  }
  {
    float lo, hi;
    up2(s2, lo, hi);
    a.s += lo + hi;
    up2(u2, lo, hi);
    a.u += lo + hi;
  }
  a.n = warp_sum(a.n);
  a.s = warp_sum(a.s);
  a.u = warp_sum(a.u);
  if (bad) a = Part{neg_inf(), 0.0f, qnan(), 0.0f};

  // join the warps, then the CTAs
  const int n = p.top_n;
  float nth = neg_inf(), rth = neg_inf();
  if (n > 0) {
    const float sorted = warp_sort_desc(lm, lane);
    nth = __shfl_sync(FULL, sorted, n - 1);
    rth = __shfl_sync(FULL, sorted, (n + warps * cs - 1) / (warps * cs) - 1);
  }
  if (warps > 1) {
    if (lane == 0) {
      sh.part[warp] = a;
      sh.nth[warp] = nth;
      sh.rth[warp] = rth;
    }
    __syncthreads();
    const int width = MAX_WARPS;
    a = lane < warps ? sh.part[lane] : empty_part();
    a = lanes_join(a, width, scale);
    nth = lane < warps ? sh.nth[lane] : neg_inf();
    rth = lane < warps ? sh.rth[lane] : pos_inf();
#pragma unroll
    for (int o = 1; o < MAX_WARPS; o <<= 1) {
      nth = fmaxf(nth, __shfl_xor_sync(FULL, nth, o));
      rth = fminf(rth, __shfl_xor_sync(FULL, rth, o));
    }
    // lanes 8 .. 31 joined empty parts: lane 0 has the CTA's
    a = Part{__shfl_sync(FULL, a.m, 0), __shfl_sync(FULL, a.n, 0), __shfl_sync(FULL, a.s, 0), __shfl_sync(FULL, a.u, 0)};
    nth = __shfl_sync(FULL, nth, 0);
    rth = __shfl_sync(FULL, rth, 0);
  } else {
    __syncwarp();  // sh.count = 0 before the first candidate
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (cs > 1) {
    if (tid == 0) {
      sh.cta = a;
      sh.cta_nth = nth;
      sh.cta_rth = rth;
    }
    cluster.sync();
    Part q = empty_part();
    float qn = neg_inf(), qr = pos_inf();
    if (lane < cs) {
      const Shared* other = cluster.map_shared_rank(&sh, lane);
      q = other->cta;
      qn = other->cta_nth;
      qr = other->cta_rth;
    }
    a = lanes_join(q, MAX_CLUSTER, scale);
#pragma unroll
    for (int o = 1; o < MAX_CLUSTER; o <<= 1) {
      qn = fmaxf(qn, __shfl_xor_sync(FULL, qn, o));
      qr = fminf(qr, __shfl_xor_sync(FULL, qr, o));
    }
    a = Part{__shfl_sync(FULL, a.m, 0), __shfl_sync(FULL, a.n, 0), __shfl_sync(FULL, a.s, 0), __shfl_sync(FULL, a.u, 0)};
    nth = __shfl_sync(FULL, qn, 0);
    rth = __shfl_sync(FULL, qr, 0);
  }
  const Row r = row_of(a, p.inv_t);
  if (tid == 0 && rank == 0) {
    uint32_t st = r.bad ? MTR_ROW_NONFINITE : r.none ? MTR_ROW_ALL_MASKED : 0u;
    if (p.tokens) {
      if (token >= V) st |= MTR_ROW_BAD_ID;
      if (p.logprobs) p.logprobs[row] = (token < 0 || token >= V) ? 0.0f : log_prob(token_x, r, p.inv_t);
    }
    if (p.entropy) p.entropy[row] = r.entropy;
    if (p.lse) p.lse[row] = r.lse;
    if (p.stats) p.stats[row] = make_float4(r.m, r.log_s, r.entropy, 0.0f);
    if (p.status) p.status[row] = st;
  }
  if (n == 0) {
    if (cs > 1) cluster.sync();  // this CTA's parts have been read
    return;
  }

  // candidates
  const float bound = fmaxf(nth, rth);
  auto push = [&](float f, int id) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < LIST) sh.list[at] = order_key(f, (uint32_t)id);
  };
  if (!r.bad && !r.none) {
    if (single >= bound && single > neg_inf()) push(single, single_id);
    // the winners' vectors, dealt to the lanes in turn, four loads in flight each
    const bool won = lm >= bound && lm > neg_inf();
    const unsigned winners = __ballot_sync(FULL, won);
    if (won) sh.winner[warp][__popc(winners & ((1u << lane) - 1u))] = (uint8_t)lane;
    __syncwarp();
    const int each = (v1 - v0 - warp * 32 + threads - 1) / threads;  // vectors of the warp's first lane
    const int all = each > 0 ? __popc(winners) * each : 0;
    for (int base = 0; base < all; base += 128) {
      uint4 w[4];
      int at[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = base + j * 32 + lane, who = k / each;
        at[j] = k < all ? v0 + warp * 32 + sh.winner[warp][who] + (k - who * each) * threads : v1;
        w[j] = at[j] < v1 ? body[at[j]] : make_uint4(X::FILL, X::FILL, X::FILL, X::FILL);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float most = X::value(X::top(w[j]));
        if (most >= bound && most > neg_inf()) {
          float f[E];
          X::unpack(w[j], f);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (f[e] >= bound && f[e] > neg_inf()) push(f[e], head + at[j] * E + e);
        }
      }
    }
  }
  __syncthreads();
  int c = sh.count;
  if (cs > 1) {
    cluster.sync();
    if (rank == 0 && c <= LIST) {
      for (int k = 1; k < cs && c <= LIST; ++k) {
        const Shared* other = cluster.map_shared_rank(&sh, k);
        const int more = other->count;
        if (c + more <= LIST)
          for (int i = tid; i < more; i += threads) sh.list[c + i] = other->list[i];
        c += more;
      }
    }
    __syncthreads();
    cluster.sync();  // the others' lists have been read
    if (rank != 0) return;
  }
  int64_t* ids = p.top_ids + row * n;
  float* lps = p.top_logprobs + row * n;
  if (c <= LIST) {
    for (int i = tid; i < c; i += threads) {
      const u64 k = sh.list[i];
      int place = 0;
      for (int j = 0; j < c; ++j) place += sh.list[j] > k;
      if (place < n) {
        ids[place] = key_id(k);
        lps[place] = log_prob(key_value(k), r, p.inv_t);
      }
    }
    for (int j = c + tid; j < n; j += threads) {
      ids[j] = -1;
      lps[j] = r.bad ? qnan() : neg_inf();
    }
    return;
  }
  // the list overflowed: the largest key below the last one, n times
  u64 last = ~0ull;
  for (int j = 0; j < n; ++j) {
    u64 best = 0;
    if (last)
      for (int v = tid; v < V; v += threads) {
        const float f = to_f(x[v]);
        const u64 k = f > neg_inf() ? order_key(f, (uint32_t)v) : 0;
        if (k < last && k > best) best = k;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 q = __shfl_xor_sync(FULL, best, o);
      best = q > best ? q : best;
    }
    if (lane == 0) sh.key[warp] = best;
    __syncthreads();
    for (int w = 0; w < warps; ++w) best = sh.key[w] > best ? sh.key[w] : best;
    __syncthreads();
    if (tid == 0) {
      ids[j] = best ? key_id(best) : -1;
      lps[j] = best ? log_prob(key_value(best), r, p.inv_t) : neg_inf();
    }
    last = best;
  }
}

// grad_v = p_v (a + b log2 p_v) + (what is given to v alone), a and b one row's
// two numbers (both divided by T).  One CTA owns a run of a row's vectors and
// asks for them before anything else; the row's numbers arrive meanwhile.  The
// few ids that are given something of their own (the token, the alternatives)
// are written once more, in full precision, after the run: one thread for each
// distinct id, so a token that is also an alternative is summed before the
// rounding.  4 bytes of traffic for a bf16 score and about 6 instructions: HBM
// bounds it.
struct GradRow {
  float m, log2_s, a, b;
};
template <typename T>
__device__ __forceinline__ float grad_of(T x, const GradRow& r, float scale) {
  const float d = max_nan(fmaf(to_f(x) - r.m, scale, -r.log2_s), -1000.0f);
  return ex2(d) * fmaf(r.b, d, r.a);
}

constexpr int GRAD_VECS = 4;  // vectors a thread holds
constexpr int MAX_SLOTS = MTR_MAX_TOP_N + 1;

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

// ALIKE: logits and gradient rows lie alike about the 16-byte boundaries, so one
// division into vectors serves both; else every logit is its own access.
template <typename T, bool ALIKE>
__global__ void __launch_bounds__(256) logprob_grad_kernel(const GradParams p) {
  typedef Vec<T> X;
  constexpr int E = X::E;
  __shared__ int32_t slot_id[MAX_SLOTS];
  __shared__ float slot_g[MAX_SLOTS];
  const int tid = threadIdx.x, threads = blockDim.x;
  wait_prior_grid();
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.logits + row * p.stride;
  T* g = (T*)p.grad + row * p.grad_stride;
  const int V = p.vocab, span = threads * GRAD_VECS;
  const int off = ALIKE ? (int)(((uintptr_t)x & 15u) / sizeof(T)) : 0;
  const int head = min(off ? E - off : 0, V), vecs = (V - head) / E;
  const int v0 = (int)blockIdx.y * span, v1 = min(v0 + span, vecs);
  // the CTA's scores: its vectors, the first run those before them, the last those behind
  const bool last = blockIdx.y == gridDim.y - 1;
  const int from = v0 == 0 ? 0 : head + min(v0, vecs) * E, to = last ? V : head + v1 * E;
  uint4 w[GRAD_VECS];
  if (ALIKE) {
#pragma unroll
    for (int j = 0; j < GRAD_VECS; ++j) {
      const int i = v0 + j * threads + tid;
      if (i < v1) w[j] = reinterpret_cast<const uint4*>(x + head)[i];
    }
  }

  const float4 st = p.stats[row];
  const int64_t tok = p.tokens ? load_id(p.tokens, p.ids32, row) : -1;
  const bool has = tok >= 0 && tok < V;
  const float gt = has && p.g_logprobs ? p.g_logprobs[row] : 0.0f;
  const float gh = p.g_entropy ? p.g_entropy[row] : 0.0f;
  float even = (p.g_lse ? p.g_lse[row] : 0.0f) - gt - gh * st.z;
  const int slots = 1 + p.top_n;
  if (p.top_n > 0) {
    if (tid < p.top_n) {
      const int64_t id = p.top_ids[row * p.top_n + tid];
      const bool ok = id >= 0 && id < V;
      slot_id[1 + tid] = ok ? (int32_t)id : -1;
      slot_g[1 + tid] = ok ? p.g_top[row * p.top_n + tid] : 0.0f;
    }
    if (tid == 0) {
      slot_id[0] = has ? (int32_t)tok : -1;
      slot_g[0] = gt;
    }
    __syncthreads();
    for (int j = 1; j < slots; ++j) even -= slot_g[j];
  }
  const bool bad = !(st.y == st.y), none = st.x == neg_inf();
  // a row without a finite score has gradient 0, one with a NaN NaN: 2^d with d = -1000 or NaN times a = 0
  GradRow r;
  r.m = none ? 0.0f : st.x;
  r.log2_s = st.y * LOG2E_D;
  r.a = none ? 0.0f : bad ? qnan() : even * p.inv_t;
  r.b = none ? 0.0f : -gh * LN2 * p.inv_t;

  if (ALIKE) {
    const u64 nm2 = pk2(-r.m, -r.m), sc2 = pk2(p.scale, p.scale), nl2 = pk2(-r.log2_s, -r.log2_s), a2 = pk2(r.a, r.a), b2 = pk2(r.b, r.b);
#pragma unroll
    for (int j = 0; j < GRAD_VECS; ++j) {
      const int i = v0 + j * threads + tid;
      if (i < v1) {
        float f[E];
        X::unpack(w[j], f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          float d0, d1;
          up2(fma2(add2(pk2(f[e], f[e + 1]), nm2), sc2, nl2), d0, d1);
          d0 = max_nan(d0, -1000.0f);
          d1 = max_nan(d1, -1000.0f);
          up2(mul2(pk2(ex2(d0), ex2(d1)), fma2(b2, pk2(d0, d1), a2)), f[e], f[e + 1]);
        }
        reinterpret_cast<uint4*>(g + head)[i] = pack<T>(f);
      }
    }
    if (v0 == 0 && tid < head) g[tid] = from_f<T>(grad_of(x[tid], r, p.scale));
    const int behind = head + vecs * E;
    if (last && tid < V - behind) g[behind + tid] = from_f<T>(grad_of(x[behind + tid], r, p.scale));
  } else {
    for (int v = from + tid; v < to; v += threads) g[v] = from_f<T>(grad_of(x[v], r, p.scale));
  }

  if (none || bad) return;
  if (p.top_n == 0) {
    if (!has || tok < from || tok >= to) return;
    __syncthreads();  // after the run's own store of this id
    if (tid == 0) g[tok] = from_f<T>(fmaf(gt, p.inv_t, grad_of(x[tok], r, p.scale)));
    return;
  }
  __syncthreads();
  if (tid < slots) {
    const int id = slot_id[tid];
    bool mine = id >= from && id < to;
    float own = 0.0f;
    for (int j = 0; j < slots; ++j)
      if (slot_id[j] == id) {
        if (j < tid) mine = false;  // an earlier slot writes it
        own += slot_g[j];
      }
    if (mine) g[id] = from_f<T>(fmaf(own, p.inv_t, grad_of(x[id], r, p.scale)));
  }
}

template <typename K, typename P>
static cudaError_t launch(K kern, const P& p, dim3 grid, int threads, int cluster, cudaStream_t s) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = launch_attrs(attr, cluster, true);
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

static int esize(int32_t dtype) { return dtype == MTR_DTYPE_F32 ? 4 : 2; }

constexpr int TILE = 16;

// Warps and CTAs of a row.
struct Shape {
  int threads, cluster;
};
static Shape shape_for(int64_t rows, int vocab, int es) {
  const int64_t vecs = ((int64_t)vocab * es + 15) / 16, sms = device_sms();
  const char* ov = getenv("LPSHAPE");
  if (ov) { int w, c; sscanf(ov, "%d,%d", &w, &c); return {32 * w, c}; }
  int warps = 1;
  while (warps < MAX_WARPS && (vecs > 32ll * TILE * warps || (rows * warps < 16 * sms && vecs > 128 * warps))) warps *= 2;
  int cluster = 1;
  while (cluster < MAX_CLUSTER && vecs > 4096ll * cluster) cluster *= 2;
  return {32 * warps, cluster};
}

template <typename T>
static cudaError_t launch_grad(const GradParams& p, cudaStream_t s) {
  const int64_t es = sizeof(T), vecs = (p.vocab * es + 15) / 16;
  int threads = 64;
  while (threads < 256 && vecs > threads * GRAD_VECS) threads *= 2;
  const dim3 grid((unsigned)p.rows, (unsigned)((vecs + threads * GRAD_VECS - 1) / (threads * GRAD_VECS)), 1);
  // alike in row 0 and in every step to the next row
  const bool alike = (((uintptr_t)p.logits ^ (uintptr_t)p.grad) & 15u) == 0 && ((p.stride - p.grad_stride) * es) % 16 == 0;
  return alike ? launch(logprob_grad_kernel<T, true>, p, grid, threads, 1, s)
               : launch(logprob_grad_kernel<T, false>, p, grid, threads, 1, s);
}

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
  if (a->rows < 0 || a->rows > MTR_MAX_SCORE_ROWS || a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
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
  const Shape g = shape_for(p.rows, p.vocab, esize(a->logits_dtype));
  p.cluster = g.cluster;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  const dim3 grid((unsigned)(p.rows * g.cluster), 1, 1);
  switch (a->logits_dtype) {
    case MTR_DTYPE_F32: e = launch(logprob_kernel<float, TILE>, p, grid, g.threads, g.cluster, s); break;
    case MTR_DTYPE_BF16: { const char* tv = getenv("LPTV"); int t = tv ? atoi(tv) : TILE;
      e = t == 4 ? launch(logprob_kernel<__nv_bfloat16, 4>, p, grid, g.threads, g.cluster, s) : t == 8 ? launch(logprob_kernel<__nv_bfloat16, 8>, p, grid, g.threads, g.cluster, s) : launch(logprob_kernel<__nv_bfloat16, TILE>, p, grid, g.threads, g.cluster, s); break; }
    default: e = launch(logprob_kernel<__half, TILE>, p, grid, g.threads, g.cluster, s); break;
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
    case MTR_DTYPE_F32: e = launch_grad<float>(p, s); break;
    case MTR_DTYPE_BF16: e = launch_grad<__nv_bfloat16>(p, s); break;
    default: e = launch_grad<__half>(p, s); break;
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}
