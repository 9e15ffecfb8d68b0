// mtr_distill.cu -- losses of a student's logits against a teacher's top ids, and
// their gradient.
//
// A row has n ids with the teacher's log probabilities l_j.  With q the student's
// softmax(logits / T), S the set of the ids and q_t the student's mass outside S:
//   renormalised   p_j = e^(l_j) / sum e^(l),  L = sum_j p_j (log p_j - log q_j)
//   with the tail  p_j = e^(l_j), p_t = 1 - sum p_j,  L + p_t (log p_t - log q_t)
//   T dL / dlogit_v = q_v (P + p_t) - sum_j [v = id_j] p_j       for v in S
//                     q_v P - p_t (1 - q_t) (q_v / q_t)          for the others
// where P = sum_j p_j and p_t = 0 in the first form.
//
// The loss is a difference of nearly equal logarithms, and q_t may be a small part
// of the whole, so nothing is subtracted from a sum: a bitmap of S in shared
// memory takes the ids of S out of the pass over the row (one byte of it a
// 16-byte vector), which gives the sum outside S about the largest logit there
// (fp32 terms, joined in double), and the n terms of S are computed in double.
// Then q_v / q_t is 2^d times one number of the row whose sum is at least 1, and no
// factor leaves the fp32 range.
//
// A row is read from HBM once and its gradient written once.  A CTA, or a cluster of
// them, owns a row and keeps its first HOLD vectors a thread in registers between the
// two passes; what a longer row has behind them comes from L2 the second time.  The
// work of S in double goes on in the first warp while the row is under way.  Losses
// alone run at 6.0 TB/s (1024 x 131072 fp32, 89.3 us).  With gradients of 2-byte rows
// nothing is full (8192 x 4096 bf16 34.3 us where its bytes take 20.8 at HBM's copy rate:
// 0.64 instructions a clock and scheduler, exponentials 51 % of their rate, HBM 29 %
// under the profiler): a row is a chain -- ids, the logits at them, the vectors, sums,
// the row's work in double, the gradient -- that only the SM's other rows cover, of which
// 28 fit at 72 registers.  2000 x 65533 takes 125 us, its bytes 80.  Some 6 us of the 34
// are the rows' work in double, which makes do with one division and one logarithm a
// lane (35.8 with each formed apart).
// More than 32 ids (SLOTS 4) spill under these registers, up to 224 bytes a thread: 8192 x
// 4096 bf16 takes 47 us with 50 ids and 58 with 128, where 20 take 34, 2000 x 65533
// 153 with 50.
#include "mtr_vec.cuh"

namespace mtr {
namespace ds {

constexpr double LEAST_REST = 0x1p-20;  // a smaller p_t is the rounding of the given log probabilities: none

struct Params {
  const void* logits;
  int64_t stride;
  const void* ids;
  int64_t ids_stride;
  const float* lps;
  int64_t lps_stride;
  int32_t ids32;
  int32_t vocab;
  int32_t n;
  int32_t tail;
  int32_t cluster; // CTAs of a row
  int32_t alike;  // logits and gradient rows lie alike about the 16-byte boundaries
  float scale;    // log2(e) / T
  double inv_t;
  float* loss;
  double2* stats;  // written with the loss; read where only the gradient is asked for
  const float* g_loss;
  void* grad;
  int64_t grad_stride;
  uint32_t* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}

// the values of a vector whose bits are set become masked scores
__device__ __forceinline__ void drop(uint4& w, uint32_t bits, float) {
  if (bits & 1u) w.x = 0xff800000u;
  if (bits & 2u) w.y = 0xff800000u;
  if (bits & 4u) w.z = 0xff800000u;
  if (bits & 8u) w.w = 0xff800000u;
}
template <typename T>
__device__ __forceinline__ void drop(uint4& w, uint32_t bits, T) {
  constexpr uint32_t F = Vec<T>::FILL;
  auto half = [&](uint32_t& x, uint32_t two) {
    const uint32_t m = ((two & 1u) ? 0xffffu : 0u) | ((two & 2u) ? 0xffff0000u : 0u);
    x = (x & ~m) | (F & m);
  };
  half(w.x, bits);
  half(w.y, bits >> 2);
  half(w.z, bits >> 4);
  half(w.w, bits >> 6);
}

constexpr int MOST_THREADS = 512;  // whose CTAs may share a row

template <int WARPS>
struct Shared {
  float m[WARPS];    // a warp's largest logit outside S
  double s[WARPS];   // and its sum about it; NaN: a NaN or +inf
  float row_m, row_c;
  float cta_m;       // read by the cluster's other CTAs
  double cta_s;
  int dup;
  int32_t id[MTR_MAX_TEACHER_IDS];
  double p[MTR_MAX_TEACHER_IDS];
};

// HOLD: vectors a thread keeps; CTAS: CTAs of an SM; SLOTS: entries a lane of the
// first warp has (1 or 4)
template <typename T, int THREADS, int HOLD, int CTAS, int SLOTS, bool SCAN, bool GRAD>
__global__ void __launch_bounds__(THREADS, CTAS) distill_kernel(const Params p) {
  typedef Vec<T> X;
  constexpr int E = X::E, WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint32_t bits[];  // bit 8 + id - head
  __shared__ Shared<WARPS> sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int V = p.vocab;
  const int cs = THREADS == MOST_THREADS ? p.cluster : 1, rank = cs > 1 ? (int)(blockIdx.x % cs) : 0;
  const int64_t row = cs > 1 ? blockIdx.x / cs : blockIdx.x;
  cg::cluster_group cluster = cg::this_cluster();
  auto sync = [] {
    if constexpr (THREADS > 32) __syncthreads();
    else __syncwarp();
  };
  wait_prior_grid();

  const T* x = (const T*)p.logits + row * p.stride;
  const int off = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int head = min(off ? E - off : 0, V), vecs = (V - head) / E, behind = V - head - vecs * E;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  // the CTA's vectors [v0, v1); the first one has the single logits before the first 16-byte boundary and behind the last too
  const int run = cs > 1 ? (vecs + cs - 1) / cs : vecs, v0 = min(rank * run, vecs), v1 = min(v0 + run, vecs);
  uint4 w[HOLD];
#pragma unroll
  for (int j = 0; j < HOLD; ++j) {
    const int i = v0 + tid + j * THREADS;
    w[j] = i < v1 ? body[i] : make_uint4(X::FILL, X::FILL, X::FILL, X::FILL);
  }
  const int single = rank > 0 ? -1 : tid < head ? tid : tid >= 16 && tid < 16 + behind ? V - behind + tid - 16 : -1;
  float one = single >= 0 ? to_f(x[single]) : neg_inf();

  // the teacher's entries, of the first warp: entry lane + 32 k
  int id[SLOTS];
  float lp[SLOTS], xs[SLOTS];
  bool wrong = false;
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const int j = lane + 32 * k;
      id[k] = -1;
      lp[k] = xs[k] = neg_inf();
      if (32 * k < p.n && j < p.n) {
        const int64_t at = row * p.ids_stride + j;
        const int64_t v = p.ids32 ? (int64_t)((const int32_t*)p.ids)[at] : ((const int64_t*)p.ids)[at];
        if (v >= 0 && v < V) {
          id[k] = (int)v;
          lp[k] = p.lps[row * p.lps_stride + j];
          xs[k] = to_f(x[v]);
        } else if (v >= V) {
          wrong = true;
        }
      }
    }
  }
  for (int i = tid; i < (V + 8 + 31) / 32; i += THREADS) bits[i] = 0u;
  if (tid == 0) sh.dup = 0;
  sync();
  bool lead[SLOTS];  // the first of equal ids
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      lead[k] = false;
      if (id[k] >= 0) {
        const int b = 8 + id[k] - head;
        lead[k] = !(atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u);
        if (!lead[k]) sh.dup = 1;
      }
    }
  }
  sync();

  auto listed = [&](int i) {  // which values of vector i are of S
    if constexpr (E == 8) return (uint32_t) reinterpret_cast<const uint8_t*>(bits)[i + 1];
    else return ((uint32_t) reinterpret_cast<const uint8_t*>(bits)[(i + 2) >> 1] >> ((i & 1) * 4)) & 15u;
  };
  // the ids of S leave the vectors i0, i0 + THREADS, ...: few batches have any
  auto leave = [&](uint4 (&v)[HOLD], int i0) {
    uint32_t b[HOLD], any = 0;
#pragma unroll
    for (int j = 0; j < HOLD; ++j) any |= b[j] = i0 + j * THREADS < v1 ? listed(i0 + j * THREADS) : 0u;
    if (any) {
#pragma unroll
      for (int j = 0; j < HOLD; ++j) drop(v[j], b[j], T());
    }
  };
  leave(w, v0 + tid);
  if (single >= 0) {
    const int b = 8 + single - head;
    if (bits[b >> 5] >> (b & 31) & 1u) one = neg_inf();
  }

  // largest logit outside S and the sum about it, of a thread, then of a warp
  float m = neg_inf();
  double s = 0.0;
  if constexpr (SCAN) {
    bool bad = false;
    auto rise = [&](float v) {
      if (!(v < pos_inf())) bad = true;
      if (v > m) {
        s *= (double)ex2((m - v) * p.scale);  // m = -inf: 0
        m = v;
      }
    };
    auto take = [&](const uint4 (&w)[HOLD]) {
      typename X::Top top = X::top(w[0]);
#pragma unroll
      for (int j = 1; j < HOLD; ++j) top = X::larger(top, X::top(w[j]));
      rise(X::value(top));
      if (bad || !(m > neg_inf())) return;
      const u64 nm2 = pk2(-m, -m), sc2 = pk2(p.scale, p.scale);
      u64 s2 = 0;
#pragma unroll
      for (int j = 0; j < HOLD; ++j) {
        float f[E];
        X::unpack(w[j], f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          float d0, d1;
          up2(mul2(add2(pk2(f[e], f[e + 1]), nm2), sc2), d0, d1);
          s2 = add2(s2, pk2(ex2(d0), ex2(d1)));
        }
      }
      float lo, hi;
      up2(s2, lo, hi);
      s += (double)lo + (double)hi;
    };
    take(w);
    for (int i0 = v0 + tid + HOLD * THREADS; i0 < v1; i0 += HOLD * THREADS) {
      uint4 v[HOLD];
#pragma unroll
      for (int j = 0; j < HOLD; ++j) {
        const int i = i0 + j * THREADS;
        v[j] = i < v1 ? body[i] : make_uint4(X::FILL, X::FILL, X::FILL, X::FILL);
      }
      leave(v, i0);
      take(v);
    }
    if (single >= 0) {
      rise(one);
      if (!bad && m > neg_inf()) s += (double)ex2((one - m) * p.scale);
    }
    const float most = warp_max(bad ? neg_inf() : m);
    if (m > neg_inf() && !bad) s *= (double)ex2((m - most) * p.scale);
    if (bad) s = __longlong_as_double(0x7ff8000000000000LL);
    s = warp_sum(s);
    if (lane == 0) {
      sh.m[warp] = most;
      sh.s[warp] = s;
    }
  }

  // What needs no sum, by the first warp: the teacher's probabilities, and the terms
  // of S about its largest logit x_s.
  constexpr double NAN_D = 0.0 / 0.0;
  // The teacher's are left divided by `whole` until one division serves the row.
  double pj[SLOTS], ej[SLOTS], mass = 0.0, rest = 0.0, in = 0.0, cross = 0.0, whole = 1.0;
  float x_s = neg_inf();
  bool empty = false, odd = false, bad_s = false;
  if (warp == 0) {
    bool any = false;
    float lp_top = neg_inf();
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      any |= id[k] >= 0;
      if (id[k] >= 0) {
        odd |= !(lp[k] < pos_inf());
        bad_s |= !(xs[k] < pos_inf());
      }
      lp_top = fmaxf(lp_top, lp[k]);
      x_s = fmaxf(x_s, xs[k]);
    }
    any = __any_sync(FULL, any);
    odd = __any_sync(FULL, odd);
    bad_s = __any_sync(FULL, bad_s);
    lp_top = warp_max(lp_top);
    x_s = warp_max(x_s);
    empty = !any || (!p.tail && lp_top == neg_inf() && !odd);
    const double shift = p.tail || odd || empty ? 0.0 : (double)lp_top, about = x_s > neg_inf() && !bad_s ? (double)x_s : 0.0;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      pj[k] = ej[k] = 0.0;
      if (id[k] >= 0) {
        pj[k] = exp((double)lp[k] - shift);
        ej[k] = exp(((double)xs[k] - about) * p.inv_t);
        if (lead[k]) in += ej[k];
      }
      mass += pj[k];
    }
    mass = warp_sum(mass);
    in = warp_sum(in);
    if (p.tail) {
      rest = 1.0 - mass;
      if (rest < LEAST_REST) rest = 0.0;
    } else if (!empty && !odd) {
      whole = mass;
      mass = 1.0;
    }
    if (SCAN && p.loss) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (pj[k] > 0.0) cross += pj[k] * (((double)lp[k] - shift) - ((double)xs[k] - about) * p.inv_t);
      cross = warp_sum(cross);
    }
  }
  sync();

  // the warps' sums joined, then the CTAs'
  float m_all = neg_inf();
  double s_all = 0.0;
  auto join = [&](float m, double s) {  // of the lanes
    m_all = warp_max(m);
    if (m > neg_inf()) s *= (double)ex2((m - m_all) * p.scale);
    s_all = warp_sum(s);
  };
  if constexpr (SCAN) {
    if (WARPS == 1) {
      m_all = sh.m[0];
      s_all = sh.s[0];
    } else if (warp == 0) {
      join(lane < WARPS ? sh.m[lane] : neg_inf(), lane < WARPS ? sh.s[lane] : 0.0);
    }
    if (cs > 1) {
      if (tid == 0) {
        sh.cta_m = m_all;
        sh.cta_s = s_all;
      }
      cluster.sync();
      if (warp == 0) {
        const Shared<WARPS>* other = cluster.map_shared_rank(&sh, lane % cs);
        join(lane < cs ? other->cta_m : neg_inf(), lane < cs ? other->cta_s : 0.0);
      }
      cluster.sync();  // this CTA's have been read
    }
  }

  // the row's
  double q_scale = 0.0, own_scale = 0.0;
  if (warp == 0) {
    double sum_rest;
    float m_rest;
    if constexpr (SCAN) {
      m_rest = m_all;
      sum_rest = s_all;
    } else {
      const double2 st = p.stats[row];
      m_rest = (float)st.x;
      sum_rest = st.y;
    }
    const bool bad = bad_s || !(sum_rest < (double)pos_inf());
    const bool some = m_rest > neg_inf(), none = !bad && !some && !(x_s > neg_inf());
    // both sums about the larger of m_rest and x_s
    const double apart = some && x_s > neg_inf() ? ((double)m_rest - (double)x_s) * p.inv_t : 0.0, shrink = exp(-fabs(apart));
    const double in_part = apart > 0.0 ? in * shrink : in, rest_part = some ? (apart < 0.0 ? sum_rest * shrink : sum_rest) : 0.0;
    const double all = in_part + rest_part;
    // one division for three: all >= 1 or there is nothing, sum_rest >= 1 or there is no rest, whole in [1, n]
    const double sum_1 = some && !bad ? sum_rest : 1.0, inv = 1.0 / (all * sum_1 * whole), over_all = inv * (sum_1 * whole);
    const double over_rest = inv * (all * whole), over_whole = p.tail ? 1.0 : inv * (all * sum_1);
    if constexpr (GRAD) {
      const double g = (p.g_loss ? (double)p.g_loss[row] : 1.0) * p.inv_t;
      // e = 2^((x - m_rest) scale): q = e rest_part / (sum_rest all), q / q_t = e / sum_rest
      double c = 0.0;
      if (!empty && !none && some) c = g * (mass * (rest_part * over_all) - rest * (in_part * over_all)) * over_rest;
      if (!empty && (bad || odd)) c = NAN_D;
      q_scale = empty || none ? 0.0 : g * (mass + rest) * over_all * (apart > 0.0 ? shrink : 1.0);
      own_scale = empty || none ? 0.0 : g * over_whole;
      if (bad || odd) q_scale = empty ? 0.0 : NAN_D;
      if (lane == 0) {
        sh.row_m = some && !empty && !bad ? m_rest : 0.0f;
        sh.row_c = (float)c;
      }
    }
    if constexpr (GRAD && THREADS > 32) sync();  // the others go on with the gradient
    if (SCAN && p.loss && rank == 0) {
      // log sum about x_s: log q_j = (x_j - x_s) / T - log_s, and log p_j = l_j - shift - log whole; a lane each
      // takes the logarithms of all / whole and of what the tail needs
      const double logs = log(lane == 0 ? all * over_whole : rest * over_rest), log_tail = __shfl_sync(FULL, logs, 1);
      const double log_s = none ? 0.0 : logs + (apart > 0.0 ? apart : 0.0);
      double loss = cross * over_whole + mass * log_s;
      if (!(x_s > neg_inf()) && mass > 0.0) loss = (double)pos_inf();
      if (rest > 0.0) loss += some ? rest * (log_tail + logs - fmin(apart, 0.0)) : (double)pos_inf();
      if (lane == 0) p.loss[row] = empty ? 0.0f : bad || odd ? (float)NAN_D : (float)loss;
    }
    if (SCAN && lane == 0 && rank == 0 && p.stats) p.stats[row] = make_double2((double)m_rest, sum_rest);
    if (SCAN && p.status) {
      wrong = __any_sync(FULL, wrong);
      uint32_t st = wrong ? MTR_ROW_BAD_ID : 0u;
      if (!empty) st |= bad || odd ? MTR_ROW_NONFINITE : none ? MTR_ROW_ALL_MASKED : 0u;
      if (lane == 0 && rank == 0) p.status[row] = st;
    }
    if constexpr (GRAD) {
      if (sh.dup) {  // equal ids: the leading one gets all of their probability
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
          const int j = lane + 32 * k;
          if (j < p.n) {
            sh.id[j] = id[k];
            sh.p[j] = pj[k];
          }
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < SLOTS; ++k)
          if (lead[k]) {
            double sum = 0.0;
            for (int j = 0; j < p.n; ++j)
              if (sh.id[j] == id[k]) sum += sh.p[j];
            pj[k] = sum;
          }
      }
      __syncwarp();
    }
  } else if constexpr (GRAD) {
    sync();
  }
  if constexpr (!GRAD) return;
  const float rm = sh.row_m, rc = sh.row_c;
  T* g = (T*)p.grad + row * p.grad_stride;
  const u64 nm2 = pk2(-rm, -rm), sc2 = pk2(p.scale, p.scale), c2 = pk2(rc, rc);
  // a row of gradient 0 may hold NaN, which has no gradient then
  const bool zero = rc == 0.0f;
  auto store = [&](int i, const uint4& packed, const float (&f)[E]) {
    if (p.alike) {
      reinterpret_cast<uint4*>(g + head)[i] = packed;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) g[head + i * E + e] = from_f<T>(f[e]);
    }
  };
  auto put = [&](int i, const uint4& v) {
    float f[E];
    X::unpack(v, f);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float d0, d1;
      up2(mul2(add2(pk2(f[e], f[e + 1]), nm2), sc2), d0, d1);
      up2(mul2(pk2(ex2(d0), ex2(d1)), c2), f[e], f[e + 1]);
    }
    store(i, pack<T>(f), f);
  };
  if (zero) {
    const float f[E] = {};
    for (int i = v0 + tid; i < v1; i += THREADS) store(i, make_uint4(0u, 0u, 0u, 0u), f);
  } else {
#pragma unroll
    for (int j = 0; j < HOLD; ++j)
      if (v0 + tid + j * THREADS < v1) put(v0 + tid + j * THREADS, w[j]);
    for (int i0 = v0 + tid + HOLD * THREADS; i0 < v1; i0 += HOLD * THREADS) {
#pragma unroll
      for (int j = 0; j < HOLD; ++j)
        if (i0 + j * THREADS < v1) w[j] = body[i0 + j * THREADS];
#pragma unroll
      for (int j = 0; j < HOLD; ++j)
        if (i0 + j * THREADS < v1) put(i0 + j * THREADS, w[j]);
    }
  }
  if (single >= 0) g[single] = from_f<T>(zero ? 0.0f : ex2((one - rm) * p.scale) * rc);
  sync();  // the entries of S are written over, by the CTA that wrote there
  const int from = rank == 0 ? 0 : head + v0 * E, to = head + v1 * E, last = rank == 0 ? V - behind : V;
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
      if (lead[k] && ((id[k] >= from && id[k] < to) || id[k] >= last)) g[id[k]] = from_f<T>(empty ? 0.0f : (float)(ej[k] * q_scale - pj[k] * own_scale));
  }
}

static int esize(int32_t dtype) { return dtype == MTR_DTYPE_F32 ? 4 : 2; }

// vectors of a thread in registers: more warps pay more than longer runs (8192 x 4096 bf16: 16 vectors 51.1 us, 4 35.1)
constexpr int HELD = 4;
template <typename T, int THREADS, int CTAS, int SLOTS>
static cudaError_t launch_of(const Params& p, int64_t rows, bool scan, cudaStream_t s) {
  const int dyn = (p.vocab + 8 + 31) / 32 * 4;  // at most 16.4 KB
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(rows * p.cluster), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = (size_t)dyn;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = launch_attrs(attr, p.cluster, true);
  cfg.attrs = attr;
  if (!p.grad) return cudaLaunchKernelEx(&cfg, distill_kernel<T, THREADS, HELD, CTAS, SLOTS, true, false>, p);
  return scan ? cudaLaunchKernelEx(&cfg, distill_kernel<T, THREADS, HELD, CTAS, SLOTS, true, true>, p)
              : cudaLaunchKernelEx(&cfg, distill_kernel<T, THREADS, HELD, CTAS, SLOTS, false, true>, p);
}
template <typename T, int THREADS, int CTAS>
static cudaError_t launch(const Params& p, int64_t rows, bool scan, cudaStream_t s) {
  return p.n <= 32 ? launch_of<T, THREADS, CTAS, 1>(p, rows, scan, s) : launch_of<T, THREADS, CTAS, MTR_MAX_TEACHER_IDS / 32>(p, rows, scan, s);
}

// Threads of a row, by how many rows there are to fill the device's 16 warps an SM
// and how long they are; CTAs share a row only where they give idle SMs work, and not
// where the gradient alone is asked for (4 x 131072 fp32, 32 ids: 16.3 us, the loss before
// it 6.1, both from one reading in clusters 8.1).
// Loss and gradient together, with 20 ids (us, 32 / 128 / 256 threads, 148 SMs):
//   8192 x 1000 bf16    14.9 / 39.5 / 64.2     enough rows: a warp each
//   8192 x 4096 bf16    34.4 / 47.3 / 75.4
//   8192 x 8192 bf16    63.0 / 71.7 / 85.0
//   3000 x 4096 fp32    23.3 / 24.2 / 31.2
//   1000 x 4096 bf16    10.2 /  7.9 / 12.2     few rows: more warps each
//   2000 x 16384 bf16   44.3 / 32.5 / 38.0     long rows: 128 threads, then 256
//   3000 x 32768 bf16    108 / 91.3 / 85.1
//   300 x 16384 fp32    38.6 / 15.4 / 12.3
//   2000 x 65533 bf16    181 /  135 /  124, 512 threads 125
template <typename T>
static cudaError_t launch(Params p, int64_t rows, bool scan, cudaStream_t s) {
  const int64_t vecs = (int64_t)p.vocab * (int)sizeof(T) / 16, sms = device_sms();
  int threads = vecs > 2560 ? 256 : vecs > 1024 ? 128 : 32;
  while (threads < MOST_THREADS && rows * threads < 16 * 32 * sms && vecs >= 8 * threads) threads *= threads == 32 ? 4 : 2;
  p.cluster = 1;
  while (threads == MOST_THREADS && p.cluster < 8 && scan && vecs >= 2ll * HELD * MOST_THREADS * p.cluster && rows * p.cluster * 2 <= sms)
    p.cluster *= 2;
  switch (threads) {
    case 32: return launch<T, 32, 28>(p, rows, scan, s);
    case 128: return launch<T, 128, 7>(p, rows, scan, s);
    case 256: return launch<T, 256, 4>(p, rows, scan, s);
    default: return launch<T, 512, 2>(p, rows, scan, s);
  }
}

}  // namespace ds
}  // namespace mtr

// ---------------------------------------------------------------- C ABI
using namespace mtr::ds;

int mtr_distill_validate(const MtrDistillArgs* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrDistillArgs)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->rows > MTR_MAX_SCORE_ROWS || a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
  if (a->n < 1 || a->n > MTR_MAX_TEACHER_IDS) return MTR_ERR_BAD_PARAM;
  if (a->logits_dtype < MTR_DTYPE_F32 || a->logits_dtype > MTR_DTYPE_F16) return MTR_ERR_BAD_PARAM;
  if (a->ids_dtype != MTR_IDS_I64 && a->ids_dtype != MTR_IDS_I32) return MTR_ERR_BAD_PARAM;
  if (a->tail != 0 && a->tail != 1) return MTR_ERR_BAD_PARAM;
  if (!(a->temperature > 0.0) || !(a->temperature <= (double)MTR_MAX_TEMPERATURE) || !((float)(1.4426950408889634 / a->temperature) < INFINITY))
    return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  if (!a->logits || !a->teacher_ids || !a->teacher_logprobs) return MTR_ERR_NULL_ARG;
  if (!a->out_loss && !(a->grad_logits && a->stats)) return MTR_ERR_NULL_ARG;
  if (a->logits_row_stride < a->vocab || a->ids_row_stride < 0 || a->logprobs_row_stride < 0) return MTR_ERR_BAD_SHAPE;
  if (a->grad_logits && a->grad_row_stride < a->vocab) return MTR_ERR_BAD_SHAPE;
  const int64_t es = esize(a->logits_dtype);
  if ((uintptr_t)a->logits % es || (uintptr_t)a->teacher_ids % (a->ids_dtype == MTR_IDS_I64 ? 8 : 4) ||
      (uintptr_t)a->teacher_logprobs % 4 || (uintptr_t)a->out_loss % 4 || (uintptr_t)a->stats % 16 ||
      (uintptr_t)a->g_loss % 4 || (uintptr_t)a->grad_logits % es || (uintptr_t)a->out_status % 4)
    return MTR_ERR_ALIGNMENT;
  const int64_t ids_size = a->ids_dtype == MTR_IDS_I64 ? 8 : 4;
  if (a->grad_logits) {  // a CTA's gradient row must be nothing that another CTA has yet to read
    const mtr::Bytes grad = mtr::bytes_of(a->grad_logits, a->rows, a->grad_row_stride, a->vocab, es);
    auto hits = [&](const void* at, int64_t stride, int64_t cols, int64_t size) {  // stride 0: one row for all
      return at && overlap(grad, mtr::bytes_of(at, stride ? a->rows : 1, stride ? stride : cols, cols, size));
    };
    if (hits(a->logits, a->logits_row_stride, a->vocab, es) || hits(a->teacher_ids, a->ids_row_stride, a->n, ids_size) ||
        hits(a->teacher_logprobs, a->logprobs_row_stride, a->n, 4) || hits(a->g_loss, 1, 1, 4) ||
        mtr::meets(a->stats, 16ll * a->rows, a->grad_logits, a->rows, a->grad_row_stride * es, 1, 0, a->vocab * es))
      return MTR_ERR_BAD_PARAM;
  }
  if (a->out_loss) {  // and so its loss, statistics and status
    const struct {
      const void* at;
      int64_t size;
    } outs[3] = {{a->out_loss, 4}, {a->stats, 16}, {a->out_status, 4}};
    for (const auto& o : outs) {
      auto hits = [&](const void* at, int64_t stride, int64_t cols, int64_t size) {
        return mtr::meets(o.at, o.size * a->rows, at, a->rows, stride * size, 1, 0, cols * size);
      };
      if (o.at && (hits(a->logits, a->logits_row_stride, a->vocab, es) || hits(a->teacher_ids, a->ids_row_stride, a->n, ids_size) ||
                   hits(a->teacher_logprobs, a->logprobs_row_stride, a->n, 4) || hits(a->g_loss, 1, 1, 4) ||
                   hits(a->grad_logits, a->grad_row_stride, a->vocab, es)))
        return MTR_ERR_BAD_PARAM;
    }
  }
  return MTR_OK;
}

int mtr_distill_launch(const MtrDistillArgs* a, void* stream) {
  const int v = mtr_distill_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  Params p;
  p.logits = a->logits;
  p.stride = a->logits_row_stride;
  p.ids = a->teacher_ids;
  p.ids_stride = a->ids_row_stride;
  p.lps = a->teacher_logprobs;
  p.lps_stride = a->logprobs_row_stride;
  p.ids32 = a->ids_dtype == MTR_IDS_I32;
  p.vocab = a->vocab;
  p.n = a->n;
  p.tail = a->tail;
  const int64_t es = esize(a->logits_dtype);
  p.alike = (((uintptr_t)a->logits ^ (uintptr_t)a->grad_logits) & 15u) == 0 && ((a->logits_row_stride - a->grad_row_stride) * es) % 16 == 0;
  p.scale = (float)(1.4426950408889634 / a->temperature);
  p.inv_t = 1.0 / a->temperature;
  p.loss = a->out_loss;
  p.stats = (double2*)a->stats;
  p.g_loss = a->g_loss;
  p.grad = a->grad_logits;
  p.grad_stride = a->grad_row_stride;
  p.status = a->out_status;
  cudaStream_t s = (cudaStream_t)stream;
  const bool scan = a->out_loss != nullptr;
  cudaError_t e;
  switch (a->logits_dtype) {
    case MTR_DTYPE_F32: e = launch<float>(p, a->rows, scan, s); break;
    case MTR_DTYPE_BF16: e = launch<__nv_bfloat16>(p, a->rows, scan, s); break;
    default: e = launch<__half>(p, a->rows, scan, s); break;
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}
