// mtr_verify.cu -- drafted tokens accepted or replaced under the target's
// distribution (speculative sampling).
//
// With p_j the target's softmax(logits / T) of position j, q_j the draft's (or all
// mass on the drafted token t_j where no draft logits are given) and u the caller's
// uniforms, draft j is accepted while u_j q_j(t_j) < p_j(t_j).  At the first that is
// not, j = a, a token is drawn from w = max(p_a - q_a, 0): the smallest id v with
// sum_{i <= v} w_i > u_K sum w; behind the last draft from w = p.
//
// Tokens are decisions, so each is what real arithmetic decides (but for borders
// nearer than double's rounding):
//   rows_kernel   reads every row that may count once and keeps its largest
//                 logit and the sum of e^((x - max) / T) about it, fp32 terms, within
//                 E = 2^-15 relative (below).  HBM bounds it.
//   pick_kernel   decides the drafts in turn: log u + log q - log p in double from
//                 these sums, clear when it is further than 2 E from 0; else (about
//                 once in 10^4 drafts) both sums are formed again in double.  Then it
//                 draws from the one position that counts, all in double.  It reads
//                 short rows itself, and one launch does it all.
// rows_kernel reads 571 MB (128 x 17 rows of 131072 bf16) in 102 us, 5.6 TB/s, and the draw
// of 128 sequences takes 62 behind it.  Neither its instructions (69 for an id's two
// terms, 0.56 a clock and scheduler) nor the double rate (41 %) fill that time: one CTA of
// 16 warps an SM at 126 registers waits for its own chains.  Rows that do not lie alike
// about 16 bytes (odd vocabularies with a draft's logits) are drawn from a value an
// access: 182 us at V = 131071 where 131072 takes 167, 59.5 at 64 x 5, V = 65533 fp16 where
// 65536 takes 54.7.
// The bound E: ex2.approx is within 2^-22, its argument within 3 2^-24 |d| of d (over
// all moves together, whose distances add up to d), and the mean of |d| under the
// softmax is at most log V < 12; a thread adds at most 16 pairs in fp32 before double
// takes over, and its sum moves to a larger maximum at most 40 times (MOVES), within
// 2^-22 each: 2.4e-7 + 2.2e-6 + 1e-6 + 9.6e-6 < 2^-15 = 3.1e-5.
#include "mtr_vec.cuh"

namespace mtr {
namespace vf {

constexpr double BORDER = 0x1p-14;  // 2 E: two sums
// (logit - largest) / T of an id that has no probability, 2^-1000 of the largest or less:
// a mask of the type's lowest value forbids a token whatever the uniform, as -inf does
constexpr double FAR_LOG = -1000.0 * 0.69314718055994530942;

struct Part {  // of a run of a row
  float m;
  int32_t id;  // the first id of the largest logit (greedy only)
  double s;    // NaN: a NaN or +inf
};

struct Params {
  const void* target;
  int64_t t_batch, t_pos;
  const void* draft;  // NULL: one-hot
  int64_t d_batch, d_pos;
  const void* ids;
  int64_t ids_stride;
  int32_t ids32;
  const float* uniforms;
  int64_t u_stride;
  int32_t batch, drafts, vocab;
  int32_t runs;     // of a row, a CTA each
  int32_t run;      // vectors of a run
  int32_t greedy;
  int32_t cluster;
  float t_scale, d_scale;    // log2(e) / T
  double t_inv, d_inv;       // 1 / T
  int64_t pad_id;
  Part* parts;               // [batch (2 drafts + 1)] rows of runs: the targets, then the drafts
  int64_t* tokens;
  int32_t* accepted;
  float* logprobs;
  uint32_t* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double nan_d() { return __longlong_as_double(0x7ff8000000000000LL); }
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
__device__ __forceinline__ int64_t draft_id(const Params& p, int64_t b, int j) {
  const int64_t at = b * p.ids_stride + j;
  return p.ids32 ? (int64_t)((const int32_t*)p.ids)[at] : ((const int64_t*)p.ids)[at];
}

constexpr int HOLD = 4;  // vectors of a thread's tile

// Moves of a sum: an unsplit fp32 row is 32 tiles of 256 threads, 31 of them behind the
// first; the single logit, the warp's maximum, 7 of the 8 warps in join.  (r runs have 32 / r
// tiles and r - 1 more joins: fewer.)
constexpr int MOVES = MTR_MAX_VOCAB / 4 / (256 * HOLD) - 1 + 1 + 1 + 7;
static_assert((1 + MOVES) * 0x1p-22 + (3 * 12 + 16) * 0x1p-24 < BORDER / 2, "the fp32 sums' error bound");

// A row's parts joined; every lane the same.
__device__ __forceinline__ Part join(const Part* parts, int runs, float scale) {
  Part r = parts[0];
  for (int i = 1; i < runs; ++i) {
    const Part q = parts[i];
    const float m = fmaxf(r.m, q.m);
    if (q.m > r.m || (q.m == r.m && q.id < r.id)) r.id = q.id;
    r.s = (r.m > neg_inf() ? r.s * (double)ex2((r.m - m) * scale) : r.s) + (q.m > neg_inf() ? q.s * (double)ex2((q.m - m) * scale) : q.s);
    r.m = m;
  }
  return r;
}

// A warp's part of the vectors [v0, v1) of a row, which THREADS threads take 32 by 32
// (tid of them); `singles`: with the single logits before the first 16-byte boundary
// and behind the last.  The first tile is asked for before `counts` says whether the
// row does; nothing is returned where it does not.
template <typename T, int THREADS, bool GREEDY, typename F>
__device__ __forceinline__ bool warp_run(const T* x, int V, int v0, int v1, bool singles, float scale, int tid, F counts, Part& part) {
  typedef Vec<T> X;
  constexpr int E = X::E;
  const int off = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int head = min(off ? E - off : 0, V), vecs = (V - head) / E, behind = V - head - vecs * E;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  v0 = min(v0, vecs);
  v1 = min(v1, vecs);
  uint4 w[HOLD];
  auto ask = [&](int i0) {
#pragma unroll
    for (int k = 0; k < HOLD; ++k) {
      const int i = i0 + k * THREADS;
      w[k] = i < v1 ? body[i] : make_uint4(X::FILL, X::FILL, X::FILL, X::FILL);
    }
  };
  ask(v0 + tid);
  if (!counts()) return false;

  float m = neg_inf();
  double s = 0.0;
  bool bad = false;
  int at = 0x7fffffff;
  auto rise = [&](float v) {
    if (!(v < pos_inf())) bad = true;
    if (v > m) {
      s *= (double)ex2((m - v) * scale);  // m = -inf: 0
      m = v;
    }
  };
  const int single = !singles ? -1 : tid < head ? tid : tid >= 16 && tid < 16 + behind ? V - behind + tid - 16 : -1;
  const float one = single >= 0 ? to_f(x[single]) : neg_inf();
  for (int i0 = v0 + tid; i0 < v1; i0 += HOLD * THREADS) {
    if (i0 != v0 + tid) ask(i0);
    if constexpr (GREEDY) {
      float best = m;
#pragma unroll
      for (int k = 0; k < HOLD; ++k) {
        const float v = X::value(X::top(w[k]));
        if (v > best) {
          best = v;
          at = i0 + k * THREADS;
        }
      }
    }
    typename X::Top top = X::top(w[0]);
#pragma unroll
    for (int k = 1; k < HOLD; ++k) top = X::larger(top, X::top(w[k]));
    rise(X::value(top));
    if (bad || !(m > neg_inf())) continue;
    const u64 nm2 = pk2(-m, -m), sc2 = pk2(scale, scale);
    u64 s2 = 0;
#pragma unroll
    for (int k = 0; k < HOLD; ++k) {
      float f[E];
      X::unpack(w[k], f);
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
  }
  const float vector_m = m;  // what `at` holds
  if (single >= 0) {
    rise(one);
    if (!bad && m > neg_inf()) s += (double)ex2((one - m) * scale);
  }
  part.m = warp_max(bad ? neg_inf() : m);
  if (!bad && m > neg_inf()) s *= (double)ex2((m - part.m) * scale);
  if (bad) s = nan_d();
  part.s = warp_sum(s);
  part.id = 0x7fffffff;
  if constexpr (GREEDY) {
    // the first id whose logit is the largest
    int id = single >= 0 && one == part.m ? single : 0x7fffffff;
    if (vector_m == part.m && at < vecs) {
      float f[E];
      X::unpack(body[at], f);
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (f[e] == part.m) id = min(id, head + at * E + e);
    }
    part.id = __reduce_min_sync(FULL, id);
  }
  return true;
}
// a position counts only behind drafts that are ids: whether the first n are
__device__ __forceinline__ bool drafts_are_ids(const Params& p, int64_t b, int n) {
  const int lane = threadIdx.x & 31;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int64_t id = i0 + lane < n ? draft_id(p, b, i0 + lane) : 0;
    if (__any_sync(FULL, id < 0 || id >= p.vocab)) return false;
  }
  return true;
}

// One run of one row: its largest logit and the sum about it.
template <typename T, int THREADS, bool GREEDY>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Params p) {
  constexpr int WARPS = THREADS / 32;
  __shared__ Part parts[WARPS];
  const int tid = threadIdx.x, K = p.drafts;
  const int64_t row = blockIdx.x, targets = (int64_t)p.batch * (K + 1);
  const bool draft = row >= targets;
  const int64_t b = draft ? (row - targets) / K : row / (K + 1);
  const int j = (int)(draft ? (row - targets) % K : row % (K + 1));
  wait_prior_grid();
  const T* x = draft ? (const T*)p.draft + b * p.d_batch + j * p.d_pos : (const T*)p.target + b * p.t_batch + j * p.t_pos;
  const float scale = draft ? p.d_scale : p.t_scale;
  const int v0 = (int)blockIdx.y * p.run;
  Part part;
  if (!warp_run<T, THREADS, GREEDY>(x, p.vocab, v0, blockIdx.y == gridDim.y - 1 ? p.vocab : v0 + p.run, blockIdx.y == 0, scale, tid,
                                    [&] { return drafts_are_ids(p, b, draft ? j + 1 : j); }, part))
    return;
  if ((tid & 31) == 0) parts[tid >> 5] = part;
  __syncthreads();
  if (tid == 0) p.parts[row * p.runs + blockIdx.y] = join(parts, WARPS, scale);
}

// Threads of a CTA that draws.  Where it has few ids (kept) a thread's terms stay in
// registers.  640, 768 and 1024 threads for the others: 172, 177 and 169 us where 512
// take 167 (128 x 8, V = 131072 bf16).
constexpr int FEW = 512, MANY = 512;
constexpr int KEPT = 8;  // ids of a thread whose terms stay in registers
constexpr int NEAR = 64; // ids of a warp next to the border between p > q and p < q
// A sum of weights by term() is above this where an id has weight: n ids without any add
// at most n 2^-1000.  A CTA's share above NOTHING has a warp's piece above LITTLE.
// Sums by term_or_0 are 0 there.
constexpr double NOTHING = 0x1p-900, LITTLE = 0x1p-910;

// e^((x - m) / T) in double, x <= m finite or -inf: with c = 64 log2(e) / T,
// z = (x - m) c = k + r, k whole and |r| <= 1/2, the value is 2^(k / 64) 2^(r / 64): a
// table of 64 powers, an exponent, and the series of e^(r ln2 / 64) to r^4 (within
// 4e-14).  Ten double operations, which bound the kernel (64 a clock and SM); the
// library's exp has about twice as many.  z is held to -64000, where the value is
// 2^-1000 (one unsigned minimum of high words): far and masked ids then add next to
// nothing to a sum of at least 1, and term_or_0 gives them nothing.
struct Exp {
  double m, c;
};
constexpr uint32_t FAR = 0xc0ef4000u;  // the high word of -64000.0
__device__ __forceinline__ Exp exp_of(float m, double inv) { return Exp{(double)m, 64.0 * 1.4426950408889634074 * inv}; }
__device__ __forceinline__ double term(float x, const Exp& e, const double* powers, bool& far) {
  constexpr double STEP = 0.69314718055994530942 / 64.0, MAGIC = 6755399441055744.0;  // 1.5 2^52
  const double d = ((double)x - e.m) * e.c;
  far = (uint32_t)__double2hiint(d) >= FAR;
  const double z = __hiloint2double((int)min((uint32_t)__double2hiint(d), FAR), __double2loint(d)), y = z + MAGIC, r = z - (y - MAGIC);
  const int k = __double2loint(y);
  const double v = fma(fma(fma(fma(STEP * STEP * STEP * STEP / 24.0, r, STEP * STEP * STEP / 6.0), r, STEP * STEP / 2.0), r, STEP), r, 1.0) *
                   powers[k & 63];
  return __hiloint2double(__double2hiint(v) + ((k >> 6) << 20), __double2loint(v));
}
__device__ __forceinline__ double term(float x, const Exp& e, const double* powers) {
  bool far;
  return term(x, e, powers, far);
}
__device__ __forceinline__ double term_or_0(float x, const Exp& e, const double* powers) {
  bool far;
  const double v = term(x, e, powers, far);
  return far ? 0.0 : v;
}

struct Sums {
  double t, d;
  double over;  // ids next to the border that a list had no room for
};

template <int PICK_WARPS>
struct PickShared {
  double powers[64];
  double warp_t[PICK_WARPS], warp_d[PICK_WARPS], warp_over[PICK_WARPS];
  Sums cta;                      // read by the cluster's other CTAs
  double weight;                 // likewise
  double piece[PICK_WARPS];
  int stop, unclear, token;
  int32_t near[PICK_WARPS][NEAR];
  Part parts[2 * MTR_MAX_DRAFTS + 1];  // where the rows are read here
};

template <typename T, bool kept>
__global__ void __launch_bounds__(kept ? FEW : MANY, 1) pick_kernel(const Params p) {
  constexpr int PICK = kept ? FEW : MANY, PICK_WARPS = PICK / 32;
  constexpr int PIECE = (MTR_MAX_VOCAB + PICK_WARPS - 1) / PICK_WARPS;         // a warp's ids at most
  constexpr int MOST = kept ? KEPT : (PIECE + PICK - 1) / PICK;               // and a thread's in the last search
  __shared__ PickShared<PICK_WARPS> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = p.cluster, rank = cs > 1 ? (int)(blockIdx.x % cs) : 0;
  const int64_t b = cs > 1 ? blockIdx.x / cs : blockIdx.x;
  const int K = p.drafts, V = p.vocab;
  wait_prior_grid();

  const Part* t_parts = kept && !p.parts ? sh.parts : p.parts + b * (K + 1) * p.runs;
  const Part* d_parts = kept && !p.parts ? sh.parts + K + 1 : p.parts + ((int64_t)p.batch * (K + 1) + b * K) * p.runs;
  auto t_row = [&](int j) { return (const T*)p.target + b * p.t_batch + j * p.t_pos; };
  auto d_row = [&](int j) { return (const T*)p.draft + b * p.d_batch + j * p.d_pos; };
  auto uniform = [&](int j, uint32_t& st) {
    float u = p.uniforms[b * p.u_stride + j];
    if (!(u >= 0.0f)) {
      u = 0.0f;
      st |= MTR_ROW_BAD_UNIFORM;
    } else if (u >= 1.0f) {
      u = 0x1.fffffep-1f;
      st |= MTR_ROW_BAD_UNIFORM;
    }
    return (double)u;
  };
  if constexpr (kept) {
    if (!p.parts) {  // short rows: a warp each, the targets, then the drafts
      const int rows = p.draft ? 2 * K + 1 : K + 1;
      for (int r = warp; r < rows; r += PICK_WARPS) {
        const bool of_draft = r > K;
        const int j = of_draft ? r - K - 1 : r;
        const T* x = of_draft ? d_row(j) : t_row(j);
        const float scale = of_draft ? p.d_scale : p.t_scale;
        auto counts = [&] { return drafts_are_ids(p, b, of_draft ? j + 1 : j); };
        Part part;
        const bool some = p.greedy ? warp_run<T, 32, true>(x, V, 0, V, true, scale, lane, counts, part)
                                   : warp_run<T, 32, false>(x, V, 0, V, true, scale, lane, counts, part);
        if (some && lane == 0) sh.parts[r] = part;
      }
    }
  }
  if (tid < 64) sh.powers[tid] = exp2(tid / 64.0);
  __syncthreads();
  const double* powers = sh.powers;
  // this CTA's ids [c0, c1); kept: a thread has KEPT of them, one after another, at most
  const int share = (V + cs - 1) / cs, c0 = min(rank * share, V), c1 = min(c0 + share, V);
  // part `k` of [from, to) cut into n
  auto part_of = [](int from, int to, int n, int k, int& a, int& z) {
    const int each = (to - from + n - 1) / n;
    a = min(from + k * each, to);
    z = min(a + each, to);
  };
  // sums over the CTA, then over the cluster; the same in every thread
  auto total = [&](Sums s) {
    s.t = warp_sum(s.t);
    s.d = warp_sum(s.d);
    if (lane == 0) {
      sh.warp_t[warp] = s.t;
      sh.warp_d[warp] = s.d;
      sh.warp_over[warp] = s.over;
    }
    __syncthreads();
    s = Sums{0.0, 0.0, 0.0};
    for (int k = 0; k < PICK_WARPS; ++k) {
      s.t += sh.warp_t[k];
      s.d += sh.warp_d[k];
      s.over += sh.warp_over[k];
    }
    if (cs > 1) {
      if (tid == 0) sh.cta = s;
      cluster.sync();
      s = Sums{0.0, 0.0, 0.0};
      for (int k = 0; k < cs; ++k) {
        const Sums o = cluster.map_shared_rank(&sh, k)->cta;
        s.t += o.t;
        s.d += o.d;
        s.over += o.over;
      }
      cluster.sync();  // read before it is written again
    } else {
      __syncthreads();
    }
    return s;
  };
  // A warp's ids [a, z) of two rows (y may be missing): f(id, x, y);
  // the warp is in step, ids behind the end are z and their values -inf.  Rows that lie
  // alike about the 16-byte boundaries are read in vectors, the next ones under way
  // while these are summed; else every value is its own access.
  auto stream = [&](const T* x, const T* y, int a, int z, auto f) {
    constexpr int E = Vec<T>::E;
    auto singles = [&](int from, int to) {
      constexpr int U = 8;
      for (int v0 = from + lane; v0 - lane < to; v0 += 32 * U) {
        float xs[U], ys[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int v = v0 + 32 * i;
          xs[i] = v < to ? to_f(x[v]) : neg_inf();
          ys[i] = y && v < to ? to_f(y[v]) : neg_inf();
        }
#pragma unroll
        for (int i = 0; i < U; ++i) f(min(v0 + 32 * i, to), xs[i], ys[i]);
      }
    };
    if (y && (((uintptr_t)x ^ (uintptr_t)y) & 15u)) {
      singles(a, z);
      return;
    }
    const int off = (int)(((uintptr_t)(x + a) & 15u) / sizeof(T)), head = min(off ? E - off : 0, z - a), vecs = (z - a - head) / E;
    const uint4 *xv = reinterpret_cast<const uint4*>(x + a + head), *yv = reinterpret_cast<const uint4*>(y + a + head);
    const uint4 fill = make_uint4(Vec<T>::FILL, Vec<T>::FILL, Vec<T>::FILL, Vec<T>::FILL);
    uint4 nx = lane < vecs ? xv[lane] : fill, ny = y && lane < vecs ? yv[lane] : fill;
    singles(a, a + head);
    singles(a + head + vecs * E, z);
    for (int i = lane; i - lane < vecs; i += 32) {
      float xs[E], ys[E];
      Vec<T>::unpack(nx, xs);
      Vec<T>::unpack(ny, ys);
      nx = i + 32 < vecs ? xv[i + 32] : fill;
      ny = y && i + 32 < vecs ? yv[i + 32] : fill;
      const int v = i < vecs ? a + head + i * E : z;
#pragma unroll
      for (int e = 0; e < E; ++e) f(v + e, xs[e], ys[e]);
    }
  };
  // sums of e^((x - m) / T) over the whole row(s)
  auto exact_sums = [&](const T* t, const Exp& te, const T* d, const Exp& de) {
    int a, z;
    part_of(c0, c1, PICK_WARPS, warp, a, z);
    Sums s{0.0, 0.0, 0.0};
    if (d)
      stream(t, d, a, z, [&](int, float x, float y) {
        s.t += term(x, te, powers);
        s.d += term(y, de, powers);
      });
    else
      stream(t, d, a, z, [&](int, float x, float) { s.t += term(x, te, powers); });
    return total(s);
  };

  // The drafts in turn, 32 at a time: lane l decides draft first + l.
  uint32_t status = 0;
  int stop = 0;          // accepted so far
  bool open = true;
  while (open) {
    if (warp == 0) {
      const int j = stop + lane;
      int verdict = 2;  // 0 accepted, 1 refused (or no draft), 2 unclear
      uint32_t st = 0;
      const int64_t id = j < K ? draft_id(p, b, j) : -1;
      if (id < 0 || id >= V) {
        verdict = 1;
        if (id >= V) st |= MTR_ROW_BAD_ID;
      }
      // positions behind the first that is no draft have no parts
      const unsigned ends = __ballot_sync(FULL, verdict == 1);
      const int known = ends ? __ffs(ends) - 1 : 32;
      if (lane < known) {
        const Part t = join(t_parts + (int64_t)j * p.runs, p.runs, p.t_scale);
        const bool t_bad = !(t.s < (double)pos_inf()), t_none = !t_bad && !(t.m > neg_inf());
        if (t_bad || t_none) {
          verdict = 1;  // the draw reports it
        } else if (p.greedy) {
          verdict = t.id == (int)id ? 0 : 1;
        } else {
          const double z = ((double)to_f(t_row(j)[id]) - (double)t.m) * p.t_inv;
          const double u = uniform(j, st);
          bool q_zero = false, q_bad = false;
          double lq = 0.0;
          if (p.draft) {
            const Part d = join(d_parts + (int64_t)j * p.runs, p.runs, p.d_scale);
            if (!(d.s < (double)pos_inf())) {
              st |= MTR_ROW_NONFINITE;
              q_bad = true;
            } else if (!(d.m > neg_inf())) {
              st |= MTR_ROW_ALL_MASKED;
              q_bad = true;
            } else {
              const double z = ((double)to_f(d_row(j)[id]) - (double)d.m) * p.d_inv;
              q_zero = z <= FAR_LOG;
              lq = z - log(d.s);
            }
          }
          if (q_bad || z <= FAR_LOG) verdict = 1;
          else if (q_zero || u == 0.0) verdict = 0;
          else {
            const double far = log(u) + lq - (z - log(t.s));
            verdict = far < -BORDER ? 0 : far > BORDER ? 1 : 2;
          }
        }
      }
      const unsigned not_yes = __ballot_sync(FULL, verdict != 0);
      const int n = not_yes ? __ffs(not_yes) - 1 : 32;
      // the bits of the positions that were looked at in earnest
      status |= __reduce_or_sync(FULL, lane <= n ? st : 0u);
      const int what = n < 32 ? __shfl_sync(FULL, verdict, n) : 3;
      if (lane == 0) {
        sh.stop = stop + n;
        sh.unclear = what;
      }
    }
    __syncthreads();
    stop = sh.stop;
    const int what = sh.unclear;
    __syncthreads();
    if (what == 1) {
      open = false;
    } else if (what == 2) {
      const int j = stop;
      const Part t = join(t_parts + (int64_t)j * p.runs, p.runs, p.t_scale);
      const Part d = p.draft ? join(d_parts + (int64_t)j * p.runs, p.runs, p.d_scale) : Part{0.0f, 0, 1.0};
      const Exp te = exp_of(t.m, p.t_inv), de = exp_of(d.m, p.d_inv);
      const Sums s = exact_sums(t_row(j), te, p.draft ? d_row(j) : nullptr, de);
      const int64_t id = draft_id(p, b, j);
      uint32_t st = 0;
      const double pt = term_or_0(to_f(t_row(j)[id]), te, powers) / s.t;
      const double qd = p.draft ? term_or_0(to_f(d_row(j)[id]), de, powers) / s.d : 1.0;
      if (uniform(j, st) * qd < pt) ++stop;
      else open = false;
    }
  }

  // The draw from position `stop`.
  const int64_t drafted = stop < K ? draft_id(p, b, stop) : -1;
  const bool refused = drafted >= 0 && drafted < V;
  const Part t = join(t_parts + (int64_t)stop * p.runs, p.runs, p.t_scale);
  const bool t_bad = !(t.s < (double)pos_inf()), t_none = !t_bad && !(t.m > neg_inf());
  const T* x = t_row(stop);
  int token = -1;
  double token_s = t.s;
  if (t_bad || t_none) {
    status |= t_bad ? MTR_ROW_NONFINITE : MTR_ROW_ALL_MASKED;
  } else if (p.greedy) {
    token = t.id;
  } else {
    const T* y = nullptr;
    float dm = 0.0f;
    if (refused && p.draft) {
      const Part d = join(d_parts + (int64_t)stop * p.runs, p.runs, p.d_scale);
      if (d.s < (double)pos_inf() && d.m > neg_inf()) {
        y = d_row(stop);
        dm = d.m;
      }
    }
    const int hot = refused && !p.draft ? (int)drafted : -1;
    const Exp te = exp_of(t.m, p.t_inv), de = exp_of(dm, p.d_inv);
    int a, z;  // the thread's run of ids, where terms are kept
    part_of(c0, c1, PICK, tid, a, z);
    int from = 0, to = 0;  // or the warp's piece
    double et[KEPT], ed[KEPT], above_t = 0.0, above_d = 0.0;
    int listed = 0;
    Sums s;
    if constexpr (kept) {
      float xs[KEPT], ys[KEPT];
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        xs[i] = a + i < z ? to_f(x[a + i]) : neg_inf();
        ys[i] = y && a + i < z ? to_f(y[a + i]) : neg_inf();
      }
      s = Sums{0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        et[i] = term_or_0(xs[i], te, powers);
        ed[i] = y ? term_or_0(ys[i], de, powers) : 0.0;
        s.t += et[i];
        s.d += ed[i];
      }
      s = total(s);
    } else {
      // One pass: the sums, and of the warp's piece those of the ids whose p is above
      // q.  Which they are is clear from the fp32 sums but for ids with |p - q| <
      // 2^-12 p or so, which are listed and looked at when the sums are known.
      part_of(c0, c1, PICK_WARPS, warp, from, to);
      s = Sums{0.0, 0.0, 0.0};
      if (y) {
        const Part d = join(d_parts + (int64_t)stop * p.runs, p.runs, p.d_scale);
        const double ratio = t.s / d.s;
        stream(x, y, from, to, [&](int v, float xv, float yv) {
          const double e = term(xv, te, powers), q = term(yv, de, powers), over = fma(-q, ratio, e);
          s.t += e;
          s.d += q;
          // |over| against 2^-12 of the larger term, by exponents: within a factor of two
          const int high = __double2hiint(over), size = max(__double2hiint(e), __double2hiint(q * ratio));
          const bool close = (high & 0x7fffffff) + (12 << 20) < size && size > (40 << 20);  // not both far
          if (high >= 0 && !close) {
            above_t += e;
            above_d += q;
          }
          const unsigned some = __ballot_sync(FULL, close && v < to);
          if (some) {
            const int at = listed + __popc(some & ((1u << lane) - 1u));
            if (close && v < to && at < NEAR) sh.near[warp][at] = v;
            listed += __popc(some);
          }
        });
        if (listed > NEAR) s.over = 1.0;
        __syncwarp();
      } else {
        auto add = [&](int, float xv, float) { above_t += term(xv, te, powers); };
        if (hot >= from && hot < to) {  // the drafted token has no part in the draw
          stream(x, nullptr, from, hot, add);
          stream(x, nullptr, hot + 1, to, add);
          if (lane == 0) s.t = term(to_f(x[hot]), te, powers);
        } else {
          stream(x, nullptr, from, to, add);
        }
        s.t += above_t;
      }
      s = total(s);
    }
    const bool summed = s.over == 0.0;  // the pieces' sums are complete
    token_s = s.t;
    const double over_t = 1.0 / s.t, over_d = y ? 1.0 / s.d : 0.0;
    bool from_p = false;
    // p - q of an id from its two terms, each rounded by itself: 0 where they are equal (a
    // fused product would leave its rounding, and a token be drawn from that)
    auto apart = [&](double e, double q) { return __dsub_rn(__dmul_rn(e, over_t), __dmul_rn(q, over_d)); };
    auto weight = [&](int v, double e, double q) {  // of id v
      if (from_p) return e * over_t;
      return v == hot ? 0.0 : fmax(apart(e, q), 0.0);
    };
    // the CTA's weight by pieces of a warp each, in sh.piece; the sum over the cluster
    auto weigh = [&]() {
      double w = 0.0;
      if constexpr (kept) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) w += a + i < z ? weight(a + i, et[i], ed[i]) : 0.0;
      } else if (summed && !from_p) {
        w = above_t * over_t - above_d * over_d;
        for (int i = lane; i < listed; i += 32) {
          const int v = sh.near[warp][i];
          w += weight(v, term(to_f(x[v]), te, powers), term(to_f(y[v]), de, powers));
        }
      } else {
        if (y && !from_p) {
          stream(x, y, from, to, [&](int, float xv, float yv) {
            const double one = apart(term(xv, te, powers), term(yv, de, powers));
            if (__double2hiint(one) >= 0) w += one;
          });
        } else {
          auto add = [&](int, float xv, float) { w += term(xv, te, powers); };
          if (!from_p && hot >= from && hot < to) {  // the drafted token has no part
            stream(x, nullptr, from, hot, add);
            stream(x, nullptr, hot + 1, to, add);
          } else {
            stream(x, nullptr, from, to, add);
          }
          w *= over_t;
        }
      }
      w = warp_sum(w);
      __syncthreads();
      if (lane == 0) sh.piece[warp] = w;
      __syncthreads();
      w = 0.0;
      for (int k = 0; k < PICK_WARPS; ++k) w += sh.piece[k];
      if (cs > 1) {
        cluster.sync();  // an earlier weight has been read
        if (tid == 0) sh.weight = w;
        cluster.sync();
        w = 0.0;
        for (int k = 0; k < cs; ++k) w += cluster.map_shared_rank(&sh, k)->weight;
      }
      return w;
    };
    // first piece of n whose running sum passes u (or the last that has any): its index,
    // and the sum before it.  What has none (w <= none) is passed over: u may be 0.
    auto choose = [](auto piece, int n, double u, double none, double& before) {
      double run = before, at = before;
      int last = 0;
      for (int k = 0; k < n; ++k) {
        const double w = piece(k);
        if (!(w > none)) continue;
        last = k;
        at = run;
        run += w;
        if (run > u) break;
      }
      before = at;
      return last;
    };
    double all = weigh();
    if (!(all > NOTHING)) {  // target and draft are the same: draw from the target
      from_p = true;
      all = weigh();
    }
    const double u = uniform(K, status) * all;
    double before = 0.0;
    int owner = 0;
    if (cs > 1) {
      owner = choose([&](int k) { return cluster.map_shared_rank(&sh, k)->weight; }, cs, u, kept ? 0.0 : NOTHING, before);
      cluster.sync();
      if (rank != owner) return;
    }
    // the piece that decides: a warp's, where terms are kept; else one that is weighed again by runs of a thread
    int k = choose([&](int k) { return sh.piece[k]; }, PICK_WARPS, u, kept ? 0.0 : LITTLE, before);
    double w[MOST], mine = 0.0;
    if constexpr (kept) {
#pragma unroll
      for (int i = 0; i < MOST; ++i) w[i] = a + i < z ? weight(a + i, et[i % KEPT], ed[i % KEPT]) : 0.0;
    } else {
      part_of(c0, c1, PICK_WARPS, k, from, to);
      part_of(from, to, PICK, tid, a, z);
      float xs[MOST], ys[MOST];
#pragma unroll
      for (int i = 0; i < MOST; ++i) {
        xs[i] = a + i < z ? to_f(x[a + i]) : neg_inf();
        ys[i] = y && a + i < z ? to_f(y[a + i]) : neg_inf();
      }
#pragma unroll
      for (int i = 0; i < MOST; ++i) w[i] = a + i < z ? weight(a + i, term_or_0(xs[i], te, powers), y ? term_or_0(ys[i], de, powers) : 0.0) : 0.0;
    }
#pragma unroll
    for (int i = 0; i < MOST; ++i) mine += w[i];
    if constexpr (!kept) {
      const double sum = warp_sum(mine);
      __syncthreads();
      if (lane == 0) sh.piece[warp] = sum;
      __syncthreads();
      k = choose([&](int k) { return sh.piece[k]; }, PICK_WARPS, u, 0.0, before);
    }
    if (warp == k) {
      double up = mine;  // running sums of the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double q = __shfl_up_sync(FULL, up, o);
        if (lane >= o) up += q;
      }
      const unsigned past = __ballot_sync(FULL, mine > 0.0 && before + up > u), some = __ballot_sync(FULL, mine > 0.0);
      const int who = past ? __ffs(past) - 1 : some ? 31 - __clz(some) : 0;
      if (lane == who) {
        double run = before + (up - mine);
        int last = -1;
        bool open = true;
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
          run += w[i];  // rounded otherwise than the lanes' sums: it may pass u before an id with weight
          if (open && w[i] > 0.0) {
            last = a + i;
            open = !(run > u);
          }
        }
        sh.token = last;
      }
    }
    __syncthreads();
    token = sh.token;
  }
  if (p.greedy || t_bad || t_none) {
    if (rank != 0) return;
  }

  for (int j = tid; j <= K; j += PICK) {
    int64_t out = p.pad_id;
    float lp = 0.0f;
    const int64_t id = j < stop ? draft_id(p, b, j) : j == stop && token >= 0 ? token : -1;
    if (id >= 0) {
      out = id;
      const Part r = j < stop ? join(t_parts + (int64_t)j * p.runs, p.runs, p.t_scale) : t;
      lp = (float)(((double)to_f(t_row(j)[id]) - (double)r.m) * p.t_inv - log(j < stop ? r.s : token_s));
    }
    p.tokens[b * (K + 1) + j] = out;
    if (p.logprobs) p.logprobs[b * (K + 1) + j] = lp;
  }
  if (tid == 0) {
    p.accepted[b] = stop;
    if (p.status) p.status[b] = status;
  }
}

static int esize(int32_t dtype) { return dtype == MTR_DTYPE_F32 ? 4 : 2; }

// Runs of a row (a CTA each), and vectors of a run: rows are split until there are
// four CTAs an SM or a run is a tile.  The workspace goes by this and by in_one, so
// they ask no device.
constexpr int64_t SMS = 148, ENOUGH = 4 * SMS;
struct Shape {
  int threads, runs, run;
};
static Shape shape_for(int64_t rows, int vocab, int es) {
  const int64_t vecs = ((int64_t)vocab * es + 15) / 16;
  const int threads = vecs <= 128 * HOLD ? 128 : 256;
  const int64_t tile = (int64_t)threads * HOLD, tiles = (vecs + tile - 1) / tile;
  int64_t runs = 1;
  while (runs < MTR_VERIFY_MAX_RUNS && runs < tiles && rows * runs < ENOUGH) runs *= 2;
  const int64_t each = (tiles + runs - 1) / runs;
  runs = (tiles + each - 1) / each;
  return {threads, (int)(runs > 0 ? runs : 1), (int)(each * tile)};
}
static int64_t rows_of(const MtrVerifyArgs& a) {
  return (int64_t)a.batch * (a.drafts + 1) + (a.draft_logits && a.do_sample ? (int64_t)a.batch * a.drafts : 0);
}

// Whether one launch does it all: there is a CTA for each sequence at once, and its
// rows are short enough for it.  A call from Python then costs the host 4 to 5 us less
// (a launch, and no workspace), and is bound by it; on the GPU, which is what a replayed
// graph pays, it is 2.3 us slower to 0.9 faster (us, one launch / two, GPU and call):
//   1 x 4 drafts, V = 4096 fp32    12.2 / 11.0   18.9 / 23.5
//   the same, greedy                6.5 /  5.8   16.5 / 20.8
//   64 x 8, V = 4096 bf16          16.6 / 14.3   19.9 / 24.1
//   the same, looked up            10.1 / 11.0   17.9 / 22.1
//   1 x 8, V = 600 bf16             9.8 / 10.7   19.0 / 23.2
//   256 x 8, V = 4096 bf16         32.5 / 30.1   26.4 / 26.8   (more sequences than SMs: two)
static bool in_one(int64_t batch, int64_t rows, int vocab, int es) {
  return batch <= SMS && vocab <= FEW * KEPT && rows * vocab * es <= 160 * 1024;
}

template <typename K>
static cudaError_t launch(K kern, const Params& p, dim3 grid, int threads, int cluster, cudaStream_t s) {
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

template <typename T>
static cudaError_t launch_all(Params p, int64_t rows, cudaStream_t s) {
  const Shape g = shape_for(rows, p.vocab, sizeof(T));
  p.runs = g.runs;
  p.run = g.run;
  const dim3 grid((unsigned)rows, (unsigned)g.runs, 1);
  cudaError_t e;
  if (in_one(p.batch, rows / p.batch, p.vocab, sizeof(T))) {
    p.parts = nullptr;
    p.runs = 1;
    p.cluster = 1;
    return launch(pick_kernel<T, true>, p, dim3((unsigned)p.batch, 1, 1), FEW, 1, s);
  }
  if (g.threads == 128)
    e = p.greedy ? launch(rows_kernel<T, 128, true>, p, grid, 128, 1, s) : launch(rows_kernel<T, 128, false>, p, grid, 128, 1, s);
  else
    e = p.greedy ? launch(rows_kernel<T, 256, true>, p, grid, 256, 1, s) : launch(rows_kernel<T, 256, false>, p, grid, 256, 1, s);
  if (e != cudaSuccess) return e;
  int cluster = 1;
  while (!p.greedy && cluster < 8 && p.batch * cluster * 2 <= device_sms() && p.vocab > FEW * KEPT * cluster) cluster *= 2;
  p.cluster = cluster;
  const dim3 ctas((unsigned)(p.batch * cluster), 1, 1);
  if (p.greedy || (p.vocab + cluster - 1) / cluster <= FEW * KEPT) return launch(pick_kernel<T, true>, p, ctas, FEW, cluster, s);
  return launch(pick_kernel<T, false>, p, ctas, MANY, cluster, s);
}

}  // namespace vf
}  // namespace mtr

// ---------------------------------------------------------------- C ABI
using namespace mtr::vf;

int64_t mtr_verify_workspace(int32_t batch, int32_t drafts, int32_t vocab, int32_t logits_dtype) {
  if (batch <= 0 || drafts < 0 || vocab <= 0) return 0;
  const int es = esize(logits_dtype);
  if (in_one(batch, 2 * (int64_t)drafts + 1, vocab, es)) return 0;
  const int64_t targets = (int64_t)batch * (drafts + 1), both = targets + (int64_t)batch * drafts;
  const int64_t a = targets * shape_for(targets, vocab, es).runs, b = both * shape_for(both, vocab, es).runs;
  return (a > b ? a : b) * (int64_t)sizeof(Part);
}

int mtr_verify_validate(const MtrVerifyArgs* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrVerifyArgs)) return MTR_ERR_ABI;
  if (a->batch < 0 || a->batch > MTR_MAX_VERIFY_BATCH || a->drafts < 0 || a->drafts > MTR_MAX_DRAFTS) return MTR_ERR_BAD_SHAPE;
  if (a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
  if (a->logits_dtype < MTR_DTYPE_F32 || a->logits_dtype > MTR_DTYPE_F16) return MTR_ERR_BAD_PARAM;
  if (a->ids_dtype != MTR_IDS_I64 && a->ids_dtype != MTR_IDS_I32) return MTR_ERR_BAD_PARAM;
  if (a->do_sample != 0 && a->do_sample != 1) return MTR_ERR_BAD_PARAM;
  const double temps[2] = {a->temperature, a->draft_temperature};
  for (double t : temps)
    if (!(t > 0.0) || !(t <= (double)MTR_MAX_TEMPERATURE) || !((float)(1.4426950408889634 / t) < INFINITY)) return MTR_ERR_BAD_PARAM;
  if (a->batch == 0) return MTR_OK;
  const int64_t need = mtr_verify_workspace(a->batch, a->drafts, a->vocab, a->logits_dtype);
  if (!a->target_logits || !a->out_tokens || !a->out_accepted || (need > 0 && !a->workspace)) return MTR_ERR_NULL_ARG;
  if ((a->drafts > 0 && !a->draft_ids) || (a->do_sample && !a->uniforms)) return MTR_ERR_NULL_ARG;
  if (a->target_pos_stride < a->vocab || a->target_batch_stride < 0) return MTR_ERR_BAD_SHAPE;
  if (a->draft_logits && (a->draft_pos_stride < a->vocab || a->draft_batch_stride < 0)) return MTR_ERR_BAD_SHAPE;
  if (a->ids_row_stride < 0 || a->uniforms_row_stride < 0) return MTR_ERR_BAD_SHAPE;
  if (a->workspace_bytes < need) return MTR_ERR_BAD_SHAPE;
  const int es = esize(a->logits_dtype);
  if ((uintptr_t)a->target_logits % es || (uintptr_t)a->draft_logits % es || (uintptr_t)a->draft_ids % (a->ids_dtype == MTR_IDS_I64 ? 8 : 4) ||
      (uintptr_t)a->uniforms % 4 || (uintptr_t)a->out_tokens % 8 || (uintptr_t)a->out_accepted % 4 || (uintptr_t)a->out_logprobs % 4 ||
      (uintptr_t)a->out_status % 4 || (uintptr_t)a->workspace % 16)
    return MTR_ERR_ALIGNMENT;
  // no sequence's results in what another has yet to read
  const int64_t more = a->drafts + 1, all = a->batch * more, ids_size = a->ids_dtype == MTR_IDS_I64 ? 8 : 4;
  struct Run {
    const void* at;
    int64_t n;
  };
  const Run outs[5] = {{a->workspace, need}, {a->out_tokens, 8 * all}, {a->out_accepted, 4ll * a->batch}, {a->out_logprobs, 4 * all},
                       {a->out_status, 4ll * a->batch}};
  for (const Run& o : outs) {
    if (!o.at || o.n == 0) continue;
    if (&o != outs && mtr::meets(o.at, o.n, a->workspace, 1, 0, 1, 0, need)) return MTR_ERR_BAD_PARAM;
    if (mtr::meets(o.at, o.n, a->target_logits, a->batch, a->target_batch_stride * es, more, a->target_pos_stride * es, (int64_t)a->vocab * es) ||
        mtr::meets(o.at, o.n, a->draft_ids, a->batch, a->ids_row_stride * ids_size, 1, 0, a->drafts * ids_size))
      return MTR_ERR_BAD_PARAM;
    if (a->do_sample &&
        (mtr::meets(o.at, o.n, a->draft_logits, a->batch, a->draft_batch_stride * es, a->drafts, a->draft_pos_stride * es, (int64_t)a->vocab * es) ||
         mtr::meets(o.at, o.n, a->uniforms, a->batch, a->uniforms_row_stride * 4, 1, 0, more * 4)))
      return MTR_ERR_BAD_PARAM;
  }
  return MTR_OK;
}

int mtr_verify_launch(const MtrVerifyArgs* a, void* stream) {
  const int v = mtr_verify_validate(a);
  if (v != MTR_OK) return v;
  if (a->batch == 0) return MTR_OK;
  Params p;
  memset(&p, 0, sizeof(p));
  p.target = a->target_logits;
  p.t_batch = a->target_batch_stride;
  p.t_pos = a->target_pos_stride;
  p.draft = a->do_sample ? a->draft_logits : nullptr;
  p.d_batch = a->draft_batch_stride;
  p.d_pos = a->draft_pos_stride;
  p.ids = a->draft_ids;
  p.ids_stride = a->ids_row_stride;
  p.ids32 = a->ids_dtype == MTR_IDS_I32;
  p.uniforms = a->uniforms;
  p.u_stride = a->uniforms_row_stride;
  p.batch = a->batch;
  p.drafts = a->drafts;
  p.vocab = a->vocab;
  p.greedy = !a->do_sample;
  p.t_scale = (float)(1.4426950408889634 / a->temperature);
  p.d_scale = (float)(1.4426950408889634 / a->draft_temperature);
  p.t_inv = 1.0 / a->temperature;
  p.d_inv = 1.0 / a->draft_temperature;
  p.pad_id = a->pad_id;
  p.parts = (Part*)a->workspace;
  p.tokens = a->out_tokens;
  p.accepted = a->out_accepted;
  p.logprobs = a->out_logprobs;
  p.status = a->out_status;
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t rows = rows_of(*a);
  cudaError_t e;
  switch (a->logits_dtype) {
    case MTR_DTYPE_F32: e = launch_all<float>(p, rows, s); break;
    case MTR_DTYPE_BF16: e = launch_all<__nv_bfloat16>(p, rows, s); break;
    default: e = launch_all<__half>(p, rows, s); break;
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}
