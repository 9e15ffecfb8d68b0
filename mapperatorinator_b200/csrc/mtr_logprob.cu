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
// all there are (fp32 rows reach HBM's rate; 2-byte rows 3.9 TB/s at 2.5
// instructions a cycle, with neither full).  Per score: unpack (1), the two packed steps of
// d = (x - m) (log2(e) / T) (2 x 1/2), one signed minimum, 2^d (1), and the
// packed sums of 2^d and of 2^d d (2 x 1/2); the maximum is packed too (1/2).
// The minimum does three things at once: d <= 0 compares as a signed word from
// -0 = 0x80000000 up to -inf, so masked scores (d = -inf) and far ones become
// d = -1000, whose 2^d is 0 and whose product with d is 0 as well (-inf would
// give NaN), and a score equal to the maximum, whose d is +0 = 0, becomes -1000
// too and so leaves the sums: it is counted in n.  NaN is found by the maximum,
// which keeps it.  Terms below 2^-126 count as 0, in the sums and in the gradient;
// so do those whose x - m passes the fp32 range (T <= 2^100 leaves less than
// -2^27 of it), but their log probabilities are finite again (log_prob).
#include "mtr_vec.cuh"

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
  float part, part_inv_t;  // 1/2 and 2 / T where T > 1, which may bring back what x - m takes out of the range; else 1 and 1 / T
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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
  float s;   // sum of 2^d over the others
  float u;   // sum of 2^d d
};

__device__ __forceinline__ Part empty_part() { return Part{neg_inf(), 0.0f, 0.0f, 0.0f}; }

// `p` about a larger maximum M: its terms shrink by 2^g, g = (m - M) scale, and
// each d falls by |g|; what equalled m is one of the others now.
__device__ __forceinline__ void move_to(Part& p, float M, float scale) {
  if (p.m > neg_inf()) {
    const float g = fmaxf((p.m - M) * scale, -1000.0f), f = ex2(g), t = p.s + p.n;
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
    r.entropy = r.log_s - __fdividef(LN2 * p.u, 1.0f + rest);
    r.lse = fmaf(p.m, inv_t, r.log_s);
  }
  return r;
}
__device__ __forceinline__ float log_prob(float x, const Row& r, const FwdParams& p) {
  if (r.bad) return qnan();
  if (r.none || x == neg_inf()) return neg_inf();
  return fmaf(fmaf(x, p.part, -(r.m * p.part)), p.part_inv_t, -r.log_s);
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
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

template <int W>
struct Shared {
  static constexpr int LIST = 64 * (W + 1);  // candidates of a row's alternatives
  u64 list[LIST];
  u64 best[MTR_MAX_TOP_N];  // a cluster CTA's own n largest, and how many they are
  int best_count;
  u64 bound[2];
  // by the row's parity: a warp may be a row ahead of another
  Part part[2][W];
  float nth[2][W], rth[2][W];
  int count[2];     // candidates found (where they pass LIST, the list is not complete)
  Part cta;         // read by the cluster's other CTAs
  float cta_nth, cta_rth;
  uint8_t winner[W][32];
};

// A row as one CTA sees it: single logits before the first 16-byte boundary
// and behind the last, and the CTA's run [v0, v1) of the vectors between.
template <typename T>
struct Span {
  const T* x;
  int head, vecs, v0, v1;
  __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(x + head); }
};
template <typename T>
__device__ __forceinline__ Span<T> span_of(const FwdParams& p, int64_t row, int rank) {
  constexpr int E = Vec<T>::E;
  Span<T> r;
  r.x = (const T*)p.logits + row * p.stride;
  const int off = (int)(((uintptr_t)r.x & 15u) / sizeof(T));
  r.head = min(off ? E - off : 0, p.vocab);
  r.vecs = (p.vocab - r.head) / E;
  const int run = p.cluster > 1 ? (r.vecs + p.cluster - 1) / p.cluster : r.vecs;
  r.v0 = min(rank * run, r.vecs);
  r.v1 = min(r.v0 + run, r.vecs);
  return r;
}

// Vectors of a thread's tile, and warps of an SM (so its registers).  A warp that
// has a row to itself walks a long chain a row (joins, candidates) that other
// warps must fill: more warps with smaller tiles of 32 scores a lane.  us, tiles
// of 8 vectors and 16 warps / 4 and 24 (4 and 20, 4 and 28 lie between): 8192 x
// 4096 bf16 18.2 / 16.8, with 8 alternatives 29.8 / 26.3; but fp32, whose 4
// vectors are 16 scores, 33.7 / 34.7.  Rows shared by warps want the bytes in
// flight: 1024 x 131072 fp32 81.4 / 114, 2000 x 65533 bf16 48.9 / 54.8.
template <typename T, int W>
struct Plan {
  static constexpr int TILE = W == 1 ? 32 / Vec<T>::E : 8;
  static constexpr int WARPS = W == 1 && Vec<T>::E == 8 ? 24 : 16;
};

// tile starting at vector t0 of the CTA's run; masked scores behind its end
template <int THREADS, int TILE, typename T>
__device__ __forceinline__ void load_tile(uint4 (&w)[TILE], const Span<T>& r, int t0, int tid) {
  const uint4* b = r.body() + t0 + tid;
  if (t0 + THREADS * TILE <= r.v1) {
#pragma unroll
    for (int j = 0; j < TILE; ++j) w[j] = b[j * THREADS];
  } else {
    constexpr uint32_t F = Vec<T>::FILL;
#pragma unroll
    for (int j = 0; j < TILE; ++j) w[j] = t0 + tid + j * THREADS < r.v1 ? b[j * THREADS] : make_uint4(F, F, F, F);
  }
}

// how many of list[0 .. c) are larger than k
__device__ __forceinline__ int place_of(const u64* list, int c, u64 k) {
  int place = 0;
#pragma unroll 4
  for (int j = 0; j < c; ++j) place += list[j] > k;
  return place;
}

// A CTA of W warps takes one row after another (a cluster of CTAs takes one).
//
// A thread's tile is TILE vectors; the next tile, of this row or of the CTA's
// next one, is under way while one is summed.  A warp keeps one maximum (one
// redux a tile), so that its lanes' sums move to a new maximum together and
// rarely.
//
// Alternatives: with lm the lanes' maxima, any T with at least n logits >= T
// bounds the n largest from below.  Two such T are at hand: the n-th largest lm
// of a warp, the best warp's taken, and the smallest over all warps of the r-th
// largest lm, r n-th part of the warps (n <= r warps).  (The n-th of 32 maxima
// is a poor bound when n is near 32; then a lane keeps two maxima.)  The larger
// of the two leaves about n to 3 n lanes with lm >= T, whose vectors are read again
// (from L2) for the list of candidates, which are ranked by comparing all pairs.  A
// list that overflows (many equal logits) is left at once: it holds more than n
// candidates, the n-th of them is a better T, and they are looked for again.
template <typename T, int W>
__global__ void __launch_bounds__(W * 32, Plan<T, W>::WARPS / W) logprob_kernel(const FwdParams p) {
  typedef Vec<T> X;
  constexpr int E = X::E, THREADS = W * 32, TILE = Plan<T, W>::TILE;
  __shared__ Shared<W> sh;
  constexpr int LIST = Shared<W>::LIST;
  const int tid = threadIdx.x, warp = W > 1 ? tid >> 5 : 0, lane = tid & 31;
  const int cs = p.cluster, rank = cs > 1 ? (int)(blockIdx.x % cs) : 0;
  const int64_t step = cs > 1 ? gridDim.x / cs : gridDim.x;
  int64_t row = cs > 1 ? blockIdx.x / cs : blockIdx.x;
  const int V = p.vocab, n = p.top_n;
  const bool split = n > 24;  // bounds from 64 maxima a warp instead of 32
  const float scale = p.scale;
  auto cta_sync = [&]() {
    if (W > 1) __syncthreads();
    else __syncwarp();
  };
  if (W > 1 && tid < 2) sh.count[tid] = 0;
  wait_prior_grid();
  Span<T> sp = span_of<T>(p, row, rank);
  uint4 next[TILE];
  load_tile<THREADS>(next, sp, sp.v0, tid);

  for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
    // the token and its logit, needed last, are asked for first
    int64_t token = -1;
    float token_x = 0.0f;
    if (tid == 0 && rank == 0 && p.tokens) {
      token = load_id(p.tokens, p.ids32, row);
      if (token >= 0 && token < V) token_x = to_f(sp.x[token]);
    }
    const int tail = V - sp.head - sp.vecs * E;
    Part a = empty_part();
    float lm[2] = {neg_inf(), neg_inf()};  // the lane's largest logits, of its tiles' even and odd vectors
    bool bad = false;
    // the single scores: lanes 0 .. head - 1 and 16 .. 16 + tail - 1 of the first warp
    float single = neg_inf();
    int single_id = -1;
    if (warp == 0 && rank == 0 && sp.head + tail > 0) {
      if (lane < sp.head) single_id = lane;
      else if (lane >= 16 && lane < 16 + tail) single_id = V - tail + lane - 16;
      if (single_id >= 0) single = to_f(sp.x[single_id]);
      const float top = warp_max_nan(single);
      bad = !(top < pos_inf());
      if (!bad && top > neg_inf()) {
        a.m = top;
        if (single == top) a.n = 1.0f;
        else if (single > neg_inf()) {
          const float d = fmaxf((single - top) * scale, -1000.0f);
          a.s = ex2(d);
          a.u = a.s * d;
        }
        lm[0] = single;
      }
    }
    Span<T> after = sp;
    u64 s2 = 0, u2 = 0;  // pairs of partial sums, added to a.s, a.u when the maximum moves
    auto sum_tile = [&](const uint4 (&w)[TILE]) {
      typename X::Top top[TILE];
#pragma unroll
      for (int j = 0; j < TILE; ++j) top[j] = X::top(w[j]);
      typename X::Top even = top[0], odd = top[1];
#pragma unroll
      for (int j = 2; j < TILE; j += 2) {
        even = X::larger(even, top[j]);
        odd = X::larger(odd, top[j + 1]);
      }
      const float mine = X::value(X::larger(even, odd)), most = warp_max_nan(mine);
      if (!(most < pos_inf())) bad = true;
      if (split) {
        lm[0] = fmaxf(lm[0], X::value(even));
        lm[1] = fmaxf(lm[1], X::value(odd));
      } else {
        lm[0] = fmaxf(lm[0], mine);
      }
      if (most > a.m) {
        float lo, hi;
        up2(s2, lo, hi);
        a.s += lo + hi;
        up2(u2, lo, hi);
        a.u += lo + hi;
        s2 = u2 = 0;
        move_to(a, most, scale);
      }
      if (bad || !(a.m > neg_inf())) return;
      if (mine == a.m) {
        const typename X::Top m = X::pattern(a.m);
        uint32_t equal = 0;
#pragma unroll
        for (int j = 0; j < TILE; ++j) equal += X::equal(w[j], m);
        a.n += (float)X::count(equal);
      }
      const float nm = 0.0f - a.m;  // +0 for both zeros, so that equal scores differ by +0
      const u64 nm2 = pk2(nm, nm), sc2 = pk2(scale, scale);
#pragma unroll
      for (int j = 0; j < TILE; ++j) {
        float f[E];
        X::unpack(w[j], f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          float d0, d1;
          up2(mul2(add2(pk2(f[e], f[e + 1]), nm2), sc2), d0, d1);
          d0 = __int_as_float(min(__float_as_int(d0), (int)0xc47a0000));  // -1000
          d1 = __int_as_float(min(__float_as_int(d1), (int)0xc47a0000));
          const u64 e2 = pk2(ex2(d0), ex2(d1));
          s2 = add2(s2, e2);
          u2 = fma2(e2, pk2(d0, d1), u2);
        }
      }
    };
    // the tile behind the one at t0 - THREADS TILE: this row's, or the next row's first
    auto ask = [&](uint4 (&w)[TILE], int t0) {
      if (t0 < sp.v1) {
        load_tile<THREADS>(w, sp, t0, tid);
      } else if (row + step < p.rows) {
        after = span_of<T>(p, row + step, rank);
        load_tile<THREADS>(w, after, after.v0, tid);
      }
    };
    for (int t0 = sp.v0 + THREADS * TILE;; t0 += THREADS * TILE) {
      uint4 w[TILE];
#pragma unroll
      for (int j = 0; j < TILE; ++j) w[j] = next[j];
      ask(next, t0);
      sum_tile(w);
      if (t0 >= sp.v1) break;
    }
    {
      float lo, hi;
      up2(s2, lo, hi);
      a.s += lo + hi;
      up2(u2, lo, hi);
      a.u += lo + hi;
    }
    a.n = (float)__reduce_add_sync(FULL, (unsigned)a.n);
    u64 su = pk2(a.s, a.u);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) su = add2(su, __shfl_xor_sync(FULL, su, o));
    up2(su, a.s, a.u);
    if (bad) a = Part{neg_inf(), 0.0f, qnan(), 0.0f};

    // join the warps, then the CTAs
    float nth = neg_inf(), rth = neg_inf();
    if (n > 0) {
      float sorted = warp_sort_desc(lm[0], lane);
      if (split) {
        // the 32 largest of both halves: the larger of each pair of a descending and an ascending sequence
        sorted = fmaxf(sorted, __shfl_sync(FULL, warp_sort_desc(lm[1], lane), 31 - lane));
        sorted = warp_sort_desc(sorted, lane);
      }
      nth = __shfl_sync(FULL, sorted, n - 1);
      rth = __shfl_sync(FULL, sorted, (n + W * cs - 1) / (W * cs) - 1);
    }
    if (W > 1) {
      if (lane == 0) {
        sh.part[parity][warp] = a;
        sh.nth[parity][warp] = nth;
        sh.rth[parity][warp] = rth;
      }
      __syncthreads();
      // every group of W lanes joins the W parts
      a = lanes_join(sh.part[parity][lane % W], W, scale);
      nth = sh.nth[parity][lane % W];
      rth = sh.rth[parity][lane % W];
#pragma unroll
      for (int o = 1; o < W; o <<= 1) {
        nth = fmaxf(nth, __shfl_xor_sync(FULL, nth, o));
        rth = fminf(rth, __shfl_xor_sync(FULL, rth, o));
      }
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (cs > 1) {
      if (tid == 0) {
        sh.cta = a;
        sh.cta_nth = nth;
        sh.cta_rth = rth;
      }
      cluster.sync();
      const Shared<W>* other = cluster.map_shared_rank(&sh, lane % cs);
      a = lanes_join(other->cta, cs, scale);
      nth = other->cta_nth;
      rth = other->cta_rth;
      for (int o = 1; o < cs; o <<= 1) {
        nth = fmaxf(nth, __shfl_xor_sync(FULL, nth, o));
        rth = fminf(rth, __shfl_xor_sync(FULL, rth, o));
      }
    }
    const Row r = row_of(a, p.inv_t);
    if (tid == 0 && rank == 0) {
      uint32_t st = r.bad ? MTR_ROW_NONFINITE : r.none ? MTR_ROW_ALL_MASKED : 0u;
      if (p.tokens) {
        if (token >= V) st |= MTR_ROW_BAD_ID;
        if (p.logprobs) p.logprobs[row] = (token < 0 || token >= V) ? 0.0f : log_prob(token_x, r, p);
      }
      if (p.entropy) p.entropy[row] = r.entropy;
      if (p.lse) p.lse[row] = r.lse;
      if (p.stats) p.stats[row] = make_float4(r.m, r.log_s, r.entropy, 0.0f);
      if (p.status) p.status[row] = st;
    }
    if (n == 0) {
      if (cs > 1) cluster.sync();  // this CTA's parts have been read
      sp = after;
      continue;
    }

    // candidates: keys of the scores that reach the bound
    u64 bound = order_key(fmaxf(nth, rth), 0xffffffffu);
    int c = 0;
    if (W > 1 && tid == 0) sh.count[parity ^ 1] = 0;
    bool again = false, full = false;
    float least = 0.0f;  // the bound's score; of masked scores none is a candidate
    auto list = [&](float f, int id) {
      bool hit = f >= least;
      if (again) hit = hit && order_key(f, (uint32_t)id) >= bound;
      const unsigned hits = __ballot_sync(FULL, hit);
      if (hits == 0) return;
      int at = c;
      if (W > 1) {
        if (lane == 0) at = atomicAdd(&sh.count[parity], __popc(hits));
        at = __shfl_sync(FULL, at, 0);
      } else {
        c += __popc(hits);
      }
      full = at + __popc(hits) > LIST;
      at += __popc(hits & ((1u << lane) - 1u));
      if (hit && at < LIST) sh.list[at] = order_key(f, (uint32_t)id);
    };
    while (!r.bad && !r.none) {
      least = fmaxf(key_value(bound), X::LOWEST);
      const typename X::Top cut = X::pattern(least);
      if (warp == 0 && rank == 0 && sp.head + tail > 0) list(single, single_id);
      const float top = fmaxf(lm[0], lm[1]);
      const bool won = top >= least;
      const unsigned winners = __ballot_sync(FULL, won);
      if (won) sh.winner[warp][__popc(winners & ((1u << lane) - 1u))] = (uint8_t)lane;
      __syncwarp();
      // a half warp reads one winner's vectors, 16 at a time, for four winners in turn
      const uint4* body = sp.body();
      const int most_of = (sp.v1 - sp.v0 - warp * 32 + THREADS - 1) / THREADS;  // vectors of the warp's first lane
      const int count = __popc(winners);
      for (int first = 0; first < count && !full; first += 8)
        for (int i0 = 0; i0 < most_of && !full; i0 += 16) {
          uint32_t reach = 0;  // bits 4 j ..: the j-th vector's
          auto vector = [&](int j) {
            const int who = first + 2 * j + (lane >> 4);
            return who < count ? sp.v0 + warp * 32 + sh.winner[warp][who] + (i0 + (lane & 15)) * THREADS : sp.v1;
          };
          uint4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = vector(j);
            w[j] = at < sp.v1 ? body[at] : make_uint4(X::FILL, X::FILL, X::FILL, X::FILL);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) reach |= X::reach(w[j], cut) << (4 * j);
          while (!full && __any_sync(FULL, reach != 0u)) {  // one score a lane
            const int bit = reach ? __ffs(reach) - 1 : 0;
            const int id = sp.head + vector((bit >> 2) & 3) * E + (E == 8 ? 2 * (bit & 3) + (bit >> 4) : bit & 3);
            list(reach ? to_f(sp.x[id]) : neg_inf(), id);
            reach &= reach - 1;
          }
        }
      cta_sync();
      if (W > 1) c = sh.count[parity];
      if (c <= LIST) break;
      // overflow: the list's n-th key is the new bound (LIST > n, so the count falls)
      for (int i = tid; i < LIST; i += THREADS) {
        const u64 k = sh.list[i];
        const int place = place_of(sh.list, LIST, k);
        if (place == n - 1) sh.bound[parity] = k;
      }
      cta_sync();
      bound = sh.bound[parity];
      again = true;
      full = false;
      c = 0;
      if (W > 1 && tid == 0) sh.count[parity] = 0;
      cta_sync();
    }
    if (cs > 1) {
      // the CTAs' own n largest, ranked by the first CTA
      for (int i = tid; i < c; i += THREADS) {
        const u64 k = sh.list[i];
        const int place = place_of(sh.list, c, k);
        if (place < n) sh.best[place] = k;
      }
      if (tid == 0) sh.best_count = min(c, n);
      cluster.sync();
      if (rank == 0) {
        c = 0;
        for (int k = 0; k < cs; ++k) {
          const Shared<W>* other = cluster.map_shared_rank(&sh, k);
          const int more = other->best_count;
          for (int i = tid; i < more; i += THREADS) sh.list[c + i] = other->best[i];
          c += more;
        }
      }
      cluster.sync();  // the others' keys have been read
      if (rank != 0) return;
    }
    int64_t* ids = p.top_ids + row * n;
    float* lps = p.top_logprobs + row * n;
    for (int i = tid; i < c; i += THREADS) {
      const u64 k = sh.list[i];
      const int place = place_of(sh.list, c, k);
      if (place < n) {
        ids[place] = key_id(k);
        lps[place] = log_prob(key_value(k), r, p);
      }
    }
    for (int j = c + tid; j < n; j += THREADS) {
      ids[j] = -1;
      lps[j] = r.bad ? qnan() : neg_inf();
    }
    if (W == 1) __syncwarp();  // the list has been read before the next row's candidates
    sp = after;
  }
}

// grad_v = p_v (a + b log2 p_v) + (what is given to v alone), a and b one row's
// two numbers (both divided by T).  One CTA owns a run of a row's vectors and
// asks for them before anything else; the row's numbers arrive meanwhile.  The
// few ids that are given something of their own (the token, the alternatives)
// are written once more after the run, one thread for each distinct id, so a
// token that is also an alternative is summed before the rounding.  With o_v what
// is given to v alone, the row's `a` holds -o_v p_v: v gets o_v (1 - p_v) + p_v
// (the others' terms), 1 - p_v = -expm1(log p_v), which keeps the digits of a
// gradient that is small because p_v is near 1.  4 bytes of traffic for a bf16 score and about 6 instructions: HBM
// bounds it.
struct GradRow {
  float m, log2_s, a, b;
};
template <typename T>
__device__ __forceinline__ float grad_of(T x, const GradRow& r, float scale) {
  const float d = max_nan(fmaf(to_f(x) - r.m, scale, -r.log2_s), -1000.0f);
  return ex2(d) * fmaf(r.b, d, r.a);
}

// the same for an id that `own` is given to alone; `rest` is what the row's even part has from the others
template <typename T>
__device__ __forceinline__ float own_grad_of(T x, const GradRow& r, const GradParams& p, float log_s, float own, float rest) {
  const float logp = fmaf(to_f(x) - r.m, p.inv_t, -log_s), d = max_nan(fmaf(to_f(x) - r.m, p.scale, -r.log2_s), -1000.0f);
  return fmaf(-own * p.inv_t, expm1f(logp), ex2(d) * fmaf(r.b, d, rest * p.inv_t));
}

constexpr int GRAD_VECS = 4;  // vectors a thread holds
constexpr int MAX_SLOTS = MTR_MAX_TOP_N + 1;

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
  const float gz = p.g_lse ? p.g_lse[row] : 0.0f;
  float even = gz - gt - gh * st.z;
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
    if (tid == 0) g[tok] = from_f<T>(own_grad_of(x[tok], r, p, st.y, gt, gz - gh * st.z));
    return;
  }
  __syncthreads();
  if (tid < slots) {
    const int id = slot_id[tid];
    bool mine = id >= from && id < to;
    float own = 0.0f, rest = gz - gh * st.z;
    for (int j = 0; j < slots; ++j)
      if (slot_id[j] == id) {
        if (j < tid) mine = false;  // an earlier slot writes it
        own += slot_g[j];
      } else {
        rest -= slot_g[j];
      }
    if (mine) g[id] = from_f<T>(own_grad_of(x[id], r, p, st.y, own, rest));
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

// Warps and CTAs of a row, by how many rows there are to fill the device's 16
// warps an SM and how long they are.  Measured (us, 148 SMs):
//   8192 x 4096 bf16      1 warp 16.8, 2 23.0, 4 44.6     enough rows: a warp each
//   2000 x 65533 bf16     1 warp 50.4, 2 52.6, 4 48.1, 8 57.3   long rows: 4
//   1024 x 131072 fp32    1 warp 99.1, 2 81.7, 4 80.8, 8 83.6
//   256 x 65536 fp16      1 warp 24.6, 4 11.4, 8 10.6, 4 CTAs of 8 25.8
//   64 x 4096 fp32, n = 5 1 warp 5.4, 4 4.2, 8 4.5        256 vectors a warp at least
//   1 x 131072 fp32       8 warps 14.7, 4 CTAs of 8 9.8, 8 CTAs 9.7
// More warps than the rows need cost their joins; clusters pay only where they
// give idle SMs work.
struct Shape {
  int warps, cluster;
};
static Shape shape_for(int64_t rows, int vocab, int es) {
  const int64_t vecs = ((int64_t)vocab * es + 15) / 16, sms = device_sms();
  int warps = vecs >= 4096 ? 4 : 1;
  while (warps < MAX_WARPS && rows * warps < 16 * sms && vecs > 256 * warps) warps *= 2;
  int cluster = 1;  // only of 8 warps: MAX_CLUSTER * MTR_MAX_TOP_N keys must fit the list
  while (warps == MAX_WARPS && cluster < MAX_CLUSTER && vecs > 2048ll * cluster && rows * cluster < sms) cluster *= 2;
  return {warps, cluster};
}

template <typename T, int W>
static cudaError_t launch_fwd(FwdParams p, int cluster, cudaStream_t s) {
  auto kern = logprob_kernel<T, W>;
  p.cluster = cluster;
  if (cluster > 1) return launch(kern, p, dim3((unsigned)(p.rows * cluster), 1, 1), 32 * W, cluster, s);
  int occ = 0;
  const cudaError_t e = cached_occupancy((const void*)kern, 32 * W, 0, &occ);
  if (e != cudaSuccess) return e;
  const int64_t room = (int64_t)(occ > 0 ? occ : 1) * device_sms();
  return launch(kern, p, dim3((unsigned)(p.rows < room ? p.rows : room), 1, 1), 32 * W, 1, s);
}
template <typename T>
static cudaError_t launch_fwd(const FwdParams& p, cudaStream_t s) {
  const Shape g = shape_for(p.rows, p.vocab, sizeof(T));
  switch (g.warps) {
    case 1: return launch_fwd<T, 1>(p, g.cluster, s);
    case 2: return launch_fwd<T, 2>(p, g.cluster, s);
    case 4: return launch_fwd<T, 4>(p, g.cluster, s);
    default: return launch_fwd<T, 8>(p, g.cluster, s);
  }
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

template <typename A>
static int check_common(const A* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(A)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->rows > MTR_MAX_SCORE_ROWS || a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
  if (a->logits_dtype < MTR_DTYPE_F32 || a->logits_dtype > MTR_DTYPE_F16) return MTR_ERR_BAD_PARAM;
  if (a->tokens_dtype != MTR_IDS_I64 && a->tokens_dtype != MTR_IDS_I32) return MTR_ERR_BAD_PARAM;
  if (a->top_n < 0 || a->top_n > MTR_MAX_TOP_N) return MTR_ERR_BAD_PARAM;
  if (!(a->temperature > 0.0f) || !(a->temperature <= MTR_MAX_TEMPERATURE) || !(1.4426950408889634f / a->temperature < INFINITY))
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
  p.part = a->temperature > 1.0f ? 0.5f : 1.0f;
  p.part_inv_t = p.inv_t / p.part;
  p.logprobs = a->out_logprobs;
  p.entropy = a->out_entropy;
  p.lse = a->out_lse;
  p.top_ids = a->out_top_ids;
  p.top_logprobs = a->out_top_logprobs;
  p.stats = (float4*)a->out_stats;
  p.status = a->out_status;
  p.cluster = 1;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  switch (a->logits_dtype) {
    case MTR_DTYPE_F32: e = launch_fwd<float>(p, s); break;
    case MTR_DTYPE_BF16: e = launch_fwd<__nv_bfloat16>(p, s); break;
    default: e = launch_fwd<__half>(p, s); break;
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
  const int64_t es = esize(a->logits_dtype);
  if (overlap(mtr::bytes_of(a->logits, a->rows, a->logits_row_stride, a->vocab, es),
              mtr::bytes_of(a->grad_logits, a->rows, a->grad_row_stride, a->vocab, es)))
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
