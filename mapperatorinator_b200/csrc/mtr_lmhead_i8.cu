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
#include <type_traits>

#include "mtr_quant.cuh"
#include "mtr_tc.cuh"

namespace mtr {
namespace i8 {

using namespace tc;

constexpr int BM = 128;  // rows of a CTA's tile
constexpr int BK = 128;  // int8 elements of one 128-byte swizzled row
constexpr int UK = 32;   // K of one tcgen05.mma kind::i8
constexpr int QUANT_THREADS = 128;

struct QuantParams {
  const void* x;
  int64_t x_stride;
  int32_t rows;
  int32_t cols;
  int32_t threads_per_row;
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
  int32_t m_tiles, n_tiles;
  int32_t a_bytes;   // bytes of a hidden tile's copy
  int32_t store_tma; // logits rows are 16-byte aligned: tiles leave by TMA
  int32_t tma_ids;   // ids that may leave so: a TMA store at an edge inside 16 bytes would write all of them
  uint32_t* err;
  int32_t give_up;   // test hook: the epilogue takes its first wait as run out
};

// Rows to int8: threads_per_row threads (a power of two, 32 .. 128) take a row
// (quantize_row).  HBM bounds it: 3 bytes a bf16 value.  HOLD is 4 where a warp's
// 4 vectors a lane hold a row, else 8 (us, 4 / 8, its bytes at the measured copy
// rate): 8192 x 768 bf16 4.9 / 6.6, 2.9; 8192 x 4096 bf16 20.3 / 18.8, 15.4;
// 131072 x 1024 fp32 119 / 94, 102 (mostly reads, which run faster than a copy).
template <typename T, bool VEC, int HOLD>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_kernel(const QuantParams p) {
  __shared__ float tops[QUANT_THREADS / 32];
  const int per = p.threads_per_row, sub = threadIdx.x / per, tid = threadIdx.x % per;
  wait_prior_grid();
  const int64_t row = (int64_t)blockIdx.x * (QUANT_THREADS / per) + sub;
  const bool live = row < p.rows;
  const float scale = quantize_row<T, VEC, HOLD>((const T*)p.x + (live ? row : 0) * p.x_stride, live ? p.cols : 0, per, sub, tid, tops,
                                                 p.q + (live ? row : 0) * p.q_stride, [] { allow_dependents(); });
  if (live && tid == 0) p.scale[row] = scale;
}

// One product, operands as the low words of their shared-memory descriptors: the
// high word is the same for every tile of this layout (sw128_desc), and a stage
// or a step of K moves the low word by its bytes / 16.
template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
        : "memory");
}

// Instruction descriptor of kind::i8: int32 accumulator (bits 4-5 = 2), signed A
// and B (bits 7-9, 10-12 = 1), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Tiles of 128 rows x BN vocabulary ids for one CTA (CG = 1), or of 256 rows x BN
// for a pair of CTAs (CG = 2) whose products run on both tensor cores at once:
// each CTA loads its own 128 rows and half of the ids, and each half serves both,
// so a pair takes 64 KB a step of K out of L2 where two CTAs alone take 96.
//
// What bounds it: at d = 4096 the products (8192 x 4096 -> 16384 in 331 us without
// the quantisation, 3.3 POP/s: 2.03 times the measured bf16 rate).  At d = 768
// neither side alone: 8192 x 768 -> 4096 takes 25 us without the quantisation,
// 20 with one step of K (the epilogue and its stores), 19 with the epilogue's
// work left out (six steps of K, starts and ends of 512 tiles); an accumulator is
// free only when all of it has been read, so the two overlap in part.
//
// Persistent: a CTA (pair) takes tile after tile, with two accumulators in tensor
// memory, so that one tile is scaled and stored while the next is multiplied.
//   warp 0, one lane   producer: TMA loads into a ring of STAGES stages
//   warp 1, one lane   issues the products (of a pair: the first CTA's only);
//                      the whole warp allocates and frees the tensor memory
//   warps 2-9          epilogue: warp w owns tensor memory lanes 32 (w % 4) ..,
//                      tile rows, and half of the columns (two warps a
//                      scheduler, so that one works while the other waits for
//                      tensor memory); scales them, rounds, stages 32 rows x 128 bytes
//                      in shared memory (16-byte pieces XOR-swizzled by row) and
//                      sends them by TMA, or row by row where rows of logits are
//                      not 16-byte aligned
// Every wait is bounded; a role whose wait gives up counts it (gave_up) and stops,
// so that the others' waits give up too; the producer then gives its copies time
// to land, the epilogue writes NaN for what was not computed, and the CTA returns.
constexpr int EPI = 8;  // epilogue warps
constexpr int PROJ_THREADS = 64 + 32 * EPI;

template <int CG, int BN>
struct Geo {
  static constexpr uint32_t A_BYTES = BM * BK, B_BYTES = BN / CG * BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr uint32_t BOX_BYTES = 32 * 128;  // one epilogue warp's staging buffer
  static constexpr uint32_t OUT_BYTES = EPI * BOX_BYTES;
  static constexpr uint32_t FIXED = 2560;          // barriers, flags, column scales
  static constexpr int FIT = (int)((227 * 1024 - OUT_BYTES - FIXED) / STAGE_BYTES);
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr uint32_t DYN = STAGES * STAGE_BYTES + OUT_BYTES + FIXED;
  static constexpr uint32_t COLS = 2 * BN;  // tensor-memory columns
};

// 32 accumulators to fp32, rounded to nearest even.  Below 2^22 in magnitude
// (all but a few: the bound is 127^2 d) the sum m = acc + bits(1.5 2^23) is the
// word of the float 1.5 2^23 + acc, so an integer and half a packed float
// addition convert it; the conversion instruction runs at a quarter of that
// rate and would bound the epilogue (2048 clocks a 128 x 256 tile).
__device__ __forceinline__ void to_floats(uint32_t (&v)[32]) {
  constexpr uint32_t BIAS = 0x4b400000u;  // 1.5 2^23
  uint32_t far = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) far |= (v[i] + BIAS) ^ 0x4b000000u;
  if (__any_sync(FULL, far >= 0x800000u)) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__int2float_rn((int)v[i]));
  } else {
    const u64 back = pk2(-12582912.0f, -12582912.0f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float lo, hi;
      up2(add2(pk2(__uint_as_float(v[i] + BIAS), __uint_as_float(v[i + 1] + BIAS)), back), lo, hi);
      v[i] = __float_as_uint(lo);
      v[i + 1] = __float_as_uint(hi);
    }
  }
}

template <int CG, int BN, typename Tout>
__global__ void __launch_bounds__(PROJ_THREADS, 1)
    lmhead_i8_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_out, const ProjParams p) {
  typedef Geo<CG, BN> G;
  constexpr int S = G::STAGES;
  constexpr int CB = BN * (int)sizeof(Tout) < 128 ? BN : 128 / (int)sizeof(Tout);  // columns of a staging buffer
  constexpr int PIECES = CB * (int)sizeof(Tout) / 16;                              // 16-byte pieces of its rows
  struct Fixed {
    uint64_t full[S], empty[S], acc_full[2], acc_empty[2];
    uint32_t tmem_slot;
    __align__(16) float col_scale[EPI][64];
  };
  static_assert(sizeof(Fixed) <= G::FIXED, "fixed part of the shared memory");
  // the swizzle patterns of ring and staging repeat every 1024 bytes
  extern __shared__ __align__(1024) uint8_t ring[];
  Fixed& fx = *reinterpret_cast<Fixed*>(ring + (size_t)S * G::STAGE_BYTES + G::OUT_BYTES);
  uint64_t *const full = fx.full, *const empty = fx.empty, *const acc_full = fx.acc_full, *const acc_empty = fx.acc_empty;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = CG > 1 ? (int)(blockIdx.x % CG) : 0;  // within the pair
  auto a_tile = [&](int s) { return ring + (size_t)s * G::STAGE_BYTES; };
  auto b_tile = [&](int s) { return ring + (size_t)s * G::STAGE_BYTES + G::A_BYTES; };

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_h) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_w) : "memory");
    if (p.store_tma) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_out) : "memory");
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], EPI * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&fx.tmem_slot)), "r"(G::COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&fx.tmem_slot)), "r"(G::COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG > 1) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = fx.tmem_slot;

  // The CTA's (pair's) tiles are first, first + step, ...: sixteen row tiles by all
  // columns, rows first, so that the tiles in flight share rows and ids in L2.
  const int tiles = p.m_tiles * p.n_tiles, first = (int)(blockIdx.x / CG), step = (int)(gridDim.x / CG);
  const int KB = p.kblocks;
  auto place = [&](int t, int& m0, int& n0) {
    constexpr int GROUP = 16;
    const int per = GROUP * p.n_tiles, g = t / per, in = t - g * per;
    const int high = min(GROUP, p.m_tiles - g * GROUP);
    n0 = in / high * BN;
    m0 = ((g * GROUP + in % high) * CG + cta) * BM;
  };
  // the ids' part of a stage (CG = 2: of both CTAs, counted on the first one's barrier), with the bytes of all of it
  auto load_ids = [&](int slot, int kb, int n0) {
    const uint32_t bytes = (uint32_t)p.a_bytes + G::B_BYTES;
    if (CG == 1) {
      mbar_expect_tx(&full[slot], bytes);
      tma_load_2d(b_tile(slot), &map_w, kb * BK, n0, &full[slot]);
    } else {
      if (cta == 0) mbar_expect_tx(&full[slot], 2 * bytes);
      load_pair(b_tile(slot), &map_w, kb * BK, n0 + cta * (BN / CG), map_to(smem_u32(&full[slot]), 0));
    }
  };
  uint32_t early = 0;  // stages whose ids have been asked for ahead
  auto load_early = [&]() {
    for (int t = first; t < tiles && early < (uint32_t)S; t += step) {
      int m0, n0;
      place(t, m0, n0);
      for (int kb = 0; kb < KB && early < (uint32_t)S; ++kb, ++early) load_ids((int)early, kb, n0);
    }
  };

  // The weight tiles of the first stages are asked for before the quantisation of
  // the hidden states is waited for: that kernel lets this one in only after its
  // own wait, when whatever wrote the weight has completed.
  if (warp == 0 && lane == 0) load_early();
  wait_prior_grid();

  if (warp == 0 && lane == 0) {
    // ---------------- producer
    Turn turn;
    uint32_t it = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (mbar_wait(bar, parity, WAIT_NS)) return true;
      gave_up(p.err, 1u);
      return false;
    };
    for (int t = first; t < tiles && ok; t += step) {
      int m0, n0;
      place(t, m0, n0);
      for (int kb = 0; kb < KB && ok; ++kb, ++it, turn.next(S)) {
        ok = wait(&empty[turn.slot], turn.parity ^ 1);
        if (!ok) break;
        if (it >= early) load_ids(turn.slot, kb, n0);
        if (CG == 1) tma_load_2d(a_tile(turn.slot), &map_h, kb * BK, m0, &full[turn.slot]);
        else load_pair(a_tile(turn.slot), &map_h, kb * BK, m0, map_to(smem_u32(&full[turn.slot]), 0));
      }
    }
    // every stage is free: its copies have landed and the arrivals on its barriers are in
    for (int i = 0; ok && i < S; ++i, turn.next(S)) ok = wait(&empty[turn.slot], turn.parity ^ 1);
    if (!ok) {  // copies under way get time to land before the CTA may leave
      const uint64_t t0 = global_ns();
      while (global_ns() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 1 && lane == 0 && cta == 0) {
    // ---------------- products
    constexpr uint32_t idesc = idesc_i8(BM * CG, BN);
    Turn turn;
    uint32_t n = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (mbar_wait(bar, parity, WAIT_NS)) return true;
      gave_up(p.err, 2u);
      return false;
    };
    // this thread feeds the tensor core alone, a stage of products every 512
    // clocks at most: everything a stage needs is an addition to these
    const uint64_t desc = sw128_desc(smem_u32(ring));
    const uint32_t lo0 = (uint32_t)desc, hi = (uint32_t)(desc >> 32);
    auto commit = [&](uint64_t* bar) {
      if (CG == 1) tc_commit(bar);
      else commit_pair(bar);
    };
    for (int t = first; t < tiles && ok; t += step, ++n) {
      const int acc = n & 1;
      ok = wait(&acc_empty[acc], ((n >> 1) & 1) ^ 1);
      if (!ok) break;
      tc_fence_after();
      for (int kb = 0; kb < KB; ++kb, turn.next(S)) {
        ok = wait(&full[turn.slot], turn.parity);
        if (!ok) break;
        const uint32_t a_lo = lo0 + (uint32_t)turn.slot * (G::STAGE_BYTES >> 4), b_lo = a_lo + (G::A_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < BK / UK; ++k)
          mma_i8<CG>(tmem + acc * BN, a_lo + k * (UK >> 4), b_lo + k * (UK >> 4), hi, idesc, k > 0 ? 1u : (uint32_t)kb);
        commit(&empty[turn.slot]);
      }
      if (!ok) break;
      commit(&acc_full[acc]);
    }
  } else if (warp >= 2) {
    // a warp's columns, a staging buffer's at a time
    constexpr int PART = BN / (EPI / 4) < CB ? CB : BN / (EPI / 4);
    const int quad = warp & 3, c0 = (warp - 2) / 4 * PART;
    uint8_t* box = ring + (size_t)S * G::STAGE_BYTES + (size_t)(warp - 2) * G::BOX_BYTES;
    float* cs = fx.col_scale[warp - 2];
    // the scales of a tile, asked for a tile ahead: columns lane, lane + 32, ... and the lane's row
    float cs_next[PART / 32], rs_next = 0.0f;
    auto ask = [&](int t) {
      int m0, n0;
      place(t, m0, n0);
#pragma unroll
      for (int i = 0; i < PART / 32; ++i) {
        const int col = n0 + c0 + i * 32 + lane;
        cs_next[i] = c0 < BN && col < p.vocab ? p.col_scale[col] : 0.0f;
      }
      const int row = m0 + quad * 32 + lane;
      rs_next = row < p.rows ? p.row_scale[row] : 0.0f;
    };
    if (first < tiles) ask(first);
    uint32_t n = 0;
    for (int t = first; t < tiles; t += step, ++n) {
      const int acc = n & 1;
      int m0, n0;
      place(t, m0, n0);
      float cs_now[PART / 32];
#pragma unroll
      for (int i = 0; i < PART / 32; ++i) cs_now[i] = cs_next[i];
      const float rs = rs_next;
      if (t + step < tiles) ask(t + step);
      bool waited = true;
      if (lane == 0) waited = mbar_wait(&acc_full[acc], (n >> 1) & 1, WAIT_NS) && !p.give_up;
      waited = __shfl_sync(FULL, waited, 0) != 0;
      __syncwarp();  // a shuffle orders no memory
      if (!waited) {
        if (lane == 0) gave_up(p.err, 4u);
        // what is not computed reads NaN, which the sampler and the scores report
        for (; t < tiles; t += step) {
          place(t, m0, n0);
          for (int r = m0 + quad * 32; c0 < BN && r < min(m0 + quad * 32 + 32, p.rows); ++r)
            for (int col = n0 + c0 + lane; col < min(n0 + c0 + PART, p.vocab); col += 32)
              ((Tout*)p.out)[r * p.out_stride + col] = from_f<Tout>(__int_as_float(0x7fc00000));
        }
        break;
      }
      tc_fence_after();
      const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN + c0);
      const bool live = c0 < BN && m0 + quad * 32 < p.rows && n0 + c0 < p.vocab;
      auto scale_part = [&](auto tma) {
        constexpr bool by_tma = decltype(tma)::value;
#pragma unroll
        for (int g = 0; g < PART; g += CB) {
          uint32_t v[CB / 32][32];
#pragma unroll
          for (int h = 0; h < CB / 32; ++h) tmem_ld(base + (uint32_t)(g + h * 32), v[h]);
          __syncwarp();
#pragma unroll
          for (int h = 0; h < CB / 32; ++h) cs[h * 32 + lane] = cs_now[g / 32 + h];
          __syncwarp();
          tmem_wait_ld();
          if (g + CB >= PART) {  // the warp's part of the accumulator is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(map_to(smem_u32(&acc_empty[acc]), 0));
          }
          const u64 rs2 = pk2(rs, rs);
          constexpr int EP = 16 / (int)sizeof(Tout);
          uint4 w[PIECES];
#pragma unroll
          for (int h = 0; h < CB / 32; ++h) {
            to_floats(v[h]);
#pragma unroll
            for (int q = 0; q < 32 / EP; ++q) {
              float f[EP];
#pragma unroll
              for (int e = 0; e < EP; e += 4) {
                const float4 c4 = *reinterpret_cast<const float4*>(&cs[h * 32 + q * EP + e]);
                const uint32_t* a4 = &v[h][q * EP + e];
                up2(mul2(mul2(pk2(__uint_as_float(a4[0]), __uint_as_float(a4[1])), rs2), pk2(c4.x, c4.y)), f[e], f[e + 1]);
                up2(mul2(mul2(pk2(__uint_as_float(a4[2]), __uint_as_float(a4[3])), rs2), pk2(c4.z, c4.w)), f[e + 2], f[e + 3]);
              }
              w[h * 32 / EP + q] = pack<Tout>(f);
            }
          }
          if (by_tma || p.store_tma) {  // the buffer's previous contents have been read
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < PIECES; ++q)
            *reinterpret_cast<uint4*>(box + lane * (PIECES * 16) + (q ^ (lane & (PIECES - 1))) * 16) = w[q];
          if constexpr (by_tma) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (n0 + c0 + g < p.vocab) store_2d(&map_out, box, n0 + c0 + g, m0 + quad * 32);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            __syncwarp();
            const int high = min(32, p.rows - (m0 + quad * 32)), wide = min(CB, p.vocab - (n0 + c0 + g));
            Tout* dst = (Tout*)p.out + (int64_t)(m0 + quad * 32) * p.out_stride + n0 + c0 + g;
            for (int r = 0; r < high; ++r, dst += p.out_stride)
#pragma unroll
              for (int x = 0; x < CB; x += 32) {
                const int i = x + lane, in = i * (int)sizeof(Tout), piece = in / 16 ^ (r & (PIECES - 1));
                if (i < wide) dst[i] = *reinterpret_cast<const Tout*>(box + r * (PIECES * 16) + piece * 16 + in % 16);
              }
            __syncwarp();
          }
        }
      };
      if (live) {
        // two copies of the loop: chosen inside it, the way out costs every tile 1 %
        if (n0 + c0 + PART <= p.tma_ids) scale_part(std::true_type());
        else scale_part(std::false_type());
      }
      if (!live && lane == 0) arrive_at(map_to(smem_u32(&acc_empty[acc]), 0));  // nothing to read here
    }
    if (p.store_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (CG > 1) cluster_sync();  // the pair's products and arrivals are over
  if (warp == 1) {
    tc_fence_after();
    if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::COLS) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::COLS) : "memory");
  }
}

// ---------------------------------------------------------------- host side
static int esize(int32_t dtype) { return dtype == MTR_DTYPE_F32 ? 4 : 2; }

static cudaLaunchConfig_t config(dim3 grid, int threads, size_t dyn, int cluster, cudaStream_t s, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = dyn;
  cfg.stream = s;
  cfg.numAttrs = launch_attrs(attr, cluster, true);
  cfg.attrs = attr;
  return cfg;
}

static cudaError_t launch_quantize(const void* x, int64_t x_stride, int dtype, int rows, int cols, int8_t* q,
                                   int64_t q_stride, float* scale, cudaStream_t s) {
  const int es = esize(dtype), e = 16 / es;
  const bool vec = (uintptr_t)x % 16 == 0 && x_stride * es % 16 == 0 && (uintptr_t)q % e == 0 && q_stride % e == 0;
  const int64_t units = vec ? cols / e : cols;
  int per = 32;
  const bool wide = vec && units > 32 * 4;
  while (per < QUANT_THREADS && units > (int64_t)per * (wide ? 8 : 4)) per *= 2;
  const QuantParams p{x, x_stride, rows, cols, per, q, q_stride, scale};
  cudaLaunchAttribute attr[2];
  const int64_t high = QUANT_THREADS / per;
  const cudaLaunchConfig_t cfg = config(dim3((unsigned)((rows + high - 1) / high), 1, 1), QUANT_THREADS, 0, 1, s, attr);
  auto launch = [&](auto of, auto wide_of, auto single) {
    return cudaLaunchKernelEx(&cfg, wide ? wide_of : vec ? of : single, p);
  };
  switch (dtype) {
    case MTR_DTYPE_F32: return launch(quantize_kernel<float, true, 4>, quantize_kernel<float, true, 8>, quantize_kernel<float, false, 4>);
    case MTR_DTYPE_BF16:
      return launch(quantize_kernel<__nv_bfloat16, true, 4>, quantize_kernel<__nv_bfloat16, true, 8>,
                    quantize_kernel<__nv_bfloat16, false, 4>);
    default: return launch(quantize_kernel<__half, true, 4>, quantize_kernel<__half, true, 8>, quantize_kernel<__half, false, 4>);
  }
}

template <int CG, int BN, typename Tout>
static cudaError_t launch_tiles(const MtrLmHeadI8Args& a, const int8_t* q, int64_t q_stride, const float* row_scale, cudaStream_t s) {
  typedef Geo<CG, BN> G;
  CUtensorMap mh, mw, mo;
  // a tile of fewer rows than 128 copies only those that there are, in eights
  const int high = CG == 1 && a.rows < BM ? (a.rows + 7) / 8 * 8 : BM;
  if (!make_map(&mh, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, a.rows, a.d_model, q_stride, BK, high) ||
      !make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.weight, a.vocab, a.d_model, a.weight_row_stride, BK, BN / CG))
    return cudaErrorInvalidValue;
  const int es = sizeof(Tout);
  const bool tma = (uintptr_t)a.logits % 16 == 0 && a.logits_row_stride * es % 16 == 0;
  const CUtensorMapDataType type = std::is_same<Tout, float>::value           ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<Tout, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (tma) {
    if (!make_map(&mo, type, a.logits, a.rows, a.vocab, a.logits_row_stride * es, 128 / es, 32)) return cudaErrorInvalidValue;
  } else {
    mo = mw;
  }
  auto kern = lmhead_i8_kernel<CG, BN, Tout>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() {
    attr_err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G::DYN);
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  ProjParams p;
  p.row_scale = row_scale;
  p.col_scale = a.weight_scale;
  p.out = a.logits;
  p.out_stride = a.logits_row_stride;
  p.rows = a.rows;
  p.vocab = a.vocab;
  p.kblocks = (a.d_model + BK - 1) / BK;
  p.m_tiles = (a.rows + BM * CG - 1) / (BM * CG);
  p.n_tiles = (a.vocab + BN - 1) / BN;
  p.a_bytes = high * BK;
  p.store_tma = tma;
  // a last copy that ends inside the row's last 16 bytes leaves row by row instead
  p.tma_ids = !tma ? 0 : a.vocab * es % 16 == 0 ? INT32_MAX : a.vocab;
  p.err = a.error_word;
  p.give_up = test_waits();
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles, room = device_sms() / CG;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      config(dim3((unsigned)((tiles < room ? tiles : room) * CG), 1, 1), PROJ_THREADS, G::DYN, CG, s, attr);
  return cudaLaunchKernelEx(&cfg, kern, mh, mw, mo, p);
}

// The narrowest tiles that still make one round of CTAs; beyond that 128 x 256
// tiles, or pairs of CTAs on 256 x 256, which take less out of L2: pairs unless
// they need more rounds (rows that fill half of the last pair) or there are only
// one or two rounds of a short d, where a tile's start and end weigh most.
// Measured with the quantisation (us, 148 SMs; weights in L2, in the rows with two
// figures not; the rule's choice is starred):
//                         64     128    256    pair
//   128 x 768 -> 4096     6.9*   7.3    8.2    9.2      (tiles of 32: 7.1)
//   333 x 1001 -> 4099    11.8   10.2*  12.4   12.0
//   700 x 1024 -> 4096    13.2   10.8   9.1*   10.2
//   512 x 768 -> 16384    20.2   14.4   11.8*  12.5
//   512 x 4096 -> 16384                 34.4   31.5*
//   900 x 768 -> 32000                  29.0   26.7*
//   300 x 1024 -> 131072                54.0*  57.0
//   64 x 1024 -> 65536    23.1   16.1   12.3*  20.4
template <typename Tout>
static cudaError_t launch_proj(const MtrLmHeadI8Args& a, const int8_t* q, int64_t q_stride, const float* row_scale, cudaStream_t s) {
  const int64_t sms = device_sms(), m = (a.rows + BM - 1) / BM;
  auto tiles = [&](int bn) { return m * ((a.vocab + bn - 1) / bn); };
  if (tiles(64) <= sms) return launch_tiles<1, 64, Tout>(a, q, q_stride, row_scale, s);
  if (tiles(128) <= sms) return launch_tiles<1, 128, Tout>(a, q, q_stride, row_scale, s);
  const int64_t n = (a.vocab + 255) / 256, pairs = sms / 2;
  const int64_t rounds = (m * n + sms - 1) / sms, pair_rounds = ((m + 1) / 2 * n + pairs - 1) / pairs;
  // a round of pairs takes about 12/13 of the time
  if (m == 1 || 12 * pair_rounds > 13 * rounds || (rounds <= 2 && a.d_model <= 2048))
    return launch_tiles<1, 256, Tout>(a, q, q_stride, row_scale, s);
  return launch_tiles<2, 256, Tout>(a, q, q_stride, row_scale, s);
}

static bool dtype_ok(int32_t dtype) { return dtype >= MTR_DTYPE_F32 && dtype <= MTR_DTYPE_F16; }
static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
static mtr::Bytes run_of(const void* at, int64_t n) { return {at, 1, n, n}; }

}  // namespace i8

cudaError_t tc::read_gave_up_i8(uint32_t* n, cudaStream_t s) { return read_gave_up(n, s); }
}  // namespace mtr

// ---------------------------------------------------------------- C ABI
using namespace mtr::i8;

int mtr_quantize_rows_validate(const MtrQuantizeArgs* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrQuantizeArgs)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->cols < 1 || a->cols > MTR_MAX_I8_D_MODEL) return MTR_ERR_BAD_SHAPE;
  if (!dtype_ok(a->x_dtype)) return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  if (!a->x || !a->q || !a->scale) return MTR_ERR_NULL_ARG;
  if (a->x_row_stride < a->cols || a->q_row_stride < a->cols) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->x % esize(a->x_dtype) || (uintptr_t)a->scale % 4) return MTR_ERR_ALIGNMENT;
  const mtr::Bytes x = mtr::bytes_of(a->x, a->rows, a->x_row_stride, a->cols, esize(a->x_dtype));
  const mtr::Bytes q = mtr::bytes_of(a->q, a->rows, a->q_row_stride, a->cols, 1), scale = run_of(a->scale, 4ll * a->rows);
  if (overlap(x, q) || overlap(x, scale) || overlap(q, scale)) return MTR_ERR_BAD_PARAM;
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

int64_t mtr_lmhead_i8_workspace(int32_t rows, int32_t d_model, int32_t vocab) {
  if (rows <= 0 || d_model <= 0 || few_rows(rows, d_model, vocab)) return 0;
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
  const int64_t need = mtr_lmhead_i8_workspace(a->rows, a->d_model, a->vocab);
  if (!a->hidden || !a->weight || !a->weight_scale || !a->logits || (need > 0 && !a->workspace)) return MTR_ERR_NULL_ARG;
  if (a->hidden_row_stride < a->d_model || a->weight_row_stride < a->d_model || a->logits_row_stride < a->vocab)
    return MTR_ERR_BAD_SHAPE;
  if (a->workspace_bytes < need) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->hidden % esize(a->hidden_dtype) || (uintptr_t)a->weight % 16 || a->weight_row_stride % 16 ||
      (uintptr_t)a->weight_scale % 4 || (uintptr_t)a->logits % esize(a->logits_dtype) || (uintptr_t)a->workspace % 256 ||
      (uintptr_t)a->error_word % 4)
    return MTR_ERR_ALIGNMENT;
  const mtr::Bytes logits = mtr::bytes_of(a->logits, a->rows, a->logits_row_stride, a->vocab, esize(a->logits_dtype));
  const mtr::Bytes hidden = mtr::bytes_of(a->hidden, a->rows, a->hidden_row_stride, a->d_model, esize(a->hidden_dtype));
  const mtr::Bytes weight = mtr::bytes_of(a->weight, a->vocab, a->weight_row_stride, a->d_model, 1);
  const mtr::Bytes scale = run_of(a->weight_scale, 4ll * a->vocab), work = run_of(a->workspace, need);
  if (overlap(logits, hidden) || overlap(logits, weight) || overlap(logits, scale)) return MTR_ERR_BAD_PARAM;
  if (need > 0 && (overlap(logits, work) || overlap(work, hidden) || overlap(work, weight) || overlap(work, scale)))
    return MTR_ERR_BAD_PARAM;
  return MTR_OK;
}

static int lmhead_i8_launch_impl(const MtrLmHeadI8Args* a, cudaStream_t s) {
  if (few_rows(a->rows, a->d_model, a->vocab)) {
    const cudaError_t e = launch_few(*a, s);
    mtr::set_last_cuda_error((int)e);
    return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
  }
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
