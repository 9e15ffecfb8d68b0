// mtr_lmhead_f8.cu -- the decoder's output projection in 8-bit floating point with a
// scale for each block of 128, on the sm_100a tensor cores.
//
// Hidden states are held as e4m3 with one fp32 scale for each row's 128 values,
// weights with one for each 128 ids x 128 values: scale = max|x| RN(1/448),
// q = e4m3(RN32(x / scale)), so with b the blocks of d
//   logits[r, v] = sum_b (scale_h[r, b] scale_w[v / 128, b]) sum_{k in b} q_h[r, k] q_w[v, k].
// The inner sums are the tensor core's, in fp32 (products of two e4m3 are exact);
// each is scaled by the two scales' product, rounded to fp32 (so it has to be in
// fp32's range: beyond 2^128 the logits are not finite, below 2^-126 they lose bits),
// and added to its logit in a register: no sum runs over more than a block.  One
// rounding to the logits' type follows.
#include <type_traits>

#include "mtr_f8.cuh"
#include "mtr_tc.cuh"

namespace mtr {
namespace f8 {

using namespace tc;

constexpr int BM = 128;  // rows of a CTA's tile
constexpr int BK = 128;  // values of one 128-byte swizzled row, and of a block
constexpr int UK = 32;   // K of one tcgen05.mma kind::f8f6f4
constexpr int QUANT_THREADS = 256;
static_assert(BK == BLOCK, "a stage is a block");

struct QuantParams {
  const void* x;
  int64_t x_stride;
  int32_t rows;
  int32_t cols;
  uint8_t* q;
  int64_t q_stride;
  float* scale;
  int64_t scale_row, scale_col;  // strides of a row's (of 128 rows') scales and of a block's
};

__device__ __forceinline__ void store4(uint8_t* q, int c, int cols, uint32_t w) {
  if (c + 4 <= cols) {
    *reinterpret_cast<uint32_t*>(q + c) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < cols) q[c + e] = (uint8_t)(w >> (8 * e));
  }
}

// A row's blocks of 128, a warp for UNITS of them: four values a lane and block.
// Fewer units where rows are few, so that there are warps for all SMs.  8192 x 4096 fp32
// 29.7 us, 5.6 TB/s, which HBM bounds; bf16 30.3, 3.3 TB/s: the same 8-byte loads a lane
// and the same work for half the bytes read.  64 x 768 bf16 1.7 us, a launch.
template <typename T, bool VEC, int UNITS>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_rows_kernel(const QuantParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks = (p.cols + BLOCK - 1) / BLOCK, runs = (blocks + UNITS - 1) / UNITS;
  wait_prior_grid();
  allow_dependents();
  const int64_t unit = (int64_t)blockIdx.x * (QUANT_THREADS / 32) + warp, row = unit / runs;
  if (row >= p.rows) return;
  const int b0 = (int)(unit % runs) * UNITS;
  const T* x = (const T*)p.x + row * p.x_stride;
  float v[UNITS][4], top[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) load4<T, VEC>(x, (b0 + i) * BLOCK + 4 * lane, p.cols, v[i]);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) top[i] = largest(magnitude(v[i]));
  // lane i has block i's scale and its reciprocal
  float mine = top[0];
#pragma unroll
  for (int i = 1; i < UNITS; ++i) mine = lane == i ? top[i] : mine;
  const i8::Divisor own = i8::divisor_of(mine, RECIPROCAL);
  if (lane < UNITS && b0 + lane < blocks) p.scale[row * p.scale_row + (b0 + lane) * p.scale_col] = own.s;
  const uint32_t flags = (own.zero ? 1u : 0u) | (own.divide ? 2u : 0u);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    i8::Divisor d;
    d.s = __shfl_sync(FULL, own.s, i);
    d.inv = __shfl_sync(FULL, own.inv, i);
    const uint32_t f = __shfl_sync(FULL, flags, i);
    d.zero = f & 1u;
    d.divide = f & 2u;
    if (b0 + i < blocks) store4(p.q + row * p.q_stride, (b0 + i) * BLOCK + 4 * lane, p.cols, quotients(v[i], d));
  }
}

// 128 rows x 128 values with one scale: a CTA each.  Weights pass here once, at load
// time, and it is not tuned: 16384 x 4096 bf16 170 us, 1.2 TB/s (16 loads and 16 stores of
// 4 values a thread, a barrier between them); 4096 x 768 13.9 us.
template <typename T, bool VEC>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_tiles_kernel(const QuantParams p) {
  __shared__ float tops[QUANT_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WARPS = QUANT_THREADS / 32, EACH = BLOCK / WARPS;
  wait_prior_grid();
  const int64_t r0 = (int64_t)blockIdx.y * BLOCK;
  const int c = (int)blockIdx.x * BLOCK + 4 * lane;
  float v[EACH][4], top = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int64_t row = r0 + warp + i * WARPS;
    if (row < p.rows) load4<T, VEC>((const T*)p.x + row * p.x_stride, c, p.cols, v[i]);
    else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) top = max_nan(top, magnitude(v[i]));
  top = largest(top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < WARPS; ++k) top = max_nan(top, tops[k]);
  const i8::Divisor d = i8::divisor_of(top, RECIPROCAL);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int64_t row = r0 + warp + i * WARPS;
    if (row < p.rows) store4(p.q + row * p.q_stride, c, p.cols, quotients(v[i], d));
  }
  if (threadIdx.x == 0) p.scale[blockIdx.y * p.scale_row + blockIdx.x * p.scale_col] = d.s;
}

struct ProjParams {
  const float* row_scale;  // [kblocks][row_pitch]
  int64_t row_pitch;
  const float* w_scale;    // [ids / 128][w_pitch]
  int64_t w_pitch;
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

// One product, operands as the low words of their shared-memory descriptors: the
// high word is the same for every tile of this layout (sw128_desc), and a stage
// or a step of K moves the low word by its bytes / 16.
template <int CG>
__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
        : "memory");
}

// Instruction descriptor of kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), A and B
// e4m3 (bits 7-9, 10-12 = 0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Tiles of 128 rows x BN vocabulary ids for one CTA (CG = 1), or of 256 rows x BN
// for a pair of CTAs (CG = 2) whose products run on both tensor cores at once, each
// CTA loading its own 128 rows and half of the ids.
//
// Persistent: a CTA (pair) takes tile after tile.  The products of a block (one
// stage, K = 128) are an accumulator of their own in tensor memory, of which there
// are NACC; the epilogue warps take one after another into registers, scaled, while
// the next blocks are multiplied.
//   warp 0, one lane   producer: TMA loads into a ring of STAGES stages
//   warp 1, one lane   issues the products (of a pair: the first CTA's only);
//                      the whole warp allocates and frees the tensor memory
//   warp 2             copies the blocks' scales into a ring of their own: a trip to
//                      L2 takes longer than a block's products
//   warps 4 ..         epilogue: warp w owns tensor memory lanes 32 (w % 4) ..,
//                      tile rows, and some of the columns, whose logits it holds
//                      in registers over the tile's blocks (128 a lane at most);
//                      at the tile's end it rounds them, stages 32 rows x 128 bytes
//                      in shared memory (16-byte pieces XOR-swizzled by row) and
//                      sends them by TMA, or row by row where rows of logits are
//                      not 16-byte aligned
// Every wait is bounded; a role whose wait gives up counts it (gave_up) and stops,
// so that the others' waits give up too; the producer then gives its copies time
// to land, the epilogue writes NaN for what was not computed, and the CTA returns.
//
// What bounds it (8192 x 4096 -> 16384: 521 .. 578 us by the clock that power leaves,
// quantisation included; clock stamps): a block takes 875 clocks, of which the tensor
// core is busy 55 %.  The epilogue's own chain of a block -- see it done 140 at least,
// read, add and hand over 470, the rest of its loop 155 -- takes 730 even where no
// product is issued, and two accumulators of 256 columns are all that tensor memory
// holds.  That chain is latency: its additions are 256 issue slots a scheduler and its
// tensor-memory reads 256 clocks, so waits and loop could give way.  Sums are scalar:
// packed ones cost a move each (750 -> 605 us with the scales' ring).  Not faster: 16 epilogue warps of 64 columns (700; no registers left), tiles of
// 128 columns and four accumulators (763), halves of a product handed over one by one
// (685: N = 128 waits for shared memory), one warp that polls for all (757).
constexpr int RING = 4;  // blocks whose scales are in shared memory

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}

template <int CG, int BN>
struct Geo {
  static constexpr int EPI = 8, THREADS = 128 + 32 * EPI;  // epilogue warps
  // Registers a thread.  384 threads have 168 each at launch; where the epilogue
  // holds 128 sums a lane the control group's four warps leave most of theirs to
  // it: 128 * 56 + 256 * 224 = 384 * 168.
  static constexpr bool SPLIT = BN == 256;
  static constexpr int LAUNCH_REGS = 168, CONTROL_REGS = 56, EPI_REGS = 224;
  static_assert(!SPLIT || 128 * CONTROL_REGS + 32 * EPI * EPI_REGS <= THREADS * LAUNCH_REGS, "registers of the launch");
  static constexpr uint32_t A_BYTES = BM * BK, B_BYTES = BN / CG * BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr uint32_t ROW_BYTES = 128;                   // of a staging buffer
  static constexpr uint32_t BOX_BYTES = 32 * ROW_BYTES;        // one epilogue warp's
  static constexpr uint32_t OUT_BYTES = EPI * BOX_BYTES;
  static constexpr uint32_t FIXED = 2816;                      // barriers, scales
  static constexpr int FIT = (int)((227 * 1024 - OUT_BYTES - FIXED) / STAGE_BYTES);
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr uint32_t DYN = STAGES * STAGE_BYTES + OUT_BYTES + FIXED;
  static constexpr int NACC = BN == 256 ? 2 : 4;
  static constexpr uint32_t COLS = NACC * BN;  // tensor-memory columns
};

template <int CG, int BN, typename Tout>
__global__ void __launch_bounds__(Geo<CG, BN>::THREADS, 1)
    lmhead_f8_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_out, const ProjParams p) {
  typedef Geo<CG, BN> G;
  constexpr int S = G::STAGES, NACC = G::NACC;
  constexpr int ROW = G::ROW_BYTES, PIECES = ROW / 16;      // bytes and 16-byte pieces of a staged row
  constexpr int CB = ROW / (int)sizeof(Tout);               // columns of a staging buffer
  constexpr int MIN_PART = CB > 32 ? CB : 32;
  constexpr int EACH = BN / (G::EPI / 4), PART = EACH < MIN_PART ? MIN_PART : EACH;  // a warp's columns
  constexpr int ACTIVE = 4 * (BN / PART);                   // warps that have some
  struct Fixed {
    uint64_t full[S], done[S], acc_empty[NACC], sc_full[RING], sc_empty[RING];
    uint32_t tmem_slot;
    __align__(16) float rows[RING][BM], ids[RING][4];  // scales of a block: of the rows, of each 128 ids
  };
  static_assert(sizeof(Fixed) <= G::FIXED, "fixed part of the shared memory");
  static_assert(BN <= 256 && BLOCK % PART == 0, "a warp's columns share a weight block");
  // the swizzle patterns of ring and staging repeat every 1024 bytes
  extern __shared__ __align__(1024) uint8_t ring[];
  Fixed& fx = *reinterpret_cast<Fixed*>(ring + (size_t)S * G::STAGE_BYTES + G::OUT_BYTES);
  uint64_t *const full = fx.full, *const done = fx.done, *const acc_empty = fx.acc_empty;

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
      mbar_init(&done[s], 1);
    }
    for (int i = 0; i < NACC; ++i) mbar_init(&acc_empty[i], ACTIVE * CG);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&fx.sc_full[i], 32);
      mbar_init(&fx.sc_empty[i], ACTIVE);
    }
  }
  if (warp == 1) {
    __syncwarp();
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

  if (warp < 4) {
    if constexpr (G::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::CONTROL_REGS));
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
          ok = wait(&done[turn.slot], turn.parity ^ 1);
          if (!ok) break;
          if (it >= early) load_ids(turn.slot, kb, n0);
          if (CG == 1) tma_load_2d(a_tile(turn.slot), &map_h, kb * BK, m0, &full[turn.slot]);
          else load_pair(a_tile(turn.slot), &map_h, kb * BK, m0, map_to(smem_u32(&full[turn.slot]), 0));
        }
      }
      // every stage is free: its copies have landed and the arrivals on its barriers are in
      for (int i = 0; ok && i < S; ++i, turn.next(S)) ok = wait(&done[turn.slot], turn.parity ^ 1);
      if (!ok) {  // copies under way get time to land before the CTA may leave
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) {
        }
      }
    } else if (warp == 1 && cta == 0) {
      // ---------------- products: the warp in step, one elected lane issues
      constexpr uint32_t idesc = idesc_f8(BM * CG, BN);
      Turn turn, acc;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (__all_sync(FULL, mbar_wait(bar, parity, WAIT_NS))) return true;
        if (lane == 0) gave_up(p.err, 2u);
        return false;
      };
      // this warp feeds the tensor core alone, a stage of products every 512
      // clocks at most: everything a stage needs is an addition to these
      const uint32_t full_at = held(smem_u32(full)), done_at = held(smem_u32(done));
      const uint32_t acc_empty_at = held(smem_u32(acc_empty));
      const uint64_t desc = sw128_desc(smem_u32(ring));
      const uint32_t lo0 = (uint32_t)desc, hi = (uint32_t)(desc >> 32);
      for (int t = first; t < tiles && ok; t += step) {
        for (int kb = 0; kb < KB; ++kb, turn.next(S), acc.next(NACC)) {
          const uint32_t a_lo = lo0 + (uint32_t)turn.slot * (G::STAGE_BYTES >> 4), b_lo = a_lo + (G::A_BYTES >> 4);
          const uint32_t full_bar = full_at + 8 * turn.slot, empty_bar = acc_empty_at + 8 * acc.slot;
          if (!both_complete(lane == 0, full_bar, turn.parity, empty_bar, acc.parity ^ 1)) {
            ok = wait(full_bar, turn.parity) && wait(empty_bar, acc.parity ^ 1);
            if (!ok) break;
          }
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / UK; ++k)
              mma_f8<CG>(tmem + acc.slot * BN, a_lo + k * (UK >> 4), b_lo + k * (UK >> 4), hi, idesc, k > 0 ? 1u : 0u);
            // the stage is free for the producer and the accumulator full for the epilogue
            if (CG == 1) tc_commit(done_at + 8 * turn.slot);
            else commit_pair(done_at + 8 * turn.slot);
          }
          __syncwarp();
        }
      }
    } else if (warp == 2) {
      // ---------------- scales: RING blocks ahead of the epilogue, past tile borders
      Turn turn;
      for (int t = first; t < tiles; t += step) {
        int m0, n0;
        place(t, m0, n0);
        // four rows a lane; behind the last row and the last id any scale does
        const float* r = p.row_scale + min(m0 + 4 * lane, (p.rows - 1) & ~3);
        const float* w = p.w_scale + (int64_t)(min(n0 + lane * BLOCK, p.vocab - 1) / BLOCK) * p.w_pitch;
        bool ok = true;
        for (int kb = 0; kb < KB; ++kb, turn.next(RING), r += p.row_pitch, ++w) {
          ok = __all_sync(FULL, mbar_wait(&fx.sc_empty[turn.slot], turn.parity ^ 1, WAIT_NS));
          if (!ok) break;
          copy_async<16>(&fx.rows[turn.slot][4 * lane], r);
          if (lane * BLOCK < BN) copy_async<4>(&fx.ids[turn.slot][lane], w);
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&fx.sc_full[turn.slot])) : "memory");
        }
        if (!ok) {
          if (lane == 0) gave_up(p.err, 1u);
          break;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    if constexpr (G::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::EPI_REGS));
    if ((warp - 4) / 4 * PART < BN) {
      const int quad = warp & 3, c0 = (warp - 4) / 4 * PART;
      uint8_t* box = ring + (size_t)S * G::STAGE_BYTES + (size_t)(warp - 4) * G::BOX_BYTES;
      constexpr int LD = 32;  // columns of a load; the next one is under way while these are added
      const uint32_t tmem_at = held(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c0);
      const uint32_t done_at = held(smem_u32(done)), empty_at = held(map_to(smem_u32(acc_empty), 0));
      const uint32_t sc_full_at = held(smem_u32(fx.sc_full)), sc_empty_at = held(smem_u32(fx.sc_empty));
      const uint32_t rows_at = held(smem_u32(&fx.rows[0][quad * 32 + lane])), ids_at = held(smem_u32(&fx.ids[0][c0 / BLOCK]));
      const bool first_lane = held(lane) == 0;
      Turn acc, sc, turn;
      bool hook = p.give_up != 0;
      for (int t = first; t < tiles; t += step) {
        int m0, n0;
        place(t, m0, n0);
        const bool live = m0 + quad * 32 < p.rows && n0 + c0 < p.vocab;
        float sum[PART];
#pragma unroll
        for (int i = 0; i < PART; ++i) sum[i] = 0.0f;
        bool waited = true;
        for (int kb = 0; kb < KB; ++kb, acc.next(NACC), sc.next(RING), turn.next(S)) {
          const uint32_t sc_bar = sc_full_at + 8 * sc.slot, done_bar = done_at + 8 * turn.slot;
          if (hook || !both_complete(first_lane, sc_bar, sc.parity, done_bar, turn.parity)) {
            if (lane == 0) waited = mbar_wait(sc_bar, sc.parity, WAIT_NS) && mbar_wait(done_bar, turn.parity, WAIT_NS) && !hook;
            hook = false;
            waited = __shfl_sync(FULL, waited, 0) != 0;
            __syncwarp();  // as in both_complete
            if (!waited) break;
          }
          tc_fence_after();
          const uint32_t base = tmem_at + (uint32_t)(acc.slot * BN);
          uint32_t v[2][LD];
          if (live) tmem_ld(base, v[0]);
          const float f = __fmul_rn(load_shared(rows_at + sc.slot * (BM * 4)), load_shared(ids_at + sc.slot * 16));
          auto release = [&]() {  // the warp's part of the accumulator is in registers
            tc_fence_before();
            __syncwarp();
            arrive_both(first_lane, sc_empty_at + 8 * sc.slot, empty_at + 8 * acc.slot);
          };
          if (live) {
#pragma unroll
            for (int g = 0; g < PART / LD; ++g) {
              uint32_t(&now)[LD] = v[g % 2];
              tmem_wait_ld(now);
              if (g + 1 == PART / LD) release();
              else tmem_ld(base + (uint32_t)((g + 1) * LD), v[(g + 1) % 2]);
#pragma unroll
              for (int i = 0; i < LD; ++i) sum[g * LD + i] = fmaf(__uint_as_float(now[i]), f, sum[g * LD + i]);
            }
          } else {
            release();  // nothing to read here
          }
        }
        if (!waited) {
          if (lane == 0) gave_up(p.err, 4u);
          // what is not computed reads NaN, which the sampler and the scores report
          for (; t < tiles; t += step) {
            place(t, m0, n0);
            for (int r = m0 + quad * 32; r < min(m0 + quad * 32 + 32, p.rows); ++r)
              for (int col = n0 + c0 + lane; col < min(n0 + c0 + PART, p.vocab); col += 32)
                ((Tout*)p.out)[r * p.out_stride + col] = from_f<Tout>(__int_as_float(0x7fc00000));
          }
          break;
        }
        if (!live) continue;
        const bool by_tma = n0 + c0 + PART <= p.tma_ids;
        auto swizzle = [](int r) { return r & 7; };  // of TMA's 128-byte pattern
#pragma unroll
        for (int g = 0; g < PART; g += CB) {
          constexpr int EP = 16 / (int)sizeof(Tout);
          uint4 w[PIECES];
#pragma unroll
          for (int q = 0; q < PIECES; ++q) {
            float f[EP];
#pragma unroll
            for (int e = 0; e < EP; ++e) f[e] = sum[g + q * EP + e];
            w[q] = pack<Tout>(f);
          }
          if (p.store_tma) {  // the buffer's previous contents have been read
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < PIECES; ++q)
            *reinterpret_cast<uint4*>(box + lane * ROW + (q ^ swizzle(lane)) * 16) = w[q];
          if (by_tma) {
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
                const int i = x + lane, in = i * (int)sizeof(Tout), piece = in / 16 ^ swizzle(r);
                if (i < wide) dst[i] = *reinterpret_cast<const Tout*>(box + r * ROW + piece * 16 + in % 16);
              }
            __syncwarp();
          }
        }
      }
      if (p.store_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
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

template <typename T>
static cudaError_t launch_quantize(const QuantParams& p, bool tiles, cudaStream_t s) {
  const bool vec = (uintptr_t)p.x % (4 * sizeof(T)) == 0 && p.x_stride % 4 == 0;
  const int64_t blocks = (p.cols + BLOCK - 1) / BLOCK;
  cudaLaunchAttribute attr[2];
  if (tiles) {
    const cudaLaunchConfig_t cfg = config(dim3((unsigned)blocks, (unsigned)((p.rows + BLOCK - 1) / BLOCK), 1), QUANT_THREADS, 0, 1, s, attr);
    return vec ? cudaLaunchKernelEx(&cfg, quantize_tiles_kernel<T, true>, p) : cudaLaunchKernelEx(&cfg, quantize_tiles_kernel<T, false>, p);
  }
  auto rows = [&](auto kern, int64_t each) {
    const int64_t units = p.rows * ((blocks + each - 1) / each), warps = QUANT_THREADS / 32;
    const cudaLaunchConfig_t cfg = config(dim3((unsigned)((units + warps - 1) / warps), 1, 1), QUANT_THREADS, 0, 1, s, attr);
    return cudaLaunchKernelEx(&cfg, kern, p);
  };
  if (p.rows * blocks < 8ll * 16 * device_sms())
    return vec ? rows(quantize_rows_kernel<T, true, 2>, 2) : rows(quantize_rows_kernel<T, false, 2>, 2);
  return vec ? rows(quantize_rows_kernel<T, true, 8>, 8) : rows(quantize_rows_kernel<T, false, 8>, 8);
}
static cudaError_t launch_quantize(const QuantParams& p, int dtype, bool tiles, cudaStream_t s) {
  switch (dtype) {
    case MTR_DTYPE_F32: return launch_quantize<float>(p, tiles, s);
    case MTR_DTYPE_BF16: return launch_quantize<__nv_bfloat16>(p, tiles, s);
    default: return launch_quantize<__half>(p, tiles, s);
  }
}

struct Held {  // the quantised hidden states, in the workspace
  uint8_t* q;
  int64_t q_stride;
  float* scale;
  int64_t pitch;
};

template <int CG, int BN, typename Tout>
static cudaError_t launch_tiles(const MtrLmHeadF8Args& a, const Held& h, cudaStream_t s) {
  typedef Geo<CG, BN> G;
  CUtensorMap mh, mw, mo;
  // a tile of fewer rows than 128 copies only those that there are, in eights
  const int high = CG == 1 && a.rows < BM ? (a.rows + 7) / 8 * 8 : BM;
  if (!make_map(&mh, CU_TENSOR_MAP_DATA_TYPE_UINT8, h.q, a.rows, a.d_model, h.q_stride, BK, high) ||
      !make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.weight, a.vocab, a.d_model, a.weight_row_stride, BK, BN / CG))
    return cudaErrorInvalidValue;
  const int es = sizeof(Tout);
  const bool tma = (uintptr_t)a.logits % 16 == 0 && a.logits_row_stride * es % 16 == 0;
  const CUtensorMapDataType type = std::is_same<Tout, float>::value           ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<Tout, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (tma) {
    if (!make_map(&mo, type, a.logits, a.rows, a.vocab, a.logits_row_stride * es, (int)G::ROW_BYTES / es, 32)) return cudaErrorInvalidValue;
  } else {
    mo = mw;
  }
  auto kern = lmhead_f8_kernel<CG, BN, Tout>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() {
    cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G::DYN);
    if (G::SPLIT && err == cudaSuccess) {  // the epilogue would wait for good for registers that the launch does not have
      cudaFuncAttributes f;
      err = cudaFuncGetAttributes(&f, kern);
      if (err == cudaSuccess && f.numRegs < G::LAUNCH_REGS) err = cudaErrorInvalidKernelImage;
    }
    attr_err[dev] = err;
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  ProjParams p;
  p.row_scale = h.scale;
  p.row_pitch = h.pitch;
  p.w_scale = a.weight_scale;
  p.w_pitch = a.scale_row_stride;
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
      config(dim3((unsigned)((tiles < room ? tiles : room) * CG), 1, 1), G::THREADS, G::DYN, CG, s, attr);
  return cudaLaunchKernelEx(&cfg, kern, mh, mw, mo, p);
}

// The narrowest tiles that still make one round of CTAs; beyond that 128 x 256
// tiles, or pairs of CTAs on 256 x 256, which take less out of L2.  Measured with the
// quantisation (us, 148 SMs, weights not in L2; bf16, the second row fp16 to fp32; the
// rule's choice is starred):
//                         64     128    256    pair
//   128 x 768 -> 4096     6.4*   7.2    8.9    9.8
//   333 x 1001 -> 4099    13.2   11.1*  16.5   17.1
//   700 x 1024 -> 4096    14.2   12.8   11.9*  13.0
//   512 x 768 -> 16384    21.2   17.0   15.7*  17.2
//   64 x 4096 -> 16384    25.8   18.9*  22.9   25.3
//   300 x 1024 -> 131072  117    73.4   65.6*  81.9
//   1024 x 2048 -> 32768  144    88.3   74.1   73.6*
//   8192 x 768 -> 4096    68.9   47.7   43.5   43.7*
template <typename Tout>
static cudaError_t launch_proj(const MtrLmHeadF8Args& a, const Held& h, cudaStream_t s) {
  const int64_t sms = device_sms(), m = (a.rows + BM - 1) / BM;
  auto tiles = [&](int bn) { return m * ((a.vocab + bn - 1) / bn); };
  if (tiles(64) <= sms) return launch_tiles<1, 64, Tout>(a, h, s);
  if (tiles(128) <= sms) return launch_tiles<1, 128, Tout>(a, h, s);
  const int64_t n = (a.vocab + 255) / 256, pairs = sms / 2;
  const int64_t rounds = (m * n + sms - 1) / sms, pair_rounds = ((m + 1) / 2 * n + pairs - 1) / pairs;
  // pairs where they need no more rounds than 13/12 of the others'; near that the two are within 3 %
  if (m == 1 || 12 * pair_rounds > 13 * rounds || (rounds <= 2 && a.d_model <= 2048)) return launch_tiles<1, 256, Tout>(a, h, s);
  return launch_tiles<2, 256, Tout>(a, h, s);
}

static bool dtype_ok(int32_t dtype) { return dtype >= MTR_DTYPE_F32 && dtype <= MTR_DTYPE_F16; }
static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
static int64_t blocks_of(int64_t n) { return (n + BLOCK - 1) / BLOCK; }
static mtr::Bytes run_of(const void* at, int64_t n) { return {at, 1, n, n}; }

}  // namespace f8

cudaError_t tc::read_gave_up_f8(uint32_t* n, cudaStream_t s) { return read_gave_up(n, s); }
}  // namespace mtr

// ---------------------------------------------------------------- C ABI
using namespace mtr::f8;

int mtr_quantize_blocks_validate(const MtrQuantizeBlocksArgs* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrQuantizeBlocksArgs)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->rows > MTR_MAX_F8_ROWS || a->cols < 1 || a->cols > MTR_MAX_F8_D_MODEL) return MTR_ERR_BAD_SHAPE;
  if (!dtype_ok(a->x_dtype) || (a->block_rows != 1 && a->block_rows != BLOCK)) return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  if (!a->x || !a->q || !a->scale) return MTR_ERR_NULL_ARG;
  const int64_t blocks = blocks_of(a->cols), scale_rows = a->block_rows == 1 ? a->rows : blocks_of(a->rows);
  if (a->x_row_stride < a->cols || a->q_row_stride < a->cols || a->scale_row_stride < blocks) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->x % esize(a->x_dtype) || (uintptr_t)a->scale % 4 || (uintptr_t)a->q % 4 || a->q_row_stride % 4) return MTR_ERR_ALIGNMENT;
  const mtr::Bytes x = mtr::bytes_of(a->x, a->rows, a->x_row_stride, a->cols, esize(a->x_dtype));
  const mtr::Bytes q = mtr::bytes_of(a->q, a->rows, a->q_row_stride, a->cols, 1);
  const mtr::Bytes scale = mtr::bytes_of(a->scale, scale_rows, a->scale_row_stride, blocks, 4);
  if (overlap(x, q) || overlap(x, scale) || overlap(q, scale)) return MTR_ERR_BAD_PARAM;
  return MTR_OK;
}

int mtr_quantize_blocks_launch(const MtrQuantizeBlocksArgs* a, void* stream) {
  const int v = mtr_quantize_blocks_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  const QuantParams p{a->x, a->x_row_stride, a->rows, a->cols, a->q, a->q_row_stride, a->scale, a->scale_row_stride, 1};
  const cudaError_t e = launch_quantize(p, a->x_dtype, a->block_rows != 1, (cudaStream_t)stream);
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}

int64_t mtr_lmhead_f8_workspace(int32_t rows, int32_t d_model, int32_t vocab) {
  if (rows <= 0 || d_model <= 0 || few_rows(rows, d_model, vocab)) return 0;
  return up((int64_t)rows * up(d_model, 16), 256) + 4ll * up(rows, 4) * blocks_of(d_model);
}

int mtr_lmhead_f8_validate(const MtrLmHeadF8Args* a) {
  if (!a) return MTR_ERR_NULL_ARG;
  if (a->abi_version != MTR_ABI_VERSION || a->struct_size != sizeof(MtrLmHeadF8Args)) return MTR_ERR_ABI;
  if (a->rows < 0 || a->rows > MTR_MAX_F8_ROWS) return MTR_ERR_BAD_SHAPE;
  if (a->d_model < 1 || a->d_model > MTR_MAX_F8_D_MODEL) return MTR_ERR_BAD_SHAPE;
  if (a->vocab < 1 || a->vocab > MTR_MAX_VOCAB) return MTR_ERR_BAD_SHAPE;
  if (!dtype_ok(a->hidden_dtype) || !dtype_ok(a->logits_dtype)) return MTR_ERR_BAD_PARAM;
  if (a->rows == 0) return MTR_OK;
  const int64_t need = mtr_lmhead_f8_workspace(a->rows, a->d_model, a->vocab), blocks = blocks_of(a->d_model);
  if (!a->hidden || !a->weight || !a->weight_scale || !a->logits || (need > 0 && !a->workspace)) return MTR_ERR_NULL_ARG;
  if (a->hidden_row_stride < a->d_model || a->weight_row_stride < a->d_model || a->logits_row_stride < a->vocab ||
      a->scale_row_stride < blocks)
    return MTR_ERR_BAD_SHAPE;
  if (a->workspace_bytes < need) return MTR_ERR_BAD_SHAPE;
  if ((uintptr_t)a->hidden % esize(a->hidden_dtype) || (uintptr_t)a->weight % 16 || a->weight_row_stride % 16 ||
      (uintptr_t)a->weight_scale % 4 || (uintptr_t)a->logits % esize(a->logits_dtype) || (uintptr_t)a->workspace % 256 ||
      (uintptr_t)a->error_word % 4)
    return MTR_ERR_ALIGNMENT;
  const mtr::Bytes logits = mtr::bytes_of(a->logits, a->rows, a->logits_row_stride, a->vocab, esize(a->logits_dtype));
  const mtr::Bytes hidden = mtr::bytes_of(a->hidden, a->rows, a->hidden_row_stride, a->d_model, esize(a->hidden_dtype));
  const mtr::Bytes weight = mtr::bytes_of(a->weight, a->vocab, a->weight_row_stride, a->d_model, 1);
  const mtr::Bytes scale = mtr::bytes_of(a->weight_scale, blocks_of(a->vocab), a->scale_row_stride, blocks, 4), work = run_of(a->workspace, need);
  if (overlap(logits, hidden) || overlap(logits, weight) || overlap(logits, scale)) return MTR_ERR_BAD_PARAM;
  if (need > 0 && (overlap(logits, work) || overlap(work, hidden) || overlap(work, weight) || overlap(work, scale)))
    return MTR_ERR_BAD_PARAM;
  return MTR_OK;
}

static int lmhead_f8_launch_impl(const MtrLmHeadF8Args* a, cudaStream_t s) {
  if (few_rows(a->rows, a->d_model, a->vocab)) {
    const cudaError_t e = launch_few(*a, s);
    mtr::set_last_cuda_error((int)e);
    return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
  }
  Held h;
  h.q = (uint8_t*)a->workspace;
  h.q_stride = up(a->d_model, 16);
  h.scale = (float*)(h.q + up(a->rows * h.q_stride, 256));
  h.pitch = up(a->rows, 4);  // a block's scales of all rows side by side, 16 bytes a lane
  const QuantParams p{a->hidden, a->hidden_row_stride, a->rows, a->d_model, h.q, h.q_stride, h.scale, 1, h.pitch};
  cudaError_t e = launch_quantize(p, a->hidden_dtype, false, s);
  if (e == cudaSuccess) {
    switch (a->logits_dtype) {
      case MTR_DTYPE_F32: e = launch_proj<float>(*a, h, s); break;
      case MTR_DTYPE_BF16: e = launch_proj<__nv_bfloat16>(*a, h, s); break;
      default: e = launch_proj<__half>(*a, h, s); break;
    }
  }
  mtr::set_last_cuda_error((int)e);
  return e == cudaSuccess ? MTR_OK : MTR_ERR_CUDA;
}

int mtr_lmhead_f8_launch(const MtrLmHeadF8Args* a, void* stream) {
  const int v = mtr_lmhead_f8_validate(a);
  if (v != MTR_OK) return v;
  if (a->rows == 0) return MTR_OK;
  return lmhead_f8_launch_impl(a, (cudaStream_t)stream);
}

int mtr_lmhead_f8_sample_launch(const MtrLmHeadF8Args* lm, const MtrSamplerArgs* sa, void* stream) {
  int v = mtr_lmhead_f8_validate(lm);
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
  v = lmhead_f8_launch_impl(lm, (cudaStream_t)stream);
  if (v != MTR_OK) return v;
  return mtr::sampler_launch(sa, (cudaStream_t)stream, true);
}
