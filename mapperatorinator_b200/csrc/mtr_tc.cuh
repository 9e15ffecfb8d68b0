// mtr_tc.cuh -- PTX wrappers of the tensor-core kernels (mtr_lmhead.cu: bf16
// output projection; mtr_lmhead_i8.cu, mtr_lmhead_f8.cu: 8-bit output projections):
// mbarriers with bounded waits, TMA tile loads and stores, tensor-memory loads,
// tcgen05 fences, commits and descriptors, CTA pairs.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "mtr_common.cuh"

namespace mtr {
namespace tc {

constexpr uint64_t WAIT_NS = 200000000ull;  // 200 ms: far beyond any healthy wait

// ---------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 who;\n\t"
      "elect.sync who|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// Waits for the phase with parity `ph` to complete; false after `budget_ns`
// nanoseconds (0: a single poll).  The clock is read only every 4096 polls:
// a healthy hand-off completes long before the first read.
__device__ __forceinline__ bool mbar_wait(uint32_t a, uint32_t ph, uint64_t budget_ns) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(ph)
        : "memory");
    if (done) return true;
    if (budget_ns == 0) return false;
    if ((i & 4095u) == 0u) {
      const uint64_t t = global_ns();
      if (t0 == 0) t0 = t;
      else if (t - t0 > budget_ns) return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t ph, uint64_t budget_ns) { return mbar_wait(smem_u32(b), ph, budget_ns); }
// Whether two phases have completed, polled once, by the lanes with `mine` (one of
// the warp) and without a branch: what waits finds its barriers complete more often
// than not, and a loop that the warp leaves and joins again costs it 150 clocks each.
__device__ __forceinline__ bool both_complete(bool mine, uint32_t a, uint32_t pa, uint32_t b, uint32_t pb) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred m, p, q;\n\t"
      "setp.ne.b32 m, %1, 0;\n\t"
      "setp.ne.b32 p, 0, 0;\n\t"
      "setp.ne.b32 q, 0, 0;\n\t"
      "@m mbarrier.try_wait.parity.shared::cta.b64 p, [%2], %3;\n\t"
      "@m mbarrier.try_wait.parity.shared::cta.b64 q, [%4], %5;\n\t"
      "and.pred p, p, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"((uint32_t)mine), "r"(a), "r"(pa), "r"(b), "r"(pb)
      : "memory");
  const bool any = __any_sync(FULL, ok != 0u);
  __syncwarp();  // a vote orders no memory: what the one lane has acquired, the others may read now
  return any;
}
// A value that the compiler keeps in a register: it would form a shared-memory
// address anew, from the CTA's place in the cluster, wherever it is used.
__device__ __forceinline__ uint32_t held(uint32_t v) {
  asm volatile("mov.b32 %0, %0;" : "+r"(v));
  return v;
}
__device__ __forceinline__ float load_shared(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
// Bounded waits that gave up on this device since the library was loaded (each
// translation unit has its own count; mtr_projection_timeouts adds them), and the
// bit of one in the caller's word.
static __device__ uint32_t gave_up_count;
__device__ __forceinline__ void gave_up(uint32_t* err, uint32_t bit) {
  atomicAdd(&gave_up_count, 1u);
  if (err) atomicOr(err, bit);
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) { tc_commit(smem_u32(bar)); }
// Shared-memory matrix descriptor of a K-major tile with the 128-byte swizzle:
// rows of 128 bytes, 8-row atoms 1024 bytes apart (stride byte offset), leading
// byte offset 16 (unused by this layout), descriptor version 1, layout type 2.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)(1024u >> 4) << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&v)[32]) {
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
// waits for the tensor-memory loads of the warp; what they loaded into v is not used before it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]),
                 "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                 "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29])
               :
               : "memory");
  asm volatile("" : "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// A position in a ring of barriers: its slot, and the parity of its next completion.
struct Turn {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int slots) {
    if (++slot == slots) {
      slot = 0;
      parity ^= 1;
    }
  }
};

__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// an arrival on a barrier of the cluster, at a shared::cluster address; the
// default scope orders what the barrier is for, the reads of tensor memory
// before it (a cluster-wide release waits for the warp's shared-memory and
// global stores as well: 31.7 us where this takes 27.5, 8192 x 768 -> 4096)
__device__ __forceinline__ void arrive_at(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// arrivals of the lanes with `mine` on a barrier of this CTA and on one of the cluster
__device__ __forceinline__ void arrive_both(bool mine, uint32_t here, uint32_t there) {
  asm volatile(
      "{\n\t.reg .pred m;\n\t"
      "setp.ne.b32 m, %0, 0;\n\t"
      "@m mbarrier.arrive.shared::cta.b64 _, [%1];\n\t"
      "@m mbarrier.arrive.shared::cluster.b64 _, [%2];\n\t}" ::"r"((uint32_t)mine),
      "r"(here), "r"(there)
      : "memory");
}
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// arrives on the barrier at this offset in both CTAs of the pair
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) { commit_pair(smem_u32(bar)); }
__device__ __forceinline__ void store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- host side
static inline cudaError_t read_gave_up(uint32_t* n, cudaStream_t s) {
  return cudaMemcpyFromSymbolAsync(n, gave_up_count, sizeof(*n), 0, cudaMemcpyDeviceToHost, s);
}
cudaError_t read_gave_up_i8(uint32_t* n, cudaStream_t s);  // mtr_lmhead_i8.cu's count
cudaError_t read_gave_up_f8(uint32_t* n, cudaStream_t s);  // mtr_lmhead_f8.cu's
bool test_waits();                                         // mtr_projection_test_waits

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, []() {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)f;
  });
  return fn;
}

// 2-D tensor map over a row-major [rows, cols] matrix, box of box_cols x
// box_rows, 128-byte swizzle; reads 0 outside the matrix and writes nothing
// behind the 16 bytes that its last column ends in.
inline bool make_map(CUtensorMap* m, CUtensorMapDataType type, const void* base, int64_t rows, int64_t cols, int64_t stride_bytes,
                     int box_cols, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
}  // namespace mtr
