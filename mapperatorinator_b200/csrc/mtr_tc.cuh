// mtr_tc.cuh -- PTX wrappers of the tensor-core kernels (mtr_lmhead.cu: bf16
// output projection; mtr_lmhead_i8.cu: 8-bit output projection): mbarriers with
// bounded waits, TMA tile loads, tcgen05 fences, commits and descriptors.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "mtr_common.cuh"

namespace mtr {
namespace tc {

constexpr uint64_t WAIT_NS = 200000000ull;  // 200 ms: far beyond any healthy wait

// ---------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

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
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t ph, uint64_t budget_ns) {
  const uint32_t a = smem_u32(b);
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
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// Shared-memory matrix descriptor of a K-major tile with the 128-byte swizzle:
// rows of 128 bytes, 8-row atoms 1024 bytes apart (stride byte offset), leading
// byte offset 16 (unused by this layout), descriptor version 1, layout type 2.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)(1024u >> 4) << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

// ---------------------------------------------------------------- host side
static inline cudaError_t read_gave_up(uint32_t* n, cudaStream_t s) {
  return cudaMemcpyFromSymbolAsync(n, gave_up_count, sizeof(*n), 0, cudaMemcpyDeviceToHost, s);
}
cudaError_t read_gave_up_i8(uint32_t* n, cudaStream_t s);  // mtr_lmhead_i8.cu's count
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

}  // namespace tc
}  // namespace mtr
