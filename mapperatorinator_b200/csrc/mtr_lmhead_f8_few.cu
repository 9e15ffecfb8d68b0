// mtr_lmhead_f8_few.cu -- the output projection in 8-bit floats of few rows (one
// token of one song, or of a few), in one launch and without tensor-core tiles, 120
// of whose 128 rows would be empty.
//
// Every CTA quantises the rows into shared memory (each CTA reads them again: a few
// KB).  A warp takes 16 vocabulary ids: their weights are the first operand of
// mma.sync m16n8k32, straight from memory, 8 rows of hidden states the second, from
// shared memory.  Which k goes where in a fragment does not change the sum, so a
// lane loads 16 bytes of a weight row at once and reads the same 16 k of its hidden
// row.  A block's products are summed by the tensor core, then scaled and added in
// fp32.  The weights are read once: HBM bounds a large vocabulary, launch and two
// dependent trips to memory a small one.  Where there are fewer ids than warps a
// group's blocks are dealt to SPLIT warps, whose sums are joined in a fixed order.
#include "mtr_f8.cuh"

namespace mtr {
namespace f8 {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int CTAS = 2;           // an SM
constexpr int ROWS = 8;           // of a fragment

struct FewParams {
  const void* x;
  int64_t x_stride;
  const uint8_t* weight;
  int64_t w_stride;
  const float* w_scale;
  int64_t ws_stride;
  void* out;
  int64_t out_stride;
  int32_t x_dtype, out_dtype;
  int32_t rows, d, blocks;
  int32_t vocab;
  int32_t vec;  // rows of x allow loads of four values
};

// bytes between hidden rows: two neighbours' 64 bytes of a fragment load lie in different halves of the banks
__host__ __device__ constexpr int row_bytes(int blocks) { return blocks * BLOCK + 64; }

// The rows' blocks, a warp each.  (In the place of rows that are not there the products
// take the last one, whose sums there nobody reads.)
template <typename T, bool VEC>
__device__ __forceinline__ void hold_rows(const FewParams& p, uint8_t* held, float* scale) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, units = p.rows * p.blocks;
  constexpr int U = 4;  // blocks under way
  for (int u0 = warp; u0 < units; u0 += WARPS * U) {
    float v[U][4];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = u0 + i * WARPS, r = u / p.blocks, b = u - r * p.blocks;
      if (u < units) load4<T, VEC>((const T*)p.x + r * p.x_stride, b * BLOCK + 4 * lane, p.d, v[i]);
      else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = u0 + i * WARPS, r = u / p.blocks, b = u - r * p.blocks;
      if (u < units) {
        const i8::Divisor d = i8::divisor_of(largest(magnitude(v[i])), RECIPROCAL);
        *reinterpret_cast<uint32_t*>(held + r * row_bytes(p.blocks) + b * BLOCK + 4 * lane) = quotients(v[i], d);
        if (lane == 0) scale[b * ROWS + r] = d.s;
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ void hold_rows(const FewParams& p, uint8_t* held, float* scale) {
  if (p.vec) hold_rows<T, true>(p, held, scale);
  else hold_rows<T, false>(p, held, scale);
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int SPLIT>
__global__ void __launch_bounds__(THREADS, CTAS) few_rows_kernel(const FewParams p) {
  constexpr int GP = WARPS / SPLIT;
  extern __shared__ __align__(16) uint8_t held[];
  __shared__ float joined[SPLIT > 1 ? WARPS : 1][SPLIT > 1 ? 4 * 32 : 1];
  float* scale = reinterpret_cast<float*>(held + p.rows * row_bytes(p.blocks));  // [blocks][ROWS]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % SPLIT, sub = warp / SPLIT;
  const int KB = p.blocks, V = p.vocab, groups = (V + 15) / 16;
  const int g = lane >> 2, t = lane & 3;
  wait_prior_grid();

  // two blocks, kb and kb + SPLIT, of a group's ids g and g + 8: 16 bytes at 16 t and at 64 + 16 t of each
  auto load = [&](uint4 (&w)[2][4], int group, int kb) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int id = min(group * 16 + g + (q & 1) * 8, V - 1), b = kb + i * SPLIT, k = b * BLOCK + (q >> 1) * 64 + 16 * t;
        const uint8_t* at = p.weight + id * p.w_stride + k;
        w[i][q] = make_uint4(0u, 0u, 0u, 0u);
        if (b < KB && k + 16 <= p.d) {
          w[i][q] = *reinterpret_cast<const uint4*>(at);
        } else if (b < KB && k < p.d) {  // the last bytes of d; what lies behind them is not read
          uint32_t word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int c = 0; c < 16; ++c)
            if (k + c < p.d) word[c / 4] |= (uint32_t)at[c] << (c % 4 * 8);
          w[i][q] = make_uint4(word[0], word[1], word[2], word[3]);
        }
      }
  };
  const int step = gridDim.x * GP;
  uint4 next[2][4];
  if ((int)blockIdx.x * GP + sub < groups) load(next, blockIdx.x * GP + sub, part);
  switch (p.x_dtype) {
    case MTR_DTYPE_F32: hold_rows<float>(p, held, scale); break;
    case MTR_DTYPE_BF16: hold_rows<__nv_bfloat16>(p, held, scale); break;
    default: hold_rows<__half>(p, held, scale); break;
  }
  __syncthreads();

  for (int base = blockIdx.x * GP; base < groups; base += step) {
    const int group = base + sub;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (group < groups) {
      const float* ws = p.w_scale + (int64_t)(group / 8) * p.ws_stride;
      for (int kb = part; kb < KB; kb += 2 * SPLIT) {
        uint4 w[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) w[i][q] = next[i][q];
        const float s0 = ws[kb], s1 = kb + SPLIT < KB ? ws[kb + SPLIT] : 0.0f;
        const bool more = kb + 2 * SPLIT < KB;
        if (more) load(next, group, kb + 2 * SPLIT);
        else if (group + step < groups) load(next, group + step, part);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int b = kb + i * SPLIT;
          if (b >= KB) break;
          const uint8_t* h = held + min(g, p.rows - 1) * row_bytes(KB) + b * BLOCK + 16 * t;
          const uint4 h0 = *reinterpret_cast<const uint4*>(h), h1 = *reinterpret_cast<const uint4*>(h + 64);
          float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma(c, w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, h0.x, h0.y);
          mma(c, w[i][0].z, w[i][1].z, w[i][0].w, w[i][1].w, h0.z, h0.w);
          mma(c, w[i][2].x, w[i][3].x, w[i][2].y, w[i][3].y, h1.x, h1.y);
          mma(c, w[i][2].z, w[i][3].z, w[i][2].w, w[i][3].w, h1.z, h1.w);
          const float2 hs = *reinterpret_cast<const float2*>(scale + b * ROWS + 2 * t);
          const float f0 = __fmul_rn(hs.x, i ? s1 : s0), f1 = __fmul_rn(hs.y, i ? s1 : s0);
          acc[0] = fmaf(c[0], f0, acc[0]);
          acc[1] = fmaf(c[1], f1, acc[1]);
          acc[2] = fmaf(c[2], f0, acc[2]);
          acc[3] = fmaf(c[3], f1, acc[3]);
        }
      }
    }
    if constexpr (SPLIT > 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) joined[warp][e * 32 + lane] = acc[e];
      __syncthreads();
      if (part == 0)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 1; k < SPLIT; ++k) acc[e] += joined[warp + k][e * 32 + lane];
    }
    if (part == 0 && group < groups) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 2 * t + (e & 1), v = group * 16 + g + (e >> 1) * 8;
        if (r < p.rows && v < V) {
          const int64_t at = r * p.out_stride + v;
          switch (p.out_dtype) {
            case MTR_DTYPE_F32: ((float*)p.out)[at] = acc[e]; break;
            case MTR_DTYPE_BF16: ((__nv_bfloat16*)p.out)[at] = from_f<__nv_bfloat16>(acc[e]); break;
            default: ((__half*)p.out)[at] = from_f<__half>(acc[e]); break;
          }
        }
      }
    }
    if (SPLIT > 1) __syncthreads();  // the parts have been read
  }
}

template <int SPLIT>
cudaError_t launch_split(const FewParams& p, cudaStream_t s) {
  const int64_t groups = (p.vocab + 15) / 16, all = (groups * SPLIT + WARPS - 1) / WARPS, room = (int64_t)CTAS * device_sms();
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(all < room ? all : room), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = (size_t)(p.rows * row_bytes(p.blocks) + p.blocks * ROWS * 4);  // few_rows: 48 blocks, 8.2 KB at most
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = launch_attrs(attr, 1, true);
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, few_rows_kernel<SPLIT>, p);
}

cudaError_t launch_rows(const FewParams& p, cudaStream_t s) {
  const int64_t groups = (p.vocab + 15) / 16, warps = (int64_t)CTAS * device_sms() * WARPS;
  int split = 1;
  while (split < 8 && groups * split * 2 <= warps && split * 2 <= p.blocks) split *= 2;
  switch (split) {
    case 1: return launch_split<1>(p, s);
    case 2: return launch_split<2>(p, s);
    case 4: return launch_split<4>(p, s);
    default: return launch_split<8>(p, s);
  }
}

}  // namespace

// Where this kernel is the faster one: every CTA quantises all rows, so their blocks
// must be few, the fewer the more the vocabulary's own time weighs.  us with weights
// that are not in L2, here / there (148 SMs): 1 x 768 -> 4096 3.5 / 6.1, 2 x 768 -> 4096
// 3.7 / 6.2, 8 x 768 -> 4096 5.8 / 6.9; at the bound 8 x 300 -> 65536 12.3 / 11.8 and 1 x
// 1024 -> 65536 17.6 / 17.1, within 4 % and without a workspace; and beyond it 4 x 1024 ->
// 65536 18.9 / 17.2, 1 x 4096 -> 16384 18.4 / 17.6, 1 x 4096 -> 131072 101 / 90, 8 x 4096 ->
// 131072 119 / 91.  Large weights are far from their bytes on either side (1 x 4096 ->
// 16384 10.2, 1 x 1024 -> 65536 10.2, 8 x 300 -> 65536 3.2): here whole groups are dealt to
// warps, 4096 to 2368 in the second case, so that some have two and most one, and a step
// is two blocks where a row may have three; there 120 and more of a tile's 128 rows are
// empty, behind a launch of its own that quantises.
bool few_rows(int64_t rows, int64_t d, int64_t vocab) {
  const int64_t blocks = (d + BLOCK - 1) / BLOCK;
  return rows <= ROWS && rows * blocks <= (vocab <= 8192 ? 48 : 24);
}

cudaError_t launch_few(const MtrLmHeadF8Args& a, cudaStream_t s) {
  FewParams p;
  p.x = a.hidden;
  p.x_stride = a.hidden_row_stride;
  p.weight = (const uint8_t*)a.weight;
  p.w_stride = a.weight_row_stride;
  p.w_scale = a.weight_scale;
  p.ws_stride = a.scale_row_stride;
  p.out = a.logits;
  p.out_stride = a.logits_row_stride;
  p.x_dtype = a.hidden_dtype;
  p.out_dtype = a.logits_dtype;
  p.rows = a.rows;
  p.d = a.d_model;
  p.blocks = (a.d_model + BLOCK - 1) / BLOCK;
  p.vocab = a.vocab;
  const int es = a.hidden_dtype == MTR_DTYPE_F32 ? 4 : 2;
  p.vec = (uintptr_t)a.hidden % (4 * es) == 0 && a.hidden_row_stride % 4 == 0;
  return launch_rows(p, s);
}

}  // namespace f8
}  // namespace mtr
