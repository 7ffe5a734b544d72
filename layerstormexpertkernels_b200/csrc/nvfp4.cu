// NVFP4 quantise, dequantise and quantising permute (arithmetic: nvfp4.cuh).
//
// All three are HBM streams: the quantiser reads 2 bytes and writes 0.5625
// bytes an element, the dequantiser the reverse, and the permute reads each
// token once and writes 0.5625 bytes an element to each of its topk rows.
// A thread's access is a block of 16 elements: 32 bytes in (one access), 8 bytes
// of codes and one scale byte out, so a warp reads 1 KB and writes 256 + 32
// bytes, all contiguous; the quantiser and the dequantiser have four blocks in
// flight a thread.  Blocks do not cross rows (the row length is a multiple of
// 16), so a contiguous tensor is one flat run of blocks.  At 16 x 4096 x 7168
// each of the two takes 184 us, 6.5 TB/s; to fp32 (four 16-byte stores 64 bytes
// apart) the dequantiser takes 497 us, 4.3 TB/s.
#include "nvfp4.cuh"

namespace lsek {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;                            // blocks a thread has in flight
constexpr int kCtaBlocks = kThreads * kUnroll;

// One block of 16 elements; VEC: the address is a multiple of 32 bytes.
template <typename T, bool VEC>
__device__ __forceinline__ void load_block(const T* p, uint4& lo, uint4& hi) {
  if (VEC) {
    ldg_nc_v8(p, lo, hi);
  } else {
    uint16_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __ldg(reinterpret_cast<const uint16_t*>(p) + i);
    auto pair = [&](int i) { return static_cast<uint32_t>(v[i]) | static_cast<uint32_t>(v[i + 1]) << 16; };
    lo = make_uint4(pair(0), pair(2), pair(4), pair(6));
    hi = make_uint4(pair(8), pair(10), pair(12), pair(14));
  }
}

// `blocks` blocks in groups of `group_blocks`, one global scale per group
// (global == null: 1).  A thread takes kUnroll blocks kThreads apart and loads
// them all before it works on the first.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                    const T* __restrict__ x, const float* __restrict__ global, int64_t blocks,
                    int64_t group_blocks) {
  const int64_t first = blockIdx.x * static_cast<int64_t>(kCtaBlocks) + threadIdx.x;
  uint4 lo[kUnroll], hi[kUnroll];
  float g[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + u * kThreads;
    if (i >= blocks) break;
    load_block<T, VEC>(x + i * kFp4Block, lo[u], hi[u]);
    g[u] = global ? __ldg(global + i / group_blocks) : 1.0f;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + u * kThreads;
    if (i >= blocks) break;
    const Fp4Block q = fp4_quantize16<T>(lo[u], hi[u], g[u], __fmul_rn(6.0f, g[u]));
    codes[i] = q.codes;
    scales[i] = static_cast<uint8_t>(q.scale);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_block(T* p, const float (&v)[16]) {
  Vec8<T> o[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i / 8].v[i % 8] = Elem<T>::from_f(v[i]);
  const uint4 lo = *reinterpret_cast<const uint4*>(&o[0]), hi = *reinterpret_cast<const uint4*>(&o[1]);
  if (VEC) {
    stg_v8(p, lo, hi);
  } else {
    reinterpret_cast<uint4*>(p)[0] = lo;
    reinterpret_cast<uint4*>(p)[1] = hi;
  }
}
template <>
__device__ __forceinline__ void store_block<float, false>(float* p, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}

// code * scale is exact in fp32 (2 + 4 significand bits); the product with g
// is rounded once, and once more to a 16-bit output type.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(T* __restrict__ out, const uint2* __restrict__ codes,
                      const uint8_t* __restrict__ scales, const float* __restrict__ global,
                      int64_t blocks, int64_t group_blocks) {
  const int64_t first = blockIdx.x * static_cast<int64_t>(kCtaBlocks) + threadIdx.x;
  uint2 c[kUnroll];
  uint32_t sc[kUnroll];
  float g[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + u * kThreads;
    if (i >= blocks) break;
    c[u] = __ldg(codes + i);
    sc[u] = __ldg(scales + i);
    g[u] = global ? __ldg(global + i / group_blocks) : 1.0f;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + u * kThreads;
    if (i >= blocks) break;
    const float s = e4m3_to_f32(sc[u]);
    float v[16];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const float2 two = e2m1x2_to_f32((b < 4 ? c[u].x : c[u].y) >> (8 * (b & 3)) & 0xFFu);
      v[2 * b] = __fmul_rn(__fmul_rn(two.x, s), g[u]);
      v[2 * b + 1] = __fmul_rn(__fmul_rn(two.y, s), g[u]);
    }
    store_block<T, VEC>(out + i * kFp4Block, v);
  }
}

// Quantises each token once and stores it to its topk rows.  Grid (T, slices
// of the row); a slice is kThreads blocks.  `zero`: `zeros` words that the
// caller wants zeroed on the way, or null.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
    permute_quantize_kernel(uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                            const __nv_bfloat16* __restrict__ hidden,
                            const int32_t* __restrict__ s2d, const float* __restrict__ global,
                            int topk, int row_blocks, int32_t* __restrict__ zero, int zeros) {
  const int64_t t = blockIdx.x;
  if (zero != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < zeros)
    zero[threadIdx.x] = 0;
  const int b = blockIdx.y * kThreads + threadIdx.x;
  if (b >= row_blocks) return;
  const float g = global ? __ldg(global) : 1.0f;
  uint4 lo, hi;
  load_block<__nv_bfloat16, VEC>(hidden + (t * row_blocks + b) * kFp4Block, lo, hi);
  const Fp4Block q = fp4_quantize16<__nv_bfloat16>(lo, hi, g, __fmul_rn(6.0f, g));
  for (int k = 0; k < topk; ++k) {
    const int64_t at = static_cast<int64_t>(__ldg(s2d + t * topk + k)) * row_blocks + b;
    codes[at] = q.codes;
    scales[at] = static_cast<uint8_t>(q.scale);
  }
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

lsek_status check_blocks(const char* name, int64_t groups, int64_t rows, int32_t k) {
  LSEK_REQUIRE(groups >= 0 && rows >= 0 && k >= 0, "%s: sizes must be >= 0", name);
  LSEK_REQUIRE(k % kFp4Block == 0, "%s: the row length must be a multiple of %d, got %d", name,
               kFp4Block, k);
  LSEK_REQUIRE(groups == 0 || rows <= (1ll << 38) / groups, "%s: too many rows", name);
  LSEK_REQUIRE(k == 0 || groups * rows <= (1ll << 38) / (k / kFp4Block),
               "%s: more than 2^38 blocks of %d", name, kFp4Block);
  return LSEK_OK;
}

template <typename T>
lsek_status quantize_t(void* codes, void* scales, const void* x, const float* global,
                       int64_t blocks, int64_t group_blocks, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(ceil_div(blocks, kCtaBlocks));
  uint2* c = static_cast<uint2*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  const T* in = static_cast<const T*>(x);
  if (aligned(x, 32))
    quantize_kernel<T, true><<<grid, kThreads, 0, st>>>(c, s, in, global, blocks, group_blocks);
  else
    quantize_kernel<T, false><<<grid, kThreads, 0, st>>>(c, s, in, global, blocks, group_blocks);
  return check_launch("nvfp4_quantize");
}

}  // namespace

// Used by moe_permute_nvfp4 and the layer forward: quantises hidden [T, H]
// into the rows that src_to_dest_map gives.
lsek_status launch_permute_quantize(void* codes, void* scales, const void* hidden,
                                    const int32_t* s2d, const float* global, int T, int topk,
                                    int H, int32_t* zero, int zeros, cudaStream_t st) {
  const int row_blocks = H / kFp4Block;
  if (T == 0 || row_blocks == 0 || topk == 0) return LSEK_OK;
  const dim3 grid(static_cast<unsigned>(T), static_cast<unsigned>(ceil_div(row_blocks, kThreads)));
  uint2* c = static_cast<uint2*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  const __nv_bfloat16* in = static_cast<const __nv_bfloat16*>(hidden);
  if (aligned(hidden, 32))
    permute_quantize_kernel<true><<<grid, kThreads, 0, st>>>(c, s, in, s2d, global, topk, row_blocks,
                                                        zero, zeros);
  else
    permute_quantize_kernel<false><<<grid, kThreads, 0, st>>>(c, s, in, s2d, global, topk, row_blocks,
                                                        zero, zeros);
  return check_launch("moe_permute_nvfp4");
}

}  // namespace lsek

extern "C" lsek_status lsek_nvfp4_quantize(void* codes, void* scales, const void* x,
                                           const float* global_scale, int64_t groups, int64_t rows,
                                           int32_t k, int32_t dtype, void* stream) {
  using namespace lsek;
  lsek_status s = check_blocks("nvfp4_quantize", groups, rows, k);
  if (s != LSEK_OK) return s;
  LSEK_REQUIRE(dtype == LSEK_BF16 || dtype == LSEK_FP16, "nvfp4_quantize: dtype must be bf16 or fp16");
  const int64_t group_blocks = rows * (k / kFp4Block), blocks = groups * group_blocks;
  if (blocks == 0) return LSEK_OK;
  LSEK_REQUIRE(codes && scales && x, "nvfp4_quantize: NULL tensor pointer");
  LSEK_REQUIRE(aligned(codes, 8) && aligned(x, 2), "nvfp4_quantize: codes must be 8-byte aligned, x 2-byte");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == LSEK_BF16
             ? quantize_t<__nv_bfloat16>(codes, scales, x, global_scale, blocks, group_blocks, st)
             : quantize_t<__half>(codes, scales, x, global_scale, blocks, group_blocks, st);
}

extern "C" lsek_status lsek_nvfp4_dequantize(void* out, const void* codes, const void* scales,
                                             const float* global_scale, int64_t groups,
                                             int64_t rows, int32_t k, int32_t dtype, void* stream) {
  using namespace lsek;
  lsek_status s = check_blocks("nvfp4_dequantize", groups, rows, k);
  if (s != LSEK_OK) return s;
  LSEK_REQUIRE(dtype == LSEK_BF16 || dtype == LSEK_FP16 || dtype == LSEK_FP32,
               "nvfp4_dequantize: dtype must be bf16, fp16 or fp32");
  const int64_t group_blocks = rows * (k / kFp4Block), blocks = groups * group_blocks;
  if (blocks == 0) return LSEK_OK;
  LSEK_REQUIRE(out && codes && scales, "nvfp4_dequantize: NULL tensor pointer");
  LSEK_REQUIRE(aligned(codes, 8) && aligned(out, 16),
               "nvfp4_dequantize: codes must be 8-byte aligned, out 16-byte");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(ceil_div(blocks, kCtaBlocks));
  const uint2* c = static_cast<const uint2*>(codes);
  const uint8_t* sc = static_cast<const uint8_t*>(scales);
  const bool vec = aligned(out, 32);
  auto run = [&](auto* o, auto kernel, auto kernel_vec) {
    (vec ? kernel_vec : kernel)<<<grid, kThreads, 0, st>>>(o, c, sc, global_scale, blocks, group_blocks);
  };
  if (dtype == LSEK_BF16)
    run(static_cast<__nv_bfloat16*>(out), dequantize_kernel<__nv_bfloat16, false>,
        dequantize_kernel<__nv_bfloat16, true>);
  else if (dtype == LSEK_FP16)
    run(static_cast<__half*>(out), dequantize_kernel<__half, false>, dequantize_kernel<__half, true>);
  else
    run(static_cast<float*>(out), dequantize_kernel<float, false>, dequantize_kernel<float, false>);
  return check_launch("nvfp4_dequantize");
}

extern "C" lsek_status lsek_moe_permute_nvfp4(void* codes, void* scales, int32_t* expert_offsets,
                                              int32_t* src_to_dest_map, int32_t* permuted_idx,
                                              const void* hidden_states,
                                              const int32_t* topk_indices,
                                              const float* global_scale, int32_t num_tokens,
                                              int32_t topk, int32_t hidden_dim,
                                              int32_t num_experts, void* stream) {
  using namespace lsek;
  LSEK_REQUIRE(num_tokens >= 0 && topk >= 0 && hidden_dim >= 0,
               "moe_permute_nvfp4: sizes must be >= 0");
  LSEK_REQUIRE(hidden_dim % kFp4Block == 0,
               "moe_permute_nvfp4: hidden_dim must be a multiple of %d, got %d", kFp4Block, hidden_dim);
  const bool empty = num_tokens == 0 || topk == 0 || hidden_dim == 0;
  if (!empty) {
    LSEK_REQUIRE(codes && scales && hidden_states, "moe_permute_nvfp4: NULL tensor pointer");
    LSEK_REQUIRE(aligned(codes, 8) && aligned(hidden_states, 2),
                 "moe_permute_nvfp4: codes must be 8-byte aligned, hidden_states 2-byte");
  }
  // The route checks the expert count, topk, the slot count and its pointers.
  const lsek_status s = lsek_moe_route(expert_offsets, src_to_dest_map, permuted_idx, topk_indices,
                                       num_tokens, topk, num_experts, stream);
  if (s != LSEK_OK || empty) return s;
  return launch_permute_quantize(codes, scales, hidden_states, src_to_dest_map, global_scale,
                                 num_tokens, topk, hidden_dim, nullptr, 0,
                                 static_cast<cudaStream_t>(stream));
}
