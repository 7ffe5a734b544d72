// SwiGLU arithmetic shared by the standalone kernel and the gate/up GEMM
// epilogue, so both produce the same bits from the same 16-bit g and u.
#pragma once

#include <cuda_runtime.h>

namespace lsek {

// The clamp of ref_swiglu (tests/test_reference.py:110-125): g = min(g, L),
// u = clamp(u, -L, L), L > 0.  NaN stays NaN, as in torch.clamp, so that it is
// seen downstream; fminf and fmaxf would return the limit for it.  The second
// is one instruction: the smaller of |u| and L with the sign of u.
__device__ __forceinline__ float clamp_gate(float g, float limit) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(g), "f"(limit));
  return r;
}
__device__ __forceinline__ float clamp_up(float u, float limit) {
  float r;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(u), "f"(limit));
  return r;
}

// The clamp's limit as an operand: a swiglu_limit of 0 stands for none, which is
// a limit of infinity to the two above.  Kernels take it once, so that their
// epilogues clamp without a test (with one in each element the bf16 GEMM's took
// 1 % more at 2048 rows an expert).
__device__ __forceinline__ float clamp_limit(float swiglu_limit) {
  return swiglu_limit > 0.0f ? swiglu_limit : __int_as_float(0x7F800000);
}

// silu(g) * u in fp32; silu(g) = g / (1 + e^-g).
//
// The quotient uses the fast approximate division: an IEEE-rounded division
// costs enough instructions per element that the standalone kernel becomes
// issue-bound below the HBM stream rate (5.2 vs 6.2 TB/s at 65536 x 2048 on
// a B200).  Both __expf and __fdividef are within a few fp32 ulps of their
// exact results for the g that matter, which leaves the 16-bit result within
// one 16-bit ulp of silu(g) * u.  For g < -87 (1 + e^-g > 2^126) the quotient
// is 0 where the exact value is below 2^-120.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float s = __fdividef(g, __fadd_rn(1.0f, __expf(-g)));
  return __fmul_rn(s, u);
}

// silu(g) * u behind the clamp; `limit` from clamp_limit().
__device__ __forceinline__ float swiglu_f32(float g, float u, float limit) {
  return silu_mul(clamp_gate(g, limit), clamp_up(u, limit));
}

}  // namespace lsek
