// NVFP4 arithmetic shared by the quantiser, the quantising permute, the
// dequantiser and the gate/up GEMM's epilogue, so all produce the same codes
// from the same values.
//
// A value is code * scale * g: an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and the
// negatives; two per byte, the even element in the low nibble, as in
// ref_nvfp4_dequant, tests/test_reference.py:19-53), an E4M3 scale for 16
// consecutive elements, and a float32 global scale g for the tensor.
//
// Quantising a block of 16 values x, every operation rounded to fp32 once:
//   s    = e4m3(amax / (6 g))     nearest, halves to even, saturating at 448
//   inv  = 1 / (s g)              0 when s is 0
//   code = e2m1(x inv)            nearest, halves to even, saturating at 6
// The steps are the definition: a quotient that lies on a border of two codes
// (x = 0.75 s g is one for every s whose 16-bit x exists) falls to one side or
// the other by the rounding of inv, so an implementation with other steps
// would give other codes.  A block that holds an infinity or a NaN gets the
// scale NaN (0x7F) and codes of 0, so that it dequantises to NaN and is seen
// downstream.  g has to be positive, in [2^-100, 2^117]: s g and its reciprocal
// are normal fp32 numbers there (s is 2^-9 to 448), and the largest bf16 tensor,
// with g = amax / 2688, lies inside.
#pragma once

#include "common.cuh"

namespace lsek {

constexpr int kFp4Block = 16;           // elements that share a scale
constexpr uint32_t kE4m3Nan = 0x7Fu;

// What a value of the type has in its bits: the bits of +infinity.
template <typename T> struct Fp4Elem;
template <> struct Fp4Elem<__nv_bfloat16> { static constexpr uint32_t kInf = 0x7F80u; };
template <> struct Fp4Elem<__half> { static constexpr uint32_t kInf = 0x7C00u; };

__device__ __forceinline__ uint32_t e4m3_from_f32(float x) {  // saturating, NaN -> 0x7F
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(x));
  return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t code) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(code)));
  return __half2float(__ushort_as_half(static_cast<uint16_t>(h2)));
}
// Eight fp32 values -> eight E2M1 codes, value i in bits 4i .. 4i+3.
__device__ __forceinline__ uint32_t e2m1x8_from_f32(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Two E2M1 codes of a byte -> two fp32 values (exact through fp16).
__device__ __forceinline__ float2 e2m1x2_to_f32(uint32_t byte) {
  uint32_t h2;
  asm("{\n\t.reg .b8 b, z0, z1, z2;\n\t"
      "mov.b32 {b, z0, z1, z2}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
      : "=r"(h2)
      : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}

// Two fp32 products in one instruction, each rounded once.
__device__ __forceinline__ float2 mul_f32x2(float a0, float a1, float b0, float b1) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 c, a, b;\n\t"
      "mov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
  return r;
}

// Pairs of 16-bit values: |x|, the larger of two (NaN if either is), and fp32.
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b, __nv_bfloat16) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7FFF7FFFu), "r"(b & 0x7FFF7FFFu));
  return r;
}
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7FFF7FFFu), "r"(b & 0x7FFF7FFFu));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

struct Fp4Block {
  uint2 codes;     // 16 codes, element i in bits 4i of the 64
  uint32_t scale;  // E4M3 bits
};

// Quantises 16 consecutive 16-bit values (two 16-byte vectors); six_g = 6 g
// rounded to fp32.
template <typename T>
__device__ __forceinline__ Fp4Block fp4_quantize16(const uint4& lo, const uint4& hi, float g,
                                                   float six_g) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t m = max_abs2(w[0], w[1], T());
#pragma unroll
  for (int i = 2; i < 8; ++i) m = max_abs2(m, w[i], T());
  const uint32_t amax_bits = max_abs2(m, m >> 16, T()) & 0xFFFFu;
  const uint16_t ab = static_cast<uint16_t>(amax_bits);
  const float amax = Elem<T>::to_f(*reinterpret_cast<const T*>(&ab));
  Fp4Block q;
  q.scale = e4m3_from_f32(__fdiv_rn(amax, six_g));
  const float s = e4m3_to_f32(q.scale);
  const float inv = s > 0.0f ? __frcp_rn(__fmul_rn(s, g)) : 0.0f;
  uint32_t half[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = unpack2(w[4 * h + i], T());
      const float2 p = mul_f32x2(x.x, x.y, inv, inv);
      y[2 * i] = p.x;
      y[2 * i + 1] = p.y;
    }
    half[h] = e2m1x8_from_f32(y);
  }
  q.codes = make_uint2(half[0], half[1]);
  if (amax_bits >= Fp4Elem<T>::kInf) {
    q.scale = kE4m3Nan;
    q.codes = make_uint2(0u, 0u);
  }
  return q;
}

}  // namespace lsek
