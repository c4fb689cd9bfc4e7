// The 8-bit cache: what its rows are, how they are made, and how their codes become 16-bit floating-point operands.
//
// A row is the `hd` numbers of one token and one key/value head, keys and values apart.  With A = max(|x_i|, 2^-60):
//     scale = A / top,   code_i = round(x_i * (top / A))
// to whole numbers with ties to even (int8, top 127) or to e4m3 (fp8, top 448); the row stands for code_i * scale.  Both divisions
// and every product are single IEEE float32 operations, so that any program that follows the formula gets the same codes.  A row
// with a number that is not finite is kept as scale NaN and codes of zero: its codes stay numbers whatever it held, so that a
// weight of zero times such a row is zero, and who sees the row sees NaN.  The floor of 2^-60 keeps top / A and 1 / scale finite.
//
// Every code is exact as a float16 number (whole numbers to 127; four significant bits down to 2^-9), and the tensor cores take
// float16 operands as they take bfloat16 ones.  The attention kernels multiply codes, and apply the scales in float32: a key's to
// its scores, a value's inside the exponent (attention_quant.cuh).
#pragma once
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace edgelm {

enum : int { QF_INT8 = 0, QF_FP8 = 1 };     // formats of the C ABI
constexpr float QUANT_SMALLEST = 8.673617379884035e-19f;   // 2^-60

template <int FMT> __host__ __device__ constexpr float quant_top() { return FMT == QF_INT8 ? 127.f : 448.f; }

// |x| as an unsigned number: its order is that of the magnitudes, with infinity and then NaN above every number.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct RowScale {
  float scale, to_codes;   // to_codes 0: a row that is not finite
};
template <int FMT>
__device__ __forceinline__ RowScale row_scale(uint32_t largest_bits) {
  if (largest_bits >= 0x7f800000u) return {CUDART_NAN_F, 0.f};
  const float a = fmaxf(__uint_as_float(largest_bits), QUANT_SMALLEST);
  return {__fdiv_rn(a, quant_top<FMT>()), __fdiv_rn(quant_top<FMT>(), a)};
}

// Two products at a time, each rounded by itself.  (Sums that must not join such a product in one rounding are scalar: a packed product
// followed by a packed sum was made one multiply-add here, explicit roundings notwithstanding.)
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Four numbers of a row as four codes, the first in the lowest byte.
template <int FMT>
__device__ __forceinline__ uint32_t to_codes4(const float2& x0, const float2& x1, float f) {
  if (f == 0.f) return 0u;
  float2 y0 = mul2(x0, make_float2(f, f)), y1 = mul2(x1, make_float2(f, f));
  if (FMT == QF_INT8) {
    // |y| <= 127 (1 + 2^-22): added to 1.5 2^23, whose last place is 1, it is rounded to a whole number, ties to even, and the low byte
    // of the sum is that number (a conversion to int takes the special-function unit, a quarter as many a clock)
    const float magic = 12582912.f;
    y0 = make_float2(__fadd_rn(y0.x, magic), __fadd_rn(y0.y, magic));
    y1 = make_float2(__fadd_rn(y1.x, magic), __fadd_rn(y1.y, magic));
    return __byte_perm(__byte_perm(__float_as_uint(y0.x), __float_as_uint(y0.y), 0x0040), __byte_perm(__float_as_uint(y1.x), __float_as_uint(y1.y), 0x0040), 0x5410);
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y0.y), "f"(y0.x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y1.y), "f"(y1.x));
  return (uint32_t)lo | (uint32_t)hi << 16;
}

// The codes in the bytes of `c` as float16 pairs: (byte 0, byte 1) and (byte 2, byte 3).
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t c, uint32_t& lo, uint32_t& hi) {
  if (FMT == QF_INT8) {
    // 0x6400 + u is the float16 number 1024 + u; with u = code + 128 (the sign bit turned over), 1152 less is the code itself
    const uint32_t u = c ^ 0x80808080u;
    const __half2 off = __floats2half2_rn(1152.f, 1152.f);
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off), hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(c));
  }
}

__device__ __forceinline__ float2 half2_to_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// a cos - b sin and b cos + a sin with every product and sum rounded by itself.
__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

// Four neighbouring numbers (aligned to their size).
__device__ __forceinline__ float4 load_piece(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load_piece(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x)), hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}

}  // namespace edgelm
