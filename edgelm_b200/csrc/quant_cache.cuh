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

// Four numbers of a row as four codes, the first in the lowest byte.
template <int FMT>
__device__ __forceinline__ uint32_t to_codes4(float x0, float x1, float x2, float x3, float f) {
  if (f == 0.f) return 0u;
  const float y0 = __fmul_rn(x0, f), y1 = __fmul_rn(x1, f), y2 = __fmul_rn(x2, f), y3 = __fmul_rn(x3, f);
  if (FMT == QF_INT8) {
    // |y| <= 127 (1 + 2^-22): added to 1.5 2^23, whose last place is 1, it is rounded to a whole number, ties to even, and the low byte
    // of the sum is that number (a conversion to int takes the special-function unit, a quarter as many a clock)
    const float magic = 12582912.f;
    const uint32_t c0 = __float_as_uint(__fadd_rn(y0, magic)), c1 = __float_as_uint(__fadd_rn(y1, magic));
    const uint32_t c2 = __float_as_uint(__fadd_rn(y2, magic)), c3 = __float_as_uint(__fadd_rn(y3, magic));
    return __byte_perm(__byte_perm(c0, c1, 0x0040), __byte_perm(c2, c3, 0x0040), 0x5410);
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y1), "f"(y0));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y3), "f"(y2));
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
