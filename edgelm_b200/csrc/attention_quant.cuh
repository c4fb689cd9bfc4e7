// What the attention kernels over the 8-bit cache share: float16 products of codes, and the arithmetic of scores and weights.
//
// With codes a (keys) and c (values) and scales u_j, v_j:   out = sum_j p_j v_j c_j / sum_j p_j,   p_j = 2^(s_j - m),
// s_j = log2(e) scale u_j (q . a_j).  Let v_j = f_j 2^e_j, e_j the float's exponent (held to -60 at least).  The kernels keep
//     x_j = s_j + e_j,   t_j = 2^(x_j - M + 46),   M >= x_j for all j so far,
// and sum   w_j c_j  with w_j = t_j f_j 2^-32 (the operand of the product with the codes: a float16 number under 2^15), and t_j 2^-e_j
// (the same weight without its value's scale, in float32).  A weight is small beside the largest *weighted* row only, whatever the
// scales of the rows, so no scale pushes the operand out of float16's range: 2^14 keeps 28 bits below the largest weight above
// float16's smallest normal number (a key is off by 2^-39 of the largest weighted row at most, besides its operand's rounding; on tcgen05, whose M
// lags behind the largest by up to 2^8 and whose operand is t 2^-40, 2^6 to 2^14 and 2^-31), and where all rows' scales lie under 2^-60 (the format's smallest is 2^-67 or so) 11 bits are left down to
// 2^-87.  2^46 holds the other sum apart from both ends of float32: a term is at most 2^106, and rows drop out of it only where their
// scale lies 150 powers of two or more under that of a row they compete with.  Taking e_j off the float is exact and costs no
// logarithm.
//
// The queries' rows are brought to at most 2^13 by a power of two before they become float16 numbers (28 bits below a row's largest
// number survive); float32 models carry a second term, x - float16(x), of queries and weights: 22 bits.
#pragma once
#include "quant_cache.cuh"

namespace edgelm {

constexpr float AQ_LIFT = 46.f;            // t <= 2^46
// 46 - M loses bits once M is far from zero: from 2^26 on it is off by 2 and more, so that weights overflow as operands, or all vanish.  So M is
// taken off first, which is exact where it matters (next to M), and the lift added to the difference; on tcgen05, which the softmax
// bounds, x + (46 - M) is one sum while it loses no more than the scores themselves have lost, 2^-12, and goes the other way beyond.  (On
// mma.sync such a branch took the same time as the second sum, in decode 5 % more with 65,001 keys.)
constexpr float AQ_FAR = 4096.f;
constexpr float AQ_OPERAND = 2.3283064365386963e-10f;   // 2^-32: the largest weight as an operand is 2^14 to 2^15
constexpr float AQ_OPERAND_BACK = 4294967296.f;         // 2^32, for the finished sums of values
constexpr int AQ_QUERY_EXP = 12;           // a query row's largest number lies in [2^12, 2^13)
constexpr float AQ_LOG2E = 1.4426950408889634f;
constexpr long long AQ_WAIT_CYCLES = 2000000000LL;

__device__ __forceinline__ uint32_t aq_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float aq_exp2(float x) {   // 2^x on the special-function unit; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void aq_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t aq_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// the second term of a pair: what float16 left out
__device__ __forceinline__ uint32_t aq_rest(float lo, float hi, uint32_t first) {
  const float2 f = half2_to_floats(first);
  return aq_pack(lo - f.x, hi - f.y);
}
__device__ __forceinline__ uint32_t aq_transpose8(uint32_t x) {   // an 8 x 8 matrix of 16-bit values spread over the warp, transposed
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// A value's scale as f 2^e, f with the operand's 2^-32 (f keeps a NaN).
struct ValueScale {
  float e, f, undo;    // undo = 2^-e
};
__device__ __forceinline__ ValueScale value_scale(float v) {
  const int b = min(max((int)((__float_as_uint(v) >> 23) & 255u), 127 - 60), 253);
  const float undo = __uint_as_float((uint32_t)(254 - b) << 23);
  return {(float)(b - 127), v * undo * AQ_OPERAND, undo};
}

// The power of two that brings a query row with this largest magnitude into [2^12, 2^13).  (Rows that are not finite stay so; rows of
// zeros, or under 2^-100, keep a factor whose inverse is a number.)  Its inverse times the scores' scale is the row's factor, which a key's
// scale joins before the product does: scores are numbers as long as they, and that factor times that scale, are within float32.
__device__ __forceinline__ float query_lift(uint32_t largest_bits) {
  const int e = min(max((int)(largest_bits >> 23), 27), 254) - 127;    // floor(log2), held to -100 .. 127
  return __uint_as_float((uint32_t)(AQ_QUERY_EXP - e + 127) << 23);
}

// Bounded wait for a phase of an mbarrier: false once the clock says that it will not come.
__device__ __forceinline__ bool aq_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool aq_wait(uint32_t bar, uint32_t parity) {
  if (aq_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!aq_try(bar, parity))
    if (clock64() - t0 > AQ_WAIT_CYCLES) return false;
  return true;
}
__device__ __forceinline__ void aq_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

}  // namespace edgelm
