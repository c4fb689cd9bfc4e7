// Writing the 8-bit cache and reading it back (the format: quant_cache.cuh).
//
//   rope_quantize_append   a step's queries rotated (in place, or to rows of their own); its keys rotated and its values as they are,
//                          each row as codes and a scale into its page.  A row is held by hd / 16 neighbouring lanes (rounded up to a
//                          power of two), each with eight numbers of the row's first half and their partners of the second: the
//                          rotation needs no exchange, the row's largest magnitude log2(lanes) shuffles, and all reads and writes
//                          are pieces of 8 numbers.
//   quantized_rows         rows of given tokens as numbers, 16 codes a lane.
//
// Where there are many tokens nothing is saturated (append: DRAM 41 %, issue slots 56 %, occupancy 41 % at 64 registers): a lane waits in the
// chain position -> sequence -> slot -> page -> row that it walks before it may write (or read) a row.  So a warp stays with one token,
// walks the chain once, and has two pieces a lane on their way at a time.  With few tokens a lane has one piece, so that the token is spread over more warps.
// 8,407 tokens of 32 query and 64 kept rows of 64, bfloat16 to int8: 41 us for 174 MB (4.2 TB/s, with the rotation and rounding in 56 % of the
// issue slots), read back 25 us for 105 MB; float32 rows 63 us for 312 MB (5.0 TB/s); eight sequences of 1 to 3 tokens (9 and 6 rows) 2.4 and 2.1 us.
#include <type_traits>

#include "quant_cache.cuh"

namespace edgelm {

constexpr int QA_THREADS = 256;
constexpr int QA_MANY_PIECES = 2;
constexpr int QA_MANY_TOKENS = 64;    // from here on QA_MANY_PIECES pieces a lane

// Eight neighbouring numbers as they are stored.
template <typename T> struct Piece8;
template <> struct Piece8<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float2 (&x)[4]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
template <> struct Piece8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float2 (&x)[4]) const {
    x[0] = make_float2(a.x, a.y);
    x[1] = make_float2(a.z, a.w);
    x[2] = make_float2(b.x, b.y);
    x[3] = make_float2(b.z, b.w);
  }
};
__device__ __forceinline__ void store8(float* p, const float2 (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float2 (&x)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[i].x, x[i].y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// the larger, or NaN if either is none
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The page of a token's position, or -1 (reported by one lane).
__device__ __forceinline__ int page_of_token(int pos, int max_pos, int seq, const int32_t* seq_slot, const int32_t* page_table, int table_stride,
                                             int n_pages, bool report, int* err) {
  if (pos < 0 || pos >= max_pos) {
    if (report) atomicOr(err, ERR_POSITION_RANGE);
    return -1;
  }
  const int page = pos / PAGE < table_stride ? page_table[(size_t)seq_slot[seq] * table_stride + pos / PAGE] : -1;
  if (page < 0 || page >= n_pages) {
    if (report) atomicOr(err, ERR_PAGE_RANGE);
    return -1;
  }
  return page;
}

template <typename T, int FMT, int LANES, int PIECES>   // LANES: lanes of a row (a power of two, at least hd / 16); PIECES a lane
__global__ void __launch_bounds__(QA_THREADS, sizeof(T) == 2 ? 4 : 3)
rope_quantize_append_kernel(T* __restrict__ qkv, T* __restrict__ q_out, const int32_t* __restrict__ tok_pos, const int32_t* __restrict__ tok_seq,
                            const int32_t* __restrict__ seq_slot, const int32_t* __restrict__ page_table, int table_stride, int n_pages,
                            const float* __restrict__ cos_t, const float* __restrict__ sin_t, int max_pos, uint8_t* __restrict__ kcache,
                            uint8_t* __restrict__ vcache, float* __restrict__ k_scale, float* __restrict__ v_scale, int n_tokens, int nh,
                            int nkv, int hd, int warps_per_token, int* __restrict__ err) {
  constexpr int ROWS = 32 / LANES;      // of a warp at a time
  pdl_launch_dependents();
  pdl_wait();   // (launched as a programmatic dependent: the projections are the kernel before this one's)
  const int rows = nh + 2 * nkv, half = hd >> 1, lane = threadIdx.x & 31, part = lane % LANES, j = part * 8;
  const int warp = blockIdx.x * (QA_THREADS / 32) + (threadIdx.x >> 5);
  const int t = warp / warps_per_token, chunk = warp - t * warps_per_token;
  if (t >= n_tokens) return;            // (whole warps)
  const int row0 = chunk * ROWS * PIECES + lane / LANES;
  T* src = qkv + (size_t)t * rows * hd + j;
  Piece8<T> lo[PIECES], hi[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int r = row0 + i * ROWS;
    if (r < rows && j < half) {
      lo[i].load(src + (size_t)r * hd);
      hi[i].load(src + (size_t)r * hd + half);
    }
  }
  const int pos = tok_pos[t];
  const int page = page_of_token(pos, max_pos, tok_seq[t], seq_slot, page_table, table_stride, n_pages, lane == 0 && chunk == 0, err);
  if (page < 0) return;                 // (whole warps: the token is the warp's)
  float2 cs[4], sn[4];
  if (j < half) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const float4 c = *reinterpret_cast<const float4*>(cos_t + (size_t)pos * half + j + 2 * k), s = *reinterpret_cast<const float4*>(sin_t + (size_t)pos * half + j + 2 * k);
      cs[k] = make_float2(c.x, c.y);
      cs[k + 1] = make_float2(c.z, c.w);
      sn[k] = make_float2(s.x, s.y);
      sn[k + 1] = make_float2(s.z, s.w);
    }
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int r = row0 + i * ROWS;
    const bool mine = r < rows && j < half;
    float2 a[4] = {}, b[4] = {};
    if (mine) {
      lo[i].get(a);
      hi[i].get(b);
      if (r < nh + nkv) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {   // a c - b s, b c + a s, every product and sum rounded by itself
          const float2 ac = mul2(a[k], cs[k]), bs = mul2(b[k], sn[k]), bc = mul2(b[k], cs[k]), as = mul2(a[k], sn[k]);
          a[k] = make_float2(__fsub_rn(ac.x, bs.x), __fsub_rn(ac.y, bs.y));
          b[k] = make_float2(__fadd_rn(bc.x, as.x), __fadd_rn(bc.y, as.y));
        }
      }
    }
    float most = 0.f;
    if (row0 - lane / LANES + (i + 1) * ROWS > nh) {      // (the warp has rows that are kept)
#pragma unroll
      for (int k = 0; k < 4; ++k) most = max_or_nan(max_or_nan(most, max_or_nan(fabsf(a[k].x), fabsf(a[k].y))), max_or_nan(fabsf(b[k].x), fabsf(b[k].y)));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    if (!mine) continue;
    if (r < nh) {
      T* dst = q_out ? q_out + ((size_t)t * nh + r) * hd + j : src + (size_t)r * hd;
      store8(dst, a);
      store8(dst + half, b);
      continue;
    }
    const RowScale rs = row_scale<FMT>(__float_as_uint(most));
    const bool is_v = r >= nh + nkv;
    const size_t at = ((size_t)page * nkv + (is_v ? r - nh - nkv : r - nh)) * PAGE + pos % PAGE;
    uint8_t* codes = (is_v ? vcache : kcache) + at * hd + j;
    *reinterpret_cast<uint2*>(codes) = make_uint2(to_codes4<FMT>(a[0], a[1], rs.to_codes), to_codes4<FMT>(a[2], a[3], rs.to_codes));
    *reinterpret_cast<uint2*>(codes + half) = make_uint2(to_codes4<FMT>(b[0], b[1], rs.to_codes), to_codes4<FMT>(b[2], b[3], rs.to_codes));
    if (part == 0) (is_v ? v_scale : k_scale)[at] = rs.scale;
  }
}

// keys[t], values[t] [nkv, hd] = the numbers that the cache holds for token t; a lane 16 of a row's at a time.
template <typename T, int FMT, int PIECES>
__global__ void __launch_bounds__(QA_THREADS, 6)
quantized_rows_kernel(const uint8_t* __restrict__ kcache, const uint8_t* __restrict__ vcache, const float* __restrict__ k_scale,
                      const float* __restrict__ v_scale, const int32_t* __restrict__ tok_pos, const int32_t* __restrict__ tok_seq,
                      const int32_t* __restrict__ seq_slot, const int32_t* __restrict__ page_table, int table_stride, int n_pages,
                      T* __restrict__ keys, T* __restrict__ values, int n_tokens, int nkv, int hd, int warps_per_token, int* __restrict__ err) {
  pdl_launch_dependents();
  pdl_wait();
  const int per_row = hd >> 4, per_token = 2 * nkv * per_row, lane = threadIdx.x & 31;
  const int warp = blockIdx.x * (QA_THREADS / 32) + (threadIdx.x >> 5);
  const int t = warp / warps_per_token, chunk = warp - t * warps_per_token;
  if (t >= n_tokens) return;
  const int pos = tok_pos[t];
  const int page = page_of_token(pos, 0x7fffffff, tok_seq[t], seq_slot, page_table, table_stride, n_pages, lane == 0 && chunk == 0, err);
  const size_t first = ((size_t)max(page, 0) * nkv) * PAGE + max(pos, 0) % PAGE;
  uint4 c[PIECES];
  float scale[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int it = (chunk * PIECES + i) * 32 + lane, row = it / per_row, d = (it - row * per_row) * 16;
    c[i] = make_uint4(0, 0, 0, 0);
    scale[i] = 0.f;                     // (a token that the cache cannot hold: zeros, and the error word says so)
    if (it < per_token && page >= 0) {
      const bool is_v = row >= nkv;
      const size_t at = first + (size_t)(is_v ? row - nkv : row) * PAGE;
      c[i] = *reinterpret_cast<const uint4*>((is_v ? vcache : kcache) + at * hd + d);
      scale[i] = (is_v ? v_scale : k_scale)[at];
    }
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int it = (chunk * PIECES + i) * 32 + lane, row = it / per_row, d = (it - row * per_row) * 16;
    if (it >= per_token) break;
    const bool is_v = row >= nkv;
    T* dst = (is_v ? values : keys) + ((size_t)t * nkv + (is_v ? row - nkv : row)) * hd + d;
    const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float2 x[4] = {};
      if (page >= 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t p0, p1;
          codes_to_half<FMT>(w[2 * h + k], p0, p1);
          const float2 s = make_float2(scale[i], scale[i]);
          x[2 * k] = mul2(half2_to_floats(p0), s);
          x[2 * k + 1] = mul2(half2_to_floats(p1), s);
        }
      }
      store8(dst + 8 * h, x);
    }
  }
}

template <typename T, int FMT>
static void launch_append(const void* qkv, void* q_out, const int32_t* tok_pos, const int32_t* tok_seq, const int32_t* seq_slot, const int32_t* page_table,
                          int table_stride, int n_pages, const float* cos_t, const float* sin_t, int max_pos, void* kc, void* vc, float* ks,
                          float* vs, int n_tokens, int nh, int nkv, int hd, int* err, cudaStream_t stream) {
  const bool many = n_tokens >= QA_MANY_TOKENS;
  auto go = [&](auto kern, int lanes) {
    const int per_warp = 32 / lanes * (many ? QA_MANY_PIECES : 1), warps = (nh + 2 * nkv + per_warp - 1) / per_warp;
    launch_pdl(pdl_bit_for_tokens(n_tokens), kern, dim3((unsigned)(((long long)n_tokens * warps + QA_THREADS / 32 - 1) / (QA_THREADS / 32))), dim3(QA_THREADS),
               (size_t)0, stream, (T*)const_cast<void*>(qkv), (T*)q_out, tok_pos, tok_seq, seq_slot, page_table, table_stride, n_pages, cos_t, sin_t, max_pos,
               (uint8_t*)kc, (uint8_t*)vc, ks, vs, n_tokens, nh, nkv, hd, warps, err);
  };
  auto lanes = [&](auto n) {
    constexpr int L = decltype(n)::value;
    many ? go(rope_quantize_append_kernel<T, FMT, L, QA_MANY_PIECES>, L) : go(rope_quantize_append_kernel<T, FMT, L, 1>, L);
  };
  if (hd <= 16) lanes(std::integral_constant<int, 1>{});
  else if (hd <= 32) lanes(std::integral_constant<int, 2>{});
  else if (hd <= 64) lanes(std::integral_constant<int, 4>{});
  else if (hd <= 128) lanes(std::integral_constant<int, 8>{});
  else lanes(std::integral_constant<int, 16>{});
}

}  // namespace edgelm

using namespace edgelm;

// The entry points of the 8-bit cache take their arguments as one struct: their callers make a call a layer and token, and packing a struct
// takes a sixth of the time that converting thirty arguments one by one does (0.4 against 1.9 us in Python).  8-byte fields first.
struct QuantAppendCall {
  void *qkv, *q_out;                                        // q_out: rows [n_tokens, nh hd] for the rotated queries, or null: back in place
  const int32_t *tok_pos, *tok_seq, *seq_slot, *page_table;
  const float *cos_t, *sin_t;
  void *kcache, *vcache;
  float *k_scale, *v_scale;
  int* err;
  cudaStream_t stream;
  int dtype, format, table_stride, n_pages, max_pos, n_tokens, nh, nkv, hd;
};

extern "C" int edgelm_rope_quantize_append(const QuantAppendCall* call) {
  const QuantAppendCall& c = *call;
  if (c.n_tokens == 0) return 0;
  EL_REFUSE(c.n_tokens > 0 && c.nh > 0 && c.nkv > 0, "rope_quantize_append: bad sizes");
  EL_REFUSE(c.hd >= 16 && c.hd <= 256 && c.hd % 16 == 0, "rope_quantize_append: head size %d (takes 16..256 in steps of 16)", c.hd);
  EL_REFUSE((c.format == QF_INT8 || c.format == QF_FP8) && (c.dtype == DT_F32 || c.dtype == DT_BF16), "rope_quantize_append: format %d, dtype %d", c.format, c.dtype);
  EL_REFUSE((uintptr_t)c.qkv % 16 == 0 && (uintptr_t)c.q_out % 16 == 0 && (uintptr_t)c.cos_t % 16 == 0 && (uintptr_t)c.sin_t % 16 == 0 &&
                (uintptr_t)c.kcache % 16 == 0 && (uintptr_t)c.vcache % 16 == 0,
            "rope_quantize_append: rows must start on 16-byte boundaries");
  EL_REFUSE((long long)c.n_tokens * (c.nh + 2 * c.nkv) < 0x7fffffffLL, "rope_quantize_append: grid too large");
  auto go = [&](auto fn) { fn(c.qkv, c.q_out, c.tok_pos, c.tok_seq, c.seq_slot, c.page_table, c.table_stride, c.n_pages, c.cos_t, c.sin_t, c.max_pos, c.kcache,
                              c.vcache, c.k_scale, c.v_scale, c.n_tokens, c.nh, c.nkv, c.hd, c.err, c.stream); };
  if (c.dtype == DT_F32) c.format == QF_INT8 ? go(launch_append<float, QF_INT8>) : go(launch_append<float, QF_FP8>);
  else c.format == QF_INT8 ? go(launch_append<__nv_bfloat16, QF_INT8>) : go(launch_append<__nv_bfloat16, QF_FP8>);
  EL_LAUNCH_CHECK("rope_quantize_append");
  return 0;
}

struct QuantRowsCall {
  const void *kcache, *vcache;
  const float *k_scale, *v_scale;
  const int32_t *tok_pos, *tok_seq, *seq_slot, *page_table;
  void *keys, *values;
  int* err;
  cudaStream_t stream;
  int format, dtype, table_stride, n_pages, n_tokens, nkv, hd;
};

extern "C" int edgelm_quantized_rows(const QuantRowsCall* call) {
  const QuantRowsCall& c = *call;
  if (c.n_tokens == 0) return 0;
  EL_REFUSE(c.n_tokens > 0 && c.nkv > 0, "quantized_rows: bad sizes");
  EL_REFUSE(c.hd >= 16 && c.hd <= 256 && c.hd % 16 == 0, "quantized_rows: head size %d (takes 16..256 in steps of 16)", c.hd);
  EL_REFUSE((c.format == QF_INT8 || c.format == QF_FP8) && (c.dtype == DT_F32 || c.dtype == DT_BF16), "quantized_rows: format %d, dtype %d", c.format, c.dtype);
  EL_REFUSE((uintptr_t)c.keys % 16 == 0 && (uintptr_t)c.values % 16 == 0 && (uintptr_t)c.kcache % 16 == 0 && (uintptr_t)c.vcache % 16 == 0,
            "quantized_rows: rows must start on 16-byte boundaries");
  EL_REFUSE((long long)c.n_tokens * 2 * c.nkv < 0x7fffffffLL, "quantized_rows: grid too large");
  const bool many = c.n_tokens >= QA_MANY_TOKENS;
  const int per_warp = 32 * (many ? QA_MANY_PIECES : 1), warps = (2 * c.nkv * (c.hd / 16) + per_warp - 1) / per_warp;
  const dim3 grid((unsigned)(((long long)c.n_tokens * warps + QA_THREADS / 32 - 1) / (QA_THREADS / 32)));
  auto go = [&](auto kern, auto* out) {
    using T = std::remove_pointer_t<decltype(out)>;
    launch_pdl(pdl_bit_for_tokens(c.n_tokens), kern, grid, dim3(QA_THREADS), (size_t)0, c.stream, (const uint8_t*)c.kcache, (const uint8_t*)c.vcache, c.k_scale,
               c.v_scale, c.tok_pos, c.tok_seq, c.seq_slot, c.page_table, c.table_stride, c.n_pages, (T*)c.keys, (T*)c.values, c.n_tokens, c.nkv, c.hd, warps, c.err);
  };
  auto type = [&](auto* out) {
    using T = std::remove_pointer_t<decltype(out)>;
    if (c.format == QF_INT8) many ? go(quantized_rows_kernel<T, QF_INT8, QA_MANY_PIECES>, out) : go(quantized_rows_kernel<T, QF_INT8, 1>, out);
    else many ? go(quantized_rows_kernel<T, QF_FP8, QA_MANY_PIECES>, out) : go(quantized_rows_kernel<T, QF_FP8, 1>, out);
  };
  if (c.dtype == DT_F32) type((float*)nullptr);
  else type((__nv_bfloat16*)nullptr);
  EL_LAUNCH_CHECK("quantized_rows");
  return 0;
}
