// Writing the 8-bit cache and reading it back (the format: quant_cache.cuh).
//
//   rope_quantize_append   a step's queries rotated in place; its keys rotated and its values as they are, each row as codes and a
//                          scale into its page.  A row is held by hd / 8 neighbouring lanes (rounded up to a power of two), each
//                          with four numbers of the row's first half and their partners of the second: the rotation needs no
//                          exchange, the row's largest magnitude log2(lanes) shuffles, and all reads and writes are pieces of 4
//                          numbers.  Bound by memory: a number is read once and a code written once.
//   quantized_rows         rows of given tokens as numbers.
#include "quant_cache.cuh"

namespace edgelm {

constexpr int QA_THREADS = 256;

template <typename T, int FMT, int LANES>   // LANES: lanes of a row (a power of two, at least hd / 8)
__global__ void __launch_bounds__(QA_THREADS)
rope_quantize_append_kernel(T* __restrict__ qkv, const int32_t* __restrict__ tok_pos, const int32_t* __restrict__ tok_seq,
                            const int32_t* __restrict__ seq_slot, const int32_t* __restrict__ page_table, int table_stride, int n_pages,
                            const float* __restrict__ cos_t, const float* __restrict__ sin_t, int max_pos, uint8_t* __restrict__ kcache,
                            uint8_t* __restrict__ vcache, float* __restrict__ k_scale, float* __restrict__ v_scale, int n_tokens, int nh,
                            int nkv, int hd, int* __restrict__ err) {
  pdl_launch_dependents();
  pdl_wait();   // (launched as a programmatic dependent: the projections are the kernel before this one's)
  const int rows = nh + 2 * nkv, half = hd >> 1;
  const long long row = ((long long)blockIdx.x * QA_THREADS + threadIdx.x) / LANES;
  const int part = threadIdx.x % LANES, j = part * 4;
  const int t = (int)(row / rows), r = (int)(row - (long long)t * rows);
  bool work = t < n_tokens;
  const int pos = work ? tok_pos[t] : 0;
  int page = 0;
  if (work && (pos < 0 || pos >= max_pos)) {
    if (part == 0 && r == 0) atomicOr(err, ERR_POSITION_RANGE);
    work = false;
  }
  if (work) {
    page = pos / PAGE < table_stride ? page_table[(size_t)seq_slot[tok_seq[t]] * table_stride + pos / PAGE] : -1;
    if (page < 0 || page >= n_pages) {
      if (part == 0 && r == 0) atomicOr(err, ERR_PAGE_RANGE);
      work = false;
    }
  }
  const bool mine = work && j < half;
  T* src = qkv + (size_t)(work ? t : 0) * rows * hd + (size_t)r * hd + j;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
  if (mine) {
    a = load_piece(src);
    b = load_piece(src + half);
    if (r < nh + nkv) {
      const float4 c = *reinterpret_cast<const float4*>(cos_t + (size_t)pos * half + j), s = *reinterpret_cast<const float4*>(sin_t + (size_t)pos * half + j);
      rotate_pair(a.x, b.x, c.x, s.x);
      rotate_pair(a.y, b.y, c.y, s.y);
      rotate_pair(a.z, b.z, c.z, s.z);
      rotate_pair(a.w, b.w, c.w, s.w);
    }
  }
  uint32_t most = max(max(max(magnitude_bits(a.x), magnitude_bits(a.y)), max(magnitude_bits(a.z), magnitude_bits(a.w))),
                      max(max(magnitude_bits(b.x), magnitude_bits(b.y)), max(magnitude_bits(b.z), magnitude_bits(b.w))));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (!mine) return;
  if (r < nh) {
    store_piece(src, a);
    store_piece(src + half, b);
    return;
  }
  const RowScale rs = row_scale<FMT>(most);
  const int h = r < nh + nkv ? r - nh : r - nh - nkv;
  const size_t at = ((size_t)page * nkv + h) * PAGE + pos % PAGE;
  uint8_t* codes = (r < nh + nkv ? kcache : vcache) + at * hd + j;
  *reinterpret_cast<uint32_t*>(codes) = to_codes4<FMT>(a.x, a.y, a.z, a.w, rs.to_codes);
  *reinterpret_cast<uint32_t*>(codes + half) = to_codes4<FMT>(b.x, b.y, b.z, b.w, rs.to_codes);
  if (part == 0) (r < nh + nkv ? k_scale : v_scale)[at] = rs.scale;
}

// keys[t], values[t] [nkv, hd] = the numbers that the cache holds for token t; a lane eight of them.
template <typename T, int FMT>
__global__ void __launch_bounds__(QA_THREADS)
quantized_rows_kernel(const uint8_t* __restrict__ kcache, const uint8_t* __restrict__ vcache, const float* __restrict__ k_scale,
                      const float* __restrict__ v_scale, const int32_t* __restrict__ tok_pos, const int32_t* __restrict__ tok_seq,
                      const int32_t* __restrict__ seq_slot, const int32_t* __restrict__ page_table, int table_stride, int n_pages,
                      T* __restrict__ keys, T* __restrict__ values, int n_tokens, int nkv, int hd, int* __restrict__ err) {
  pdl_launch_dependents();
  pdl_wait();
  const int per_row = hd >> 3, per_token = 2 * nkv * per_row;
  const long long i = (long long)blockIdx.x * QA_THREADS + threadIdx.x;
  const int t = (int)(i / per_token);
  if (t >= n_tokens) return;
  const int it = (int)(i - (long long)t * per_token), row = it / per_row, d = (it - row * per_row) * 8;
  const bool is_v = row >= nkv;
  const int h = is_v ? row - nkv : row;
  const int pos = tok_pos[t];
  int page = -1;
  if (pos < 0) {
    if (it == 0) atomicOr(err, ERR_POSITION_RANGE);
  } else {
    if (pos / PAGE < table_stride) page = page_table[(size_t)seq_slot[tok_seq[t]] * table_stride + pos / PAGE];
    if (page < 0 || page >= n_pages) {
      page = -1;
      if (it == 0) atomicOr(err, ERR_PAGE_RANGE);
    }
  }
  T* dst = (is_v ? values : keys) + ((size_t)t * nkv + h) * hd + d;
  float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;     // (a token that the cache cannot hold: zeros, and the error word says so)
  if (page >= 0) {
    const size_t at = ((size_t)page * nkv + h) * PAGE + pos % PAGE;
    const uint2 c = *reinterpret_cast<const uint2*>((is_v ? vcache : kcache) + at * hd + d);
    const float s = (is_v ? v_scale : k_scale)[at];
    uint32_t p0, p1, p2, p3;
    codes_to_half<FMT>(c.x, p0, p1);
    codes_to_half<FMT>(c.y, p2, p3);
    const float2 f0 = half2_to_floats(p0), f1 = half2_to_floats(p1), f2 = half2_to_floats(p2), f3 = half2_to_floats(p3);
    lo = make_float4(f0.x * s, f0.y * s, f1.x * s, f1.y * s);
    hi = make_float4(f2.x * s, f2.y * s, f3.x * s, f3.y * s);
  }
  store_piece(dst, lo);
  store_piece(dst + 4, hi);
}

template <typename T, int FMT>
static void launch_append(const void* qkv, const int32_t* tok_pos, const int32_t* tok_seq, const int32_t* seq_slot, const int32_t* page_table,
                          int table_stride, int n_pages, const float* cos_t, const float* sin_t, int max_pos, void* kc, void* vc, float* ks,
                          float* vs, int n_tokens, int nh, int nkv, int hd, int* err, cudaStream_t stream) {
  const int lanes = hd / 8 <= 2 ? 2 : hd / 8 <= 4 ? 4 : hd / 8 <= 8 ? 8 : hd / 8 <= 16 ? 16 : 32;
  const long long threads = (long long)n_tokens * (nh + 2 * nkv) * lanes;
  auto go = [&](auto kern) {
    launch_pdl(pdl_bit_for_tokens(n_tokens), kern, dim3((unsigned)((threads + QA_THREADS - 1) / QA_THREADS)), dim3(QA_THREADS), (size_t)0, stream,
               (T*)const_cast<void*>(qkv), tok_pos, tok_seq, seq_slot, page_table, table_stride, n_pages, cos_t, sin_t, max_pos, (uint8_t*)kc,
               (uint8_t*)vc, ks, vs, n_tokens, nh, nkv, hd, err);
  };
  if (lanes == 2) go(rope_quantize_append_kernel<T, FMT, 2>);
  else if (lanes == 4) go(rope_quantize_append_kernel<T, FMT, 4>);
  else if (lanes == 8) go(rope_quantize_append_kernel<T, FMT, 8>);
  else if (lanes == 16) go(rope_quantize_append_kernel<T, FMT, 16>);
  else go(rope_quantize_append_kernel<T, FMT, 32>);
}

}  // namespace edgelm

using namespace edgelm;

extern "C" int edgelm_rope_quantize_append(void* qkv, int dtype, int format, const int32_t* tok_pos, const int32_t* tok_seq, const int32_t* seq_slot,
                                           const int32_t* page_table, int table_stride, int n_pages, const float* cos_t, const float* sin_t,
                                           int max_pos, void* kcache, void* vcache, float* k_scale, float* v_scale, int n_tokens, int nh, int nkv,
                                           int hd, int* err, cudaStream_t stream) {
  if (n_tokens == 0) return 0;
  EL_REFUSE(n_tokens > 0 && nh > 0 && nkv > 0, "rope_quantize_append: bad sizes");
  EL_REFUSE(hd >= 16 && hd <= 256 && hd % 16 == 0, "rope_quantize_append: head size %d (takes 16..256 in steps of 16)", hd);
  EL_REFUSE((format == QF_INT8 || format == QF_FP8) && (dtype == DT_F32 || dtype == DT_BF16), "rope_quantize_append: format %d, dtype %d", format, dtype);
  EL_REFUSE((uintptr_t)qkv % 16 == 0 && (uintptr_t)cos_t % 16 == 0 && (uintptr_t)sin_t % 16 == 0 && (uintptr_t)kcache % 16 == 0 && (uintptr_t)vcache % 16 == 0,
            "rope_quantize_append: rows must start on 16-byte boundaries");
  EL_REFUSE((long long)n_tokens * (nh + 2 * nkv) * 32 / QA_THREADS < 0x7fffffffLL, "rope_quantize_append: grid too large");
  auto go = [&](auto fn) { fn(qkv, tok_pos, tok_seq, seq_slot, page_table, table_stride, n_pages, cos_t, sin_t, max_pos, kcache, vcache, k_scale, v_scale,
                              n_tokens, nh, nkv, hd, err, stream); };
  if (dtype == DT_F32) format == QF_INT8 ? go(launch_append<float, QF_INT8>) : go(launch_append<float, QF_FP8>);
  else format == QF_INT8 ? go(launch_append<__nv_bfloat16, QF_INT8>) : go(launch_append<__nv_bfloat16, QF_FP8>);
  EL_LAUNCH_CHECK("rope_quantize_append");
  return 0;
}

extern "C" int edgelm_quantized_rows(const void* kcache, const void* vcache, const float* k_scale, const float* v_scale, int format,
                                     const int32_t* tok_pos, const int32_t* tok_seq, const int32_t* seq_slot, const int32_t* page_table,
                                     int table_stride, int n_pages, void* keys, void* values, int dtype, int n_tokens, int nkv, int hd, int* err,
                                     cudaStream_t stream) {
  if (n_tokens == 0) return 0;
  EL_REFUSE(n_tokens > 0 && nkv > 0, "quantized_rows: bad sizes");
  EL_REFUSE(hd >= 16 && hd <= 256 && hd % 16 == 0, "quantized_rows: head size %d (takes 16..256 in steps of 16)", hd);
  EL_REFUSE((format == QF_INT8 || format == QF_FP8) && (dtype == DT_F32 || dtype == DT_BF16), "quantized_rows: format %d, dtype %d", format, dtype);
  EL_REFUSE((uintptr_t)keys % 16 == 0 && (uintptr_t)values % 16 == 0 && (uintptr_t)kcache % 16 == 0 && (uintptr_t)vcache % 16 == 0,
            "quantized_rows: rows must start on 16-byte boundaries");
  const long long threads = (long long)n_tokens * 2 * nkv * (hd / 8);
  const dim3 grid((unsigned)((threads + QA_THREADS - 1) / QA_THREADS));
  auto go = [&](auto kern, auto* out) {
    using T = std::remove_pointer_t<decltype(out)>;
    launch_pdl(pdl_bit_for_tokens(n_tokens), kern, grid, dim3(QA_THREADS), (size_t)0, stream, (const uint8_t*)kcache, (const uint8_t*)vcache, k_scale, v_scale,
               tok_pos, tok_seq, seq_slot, page_table, table_stride, n_pages, (T*)keys, (T*)values, n_tokens, nkv, hd, err);
  };
  if (dtype == DT_F32) format == QF_INT8 ? go(quantized_rows_kernel<float, QF_INT8>, (float*)nullptr) : go(quantized_rows_kernel<float, QF_FP8>, (float*)nullptr);
  else format == QF_INT8 ? go(quantized_rows_kernel<__nv_bfloat16, QF_INT8>, (__nv_bfloat16*)nullptr)
                         : go(quantized_rows_kernel<__nv_bfloat16, QF_FP8>, (__nv_bfloat16*)nullptr);
  EL_LAUNCH_CHECK("quantized_rows");
  return 0;
}
