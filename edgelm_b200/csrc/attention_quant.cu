// Entry points of the attention over the 8-bit cache.
#include <algorithm>

#include "attention_quant_decode.cuh"
#include "attention_quant_prefill.cuh"

namespace edgelm {
int launch_decode_quant_int8(const QuantDecodeArgs& p, int dtype, int hd, int n_seqs, int n_splits, int warps, cudaStream_t stream);
int launch_decode_quant_fp8(const QuantDecodeArgs& p, int dtype, int hd, int n_seqs, int n_splits, int warps, cudaStream_t stream);
int launch_prefill_quant_int8(const QuantPrefillArgs& p, int dtype, int hd, int n_tiles, int n_splits, cudaStream_t stream);
int launch_prefill_quant_fp8(const QuantPrefillArgs& p, int dtype, int hd, int n_tiles, int n_splits, cudaStream_t stream);
bool prefill_quant_tc_takes(const void* q, long long ldq, const void* out, long long ldo, int dtype, int hd);
int launch_prefill_quant_tc(const void* q, long long ldq, void* out, long long ldo, const void* kcache, const void* vcache, const float* k_scale,
                            const float* v_scale, int format, const int32_t* page_table, int table_stride, int n_pages, const int32_t* seq_slot,
                            const int32_t* tile_seq, const int32_t* tile_tok0, const int32_t* tile_ntok, const int32_t* tile_pos0, int n_tiles,
                            int max_tile_tokens, int nh, int nkv, int hd, float scale, int n_splits, int max_keys, int window, int* err, cudaStream_t stream);
}  // namespace edgelm

using namespace edgelm;

// One new token a sequence.  With the position tables (cos_t, sin_t [max_pos, hd / 2]) `q` holds the raw q, k, v projections
// [n_seqs, (nh + 2 nkv) hd]: the kernel rotates, appends the new rows as codes (kcache, vcache, k_scale, v_scale are written) and
// attends over the cache with them.  Without: `q` holds rotated query heads and the cache every row up to seq_pos.
// n_splits: blocks that share a sequence's keys, 1 to 8 or a multiple of 8 up to 128; from 16 on `part` is scratch for n_seqs nh (n_splits / 8)
// (hd + 2) floats.  Returns 0 or a negative code.
// (Arguments as one struct, 8-byte fields first: see quant_cache.cu.)
struct QuantDecodeCall {
  const void* q;
  void* out;
  void *kcache, *vcache;
  float *k_scale, *v_scale;
  const int32_t *page_table, *seq_slot, *seq_pos;
  const float *cos_t, *sin_t;
  int* err;
  float* part;
  cudaStream_t stream;
  long long ldq, ldo;
  int dtype, format, table_stride, n_pages, max_pos, n_seqs, nh, nkv, hd, n_splits, window, meta_ready;
  float scale;
};

extern "C" int edgelm_attn_decode_quantized(const QuantDecodeCall* call) {
  const auto [q, out, kcache, vcache, k_scale, v_scale, page_table, seq_slot, seq_pos, cos_t, sin_t, err, part, stream, ldq, ldo, dtype, format, table_stride, n_pages,
              max_pos, n_seqs, nh, nkv, hd, n_splits, window, meta_ready, scale] = *call;
  if (n_seqs == 0) return 0;
  const char* who = "attn_decode_quantized";
  EL_REFUSE(nh > 0 && nkv > 0 && nh % nkv == 0, "%s: %d query heads are not a multiple of %d key/value heads", who, nh, nkv);
  EL_REFUSE(hd >= 16 && hd <= 256 && hd % 16 == 0, "%s: head size %d (takes 16..256 in steps of 16)", who, hd);
  EL_REFUSE((format == QF_INT8 || format == QF_FP8) && (dtype == DT_F32 || dtype == DT_BF16), "%s: format %d, dtype %d", who, format, dtype);
  EL_REFUSE(n_seqs > 0 && n_seqs <= 65535, "%s: %d sequences (takes up to 65,535)", who, n_seqs);
  const int chunks = (nh / nkv + QD_HEADS - 1) / QD_HEADS;
  EL_REFUSE((long long)nkv * chunks <= 65535, "%s: too many heads", who);
  EL_REFUSE(n_splits >= 1 && n_splits <= QD_CLUSTER * QD_MAX_GROUPS && (n_splits <= QD_CLUSTER || n_splits % QD_CLUSTER == 0),
            "%s: %d splits (takes 1 to %d, and multiples of %d up to %d)", who, n_splits, QD_CLUSTER, QD_CLUSTER, QD_CLUSTER * QD_MAX_GROUPS);
  EL_REFUSE(n_splits <= QD_CLUSTER || part != nullptr, "%s: %d splits need the scratch", who, n_splits);
  EL_REFUSE(n_splits <= QD_CLUSTER || nh <= 65535, "%s: too many heads", who);
  EL_REFUSE(window >= 0, "%s: a window of %d keys", who, window);
  EL_REFUSE((cos_t == nullptr) == (sin_t == nullptr) && (cos_t == nullptr || max_pos > 0), "%s: position tables", who);
  EL_REFUSE((uintptr_t)kcache % 16 == 0 && (uintptr_t)vcache % 16 == 0 && (uintptr_t)k_scale % 16 == 0 && (uintptr_t)v_scale % 16 == 0,
            "%s: the cache must start on 16-byte boundaries", who);
  EL_REFUSE((uintptr_t)out % 8 == 0 && ldo % 2 == 0, "%s: output rows must start on 8-byte boundaries", who);
  const QuantDecodeArgs p = {q, out, (uint8_t*)kcache, (uint8_t*)vcache, k_scale, v_scale, page_table, seq_slot, seq_pos, cos_t, sin_t, err, part,
                             ldq, ldo, table_stride, n_pages, max_pos, nh, nkv, window, meta_ready, n_splits < QD_CLUSTER ? n_splits : QD_CLUSTER, scale};
  // Warps a block, by how many blocks there are: a block costs about 8 us from its first read to its last, whatever it has to do, so few
  // blocks get many warps and many blocks few (an SM holds 12, 12 and 10 warps of them at a time).  us with 2, 4 and 12 warps: 2,048 blocks
  // (64 sequences of 700 to 2,300 keys, 32 heads of 64) 87, 112, 132; 320 blocks (15 heads on 5) 34, 22, 26; 80 blocks (two splits of 8
  // sequences of 130 to 2,040 keys, 15 heads on 5) 17, 11, 9.
  const long long blocks = (long long)n_seqs * nkv * chunks * n_splits;
  const int warps = blocks <= 148 ? QD_MAX_WARPS : blocks <= 592 ? 4 : 2;
  const int rc = format == QF_INT8 ? launch_decode_quant_int8(p, dtype, hd, n_seqs, n_splits, warps, stream)
                                   : launch_decode_quant_fp8(p, dtype, hd, n_seqs, n_splits, warps, stream);
  if (rc) return rc;
  EL_LAUNCH_CHECK(who);
  return 0;
}

// New tokens, any number a sequence, as tiles of at most `max_tile_tokens` (up to 128) consecutive tokens of one sequence; their keys and
// values are in the cache already.  n_splits: blocks that share a row tile's keys, 1 to 8 (0: by sizes, with
// `max_keys` as the longest sequence's keys that a token sees).  form: 0 tcgen05 where it takes the operands, else mma.sync; 1 mma.sync; 2 tcgen05.
struct QuantPrefillCall {
  const void* q;
  void* out;
  const void *kcache, *vcache;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *seq_slot, *tile_seq, *tile_tok0, *tile_ntok, *tile_pos0;
  int* err;
  cudaStream_t stream;
  long long ldq, ldo;
  int dtype, format, table_stride, n_pages, n_tiles, max_tile_tokens, nh, nkv, hd, n_splits, max_keys, window, form;
  float scale;
};

extern "C" int edgelm_attn_prefill_quantized(const QuantPrefillCall* call) {
  const auto [q, out, kcache, vcache, k_scale, v_scale, page_table, seq_slot, tile_seq, tile_tok0, tile_ntok, tile_pos0, err, stream, ldq, ldo, dtype, format,
              table_stride, n_pages, n_tiles, max_tile_tokens, nh, nkv, hd, n_splits, max_keys, window, form, scale] = *call;
  if (n_tiles == 0) return 0;
  const char* who = "attn_prefill_quantized";
  EL_REFUSE(nh > 0 && nkv > 0 && nh % nkv == 0, "%s: %d query heads are not a multiple of %d key/value heads", who, nh, nkv);
  EL_REFUSE(hd >= 16 && hd <= 256 && hd % 16 == 0, "%s: head size %d (takes 16..256 in steps of 16)", who, hd);
  EL_REFUSE((format == QF_INT8 || format == QF_FP8) && (dtype == DT_F32 || dtype == DT_BF16), "%s: format %d, dtype %d", who, format, dtype);
  EL_REFUSE(n_tiles > 0 && max_tile_tokens >= 1 && max_tile_tokens <= 128, "%s: %d tiles of up to %d tokens (takes 1 to 128)", who, n_tiles, max_tile_tokens);
  EL_REFUSE(n_splits >= 0 && n_splits <= QP_MAX_SPLITS && max_keys >= 0, "%s: %d splits (takes 1 to %d, 0: by sizes), %d keys", who, n_splits, QP_MAX_SPLITS, max_keys);
  EL_REFUSE(window >= 0 && n_pages > 0, "%s: a window of %d keys, %d pages", who, window, n_pages);
  EL_REFUSE((uintptr_t)kcache % 16 == 0 && (uintptr_t)vcache % 16 == 0 && (uintptr_t)k_scale % 16 == 0 && (uintptr_t)v_scale % 16 == 0,
            "%s: the cache must start on 16-byte boundaries", who);
  EL_REFUSE((uintptr_t)q % 16 == 0 && ldq % 4 == 0, "%s: query rows must start on a 16-byte boundary, a multiple of 4 numbers apart", who);
  EL_REFUSE((uintptr_t)out % 8 == 0 && ldo % 2 == 0, "%s: output rows must start on 8-byte boundaries", who);
  EL_REFUSE(form >= 0 && form <= 2, "%s: form %d", who, form);
  EL_REFUSE(nkv <= 65535, "%s: %d key/value heads (takes up to 65,535)", who, nkv);
  // Sequences of one page stay on mma.sync: a block there starts sooner (us on mma.sync and tcgen05, 64 tokens: 9 heads of 64 on 3 5.6, 7.4; 16 of 128
  // on 4 6.9, 9.9; 16 sequences of 12 heads of 96 on 4 8.2, 11.6; 128 tokens: 7.6, 7.6; 9.5, 10.2; 15.7, 18.4, and of 9 heads of 64 9.3, 8.2).
  const bool taken = err != nullptr && prefill_quant_tc_takes(q, ldq, out, ldo, dtype, hd), tc = form == 2 ? taken : form == 0 && taken && max_keys > PAGE;
  EL_REFUSE(form != 2 || tc, "%s: these operands are not taken on tcgen05 (bfloat16, head size up to 128, 16-byte rows, an error word)", who);
  if (tc) {
    const int rc = launch_prefill_quant_tc(q, ldq, out, ldo, kcache, vcache, k_scale, v_scale, format, page_table, table_stride, n_pages, seq_slot, tile_seq,
                                           tile_tok0, tile_ntok, tile_pos0, n_tiles, max_tile_tokens, nh, nkv, hd, scale, n_splits, max_keys, window, err, stream);
    if (rc) return rc;
    EL_LAUNCH_CHECK(who);
    return 0;
  }
  const int per_tile = (max_tile_tokens * (nh / nkv) + QP_ROWS - 1) / QP_ROWS;
  EL_REFUSE((long long)n_tiles * per_tile <= 65535, "%s: %d tiles of %d blocks (takes up to 65,535 blocks a kv head)", who, n_tiles, per_tile);
  const QuantPrefillArgs p = {q, out, (const uint8_t*)kcache, (const uint8_t*)vcache, k_scale, v_scale, page_table, seq_slot, tile_seq, tile_tok0, tile_ntok,
                              tile_pos0, err, ldq, ldo, table_stride, n_pages, nh, nkv, window, per_tile, max_keys, scale};
  const int rc = format == QF_INT8 ? launch_prefill_quant_int8(p, dtype, hd, n_tiles, n_splits, stream) : launch_prefill_quant_fp8(p, dtype, hd, n_tiles, n_splits, stream);
  if (rc) return rc;
  EL_LAUNCH_CHECK(who);
  return 0;
}
