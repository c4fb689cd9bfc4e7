// Attention of one new token a sequence over the 8-bit cache (quant_cache.cuh, attention_quant.cuh), optionally with the rotation of
// its query and key and the quantising append in the same kernel.
//
// A warp walks tiles of up to 64 keys; a tile's key codes and value codes are two contiguous pieces of a page, each ONE bulk copy into
// the warp's own ring of two stages (its scales come by 16-byte copies of the lanes), so no warp waits for
// another until the sequence is done.  The keys are the 16-row operand and up to 8 query heads the 8 columns (S^T = K Q^T,
// O^T = V^T P^T): no row of a product is padding however few heads a kv head serves.  The order of dims inside a product is free,
// so a lane reads its key row's codes in whole words (16 bytes where the head size allows), and its value codes likewise: the
// transpose that V^T asks for is one byte permutation of two keys' words.  Up to 4 heads take every other column, so that a lane, which
// holds two neighbouring columns of a product, has one score a key to deal with instead of two.  A key's scales are taken apart once a
// tile, by one lane, and not by all that use them.
//
// 64 sequences of 700 to 2,300 keys, 32 heads of 64: 87 us int8, 79 us e4m3 for 419 MB (4.8 and 5.3 TB/s; the floor is 64 us).  There the
// warps' instructions bound it (about 870 a tile of 64 keys, 376 of them on the ALU pipe, most of these the codes' way to float16; ncu: issue
// slots 47 % busy with 9 warps an SM, as many as the stages leave room for); shorter stages make room for twice the warps and need more
// instructions a key: 83 to 92 us.
//
// A sequence's tiles are dealt round over the warps of a cluster of up to 8 blocks, whose partial results meet in distributed shared
// memory in a fixed order: one launch, no scratch in memory, no counters.  Where few heads of few long sequences leave SMs idle, several
// clusters share a sequence and a small second kernel folds their results out of a scratch.  (Clusters of 16 need 16 free SMs of one
// GPC: 8 of them took 14.3 us where 8 clusters of 8 took 8.2.)  More than 8 heads a kv head: further blocks.
#pragma once
#include <cooperative_groups.h>

#include "attention_quant.cuh"

namespace edgelm {

constexpr int QD_HEADS = 8;        // query heads of a block
constexpr int QD_STAGES = 2;
constexpr int QD_MAX_WARPS = 12;
constexpr int QD_CLUSTER = 8;      // blocks of a cluster, at most
constexpr int QD_MAX_GROUPS = 16;  // clusters that share a sequence, at most

__host__ __device__ constexpr int qd_tile_keys(int hdt) { return hdt <= 4 ? 64 : hdt <= 8 ? 32 : 16; }   // about 8 KB of codes
__host__ __device__ constexpr int qd_stage_bytes(int hdt) { return qd_tile_keys(hdt) * (2 * hdt * 16 + 8); }
__host__ __device__ constexpr int qd_align(int b) { return (b + 127) / 128 * 128; }
// [terms][8][hd + 8] float16 queries | 8 factors | the new key's and value's codes and scales | barriers | [8][hd + 2] the block's result |
// the warps' key factors | the warps' stages
__host__ __device__ constexpr int qd_off_factors(int hdt, int terms) { return terms * QD_HEADS * (hdt * 16 + 8) * 2; }
__host__ __device__ constexpr int qd_off_new(int hdt, int terms) { return qd_off_factors(hdt, terms) + 32; }
__host__ __device__ constexpr int qd_off_bars(int hdt, int terms) { return qd_off_new(hdt, terms) + 2 * hdt * 16 + 16; }
__host__ __device__ constexpr int qd_off_result(int hdt, int terms, int warps) { return qd_off_bars(hdt, terms) + warps * QD_STAGES * 8; }
__host__ __device__ constexpr int qd_off_keys(int hdt, int terms, int warps) {
  return qd_align(qd_off_result(hdt, terms, warps) + QD_HEADS * (hdt * 16 + 2) * 4);
}
__host__ __device__ constexpr int qd_off_ring(int hdt, int terms, int warps) { return qd_align(qd_off_keys(hdt, terms, warps) + warps * qd_tile_keys(hdt) * 16); }
__host__ __device__ constexpr int qd_smem(int hdt, int terms, int warps) {
  return qd_off_ring(hdt, terms, warps) + warps * QD_STAGES * qd_align(qd_stage_bytes(hdt));
}

struct QuantDecodeArgs {
  const void* q;            // [n_seqs, ldq]: query heads (or q, k, v projections when rotating)
  void* out;
  uint8_t *kcache, *vcache;
  float *k_scale, *v_scale;
  const int32_t *page_table, *seq_slot, *seq_pos;
  const float *cos_t, *sin_t;   // null: the queries are rotated and the new rows in the cache already
  int* err;
  float* part;              // with several clusters a sequence: [n_seqs, nh, groups][hd + 2] (sums of weighted values, reference, sum of weights)
  long long ldq, ldo;
  int table_stride, n_pages, max_pos, nh, nkv, window, meta_ready, cluster;
  float scale;
};

// words of a key row: HDT of them for lane tig, so that word ks holds four dims of step ks (the same dims in every row)
template <int HDT>
__device__ __forceinline__ void qd_key_words(const uint8_t* row, int tig, uint32_t (&w)[HDT]) {
  if constexpr (HDT % 4 == 0) {
#pragma unroll
    for (int i = 0; i < HDT / 4; ++i) *reinterpret_cast<uint4*>(&w[4 * i]) = *reinterpret_cast<const uint4*>(row + 64 * i + 16 * tig);
  } else if constexpr (HDT % 2 == 0) {
#pragma unroll
    for (int i = 0; i < HDT / 2; ++i) *reinterpret_cast<uint2*>(&w[2 * i]) = *reinterpret_cast<const uint2*>(row + 32 * i + 8 * tig);
  } else {
#pragma unroll
    for (int i = 0; i < HDT; ++i) w[i] = *reinterpret_cast<const uint32_t*>(row + 16 * i + 4 * tig);
  }
}
template <int HDT>
__device__ __forceinline__ int qd_key_dim(int ks, int tig) {   // the first of the four dims
  if constexpr (HDT % 4 == 0) return 64 * (ks / 4) + 16 * tig + 4 * (ks % 4);
  else if constexpr (HDT % 2 == 0) return 32 * (ks / 2) + 8 * tig + 4 * (ks % 2);
  else return 16 * ks + 4 * tig;
}
// the 2 HDT neighbouring codes of a value row that lane gid holds, as words (odd HDT: the last one half full)
template <int HDT>
__device__ __forceinline__ void qd_value_words(const uint8_t* p, uint32_t (&w)[(HDT + 1) / 2]) {
  if constexpr (HDT % 8 == 0) {
#pragma unroll
    for (int i = 0; i < HDT / 8; ++i) *reinterpret_cast<uint4*>(&w[4 * i]) = *reinterpret_cast<const uint4*>(p + 16 * i);
  } else if constexpr (HDT % 4 == 0) {
#pragma unroll
    for (int i = 0; i < HDT / 4; ++i) *reinterpret_cast<uint2*>(&w[2 * i]) = *reinterpret_cast<const uint2*>(p + 8 * i);
  } else if constexpr (HDT % 2 == 0) {
#pragma unroll
    for (int i = 0; i < HDT / 2; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  } else {   // pieces of two bytes
#pragma unroll
    for (int i = 0; i < HDT; ++i) {
      const uint32_t v = *reinterpret_cast<const uint16_t*>(p + 2 * i);
      w[i / 2] = i % 2 ? w[i / 2] | v << 16 : v;
    }
  }
}

// One head row by one warp, lane pairs (j, j + half), j = lane + 32 i: read ahead of everything that says where the sequence stands ..
template <int HDT> struct QdRow {
  static constexpr int N = (HDT + 3) / 4;
  float a[N], b[N];
  template <typename T> __device__ __forceinline__ void load(const T* src) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = lane + 32 * i;
      a[i] = j < HDT * 8 ? to_f32(src[j]) : 0.f;
      b[i] = j < HDT * 8 ? to_f32(src[j + HDT * 8]) : 0.f;
    }
  }
  // .. then rotated, if `cs` says so; the row's largest magnitude
  __device__ __forceinline__ uint32_t turn(const float* cs, const float* sn) {
    const int lane = threadIdx.x & 31;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = lane + 32 * i;
      if (cs && j < HDT * 8) rotate_pair(a[i], b[i], cs[j], sn[j]);
      most = max(most, max(magnitude_bits(a[i]), magnitude_bits(b[i])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    return most;
  }
};

template <int HDT, int FMT, int HC, typename T>   // HC: scores a lane has of a key, 1 (up to 4 heads) or 2
__global__ void __launch_bounds__(QD_MAX_WARPS * 32)
attn_decode_quant_kernel(const QuantDecodeArgs p) {
  constexpr int HD = HDT * 16, HALF = HD / 2, TERMS = sizeof(T) == 4 ? 2 : 1, QP = HD + 8, KT = qd_tile_keys(HDT), MT = KT / 16, WS = HD + 2;
  constexpr int STAGE = qd_align(qd_stage_bytes(HDT));
  extern __shared__ __align__(128) uint8_t qd_raw[];
  static_assert(QD_HEADS * WS * 4 <= STAGE, "a warp's partial fits its first stage");
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3;
  __half* Qs = reinterpret_cast<__half*>(qd_raw);
  float* factors = reinterpret_cast<float*>(qd_raw + qd_off_factors(HDT, TERMS));
  uint8_t* fresh = qd_raw + qd_off_new(HDT, TERMS);                       // [2][HD] codes, two scales
  float* fresh_scale = reinterpret_cast<float*>(fresh + 2 * HD);
  uint64_t* bars = reinterpret_cast<uint64_t*>(qd_raw + qd_off_bars(HDT, TERMS)) + warp * QD_STAGES;
  float* result = reinterpret_cast<float*>(qd_raw + qd_off_result(HDT, TERMS, warps));
  float4* key_data = reinterpret_cast<float4*>(qd_raw + qd_off_keys(HDT, TERMS, warps)) + warp * KT;     // u, e, f, 2^-e (attention_quant.cuh)
  uint8_t* ring = qd_raw + qd_off_ring(HDT, TERMS, warps) + (size_t)warp * QD_STAGES * STAGE;

  const int splits = gridDim.x, split = blockIdx.x, seq = blockIdx.z;
  const int cluster_size = p.cluster, rank = split % cluster_size;
  const int g = p.nh / p.nkv, chunks = HC == 1 ? 1 : (g + QD_HEADS - 1) / QD_HEADS;
  const int kvh = blockIdx.y / chunks, h0 = (blockIdx.y - kvh * chunks) * QD_HEADS, heads = min(QD_HEADS, g - h0);
  const bool fused = p.cos_t != nullptr;
  if (lane < QD_STAGES) asm volatile("mbarrier.init.shared::cta.b64 [%0], 33;" ::"r"(aq_smem(&bars[lane])));      // the bulk copies' bytes, and each lane's own copy
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  pdl_launch_dependents();
  if (!p.meta_ready) pdl_wait();
  // rows to make: the block's query heads, then (in the block that holds the new token) its key and its value
  constexpr int AHEAD = HDT <= 4 ? 4 : HDT <= 8 ? 2 : 1;
  QdRow<HDT> ahead[AHEAD];
  auto row_at = [&](int r) {
    const int head = r < heads ? kvh * g + h0 + r : p.nh + (r > heads ? p.nkv : 0) + kvh;
    return reinterpret_cast<const T*>(p.q) + (size_t)seq * p.ldq + (size_t)head * HD;
  };
  const int n_rows = heads + (fused ? 2 : 0);
  auto read_ahead = [&]() {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (warp + i * warps < n_rows) ahead[i].load(row_at(warp + i * warps));
  };
  if (!p.meta_ready) read_ahead();
  const int nkeys = p.seq_pos[seq] + 1, pos = nkeys - 1;
  const int32_t* pages = p.page_table + (size_t)p.seq_slot[seq] * p.table_stride;
  const int first_key = p.window > 0 ? max(0, nkeys - p.window) : 0;
  const int tile0 = first_key / KT, n_tiles = nkeys > 0 ? (nkeys + KT - 1) / KT - tile0 : 0;
  const int step = splits * warps, mine = split + splits * warp;          // this warp's tiles: mine, mine + step, ..
  const int my_tiles = n_tiles > mine ? (n_tiles - mine + step - 1) / step : 0;
  auto page_of = [&](int i) {   // of the warp's i-th tile; -1: none, or not one of the cache's
    const int at = i < my_tiles ? (tile0 + mine + i * step) * KT / PAGE : p.table_stride;
    int page = at < p.table_stride ? pages[at] : -1;
    if (i < my_tiles && (page < 0 || page >= p.n_pages)) {
      if (p.err) atomicOr(p.err, ERR_PAGE_RANGE);
      page = -1;
    }
    return page;
  };
  int my_page = page_of(lane);           // a lane holds the page of one of the next 32 tiles
  const bool owner = fused && nkeys > 0 && (n_tiles - 1) % splits == split;    // this block holds the new token
  int new_page = -1;
  if (owner) {
    new_page = pos / PAGE < p.table_stride ? pages[pos / PAGE] : -1;
    if (new_page >= p.n_pages) new_page = -1;
  }
  if (p.meta_ready) {   // the queries, the new key and value and the cache rows of the step before are the earlier kernels'
    pdl_wait();
    read_ahead();
  }
  if (fused && pos >= p.max_pos && threadIdx.x == 0 && p.err) atomicOr(p.err, ERR_POSITION_RANGE);

  auto issue = [&](int i, int page) {   // the warp's i-th tile into stage i % QD_STAGES
    if (page < 0) return;
    const int s = i % QD_STAGES, row0 = ((tile0 + mine + i * step) * KT) % PAGE;
    const uint32_t bar = aq_smem(&bars[s]), dst = aq_smem(ring + s * STAGE);
    const size_t at = ((size_t)page * p.nkv + kvh) * PAGE + row0;
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * KT * HD) : "memory");
    __syncwarp();
    if (lane == 0) aq_bulk(dst, p.kcache + at * HD, KT * HD, bar);
    if (lane == 1) aq_bulk(dst + KT * HD, p.vcache + at * HD, KT * HD, bar);
    if (lane < KT / 2) {   // scales: 16 bytes a lane
      const float* from = (lane < KT / 4 ? p.k_scale : p.v_scale) + at + lane % (KT / 4) * 4;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 2 * KT * HD + lane * 16), "l"(from) : "memory");
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
  };
#pragma unroll
  for (int i = 0; i < QD_STAGES; ++i)
    if (i < my_tiles) issue(i, __shfl_sync(0xffffffffu, my_page, i));

  // ---- the block's query rows as float16 terms, and, in the block that holds it, the new token's key and value as codes
  {
    const int tpos = min(max(pos, 0), max(p.max_pos - 1, 0));
    const float* cs = fused ? p.cos_t + (size_t)tpos * HALF : nullptr;
    const float* sn = fused ? p.sin_t + (size_t)tpos * HALF : nullptr;
    // columns that no head has
    for (int i = threadIdx.x; i < TERMS * QD_HEADS * (HD / 8); i += blockDim.x) {
      const int r = i / (HD / 8) % QD_HEADS;
      if (HC == 1 ? r % 2 == 1 || r / 2 >= heads : r >= heads) *reinterpret_cast<uint4*>(Qs + (i / (HD / 8)) * QP + i % (HD / 8) * 8) = make_uint4(0, 0, 0, 0);
    }
    if (threadIdx.x < QD_HEADS) factors[threadIdx.x] = 0.f;
    __syncthreads();
    auto make = [&](int r, QdRow<HDT>& row) {
      const bool is_v = r > heads;
      const uint32_t most = row.turn(is_v ? nullptr : cs, sn);
      const auto &a = row.a, &b = row.b;
      if (r < heads) {
        const float lift = query_lift(most);
        __half* col = Qs + (HC == 1 ? 2 * r : r) * QP;                 // a head's column: r, or (HC 1) every other one
#pragma unroll
        for (int i = 0; i < (HDT + 3) / 4; ++i) {
          const int j = lane + 32 * i;
          if (j < HALF) {
            const float x = a[i] * lift, y = b[i] * lift;
            const __half hx = __float2half_rn(x), hy = __float2half_rn(y);
            col[j] = hx;
            col[j + HALF] = hy;
            if (TERMS == 2) {
              col[QD_HEADS * QP + j] = __float2half_rn(x - __half2float(hx));
              col[QD_HEADS * QP + j + HALF] = __float2half_rn(y - __half2float(hy));
            }
          }
        }
        if (lane == 0) factors[HC == 1 ? 2 * r : r] = 1.0f / lift * p.scale * AQ_LOG2E;
      } else {
        const RowScale rs = row_scale<FMT>(most);
        const size_t at = ((size_t)max(new_page, 0) * p.nkv + kvh) * PAGE + pos % PAGE;
        uint8_t* dst = (is_v ? p.vcache : p.kcache) + at * HD;
        const bool write = new_page >= 0 && h0 == 0 && pos < p.max_pos;
#pragma unroll
        for (int i = 0; i < (HDT + 3) / 4; ++i) {
          const int j = lane + 32 * i;
          if (j < HALF) {
            const uint32_t c = to_codes4<FMT>(make_float2(a[i], b[i]), make_float2(0.f, 0.f), rs.to_codes);
            fresh[(is_v ? HD : 0) + j] = (uint8_t)c;
            fresh[(is_v ? HD : 0) + j + HALF] = (uint8_t)(c >> 8);
            if (write) {
              dst[j] = (uint8_t)c;
              dst[j + HALF] = (uint8_t)(c >> 8);
            }
          }
        }
        if (lane == 0) {
          fresh_scale[is_v] = rs.scale;
          if (write) (is_v ? p.v_scale : p.k_scale)[at] = rs.scale;
        }
      }
    };
    const int wanted = heads + (owner ? 2 : 0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (warp + i * warps < wanted) make(warp + i * warps, ahead[i]);
    for (int r = warp + AHEAD * warps; r < wanted; r += warps) {
      QdRow<HDT> row;
      row.load(row_at(r));
      make(r, row);
    }
  }
  __syncthreads();
  uint32_t qb[TERMS][HDT][2];     // B fragments: head gid, the dims of qd_key_dim
#pragma unroll
  for (int tm = 0; tm < TERMS; ++tm)
#pragma unroll
    for (int ks = 0; ks < HDT; ++ks) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(Qs + (tm * QD_HEADS + gid) * QP + qd_key_dim<HDT>(ks, tig));
      qb[tm][ks][0] = w[0];
      qb[tm][ks][1] = w[1];
    }
  float qf[HC], m[HC], l[HC];
#pragma unroll
  for (int h = 0; h < HC; ++h) {
    qf[h] = factors[2 * tig + h];
    m[h] = -CUDART_INF_F;
    l[h] = 0.f;
  }
  const int pi = (gid >> 1) + 4 * (gid & 1);   // rows of a product's 16 keys: row gid is key pi, row gid + 8 key pi + 8 (see the values below)

  float o[HDT][4];
#pragma unroll
  for (int i = 0; i < HDT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  bool failed = false;
  uint32_t parity = 0;     // bit s: the parity that stage s waits for
  for (int i = 0; i < my_tiles; ++i) {
    if (i > 0 && i % 32 == 0) my_page = page_of(i + lane);
    const int s = i % QD_STAGES, page = __shfl_sync(0xffffffffu, my_page, i % 32);
    if (page >= 0) {
      failed = !__all_sync(0xffffffffu, aq_wait(aq_smem(&bars[s]), parity >> s & 1));
      if (failed) break;
      parity ^= 1u << s;
      uint8_t* Kt = ring + s * STAGE;
      uint8_t* Vt = Kt + KT * HD;
      float* Ku = reinterpret_cast<float*>(Vt + KT * HD);
      float* Vu = Ku + KT;
      const int key0 = (tile0 + mine + i * step) * KT, valid = min(KT, nkeys - key0), skip = max(0, first_key - key0);
      if (owner && key0 + KT >= nkeys) {   // the copy may have read the row before the append landed
        for (int d = lane; d < HD / 4; d += 32) {
          reinterpret_cast<uint32_t*>(Kt + (valid - 1) * HD)[d] = reinterpret_cast<const uint32_t*>(fresh)[d];
          reinterpret_cast<uint32_t*>(Vt + (valid - 1) * HD)[d] = reinterpret_cast<const uint32_t*>(fresh + HD)[d];
        }
        if (lane == 0) {
          Ku[valid - 1] = fresh_scale[0];
          Vu[valid - 1] = fresh_scale[1];
        }
      }
      if (valid < KT) {   // what lies behind the sequence's end is not its own: whatever is there, it meets weights of zero as zero
        for (int j = lane; j < (KT - valid) * (HD / 16); j += 32) reinterpret_cast<uint4*>(Vt + valid * HD)[j] = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
      for (int r = lane; r < KT; r += 32) {       // keys that are not seen: an offset of minus infinity, and no value
        const ValueScale vsc = value_scale(Vu[r]);
        key_data[r] = r >= skip && r < valid ? make_float4(Ku[r], vsc.e, vsc.f, vsc.undo) : make_float4(0.f, -CUDART_INF_F, 0.f, 0.f);
      }
      __syncwarp();
      // ---- scores: x = s + e; a lane's keys of block mt are pi and pi + 8, its heads' columns 2 tig and (HC 2) 2 tig + 1
      float x[MT][2][HC], mx[HC];
#pragma unroll
      for (int h = 0; h < HC; ++h) mx[h] = m[h];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int ra = mt * 16 + pi, rb = ra + 8;
        uint32_t wa[HDT], wb[HDT];
        qd_key_words<HDT>(Kt + ra * HD, tig, wa);
        qd_key_words<HDT>(Kt + rb * HD, tig, wb);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < HDT; ++ks) {
          uint32_t a0, a1, a2, a3;
          codes_to_half<FMT>(wa[ks], a0, a2);
          codes_to_half<FMT>(wb[ks], a1, a3);
#pragma unroll
          for (int tm = TERMS - 1; tm >= 0; --tm) aq_mma(c, a0, a1, a2, a3, qb[tm][ks][0], qb[tm][ks][1]);
        }
        const float2 ka = *reinterpret_cast<const float2*>(&key_data[ra]), kb = *reinterpret_cast<const float2*>(&key_data[rb]);
#pragma unroll
        for (int h = 0; h < HC; ++h) {            // (a code behind the sequence's end may be no number: the offset alone counts there)
          x[mt][0][h] = ka.y == -CUDART_INF_F ? ka.y : fmaf(c[h], qf[h] * ka.x, ka.y);
          x[mt][1][h] = kb.y == -CUDART_INF_F ? kb.y : fmaf(c[2 + h], qf[h] * kb.x, kb.y);
          mx[h] = fmaxf(mx[h], fmaxf(x[mt][0][h], x[mt][1][h]));
        }
      }
      float ref[HC], fold[HC];
#pragma unroll
      for (int h = 0; h < HC; ++h) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], off));   // over the lanes that hold the other keys of the same heads
        ref[h] = mx[h] == -CUDART_INF_F ? 0.f : mx[h];   // (no score above minus infinity yet)
        fold[h] = aq_exp2(m[h] - ref[h]);
        m[h] = mx[h];
        l[h] *= fold[h];
      }
#pragma unroll
      for (int dt = 0; dt < HDT; ++dt)
#pragma unroll
        for (int h = 0; h < HC; ++h) {
          o[dt][h] *= fold[h];
          o[dt][2 + h] *= fold[h];
        }
      // ---- weights and values: the weights of 16 keys, held as (key, two heads), go through a transpose to (head, two keys); row
      // 2 t of a product is then key t, 2 t + 1 key t + 4, and 8 more: the four keys whose words lane tig reads lie in four rows next
      // to each other's, half as many bank conflicts as rows 2 t and 2 t + 1 give
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int ra = mt * 16 + pi, rb = ra + 8;
        const float2 sa = *(reinterpret_cast<const float2*>(&key_data[ra]) + 1), sb = *(reinterpret_cast<const float2*>(&key_data[rb]) + 1);
        float wa[2] = {0.f, 0.f}, wb[2] = {0.f, 0.f};     // (f and 2^-e of a key that is not seen are zero, and so is its weight)
#pragma unroll
        for (int h = 0; h < HC; ++h) {
          const float ta = aq_exp2(x[mt][0][h] - ref[h] + AQ_LIFT), tb = aq_exp2(x[mt][1][h] - ref[h] + AQ_LIFT);
          l[h] = fmaf(ta, sa.y, fmaf(tb, sb.y, l[h]));
          wa[h] = ta * sa.x;
          wb[h] = tb * sb.x;
        }
        uint32_t pa[TERMS], pb[TERMS];
        {
          const uint32_t ha = aq_pack(wa[0], wa[1]), hb = aq_pack(wb[0], wb[1]);
          pa[0] = aq_transpose8(ha);
          pb[0] = aq_transpose8(hb);
          if constexpr (TERMS == 2) {
            pa[1] = aq_transpose8(aq_rest(wa[0], wa[1], ha));
            pb[1] = aq_transpose8(aq_rest(wb[0], wb[1], hb));
          }
        }
        uint32_t v0[(HDT + 1) / 2], v1[(HDT + 1) / 2], v2[(HDT + 1) / 2], v3[(HDT + 1) / 2];
        const uint8_t* vp = Vt + (mt * 16 + tig) * HD + gid * 2 * HDT;
        qd_value_words<HDT>(vp, v0);
        qd_value_words<HDT>(vp + 4 * HD, v1);
        qd_value_words<HDT>(vp + 8 * HD, v2);
        qd_value_words<HDT>(vp + 12 * HD, v3);
#pragma unroll
        for (int dt = 0; dt < HDT; ++dt) {     // dims gid 2 HDT + 2 dt and the next
          uint32_t a0, a1, a2, a3;
          const uint32_t sel = dt % 2 ? 0x7362 : 0x5140;
          codes_to_half<FMT>(__byte_perm(v0[dt / 2], v1[dt / 2], sel), a0, a1);
          codes_to_half<FMT>(__byte_perm(v2[dt / 2], v3[dt / 2], sel), a2, a3);
#pragma unroll
          for (int tm = TERMS - 1; tm >= 0; --tm) aq_mma(o[dt], a0, a1, a2, a3, pa[tm], pb[tm]);
        }
      }
      __syncwarp();
    }
    const int next = i + QD_STAGES;
    if (next < my_tiles) {
      // (the pages of the next 32 tiles are asked for when their first tile comes up here)
      const int np = next % 32 >= QD_STAGES || next < 32 ? __shfl_sync(0xffffffffu, my_page, next % 32)
                                                         : page_of(next);
      issue(next, np);
    }
  }
  if (failed) {   // a copy did not arrive: report, wait (again within bounds) for the other stage, and make the rows unmistakably wrong
    if (lane == 0 && p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);
#pragma unroll
    for (int s = 0; s < QD_STAGES; ++s) aq_wait(aq_smem(&bars[s]), parity >> s & 1);
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      m[h] = 0.f;
      l[h] = CUDART_NAN_F;
    }
  }
#pragma unroll
  for (int h = 0; h < HC; ++h)
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
  // ---- the warp's partial into its own ring (no copy is on its way there any more), then the block's into `result`
  {
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float* w = reinterpret_cast<float*>(ring) + (HC * tig + h) * WS;
#pragma unroll
      for (int dt = 0; dt < HDT; ++dt) *reinterpret_cast<float2*>(w + gid * 2 * HDT + 2 * dt) = make_float2(o[dt][h] * AQ_OPERAND_BACK, o[dt][2 + h] * AQ_OPERAND_BACK);
      if (gid == 0) *reinterpret_cast<float2*>(w + HD) = make_float2(m[h], l[h]);
    }
  }
  __syncthreads();
  T* out = reinterpret_cast<T*>(p.out) + (size_t)seq * p.ldo + (size_t)(kvh * g + h0) * HD;
  auto store2 = [&](int r, int d, float a, float b) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(out + (size_t)r * HD + d) = make_float2(a, b);
    else *reinterpret_cast<__nv_bfloat162*>(out + (size_t)r * HD + d) = __floats2bfloat162_rn(a, b);
  };
  const float* parts = reinterpret_cast<const float*>(qd_raw + qd_off_ring(HDT, TERMS, warps));
  for (int it = threadIdx.x; it < heads * (HD / 2); it += blockDim.x) {
    const int r = it / (HD / 2), d = (it - r * (HD / 2)) * 2;
    float M = -CUDART_INF_F, L = 0.f, a = 0.f, b = 0.f;
    for (int w = 0; w < warps; ++w) M = fmaxf(M, parts[w * (QD_STAGES * STAGE / 4) + r * WS + HD]);
    const float ref = M == -CUDART_INF_F ? 0.f : M;
    for (int w = 0; w < warps; ++w) {
      const float* pw = parts + w * (QD_STAGES * STAGE / 4) + r * WS;
      const float f = aq_exp2(pw[HD] - ref);
      const float2 v = *reinterpret_cast<const float2*>(pw + d);
      L = fmaf(pw[HD + 1], f, L);
      a = fmaf(v.x, f, a);
      b = fmaf(v.y, f, b);
    }
    if (splits == 1) {
      const float inv = nkeys > 0 ? 1.0f / L : 0.f;     // (a sequence of no token: a row of zeros)
      store2(r, d, a * inv, b * inv);
    } else {
      *reinterpret_cast<float2*>(result + r * WS + d) = make_float2(a, b);
      if (d == 0) *reinterpret_cast<float2*>(result + r * WS + HD) = make_float2(M, L);
    }
  }
  if (splits == 1) return;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int it = rank * blockDim.x + threadIdx.x; it < heads * (HD / 2); it += cluster_size * blockDim.x) {
    const int r = it / (HD / 2), d = (it - r * (HD / 2)) * 2;
    float2 ml[QD_CLUSTER], v[QD_CLUSTER];
#pragma unroll
    for (int c = 0; c < QD_CLUSTER; ++c) {
      if (c < cluster_size) {
        const float* pw = cluster.map_shared_rank(result, c) + r * WS;
        ml[c] = *reinterpret_cast<const float2*>(pw + HD);
        v[c] = *reinterpret_cast<const float2*>(pw + d);
      }
    }
    float M = -CUDART_INF_F, L = 0.f, a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < QD_CLUSTER; ++c)
      if (c < cluster_size) M = fmaxf(M, ml[c].x);
    const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
    for (int c = 0; c < QD_CLUSTER; ++c) {
      if (c < cluster_size) {
        const float f = aq_exp2(ml[c].x - ref);
        L = fmaf(ml[c].y, f, L);
        a = fmaf(v[c].x, f, a);
        b = fmaf(v[c].y, f, b);
      }
    }
    if (splits == cluster_size) {
      const float inv = nkeys > 0 ? 1.0f / L : 0.f;
      store2(r, d, a * inv, b * inv);
    } else {      // (no token: no tile in any block, a reference of minus infinity and sums of zero)
      float* part = p.part + (((size_t)seq * p.nh + kvh * g + h0 + r) * (splits / cluster_size) + split / cluster_size) * WS;
      *reinterpret_cast<float2*>(part + d) = make_float2(a, b);
      if (d == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(M, L);
    }
  }
  cluster.sync();   // no block ends while another reads its result
}

// The clusters' results of a (sequence, head): a block each, a thread two dims.
template <typename T>
__global__ void attn_decode_quant_fold_kernel(const float* __restrict__ part, T* __restrict__ out, long long ldo, const int32_t* __restrict__ seq_pos, int nh, int hd,
                                              int groups) {
  pdl_launch_dependents();
  pdl_wait();   // the partials are the previous kernel's
  const int seq = blockIdx.x, head = blockIdx.y, ws = hd + 2, d = threadIdx.x * 2;
  if (d >= hd) return;
  const float* p = part + ((size_t)seq * nh + head) * groups * ws;
  float2 ml[QD_MAX_GROUPS], v[QD_MAX_GROUPS];
#pragma unroll
  for (int c = 0; c < QD_MAX_GROUPS; ++c) {
    if (c < groups) {
      ml[c] = *reinterpret_cast<const float2*>(p + c * ws + hd);
      v[c] = *reinterpret_cast<const float2*>(p + c * ws + d);
    }
  }
  float M = -CUDART_INF_F, L = 0.f, a = 0.f, b = 0.f;
#pragma unroll
  for (int c = 0; c < QD_MAX_GROUPS; ++c)
    if (c < groups) M = fmaxf(M, ml[c].x);
  const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
  for (int c = 0; c < QD_MAX_GROUPS; ++c) {
    if (c < groups) {
      const float f = aq_exp2(ml[c].x - ref);
      L = fmaf(ml[c].y, f, L);
      a = fmaf(v[c].x, f, a);
      b = fmaf(v[c].y, f, b);
    }
  }
  const float inv = seq_pos[seq] >= 0 ? 1.0f / L : 0.f;
  T* dst = out + (size_t)seq * ldo + (size_t)head * hd + d;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(dst) = make_float2(a * inv, b * inv);
  else *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(a * inv, b * inv);
}

}  // namespace edgelm
