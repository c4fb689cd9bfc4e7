// Attention of one new token a sequence over the 8-bit cache (quant_cache.cuh, attention_quant.cuh), optionally with the rotation of
// its query and key and the quantising append in the same kernel.
//
// Bound by the cache's bytes: 2 (hd + 4) a token and kv head.  A warp walks tiles of up to 64 keys; a tile's key codes, value codes and
// scales are four contiguous pieces of a page, each ONE bulk copy into the warp's own ring of two stages, so no warp waits for
// another until the sequence is done.  The keys are the 16-row operand and up to 8 query heads the 8 columns (S^T = K Q^T,
// O^T = V^T P^T): no row of a product is padding however few heads a kv head serves.  The order of dims inside a product is free,
// so a lane reads its key row's codes in whole words (16 bytes where the head size allows), and its value codes likewise: the
// transpose that V^T asks for is one byte permutation of two keys' words.
//
// A sequence's tiles are dealt round over the warps of a cluster of `splits` blocks; the blocks' partial results meet in distributed
// shared memory in a fixed order.  One launch, no scratch in memory, no counters.  More than 8 heads a kv head: further blocks.
#pragma once
#include <cooperative_groups.h>

#include "attention_quant.cuh"

namespace edgelm {

constexpr int QD_HEADS = 8;        // query heads of a block
constexpr int QD_STAGES = 2;
constexpr int QD_MAX_WARPS = 8;
constexpr int QD_MAX_SPLITS = 16;  // blocks of a cluster

__host__ __device__ constexpr int qd_tile_keys(int hdt) { return hdt <= 4 ? 64 : hdt <= 8 ? 32 : 16; }   // about 8 KB of codes
__host__ __device__ constexpr int qd_stage_bytes(int hdt) { return qd_tile_keys(hdt) * (2 * hdt * 16 + 8); }
__host__ __device__ constexpr int qd_align(int b) { return (b + 127) / 128 * 128; }
// [terms][8][hd + 8] float16 queries | 8 factors | the new key's and value's codes and scales | barriers | [8][hd + 2] the block's result
__host__ __device__ constexpr int qd_off_factors(int hdt, int terms) { return terms * QD_HEADS * (hdt * 16 + 8) * 2; }
__host__ __device__ constexpr int qd_off_new(int hdt, int terms) { return qd_off_factors(hdt, terms) + 32; }
__host__ __device__ constexpr int qd_off_bars(int hdt, int terms) { return qd_off_new(hdt, terms) + 2 * hdt * 16 + 16; }
__host__ __device__ constexpr int qd_off_result(int hdt, int terms, int warps) { return qd_off_bars(hdt, terms) + warps * QD_STAGES * 8; }
__host__ __device__ constexpr int qd_off_ring(int hdt, int terms, int warps) {
  return qd_align(qd_off_result(hdt, terms, warps) + QD_HEADS * (hdt * 16 + 2) * 4);
}
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
  long long ldq, ldo;
  int table_stride, n_pages, max_pos, nh, nkv, window, meta_ready;
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

// One head row by one warp: lane pairs (j, j + half), j = lane + 32 i, rotated if `cs` says so; `most` is the row's largest magnitude.
template <int HDT, typename T>
__device__ __forceinline__ void qd_row(const T* src, const float* cs, const float* sn, float (&a)[(HDT + 3) / 4], float (&b)[(HDT + 3) / 4], uint32_t& most) {
  constexpr int HALF = HDT * 8;
  const int lane = threadIdx.x & 31;
  most = 0;
#pragma unroll
  for (int i = 0; i < (HDT + 3) / 4; ++i) {
    const int j = lane + 32 * i;
    a[i] = b[i] = 0.f;
    if (j < HALF) {
      a[i] = to_f32(src[j]);
      b[i] = to_f32(src[j + HALF]);
      if (cs) rotate_pair(a[i], b[i], cs[j], sn[j]);
    }
    most = max(most, max(magnitude_bits(a[i]), magnitude_bits(b[i])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
}

template <int HDT, int FMT, typename T>
__global__ void __launch_bounds__(256)
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
  uint8_t* ring = qd_raw + qd_off_ring(HDT, TERMS, warps) + (size_t)warp * QD_STAGES * STAGE;

  const int splits = gridDim.x, split = blockIdx.x, seq = blockIdx.z;
  const int g = p.nh / p.nkv, chunks = (g + QD_HEADS - 1) / QD_HEADS;
  const int kvh = blockIdx.y / chunks, h0 = (blockIdx.y - kvh * chunks) * QD_HEADS, heads = min(QD_HEADS, g - h0);
  if (lane < QD_STAGES) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(aq_smem(&bars[lane])));
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  pdl_launch_dependents();
  if (!p.meta_ready) pdl_wait();
  const int nkeys = p.seq_pos[seq] + 1, pos = nkeys - 1;
  const int32_t* pages = p.page_table + (size_t)p.seq_slot[seq] * p.table_stride;
  const int first_key = p.window > 0 ? max(0, nkeys - p.window) : 0;
  const int tile0 = first_key / KT, n_tiles = nkeys > 0 ? (nkeys + KT - 1) / KT - tile0 : 0;
  const bool fused = p.cos_t != nullptr;
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
  if (p.meta_ready) pdl_wait();   // the queries, the new key and value and the cache rows of the step before are the earlier kernels'
  if (fused && pos >= p.max_pos && threadIdx.x == 0 && p.err) atomicOr(p.err, ERR_POSITION_RANGE);

  auto issue = [&](int i, int page) {   // the warp's i-th tile into stage i % QD_STAGES
    if (page < 0) return;
    const int s = i % QD_STAGES, row0 = ((tile0 + mine + i * step) * KT) % PAGE;
    const uint32_t bar = aq_smem(&bars[s]), dst = aq_smem(ring + s * STAGE);
    const size_t at = ((size_t)page * p.nkv + kvh) * PAGE + row0;
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(qd_stage_bytes(HDT)) : "memory");
    __syncwarp();
    if (lane == 0) aq_bulk(dst, p.kcache + at * HD, KT * HD, bar);
    if (lane == 1) aq_bulk(dst + KT * HD, p.vcache + at * HD, KT * HD, bar);
    if (lane == 2) aq_bulk(dst + 2 * KT * HD, p.k_scale + at, KT * 4, bar);
    if (lane == 3) aq_bulk(dst + 2 * KT * HD + KT * 4, p.v_scale + at, KT * 4, bar);
  };
#pragma unroll
  for (int i = 0; i < QD_STAGES; ++i)
    if (i < my_tiles) issue(i, __shfl_sync(0xffffffffu, my_page, i));

  // ---- the block's query rows as float16 terms, and, in the block that holds it, the new token's key and value as codes
  {
    const T* tok = reinterpret_cast<const T*>(p.q) + (size_t)seq * p.ldq;
    const int tpos = min(max(pos, 0), max(p.max_pos - 1, 0));
    const float* cs = fused ? p.cos_t + (size_t)tpos * HALF : nullptr;
    const float* sn = fused ? p.sin_t + (size_t)tpos * HALF : nullptr;
    for (int r = warp; r < QD_HEADS + (owner ? 2 : 0); r += warps) {
      float a[(HDT + 3) / 4], b[(HDT + 3) / 4];
      uint32_t most = 0;
      if (r < QD_HEADS) {
        if (r < heads) qd_row<HDT, T>(tok + (size_t)(kvh * g + h0 + r) * HD, cs, sn, a, b, most);
        const float lift = query_lift(most);
#pragma unroll
        for (int i = 0; i < (HDT + 3) / 4; ++i) {
          const int j = lane + 32 * i;
          if (j < HALF) {
            const float x = r < heads ? a[i] * lift : 0.f, y = r < heads ? b[i] * lift : 0.f;
            const __half hx = __float2half_rn(x), hy = __float2half_rn(y);
            Qs[r * QP + j] = hx;
            Qs[r * QP + j + HALF] = hy;
            if (TERMS == 2) {
              Qs[(QD_HEADS + r) * QP + j] = __float2half_rn(x - __half2float(hx));
              Qs[(QD_HEADS + r) * QP + j + HALF] = __float2half_rn(y - __half2float(hy));
            }
          }
        }
        if (lane == 0) factors[r] = 1.0f / lift * p.scale * AQ_LOG2E;
      } else {
        const bool is_v = r > QD_HEADS;
        qd_row<HDT, T>(tok + (size_t)(p.nh + (is_v ? p.nkv : 0) + kvh) * HD, is_v ? nullptr : cs, sn, a, b, most);
        const RowScale rs = row_scale<FMT>(most);
        const size_t at = ((size_t)max(new_page, 0) * p.nkv + kvh) * PAGE + pos % PAGE;
        uint8_t* dst = (is_v ? p.vcache : p.kcache) + at * HD;
        const bool write = new_page >= 0 && h0 == 0 && pos < p.max_pos;
#pragma unroll
        for (int i = 0; i < (HDT + 3) / 4; ++i) {
          const int j = lane + 32 * i;
          if (j < HALF) {
            const uint32_t c = to_codes4<FMT>(a[i], b[i], 0.f, 0.f, rs.to_codes);
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
  const float qf0 = factors[2 * tig], qf1 = factors[2 * tig + 1];
  const int pi = (gid >> 1) + 4 * (gid & 1);   // rows of a product's 16 keys: row gid is key pi, row gid + 8 key pi + 8 (see the values below)

  float o[HDT][4];
#pragma unroll
  for (int i = 0; i < HDT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
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
      // ---- scores: x = s + e, in place; a lane's keys of block mt are pi and pi + 8, its heads 2 tig and 2 tig + 1
      float x[MT][4];
      float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
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
        const bool va = ra >= skip && ra < valid, vb = rb >= skip && rb < valid;
        const float ua = Ku[ra], ub = Ku[rb], ea = value_scale(Vu[ra]).e, eb = value_scale(Vu[rb]).e;
        x[mt][0] = va ? fmaf(c[0], qf0 * ua, ea) : -CUDART_INF_F;
        x[mt][1] = va ? fmaf(c[1], qf1 * ua, ea) : -CUDART_INF_F;
        x[mt][2] = vb ? fmaf(c[2], qf0 * ub, eb) : -CUDART_INF_F;
        x[mt][3] = vb ? fmaf(c[3], qf1 * ub, eb) : -CUDART_INF_F;
        mx0 = fmaxf(mx0, fmaxf(x[mt][0], x[mt][2]));
        mx1 = fmaxf(mx1, fmaxf(x[mt][1], x[mt][3]));
      }
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {   // over the lanes that hold the other keys of the same heads
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
      }
      mx0 = fmaxf(mx0, m0);
      mx1 = fmaxf(mx1, m1);
      const float r0 = mx0 == -CUDART_INF_F ? 0.f : mx0, r1 = mx1 == -CUDART_INF_F ? 0.f : mx1;   // (no score above minus infinity yet)
      const float f0 = aq_exp2(m0 - r0), f1 = aq_exp2(m1 - r1);
      m0 = mx0;
      m1 = mx1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int dt = 0; dt < HDT; ++dt) {
        o[dt][0] *= f0;
        o[dt][1] *= f1;
        o[dt][2] *= f0;
        o[dt][3] *= f1;
      }
      const float b0 = AQ_LIFT - r0, b1 = AQ_LIFT - r1;
      // ---- weights and values: the weights of 16 keys, held as (key, two heads), go through a transpose to (head, two keys); row
      // 2 t of a product is then key t, 2 t + 1 key t + 4, and 8 more: the four keys whose words lane tig reads lie in four rows next
      // to each other's, half as many bank conflicts as rows 2 t and 2 t + 1 give
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int ra = mt * 16 + pi, rb = ra + 8;
        const bool va = ra >= skip && ra < valid, vb = rb >= skip && rb < valid;
        const ValueScale sa = value_scale(Vu[ra]), sb = value_scale(Vu[rb]);
        const float t0 = aq_exp2(x[mt][0] + b0), t1 = aq_exp2(x[mt][1] + b1), t2 = aq_exp2(x[mt][2] + b0), t3 = aq_exp2(x[mt][3] + b1);
        l0 = fmaf(t0, sa.undo, fmaf(t2, sb.undo, l0));
        l1 = fmaf(t1, sa.undo, fmaf(t3, sb.undo, l1));
        const float w0 = va ? t0 * sa.f : 0.f, w1 = va ? t1 * sa.f : 0.f, w2 = vb ? t2 * sb.f : 0.f, w3 = vb ? t3 * sb.f : 0.f;
        uint32_t pa[TERMS], pb[TERMS];
        {
          const uint32_t ha = aq_pack(w0, w1), hb = aq_pack(w2, w3);
          pa[0] = aq_transpose8(ha);
          pb[0] = aq_transpose8(hb);
          if constexpr (TERMS == 2) {
            pa[1] = aq_transpose8(aq_rest(w0, w1, ha));
            pb[1] = aq_transpose8(aq_rest(w2, w3, hb));
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
    m0 = m1 = 0.f;
    l0 = l1 = CUDART_NAN_F;
  }
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, off);
    l1 += __shfl_xor_sync(0xffffffffu, l1, off);
  }
  // ---- the warp's partial into its own ring (no copy is on its way there any more), then the block's into `result`
  {
    float* wa = reinterpret_cast<float*>(ring) + (2 * tig) * WS;
    float* wb = wa + WS;
#pragma unroll
    for (int dt = 0; dt < HDT; ++dt) {
      const int d = gid * 2 * HDT + 2 * dt;
      *reinterpret_cast<float2*>(wa + d) = make_float2(o[dt][0] * AQ_OPERAND_BACK, o[dt][2] * AQ_OPERAND_BACK);
      *reinterpret_cast<float2*>(wb + d) = make_float2(o[dt][1] * AQ_OPERAND_BACK, o[dt][3] * AQ_OPERAND_BACK);
    }
    if (gid == 0) {
      *reinterpret_cast<float2*>(wa + HD) = make_float2(m0, l0);
      *reinterpret_cast<float2*>(wb + HD) = make_float2(m1, l1);
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
  for (int it = split * blockDim.x + threadIdx.x; it < heads * (HD / 2); it += splits * blockDim.x) {
    const int r = it / (HD / 2), d = (it - r * (HD / 2)) * 2;
    float2 ml[QD_MAX_SPLITS], v[QD_MAX_SPLITS];
#pragma unroll
    for (int c = 0; c < QD_MAX_SPLITS; ++c) {
      if (c < splits) {
        const float* pw = cluster.map_shared_rank(result, c) + r * WS;
        ml[c] = *reinterpret_cast<const float2*>(pw + HD);
        v[c] = *reinterpret_cast<const float2*>(pw + d);
      }
    }
    float M = -CUDART_INF_F, L = 0.f, a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < QD_MAX_SPLITS; ++c)
      if (c < splits) M = fmaxf(M, ml[c].x);
    const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
    for (int c = 0; c < QD_MAX_SPLITS; ++c) {
      if (c < splits) {
        const float f = aq_exp2(ml[c].x - ref);
        L = fmaf(ml[c].y, f, L);
        a = fmaf(v[c].x, f, a);
        b = fmaf(v[c].y, f, b);
      }
    }
    const float inv = nkeys > 0 ? 1.0f / L : 0.f;
    store2(r, d, a * inv, b * inv);
  }
  cluster.sync();   // no block ends while another reads its result
}

}  // namespace edgelm
