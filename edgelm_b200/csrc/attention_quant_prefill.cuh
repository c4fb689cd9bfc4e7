// Causal attention of many new tokens over the 8-bit cache on mma.sync tensor cores (any head size, bfloat16 and float32 models).
//
// A block takes 64 (token, query head) rows of one kv head, token-major, so that all query heads of a kv head share what is read; a
// warp owns 16 of them.  A tile of keys (64, from head size 144 on 32) arrives as four bulk copies of codes and scales into a ring
// of two stages; the block's threads turn it ONCE into float16 rows (padded by 16 bytes, so that ldmatrix reads hit distinct
// banks) and per key {u, e, f, 2^-e} (attention_quant.cuh), one tile ahead of the one that is being multiplied.  A tile's
// weighted values are a sum of their own that joins the running one by a rounded multiply-add.
//
// Few rows over many keys (a short turn of a long conversation): a cluster of up to 8 blocks shares a row tile's keys, and the
// partial results meet in distributed shared memory in a fixed order.
//
// Bound by a block's own chain, not by its operations: a warp has the products and exponents of 16 rows by itself, 3,600 clocks a tile of 64
// keys (float32, head size 64: two terms of queries and weights), and two or three blocks of four warps an SM.  61 to 701 new tokens of
// 9 heads of 64 on 3, three sequences, float32, e4m3: 22 us; 2,048 tokens 59; 64 tokens 6.0.
#pragma once
#include <cooperative_groups.h>

#include "attention_quant.cuh"

namespace edgelm {

constexpr int QP_ROWS = 64, QP_THREADS = 128, QP_STAGES = 2, QP_MAX_SPLITS = 8;

__host__ __device__ constexpr int qp_tile_keys(int hdt) { return hdt <= 8 ? 64 : 32; }
__host__ __device__ constexpr int qp_align(int b) { return (b + 127) / 128 * 128; }
__host__ __device__ constexpr int qp_stage_bytes(int hdt) { return qp_align(qp_tile_keys(hdt) * (2 * hdt * 16 + 8)); }
// barriers | factors [64] | queries [terms][64][hd + 8] | {u, e, f, undo} [2][keys] | codes | keys and values [2][2][keys][hd + 8]
__host__ __device__ constexpr int qp_off_queries() { return 128 + QP_ROWS * 4; }
__host__ __device__ constexpr int qp_off_key_data(int hdt, int terms) { return qp_align(qp_off_queries() + terms * QP_ROWS * (hdt * 16 + 8) * 2); }
__host__ __device__ constexpr int qp_off_codes(int hdt, int terms) { return qp_align(qp_off_key_data(hdt, terms) + 2 * qp_tile_keys(hdt) * 16); }
__host__ __device__ constexpr int qp_off_halves(int hdt, int terms) { return qp_off_codes(hdt, terms) + QP_STAGES * qp_stage_bytes(hdt); }
__host__ __device__ constexpr int qp_halves_bytes(int hdt) { return 2 * 2 * qp_tile_keys(hdt) * (hdt * 16 + 8) * 2; }
// over the halves, once they are done with: rows of {numbers, reference, sum, -, -}, and what each block's rows count for
__host__ __device__ constexpr int qp_result_bytes(int hdt) { return QP_ROWS * (hdt * 16 + 4 + QP_MAX_SPLITS) * 4; }
__host__ __device__ constexpr int qp_smem(int hdt, int terms) {
  return qp_off_halves(hdt, terms) + (qp_halves_bytes(hdt) > qp_result_bytes(hdt) ? qp_halves_bytes(hdt) : qp_result_bytes(hdt));
}

struct QuantPrefillArgs {
  const void* q;
  void* out;
  const uint8_t *kcache, *vcache;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *seq_slot, *tile_seq, *tile_tok0, *tile_ntok, *tile_pos0;
  int* err;
  long long ldq, ldo;
  int table_stride, n_pages, nh, nkv, window, blocks_per_tile, max_keys;
  float scale;
};

__device__ __forceinline__ void aq_ldmatrix_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void aq_ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}

template <int HDT, int FMT, typename T>
__global__ void __launch_bounds__(QP_THREADS)
attn_prefill_quant_kernel(const QuantPrefillArgs p) {
  constexpr int HD = HDT * 16, TERMS = sizeof(T) == 4 ? 2 : 1, PITCH = HD + 8, KT = qp_tile_keys(HDT), NT = KT / 8, STAGE = qp_stage_bytes(HDT);
  extern __shared__ __align__(128) uint8_t qp_raw[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(qp_raw);
  float* factors = reinterpret_cast<float*>(qp_raw + 128);
  __half* Qs = reinterpret_cast<__half*>(qp_raw + qp_off_queries());
  float4* key_data = reinterpret_cast<float4*>(qp_raw + qp_off_key_data(HDT, TERMS));     // [2][KT]
  uint8_t* codes = qp_raw + qp_off_codes(HDT, TERMS);
  __half* halves = reinterpret_cast<__half*>(qp_raw + qp_off_halves(HDT, TERMS));         // [2][keys, values][KT][PITCH]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3, mi = lane >> 3;
  const int splits = gridDim.x, split = blockIdx.x, kvh = blockIdx.y, g = p.nh / p.nkv;
  pdl_launch_dependents();
  if (threadIdx.x < QP_STAGES) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(aq_smem(&bars[threadIdx.x])));
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  const int at = gridDim.z - 1 - blockIdx.z, tile = at / p.blocks_per_tile, row_base = (at - tile * p.blocks_per_tile) * QP_ROWS;   // (tiles of the most keys first)
  const int tok0 = p.tile_tok0[tile], ntok = p.tile_ntok[tile], pos0 = p.tile_pos0[tile];
  const int rows_total = ntok * g;
  if (row_base >= rows_total) return;     // (every block of the cluster)
  const int rows = min(QP_ROWS, rows_total - row_base);
  const int32_t* pages = p.page_table + (size_t)p.seq_slot[p.tile_seq[tile]] * p.table_stride;
  const int first_pos = pos0 + row_base / g, last_pos = pos0 + (row_base + rows - 1) / g;
  const int nkeys = last_pos + 1, tile0 = p.window > 0 ? max(0, first_pos - p.window + 1) / KT : 0;
  const int all_tiles = (nkeys + KT - 1) / KT - tile0;
  const int n_tiles = all_tiles > split ? (all_tiles - split + splits - 1) / splits : 0;   // this block's: split, split + splits, ..

  auto key0_of = [&](int i) { return (tile0 + split + i * splits) * KT; };
  auto page_of = [&](int i) {
    const int at = i < n_tiles ? key0_of(i) / PAGE : p.table_stride;
    int page = at < p.table_stride ? pages[at] : -1;
    if (i < n_tiles && (page < 0 || page >= p.n_pages)) {
      if (p.err) atomicOr(p.err, ERR_PAGE_RANGE);
      page = -1;
    }
    return max(page, 0);      // (a page that is not there: reported, and some other one read in its place)
  };
  int my_page = 0;
  if (warp == 0) my_page = page_of(lane);
  auto issue = [&](int i) {   // warp 0: the i-th tile's codes into stage i % QP_STAGES
    const int page = __shfl_sync(0xffffffffu, my_page, i % 32);
    const int s = i % QP_STAGES;
    const uint32_t bar = aq_smem(&bars[s]), dst = aq_smem(codes + s * STAGE);
    const size_t at = ((size_t)page * p.nkv + kvh) * PAGE + key0_of(i) % PAGE;
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(KT * (2 * HD + 8)) : "memory");
    __syncwarp();
    if (lane == 0) aq_bulk(dst, p.kcache + at * HD, KT * HD, bar);
    if (lane == 1) aq_bulk(dst + KT * HD, p.vcache + at * HD, KT * HD, bar);
    if (lane == 2) aq_bulk(dst + 2 * KT * HD, p.k_scale + at, KT * 4, bar);
    if (lane == 3) aq_bulk(dst + 2 * KT * HD + KT * 4, p.v_scale + at, KT * 4, bar);
  };
  __syncthreads();     // the barriers are there
  if (warp == 0) {
    if (n_tiles > 0) issue(0);
    if (n_tiles > 1) issue(1);
  }
  // ---- the warp's query rows as float16 terms, two lanes a row, the row read before any of it is written.  (A row at a time by the whole
  // warp cost sixteen times a read's latency and a division: 16,000 clocks a block, 64 new tokens of 9 heads of 64 13 us.)
  {
    const int row = warp * 16 + (lane >> 1), rr = row_base + row, tok = rr / g;
    const T* src = reinterpret_cast<const T*>(p.q) + (size_t)(tok0 + tok) * p.ldq + (size_t)(kvh * g + rr - tok * g) * HD + (lane & 1) * 4;
    float4 v[2 * HDT];
#pragma unroll
    for (int i = 0; i < 2 * HDT; ++i) v[i] = row < rows ? load_piece(src + 8 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 2 * HDT; ++i) most = max(most, max(max(magnitude_bits(v[i].x), magnitude_bits(v[i].y)), max(magnitude_bits(v[i].z), magnitude_bits(v[i].w))));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const float lift = query_lift(most);
    __half* dst = Qs + row * PITCH + (lane & 1) * 4;
#pragma unroll
    for (int i = 0; i < 2 * HDT; ++i) {
      const float x0 = v[i].x * lift, x1 = v[i].y * lift, x2 = v[i].z * lift, x3 = v[i].w * lift;
      const uint32_t lo = aq_pack(x0, x1), hi = aq_pack(x2, x3);
      *reinterpret_cast<uint2*>(dst + 8 * i) = make_uint2(lo, hi);
      if (TERMS == 2) *reinterpret_cast<uint2*>(dst + QP_ROWS * PITCH + 8 * i) = make_uint2(aq_rest(x0, x1, lo), aq_rest(x2, x3, hi));
    }
    if ((lane & 1) == 0) factors[row] = 1.0f / lift * (p.scale * AQ_LOG2E);
  }
  __syncwarp();
  const int ra = warp * 16 + gid, rb = ra + 8;             // this lane's rows
  const float qa = factors[ra], qb = factors[rb];
  const int pos_a = ra < rows ? pos0 + (row_base + ra) / g : -1, pos_b = rb < rows ? pos0 + (row_base + rb) / g : -1;   // -1: no row, it sees nothing
  const int low_a = p.window > 0 ? pos_a - p.window : -1, low_b = p.window > 0 ? pos_b - p.window : -1;                  // keys above these
  const int warp_first = pos0 + (row_base + min(warp * 16, rows - 1)) / g, warp_last = pos0 + (row_base + min(warp * 16 + 15, rows - 1)) / g;
  const bool whole_warp = warp * 16 + 15 < rows;

  auto convert = [&](int i) {   // all threads: tile i from its codes
    const int b = i & 1, key0 = key0_of(i), valid = min(KT, nkeys - key0);
    const uint8_t* src = codes + (i % QP_STAGES) * STAGE;
    __half* dst = halves + b * 2 * KT * PITCH;
    for (int j = threadIdx.x; j < 2 * KT * HDT; j += QP_THREADS) {
      const int row = j / HDT, d = (j - row * HDT) * 16;
      uint4 c = *reinterpret_cast<const uint4*>(src + (size_t)j * 16);
      if (row >= KT + valid) c = make_uint4(0, 0, 0, 0);   // values behind this block's last key: whatever is there, it meets weights of zero as zero
      uint4 lo, hi;
      codes_to_half<FMT>(c.x, lo.x, lo.y);
      codes_to_half<FMT>(c.y, lo.z, lo.w);
      codes_to_half<FMT>(c.z, hi.x, hi.y);
      codes_to_half<FMT>(c.w, hi.z, hi.w);
      *reinterpret_cast<uint4*>(dst + row * PITCH + d) = lo;
      *reinterpret_cast<uint4*>(dst + row * PITCH + d + 8) = hi;
    }
    if (threadIdx.x < KT) {
      const float* u = reinterpret_cast<const float*>(src + 2 * KT * HD);
      const ValueScale s = value_scale(u[KT + threadIdx.x]);
      key_data[b * KT + threadIdx.x] = make_float4(u[threadIdx.x], s.e, s.f, s.undo);
    }
  };
  float o[2 * HDT][4];
#pragma unroll
  for (int i = 0; i < 2 * HDT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float ma = -CUDART_INF_F, mb = -CUDART_INF_F, la = 0.f, lb = 0.f;

  bool arrived = n_tiles == 0 || aq_wait(aq_smem(&bars[0]), 0);
  bool failed = __syncthreads_or(!arrived);
  if (n_tiles > 0 && !failed) convert(0);
  __syncthreads();
  int i = 0;
  for (; i < n_tiles && !failed; ++i) {
    if (warp == 0 && i + 2 < n_tiles) {
      if ((i + 2) % 32 == 0) my_page = page_of(i + 2 + lane);
      issue(i + 2);
    }
    if (i + 1 < n_tiles) {
      arrived = aq_wait(aq_smem(&bars[(i + 1) % QP_STAGES]), (i + 1) / QP_STAGES & 1);
      if (arrived) convert(i + 1);
    }
    const int key0 = key0_of(i);
    if (key0 <= warp_last && (p.window == 0 || key0 + KT - 1 > warp_first - p.window)) {    // (else no row of the warp sees the tile)
      const __half* Kt = halves + (i & 1) * 2 * KT * PITCH;
      const __half* Vt = Kt + KT * PITCH;
      const float4* kd = key_data + (i & 1) * KT;
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < HDT; ++ks) {
        uint32_t a[TERMS][4];
#pragma unroll
        for (int tm = 0; tm < TERMS; ++tm)
          aq_ldmatrix_x4(aq_smem(Qs + (tm * QP_ROWS + warp * 16 + (mi & 1) * 8 + (lane & 7)) * PITCH + ks * 16 + (mi >> 1) * 8), a[tm][0], a[tm][1], a[tm][2], a[tm][3]);
#pragma unroll
        for (int nt = 0; nt < NT; nt += 2) {
          uint32_t b0, b1, b2, b3;
          aq_ldmatrix_x4(aq_smem(Kt + ((nt + (mi >> 1)) * 8 + (lane & 7)) * PITCH + ks * 16 + (mi & 1) * 8), b0, b1, b2, b3);
#pragma unroll
          for (int tm = TERMS - 1; tm >= 0; --tm) {
            aq_mma(s[nt], a[tm][0], a[tm][1], a[tm][2], a[tm][3], b0, b1);
            aq_mma(s[nt + 1], a[tm][0], a[tm][1], a[tm][2], a[tm][3], b2, b3);
          }
        }
      }
      const bool masked = !whole_warp || key0 + KT - 1 > warp_first || (p.window > 0 && key0 <= warp_last - p.window);
      float xa = -CUDART_INF_F, xb = -CUDART_INF_F;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int key = key0 + nt * 8 + 2 * tig;
        const float2 k0 = *reinterpret_cast<const float2*>(&kd[nt * 8 + 2 * tig]), k1 = *reinterpret_cast<const float2*>(&kd[nt * 8 + 2 * tig + 1]);
        s[nt][0] = fmaf(s[nt][0], qa * k0.x, k0.y);
        s[nt][1] = fmaf(s[nt][1], qa * k1.x, k1.y);
        s[nt][2] = fmaf(s[nt][2], qb * k0.x, k0.y);
        s[nt][3] = fmaf(s[nt][3], qb * k1.x, k1.y);
        if (masked) {
          if (key > pos_a || key <= low_a) s[nt][0] = -CUDART_INF_F;
          if (key + 1 > pos_a || key + 1 <= low_a) s[nt][1] = -CUDART_INF_F;
          if (key > pos_b || key <= low_b) s[nt][2] = -CUDART_INF_F;
          if (key + 1 > pos_b || key + 1 <= low_b) s[nt][3] = -CUDART_INF_F;
        }
        xa = fmaxf(xa, fmaxf(s[nt][0], s[nt][1]));
        xb = fmaxf(xb, fmaxf(s[nt][2], s[nt][3]));
      }
      xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 1));
      xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 2));
      xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 1));
      xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 2));
      xa = fmaxf(xa, ma);
      xb = fmaxf(xb, mb);
      const float ref_a = xa == -CUDART_INF_F ? 0.f : xa, ref_b = xb == -CUDART_INF_F ? 0.f : xb;
      const float fa = aq_exp2(ma - ref_a), fb = aq_exp2(mb - ref_b);
      ma = xa;
      mb = xb;
      la *= fa;
      lb *= fb;
      uint32_t w[TERMS][NT][2];      // the weights as the A operand: rows gid and gid + 8, keys 2 tig and the next of every 8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 k0 = *(reinterpret_cast<const float2*>(&kd[nt * 8 + 2 * tig]) + 1), k1 = *(reinterpret_cast<const float2*>(&kd[nt * 8 + 2 * tig + 1]) + 1);
        const float t0 = aq_exp2(s[nt][0] - ref_a + AQ_LIFT), t1 = aq_exp2(s[nt][1] - ref_a + AQ_LIFT), t2 = aq_exp2(s[nt][2] - ref_b + AQ_LIFT), t3 = aq_exp2(s[nt][3] - ref_b + AQ_LIFT);
        la = fmaf(t0, k0.y, fmaf(t1, k1.y, la));
        lb = fmaf(t2, k0.y, fmaf(t3, k1.y, lb));
        float w0 = t0 * k0.x, w1 = t1 * k1.x, w2 = t2 * k0.x, w3 = t3 * k1.x;
        if (masked) {      // (a key that a row does not see may be a row of no numbers)
          if (s[nt][0] == -CUDART_INF_F) w0 = 0.f;
          if (s[nt][1] == -CUDART_INF_F) w1 = 0.f;
          if (s[nt][2] == -CUDART_INF_F) w2 = 0.f;
          if (s[nt][3] == -CUDART_INF_F) w3 = 0.f;
        }
        w[0][nt][0] = aq_pack(w0, w1);
        w[0][nt][1] = aq_pack(w2, w3);
        if constexpr (TERMS == 2) {
          w[1][nt][0] = aq_rest(w0, w1, w[0][nt][0]);
          w[1][nt][1] = aq_rest(w2, w3, w[0][nt][1]);
        }
      }
#pragma unroll
      for (int dt = 0; dt < 2 * HDT; dt += 2) {
        float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kt = 0; kt < NT / 2; ++kt) {
          uint32_t b0, b1, b2, b3;
          aq_ldmatrix_x4_trans(aq_smem(Vt + (kt * 16 + (mi & 1) * 8 + (lane & 7)) * PITCH + (dt + (mi >> 1)) * 8), b0, b1, b2, b3);
#pragma unroll
          for (int tm = TERMS - 1; tm >= 0; --tm) {
            aq_mma(c0, w[tm][2 * kt][0], w[tm][2 * kt][1], w[tm][2 * kt + 1][0], w[tm][2 * kt + 1][1], b0, b1);
            aq_mma(c1, w[tm][2 * kt][0], w[tm][2 * kt][1], w[tm][2 * kt + 1][0], w[tm][2 * kt + 1][1], b2, b3);
          }
        }
        o[dt][0] = fmaf(o[dt][0], fa, c0[0]);
        o[dt][1] = fmaf(o[dt][1], fa, c0[1]);
        o[dt][2] = fmaf(o[dt][2], fb, c0[2]);
        o[dt][3] = fmaf(o[dt][3], fb, c0[3]);
        o[dt + 1][0] = fmaf(o[dt + 1][0], fa, c1[0]);
        o[dt + 1][1] = fmaf(o[dt + 1][1], fa, c1[1]);
        o[dt + 1][2] = fmaf(o[dt + 1][2], fb, c1[2]);
        o[dt + 1][3] = fmaf(o[dt + 1][3], fb, c1[3]);
      }
    }
    failed = __syncthreads_or(!arrived);
  }
  if (failed) {   // a copy did not arrive: report, wait (again within bounds) for what else is on its way, and make the rows unmistakably wrong
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);
    const int issued = min(n_tiles, i + QP_STAGES);     // (an iteration issues one tile, and the first two were before them)
    for (int k = max(0, issued - QP_STAGES); k < issued; ++k) aq_wait(aq_smem(&bars[k % QP_STAGES]), k / QP_STAGES & 1);
    ma = mb = 0.f;
    la = lb = CUDART_NAN_F;
  }
  la += __shfl_xor_sync(0xffffffffu, la, 1);
  la += __shfl_xor_sync(0xffffffffu, la, 2);
  lb += __shfl_xor_sync(0xffffffffu, lb, 1);
  lb += __shfl_xor_sync(0xffffffffu, lb, 2);
  T* out = reinterpret_cast<T*>(p.out);
  auto place = [&](int row) {
    const int rr = row_base + row, tok = rr / g;
    return out + (size_t)(tok0 + tok) * p.ldo + (size_t)(kvh * g + rr - tok * g) * HD;
  };
  auto store2 = [](T* dst, float a, float b) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(dst) = make_float2(a, b);
    else *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(a, b);
  };
  if (splits == 1) {
    const float ia = AQ_OPERAND_BACK / la, ib = AQ_OPERAND_BACK / lb;
    T *da = ra < rows ? place(ra) : nullptr, *db = rb < rows ? place(rb) : nullptr;
#pragma unroll
    for (int dt = 0; dt < 2 * HDT; ++dt) {
      if (da) store2(da + dt * 8 + 2 * tig, o[dt][0] * ia, o[dt][1] * ia);
      if (db) store2(db + dt * 8 + 2 * tig, o[dt][2] * ib, o[dt][3] * ib);
    }
    return;
  }
  constexpr int WS = HD + 4;
  float* result = reinterpret_cast<float*>(halves);        // (the loop's last barrier is behind every read of the halves)
#pragma unroll
  for (int dt = 0; dt < 2 * HDT; ++dt) {
    *reinterpret_cast<float2*>(result + ra * WS + dt * 8 + 2 * tig) = make_float2(o[dt][0] * AQ_OPERAND_BACK, o[dt][1] * AQ_OPERAND_BACK);
    *reinterpret_cast<float2*>(result + rb * WS + dt * 8 + 2 * tig) = make_float2(o[dt][2] * AQ_OPERAND_BACK, o[dt][3] * AQ_OPERAND_BACK);
  }
  if (tig == 0) {
    *reinterpret_cast<float2*>(result + ra * WS + HD) = make_float2(ma, la);
    *reinterpret_cast<float2*>(result + rb * WS + HD) = make_float2(mb, lb);
  }
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  float* counts = result + QP_ROWS * WS;                   // [row][block]
  if (threadIdx.x < rows) {
    float2 ml[QP_MAX_SPLITS];
    float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
    for (int c = 0; c < QP_MAX_SPLITS; ++c)
      if (c < splits) ml[c] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(result, c) + threadIdx.x * WS + HD);
#pragma unroll
    for (int c = 0; c < QP_MAX_SPLITS; ++c)
      if (c < splits) M = fmaxf(M, ml[c].x);
    const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
    for (int c = 0; c < QP_MAX_SPLITS; ++c) {
      if (c < splits) {
        ml[c].x = aq_exp2(ml[c].x - ref);
        L = fmaf(ml[c].y, ml[c].x, L);
      }
    }
    const float inv = 1.0f / L;
#pragma unroll
    for (int c = 0; c < QP_MAX_SPLITS; ++c)
      if (c < splits) counts[threadIdx.x * QP_MAX_SPLITS + c] = ml[c].x * inv;
  }
  __syncthreads();
  // four numbers a piece, two pieces of every block's on their way at a time
  constexpr int PER_ROW = HD / 4;
  for (int it = split * QP_THREADS + threadIdx.x; it < rows * PER_ROW; it += 2 * splits * QP_THREADS) {
    const int at[2] = {it, it + splits * QP_THREADS};
    float4 v[2][QP_MAX_SPLITS];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < QP_MAX_SPLITS; ++c)
        if (c < splits && at[k] < rows * PER_ROW)
          v[k][c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(result, c) + at[k] / PER_ROW * WS + at[k] % PER_ROW * 4);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (at[k] >= rows * PER_ROW) continue;
      const int r = at[k] / PER_ROW, d = at[k] % PER_ROW * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < QP_MAX_SPLITS; ++c) {
        if (c < splits) {
          const float f = counts[r * QP_MAX_SPLITS + c];
          x = make_float4(fmaf(v[k][c].x, f, x.x), fmaf(v[k][c].y, f, x.y), fmaf(v[k][c].z, f, x.z), fmaf(v[k][c].w, f, x.w));
        }
      }
      T* dst = place(r) + d;
      store2(dst, x.x, x.y);
      store2(dst + 2, x.z, x.w);
    }
  }
  cluster.sync();   // no block ends while another reads its result
}

}  // namespace edgelm
