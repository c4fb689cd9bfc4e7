// Causal attention of many new tokens over the 8-bit cache on the fifth-generation tensor cores (tcgen05): bfloat16 models, head
// sizes up to 128.  The other head sizes, float32 models and sequences of one page stay on mma.sync (attention_quant_prefill.cuh).
//
// The tensor cores take float16 operands, so the codes become float16 on the chip.  Scales are applied 32 keys (a group) at a time: with
// 2^k and 2^e the largest powers of two in the group's key and value scales, the tiles hold a_j (u_j / 2^k) and c_j (v_j / 2^e), two more
// roundings to 11 bits each (the factor u_j / 2^k, which all of a key's products share, and its product with a code), and   x_ij = log2(e) scale 2^k (q_i . tile_j) + e,   t_ij = 2^(x_ij - M_i + 46),
// out_i = 2^40 sum (t_ij 2^-40) (tile_j) / sum t_ij 2^-e   (attention_quant.cuh, with one e a group).  A softmax thread has one group: two
// numbers for 32 scores.  (Scales applied a key at a time cost a thread four shared-memory reads for four scores, 16 bytes to every lane
// though all lanes read the same: 2,048 clocks a block of keys, twice its 1,024 of exponentials; 2,048 tokens of 32 heads of 64: 82 us, now 68.)
// Where a group's key or value scales differ by more than 2^8 the tiles hold its codes as they are and the thread takes the slow way,
// scales a key at a time: a row must not lose digits to a neighbour that it may not even see.  A row that is no number makes its key's
// tile one of not-a-numbers (or, the slow way, its factor): who sees the key sees NaN, and only numbers enter the product with the values.
// M moves only when a row's largest x has outgrown it by 2^8, so a weight is at most 2^15 as an operand.
//
// A block takes 128 (token, query head) rows of one kv head, token-major, and walks the keys that they see in blocks of two pages.
// Roles: warp 0 brings codes and scales (bulk copies, two stages); warps 4 to 7 turn them into swizzled float16 tiles (keys K-major, values
// MN-major as they lie) and factors; warp 1 issues S = Q K^T, warp 2 O += P V with P out of tensor memory; warps 8 to 23 are the
// softmax, four threads a row, a group each, which share the row's reference through shared memory.  S has two buffers of 128 columns,
// so that S of block j + 1 is computed beside the softmax of block j; the weights go back over the scores that they came from.
// Few rows over many keys (a short turn of a long conversation): a cluster of up to 8 blocks shares a row tile's key blocks, and the partial
// results meet in distributed shared memory in a fixed order.
// Bound by the softmax: a block of 128 keys takes 3,050 clocks (before the branch for scores far from zero, which costs 1 to 2 %), of them 630 to read and find the maxima, 440 at the exchange between a row's
// threads, 1,280 for exponents, weights and sums, 305 waiting for S; the matrix products fill a sixth of it.  All 16 warps stand at the
// same place; two teams of softmax warps on alternate blocks (28 warps, one block of keys behind the other) took 69.5 us for 68, and 88 for
// 78 at a head size of 128: the registers of a thread then hold half of what they do now.  2,048 tokens of 32 heads of 64, e4m3: 68 us, 253
// TFLOP/s by the products that the mask leaves; four turns of 65 to 701 tokens behind 1,501, 16 heads of 128 on 4, int8: 82 us.
// Every wait is bounded; where one runs out the block reports it, writes not-a-numbers and waits for what it has in flight before
// it gives its memory back.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>
#include <utility>

#include "attention_quant.cuh"
#include "tc_common.cuh"

namespace edgelm {

constexpr int QT_ROWS = 128, QT_KEYS = 128, QT_THREADS = 768, QT_SOFT_WARPS = 16, QT_GROUPS = 4, QT_CONVERTERS = 4, QT_MAX_SPLITS = 8;
constexpr int QT_TILE = 128 * 128;             // bytes of 128 rows of 64 float16
constexpr float QT_LAZY = 8.f;
constexpr int QT_SPREAD = 8;                   // powers of two between the scales of a group that tiles of scaled codes take
constexpr float QT_OPERAND = 9.094947017729282e-13f, QT_OPERAND_BACK = 1099511627776.f;    // 2^-40, 2^40

template <int HD> struct QtSizes {
  static constexpr int KC = (HD + 63) / 64;                   // tiles of 64 dims (what lies behind a row's end in the last is not read, or its products are not)
  static constexpr int KS = 2, VS = KC == 1 ? 2 : 1;          // stages of keys and values (shared memory has room for one of values at 128)
  static constexpr int CODES = QT_KEYS * (2 * HD + 8);        // a stage: key codes, value codes, key scales, value scales
  static constexpr int KEY_DATA = QT_GROUPS * 16 + 4 * QT_KEYS * 4;   // a block's groups {2^k, e, 2^-e, slow}, and of every key (where
                                                                      // its group is slow) u, e, f 2^-40, 2^-e; four blocks' worth
  // where things lie, from a 1,024-byte boundary on
  static constexpr int KEYS = KC * QT_TILE, VALUES = KEYS + KS * KC * QT_TILE, CODES_AT = VALUES + VS * KC * QT_TILE, KEY_DATA_AT = CODES_AT + 2 * CODES;
  static constexpr int ROW_MAX = KEY_DATA_AT + 4 * KEY_DATA;                      // [block & 1][group][128 rows]
  static constexpr int ROW_SUM = ROW_MAX + 2 * QT_GROUPS * QT_ROWS * 4;           // [group][128 rows]
  static constexpr int BARS = ROW_SUM + QT_GROUPS * QT_ROWS * 4;
  static constexpr int N_BARS = 1 + 2 + 2 + 2 * KS + 2 * VS + 2 + 2 + 2 + 4 + 1;
  static constexpr int needed = 1024 + BARS + N_BARS * 8 + 8;                     // (behind the barriers: the tensor memory's address and the abort flag)
  // one block an SM, whose tensor memory has room for one: a second would wait there for the first instead of going to the next free SM
  static constexpr int smem = needed > 114 * 1024 ? needed : 114 * 1024;
  static_assert(CODES % 16 == 0 && KEY_DATA % 16 == 0 && BARS % 8 == 0, "alignment");
  static_assert(2 * (smem + 1024) > 228 * 1024, "one block an SM");
};

// Instruction descriptor of kind::f16 with float16 operands: D float32, both K-major, M x N.
__host__ __device__ constexpr uint32_t qt_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

struct QuantTcArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const uint8_t *kcache, *vcache;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *seq_slot, *tile_seq, *tile_tok0, *tile_ntok, *tile_pos0;
  int* err;
  long long ldq, ldo;
  int table_stride, n_pages, nh, nkv, window, blocks_per_tile;
  float scale;
};

__device__ __forceinline__ uint64_t qt_pair(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 qt_unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t qt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t qt_mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t qt_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void qt_tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// A block's last wait for what it has in flight, bounded and without a report (the wait that ran out before has made one)
__device__ __forceinline__ void qt_drain(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try(bar, parity) && clock64() - t0 < TC_WAIT_CYCLES) {}
}
// where eight dims d .. d + 7 of row r lie in tiles of 128 rows of 64 float16 numbers, swizzled
__device__ __forceinline__ uint8_t* qt_place(uint8_t* tiles, int r, int d) { return tiles + d / 64 * QT_TILE + r * 128 + (((d % 64 / 8) ^ (r & 7)) << 4); }

template <int HD, int FMT>
__global__ void __launch_bounds__(QT_THREADS, 1)
attn_prefill_quant_tc_kernel(const QuantTcArgs a) {
  using Z = QtSizes<HD>;
  constexpr int KC = Z::KC, KS = Z::KS, VS = Z::VS;
  extern __shared__ uint8_t qt_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(qt_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_s = smem;                             // [KC][128 rows][128 bytes]
  uint8_t* k_s = smem + Z::KEYS;                   // [KS][KC][128 keys][128 bytes]
  uint8_t* v_s = smem + Z::VALUES;                 // [VS][KC][128 keys][128 bytes]
  uint8_t* codes = smem + Z::CODES_AT;             // [2][CODES]
  uint8_t* key_data = smem + Z::KEY_DATA_AT;       // [4][KEY_DATA]
  float* row_max = reinterpret_cast<float*>(smem + Z::ROW_MAX);
  float* row_sum = reinterpret_cast<float*>(smem + Z::ROW_SUM);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Z::BARS);
  uint64_t *q_ready = bars, *c_full = bars + 1, *c_empty = c_full + 2, *k_full = c_empty + 2, *k_empty = k_full + KS, *v_full = k_empty + KS;
  uint64_t *v_empty = v_full + VS, *s_ready = v_empty + VS, *p_ready = s_ready + 2, *o_done = p_ready + 2;
  uint64_t* d_full = o_done + 2;                   // [4] key factors
  uint64_t* all_done = d_full + 4;                 // both issuers' MMAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Z::N_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (uint64_t* b = bars; b < all_done; ++b)
      mbar_init(smem_u32(b), b == q_ready || (b >= p_ready && b < o_done) ? QT_SOFT_WARPS
                             : (b >= c_empty && b < k_empty) || (b >= v_full && b < v_empty) || b >= d_full ? QT_CONVERTERS : 1);
    mbar_init(smem_u32(all_done), 2);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();      // (behind the allocation: a block of the next kernel must not hold tensor memory that this one waits for)
  pdl_wait();

  const int splits = gridDim.x, split = blockIdx.x, g = a.nh / a.nkv, kvh = blockIdx.y, at = gridDim.z - 1 - blockIdx.z;      // (tiles of the most keys first)
  const int tile = at / a.blocks_per_tile, row_base = (at - tile * a.blocks_per_tile) * QT_ROWS;
  const int tok0 = a.tile_tok0[tile], rows_total = a.tile_ntok[tile] * g, pos0 = a.tile_pos0[tile];
  const int rows = min(QT_ROWS, rows_total - row_base);
  const int first_pos = pos0 + row_base / g, last_pos = pos0 + (row_base + max(rows, 1) - 1) / g;
  const int n_keys = last_pos + 1, page0 = a.window > 0 ? max(0, first_pos - a.window + 1) / PAGE : 0, n_pg = (n_keys + PAGE - 1) / PAGE - page0;
  const int all_blk = rows > 0 ? (n_pg + 1) / 2 : 0;   // (no rows: a block of a tile that has fewer tokens than the longest)
  const int n_blk = all_blk > split ? (all_blk - split + splits - 1) / splits : 0;     // this block's: split, split + splits, ..
  auto pages_ahead = [&](int j) { return 2 * (split + j * splits); };                  // of the j-th of them, from page0 on
  auto key_of = [&](int j) { return (page0 + pages_ahead(j)) * PAGE; };
  constexpr uint32_t S_COLS = 128, O_COL = 256;
  // scores in units of log 2; the scale's sign (or a scale of 0) goes to the queries, so that the largest product has the largest weight
  const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * AQ_LOG2E, turn = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
  auto wait = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, mbar_wait_parked(smem_u32(bar), (uint32_t)parity, abort_flag, a.err)); };

  // a block's results, where several share the rows: [128][dims, reference, sum], over its tiles of keys and values
  constexpr int RESULT_PITCH = HD + 2;
  static_assert(QT_ROWS * RESULT_PITCH * 4 <= (KS + VS) * KC * QT_TILE, "a block's results fit its tiles");
  float* result = reinterpret_cast<float*>(k_s);

  if (n_blk == 0) {
    if (splits > 1 && rows > 0)
      for (int i = threadIdx.x; i < QT_ROWS * RESULT_PITCH; i += QT_THREADS) result[i] = i % RESULT_PITCH == HD ? -CUDART_INF_F : 0.f;
  } else if (warp == 0) {
    // ---- codes and scales: lanes 0 to 3 the block's first page, 4 to 7 its second
    const int32_t* pages = a.page_table + (size_t)a.seq_slot[a.tile_seq[tile]] * a.table_stride;
    auto page_of = [&](int j) {
      const int ahead = pages_ahead(j) + (lane >> 2), i = page0 + ahead;
      int page = lane < 8 && j < n_blk && ahead < n_pg ? (i < a.table_stride ? pages[i] : -1) : 0;
      if (page < 0 || page >= a.n_pages) {
        atomicOr(a.err, ERR_PAGE_RANGE);
        page = 0;                                  // (reported; some page is read in its place)
      }
      return page;
    };
    int issued = 0, page = page_of(0);
    for (int j = 0; j < n_blk; ++j) {
      const int st = j & 1, both = pages_ahead(j) + 1 < n_pg ? 2 : 1;
      const int next = page_of(j + 1);
      if (j >= 2 && !wait(&c_empty[st], (j >> 1 & 1) ^ 1)) break;
      const uint32_t bar = smem_u32(&c_full[st]), dst = smem_u32(codes + st * Z::CODES);
      if (lane == 0) mbar_expect_tx(bar, both * PAGE * (2 * HD + 8));
      __syncwarp();
      if (lane < 4 * both) {
        const int h = lane >> 2, what = lane & 3;
        const size_t row = ((size_t)page * a.nkv + kvh) * PAGE;
        if (what < 2) aq_bulk(dst + what * QT_KEYS * HD + h * PAGE * HD, (what ? a.vcache : a.kcache) + row * HD, PAGE * HD, bar);
        else aq_bulk(dst + 2 * QT_KEYS * HD + (what - 2) * QT_KEYS * 4 + h * PAGE * 4, (what == 2 ? a.k_scale : a.v_scale) + row, PAGE * 4, bar);
      }
      issued = j + 1;
      page = next;
      __syncwarp();
    }
    // (also where a wait ran out: no copy may be on its way when the block's memory is given back)
    for (int i = max(0, issued - 2); i < issued; ++i) qt_drain(smem_u32(&c_full[i & 1]), i >> 1 & 1);
  } else if (warp == 1) {
    constexpr uint32_t idesc = qt_idesc(QT_ROWS, QT_KEYS);
    const bool leader = elect_one();
    const uint64_t dq = umma_desc(smem_u32(q_s));
    bool ok = wait(q_ready, 0);
    for (int j = 0; j < n_blk && ok; ++j) {
      const int b = j & 1, st = j % KS;
      if (j >= 2) ok = wait(&o_done[b], (j >> 1) - 1 & 1);            // (the block before last has left this buffer)
      if (ok) ok = wait(&k_full[st], j / KS & 1);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t dk = umma_desc(smem_u32(k_s + st * KC * QT_TILE));
      if (leader) {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
          umma_f16(tmem + b * S_COLS, dq + (s / 4 * QT_TILE >> 4) + 2 * (s % 4), dk + (s / 4 * QT_TILE >> 4) + 2 * (s % 4), idesc, s != 0);
        umma_commit(smem_u32(&s_ready[b]));
        umma_commit(smem_u32(&k_empty[st]));
      }
      __syncwarp();
    }
    if (leader) umma_commit(smem_u32(all_done));
    __syncwarp();
    qt_drain(smem_u32(all_done), 0);
  } else if (warp == 2) {
    constexpr uint32_t idesc = qt_idesc(QT_ROWS, 64) | (1u << 16);    // B (the values) is MN-major
    const bool leader = elect_one();
    bool ok = true;
    for (int j = 0; j < n_blk && ok; ++j) {
      const int b = j & 1, st = j % VS;
      ok = wait(&v_full[st], j / VS & 1) && wait(&p_ready[b], j >> 1 & 1);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t dv = umma_desc(smem_u32(v_s + st * KC * QT_TILE));
      if (leader) {
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int s = 0; s < 8; ++s)                                 // 16 keys: 8 columns of the weights of group s / 2
            umma_f16_ts(tmem + O_COL + c * 64, tmem + b * S_COLS + s / 2 * 32 + s % 2 * 8, (uint32_t)dv + (c * QT_TILE + s * 16 * 128 >> 4), (uint32_t)(dv >> 32), idesc,
                        j > 0 || s != 0);
        umma_commit(smem_u32(&o_done[b]));
        umma_commit(smem_u32(&v_empty[st]));
      }
      __syncwarp();
    }
    if (leader) umma_commit(smem_u32(all_done));
    __syncwarp();
    qt_drain(smem_u32(all_done), 0);
  } else if (warp >= 4 && warp < 8) {
    // ---- 32 keys a warp: their factors, and their codes as float16 tiles
    constexpr int PER_ROW = HD / 16;                                  // pieces of 16 codes, and passes over the warp's rows
    const int cw = warp - 4;
    for (int j = 0; j < n_blk; ++j) {
      const int cs = j & 1, ks = j % KS, vs = j % VS;
      if (!wait(&c_full[cs], j >> 1 & 1)) break;
      if (j >= KS && !wait(&k_empty[ks], (j / KS & 1) ^ 1)) break;    // (and with S of block j - 2 done, the softmax is done with block j - 4's factors)
      const uint8_t* src = codes + cs * Z::CODES + cw * 32 * HD;
      const float* scales = reinterpret_cast<const float*>(codes + cs * Z::CODES + 2 * QT_KEYS * HD) + cw * 32 + lane;
      const bool there = key_of(j) + cw * 32 + lane < n_keys;
      const float u = there ? scales[0] : 0.f, v = there ? scales[QT_KEYS] : 0.f;
      // the largest and smallest powers of two of the group's scales; rows that are no number, or as good as zero, have no say
      const int ub = (int)(__float_as_uint(u) >> 23 & 255u), vb = (int)(__float_as_uint(v) >> 23 & 255u);
      const bool fine = ub < 255 && vb < 255, counts = there && fine;
      constexpr int ZERO = 127 - 66;
      const int umax = __reduce_max_sync(0xffffffffu, counts ? max(ub, 1) : 1), umin = __reduce_min_sync(0xffffffffu, counts && ub > ZERO ? ub : 255);
      const int vmax = __reduce_max_sync(0xffffffffu, counts ? max(vb, 127 - 60) : 127 - 60), vmin = __reduce_min_sync(0xffffffffu, counts && vb > ZERO ? vb : 255);
      const bool slow = umax - umin > QT_SPREAD || vmax - vmin > QT_SPREAD;
      const float un_k = __uint_as_float((uint32_t)(254 - min(umax, 253)) << 23), un_e = __uint_as_float((uint32_t)(254 - min(vmax, 253)) << 23);
      float* kd = reinterpret_cast<float*>(key_data + (j & 3) * Z::KEY_DATA);
      if (lane == 0)
        reinterpret_cast<float4*>(kd)[cw] = make_float4(1.0f / un_k, (float)(min(vmax, 253) - 127), un_e, slow ? 1.f : 0.f);
      float mk = fine ? u * un_k : CUDART_NAN_F, mv = fine ? v * un_e : 0.f;
      if (slow) {
        const ValueScale vsc = value_scale(fine ? v : 0.f);
        kd += QT_GROUPS * 4 + cw * 32 + lane;
        kd[0] = fine ? u : CUDART_NAN_F;
        kd[QT_KEYS] = vsc.e;
        kd[2 * QT_KEYS] = vsc.f * (QT_OPERAND / AQ_OPERAND);
        kd[3 * QT_KEYS] = vsc.undo;
        mk = mv = 1.f;
      }
      const __half2 hk = __float2half2_rn(mk), hv = __float2half2_rn(mv);
      const uint32_t fk = *reinterpret_cast<const uint32_t*>(&hk), fv = *reinterpret_cast<const uint32_t*>(&hv);
      auto tile = [&](const uint8_t* from, uint8_t* to, uint32_t factor, bool values) {
        uint4 c[PER_ROW];
#pragma unroll
        for (int i = 0; i < PER_ROW; ++i) {
          const int r = (i * 32 + lane) / PER_ROW, d = (i * 32 + lane) % PER_ROW * 16;
          c[i] = *reinterpret_cast<const uint4*>(from + r * HD + d);
          if (values && key_of(j) + cw * 32 + r >= n_keys) c[i] = make_uint4(0, 0, 0, 0);      // whatever lies there, it meets weights of zero as zero
        }
#pragma unroll
        for (int i = 0; i < PER_ROW; ++i) {
          const int r = (i * 32 + lane) / PER_ROW, d = (i * 32 + lane) % PER_ROW * 16;
          const uint32_t fr = __shfl_sync(0xffffffffu, factor, r);
          uint32_t w[8];
          codes_to_half<FMT>(c[i].x, w[0], w[1]);
          codes_to_half<FMT>(c[i].y, w[2], w[3]);
          codes_to_half<FMT>(c[i].z, w[4], w[5]);
          codes_to_half<FMT>(c[i].w, w[6], w[7]);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&w[k]), *reinterpret_cast<const __half2*>(&fr));
            w[k] = *reinterpret_cast<const uint32_t*>(&x);
          }
          *reinterpret_cast<uint4*>(qt_place(to, cw * 32 + r, d)) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(qt_place(to, cw * 32 + r, d + 8)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      };
      tile(src, k_s + ks * KC * QT_TILE, fk, false);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&k_full[ks]));
        mbar_arrive(smem_u32(&d_full[j & 3]));
      }
      if (j >= VS && !wait(&v_empty[vs], (j / VS & 1) ^ 1)) break;
      tile(src + QT_KEYS * HD, v_s + vs * KC * QT_TILE, fv, true);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&v_full[vs]));
        mbar_arrive(smem_u32(&c_empty[cs]));
      }
    }
  } else if (warp >= 8) {
    const int part = (warp - 8) >> 2, quarter = warp & 3, row = quarter * 32 + lane;      // the group of each block, the row
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int rr = row_base + row, tok = rr / g;
    const bool mine = row < rows;
    auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(quarter + 1) : "memory"); };      // the row's four threads (warps w, w + 4, w + 8, w + 12)
    auto all_four = [&](const float* at) { return fmaxf(fmaxf(at[row], at[QT_ROWS + row]), fmaxf(at[2 * QT_ROWS + row], at[3 * QT_ROWS + row])); };
    // ---- this thread's pieces of eight numbers of its row (part, part + 4, ..) as float16 numbers, lifted by a power of two (exact)
    constexpr int PIECES = HD / 8, N = (PIECES + 3) / 4;
    float qf;
    {
      uint4 v[N];
      uint32_t most = 0;
      const __nv_bfloat16* src = a.q + (size_t)(tok0 + tok) * a.ldq + (size_t)(kvh * g + rr - tok * g) * HD;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = mine && part + 4 * i < PIECES ? *reinterpret_cast<const uint4*>(src + 8 * (part + 4 * i)) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(w[k] << 16 & 0x7fffffffu, w[k] & 0x7fff0000u));
      }
      // (magnitudes compare as whole numbers whatever they stand for: kept as such)
      uint32_t* at = reinterpret_cast<uint32_t*>(row_max);
      at[part * QT_ROWS + row] = most;
      meet();
      most = max(max(at[row], at[QT_ROWS + row]), max(at[2 * QT_ROWS + row], at[3 * QT_ROWS + row]));
      meet();                                      // (all have read, before the maxima are written over)
      const float lift = query_lift(most);
      qf = 1.0f / lift * scale2;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = aq_pack(__uint_as_float(w[k] << 16) * (lift * turn), __uint_as_float(w[k] & 0xffff0000u) * (lift * turn));
        if (part + 4 * i < PIECES) *reinterpret_cast<uint4*>(qt_place(q_s, row, 8 * (part + 4 * i))) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(q_ready));
    }
    const int pos = mine ? pos0 + tok : last_pos;
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_blk; ++j) {              // (also behind a wait that ran out: the row's other threads may be at the exchange)
      const int b = j & 1, key0 = key_of(j) + part * 32;
      const uint32_t s_addr = tmem + lanes + b * S_COLS + part * 32;
      const float4* gd = reinterpret_cast<const float4*>(key_data + (j & 3) * Z::KEY_DATA);
      const ulonglong2* kd = reinterpret_cast<const ulonglong2*>(gd + QT_GROUPS) + part * 8;      // (slow) four keys' u; 32 further their e, f, 2^-e
      if (ok) ok = wait(&d_full[j & 3], j >> 2 & 1) && wait(&s_ready[b], j >> 1 & 1);
      float x[32], f = 1.f, e = 0.f, mx = -CUDART_INF_F;
      float4 group = make_float4(0.f, 0.f, 0.f, 0.f);
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        group = gd[part];
        tmem_ld32(s_addr, reinterpret_cast<uint32_t*>(x));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (group.w == 0.f) {                      // x = f s + e, left to the exponent's multiply-add
          f = fmaxf(qf * group.x, 1e-37f);         // (above zero: minus infinity times it stays so)
          e = group.y;
        } else {
          const uint64_t f2 = qt_pair(qf, qf);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const ulonglong2 u = kd[i / 4], o = kd[32 + i / 4];
            const float2 y = qt_unpair(qt_fma2(qt_pair(x[i], x[i + 1]), qt_mul2(u.x, f2), o.x)), z = qt_unpair(qt_fma2(qt_pair(x[i + 2], x[i + 3]), qt_mul2(u.y, f2), o.y));
            x[i] = y.x;
            x[i + 1] = y.y;
            x[i + 2] = z.x;
            x[i + 3] = z.y;
          }
        }
        if (key0 + 31 > first_pos || (a.window > 0 && key0 <= last_pos - a.window)) {
          const int hi = pos - key0, lo = a.window > 0 ? hi - a.window : -1;      // keys lo + 1 .. hi of the thread's 32
          uint32_t seen = hi >= 31 ? ~0u : hi < 0 ? 0u : ~(~1u << hi);
          seen &= lo >= 31 ? 0u : lo < 0 ? ~0u : ~1u << lo;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen >> i & 1)) x[i] = -CUDART_INF_F;
        }
        float mx1 = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          mx = fmaxf(mx, fmaxf(x[i], x[i + 1]));
          mx1 = fmaxf(mx1, fmaxf(x[i + 2], x[i + 3]));
        }
        mx = fmaf(fmaxf(mx, mx1), f, e);
      }
      float* maxima = row_max + b * QT_GROUPS * QT_ROWS;
      maxima[part * QT_ROWS + row] = mx;
      meet();
      if (!ok) continue;
      mx = all_four(maxima);
      float rescale = 1.f;
      if (j == 0) {
        m = mx;
      } else if (mx - m > QT_LAZY) {              // (a difference: far from zero m + 8 may be m, or m + 16)
        rescale = aq_exp2(m - mx);                 // (0 if the row has seen no key so far)
        m = mx;
        l *= rescale;
      }
      if (__any_sync(0xffffffffu, rescale != 1.f)) {       // (rare after the first blocks; all four warps of the rows take it)
        ok = wait(&o_done[b ^ 1], (j - 1) >> 1 & 1);
        if (!ok) continue;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c = part; c < PIECES; c += 4) {
          uint32_t o[8];
          const uint32_t o_addr = tmem + lanes + O_COL + 8 * c;
          tmem_ld8(o_addr, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * rescale);
          qt_tmem_st8(o_addr, o);
        }
      }
      const float reference = m == -CUDART_INF_F ? 0.f : m;
      float bias = AQ_LIFT - reference;
      if (fabsf(reference) > AQ_FAR) {             // (attention_quant.cuh; x - M as it was rounded for the maximum)
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = fmaf(x[i], f, e) - reference;
        f = 1.f;
        e = 0.f;
        bias = AQ_LIFT;
      }
      const uint64_t f2 = qt_pair(f, f), bias2 = qt_pair(e + bias, e + bias);
      uint64_t sum0 = 0, sum1 = 0;
      if (group.w == 0.f) {
        const uint64_t operand2 = qt_pair(QT_OPERAND, QT_OPERAND);
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const float2 y = qt_unpair(qt_fma2(qt_pair(x[i + k], x[i + k + 1]), f2, bias2));
            const uint64_t t = qt_pair(aq_exp2(y.x), aq_exp2(y.y));
            if (k & 2) sum1 = qt_add2(sum1, t);
            else sum0 = qt_add2(sum0, t);
            const float2 p = qt_unpair(qt_mul2(t, operand2));
            w[k / 2] = aq_pack(p.x, p.y);
          }
          qt_tmem_st8(s_addr + i / 2, w);
        }
        const float2 sum = qt_unpair(qt_add2(sum0, sum1));
        l = fmaf(sum.x + sum.y, group.z, l);
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            const ulonglong2 f = kd[64 + (i + k) / 4], un = kd[96 + (i + k) / 4];
            const float2 y = qt_unpair(qt_fma2(qt_pair(x[i + k], x[i + k + 1]), f2, bias2)), z = qt_unpair(qt_fma2(qt_pair(x[i + k + 2], x[i + k + 3]), f2, bias2));
            const uint64_t t0 = qt_pair(aq_exp2(y.x), aq_exp2(y.y)), t1 = qt_pair(aq_exp2(z.x), aq_exp2(z.y));
            sum0 = qt_fma2(t0, un.x, sum0);
            sum1 = qt_fma2(t1, un.y, sum1);
            const float2 p0 = qt_unpair(qt_mul2(t0, f.x)), p1 = qt_unpair(qt_mul2(t1, f.y));
            w[k / 2] = aq_pack(p0.x, p0.y);
            w[k / 2 + 1] = aq_pack(p1.x, p1.y);
          }
          qt_tmem_st8(s_addr + i / 2, w);
        }
        const float2 sum = qt_unpair(qt_add2(sum0, sum1));
        l += sum.x + sum.y;
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&p_ready[b]));
    }
    if (ok) ok = wait(&o_done[(n_blk - 1) & 1], (n_blk - 1) >> 1 & 1);
    row_sum[part * QT_ROWS + row] = l;
    meet();
    const float sum = ok ? (row_sum[row] + row_sum[QT_ROWS + row]) + (row_sum[2 * QT_ROWS + row] + row_sum[3 * QT_ROWS + row])
                         : CUDART_NAN_F;           // a wait that ran out: nothing that could pass for a result
    const float inv = QT_OPERAND_BACK / sum;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (splits > 1) {                              // (every MMA has read its tiles: the results take their place)
      float* res = result + row * RESULT_PITCH;
#pragma unroll
      for (int c = part; c < PIECES; c += 4) {
        uint32_t o[8];
        tmem_ld8(tmem + lanes + O_COL + 8 * c, o);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int k = 0; k < 8; ++k) res[8 * c + k] = __uint_as_float(o[k]);
      }
      if (part == 0) {
        res[HD] = m;
        res[HD + 1] = sum;
      }
    }
    __nv_bfloat16* dst = a.out + (size_t)(tok0 + tok) * a.ldo + (size_t)(kvh * g + rr - tok * g) * HD;
#pragma unroll
    for (int c = part; c < PIECES; c += 4) {
      uint32_t o[8], h[4];
      tmem_ld8(tmem + lanes + O_COL + 8 * c, o);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(o[2 * k]) * inv, __uint_as_float(o[2 * k + 1]) * inv);
        h[k] = *reinterpret_cast<const uint32_t*>(&y);
      }
      if (mine && splits == 1) *reinterpret_cast<uint4*>(dst + 8 * c) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    __syncwarp();
  }
  if (splits > 1 && rows > 0) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int it = split * QT_THREADS + threadIdx.x; it < rows * (HD / 2); it += splits * QT_THREADS) {
      const int r = it / (HD / 2), d = (it - r * (HD / 2)) * 2;
      float2 ml[QT_MAX_SPLITS], v[QT_MAX_SPLITS];
#pragma unroll
      for (int c = 0; c < QT_MAX_SPLITS; ++c) {
        if (c < splits) {
          const float* from = cluster.map_shared_rank(result, c) + r * RESULT_PITCH;
          ml[c] = *reinterpret_cast<const float2*>(from + HD);
          v[c] = *reinterpret_cast<const float2*>(from + d);
        }
      }
      float M = -CUDART_INF_F, L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int c = 0; c < QT_MAX_SPLITS; ++c)
        if (c < splits) M = fmaxf(M, ml[c].x);
      const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
      for (int c = 0; c < QT_MAX_SPLITS; ++c) {
        if (c < splits) {
          const float f = aq_exp2(ml[c].x - ref);
          L = fmaf(ml[c].y, f, L);
          x = fmaf(v[c].x, f, x);
          y = fmaf(v[c].y, f, y);
        }
      }
      const float inv = QT_OPERAND_BACK / L;
      const int row = row_base + r, t = row / g;
      *reinterpret_cast<__nv_bfloat162*>(a.out + (size_t)(tok0 + t) * a.ldo + (size_t)(kvh * g + row - t * g) * HD + d) = __floats2bfloat162_rn(x * inv, y * inv);
    }
    cluster.sync();   // no block ends while another reads its result
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <int HD, int FMT>
static int launch_quant_tc(const QuantTcArgs& a, int n_tiles, int n_splits, cudaStream_t stream) {
  // A cluster's blocks wait for one another with their tensor memory in hand.  They take all of an SM's shared memory, so that no block of
  // another kernel's cluster (another stream's matrix product) can hold the tensor memory that one of them waits for and wait for another.
  constexpr int all = 227 * 1024;
  static_assert(QtSizes<HD>::smem <= all, "shared memory");
  const int smem = n_splits > 1 ? all : QtSizes<HD>::smem;
  auto kern = attn_prefill_quant_tc_kernel<HD, FMT>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, all);
  EL_REFUSE(e == cudaSuccess, "attn_prefill_quantized: %d bytes of shared memory refused: %s", all, cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n_splits, a.nkv, n_tiles * a.blocks_per_tile);
  cfg.blockDim = dim3(QT_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (n_splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = n_splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled() & 16) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, a);
  EL_REFUSE(le == cudaSuccess, "attn_prefill_quantized: launch failed: %s", cudaGetErrorString(le));
  return 0;
}

template <int... I>
static int launch_quant_tc_sizes(std::integer_sequence<int, I...>, const QuantTcArgs& a, int format, int hd, int n_tiles, int n_splits, cudaStream_t stream) {
  int rc = -1;
  ((hd == 16 * (I + 1) ? (void)(rc = format == QF_INT8 ? launch_quant_tc<16 * (I + 1), QF_INT8>(a, n_tiles, n_splits, stream)
                                                       : launch_quant_tc<16 * (I + 1), QF_FP8>(a, n_tiles, n_splits, stream)) : (void)0), ...);
  return rc;
}

// Rows of the operands are checked by the entry point (attention_quant.cu); this form also wants 16-byte rows of queries and outputs.
bool prefill_quant_tc_takes(const void* q, long long ldq, const void* out, long long ldo, int dtype, int hd) {
  return dtype == DT_BF16 && hd % 16 == 0 && hd >= 16 && hd <= 128 && (uintptr_t)q % 16 == 0 && ldq % 8 == 0 && (uintptr_t)out % 16 == 0 && ldo % 8 == 0;
}

int launch_prefill_quant_tc(const void* q, long long ldq, void* out, long long ldo, const void* kcache, const void* vcache, const float* k_scale,
                            const float* v_scale, int format, const int32_t* page_table, int table_stride, int n_pages, const int32_t* seq_slot,
                            const int32_t* tile_seq, const int32_t* tile_tok0, const int32_t* tile_ntok, const int32_t* tile_pos0, int n_tiles,
                            int max_tile_tokens, int nh, int nkv, int hd, float scale, int n_splits, int max_keys, int window, int* err, cudaStream_t stream) {
  const int per_tile = (max_tile_tokens * (nh / nkv) + QT_ROWS - 1) / QT_ROWS;
  EL_REFUSE((long long)n_tiles * per_tile <= 65535, "attn_prefill_quantized: %d tiles of %d blocks (takes up to 65,535 blocks a kv head)", n_tiles, per_tile);
  if (n_splits == 0) {
    // Blocks that share a row tile's keys: what one wave of blocks, one an SM, leaves free (a quarter of the SMs stays out of the count: clusters
    // lie within a GPC), as long as each has a block of keys and more.  17 new tokens of 9 heads of 64 on 3 behind 4,000: 54.7 us with one block, 13.9 with 8.
    const long long blocks = (long long)nkv * n_tiles * per_tile;
    n_splits = (int)std::max(1LL, std::min({(long long)QT_MAX_SPLITS, 111 / blocks, (long long)max_keys / QT_KEYS - 1}));
  }
  const QuantTcArgs a = {(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const uint8_t*)kcache, (const uint8_t*)vcache, k_scale, v_scale, page_table, seq_slot,
                         tile_seq, tile_tok0, tile_ntok, tile_pos0, err, ldq, ldo, table_stride, n_pages, nh, nkv, window, per_tile, scale};
  return launch_quant_tc_sizes(std::make_integer_sequence<int, 8>{}, a, format, hd, n_tiles, n_splits, stream);
}

}  // namespace edgelm
