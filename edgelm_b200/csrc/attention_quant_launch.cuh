// Host side of the attention over the 8-bit cache: one instantiation a head size, format and type (a source file a kernel and format).
#pragma once
#include <algorithm>
#include <atomic>
#include <utility>

#include "attention_quant_decode.cuh"
#include "attention_quant_prefill.cuh"

namespace edgelm {

// What a kernel needs once a device (a bit a device): its shared memory.
template <typename K>
static cudaError_t quant_kernel_ready(K kern, int smem, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && done.load(std::memory_order_acquire) >> dev & 1)) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return e;
}

template <typename K, typename A>
static cudaError_t launch_quant_kernel(K kern, dim3 grid, int cluster, int threads, int smem, int pdl_bit, const A& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {      // the blocks that share keys
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled() & pdl_bit) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int FMT, typename T, int HDT, int HC>
static cudaError_t launch_decode_quant_heads(const QuantDecodeArgs& p, int n_seqs, int n_splits, int warps, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  auto kern = attn_decode_quant_kernel<HDT, FMT, HC, T>;
  const cudaError_t e = quant_kernel_ready(kern, qd_smem(HDT, TERMS, QD_MAX_WARPS), done);
  if (e != cudaSuccess) return e;
  const int chunks = (p.nh / p.nkv + QD_HEADS - 1) / QD_HEADS;
  return launch_quant_kernel(kern, dim3(n_splits, p.nkv * chunks, n_seqs), p.cluster, warps * 32, qd_smem(HDT, TERMS, warps), 2, p, stream);
}
template <int FMT, typename T, int HDT>
static cudaError_t launch_decode_quant_one(const QuantDecodeArgs& p, int n_seqs, int n_splits, int warps, cudaStream_t stream) {
  return p.nh / p.nkv <= QD_HEADS / 2 ? launch_decode_quant_heads<FMT, T, HDT, 1>(p, n_seqs, n_splits, warps, stream)
                                      : launch_decode_quant_heads<FMT, T, HDT, 2>(p, n_seqs, n_splits, warps, stream);
}

template <int FMT, typename T, int HDT>
static cudaError_t launch_prefill_quant_one(const QuantPrefillArgs& p, int n_tiles, int n_splits, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  auto kern = attn_prefill_quant_kernel<HDT, FMT, T>;
  cudaError_t e = quant_kernel_ready(kern, qp_smem(HDT, TERMS), done);
  if (e != cudaSuccess) return e;
  if (n_splits == 0) {
    // Blocks that share a row tile's keys: as many as make one wave, two tiles of keys each at the least; or up to two waves where each
    // has four (the last rows of a prompt see twice the average's keys, and the tiles of the most keys go first).  us with 1, 2, 3 and 8 blocks,
    // float32: 180 row tiles of up to 701 keys (9 heads of 64 on 3) 30, 22, 23, 52; 288 of up to 2,000 85, 55, 69, 121; 432 of up to
    // 300 23, 33, 40, 107; 96 of 1,600 to 1,700 (16 heads of 128 on 4) 93, 93, 72, 114.
    static std::atomic<int> resident{0};
    int per_sm = resident.load(std::memory_order_relaxed);
    if (per_sm == 0) {
      if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, QP_THREADS, qp_smem(HDT, TERMS))) != cudaSuccess) return e;
      resident.store(per_sm, std::memory_order_relaxed);
    }
    const long long blocks = (long long)p.nkv * n_tiles * p.blocks_per_tile, wave = 148LL * per_sm, tiles = p.max_keys / qp_tile_keys(HDT);
    const long long one = std::min(wave / blocks, tiles / 2), two = std::min((2 * wave + blocks / 2) / blocks, tiles / 4);
    n_splits = (int)std::max(1LL, std::min((long long)QP_MAX_SPLITS, std::max(one, two)));
  }
  return launch_quant_kernel(kern, dim3(n_splits, p.nkv, n_tiles * p.blocks_per_tile), n_splits, QP_THREADS, qp_smem(HDT, TERMS), 16, p, stream);
}

template <int FMT, typename T, int... I>
static cudaError_t launch_decode_quant_sizes(std::integer_sequence<int, I...>, const QuantDecodeArgs& p, int hd, int n_seqs, int n_splits, int warps,
                                             cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  ((hd == 16 * (I + 1) ? (void)(e = launch_decode_quant_one<FMT, T, I + 1>(p, n_seqs, n_splits, warps, stream)) : (void)0), ...);
  return e;
}

template <int FMT>
static int launch_decode_quant(const QuantDecodeArgs& p, int dtype, int hd, int n_seqs, int n_splits, int warps, cudaStream_t stream) {
  const auto sizes = std::make_integer_sequence<int, 16>{};
  cudaError_t e = dtype == DT_F32 ? launch_decode_quant_sizes<FMT, float>(sizes, p, hd, n_seqs, n_splits, warps, stream)
                                  : launch_decode_quant_sizes<FMT, __nv_bfloat16>(sizes, p, hd, n_seqs, n_splits, warps, stream);
  if (e == cudaSuccess && n_splits > p.cluster) {
    const dim3 grid(n_seqs, p.nh), block((hd / 2 + 31) / 32 * 32);
    const int groups = n_splits / p.cluster;
    e = dtype == DT_F32 ? launch_pdl(2, attn_decode_quant_fold_kernel<float>, grid, block, (size_t)0, stream, (const float*)p.part, (float*)p.out, p.ldo, p.seq_pos, p.nh, hd, groups)
                        : launch_pdl(2, attn_decode_quant_fold_kernel<__nv_bfloat16>, grid, block, (size_t)0, stream, (const float*)p.part, (__nv_bfloat16*)p.out, p.ldo, p.seq_pos,
                                     p.nh, hd, groups);
  }
  if (e != cudaSuccess) {
    set_error("attn_decode_quantized: launch failed: %s", cudaGetErrorString(e));
    return -2;
  }
  return 0;
}

template <int FMT, typename T, int... I>
static cudaError_t launch_prefill_quant_sizes(std::integer_sequence<int, I...>, const QuantPrefillArgs& p, int hd, int n_tiles, int n_splits, cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  ((hd == 16 * (I + 1) ? (void)(e = launch_prefill_quant_one<FMT, T, I + 1>(p, n_tiles, n_splits, stream)) : (void)0), ...);
  return e;
}

template <int FMT>
static int launch_prefill_quant(const QuantPrefillArgs& p, int dtype, int hd, int n_tiles, int n_splits, cudaStream_t stream) {
  const auto sizes = std::make_integer_sequence<int, 16>{};
  const cudaError_t e = dtype == DT_F32 ? launch_prefill_quant_sizes<FMT, float>(sizes, p, hd, n_tiles, n_splits, stream)
                                        : launch_prefill_quant_sizes<FMT, __nv_bfloat16>(sizes, p, hd, n_tiles, n_splits, stream);
  if (e != cudaSuccess) {
    set_error("attn_prefill_quantized: launch failed: %s", cudaGetErrorString(e));
    return -2;
  }
  return 0;
}

}  // namespace edgelm
