// Host side of the decode attention over the 8-bit cache: one instantiation a head size, format and type (a source file a format).
#pragma once
#include <utility>

#include "attention_quant_decode.cuh"

namespace edgelm {

template <int FMT, typename T, int HDT>
static cudaError_t launch_decode_quant_one(const QuantDecodeArgs& p, int n_seqs, int n_splits, int warps, cudaStream_t stream) {
  auto kern = attn_decode_quant_kernel<HDT, FMT, T>;
  const int smem = qd_smem(HDT, sizeof(T) == 4 ? 2 : 1, warps);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && n_splits > 8) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  const int chunks = (p.nh / p.nkv + QD_HEADS - 1) / QD_HEADS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n_splits, p.nkv * chunks, n_seqs);
  cfg.blockDim = dim3(warps * 32);
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
  if (pdl_enabled() & 2) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, p);
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
  const cudaError_t e = dtype == DT_F32 ? launch_decode_quant_sizes<FMT, float>(sizes, p, hd, n_seqs, n_splits, warps, stream)
                                        : launch_decode_quant_sizes<FMT, __nv_bfloat16>(sizes, p, hd, n_seqs, n_splits, warps, stream);
  if (e != cudaSuccess) {
    set_error("attn_decode_quantized: launch failed: %s", cudaGetErrorString(e));
    return -2;
  }
  return 0;
}

}  // namespace edgelm
