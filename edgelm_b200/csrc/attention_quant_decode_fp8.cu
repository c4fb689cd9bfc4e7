// The e4m3 instantiations of the decode attention over the 8-bit cache (attention_quant_decode.cuh).
#include "attention_quant_launch.cuh"

namespace edgelm {
int launch_decode_quant_fp8(const QuantDecodeArgs& p, int dtype, int hd, int n_seqs, int n_splits, int warps, cudaStream_t stream) {
  return launch_decode_quant<QF_FP8>(p, dtype, hd, n_seqs, n_splits, warps, stream);
}
}  // namespace edgelm
