// The e4m3 instantiations of the prompt attention over the 8-bit cache (attention_quant_prefill.cuh).
#include "attention_quant_launch.cuh"

namespace edgelm {
int launch_prefill_quant_fp8(const QuantPrefillArgs& p, int dtype, int hd, int n_tiles, int n_splits, cudaStream_t stream) {
  return launch_prefill_quant<QF_FP8>(p, dtype, hd, n_tiles, n_splits, stream);
}
}  // namespace edgelm
