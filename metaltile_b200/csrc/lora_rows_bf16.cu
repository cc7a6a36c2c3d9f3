// The warp-level tensor-core kernels of low-rank adapters, bf16 (a file a type: they are many forms)
#include "lora_rows.cuh"

namespace mtc {
template cudaError_t launch_lora_mma<MTC_BF16>(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none);
}  // namespace mtc
