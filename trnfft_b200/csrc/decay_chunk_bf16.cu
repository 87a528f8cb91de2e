// Decayed linear attention in chunks, bf16 operands (decay_chunk.cuh).
#include "decay_chunk.cuh"

namespace tfb {
cudaError_t launch_decay_chunks_bf16(const DecayArgs& a, cudaStream_t st) { return chunk::run_all<__nv_bfloat16>(a, st); }
}  // namespace tfb
