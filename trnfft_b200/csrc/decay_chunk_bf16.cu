// Decayed linear attention in chunks, bf16 operands (decay_chunk.cuh).
#include "decay_chunk.cuh"

namespace tfb {
cudaError_t launch_decay_chunks_bf16(const DecayArgs& a, cudaStream_t st) { return chunk::run_all<__nv_bfloat16>(a, st); }
cudaError_t launch_decay_flagged_bf16(const DecayArgs& a, int pass, cudaStream_t st) {
  return chunk::run_chunks<__nv_bfloat16>(a, static_cast<chunk::Pass>(pass), st);
}
}  // namespace tfb
