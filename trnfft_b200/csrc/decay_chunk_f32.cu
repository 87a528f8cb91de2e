// Decayed linear attention in chunks, f32 operands (decay_chunk.cuh).
#include "decay_chunk.cuh"

namespace tfb {
cudaError_t launch_decay_chunks_f32(const DecayArgs& a, cudaStream_t st) { return chunk::run_all<float>(a, st); }
}  // namespace tfb
