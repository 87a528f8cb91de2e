// Decayed linear attention in chunks, f16 operands (decay_chunk.cuh).
#include "decay_chunk.cuh"

namespace tfb {
cudaError_t launch_decay_chunks_f16(const DecayArgs& a, cudaStream_t st) { return chunk::run_all<__half>(a, st); }
}  // namespace tfb
