// Decayed linear attention for one new token of each stream:
//   S' = g S + k v^T,   o = scale q S',   g = exp(log_decay[head]).
// Bound by reading S and writing S' (float32): 8 bytes per element.
#include "decay_attn.h"
#include "elem.cuh"

namespace tfb {

// One block per (stream, head); thread = column of the state.
template <typename T>
__global__ void __launch_bounds__(128) k_decay_step(const __grid_constant__ DecayStepArgs a) {
  const int h = blockIdx.x, b = blockIdx.y;
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[1];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + (h / a.group) * a.ks[1];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + (h / a.group) * a.vs[1];
  const float* s = a.state + b * a.state_s + (long long)h * a.dk * a.dv;
  float* n = a.next + b * a.next_s + (long long)h * a.dk * a.dv;
  const double gd = exp((double)a.log_decay[h]);
  const float ghi = (float)gd, glo = (float)(gd - (double)ghi);
  for (int j = threadIdx.x; j < a.dv; j += blockDim.x) {
    const float vj = to_f32(v[j]);
    float acc = 0.f;
    for (int c = 0; c < a.dk; ++c) {
      const float x = s[c * a.dv + j];
      const float y = fmaf(x, ghi, fmaf(x, glo, to_f32(k[c]) * vj));
      n[c * a.dv + j] = y;
      acc = fmaf(to_f32(q[c]), y, acc);
    }
    static_cast<T*>(a.o)[((long long)b * a.heads + h) * a.dv + j] = from_f32<T>(acc * a.scale);
  }
}

cudaError_t launch_decay_step(ElemType t, const DecayStepArgs& a, cudaStream_t st) {
  const dim3 grid(a.heads, a.batch);
  switch (t) {
    case kF32: k_decay_step<float><<<grid, 128, 0, st>>>(a); break;
    case kBF16: k_decay_step<__nv_bfloat16><<<grid, 128, 0, st>>>(a); break;
    default: k_decay_step<__half><<<grid, 128, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace tfb
