// Decayed linear attention for one new token of each stream:
//   S' = g S + k v^T,   o = scale q S',   g = exp(log_decay[head]).
//
// Bound by reading S and writing S' (float32): 8 bytes per element against 5
// flops.  One block of 256 threads per (stream, head): a thread owns 4
// neighbouring columns (1 where rows are not 16-byte aligned) and every
// 256/lanes-th row, four rows in flight, so that a warp reads whole row runs;
// the partial sums of o meet in shared memory.  The factor g is kept as the
// sum of two float32, so that thousands of steps do not drift by its rounding
// (decay_state.cuh).
#include "decay_attn.h"
#include "decay_state.cuh"
#include "elem.cuh"

namespace tfb {

namespace {
constexpr int kStepThreads = 256;
constexpr int kMaxWidth = 128;

template <int V>
struct Vec;
template <>
struct Vec<4> {
  float x[4];
  __device__ __forceinline__ void load(const float* p) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
  __device__ __forceinline__ void store(float* p) const {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  }
};
template <>
struct Vec<1> {
  float x[1];
  __device__ __forceinline__ void load(const float* p) { x[0] = __ldcs(p); }
  __device__ __forceinline__ void store(float* p) const { __stcs(p, x[0]); }
};
}  // namespace

// lanes: threads of a row, a power of two >= dv / V; rows of threads = 256 / lanes.
template <typename T, int V>
__global__ void __launch_bounds__(kStepThreads) k_decay_step(const __grid_constant__ DecayStepArgs a, int lanes_log) {
  constexpr int U = 4;  // rows in flight
  __shared__ float sq[kMaxWidth], sk[kMaxWidth], red[kStepThreads * V];
  const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int tid = threadIdx.x, lane = tid & ((1 << lanes_log) - 1), row = tid >> lanes_log;
  const int rows = kStepThreads >> lanes_log, col = lane * V;
  const bool mine = col < a.dv;
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[1];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + (h / a.group) * a.ks[1];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + (h / a.group) * a.vs[1];
  const long long at = (long long)h * a.dk * a.dv + col;
  const float* s = a.state + b * a.state_s + at;
  float* n = a.next + b * a.next_s + at;
  Vec<V> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (mine && row + u * rows < a.dk) x[u].load(s + (row + u * rows) * a.dv);
  for (int c = tid; c < a.dk; c += kStepThreads) {
    sq[c] = to_f32(q[c]);
    sk[c] = to_f32(k[c]);
  }
  float vj[V], acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    vj[i] = mine ? to_f32(v[col + i]) : 0.f;
    acc[i] = 0.f;
  }
  const DecayFactor decay(exp((double)a.log_decay[h]), a.log_decay[h]);
  __syncthreads();
  if (mine) {
    for (int c0 = row; c0 < a.dk; c0 += U * rows) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * rows;
        if (c >= a.dk) break;
        const float kc = sk[c], qc = sq[c];
        Vec<V> y;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          y.x[i] = decay.step(x[u].x[i], kc * vj[i]);
          acc[i] = fmaf(qc, y.x[i], acc[i]);
        }
        y.store(n + c * a.dv);
        const int next = c + U * rows;
        if (next < a.dk) x[u].load(s + next * a.dv);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) red[tid * V + i] = acc[i];
  __syncthreads();
  for (int j = tid; j < a.dv; j += kStepThreads) {
    float sum = 0.f;
    for (int r = 0; r < rows; ++r) sum += red[(r << lanes_log) * V + j];
    static_cast<T*>(a.o)[((long long)b * a.heads + h) * a.dv + j] = from_f32<T>(sum * a.scale);
  }
}

template <typename T>
static cudaError_t run_step(const DecayStepArgs& a, cudaStream_t st) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.next);
  const bool wide = (al & 15) == 0 && a.dv % 4 == 0 && a.state_s % 4 == 0 && a.next_s % 4 == 0;
  const int need = wide ? a.dv / 4 : a.dv;
  int lg = 0;
  while ((1 << lg) < need) ++lg;
  const unsigned grid = (unsigned)a.batch * (unsigned)a.heads;
  if (wide)
    k_decay_step<T, 4><<<grid, kStepThreads, 0, st>>>(a, lg);
  else
    k_decay_step<T, 1><<<grid, kStepThreads, 0, st>>>(a, lg);
  return cudaGetLastError();
}

cudaError_t launch_decay_step(ElemType t, const DecayStepArgs& a, cudaStream_t st) {
  switch (t) {
    case kF32: return run_step<float>(a, st);
    case kBF16: return run_step<__nv_bfloat16>(a, st);
    default: return run_step<__half>(a, st);
  }
}

}  // namespace tfb
