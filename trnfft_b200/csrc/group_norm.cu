// Group normalisation with an activation over channels-last features:
//
//   mean, var over the spots and the channels of one group of one sample,
//   h = (x - mean) rstd,  z = h w + b,  y = act(z),   rstd = 1 / sqrt(var + eps)
//
// Backward, with dz = dy act'(z), u = dz w and means over the same values:
//   dx = rstd (u - mean(u) - h mean(u h)),  dw = sum dz h,  db = sum dz
#include "elem.cuh"
#include "group_norm.h"

namespace tfb {

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if (ACT == kActSilu) return z / (1.f + __expf(-z));
  if (ACT == kActGelu) return z * (0.5f + 0.5f * erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (ACT == kActSilu) {
    const float s = 1.f / (1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  if (ACT == kActGelu)
    return 0.5f + 0.5f * erff(z * 0.70710678118654752f) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
  return 1.f;
}

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) s += red[i];
  return s;
}

// One block per (sample, group): mean, then variance, then the values.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_gn_simple(const __grid_constant__ GroupNormArgs a) {
  __shared__ float red[8];
  const long long n = blockIdx.x / a.groups;
  const int g = blockIdx.x % a.groups, w = a.channels / a.groups;
  const long long base = n * a.spots * a.channels + (long long)g * w, count = a.spots * w;
  const T* x = static_cast<const T*>(a.x) + base;
  float s = 0.f;
  for (long long i = threadIdx.x; i < count; i += blockDim.x) s += to_f32(x[i / w * a.channels + i % w]);
  const float mean = block_sum(s, red) / (float)count;
  s = 0.f;
  for (long long i = threadIdx.x; i < count; i += blockDim.x) {
    const float d = to_f32(x[i / w * a.channels + i % w]) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = rsqrtf(block_sum(s, red) / (float)count + a.eps);
  for (long long i = threadIdx.x; i < count; i += blockDim.x) {
    const long long at = i / w * a.channels + i % w;
    const int c = g * w + (int)(i % w);
    const float z = fmaf((to_f32(x[at]) - mean) * rstd, a.weight ? a.weight[c] : 1.f, a.bias ? a.bias[c] : 0.f);
    static_cast<T*>(a.y)[base + at] = from_f32<T>(activate<ACT>(z));
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = rstd;
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_gn_simple_dx(const __grid_constant__ GroupNormArgs a) {
  __shared__ float red[8];
  const long long n = blockIdx.x / a.groups;
  const int g = blockIdx.x % a.groups, w = a.channels / a.groups;
  const long long base = n * a.spots * a.channels + (long long)g * w, count = a.spots * w;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* dy = static_cast<const T*>(a.dy) + base;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
  float su = 0.f, suh = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    if (pass) {
      su = block_sum(su, red) / (float)count;
      suh = block_sum(suh, red) / (float)count;
    }
    for (long long i = threadIdx.x; i < count; i += blockDim.x) {
      const long long at = i / w * a.channels + i % w;
      const int c = g * w + (int)(i % w);
      const float wc = a.weight ? a.weight[c] : 1.f;
      const float h = (to_f32(x[at]) - mean) * rstd;
      const float u = to_f32(dy[at]) * slope<ACT>(fmaf(h, wc, a.bias ? a.bias[c] : 0.f)) * wc;
      if (pass)
        static_cast<T*>(a.y)[base + at] = from_f32<T>(rstd * (u - su - h * suh));
      else {
        su += u;
        suh = fmaf(u, h, suh);
      }
    }
  }
}

// One block per channel.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_gn_simple_dw(const __grid_constant__ GroupNormArgs a) {
  __shared__ float red[8];
  const int c = blockIdx.x, g = c / (a.channels / a.groups);
  const float wc = a.weight ? a.weight[c] : 1.f, bc = a.bias ? a.bias[c] : 0.f;
  float sw = 0.f, sb = 0.f;
  for (long long i = threadIdx.x; i < a.batch * a.spots; i += blockDim.x) {
    const long long n = i / a.spots;
    const float h = (to_f32(static_cast<const T*>(a.x)[i * a.channels + c]) - a.mean[n * a.groups + g]) *
                    a.rstd[n * a.groups + g];
    const float dz = to_f32(static_cast<const T*>(a.dy)[i * a.channels + c]) * slope<ACT>(fmaf(h, wc, bc));
    sb += dz;
    sw = fmaf(dz, h, sw);
  }
  sw = block_sum(sw, red);
  sb = block_sum(sb, red);
  if (threadIdx.x == 0) {
    if (a.dw) a.dw[c] = sw;
    if (a.db) a.db[c] = sb;
  }
}

template <typename T, int ACT>
static cudaError_t run(const GroupNormArgs& a, bool backward, cudaStream_t st) {
  const unsigned blocks = (unsigned)(a.batch * a.groups);
  if (!backward) {
    k_gn_simple<T, ACT><<<blocks, 256, 0, st>>>(a);
  } else {
    if (a.y) k_gn_simple_dx<T, ACT><<<blocks, 256, 0, st>>>(a);
    if (a.dw || a.db) k_gn_simple_dw<T, ACT><<<a.channels, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t run_act(const GroupNormArgs& a, bool backward, cudaStream_t st) {
  switch (a.act) {
    case kActRelu: return run<T, kActRelu>(a, backward, st);
    case kActSilu: return run<T, kActSilu>(a, backward, st);
    case kActGelu: return run<T, kActGelu>(a, backward, st);
    default: return run<T, kActNone>(a, backward, st);
  }
}

static cudaError_t run_type(ElemType t, const GroupNormArgs& a, bool backward, cudaStream_t st) {
  switch (t) {
    case kF32: return run_act<float>(a, backward, st);
    case kBF16: return run_act<__nv_bfloat16>(a, backward, st);
    default: return run_act<__half>(a, backward, st);
  }
}

int64_t group_norm_work_bytes(ElemType, const GroupNormArgs&, bool) { return 0; }

cudaError_t launch_group_norm(ElemType t, const GroupNormArgs& a, cudaStream_t st) { return run_type(t, a, false, st); }
cudaError_t launch_group_norm_backward(ElemType t, const GroupNormArgs& a, cudaStream_t st) {
  return run_type(t, a, true, st);
}

}  // namespace tfb
