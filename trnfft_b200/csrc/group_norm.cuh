// Device code shared by the forward and backward group normalisation kernels.
#pragma once

#include "elem.cuh"
#include "group_norm.h"
#include "tma.cuh"

namespace tfb {
namespace gn {

// float32 results keep the accurate exponential and division; a 16-bit result's own rounding is
// 2^-9 or 2^-12, where the fast ones (a few 2^-22) make no difference.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  return __fdividef(1.f, 1.f + __expf(-fmaxf(z, -80.f)));
}

template <typename T, int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if (ACT == kActSilu) return z * sigmoid<T>(z);
  if (ACT == kActGelu) return z * (0.5f + 0.5f * erff(z * 0.70710678118654752f));
  return z;
}

template <typename T, int ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (ACT == kActSilu) {
    const float s = sigmoid<T>(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == kActGelu) {
    const float p = sizeof(T) == 4 ? expf(-0.5f * z * z) : __expf(-0.5f * z * z);
    return fmaf(0.5f, erff(z * 0.70710678118654752f), 0.5f) + z * p * 0.39894228040143268f;
  }
  return 1.f;
}

// V elements of one access of V * sizeof(T) bytes, as float32.
template <typename T, int V>
struct Pack {
  float x[V];
  __device__ __forceinline__ void load(const T* p) {
    constexpr int B = V * sizeof(T);
    if constexpr (B == 16) {
      const uint4 r = *reinterpret_cast<const uint4*>(p);
      unpack(reinterpret_cast<const T*>(&r));
    } else if constexpr (B == 8) {
      const uint2 r = *reinterpret_cast<const uint2*>(p);
      unpack(reinterpret_cast<const T*>(&r));
    } else if constexpr (B == 4 && V > 1) {
      const uint32_t r = *reinterpret_cast<const uint32_t*>(p);
      unpack(reinterpret_cast<const T*>(&r));
    } else {
      static_assert(V == 1, "access width");
      x[0] = to_f32(p[0]);
    }
  }
  __device__ __forceinline__ void unpack(const T* v) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f32(v[i]);
  }
  __device__ __forceinline__ void store(T* p) const {
    alignas(16) T v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = from_f32<T>(x[i]);
    constexpr int B = V * sizeof(T);
    if constexpr (B == 16)
      __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(v));
    else if constexpr (B == 8)
      __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(v));
    else if constexpr (B == 4 && V > 1)
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(v);
    else
      p[0] = v[0];
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Sum over aligned groups of `lanes` threads (a power of two).
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The parts of one sample meet here: each block adds itself to the sample's
// counter after writing its partial results, and waits until all have.  All
// blocks are resident (cooperative launch), so the wait ends; it is bounded
// all the same, and on giving up records the device status word.
__device__ __forceinline__ void sample_arrive(unsigned* counter) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(counter, 1u);
  }
}
__device__ __forceinline__ void sample_wait(unsigned* counter, unsigned target) {
  if (threadIdx.x == 0) {
    unsigned v = 0;
    int i = 0;
    for (; i < (1 << 24); ++i) {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
      if (v >= target) break;
      __nanosleep(20);
    }
    if (i == (1 << 24)) atomicExch(&g_dev_status, kStatusWaitTimeout);
    __threadfence();
  }
  __syncthreads();
}

// Rows of part k of a sample of `spots` rows cut into `parts`.
__device__ __forceinline__ void part_rows(long long spots, int parts, int k, long long& lo, long long& hi) {
  lo = spots * k / parts;
  hi = spots * (k + 1) / parts;
}

// How many rows of [lo, hi) slot s has: lo + s, lo + s + slots, ...
__device__ __forceinline__ int slot_rows(long long lo, long long hi, int s, int slots) {
  const int n = (int)(hi - lo);
  return n > s ? (n - s + slots - 1) / slots : 0;
}

}  // namespace gn
}  // namespace tfb
