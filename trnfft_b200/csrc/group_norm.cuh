// Device code shared by the forward and backward group normalisation kernels.
#pragma once

#include <type_traits>

#include "elem.cuh"
#include "group_norm.h"
#include "tma.cuh"

namespace tfb {
namespace gn {

// The special function unit's 2^x and 1/x, to about 2^-22, without the handling of denormal numbers
// that would triple their instructions (a result below 2^-126 is 0).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2E = 1.4426950408889634f;

// 1 / (1 + e^-z); e^-z = inf gives 0.
__device__ __forceinline__ float sigmoid(float z) { return rcp_fast(1.f + exp2_fast(-kLog2E * z)); }

// The normal distribution function of z, and e = exp(-z^2 / 2), from one exponential:
// erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + 0.3275911 x), x >= 0, to 1.5e-7
// (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26).  A library erf of twice
// the instructions made the float32 passes bound by instructions instead of memory.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = rcp_fast(fmaf(0.3275911f, x, 1.f));
  e = exp2_fast(x * x * -kLog2E);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float half = 0.5f * (p * t * e);
  return z < 0.f ? half : 1.f - half;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if (ACT == kActSilu) return z * sigmoid(z);
  if (ACT == kActGelu) {
    float e;
    return z * normal_cdf(z, e);
  }
  return z;
}

template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (ACT == kActSilu) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == kActGelu) {
    float e;
    const float p = normal_cdf(z, e);
    return fmaf(z * 0.39894228040143268f, e, p);
  }
  return 1.f;
}

// The bytes of one access, as loaded.
template <int B>
struct Bytes;
template <>
struct Bytes<16> { using type = uint4; };
template <>
struct Bytes<8> { using type = uint2; };
template <>
struct Bytes<4> { using type = uint32_t; };
template <>
struct Bytes<2> { using type = uint16_t; };

// V elements of one access of V * sizeof(T) bytes, as float32.
template <typename T, int V>
struct Pack {
  using Raw = typename Bytes<V * sizeof(T)>::type;
  float x[V];
  static __device__ __forceinline__ Raw raw(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void unpack(Raw r) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value && V % 2 == 0) {
      const uint32_t* v = reinterpret_cast<const uint32_t*>(&r);  // a bfloat16 is the upper half of its float32
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        x[2 * i] = __uint_as_float(v[i] << 16);
        x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      }
    } else {
      const T* v = reinterpret_cast<const T*>(&r);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = to_f32(v[i]);
    }
  }
  __device__ __forceinline__ void load(const T* p) { unpack(raw(p)); }
  __device__ __forceinline__ void store(T* p) const {
    alignas(16) T v[V];
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
      for (int i = 0; i < V; i += 2) from_f32_pair(x[i], x[i + 1], v + i);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = from_f32<T>(x[i]);
    }
    __stcs(reinterpret_cast<Raw*>(p), *reinterpret_cast<const Raw*>(v));
  }
};

// Two sums over aligned groups of `lanes` threads (a power of two).
__device__ __forceinline__ void lanes_sum(float& u, float& v, int lanes) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    if (o < lanes) {
      u += __shfl_xor_sync(~0u, u, o);
      v += __shfl_xor_sync(~0u, v, o);
    }
}

// Blocks of 256 threads an SM holds with a thread's NV accesses and their parameters in registers.
constexpr int small_blocks(int nv) { return nv == 1 ? 4 : (nv == 2 ? 3 : 2); }
constexpr int small_blocks_bwd(int nv) { return nv == 1 ? 3 : (nv == 2 ? 2 : 1); }

// kAny: a thread's elements of a group of w channels, every kNormThreads-th of the rows one after the other.
struct AnyPlace {
  long long row;
  int c, w;
  __device__ __forceinline__ explicit AnyPlace(int width) : row(threadIdx.x / width), c(threadIdx.x % width), w(width) {}
  __device__ __forceinline__ void next() {
    row += kNormThreads / w;
    c += kNormThreads % w;
    if (c >= w) c -= w, ++row;
  }
};

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < kNormThreads / 32; ++i) v += red[i];
  return v;
}

// True in the block that is the last of its sample's `parts` to come here; it sees what all of
// them wrote before.
__device__ __forceinline__ bool last_of_sample(unsigned* counter, int parts) {
  __shared__ unsigned before;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    before = atomicAdd(counter, 1u);
    __threadfence();
  }
  __syncthreads();
  return before == parts - 1;
}

constexpr int kMostShared = 220 * 1024;  // more than any launch here asks for
template <auto K>
cudaError_t allow_smem(int bytes) {
  return bytes <= 48 * 1024 ? cudaSuccess : allow_shared<K>(kMostShared);
}

// c / w for 0 <= c < 2^20, w >= 1, where inv = 1.f / w: (c + 1/2) / w is at least 1 / (2 w) from a whole
// number, c + 1/2 is exact, and inv and the product are off by 2^-24 of themselves each: by less than
// c / w * 2^-22 < 1 / (2 w) together.  (kSplit has at most 25600 channels: their sets fill kMaxSplitSmem.)
__device__ __forceinline__ int quotient(int c, float inv) { return (int)(((float)c + 0.5f) * inv); }

// A block's rows of a sample, part k, and a thread's place among them: its column of a tile of
// channels, and the rows slot, slot + slots, ... of which there are `mine`.
struct SplitPlace {
  int rows, slot, col, mine;
  long long step;   // elements between two rows of a slot
  long long first;  // element of a thread's first row, channel 0, in sample 0
  __device__ __forceinline__ SplitPlace(const GroupNormArgs& a, const GroupNormPlan& p, int k) {
    rows = k == p.parts - 1 ? (int)(a.spots - (long long)k * p.part_rows) : p.part_rows;
    slot = threadIdx.x / p.cols;
    col = threadIdx.x % p.cols;
    mine = slot < p.slots && rows > slot ? (rows - slot + p.slots - 1) / p.slots : 0;
    step = (long long)p.slots * a.channels;
    first = ((long long)k * p.part_rows + slot) * a.channels;
  }
};

// A thread's V channels of one tile: the first, and their parameters.  With one tile (up to 1024
// channels) they are read once for all samples.
template <int V>
struct SplitColumn {
  int c;
  float inv_w;
  float wt[V], bs[V];
  bool live;
  __device__ __forceinline__ int group(int v) const { return quotient(c + v, inv_w); }
  __device__ __forceinline__ void set(const GroupNormArgs& a, const GroupNormPlan& p, const SplitPlace& at, int tile) {
    c = (tile * p.cols + at.col) * V;
    live = at.slot < p.slots && c < a.channels;
    if (!live) return;
    inv_w = 1.f / (float)(a.channels / a.groups);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      wt[v] = a.weight ? a.weight[c + v] : 1.f;
      bs[v] = a.bias ? a.bias[c + v] : 0.f;
    }
  }
};

// A block's rows of N tensors (contiguous in memory), streamed through kStages buffers in shared memory
// by bulk copies that one thread issues ahead: bytes on their way take no registers, and the first
// kStages buffers are asked for at once.
template <int N>
struct RowStream {
  static constexpr int kBuffer = kStreamBytes / kStages / N;
  unsigned char* buffers;
  uint64_t* full;
  const char* from[N];
  long long row_bytes;
  int rows, per, count;  // rows in all, of a buffer; buffers
  int gave_up = -1;      // the buffer at which this thread's wait ran out
  __device__ __forceinline__ void issue(int i) {
    const int first = i * per;
    const uint32_t bytes = (uint32_t)(min(per, rows - first) * row_bytes);
    uint64_t* bar = full + i % kStages;
    mbar_arrive_expect_tx(bar, N * bytes);
#pragma unroll
    for (int j = 0; j < N; ++j) bulk_g2s(buffers + (i % kStages * N + j) * kBuffer, from[j] + first * row_bytes, bytes, bar);
  }
  __device__ __forceinline__ RowStream(unsigned char* smem, const GroupNormPlan& p, int row_count, long long bytes_per_row,
                                       const void* const (&src)[N])
      : buffers(smem), full(reinterpret_cast<uint64_t*>(smem + kStreamBytes)), row_bytes(bytes_per_row), rows(row_count),
        per(p.stage_rows) {
#pragma unroll
    for (int j = 0; j < N; ++j) from[j] = static_cast<const char*>(src[j]);
    count = (rows + per - 1) / per;
    if (threadIdx.x == 0) {
      for (int i = 0; i < kStages; ++i) mbar_init(full + i, 1);
      mbar_init_fence();
      for (int i = 0; i < min(kStages, count); ++i) issue(i);
    }
    __syncthreads();
  }
  // Waits for buffer i.  A thread whose wait gives up goes on with whatever the buffer holds, through the
  // same barriers as the others, and waits no more; finish() says so in the status word.
  __device__ __forceinline__ void wait(int i) {
    if (gave_up < 0 && !mbar_wait_bounded(full + i % kStages, i / kStages & 1)) gave_up = i;
  }
  __device__ __forceinline__ const unsigned char* buffer(int i, int tensor) const {
    return buffers + (i % kStages * N + tensor) * kBuffer;
  }
  __device__ __forceinline__ int rows_of(int i) const { return min(per, rows - i * per); }
  // All have read buffer i: it may be filled again.
  __device__ __forceinline__ void release(int i) {
    __syncthreads();
    if (threadIdx.x == 0 && gave_up < 0 && i + kStages < count) issue(i + kStages);
  }
  // After the last buffer: nothing is on its way to shared memory when the block ends.
  __device__ __forceinline__ void finish() {
    if (gave_up < 0) return;
    atomicExch(&g_dev_status, kStatusWaitTimeout);
    if (threadIdx.x == 0)
      for (int i = gave_up; i < min(gave_up + kStages, count); ++i) (void)mbar_wait_bounded(full + i % kStages, i / kStages & 1);
  }
};

// A block's samples blockIdx.x, blockIdx.x + gridDim.x, ... of N tensors, streamed whole through
// p.sample_buffers buffers.
template <int N>
struct SampleStream {
  unsigned char* buffers;
  uint64_t* full;
  const char* from[N];
  long long bytes;  // of a sample of one tensor
  int count, ring;
  int gave_up = -1;
  __device__ __forceinline__ void issue(int i) {
    uint64_t* bar = full + i % ring;
    mbar_arrive_expect_tx(bar, (uint32_t)(N * bytes));
#pragma unroll
    for (int j = 0; j < N; ++j)
      bulk_g2s(buffers + (i % ring * N + j) * bytes, from[j] + (blockIdx.x + (long long)i * gridDim.x) * bytes,
               (uint32_t)bytes, bar);
  }
  __device__ __forceinline__ SampleStream(unsigned char* smem, const GroupNormPlan& p, long long samples,
                                          long long sample_bytes, const void* const (&src)[N])
      : buffers(smem), full(reinterpret_cast<uint64_t*>(smem + p.sample_buffers * N * sample_bytes)), bytes(sample_bytes),
        ring(p.sample_buffers) {
#pragma unroll
    for (int j = 0; j < N; ++j) from[j] = static_cast<const char*>(src[j]);
    count = (int)((samples - blockIdx.x + gridDim.x - 1) / gridDim.x);
    if (threadIdx.x == 0) {
      for (int i = 0; i < ring; ++i) mbar_init(full + i, 1);
      mbar_init_fence();
      for (int i = 0; i < min(ring, count); ++i) issue(i);
    }
    __syncthreads();
  }
  __device__ __forceinline__ void wait(int i) {  // this, release() and finish() as above
    if (gave_up < 0 && !mbar_wait_bounded(full + i % ring, i / ring & 1)) gave_up = i;
  }
  __device__ __forceinline__ const unsigned char* buffer(int i, int tensor) const {
    return buffers + (i % ring * N + tensor) * bytes;
  }
  __device__ __forceinline__ void release(int i) {
    __syncthreads();
    if (threadIdx.x == 0 && gave_up < 0 && i + ring < count) issue(i + ring);
  }
  __device__ __forceinline__ void finish() {
    if (gave_up < 0) return;
    atomicExch(&g_dev_status, kStatusWaitTimeout);
    if (threadIdx.x == 0)
      for (int i = gave_up; i < min(gave_up + ring, count); ++i) (void)mbar_wait_bounded(full + i % ring, i / ring & 1);
  }
};
constexpr int kMaxSampleBuffers = 8;

}  // namespace gn
}  // namespace tfb
