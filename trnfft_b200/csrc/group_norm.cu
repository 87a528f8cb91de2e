// Group normalisation with an activation over channels-last features:
//
//   mean, var over the spots and the channels of one group of one sample,
//   h = (x - mean) rstd,  z = h w + b,  y = act(z),   rstd = 1 / sqrt(var + eps)
//
// Bound by HBM: x read once, y written once.  Two forms reach that.
//   kSmall  a group of one sample has few values (a frame's features, the
//           heads of an attention's output): a few threads keep them in
//           registers between the statistics and the result.
//   kSplit  `parts` blocks share a sample, each a run of whole rows (any
//           number of channels, any grouping, contiguous in memory).  A
//           block takes the statistics of its run, hands them to the others
//           through global memory, takes those of its next sample's run
//           while they arrive, and comes back for the first: its second
//           read of x hits L2, because the parts are chosen so that the
//           samples in flight fit there.
// The variance is never a difference of large sums: a thread takes the mean
// and the squared distances of 4 rows at a time and joins such sets by
//   M2 = M2a + M2b + (mean_b - mean_a)^2 na nb / (na + nb).
#include "group_norm.cuh"

#include <algorithm>

namespace tfb {
namespace gn {

// ---------------------------------------------------------------- kSmall
// `lanes` threads per (sample, group), NV accesses of V elements each.  The
// element with index i of a group is channel i % w of spot i / w; accesses of
// V > 1 elements are used for one spot only.  A thread's groups are a
// multiple of `groups` apart, so its channels and their parameters stay.
template <typename T, int V, int NV, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_small(const __grid_constant__ GroupNormArgs a, int lanes) {
  const int w = a.channels / a.groups, count = (int)a.spots * w;
  const int per = kNormThreads / lanes, lane = threadIdx.x & (lanes - 1);
  const long long slots = (long long)gridDim.x * per / a.groups * a.groups;
  const long long first = (long long)blockIdx.x * per + threadIdx.x / lanes, total = a.batch * a.groups;
  const int g = (int)(first % a.groups);
  int off[NV];
  float wt[NV][V], bs[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = (lane + j * lanes) * V;
    off[j] = i < count ? (V > 1 ? i : i / w * a.channels + i % w) : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = g * w + (V > 1 ? i + v : i % w);
      wt[j][v] = a.weight && i < count ? a.weight[c] : 1.f;
      bs[j][v] = a.bias && i < count ? a.bias[c] : 0.f;
    }
  }
  const float inv = 1.f / (float)count;
  // every thread of a warp takes the same number of turns: the shuffles need them all
  const long long turns = (total + slots - 1) / slots;
  for (long long k = 0; k < turns; ++k) {
    const long long id = first + k * slots;
    const bool live = first < slots && id < total;
    const long long base = live ? id / a.groups * a.spots * a.channels + (long long)g * w : 0;
    const T* x = static_cast<const T*>(a.x) + base;
    Pack<T, V> p[NV];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (live && off[j] >= 0) {
        p[j].load(x + off[j]);
#pragma unroll
        for (int v = 0; v < V; ++v) s += p[j].x[v];
      }
    }
    const float mean = lanes_sum(s, lanes) * inv;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (live && off[j] >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          p[j].x[v] -= mean;
          s = fmaf(p[j].x[v], p[j].x[v], s);
        }
      }
    const float rstd = __frsqrt_rn(lanes_sum(s, lanes) * inv + a.eps);
    if (live) {
      T* y = static_cast<T*>(a.y) + base;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (off[j] >= 0) {
#pragma unroll
          for (int v = 0; v < V; ++v) p[j].x[v] = activate<T, ACT>(fmaf(p[j].x[v] * rstd, wt[j][v], bs[j][v]));
          p[j].store(y + off[j]);
        }
      if (lane == 0 && a.mean) {
        a.mean[id] = mean;
        a.rstd[id] = rstd;
      }
    }
  }
}

// ---------------------------------------------------------------- kSplit

// Shared memory: per-slot sets (mean, M2) of a tile of channels, then the
// channels' of the block's rows, then the groups' results.
struct SplitSmem {
  float2* red;    // slots * cols * V
  float2* chan;   // channels
  float2* group;  // groups: (mean, rstd)
};

template <typename T, int V>
__device__ __forceinline__ void split_stats(const GroupNormArgs& a, const GroupNormPlan& p, const SplitSmem& sm,
                                            long long n, int k, float2* part) {
  constexpr int U = 4;
  const int slot = threadIdx.x / p.cols, col = threadIdx.x % p.cols;
  long long lo, hi;
  part_rows(a.spots, p.parts, k, lo, hi);
  const T* x = static_cast<const T*>(a.x) + n * a.spots * a.channels;
  const int w = a.channels / a.groups;
  for (int tile = 0; tile < p.tiles; ++tile) {
    const int c = (tile * p.cols + col) * V;
    float mean[V], m2[V];
    float cnt = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.f;
    if (slot < p.slots && c < a.channels) {
      const T* q = x + (lo + slot) * a.channels + c;
      const long long step = (long long)p.slots * a.channels;
      for (int left = slot_rows(lo, hi, slot, p.slots); left > 0; left -= U, q += U * step) {
        Pack<T, V> b[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < left) b[u].load(q + u * step);
        const float nb = (float)min(left, U), inv = 1.f / nb, all = cnt + nb, share = nb / all, cross = cnt * share;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float s = 0.f;
#pragma unroll
          for (int u = 0; u < U; ++u) s += u < left ? b[u].x[v] : 0.f;
          const float mb = s * inv;
          float d2 = 0.f;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const float d = u < left ? b[u].x[v] - mb : 0.f;
            d2 = fmaf(d, d, d2);
          }
          const float d = mb - mean[v];
          m2[v] += fmaf(d * d, cross, d2);
          mean[v] = fmaf(d, share, mean[v]);
        }
        cnt = all;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) sm.red[(slot * p.cols + col) * V + v] = make_float2(mean[v], m2[v]);
    }
    __syncthreads();
    // join the slots: slot s has the rows lo + s, lo + s + slots, ...
    const int width = p.cols * V;
    for (int i = threadIdx.x; i < width && tile * width + i < a.channels; i += blockDim.x) {
      float na = 0.f, m = 0.f, q = 0.f;
      for (int s = 0; s < p.slots && lo + s < hi; ++s) {
        const float nb = (float)slot_rows(lo, hi, s, p.slots), all = na + nb;
        const float2 b = sm.red[s * width + i];
        const float d = b.x - m;
        q += fmaf(d * d, na * nb / all, b.y);
        m = fmaf(d, nb / all, m);
        na = all;
      }
      sm.chan[tile * width + i] = make_float2(m, q);
    }
    __syncthreads();
  }
  // a group's channels have the same number of rows
  const float rows = (float)(hi - lo);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  for (int g = warp; g < a.groups; g += warps) {
    float s = 0.f;
    for (int c = lane; c < w; c += 32) s += sm.chan[g * w + c].x;
    const float m = warp_sum(s) / (float)w;
    s = 0.f;
    for (int c = lane; c < w; c += 32) {
      const float2 b = sm.chan[g * w + c];
      const float d = b.x - m;
      s += fmaf(d * d, rows, b.y);
    }
    s = warp_sum(s);
    if (lane == 0) {
      if (p.parts > 1)
        part[((long long)n * p.parts + k) * a.groups + g] = make_float2(m, s);
      else
        sm.group[g] = make_float2(m, s);
    }
  }
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void split_apply(const GroupNormArgs& a, const GroupNormPlan& p, const SplitSmem& sm,
                                            long long n, int k, const float2* part) {
  constexpr int U = 4;
  const int w = a.channels / a.groups;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const float total = (float)(a.spots * w);
  __syncthreads();
  for (int g = warp; g < a.groups; g += warps) {
    float m, q;
    if (p.parts > 1) {
      const float2* at = part + (long long)n * p.parts * a.groups + g;
      float s = 0.f;
      for (int i = lane; i < p.parts; i += 32) {
        long long lo, hi;
        part_rows(a.spots, p.parts, i, lo, hi);
        s = fmaf(__ldcg(at + (long long)i * a.groups).x, (float)((hi - lo) * w) / total, s);
      }
      m = warp_sum(s);
      s = 0.f;
      for (int i = lane; i < p.parts; i += 32) {
        long long lo, hi;
        part_rows(a.spots, p.parts, i, lo, hi);
        const float2 b = __ldcg(at + (long long)i * a.groups);
        const float d = b.x - m;
        s += fmaf(d * d, (float)((hi - lo) * w), b.y);
      }
      q = warp_sum(s);
    } else {
      m = sm.group[g].x;
      q = sm.group[g].y;
    }
    const float rstd = __frsqrt_rn(q / total + a.eps);
    __syncwarp();
    if (lane == 0) {
      sm.group[g] = make_float2(m, rstd);
      if (k == 0 && a.mean) {
        a.mean[n * a.groups + g] = m;
        a.rstd[n * a.groups + g] = rstd;
      }
    }
  }
  __syncthreads();
  const int slot = threadIdx.x / p.cols, col = threadIdx.x % p.cols;
  long long lo, hi;
  part_rows(a.spots, p.parts, k, lo, hi);
  const T* x = static_cast<const T*>(a.x) + n * a.spots * a.channels;
  T* y = static_cast<T*>(a.y) + n * a.spots * a.channels;
  for (int tile = 0; tile < p.tiles; ++tile) {
    const int c = (tile * p.cols + col) * V;
    if (slot >= p.slots || c >= a.channels) continue;
    float mean[V], gain[V], bias[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 s = sm.group[(c + v) / w];
      mean[v] = s.x;
      gain[v] = s.y * (a.weight ? a.weight[c + v] : 1.f);
      bias[v] = a.bias ? a.bias[c + v] : 0.f;
    }
    const long long step = (long long)p.slots * a.channels, at = (lo + slot) * a.channels + c;
    const T* from = x + at;
    T* to = y + at;
    for (int left = slot_rows(lo, hi, slot, p.slots); left > 0; left -= U, from += U * step, to += U * step) {
      Pack<T, V> q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) q[u].load(from + u * step);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) {
#pragma unroll
          for (int v = 0; v < V; ++v) q[u].x[v] = activate<T, ACT>(fmaf(q[u].x[v] - mean[v], gain[v], bias[v]));
          q[u].store(to + u * step);
        }
    }
  }
  __syncthreads();
}

// parts == 1: block = sample.  parts > 1: the grid is a multiple of `parts`
// and resident; block b takes part b % parts of the samples b / parts,
// b / parts + grid / parts, ...
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, kSplitThreadsPerSm / kNormThreads) k_gn_split(const __grid_constant__ GroupNormArgs a,
                                                  const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(16) float2 smem[];
  SplitSmem sm;
  sm.red = smem;
  sm.chan = sm.red + p.slots * p.cols * V;
  sm.group = sm.chan + a.channels;
  if (p.parts == 1) {
    for (long long n = blockIdx.x; n < a.batch; n += gridDim.x) {
      split_stats<T, V>(a, p, sm, n, 0, nullptr);
      split_apply<T, V, ACT>(a, p, sm, n, 0, nullptr);
    }
    return;
  }
  float2* part = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.off_stats);
  unsigned* sync = reinterpret_cast<unsigned*>(static_cast<char*>(a.work) + p.off_sync);
  const int k = blockIdx.x % p.parts, step = gridDim.x / p.parts;
  long long n = blockIdx.x / p.parts;
  if (n >= a.batch) return;
  split_stats<T, V>(a, p, sm, n, k, part);
  sample_arrive(sync + n);
  for (; n < a.batch; n += step) {
    const long long next = n + step;
    if (next < a.batch) {
      split_stats<T, V>(a, p, sm, next, k, part);
      sample_arrive(sync + next);
    }
    sample_wait(sync + n, (unsigned)p.parts);
    split_apply<T, V, ACT>(a, p, sm, n, k, part);
  }
}

// ---------------------------------------------------------------- kAny
// More channels than the other forms' shared memory holds: three passes over
// a group by one block.
template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_any(const __grid_constant__ GroupNormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const int w = a.channels / a.groups;
  const float inv = 1.f / (float)(a.spots * w);
  for (long long id = blockIdx.x; id < a.batch * a.groups; id += gridDim.x) {
    const int g = (int)(id % a.groups);
    const long long base = id / a.groups * a.spots * a.channels + (long long)g * w;
    float stat[2] = {0.f, 0.f};
    for (int pass = 0; pass < 3; ++pass) {
      float s = 0.f;
      for (long long r = 0; r < a.spots; ++r)
        for (int c = threadIdx.x; c < w; c += kNormThreads) {
          const long long at = base + r * a.channels + c;
          const float x = to_f32(static_cast<const T*>(a.x)[at]), d = x - stat[0];
          if (pass == 0) s += x;
          if (pass == 1) s = fmaf(d, d, s);
          if (pass == 2) {
            const float z = fmaf(d * stat[1], a.weight ? a.weight[g * w + c] : 1.f, a.bias ? a.bias[g * w + c] : 0.f);
            static_cast<T*>(a.y)[at] = from_f32<T>(activate<T, ACT>(z));
          }
        }
      if (pass == 2) break;
      s = warp_sum(s);
      __syncthreads();
      if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
      __syncthreads();
      s = 0.f;
      for (int i = 0; i < kNormThreads / 32; ++i) s += red[i];
      stat[pass] = pass == 0 ? s * inv : __frsqrt_rn(s * inv + a.eps);
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[id] = stat[0];
      a.rstd[id] = stat[1];
    }
  }
}

template <typename T, int V, int ACT>
static cudaError_t run_small(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  switch (p.nv) {
    case 1: k_gn_small<T, V, 1, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes); break;
    case 2: k_gn_small<T, V, 2, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes); break;
    case 4: k_gn_small<T, V, 4, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes); break;
    default:
      if constexpr (V == 1) k_gn_small<T, 1, 8, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes);
  }
  return cudaGetLastError();
}

template <typename T, int V, int ACT>
static cudaError_t run_split(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (p.smem > 48 * 1024)
    e = cudaFuncSetAttribute(k_gn_split<T, V, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem);
  if (e != cudaSuccess) return e;
  if (p.parts == 1) {
    k_gn_split<T, V, ACT><<<p.grid, p.threads, p.smem, st>>>(a, p);
    return cudaGetLastError();
  }
  e = cudaMemsetAsync(static_cast<char*>(a.work) + p.off_sync, 0, sizeof(unsigned) * a.batch, st);
  if (e != cudaSuccess) return e;
  GroupNormArgs a2 = a;
  GroupNormPlan p2 = p;
  void* args[] = {&a2, &p2};
  return cudaLaunchCooperativeKernel(k_gn_split<T, V, ACT>, dim3(p.grid), dim3(p.threads), args, (size_t)p.smem, st);
}

template <typename T, int ACT>
static cudaError_t run(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  if (p.kind == GroupNormPlan::kAny) {
    k_gn_any<T, ACT><<<p.grid, kNormThreads, 0, st>>>(a);
    return cudaGetLastError();
  }
  if (p.kind == GroupNormPlan::kSmall)
    return p.vec == W ? run_small<T, W, ACT>(a, p, st) : run_small<T, 1, ACT>(a, p, st);
  if (p.vec == 4) return run_split<T, 4, ACT>(a, p, st);
  if constexpr (sizeof(T) == 2)
    if (p.vec == 2) return run_split<T, 2, ACT>(a, p, st);
  return run_split<T, 1, ACT>(a, p, st);
}

template <typename T>
static cudaError_t run_act(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  switch (a.act) {
    case kActRelu: return run<T, kActRelu>(a, p, st);
    case kActSilu: return run<T, kActSilu>(a, p, st);
    case kActGelu: return run<T, kActGelu>(a, p, st);
    default: return run<T, kActNone>(a, p, st);
  }
}

}  // namespace gn

GroupNormPlan plan_group_norm(ElemType t, const GroupNormArgs& a, bool backward, int align) {
  GroupNormPlan p = {};
  const int size = t == kF32 ? 4 : 2, wide = 16 / size, w = a.channels / a.groups;
  const long long count = a.spots * w, total = a.batch * a.groups;
  const bool vec_row = a.channels % wide == 0 && align % 16 == 0;
  // A group's values in the registers of at most 32 threads: up to 4 wide accesses each for one
  // spot, else up to 8 single elements.
  const bool small_wide = a.spots == 1 && w % wide == 0 && vec_row && w / wide <= 128;
  if (small_wide || (count <= 256 && a.groups <= 4096)) {
    p.kind = GroupNormPlan::kSmall;
    p.vec = small_wide ? wide : 1;
    const int need = (int)((count + p.vec - 1) / p.vec);
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes < need) p.lanes *= 2;
    p.nv = 1;
    while (p.nv * p.lanes < need) p.nv *= 2;
    const int per = kNormThreads / p.lanes;
    const long long blocks = (total + per - 1) / per;
    const long long least = (a.groups + per - 1) / per;  // a thread group for each group of channels
    const long long most = std::max<long long>(least, (long long)kSms * (backward ? 4 : 8));
    p.grid = (int)std::max(least, std::min(blocks, most));
    if (backward) {
      const long long slots = (long long)p.grid * per / a.groups * a.groups;
      p.channel_rows = std::min(slots, total) / a.groups * a.spots;
      p.bytes = p.channel_rows * a.channels * 8;
    }
    return p;
  }
  if (a.channels > kMaxSplitChannels) {
    p.kind = GroupNormPlan::kAny;
    p.vec = 1;
    p.grid = (int)std::min<long long>(total, 16LL * kSms);
    return p;
  }
  p.kind = GroupNormPlan::kSplit;
  // 4 elements per access: with 8 of a 16-bit type the channels' parameters would not fit the registers
  p.vec = a.channels % 4 == 0 && align % (4 * size) == 0 ? 4 : (size == 2 && a.channels % 2 == 0 && align % 4 == 0 ? 2 : 1);
  const int columns = (a.channels + p.vec - 1) / p.vec;
  p.cols = std::min(columns, kNormThreads);
  p.tiles = (columns + p.cols - 1) / p.cols;
  p.slots = (int)std::min<long long>(kNormThreads / p.cols, a.spots);
  p.threads = std::max(64, (p.slots * p.cols + 31) / 32 * 32);
  p.smem = (int)sizeof(float2) * (p.slots * p.cols * p.vec + (backward ? 2 : 1) * a.channels + a.groups);
  // resident blocks per SM: the launch bounds leave registers for 768 threads
  const int resident = std::max(1, std::min(kSplitThreadsPerSm / p.threads, 200 * 1024 / (p.smem + 1024)));
  const long long most = (long long)kSms * resident;
  const long long bytes = a.spots * a.channels * size * (backward ? 2 : 1);
  // The samples in flight (two per `parts` blocks: one that is read, one that is written) stay
  // within 48 MB of L2; with few samples their blocks fill the GPU, each with 16 KB at least.
  long long parts = (most * bytes * 2 + (48LL << 20) - 1) / (48LL << 20);
  parts = std::max(parts, (most + a.batch - 1) / a.batch);
  parts = std::min({parts, most, bytes / (16 << 10), (long long)a.spots});
  p.parts = bytes <= (48 << 10) ? 1 : (int)std::max<long long>(1, parts);
  p.grid = (int)(p.parts == 1 ? std::min(a.batch, most) : std::min(a.batch, most / p.parts) * p.parts);
  p.off_channels = ((p.parts > 1 ? a.batch * p.parts * a.groups * 8 : 0) + 15) & ~15LL;
  p.channel_rows = backward ? p.grid : 0;
  p.off_sync = p.off_channels + ((p.channel_rows * a.channels * 8 + 15) & ~15LL);
  p.bytes = p.off_sync + (p.parts > 1 ? a.batch * 4 : 0);
  return p;
}

int group_norm_align(const GroupNormArgs& a) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.dy);
  return al % 16 == 0 ? 16 : (al % 8 == 0 ? 8 : (al % 4 == 0 ? 4 : 2));
}

int64_t group_norm_work_bytes(ElemType t, const GroupNormArgs& a, bool backward) {
  int64_t most = 0;  // whatever the alignment
  for (int align : {16, 8, 4, 2}) most = std::max<int64_t>(most, plan_group_norm(t, a, backward, align).bytes);
  return most;
}

cudaError_t launch_group_norm(ElemType t, const GroupNormArgs& a, cudaStream_t st) {
  const GroupNormPlan p = plan_group_norm(t, a, false, group_norm_align(a));
  switch (t) {
    case kF32: return gn::run_act<float>(a, p, st);
    case kBF16: return gn::run_act<__nv_bfloat16>(a, p, st);
    default: return gn::run_act<__half>(a, p, st);
  }
}

}  // namespace tfb
