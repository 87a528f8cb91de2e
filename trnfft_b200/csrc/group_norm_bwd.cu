// Gradients of the group normalisation with an activation (group_norm.cu).
// With h and z as there, dz = dy act'(z), u = dz w and means over a group:
//   dx = rstd (u - mean(u) - h mean(u h)),  dw = sum dz h,  db = sum dz
//
// Bound by HBM: x and dy read once, dx written once.  The same two forms as
// the forward pass.  Per sample the channels' sums of dz and dz h give the
// group means as well (sum over its channels, times w), so one pass over x
// and dy serves dx, dw and db.  Blocks add up the sums of all their samples
// and leave one row each, which a last small kernel adds in a fixed order:
// no atomics, the same result every time.
#include "group_norm.cuh"

namespace tfb {
namespace gn {

template <typename T, int V, int NV, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_small_bwd(const __grid_constant__ GroupNormArgs a, int lanes) {
  const int w = a.channels / a.groups, count = (int)a.spots * w;
  const int per = kNormThreads / lanes, lane = threadIdx.x & (lanes - 1);
  const long long slots = (long long)gridDim.x * per / a.groups * a.groups;
  const long long first = (long long)blockIdx.x * per + threadIdx.x / lanes, total = a.batch * a.groups;
  const int g = (int)(first % a.groups);
  int off[NV];
  float wt[NV][V], bs[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = (lane + j * lanes) * V;
    off[j] = i < count ? (V > 1 ? i : i / w * a.channels + i % w) : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = g * w + (V > 1 ? i + v : i % w);
      wt[j][v] = a.weight && i < count ? a.weight[c] : 1.f;
      bs[j][v] = a.bias && i < count ? a.bias[c] : 0.f;
      dw[j][v] = db[j][v] = 0.f;
    }
  }
  const float inv = 1.f / (float)count;
  const long long turns = (total + slots - 1) / slots;
  for (long long k = 0; k < turns; ++k) {
    const long long id = first + k * slots;
    const bool live = first < slots && id < total;
    const long long base = live ? id / a.groups * a.spots * a.channels + (long long)g * w : 0;
    const T* x = static_cast<const T*>(a.x) + base;
    const T* dy = static_cast<const T*>(a.dy) + base;
    Pack<T, V> h[NV], u[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (live && off[j] >= 0) {
        h[j].load(x + off[j]);
        u[j].load(dy + off[j]);
      }
    const float mean = live ? a.mean[id] : 0.f, rstd = live ? a.rstd[id] : 0.f;
    float su = 0.f, suh = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (live && off[j] >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float hv = (h[j].x[v] - mean) * rstd;
          const float dz = u[j].x[v] * slope<T, ACT>(fmaf(hv, wt[j][v], bs[j][v]));
          db[j][v] += dz;
          dw[j][v] = fmaf(dz, hv, dw[j][v]);
          h[j].x[v] = hv;
          u[j].x[v] = dz * wt[j][v];
          su += u[j].x[v];
          suh = fmaf(u[j].x[v], hv, suh);
        }
      }
    if (!a.y) continue;
    su = lanes_sum(su, lanes) * inv;
    suh = lanes_sum(suh, lanes) * inv;
    if (live) {
      T* dx = static_cast<T*>(a.y) + base;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (off[j] >= 0) {
#pragma unroll
          for (int v = 0; v < V; ++v) u[j].x[v] = rstd * (u[j].x[v] - su - h[j].x[v] * suh);
          u[j].store(dx + off[j]);
        }
    }
  }
  if ((a.dw || a.db) && first < slots && first < total) {
    float2* out = static_cast<float2*>(a.work) + first / a.groups * a.spots * a.channels + g * w;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (off[j] >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) out[off[j] + v] = make_float2(dw[j][v], db[j][v]);
      }
  }
}

struct SplitBwdSmem {
  float2* red;    // slots * cols * V: sums of (dz h, dz) of a slot
  float2* chan;   // channels: of the block's rows of one sample
  float2* acc;    // channels: of all its samples
  float2* group;  // groups: (mean of u, mean of u h)
};

template <typename T, int V, int ACT>
__device__ __forceinline__ void split_sums(const GroupNormArgs& a, const GroupNormPlan& p, const SplitBwdSmem& sm,
                                           long long n, int k, float2* part) {
  constexpr int U = 2;
  const int slot = threadIdx.x / p.cols, col = threadIdx.x % p.cols;
  long long lo, hi;
  part_rows(a.spots, p.parts, k, lo, hi);
  const T* x = static_cast<const T*>(a.x) + n * a.spots * a.channels;
  const T* dy = static_cast<const T*>(a.dy) + n * a.spots * a.channels;
  const int w = a.channels / a.groups;
  for (int tile = 0; tile < p.tiles; ++tile) {
    const int c = (tile * p.cols + col) * V;
    if (slot < p.slots && c < a.channels) {
      float mean[V], rstd[V], wt[V], bs[V], sw[V], sb[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const long long at = n * a.groups + (c + v) / w;
        mean[v] = a.mean[at];
        rstd[v] = a.rstd[at];
        wt[v] = a.weight ? a.weight[c + v] : 1.f;
        bs[v] = a.bias ? a.bias[c + v] : 0.f;
        sw[v] = sb[v] = 0.f;
      }
      const long long step = (long long)p.slots * a.channels, at = (lo + slot) * a.channels + c;
      const T *px = x + at, *pd = dy + at;
      for (int left = slot_rows(lo, hi, slot, p.slots); left > 0; left -= U, px += U * step, pd += U * step) {
        Pack<T, V> q[U], d[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (i < left) {
            q[i].load(px + i * step);
            d[i].load(pd + i * step);
          }
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (i < left) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const float h = (q[i].x[v] - mean[v]) * rstd[v];
              const float dz = d[i].x[v] * slope<T, ACT>(fmaf(h, wt[v], bs[v]));
              sb[v] += dz;
              sw[v] = fmaf(dz, h, sw[v]);
            }
          }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) sm.red[(slot * p.cols + col) * V + v] = make_float2(sw[v], sb[v]);
    }
    __syncthreads();
    const int width = p.cols * V;
    for (int i = threadIdx.x; i < width && tile * width + i < a.channels; i += blockDim.x) {
      float2 s = make_float2(0.f, 0.f);
      for (int j = 0; j < p.slots; ++j) {
        const float2 b = sm.red[j * width + i];
        s.x += b.x;
        s.y += b.y;
      }
      sm.chan[tile * width + i] = s;
      float2& acc = sm.acc[tile * width + i];
      acc.x += s.x;
      acc.y += s.y;
    }
    __syncthreads();
  }
  if (!a.y) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  for (int g = warp; g < a.groups; g += warps) {
    float su = 0.f, suh = 0.f;
    for (int c = lane; c < w; c += 32) {
      const float2 b = sm.chan[g * w + c];
      const float wc = a.weight ? a.weight[g * w + c] : 1.f;
      su = fmaf(b.y, wc, su);
      suh = fmaf(b.x, wc, suh);
    }
    su = warp_sum(su);
    suh = warp_sum(suh);
    if (lane == 0) {
      if (p.parts > 1)
        part[((long long)n * p.parts + k) * a.groups + g] = make_float2(su, suh);
      else
        sm.group[g] = make_float2(su, suh);
    }
  }
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void split_dx(const GroupNormArgs& a, const GroupNormPlan& p, const SplitBwdSmem& sm, long long n,
                                         int k, const float2* part) {
  constexpr int U = 2;
  const int w = a.channels / a.groups;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const float inv = 1.f / (float)(a.spots * w);
  __syncthreads();
  for (int g = warp; g < a.groups; g += warps) {
    float su = 0.f, suh = 0.f;
    if (p.parts > 1) {
      const float2* at = part + (long long)n * p.parts * a.groups + g;
      for (int i = lane; i < p.parts; i += 32) {
        const float2 b = __ldcg(at + (long long)i * a.groups);
        su += b.x;
        suh += b.y;
      }
      su = warp_sum(su);
      suh = warp_sum(suh);
    } else {
      su = sm.group[g].x;
      suh = sm.group[g].y;
    }
    __syncwarp();
    if (lane == 0) sm.group[g] = make_float2(su * inv, suh * inv);
  }
  __syncthreads();
  const int slot = threadIdx.x / p.cols, col = threadIdx.x % p.cols;
  long long lo, hi;
  part_rows(a.spots, p.parts, k, lo, hi);
  const long long base = n * a.spots * a.channels;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* dy = static_cast<const T*>(a.dy) + base;
  T* dx = static_cast<T*>(a.y) + base;
  for (int tile = 0; tile < p.tiles; ++tile) {
    const int c = (tile * p.cols + col) * V;
    if (slot >= p.slots || c >= a.channels) continue;
    float mean[V], rstd[V], wt[V], bs[V], mu[V], muh[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = (c + v) / w;
      mean[v] = a.mean[n * a.groups + g];
      rstd[v] = a.rstd[n * a.groups + g];
      wt[v] = a.weight ? a.weight[c + v] : 1.f;
      bs[v] = a.bias ? a.bias[c + v] : 0.f;
      mu[v] = sm.group[g].x;
      muh[v] = sm.group[g].y;
    }
    const long long step = (long long)p.slots * a.channels, at = (lo + slot) * a.channels + c;
    const T *px = x + at, *pd = dy + at;
    T* to = dx + at;
    for (int left = slot_rows(lo, hi, slot, p.slots); left > 0;
         left -= U, px += U * step, pd += U * step, to += U * step) {
      Pack<T, V> q[U], d[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i < left) {
          q[i].load(px + i * step);
          d[i].load(pd + i * step);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i < left) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float h = (q[i].x[v] - mean[v]) * rstd[v];
            const float u = d[i].x[v] * slope<T, ACT>(fmaf(h, wt[v], bs[v])) * wt[v];
            q[i].x[v] = rstd[v] * (u - mu[v] - h * muh[v]);
          }
          q[i].store(to + i * step);
        }
    }
  }
  __syncthreads();
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, kSplitThreadsPerSm / kNormThreads)
    k_gn_split_bwd(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(16) float2 smem[];
  SplitBwdSmem sm;
  sm.red = smem;
  sm.chan = sm.red + p.slots * p.cols * V;
  sm.acc = sm.chan + a.channels;
  sm.group = sm.acc + a.channels;
  for (int c = threadIdx.x; c < a.channels; c += blockDim.x) sm.acc[c] = make_float2(0.f, 0.f);
  __syncthreads();
  if (p.parts == 1) {
    for (long long n = blockIdx.x; n < a.batch; n += gridDim.x) {
      split_sums<T, V, ACT>(a, p, sm, n, 0, nullptr);
      if (a.y) split_dx<T, V, ACT>(a, p, sm, n, 0, nullptr);
    }
  } else {
    float2* part = static_cast<float2*>(a.work);
    unsigned* sync = reinterpret_cast<unsigned*>(static_cast<char*>(a.work) + p.off_sync);
    const int k = blockIdx.x % p.parts, step = gridDim.x / p.parts;
    long long n = blockIdx.x / p.parts;
    split_sums<T, V, ACT>(a, p, sm, n, k, part);
    if (a.y) sample_arrive(sync + n);
    for (; n < a.batch; n += step) {
      const long long next = n + step;
      if (next < a.batch) {
        split_sums<T, V, ACT>(a, p, sm, next, k, part);
        if (a.y) sample_arrive(sync + next);
      }
      if (a.y) {
        sample_wait(sync + n, (unsigned)p.parts);
        split_dx<T, V, ACT>(a, p, sm, n, k, part);
      }
    }
  }
  __syncthreads();
  float2* out = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.off_channels) + (long long)blockIdx.x * a.channels;
  for (int c = threadIdx.x; c < a.channels; c += blockDim.x) out[c] = sm.acc[c];
}

// dw, db = the sums of the blocks' rows of channel sums.
constexpr int kSumCols = 16, kSumRows = 32;
__global__ void __launch_bounds__(kSumCols * kSumRows) k_gn_sum_rows(const float2* __restrict__ rows, long long count,
                                                                     int channels, float* __restrict__ dw,
                                                                     float* __restrict__ db) {
  __shared__ float2 red[kSumRows][kSumCols];
  const int col = threadIdx.x % kSumCols, slot = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + col;
  float2 s = make_float2(0.f, 0.f);
  if (c < channels) {
#pragma unroll 4
    for (long long r = slot; r < count; r += kSumRows) {
      const float2 b = rows[r * channels + c];
      s.x += b.x;
      s.y += b.y;
    }
  }
  red[slot][col] = s;
  __syncthreads();
  for (int o = kSumRows / 2; o; o >>= 1) {
    if (slot < o) {
      red[slot][col].x += red[slot + o][col].x;
      red[slot][col].y += red[slot + o][col].y;
    }
    __syncthreads();
  }
  if (slot == 0 && c < channels) {
    if (dw) dw[c] = red[0][col].x;
    if (db) db[c] = red[0][col].y;
  }
}

// Any number of channels: one block per group for dx, one per channel for dw and db.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < kNormThreads / 32; ++i) v += red[i];
  return v;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_any_dx(const __grid_constant__ GroupNormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const int w = a.channels / a.groups;
  const float inv = 1.f / (float)(a.spots * w);
  for (long long id = blockIdx.x; id < a.batch * a.groups; id += gridDim.x) {
    const int g = (int)(id % a.groups);
    const long long base = id / a.groups * a.spots * a.channels + (long long)g * w;
    const float mean = a.mean[id], rstd = a.rstd[id];
    float su = 0.f, suh = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass) {
        su = block_sum(su, red) * inv;
        suh = block_sum(suh, red) * inv;
      }
      for (long long r = 0; r < a.spots; ++r)
        for (int i = threadIdx.x; i < w; i += kNormThreads) {
          const long long at = base + r * a.channels + i;
          const int c = g * w + i;
          const float wc = a.weight ? a.weight[c] : 1.f, h = (to_f32(static_cast<const T*>(a.x)[at]) - mean) * rstd;
          const float u = to_f32(static_cast<const T*>(a.dy)[at]) * slope<T, ACT>(fmaf(h, wc, a.bias ? a.bias[c] : 0.f)) * wc;
          if (pass) {
            static_cast<T*>(a.y)[at] = from_f32<T>(rstd * (u - su - h * suh));
          } else {
            su += u;
            suh = fmaf(u, h, suh);
          }
        }
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_any_dw(const __grid_constant__ GroupNormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const int c = blockIdx.x, g = c / (a.channels / a.groups);
  const float wc = a.weight ? a.weight[c] : 1.f, bc = a.bias ? a.bias[c] : 0.f;
  float sw = 0.f, sb = 0.f;
  for (long long i = threadIdx.x; i < a.batch * a.spots; i += kNormThreads) {
    const long long n = i / a.spots * a.groups + g;
    const float h = (to_f32(static_cast<const T*>(a.x)[i * a.channels + c]) - a.mean[n]) * a.rstd[n];
    const float dz = to_f32(static_cast<const T*>(a.dy)[i * a.channels + c]) * slope<T, ACT>(fmaf(h, wc, bc));
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

template <typename T, int V, int ACT>
static cudaError_t run_small(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  switch (p.nv) {
    case 1: k_gn_small_bwd<T, V, 1, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes); break;
    case 2: k_gn_small_bwd<T, V, 2, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes); break;
    case 4: k_gn_small_bwd<T, V, 4, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes); break;
    default:
      if constexpr (V == 1) k_gn_small_bwd<T, 1, 8, ACT><<<p.grid, kNormThreads, 0, st>>>(a, p.lanes);
  }
  return cudaGetLastError();
}

template <typename T, int V, int ACT>
static cudaError_t run_split(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (p.smem > 48 * 1024)
    e = cudaFuncSetAttribute(k_gn_split_bwd<T, V, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem);
  if (e != cudaSuccess) return e;
  if (p.parts == 1) {
    k_gn_split_bwd<T, V, ACT><<<p.grid, p.threads, p.smem, st>>>(a, p);
    return cudaGetLastError();
  }
  e = cudaMemsetAsync(static_cast<char*>(a.work) + p.off_sync, 0, sizeof(unsigned) * a.batch, st);
  if (e != cudaSuccess) return e;
  GroupNormArgs a2 = a;
  GroupNormPlan p2 = p;
  void* args[] = {&a2, &p2};
  return cudaLaunchCooperativeKernel(k_gn_split_bwd<T, V, ACT>, dim3(p.grid), dim3(p.threads), args, (size_t)p.smem, st);
}

template <typename T, int ACT>
static cudaError_t run(const GroupNormArgs& a, const GroupNormPlan& p, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  cudaError_t e;
  if (p.kind == GroupNormPlan::kAny) {
    if (a.y) k_gn_any_dx<T, ACT><<<p.grid, kNormThreads, 0, st>>>(a);
    if (a.dw || a.db) k_gn_any_dw<T, ACT><<<a.channels, kNormThreads, 0, st>>>(a);
    return cudaGetLastError();
  }
  if (p.kind == GroupNormPlan::kSmall) {
    e = p.vec == W ? run_small<T, W, ACT>(a, p, st) : run_small<T, 1, ACT>(a, p, st);
  } else if (p.vec == 4) {
    e = run_split<T, 4, ACT>(a, p, st);
  } else {
    if constexpr (sizeof(T) == 2)
      e = p.vec == 2 ? run_split<T, 2, ACT>(a, p, st) : run_split<T, 1, ACT>(a, p, st);
    else
      e = run_split<T, 1, ACT>(a, p, st);
  }
  if (e == cudaSuccess && (a.dw || a.db)) {
    const float2* rows = reinterpret_cast<const float2*>(static_cast<const char*>(a.work) + p.off_channels);
    k_gn_sum_rows<<<(a.channels + kSumCols - 1) / kSumCols, kSumCols * kSumRows, 0, st>>>(rows, p.channel_rows, a.channels,
                                                                                        a.dw, a.db);
    e = cudaGetLastError();
  }
  return e;
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

cudaError_t launch_group_norm_backward(ElemType t, const GroupNormArgs& a, cudaStream_t st) {
  const GroupNormPlan p = plan_group_norm(t, a, true, group_norm_align(a));
  switch (t) {
    case kF32: return gn::run_act<float>(a, p, st);
    case kBF16: return gn::run_act<__nv_bfloat16>(a, p, st);
    default: return gn::run_act<__half>(a, p, st);
  }
}

}  // namespace tfb
