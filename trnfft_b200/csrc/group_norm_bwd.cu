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
__global__ void __launch_bounds__(kNormThreads, small_blocks_bwd(NV)) k_gn_small_bwd(const __grid_constant__ GroupNormArgs a, int lanes) {
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
  const long long step = slots / a.groups * a.spots * a.channels;  // from one of a thread's groups to its next
  const long long base = first / a.groups * a.spots * a.channels + (long long)g * w;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* dy = static_cast<const T*>(a.dy) + base;
  T* dx = static_cast<T*>(a.y) + base;
  int left = first < slots && first < total ? (int)((total - first + slots - 1) / slots) : 0;
  int turns = (int)((total + slots - 1) / slots);
  const float *mean_at = a.mean + first, *rstd_at = a.rstd + first;
  typename Pack<T, V>::Raw ahead_x[NV], ahead_dy[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  if (left > 0) {
    next_mean = *mean_at;
    next_rstd = *rstd_at;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (left > 0 && off[j] >= 0) {
      ahead_x[j] = Pack<T, V>::raw(x + off[j]);
      ahead_dy[j] = Pack<T, V>::raw(dy + off[j]);
    }
  for (; turns > 0; --turns, --left, x += step, dy += step, dx += step) {
    Pack<T, V> h[NV], u[NV];
    const float mean = next_mean, rstd = next_rstd;
    if (left > 1) {
      mean_at += slots;
      rstd_at += slots;
      next_mean = *mean_at;
      next_rstd = *rstd_at;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      h[j].unpack(ahead_x[j]);
      u[j].unpack(ahead_dy[j]);
      if (left > 1 && off[j] >= 0) {
        ahead_x[j] = Pack<T, V>::raw(x + step + off[j]);
        ahead_dy[j] = Pack<T, V>::raw(dy + step + off[j]);
      }
    }
    float su = 0.f, suh = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (left > 0 && off[j] >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float hv = (h[j].x[v] - mean) * rstd;
          const float dz = u[j].x[v] * slope<ACT>(fmaf(hv, wt[j][v], bs[j][v]));
          db[j][v] += dz;
          dw[j][v] = fmaf(dz, hv, dw[j][v]);
          h[j].x[v] = hv;
          u[j].x[v] = dz * wt[j][v];
          su += u[j].x[v];
          suh = fmaf(u[j].x[v], hv, suh);
        }
      }
    if (!a.y) continue;
    lanes_sum(su, suh, lanes);
    su *= inv;
    suh *= inv;
    if (left > 0) {
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
  float2* red;    // slots * channels: sums of (dz h, dz) of a slot
  float2* chan;   // channels: of the block's rows of one sample
  float2* acc;    // channels: of all its samples
  float2* group;  // groups: (mean of u, mean of u h)
};

// The slots' sums joined: of each channel, added to the block's; of each group.
__device__ __forceinline__ void join_slots_bwd(const GroupNormArgs& a, const GroupNormPlan& p, const SplitBwdSmem& sm,
                                               float2* out) {
  const int w = a.channels / a.groups;
  __syncthreads();
  for (int i = threadIdx.x; i < a.channels; i += blockDim.x) {
    float2 s = make_float2(0.f, 0.f);
    for (int j = 0; j < p.slots; ++j) {
      const float2 b = sm.red[j * a.channels + i];
      s.x += b.x;
      s.y += b.y;
    }
    float2& acc = sm.acc[i];
    acc.x += s.x;
    acc.y += s.y;
    const float wc = a.weight ? a.weight[i] : 1.f;
    sm.chan[i] = make_float2(s.y * wc, s.x * wc);
  }
  __syncthreads();
  if (!out) return;
  const int lanes = p.glanes, lane = threadIdx.x & (lanes - 1);
  for (int g0 = 0; g0 < a.groups; g0 += blockDim.x / lanes) {
    const int g = g0 + threadIdx.x / lanes;
    float su = 0.f, suh = 0.f;
    if (g < a.groups)
      for (int c = lane; c < w; c += lanes) {
        const float2 b = sm.chan[g * w + c];
        su += b.x;
        suh += b.y;
      }
    lanes_sum(su, suh, lanes);
    if (g < a.groups && lane == 0) out[g] = make_float2(su, suh);
  }
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void split_sums(const GroupNormArgs& a, const GroupNormPlan& p, const SplitBwdSmem& sm,
                                           const SplitPlace& at, SplitColumn<V>& col, long long n, float2* out) {
  constexpr int U = rows_ahead(2 * V * sizeof(T));
  const long long base = n * a.spots * a.channels + at.first;
  for (int tile = 0; tile < p.tiles; ++tile) {
    if (p.tiles > 1) col.set(a, p, at, tile);
    if (!col.live) continue;
    float mean[V], gain[V], sw[V], sb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const long long g = n * a.groups + col.group(v);
      mean[v] = a.mean[g];
      gain[v] = a.rstd[g] * col.wt[v];
      sw[v] = sb[v] = 0.f;
    }
    const T* px = static_cast<const T*>(a.x) + base + col.c;
    const T* pd = static_cast<const T*>(a.dy) + base + col.c;
    for (int left = at.mine; left > 0; left -= U, px += U * at.step, pd += U * at.step) {
      typename Pack<T, V>::Raw rx[U], rd[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i < left) {
          rx[i] = Pack<T, V>::raw(px + i * at.step);
          rd[i] = Pack<T, V>::raw(pd + i * at.step);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i < left) {
          Pack<T, V> q, d;
          q.unpack(rx[i]);
          d.unpack(rd[i]);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float e = q.x[v] - mean[v], dz = d.x[v] * slope<ACT>(fmaf(e, gain[v], col.bs[v]));
            sb[v] += dz;
            sw[v] = fmaf(dz, e, sw[v]);
          }
        }
    }
    float2* red = sm.red + at.slot * a.channels + col.c;
#pragma unroll
    for (int v = 0; v < V; ++v) red[v] = make_float2(sw[v] * a.rstd[n * a.groups + col.group(v)], sb[v]);
  }
  join_slots_bwd(a, p, sm, out);
}

// The same from the block's stream of rows.
template <typename T, int V, int ACT>
__device__ __forceinline__ void stream_sums(const GroupNormArgs& a, const GroupNormPlan& p, unsigned char* raw,
                                            const SplitBwdSmem& sm, const SplitPlace& at, const SplitColumn<V>& col,
                                            long long n, int k, float2* out) {
  const long long base = (n * a.spots + (long long)k * p.part_rows) * a.channels;
  const void* const src[2] = {static_cast<const T*>(a.x) + base, static_cast<const T*>(a.dy) + base};
  RowStream<2> rows(raw, p, at.rows, (long long)a.channels * sizeof(T), src);
  float mean[V], gain[V], sw[V], sb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const long long g = n * a.groups + (col.live ? col.group(v) : 0);
    mean[v] = a.mean[g];
    gain[v] = a.rstd[g] * col.wt[v];
    sw[v] = sb[v] = 0.f;
  }
  for (int i = 0; i < rows.count; ++i) {
    rows.wait(i);
    if (col.live) {
      const T* px = reinterpret_cast<const T*>(rows.buffer(i, 0)) + at.slot * a.channels + col.c;
      const T* pd = reinterpret_cast<const T*>(rows.buffer(i, 1)) + at.slot * a.channels + col.c;
      const int mine = rows.rows_of(i);
#pragma unroll 4
      for (int r = at.slot; r < mine; r += p.slots, px += at.step, pd += at.step) {
        Pack<T, V> q, d;
        q.load(px);
        d.load(pd);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float e = q.x[v] - mean[v], dz = d.x[v] * slope<ACT>(fmaf(e, gain[v], col.bs[v]));
          sb[v] += dz;
          sw[v] = fmaf(dz, e, sw[v]);
        }
      }
    }
    rows.release(i);
  }
  rows.finish();
  if (col.live) {
    float2* red = sm.red + at.slot * a.channels + col.c;
#pragma unroll
    for (int v = 0; v < V; ++v) red[v] = make_float2(sw[v] * a.rstd[n * a.groups + col.group(v)], sb[v]);
  }
  join_slots_bwd(a, p, sm, out);
}

// dx of the block's rows of sample n, given the sums of (u, u h) over its groups times `inv`.
template <typename T, int V, int ACT>
__device__ __forceinline__ void split_dx(const GroupNormArgs& a, const GroupNormPlan& p, const SplitPlace& at,
                                         SplitColumn<V>& col, long long n, const float2* group, float inv) {
  constexpr int U = rows_ahead(2 * V * sizeof(T));
  const long long first = n * a.spots * a.channels + at.first;
  for (int tile = 0; tile < p.tiles; ++tile) {
    if (p.tiles > 1) col.set(a, p, at, tile);
    if (!col.live) continue;
    // with e = x - mean: dx = gain dz - rstd mean(u) - e rstd^2 mean(u h)
    float mean[V], gain[V], mu[V], muh[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = col.group(v);
      const float rstd = a.rstd[n * a.groups + g];
      const float2 m = group[g];
      mean[v] = a.mean[n * a.groups + g];
      gain[v] = rstd * col.wt[v];
      mu[v] = rstd * (m.x * inv);
      muh[v] = rstd * rstd * (m.y * inv);
    }
    const T* px = static_cast<const T*>(a.x) + first + col.c;
    const T* pd = static_cast<const T*>(a.dy) + first + col.c;
    T* to = static_cast<T*>(a.y) + first + col.c;
    for (int left = at.mine; left > 0; left -= U, px += U * at.step, pd += U * at.step, to += U * at.step) {
      typename Pack<T, V>::Raw rx[U], rd[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i < left) {
          rx[i] = Pack<T, V>::raw(px + i * at.step);
          rd[i] = Pack<T, V>::raw(pd + i * at.step);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i < left) {
          Pack<T, V> q, d;
          q.unpack(rx[i]);
          d.unpack(rd[i]);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float e = q.x[v] - mean[v], dz = d.x[v] * slope<ACT>(fmaf(e, gain[v], col.bs[v]));
            q.x[v] = fmaf(-e, muh[v], fmaf(dz, gain[v], -mu[v]));
          }
          q.store(to + i * at.step);
        }
    }
  }
}

__device__ __forceinline__ SplitBwdSmem bwd_smem(const GroupNormArgs& a, const GroupNormPlan& p, float2* smem) {
  SplitBwdSmem sm;
  sm.red = smem;
  sm.chan = sm.red + p.slots * a.channels;
  sm.acc = sm.chan + a.channels;
  sm.group = sm.acc + a.channels;
  for (int c = threadIdx.x; c < a.channels; c += blockDim.x) sm.acc[c] = make_float2(0.f, 0.f);
  __syncthreads();
  return sm;
}

__device__ __forceinline__ void leave_channels(const GroupNormArgs& a, const GroupNormPlan& p, const SplitBwdSmem& sm) {
  __syncthreads();
  float2* out = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.off_channels) + (long long)blockIdx.x * a.channels;
  for (int c = threadIdx.x; c < a.channels; c += blockDim.x) out[c] = sm.acc[c];
}

// A block takes whole samples.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_whole_bwd(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(16) float2 smem[];
  const SplitBwdSmem sm = bwd_smem(a, p, smem);
  const SplitPlace at(a, p, 0);
  SplitColumn<V> col;
  col.set(a, p, at, 0);
  const float inv = 1.f / ((float)a.spots * (float)(a.channels / a.groups));
  for (long long n = blockIdx.x; n < a.batch; n += gridDim.x) {
    split_sums<T, V, ACT>(a, p, sm, at, col, n, sm.group);
    __syncthreads();
    if (a.y) split_dx<T, V, ACT>(a, p, at, col, n, sm.group, inv);
  }
  leave_channels(a, p, sm);
}

// The same on samples streamed into shared memory, where both passes read them.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_whole_stream_bwd(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(128) unsigned char raw[];
  const long long size = a.spots * a.channels;
  const void* const src[2] = {a.x, a.dy};
  SampleStream<2> samples(raw, p, a.batch, size * (long long)sizeof(T), src);
  const SplitBwdSmem sm =
      bwd_smem(a, p, reinterpret_cast<float2*>(raw + p.sample_buffers * 2 * size * sizeof(T) + 8 * kMaxSampleBuffers));
  const SplitPlace at(a, p, 0);
  SplitColumn<V> col;
  col.set(a, p, at, 0);
  const float inv = 1.f / ((float)a.spots * (float)(a.channels / a.groups));
  for (int i = 0; i < samples.count; ++i) {
    const long long n = blockIdx.x + (long long)i * gridDim.x;
    samples.wait(i);
    const T* x = reinterpret_cast<const T*>(samples.buffer(i, 0)) + at.slot * a.channels + col.c;
    const T* dy = reinterpret_cast<const T*>(samples.buffer(i, 1)) + at.slot * a.channels + col.c;
    float mean[V], rstd[V], gain[V];
    if (col.live) {
      float sw[V], sb[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const long long g = n * a.groups + col.group(v);
        mean[v] = a.mean[g];
        rstd[v] = a.rstd[g];
        gain[v] = rstd[v] * col.wt[v];
        sw[v] = sb[v] = 0.f;
      }
      const T *px = x, *pd = dy;
#pragma unroll 2
      for (int r = 0; r < at.mine; ++r, px += at.step, pd += at.step) {
        Pack<T, V> q, d;
        q.load(px);
        d.load(pd);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float e = q.x[v] - mean[v], dz = d.x[v] * slope<ACT>(fmaf(e, gain[v], col.bs[v]));
          sb[v] += dz;
          sw[v] = fmaf(dz, e, sw[v]);
        }
      }
      float2* red = sm.red + at.slot * a.channels + col.c;
#pragma unroll
      for (int v = 0; v < V; ++v) red[v] = make_float2(sw[v] * rstd[v], sb[v]);
    }
    join_slots_bwd(a, p, sm, sm.group);
    __syncthreads();
    if (a.y && col.live) {
      float mu[V], muh[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = sm.group[col.group(v)];
        mu[v] = rstd[v] * (m.x * inv);
        muh[v] = rstd[v] * rstd[v] * (m.y * inv);
      }
      T* to = static_cast<T*>(a.y) + n * size + at.first + col.c;
      const T *px = x, *pd = dy;
#pragma unroll 2
      for (int r = 0; r < at.mine; ++r, px += at.step, pd += at.step, to += at.step) {
        Pack<T, V> q, d;
        q.load(px);
        d.load(pd);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float e = q.x[v] - mean[v], dz = d.x[v] * slope<ACT>(fmaf(e, gain[v], col.bs[v]));
          q.x[v] = fmaf(-e, muh[v], fmaf(dz, gain[v], -mu[v]));
        }
        q.store(to);
      }
    }
    samples.release(i);
  }
  samples.finish();
  leave_channels(a, p, sm);
}

// Block = part blockIdx.x % parts of sample blockIdx.x / parts: its channels' and groups' sums; the
// sample's last block adds up the groups'.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_sums(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(128) unsigned char raw[];
  const SplitBwdSmem sm = bwd_smem(a, p, reinterpret_cast<float2*>(raw + (p.stage_rows ? kStreamBytes + 64 : 0)));
  const long long n = blockIdx.x / p.parts;
  const int k = blockIdx.x % p.parts;
  float2* part = static_cast<float2*>(a.work) + n * p.parts * a.groups;
  {
    const SplitPlace at(a, p, k);
    SplitColumn<V> col;
    col.set(a, p, at, 0);
    float2* out = a.y ? part + (long long)k * a.groups : nullptr;
    if (p.stage_rows)
      stream_sums<T, V, ACT>(a, p, raw, sm, at, col, n, k, out);
    else
      split_sums<T, V, ACT>(a, p, sm, at, col, n, out);
  }
  leave_channels(a, p, sm);
  if (!a.y) return;
  unsigned* count = reinterpret_cast<unsigned*>(static_cast<char*>(a.work) + p.off_sync);
  if (!last_of_sample(count + n, p.parts)) return;
  float2* result = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.off_result) + n * a.groups;
  const int lanes = p.planes, lane = threadIdx.x & (lanes - 1);
  for (int g0 = 0; g0 < a.groups; g0 += blockDim.x / lanes) {
    const int g = g0 + threadIdx.x / lanes;
    float su = 0.f, suh = 0.f;
    if (g < a.groups) {
#pragma unroll 8
      for (int i = lane; i < p.parts; i += lanes) {
        const float2 b = __ldcg(part + (long long)i * a.groups + g);
        su += b.x;
        suh += b.y;
      }
    }
    lanes_sum(su, suh, lanes);
    if (g < a.groups && lane == 0) result[g] = make_float2(su, suh);
  }
}

// From the last sample to the first: the end of x and dy is in L2 still.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_dx(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(128) unsigned char raw[];
  const unsigned b = gridDim.x - 1 - blockIdx.x;
  const long long n = b / p.parts;
  const int k = b % p.parts;
  const SplitPlace at(a, p, k);
  SplitColumn<V> col;
  col.set(a, p, at, 0);
  const float2* result = reinterpret_cast<const float2*>(static_cast<const char*>(a.work) + p.off_result) + n * a.groups;
  const float inv = 1.f / ((float)a.spots * (float)(a.channels / a.groups));
  if (!p.stage_rows) {
    split_dx<T, V, ACT>(a, p, at, col, n, result, inv);
    return;
  }
  const long long base = (n * a.spots + (long long)k * p.part_rows) * a.channels;
  const void* const src[2] = {static_cast<const T*>(a.x) + base, static_cast<const T*>(a.dy) + base};
  RowStream<2> rows(raw, p, at.rows, (long long)a.channels * sizeof(T), src);
  float mean[V], gain[V], mu[V], muh[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int g = col.live ? col.group(v) : 0;
    const float rstd = a.rstd[n * a.groups + g];
    const float2 m = result[g];
    mean[v] = a.mean[n * a.groups + g];
    gain[v] = rstd * col.wt[v];
    mu[v] = rstd * (m.x * inv);
    muh[v] = rstd * rstd * (m.y * inv);
  }
  T* to = static_cast<T*>(a.y) + base + (long long)at.slot * a.channels + col.c;
  for (int i = 0; i < rows.count; ++i) {
    rows.wait(i);
    if (col.live) {
      const T* px = reinterpret_cast<const T*>(rows.buffer(i, 0)) + at.slot * a.channels + col.c;
      const T* pd = reinterpret_cast<const T*>(rows.buffer(i, 1)) + at.slot * a.channels + col.c;
      const int mine = rows.rows_of(i);
#pragma unroll 4
      for (int r = at.slot; r < mine; r += p.slots, px += at.step, pd += at.step, to += at.step) {
        Pack<T, V> q, d;
        q.load(px);
        d.load(pd);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float e = q.x[v] - mean[v], dz = d.x[v] * slope<ACT>(fmaf(e, gain[v], col.bs[v]));
          q.x[v] = fmaf(-e, muh[v], fmaf(dz, gain[v], -mu[v]));
        }
        q.store(to);
      }
    }
    rows.release(i);
  }
  rows.finish();
}

// dw, db = the sums of the blocks' rows of channel sums.
constexpr int kSumCols = 8, kSumRows = 64;
__global__ void __launch_bounds__(kSumCols * kSumRows) k_gn_sum_rows(const float2* __restrict__ rows, long long count,
                                                                     int channels, float* __restrict__ dw,
                                                                     float* __restrict__ db) {
  __shared__ float2 red[kSumRows][kSumCols];
  const int col = threadIdx.x % kSumCols, slot = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + col;
  float2 s = make_float2(0.f, 0.f);
  if (c < channels) {
#pragma unroll 8
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

// Any number of channels: one block per group for dx, one per channel for dw and db, sums in 64 bits.
template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_any_dx(const __grid_constant__ GroupNormArgs a) {
  __shared__ double red[kNormThreads / 32];
  const int w = a.channels / a.groups;
  const double inv = 1.0 / ((double)a.spots * w);
  for (long long id = blockIdx.x; id < a.batch * a.groups; id += gridDim.x) {
    const int g = (int)(id % a.groups);
    const long long base = id / a.groups * a.spots * a.channels + (long long)g * w;
    const float mean = a.mean[id], rstd = a.rstd[id];
    double sum = 0.0, sum_h = 0.0;
    float mu = 0.f, muh = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass) {
        mu = (float)(block_sum(sum, red) * inv);
        muh = (float)(block_sum(sum_h, red) * inv);
      }
      for (AnyPlace at(w); at.row < a.spots; at.next()) {
        const long long i = base + at.row * a.channels + at.c;
        const int c = g * w + at.c;
        const float wc = a.weight ? a.weight[c] : 1.f, h = (to_f32(static_cast<const T*>(a.x)[i]) - mean) * rstd;
        const float u = to_f32(static_cast<const T*>(a.dy)[i]) * slope<ACT>(fmaf(h, wc, a.bias ? a.bias[c] : 0.f)) * wc;
        if (pass) {
          static_cast<T*>(a.y)[i] = from_f32<T>(rstd * (u - mu - h * muh));
        } else {
          sum += u;
          sum_h += (double)u * h;
        }
      }
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_any_dw(const __grid_constant__ GroupNormArgs a) {
  __shared__ double red[kNormThreads / 32];
  const int c = blockIdx.x, g = c / (a.channels / a.groups);
  const float wc = a.weight ? a.weight[c] : 1.f, bc = a.bias ? a.bias[c] : 0.f;
  double sw = 0.0, sb = 0.0;
  for (long long i = threadIdx.x; i < a.batch * a.spots; i += kNormThreads) {
    const long long n = i / a.spots * a.groups + g;
    const float h = (to_f32(static_cast<const T*>(a.x)[i * a.channels + c]) - a.mean[n]) * a.rstd[n];
    const float dz = to_f32(static_cast<const T*>(a.dy)[i * a.channels + c]) * slope<ACT>(fmaf(h, wc, bc));
    sb += dz;
    sw += (double)dz * h;
  }
  sw = block_sum(sw, red);
  sb = block_sum(sb, red);
  if (threadIdx.x == 0) {
    if (a.dw) a.dw[c] = (float)sw;
    if (a.db) a.db[c] = (float)sb;
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
  cudaError_t e;
  if (p.sample_buffers) {
    const int smem = (int)(p.sample_buffers * 2 * a.spots * a.channels * sizeof(T)) + 8 * kMaxSampleBuffers + p.smem;
    e = allow_smem<k_gn_whole_stream_bwd<T, V, ACT>>(smem);
    if (e == cudaSuccess) k_gn_whole_stream_bwd<T, V, ACT><<<p.grid, p.threads, smem, st>>>(a, p);
    return e == cudaSuccess ? cudaGetLastError() : e;
  }
  if (p.parts == 1) {
    e = allow_smem<k_gn_whole_bwd<T, V, ACT>>(p.smem);
    if (e == cudaSuccess) k_gn_whole_bwd<T, V, ACT><<<p.grid, p.threads, p.smem, st>>>(a, p);
    return e == cudaSuccess ? cudaGetLastError() : e;
  }
  const int stream = p.stage_rows ? kStreamBytes + 64 : 0;
  e = allow_smem<k_gn_sums<T, V, ACT>>(p.smem + stream);
  if (e == cudaSuccess) e = allow_smem<k_gn_dx<T, V, ACT>>(stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(static_cast<char*>(a.work) + p.off_sync, 0, sizeof(unsigned) * a.batch, st);
  if (e != cudaSuccess) return e;
  k_gn_sums<T, V, ACT><<<p.grid, p.threads, p.smem + stream, st>>>(a, p);
  if (a.y) k_gn_dx<T, V, ACT><<<p.grid, p.threads, stream, st>>>(a, p);
  return cudaGetLastError();
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
