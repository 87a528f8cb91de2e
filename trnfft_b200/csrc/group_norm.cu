// Group normalisation with an activation over channels-last features:
//
//   mean, var over the spots and the channels of one group of one sample,
//   h = (x - mean) rstd,  z = h w + b,  y = act(z),   rstd = 1 / sqrt(var + eps)
//
// Bound by HBM: x read once, y written once.  Two forms reach that.
//   kSmall  a group of one sample has few values (a frame's features, the
//           heads of an attention's output): a few threads keep them in
//           registers between the statistics and the result.
//   kSplit  blocks of whole rows (any number of channels, any grouping,
//           contiguous in memory).  A sample of up to 48 KB is one block's,
//           which reads it twice, the second time from L1 or L2.  A larger one
//           is cut into parts: a first kernel takes their statistics (the last
//           block of a sample joins them), a second one applies them, from
//           the last sample to the first, since the end of x is in L2 still.
//           Keeping parts resident that wait for one another, so that the
//           second read always hits L2, was slower: what then fits L2 leaves
//           each thread a dozen rows between two meetings
//           (8 x 257 x 626 x 48 fp32: 206 us).
// The variance is never a difference of large sums: a thread sums a channel's
// distances d from its first value there, and their squares, and leaves
// mean = first + sum(d) / n and M2 = sum(d^2) - sum(d)^2 / n.  However far off
// that first value is, it is one of the values, so M2 of the group is at least
// its own square and the difference loses at most n 2^-24 of it (n: rows of
// one thread, dozens to hundreds).  Sets join by M2 = sum(M2_i + n_i (mean_i -
// mean)^2), where an estimate of the mean, the first set's, serves first: if
// its distance from the mean is more than 4 deviations (kFar), so that the
// difference would lose more than 17 roundings, the sets are joined again
// from the mean.  The values of a small group, which stay in registers, alike
// (512 values, the first a thousand deviations off: 1.9e-5 -> 5.7e-7 off).
#include "group_norm.cuh"

#include <algorithm>

namespace tfb {
namespace gn {

constexpr float kFar = 16.f;  // square of the distance, over the variance

// ---------------------------------------------------------------- kSmall
// `lanes` threads per (sample, group), NV accesses of V elements each.  The
// element with index i of a group is channel i % w of spot i / w; accesses of
// V > 1 elements are used for one spot only.  A thread's groups are a
// multiple of `groups` apart, so its channels and their parameters stay.
template <typename T, int V, int NV, int ACT>
__global__ void __launch_bounds__(kNormThreads, small_blocks(NV)) k_gn_small(const __grid_constant__ GroupNormArgs a, int lanes) {
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
  const long long step = slots / a.groups * a.spots * a.channels;  // from one of a thread's groups to its next
  const long long base = first / a.groups * a.spots * a.channels + (long long)g * w;
  const T* x = static_cast<const T*>(a.x) + base;
  T* y = static_cast<T*>(a.y) + base;
  // every thread of a warp takes the same number of turns: the shuffles need them all
  int left = first < slots && first < total ? (int)((total - first + slots - 1) / slots) : 0;
  int turns = (int)((total + slots - 1) / slots);
  float *mean_at = a.mean ? a.mean + first : nullptr, *rstd_at = a.rstd + first;
  typename Pack<T, V>::Raw ahead[2][NV];  // the next two groups' values, on their way
#pragma unroll
  for (int d = 0; d < 2; ++d)
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (left > d && off[j] >= 0) ahead[d][j] = Pack<T, V>::raw(x + d * step + off[j]);
  for (; turns > 0; --turns, --left, x += step, y += step) {
    Pack<T, V> p[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      p[j].unpack(ahead[0][j]);
      ahead[0][j] = ahead[1][j];
      if (left > 2 && off[j] >= 0) ahead[1][j] = Pack<T, V>::raw(x + 2 * step + off[j]);
    }
    // distances from the group's first value (see the note on the variance above)
    const float origin = __shfl_sync(~0u, p[0].x[0], threadIdx.x & 31 & -lanes);
    float s = 0.f, ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (off[j] >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          p[j].x[v] -= origin;
          s += p[j].x[v];
          ss = fmaf(p[j].x[v], p[j].x[v], ss);
        }
      }
    lanes_sum(s, ss, lanes);
    float mean = s * inv, var = fmaxf(fmaf(-mean, mean, ss * inv), 0.f);
    // (a first value far from the others: distances from their mean, in that group alone)
    const bool far = mean * mean > kFar * var;
    if (__any_sync(~0u, far)) {
      float s = 0.f, ss = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (off[j] >= 0) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float d = p[j].x[v] - mean;
            s += d;
            ss = fmaf(d, d, ss);
          }
        }
      lanes_sum(s, ss, lanes);
      if (far) {
        const float rest = s * inv;
        mean += rest;
        var = fmaxf(fmaf(-rest, rest, ss * inv), 0.f);
      }
    }
    const float rstd = __frsqrt_rn((ss - ss == 0.f ? var : ss) + a.eps);  // NaN stays NaN
    if (left > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (off[j] >= 0) {
#pragma unroll
          for (int v = 0; v < V; ++v) p[j].x[v] = activate<ACT>(fmaf((p[j].x[v] - mean) * rstd, wt[j][v], bs[j][v]));
          p[j].store(y + off[j]);
        }
      if (mean_at) {
        if (lane == 0) {
          *mean_at = origin + mean;
          *rstd_at = rstd;
        }
        mean_at += slots;
        rstd_at += slots;
      }
    }
  }
}

// ---------------------------------------------------------------- kSplit

__device__ __forceinline__ float rstd_of(float var, float eps) { return __frsqrt_rn((var < 0.f ? 0.f : var) + eps); }

// The join of sets by `lanes` threads: sums(origin, t, tt) adds up, over a thread's sets, n_i (mean_i -
// origin) and M2_i + n_i (mean_i - origin)^2.  inv: 1 / all n.
struct Joined {
  float mean, m2;
};
template <typename Sums>
__device__ __forceinline__ Joined join_sets(float origin, float inv, int lanes, const Sums& sums) {
  float t = 0.f, tt = 0.f;
  sums(origin, t, tt);
  lanes_sum(t, tt, lanes);
  Joined all{fmaf(t, inv, origin), fmaf(-t * inv, t, tt)};
  const bool far = t * inv * t > kFar * fmaxf(all.m2, 0.f);
  if (__any_sync(~0u, far)) {
    t = tt = 0.f;
    sums(all.mean, t, tt);
    lanes_sum(t, tt, lanes);
    if (far) all = {fmaf(t, inv, all.mean), fmaf(-t * inv, t, tt)};
  }
  return all;
}

// Joins the slots' sets of each group, by `glanes` threads: the distances of their means from the first of
// them, as above.  Slots below `extra` have one row more than the others.
__device__ __forceinline__ void join_slots(const GroupNormArgs& a, const GroupNormPlan& p, const float2* red,
                                           const SplitPlace& at, float2* out) {
  __syncthreads();
  const int w = a.channels / a.groups, lanes = p.glanes, lane = threadIdx.x & (lanes - 1), full = at.rows / p.slots, extra = at.rows % p.slots;
  const float inv = 1.f / ((float)at.rows * (float)w);
  for (int g0 = 0; g0 < a.groups; g0 += blockDim.x / lanes) {
    const int g = g0 + threadIdx.x / lanes;
    const Joined all = join_sets(g < a.groups ? red[g * w].x : 0.f, inv, lanes, [&](float origin, float& t, float& tt) {
      if (g >= a.groups) return;
      for (int j = 0, c = lane; j < p.slots; c += lanes) {
        while (c >= w) c -= w, ++j;
        if (j >= p.slots) break;
        const float2 b = red[j * a.channels + g * w + c];
        const float d = b.x - origin, nd = d * (float)(full + (j < extra));
        t += nd;
        tt += fmaf(nd, d, b.y);
      }
    });
    if (g < a.groups && lane == 0) out[g] = make_float2(all.mean, all.m2);
  }
}

// The sets of the block's rows of sample n, joined for each group: out[g], as (mean, M2).
template <typename T, int V>
__device__ __forceinline__ void split_stats(const GroupNormArgs& a, const GroupNormPlan& p, float2* red,
                                            const SplitPlace& at, SplitColumn<V>& col, long long n, float2* out) {
  constexpr int U = rows_ahead(V * sizeof(T));
  const T* x = static_cast<const T*>(a.x) + n * a.spots * a.channels + at.first;
  for (int tile = 0; tile < p.tiles; ++tile) {
    if (p.tiles > 1) col.set(a, p, at, tile);
    if (!col.live) continue;
    const T* q = x + col.c;
    Pack<T, V> first;
    float s[V], ss[V];
#pragma unroll
    for (int v = 0; v < V; ++v) first.x[v] = s[v] = ss[v] = 0.f;
    if (at.mine) first.load(q);
    for (int left = at.mine; left > 0; left -= U, q += U * at.step) {
      typename Pack<T, V>::Raw r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) r[u] = Pack<T, V>::raw(q + u * at.step);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) {
          Pack<T, V> b;
          b.unpack(r[u]);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float d = b.x[v] - first.x[v];
            s[v] += d;
            ss[v] = fmaf(d, d, ss[v]);
          }
        }
    }
    const float inv = at.mine ? 1.f / (float)at.mine : 0.f;
    float2* to = red + at.slot * a.channels + col.c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float d = s[v] * inv;
      to[v] = make_float2(first.x[v] + d, fmaf(-s[v], d, ss[v]));
    }
  }
  join_slots(a, p, red, at, out);
}

// The same from the block's stream of rows.
template <typename T, int V>
__device__ __forceinline__ void stream_stats(const GroupNormArgs& a, const GroupNormPlan& p, unsigned char* raw, float2* red,
                                             const SplitPlace& at, const SplitColumn<V>& col, long long n, int k,
                                             float2* out) {
  const void* const src[1] = {static_cast<const T*>(a.x) + (n * a.spots + (long long)k * p.part_rows) * a.channels};
  RowStream<1> rows(raw, p, at.rows, (long long)a.channels * sizeof(T), src);
  Pack<T, V> first;
  float s[V], ss[V];
#pragma unroll
  for (int v = 0; v < V; ++v) first.x[v] = s[v] = ss[v] = 0.f;
  for (int i = 0; i < rows.count; ++i) {
    rows.wait(i);
    if (col.live) {
      const T* q = reinterpret_cast<const T*>(rows.buffer(i, 0)) + at.slot * a.channels + col.c;
      const int mine = rows.rows_of(i);
      if (i == 0 && at.slot < mine) first.load(q);
#pragma unroll 4
      for (int r = at.slot; r < mine; r += p.slots, q += at.step) {
        Pack<T, V> b;
        b.load(q);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = b.x[v] - first.x[v];
          s[v] += d;
          ss[v] = fmaf(d, d, ss[v]);
        }
      }
    }
    rows.release(i);
  }
  rows.finish();
  if (col.live) {
    const float inv = at.mine ? 1.f / (float)at.mine : 0.f;
    float2* to = red + at.slot * a.channels + col.c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float d = s[v] * inv;
      to[v] = make_float2(first.x[v] + d, fmaf(-s[v], d, ss[v]));
    }
  }
  join_slots(a, p, red, at, out);
}

// y of the block's rows of sample n, given (mean, rstd) of its groups.
template <typename T, int V, int ACT>
__device__ __forceinline__ void split_apply(const GroupNormArgs& a, const GroupNormPlan& p, const SplitPlace& at,
                                            SplitColumn<V>& col, long long n, const float2* group) {
  constexpr int U = rows_ahead(V * sizeof(T));
  const long long first = n * a.spots * a.channels + at.first;
  for (int tile = 0; tile < p.tiles; ++tile) {
    if (p.tiles > 1) col.set(a, p, at, tile);
    if (!col.live) continue;
    float mean[V], gain[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 s = group[col.group(v)];
      mean[v] = s.x;
      gain[v] = s.y * col.wt[v];
    }
    const T* from = static_cast<const T*>(a.x) + first + col.c;
    T* to = static_cast<T*>(a.y) + first + col.c;
    for (int left = at.mine; left > 0; left -= U, from += U * at.step, to += U * at.step) {
      typename Pack<T, V>::Raw r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) r[u] = Pack<T, V>::raw(from + u * at.step);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) {
          Pack<T, V> q;
          q.unpack(r[u]);
#pragma unroll
          for (int v = 0; v < V; ++v) q.x[v] = activate<ACT>(fmaf(q.x[v] - mean[v], gain[v], col.bs[v]));
          q.store(to + u * at.step);
        }
    }
  }
}

// A block takes whole samples.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_whole(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(16) float2 smem[];
  float2 *red = smem, *group = red + p.slots * a.channels;
  const SplitPlace at(a, p, 0);
  SplitColumn<V> col;
  col.set(a, p, at, 0);
  const float inv = 1.f / ((float)a.spots * (float)(a.channels / a.groups));
  for (long long n = blockIdx.x; n < a.batch; n += gridDim.x) {
    split_stats<T, V>(a, p, red, at, col, n, group);
    __syncthreads();
    for (int g = threadIdx.x; g < a.groups; g += blockDim.x) {
      const float rstd = rstd_of(group[g].y * inv, a.eps);
      group[g].y = rstd;
      if (a.mean) {
        a.mean[n * a.groups + g] = group[g].x;
        a.rstd[n * a.groups + g] = rstd;
      }
    }
    __syncthreads();
    split_apply<T, V, ACT>(a, p, at, col, n, group);
  }
}

// The same on samples streamed into shared memory, where both passes read them.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_whole_stream(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(128) unsigned char raw[];
  const long long size = a.spots * a.channels;
  const void* const src[1] = {a.x};
  SampleStream<1> samples(raw, p, a.batch, size * (long long)sizeof(T), src);
  float2* red = reinterpret_cast<float2*>(raw + p.sample_buffers * size * sizeof(T) + 8 * kMaxSampleBuffers);
  float2* group = red + p.slots * a.channels;
  const SplitPlace at(a, p, 0);
  SplitColumn<V> col;
  col.set(a, p, at, 0);
  const float inv = 1.f / ((float)a.spots * (float)(a.channels / a.groups)), inv_mine = at.mine ? 1.f / (float)at.mine : 0.f;
  for (int i = 0; i < samples.count; ++i) {
    const long long n = blockIdx.x + (long long)i * gridDim.x;
    samples.wait(i);
    const T* x = reinterpret_cast<const T*>(samples.buffer(i, 0)) + at.slot * a.channels + col.c;
    if (col.live) {
      Pack<T, V> first;
      float s[V], ss[V];
#pragma unroll
      for (int v = 0; v < V; ++v) first.x[v] = s[v] = ss[v] = 0.f;
      if (at.mine) first.load(x);
      const T* q = x;
#pragma unroll 4
      for (int r = 0; r < at.mine; ++r, q += at.step) {
        Pack<T, V> b;
        b.load(q);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = b.x[v] - first.x[v];
          s[v] += d;
          ss[v] = fmaf(d, d, ss[v]);
        }
      }
      float2* to = red + at.slot * a.channels + col.c;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = s[v] * inv_mine;
        to[v] = make_float2(first.x[v] + d, fmaf(-s[v], d, ss[v]));
      }
    }
    join_slots(a, p, red, at, group);
    __syncthreads();
    for (int g = threadIdx.x; g < a.groups; g += blockDim.x) {
      const float rstd = rstd_of(group[g].y * inv, a.eps);
      group[g].y = rstd;
      if (a.mean) {
        a.mean[n * a.groups + g] = group[g].x;
        a.rstd[n * a.groups + g] = rstd;
      }
    }
    __syncthreads();
    if (col.live) {
      float mean[V], gain[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 s = group[col.group(v)];
        mean[v] = s.x;
        gain[v] = s.y * col.wt[v];
      }
      T* to = static_cast<T*>(a.y) + n * size + at.first + col.c;
      const T* q = x;
#pragma unroll 4
      for (int r = 0; r < at.mine; ++r, q += at.step, to += at.step) {
        Pack<T, V> b;
        b.load(q);
#pragma unroll
        for (int v = 0; v < V; ++v) b.x[v] = activate<ACT>(fmaf(b.x[v] - mean[v], gain[v], col.bs[v]));
        b.store(to);
      }
    }
    samples.release(i);
  }
  samples.finish();
}

// Block = part blockIdx.x % parts of sample blockIdx.x / parts: its groups' sets; the sample's last
// block joins the parts' into (mean, rstd).
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_stats(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(128) unsigned char raw[];
  float2* smem = reinterpret_cast<float2*>(raw + (p.stage_rows ? kStreamBytes + 64 : 0));
  const long long n = blockIdx.x / p.parts;
  const int k = blockIdx.x % p.parts;
  float2* part = static_cast<float2*>(a.work) + n * p.parts * a.groups;
  {
    const SplitPlace at(a, p, k);
    SplitColumn<V> col;
    col.set(a, p, at, 0);
    if (p.stage_rows)
      stream_stats<T, V>(a, p, raw, smem, at, col, n, k, part + (long long)k * a.groups);
    else
      split_stats<T, V>(a, p, smem, at, col, n, part + (long long)k * a.groups);
  }
  unsigned* count = reinterpret_cast<unsigned*>(static_cast<char*>(a.work) + p.off_sync);
  if (!last_of_sample(count + n, p.parts)) return;
  float2* result = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.off_result) + n * a.groups;
  const int w = a.channels / a.groups, lanes = p.planes, lane = threadIdx.x & (lanes - 1);
  const float inv = 1.f / ((float)a.spots * (float)w), most = (float)p.part_rows * (float)w;
  const float last = (float)(a.spots - (long long)(p.parts - 1) * p.part_rows) * (float)w;
  for (int g0 = 0; g0 < a.groups; g0 += blockDim.x / lanes) {
    const int g = g0 + threadIdx.x / lanes;
    const Joined all = join_sets(g < a.groups ? __ldcg(part + g).x : 0.f, inv, lanes, [&](float origin, float& t, float& tt) {
      if (g >= a.groups) return;
#pragma unroll 8
      for (int i = lane; i < p.parts; i += lanes) {
        const float2 b = __ldcg(part + (long long)i * a.groups + g);
        const float d = b.x - origin, nd = d * (i == p.parts - 1 ? last : most);
        t += nd;
        tt += fmaf(nd, d, b.y);
      }
    });
    if (g < a.groups && lane == 0) {
      const float rstd = rstd_of(all.m2 * inv, a.eps);
      result[g] = make_float2(all.mean, rstd);
      if (a.mean) {
        a.mean[n * a.groups + g] = all.mean;
        a.rstd[n * a.groups + g] = rstd;
      }
    }
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3)
    k_gn_apply(const __grid_constant__ GroupNormArgs a, const __grid_constant__ GroupNormPlan p) {
  extern __shared__ __align__(128) unsigned char raw[];
  const unsigned b = gridDim.x - 1 - blockIdx.x;
  const long long n = b / p.parts;
  const int k = b % p.parts;
  const SplitPlace at(a, p, k);
  SplitColumn<V> col;
  col.set(a, p, at, 0);
  const float2* result = reinterpret_cast<const float2*>(static_cast<const char*>(a.work) + p.off_result) + n * a.groups;
  if (!p.stage_rows) {
    split_apply<T, V, ACT>(a, p, at, col, n, result);
    return;
  }
  const long long base = (n * a.spots + (long long)k * p.part_rows) * a.channels;
  const void* const src[1] = {static_cast<const T*>(a.x) + base};
  RowStream<1> rows(raw, p, at.rows, (long long)a.channels * sizeof(T), src);
  float mean[V], gain[V];
  if (col.live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 s = result[col.group(v)];
      mean[v] = s.x;
      gain[v] = s.y * col.wt[v];
    }
  }
  T* to = static_cast<T*>(a.y) + base + (long long)at.slot * a.channels + col.c;
  for (int i = 0; i < rows.count; ++i) {
    rows.wait(i);
    if (col.live) {
      const T* q = reinterpret_cast<const T*>(rows.buffer(i, 0)) + at.slot * a.channels + col.c;
      const int mine = rows.rows_of(i);
#pragma unroll 4
      for (int r = at.slot; r < mine; r += p.slots, q += at.step, to += at.step) {
        Pack<T, V> x;
        x.load(q);
#pragma unroll
        for (int v = 0; v < V; ++v) x.x[v] = activate<ACT>(fmaf(x.x[v] - mean[v], gain[v], col.bs[v]));
        x.store(to);
      }
    }
    rows.release(i);
  }
  rows.finish();
}

// ---------------------------------------------------------------- kAny
// More channels than the other forms' shared memory holds: three passes over
// a group by one block, with its sums in 64 bits (a thread may have any number
// of terms).
template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_gn_any(const __grid_constant__ GroupNormArgs a) {
  __shared__ double red[kNormThreads / 32];
  const int w = a.channels / a.groups;
  const double inv = 1.0 / ((double)a.spots * w);
  for (long long id = blockIdx.x; id < a.batch * a.groups; id += gridDim.x) {
    const int g = (int)(id % a.groups);
    const long long base = id / a.groups * a.spots * a.channels + (long long)g * w;
    double mean = 0.0;
    float rstd = 0.f;
    for (int pass = 0; pass < 3; ++pass) {
      double s = 0.0;
      for (AnyPlace at(w); at.row < a.spots; at.next()) {
        const long long i = base + at.row * a.channels + at.c;
        const double x = to_f32(static_cast<const T*>(a.x)[i]);
        if (pass == 0) s += x;
        if (pass == 1) s += (x - mean) * (x - mean);
        if (pass == 2) {
          const float wc = a.weight ? a.weight[g * w + at.c] : 1.f, bc = a.bias ? a.bias[g * w + at.c] : 0.f;
          static_cast<T*>(a.y)[i] = from_f32<T>(activate<ACT>(fmaf((float)(x - mean) * rstd, wc, bc)));
        }
      }
      if (pass == 2) break;
      s = block_sum(s, red) * inv;
      if (pass == 0) mean = s;
      else rstd = (float)(1.0 / sqrt(s + (double)a.eps));
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[id] = (float)mean;
      a.rstd[id] = rstd;
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
  cudaError_t e;
  if (p.sample_buffers) {
    const int smem = (int)(p.sample_buffers * a.spots * a.channels * sizeof(T)) + 8 * kMaxSampleBuffers + p.smem;
    e = allow_smem<k_gn_whole_stream<T, V, ACT>>(smem);
    if (e == cudaSuccess) k_gn_whole_stream<T, V, ACT><<<p.grid, p.threads, smem, st>>>(a, p);
    return e == cudaSuccess ? cudaGetLastError() : e;
  }
  if (p.parts == 1) {
    e = allow_smem<k_gn_whole<T, V, ACT>>(p.smem);
    if (e == cudaSuccess) k_gn_whole<T, V, ACT><<<p.grid, p.threads, p.smem, st>>>(a, p);
    return e == cudaSuccess ? cudaGetLastError() : e;
  }
  const int stream = p.stage_rows ? kStreamBytes + 64 : 0;
  e = allow_smem<k_gn_stats<T, V>>(p.smem + stream);
  if (e == cudaSuccess) e = allow_smem<k_gn_apply<T, V, ACT>>(stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(static_cast<char*>(a.work) + p.off_sync, 0, sizeof(unsigned) * a.batch, st);
  if (e != cudaSuccess) return e;
  k_gn_stats<T, V><<<p.grid, p.threads, p.smem + stream, st>>>(a, p);
  k_gn_apply<T, V, ACT><<<p.grid, p.threads, stream, st>>>(a, p);
  return cudaGetLastError();
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

// Threads that share a sum of n terms: 4 terms each or more, in at most a warp.
static int lanes_for(long long n) {
  int lanes = 1;
  while (lanes < 32 && lanes * 4 < n) lanes *= 2;
  return lanes;
}

using gn::small_blocks;
using gn::small_blocks_bwd;

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
    const long long most = std::max<long long>(least, (long long)kSms * (backward ? small_blocks_bwd(p.nv) : small_blocks(p.nv)));
    p.grid = (int)std::max(least, std::min(blocks, most));
    if (backward) {
      const long long slots = (long long)p.grid * per / a.groups * a.groups;
      p.channel_rows = std::min(slots, total) / a.groups * a.spots;
      p.bytes = p.channel_rows * a.channels * 8;
    }
    return p;
  }
  // 4 elements per access: with 8 of a 16-bit type the channels' parameters would not fit the registers
  p.vec = a.channels % 4 == 0 && align % (4 * size) == 0 ? 4 : (size == 2 && a.channels % 2 == 0 && align % 4 == 0 ? 2 : 1);
  const int columns = (a.channels + p.vec - 1) / p.vec;
  p.cols = std::min(columns, kNormThreads);
  p.tiles = (columns + p.cols - 1) / p.cols;
  p.slots = (int)std::min<long long>(kNormThreads / p.cols, a.spots);
  p.threads = std::max(64, (p.slots * p.cols + 31) / 32 * 32);
  // a block's sets (backward: and its channels' sums, of one sample and of all), the groups' results
  const long long smem = 8LL * ((long long)p.slots * a.channels + (backward ? 2LL * a.channels : 0) + a.groups);
  if (smem > kMaxSplitSmem) {
    p = {};
    p.kind = GroupNormPlan::kAny;
    p.vec = 1;
    p.grid = (int)std::min<long long>(total, 16LL * kSms);
    return p;
  }
  p.smem = (int)smem;
  p.kind = GroupNormPlan::kSplit;
  const long long most = 4LL * kSms * kNormThreads / p.threads;  // blocks that fill the GPU, and then some
  const long long bytes = a.spots * a.channels * size * (backward ? 2 : 1);
  // parts of 32 KB at least, as many as fill the GPU, and no more than one block joins in a few rounds
  // of loads (1 x 16384 x 1024 in 32 groups: 592 parts 57 us, 296 parts 42 us)
  long long parts = 1;
  if (bytes > (48 << 10) && !(a.batch >= 2 * kSms && bytes <= (128 << 10)))
    parts = std::max<long long>(1, std::min({(most + a.batch - 1) / a.batch, bytes / (32 << 10), (long long)a.spots,
                                             std::max<long long>(kSms, 8192 / a.groups)}));
  // a block of one part only: cut large samples of a large batch as well, for the sake of L2
  if (parts == 1 && bytes > (128 << 10)) parts = std::min<long long>(a.spots, (bytes + (128 << 10) - 1) / (128 << 10));
  p.part_rows = (int)((a.spots + parts - 1) / parts);
  p.parts = (int)((a.spots + p.part_rows - 1) / p.part_rows);
  // rows whose addresses and sizes are multiples of 16 bytes are streamed, whole rounds of slots at a time
  const long long row_bytes = (long long)a.channels * size;
  if (p.parts > 1 && p.tiles == 1 && row_bytes % 16 == 0 && align % 16 == 0)
    p.stage_rows = (int)(kStreamBytes / kStages / (backward ? 2 : 1) / (row_bytes * p.slots)) * p.slots;
  // samples of whole 16-byte pieces are streamed: some 64 KB of buffers per block, two blocks per SM or more
  if (p.parts == 1 && p.tiles == 1 && a.spots * row_bytes % 16 == 0 && align % 16 == 0 && bytes <= (48 << 10)) {
    p.sample_buffers = (int)std::min<long long>(gn::kMaxSampleBuffers, std::max<long long>(2, (64 << 10) / bytes));
    if ((long long)p.sample_buffers * bytes + p.smem > (112 << 10)) p.sample_buffers = 0;
  }
  p.glanes = lanes_for((long long)(backward ? 1 : p.slots) * w);
  p.planes = p.parts > 1 ? lanes_for(p.parts) : 1;
  const long long per_sm = p.sample_buffers ? std::min<long long>(768 / p.threads, (220 << 10) / (p.sample_buffers * bytes + p.smem + 1024 + 64)) : 0;
  p.grid = (int)(p.sample_buffers ? std::min(a.batch, kSms * per_sm) : p.parts == 1 ? std::min(a.batch, most) : a.batch * p.parts);
  const long long result = p.parts > 1 ? a.batch * a.groups * 8 : 0;
  p.off_result = (result * p.parts + 15) & ~15LL;
  p.off_channels = (p.off_result + result + 15) & ~15LL;
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
