// Linear attention with a decay for each head, over whole sequences.
//
//   S_t = g S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   g = exp(log_decay[head])
//
// Backward: with dO the gradient of o, G_t the gradient of S_t,
//   dq_t = scale sum_{s<=t} g^{t-s} (dO_t . v_s) k_s          (+ the initial state's part)
//   dv_s = scale sum_{t>=s} g^{t-s} (k_s . q_t) dO_t          (+ the final state's)
//   dk_s = scale sum_{t>=s} g^{t-s} (v_s . dO_t) q_t          (+ the final state's)
// so every gradient is the operator itself with the operands exchanged, two
// of them with time reversed (DecayRole); the state of dv's role ends as the
// gradient of the initial state.
#include "decay_attn.h"
#include "decay_chunk.cuh"
#include "elem.cuh"
#include "kernels.h"

#include <algorithm>

using std::max;

namespace tfb {

namespace {

// Tokens of a chunk: of the tensor-core kernel for bfloat16 (a multiple of the other kernel's), of the other one.
constexpr int chunk_of(ElemType t) { return t == kBF16 ? 128 : 64; }
constexpr int kSms = 148;

// Bits of DecayRole::wide.
int wide_bits(const DecayRole& r, int size) {
  auto rows = [&](const void* p, const long long* s, int w) {
    return (reinterpret_cast<uintptr_t>(p) | s[0] * size | s[1] * size | s[2] * size | (long long)w * size) % 16 == 0;
  };
  const int osize = r.o_f32 ? 4 : size;
  const bool o = (reinterpret_cast<uintptr_t>(r.o) | (long long)r.os[0] * osize | r.os[1] * osize | r.os[2] * osize |
                  (long long)r.wv * osize) % (2 * osize) == 0;
  return (rows(r.q, r.qs, r.wk) ? 1 : 0) | (rows(r.k, r.ks, r.wk) ? 2 : 0) | (rows(r.v, r.vs, r.wv) ? 4 : 0) | (o ? 8 : 0);
}

int64_t flag_bytes(const DecayArgs& a) { return (4LL * a.roles * a.units * a.heads + 15) & ~15LL; }

// Whether the roles' operands are as the tensor-core kernel loads and stores them: 16 bytes at a time.
bool tc_ok(const DecayArgs& a) {
  for (int i = 0; i < a.roles; ++i) {
    const DecayRole& r = a.role[i];
    if ((r.wide & 7) != 7 || r.wv % 8 || reinterpret_cast<uintptr_t>(r.o) % 16) return false;
  }
  return true;
}

}  // namespace

// A sequence is walked chunk by chunk, so with few (sequence, head, role) the GPU is filled by cutting
// sequences into segments, at the cost of a pass that takes the segments' own states (it reads k and v
// once more and does about 0.6 of a chunk's work), of the states' way through memory and each block's
// start (about 3 chunks' time for each wave of blocks) and of a scan (about 2).  The segment length, in
// chunks, is the one of least time by that count.
int64_t plan_decay_attention(ElemType t, DecayArgs& a) {
  const int chunk = chunk_of(t);
  const long long total = (a.tokens + chunk - 1) / chunk;  // chunks, of one dense or of all packed sequences
  int wide = 0;
  for (int i = 0; i < a.roles; ++i) wide = max(wide, max(a.role[i].wk, a.role[i].wv));
  const long long slots = (long long)kSms * (wide <= 64 && t != kBF16 ? 2 : 1),  // blocks at a time
                  walks = (long long)a.heads * max(a.roles, 1);
  // packed: how the rows fall on the sequences is on the device; take the longest for four times the mean
  const long long longest = a.cu ? (a.nseq ? std::min(total, 4 * total / a.nseq + 1) : 0) : total;
  auto units = [&](long long s) { return a.cu ? total / s + a.nseq : a.nseq * ((total + s - 1) / s); };
  auto waves = [&](long long n) { return (double)((n * walks + slots - 1) / slots); };
  long long best = std::max<long long>(total, 1);
  double least = std::max((double)longest, waves(a.nseq) * (a.cu ? (double)total / std::max(1, a.nseq) : (double)total));
  for (long long s = 1; s < total; s *= 2) {
    const double x = waves(units(s)) * (std::min(s, longest) * 1.6 + 3.0) + 2.0;
    if (x < 0.95 * least && units(s) * a.heads < (1LL << 30)) {
      least = x;
      best = s;
    }
  }
  a.split = best < total;
  a.seg_len = (int)(best * chunk);
  a.segs = a.cu ? 1 : (int)std::max<long long>(1, (total + best - 1) / best);
  a.units = (int)(a.split ? units(best) : a.nseq);
  int64_t bytes = t == kBF16 ? flag_bytes(a) : 0;
  if (!a.split) return bytes;
  for (int i = 0; i < a.roles; ++i) bytes += (4LL * a.units * a.heads * a.role[i].wk * a.role[i].wv + 15) & ~15LL;
  return bytes;
}

cudaError_t launch_decay_attention(ElemType t, DecayArgs a, void* work, cudaStream_t st) {
  plan_decay_attention(t, a);
  char* p = static_cast<char*>(work);
  for (int i = 0; i < a.roles; ++i) {
    DecayRole& r = a.role[i];
    r.wide = wide_bits(r, t == kF32 ? 4 : 2);
    if (a.split) {
      r.seg = reinterpret_cast<float*>(p);
      p += (4LL * a.units * a.heads * r.wk * r.wv + 15) & ~15LL;
    }
  }
  switch (t) {
    case kF32: return launch_decay_chunks_f32(a, st);
    case kBF16:
      if (!tc_ok(a)) return launch_decay_chunks_bf16(a, st);
      a.flags = reinterpret_cast<int*>(p);
      return launch_decay_tc(a, st);
    default: return launch_decay_chunks_f16(a, st);
  }
}

// The states carried into the segments of one (sequence, head, role), in place of the segments' own
// final states, and the sequence's final state.
__global__ void __launch_bounds__(256) k_decay_scan(const __grid_constant__ DecayArgs a) {
  const DecayRole& R = a.role[blockIdx.z];
  const int h = blockIdx.x % a.heads, seq = blockIdx.x / a.heads;
  __shared__ int first_unit;
  __shared__ long long shared_total;
  if (threadIdx.x < 32) {
    long long n = a.tokens;
    int before = seq * a.segs;
    if (a.cu) {
      before = 0;
      for (int i = threadIdx.x; i < seq; i += 32) {
        const long long m = chunk::cu_value(a, i + 1) - chunk::cu_value(a, i);
        before += max(1, (int)(((m < 0 ? 0 : m) + a.seg_len - 1) / a.seg_len));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(~0u, before, o);
      n = chunk::cu_value(a, seq + 1) - chunk::cu_value(a, seq);
      if (n < 0) n = 0;
    }
    if (threadIdx.x == 0) {
      first_unit = before;
      shared_total = n;
    }
  }
  __syncthreads();
  const long long total = shared_total, size = (long long)R.wk * R.wv;
  const int e = blockIdx.y * 256 + threadIdx.x;
  const int segs = max(1, (int)((total + a.seg_len - 1) / a.seg_len));
  // (units: what the work area holds; only lengths that are not ascending lead past it)
  if (e >= size || first_unit + segs > a.units) return;
  const double ld = a.log_decay[h];
  const DecayFactor f(exp(ld * a.seg_len), a.log_decay[h]);
  float s = 0.f;
  const long long sbase = ((long long)seq * a.heads + h) * size;
  if (R.first) s = R.first[sbase + e / R.wv * R.first_sk + e % R.wv * R.first_sv];
  float* p = R.seg + ((long long)first_unit * a.heads + h) * size + e;
  const long long step = a.heads * size;
  int i = 0;
  for (; i + 4 < segs; i += 4, p += 4 * step) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = p[u * step];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      p[u * step] = s;
      s = f.step(s, x[u]);
    }
  }
  for (; i < segs; ++i, p += step) {
    const bool end = i == segs - 1;
    const float x = end && !R.last ? 0.f : *p;
    *p = s;
    if (!end) {
      s = f.step(s, x);
    } else if (R.last) {
      const long long n = total - (long long)i * a.seg_len;
      R.last[sbase + e] = DecayFactor(n ? exp(ld * n) : 1.0, a.log_decay[h]).step(s, x);
    }
  }
}

cudaError_t launch_decay_scan(const DecayArgs& a, cudaStream_t st) {
  int size = 0;
  for (int i = 0; i < a.roles; ++i) size = max(size, a.role[i].wk * a.role[i].wv);
  k_decay_scan<<<dim3((unsigned)a.nseq * a.heads, (size + 255) / 256, a.roles), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(256) k_sum_heads(const float* __restrict__ in, T* __restrict__ out, long long count,
                                                   int group, int width) {
  const long long stride = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += stride) {
    const float* p = in + (i / width) * group * width + i % width;
    float s = 0.f;
    for (int g = 0; g < group; ++g) s += p[(long long)g * width];
    out[i] = from_f32<T>(s);
  }
}

cudaError_t launch_sum_heads(ElemType t, const float* in, void* out, long long rows, int kv_heads, int group, int width,
                             cudaStream_t st) {
  const long long count = rows * kv_heads * width;
  if (count == 0) return cudaSuccess;
  long long blocks = (count + 255) / 256;
  if (blocks > 148 * 16) blocks = 148 * 16;
  switch (t) {
    case kF32: k_sum_heads<<<(unsigned)blocks, 256, 0, st>>>(in, static_cast<float*>(out), count, group, width); break;
    case kBF16:
      k_sum_heads<<<(unsigned)blocks, 256, 0, st>>>(in, static_cast<__nv_bfloat16*>(out), count, group, width);
      break;
    default: k_sum_heads<<<(unsigned)blocks, 256, 0, st>>>(in, static_cast<__half*>(out), count, group, width);
  }
  return cudaGetLastError();
}

}  // namespace tfb
