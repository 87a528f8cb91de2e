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
#include "elem.cuh"
#include "kernels.h"

namespace tfb {

__device__ __forceinline__ long long cu_at(const DecayArgs& a, int i) {
  long long x = a.cu64 ? static_cast<const long long*>(a.cu)[i] : (long long)static_cast<const int*>(a.cu)[i];
  return x < 0 ? 0 : (x > a.tokens ? a.tokens : x);  // no value of cu leads outside the tensors
}

// One block per (head, sequence, role): the recurrence token by token, one
// column of the state per thread in shared memory.  Right for every size; one
// read of the operands, bound by the latency of its steps.
template <typename T>
__global__ void __launch_bounds__(128) k_decay_simple(const __grid_constant__ DecayArgs a) {
  extern __shared__ float sm[];
  const DecayRole& r = a.role[blockIdx.z];
  const int h = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const T* q = static_cast<const T*>(r.q) + (long long)(h / r.qdiv) * r.qs[2];
  const T* k = static_cast<const T*>(r.k) + (long long)(h / r.kdiv) * r.ks[2];
  const T* v = static_cast<const T*>(r.v) + (long long)(h / r.vdiv) * r.vs[2];
  long long row0, n, obase = (long long)h * r.os[2];
  if (a.cu) {
    row0 = 0;
    n = 0;
    if (seq < a.nseq) {
      row0 = cu_at(a, seq);
      n = cu_at(a, seq + 1) - row0;
    } else if (r.o) {  // the rows of no sequence
      const long long head_rows = cu_at(a, 0), tail = cu_at(a, a.nseq);
      for (long long t = 0; t < a.tokens; ++t)
        if (t < head_rows || t >= tail)
          for (int j = tid; j < r.wv; j += blockDim.x) {
            const long long at = obase + t * r.os[1] + j;
            if (r.o_f32)
              static_cast<float*>(r.o)[at] = 0.f;
            else
              static_cast<T*>(r.o)[at] = from_f32<T>(0.f);
          }
      return;
    }
    if (n < 0) n = 0;
  } else {
    row0 = 0;
    n = a.tokens;
    q += seq * r.qs[0];
    k += seq * r.ks[0];
    v += seq * r.vs[0];
    obase += seq * r.os[0];
  }
  if (seq >= a.nseq) return;
  float* S = sm;                        // wk x wv
  float* sq = S + r.wk * r.wv;          // wk
  float* sk = sq + r.wk;                // wk
  const long long sbase = ((long long)seq * a.heads + h) * r.wk * r.wv;
  for (int i = 0; i < r.wk; ++i)
    for (int j = tid; j < r.wv; j += blockDim.x)
      S[i * r.wv + j] = r.first ? r.first[sbase + i * r.first_sk + j * r.first_sv] : 0.f;
  const double gd = exp((double)a.log_decay[h]);
  const float ghi = (float)gd, glo = (float)(gd - (double)ghi);
  for (long long i = 0; i < n; ++i) {
    const long long t = row0 + (r.back ? n - 1 - i : i);
    __syncthreads();
    for (int c = tid; c < r.wk; c += blockDim.x) {
      sq[c] = r.o ? to_f32(q[t * r.qs[1] + c]) : 0.f;
      sk[c] = to_f32(k[t * r.ks[1] + c]);
    }
    __syncthreads();
    for (int j = tid; j < r.wv; j += blockDim.x) {
      const float vj = to_f32(v[t * r.vs[1] + j]) * r.c;
      float acc = 0.f;
      for (int c = 0; c < r.wk; ++c) {
        float s = S[c * r.wv + j];
        if (!(r.back && i == 0)) s = fmaf(s, ghi, s * glo);
        s = fmaf(sk[c], vj, s);
        S[c * r.wv + j] = s;
        acc = fmaf(sq[c], s, acc);
      }
      if (r.o) {
        const long long at = obase + t * r.os[1] + j;
        acc *= r.r;
        if (r.o_f32)
          static_cast<float*>(r.o)[at] = acc;
        else
          static_cast<T*>(r.o)[at] = from_f32<T>(acc);
      }
    }
  }
  if (r.last)
    for (int i = 0; i < r.wk; ++i)
      for (int j = tid; j < r.wv; j += blockDim.x) {
        float s = S[i * r.wv + j];
        if (r.back && n > 0) s = fmaf(s, ghi, s * glo);
        r.last[sbase + i * r.wv + j] = s;
      }
}

template <typename T>
static cudaError_t run_simple(const DecayArgs& a, cudaStream_t st) {
  size_t smem = 0;
  for (int i = 0; i < a.roles; ++i) {
    const size_t b = sizeof(float) * ((size_t)a.role[i].wk * a.role[i].wv + 2 * a.role[i].wk);
    smem = b > smem ? b : smem;
  }
  cudaError_t e = cudaFuncSetAttribute(k_decay_simple<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  k_decay_simple<T><<<dim3(a.heads, a.nseq + (a.cu ? 1 : 0), a.roles), 128, smem, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_decay_attention(ElemType t, const DecayArgs& a, cudaStream_t st) {
  switch (t) {
    case kF32: return run_simple<float>(a, st);
    case kBF16: return run_simple<__nv_bfloat16>(a, st);
    default: return run_simple<__half>(a, st);
  }
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
