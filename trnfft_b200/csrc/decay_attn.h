// Internal interface of the decayed linear attention kernels (decay_attn.cu,
// decay_step.cu) and their C-ABI layer (capi_layers.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace tfb {

// Allows kernel K `bytes` of dynamic shared memory on the current device; asked of the driver once per device.
template <auto K>
cudaError_t allow_shared(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ULL << dev, std::memory_order_relaxed);
  return e;
}

enum ElemType { kF32 = 0, kBF16 = 1, kF16 = 2 };

// One "role": the operator
//   o_t = a sum_{s<=t} g^{t-s} (q_t . k_s) v_s + r g^{t+1-back} q_t C
//   C'  = g^n C + c sum_s g^{n-1-s+back} k_s v_s^T
// over the n tokens of every sequence and every head, in time order
// (back = 0) or from the last token to the first (back = 1).  The forward
// pass is one role; the backward pass is three (see decay_attn.cu).
struct DecayRole {
  const void* q;
  const void* k;
  const void* v;
  void* o;                     // null: only the state is wanted
  long long qs[3], ks[3], vs[3], os[3];  // strides of batch, token, head (elements; innermost 1)
  int qdiv, kdiv, vdiv;        // head h reads head h / div
  int wk, wv;                  // widths: of q and k, of v and o
  int back;
  float a, r, c;
  int o_f32;                   // o is float32 whatever the element type
  const float* first;          // carried-in state or null; element (k, v) of (sequence, head) at
  long long first_sk, first_sv;  //   (seq*heads + head)*wk*wv + k*first_sk + v*first_sv
  float* last;                 // final state (wk x wv, row-major) or null
  float* seg;                  // states of the segments, (unit, head, wk, wv)
  int wide;                    // bits: q, k, v rows are multiples of 16 bytes from aligned addresses; o of element pairs
};

constexpr int kMaxRoles = 3;

struct DecayArgs {
  DecayRole role[kMaxRoles];
  int roles;
  int heads;
  const float* log_decay;
  // dense: nseq sequences of `tokens` rows, sequence = batch row.  packed
  // (cu != null): sequence i is rows [cu[i], cu[i+1]) of batch row 0.
  long long tokens;
  int nseq;
  const void* cu;
  int cu64;
  // work units: a unit is one segment (seg_len tokens, a multiple of the
  // chunk) of one sequence; dense: seq = unit / segs.  packed: found from cu;
  // `units` bounds their number, and unit index `units` zeroes the rows of o
  // that belong to no sequence.  split: sequences may have several segments,
  // whose states then take a pass of their own.
  int seg_len;
  int segs;
  int units;
  int split;
  int* flags;  // (role, unit, head): blocks that the tensor-core kernel leaves to the other one's walk with care, or null
};

constexpr int padded_width(int w) { return w <= 32 ? 32 : (w <= 64 ? 64 : 128); }

// Cuts the sequences into segments (seg_len, segs, units, split) by the sizes alone, and says how many
// bytes the segments' states take (roles that are there: the widths in `a`).
int64_t plan_decay_attention(ElemType t, DecayArgs& a);
// `work` holds the bytes that plan_decay_attention said.
cudaError_t launch_decay_attention(ElemType t, DecayArgs a, void* work, cudaStream_t st);
cudaError_t launch_decay_chunks_f32(const DecayArgs& a, cudaStream_t st);
cudaError_t launch_decay_chunks_bf16(const DecayArgs& a, cudaStream_t st);
cudaError_t launch_decay_chunks_f16(const DecayArgs& a, cudaStream_t st);
cudaError_t launch_decay_tc(const DecayArgs& a, cudaStream_t st);
// The blocks of a pass (chunk::Pass) that the tensor-core kernel has flagged, walked with care.
cudaError_t launch_decay_flagged_bf16(const DecayArgs& a, int pass, cudaStream_t st);
// The states carried into the segments, from the segments' own.
cudaError_t launch_decay_scan(const DecayArgs& a, cudaStream_t st);

// out[row][hk][w] = sum over g < group of in[row][hk*group + g][w], float32 in, element type out.
cudaError_t launch_sum_heads(ElemType t, const float* in, void* out, long long rows, int kv_heads, int group, int width,
                             cudaStream_t st);

struct DecayStepArgs {
  const void* q;
  const void* k;
  const void* v;
  long long qs[2], ks[2], vs[2];  // strides of batch, head
  void* o;                        // (batch, heads, dv) contiguous
  const float* state;
  float* next;
  long long state_s, next_s;      // batch strides; (head, dk, dv) contiguous
  const float* log_decay;
  int batch, heads, group, dk, dv;
  float scale;
};

cudaError_t launch_decay_step(ElemType t, const DecayStepArgs& a, cudaStream_t st);

}  // namespace tfb
