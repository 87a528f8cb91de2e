// C-ABI layer of the sequence and normalisation operators: argument checks,
// roles of the backward pass, dispatch.  See include/trnfft_b200.h.
#include <cuda_runtime.h>

#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/trnfft_b200.h"
#include "decay_attn.h"
#include "group_norm.h"
#include "kernels.h"

namespace tfb {
namespace {

int bad(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return record_failure(code, buf);
}

int cuda_bad(cudaError_t e, const char* what) {
  return bad(TRNFFT_CUDA_ERROR, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

// Makes `dev` current for the call; restores the caller's device only if it was another one.
struct OnDevice {
  int prev = -1;
  bool ok = false;
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) {
      prev = -1;
      return;
    }
    if (prev == dev) {
      prev = -1;
      ok = true;
    } else {
      ok = cudaSetDevice(dev) == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool misaligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
size_t elem_size(int t) { return t == TRNFFT_F32 ? 4 : 2; }

int check_shape(const char* fn, const trnfft_decay_shape* s) {
  if (!s) return bad(TRNFFT_INVALID_VALUE, "%s: null shape", fn);
  if (s->dtype < TRNFFT_F32 || s->dtype > TRNFFT_F16) return bad(TRNFFT_INVALID_VALUE, "%s: unknown dtype %d", fn, s->dtype);
  if (s->batch < 0 || s->tokens < 0 || s->num_seqs < 0) return bad(TRNFFT_INVALID_VALUE, "%s: negative size", fn);
  if (s->heads < 1 || s->kv_heads < 1 || s->heads % s->kv_heads)
    return bad(TRNFFT_INVALID_VALUE, "%s: %lld heads are not a multiple of %lld key/value heads", fn, (long long)s->heads,
               (long long)s->kv_heads);
  if (s->key_width < 1 || s->value_width < 1) return bad(TRNFFT_INVALID_VALUE, "%s: head widths must be positive", fn);
  if (s->key_width > 128 || s->value_width > 128)
    return bad(TRNFFT_UNSUPPORTED, "%s: head widths %lld and %lld (up to 128)", fn, (long long)s->key_width,
               (long long)s->value_width);
  if (s->cu_seqlens && s->batch != 1) return bad(TRNFFT_INVALID_VALUE, "%s: packed sequences need batch 1", fn);
  if (s->cu_seqlens && misaligned(s->cu_seqlens, s->cu_is64 ? 8 : 4))
    return bad(TRNFFT_INVALID_VALUE, "%s: misaligned cu_seqlens", fn);
  const int64_t n = s->cu_seqlens ? s->num_seqs : s->batch;
  if (s->heads > 65535 || n >= (1 << 30) / s->heads || s->tokens > INT_MAX / 2)
    return bad(TRNFFT_UNSUPPORTED, "%s: more than 65535 heads, 2^30 states or 2^30 tokens", fn);
  return TRNFFT_SUCCESS;
}

DecayArgs base_args(const trnfft_decay_shape* s, const float* log_decay) {
  DecayArgs a;
  std::memset(&a, 0, sizeof a);
  a.heads = (int)s->heads;
  a.log_decay = log_decay;
  a.tokens = s->tokens;
  a.nseq = (int)(s->cu_seqlens ? s->num_seqs : s->batch);
  a.cu = s->cu_seqlens;
  a.cu64 = s->cu_is64;
  return a;
}

struct Operand {
  const void* p;
  const int64_t* stride;
  int div;
};

// The role (q, k, v) -> o with contiguous (batch, tokens, heads, wv) output.
DecayRole make_role(const DecayArgs& a, Operand q, Operand k, Operand v, void* o, int wk, int wv, bool o_f32) {
  DecayRole r;
  std::memset(&r, 0, sizeof r);
  r.q = q.p;
  r.k = k.p;
  r.v = v.p;
  r.o = o;
  for (int i = 0; i < 3; ++i) {
    r.qs[i] = q.stride[i];
    r.ks[i] = k.stride[i];
    r.vs[i] = v.stride[i];
  }
  r.qdiv = q.div;
  r.kdiv = k.div;
  r.vdiv = v.div;
  r.os[2] = wv;
  r.os[1] = (long long)a.heads * wv;
  r.os[0] = a.tokens * r.os[1];
  r.wk = wk;
  r.wv = wv;
  r.o_f32 = o_f32;
  r.a = r.r = r.c = 1.f;
  r.first_sk = wv;
  r.first_sv = 1;
  return r;
}

int check_operands(const char* fn, const trnfft_decay_shape* s, std::initializer_list<const void*> elems,
                   std::initializer_list<const void*> floats) {
  for (const void* p : elems)
    if (p && misaligned(p, elem_size(s->dtype))) return bad(TRNFFT_INVALID_VALUE, "%s: misaligned pointer", fn);
  for (const void* p : floats)
    if (p && misaligned(p, 4)) return bad(TRNFFT_INVALID_VALUE, "%s: misaligned float pointer", fn);
  return TRNFFT_SUCCESS;
}

// float32 gradients of the query heads' own keys and values, before the heads of a group are summed
int64_t head_grad_bytes(const trnfft_decay_shape* s) {
  if (s->heads == s->kv_heads) return 0;
  return (4 * s->batch * s->tokens * s->heads * (s->key_width + s->value_width) + 15) & ~(int64_t)15;
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" {

int64_t trnfft_decay_attention_work_bytes(const trnfft_decay_shape* s, int backward) {
  if (check_shape("decay_attention_work_bytes", s)) return -1;
  DecayArgs a = base_args(s, nullptr);
  const int wk = (int)s->key_width, wv = (int)s->value_width;
  if (!backward) {
    a.roles = 1;
    a.role[0].wk = wk;
    a.role[0].wv = wv;
    return plan_decay_attention((ElemType)s->dtype, a);
  }
  // whichever of the gradients are asked for
  int64_t most = 0;
  for (a.roles = 1; a.roles <= kMaxRoles; ++a.roles) {
    for (int i = 0; i < a.roles; ++i) {
      a.role[i].wk = wk;
      a.role[i].wv = wv;
    }
    const int64_t bytes = plan_decay_attention((ElemType)s->dtype, a);
    most = bytes > most ? bytes : most;
  }
  return head_grad_bytes(s) + most;
}

int trnfft_decay_attention(const trnfft_decay_shape* s, const void* q, const void* k, const void* v, const float* log_decay,
                           const float* initial, void* o, float* final_state, void* work, int device, void* stream) {
  const char* fn = "decay_attention";
  int rc = check_shape(fn, s);
  if (rc) return rc;
  DecayArgs a = base_args(s, log_decay);
  const bool rows = s->batch > 0 && s->tokens > 0;
  if (!rows && (a.nseq == 0 || !final_state)) return TRNFFT_SUCCESS;
  if (!log_decay || (rows && (!q || !k || !v || !o))) return bad(TRNFFT_INVALID_VALUE, "%s: null pointer", fn);
  rc = check_operands(fn, s, {q, k, v, o}, {log_decay, initial, final_state});
  if (rc) return rc;
  const int g = (int)(s->heads / s->kv_heads);
  a.roles = 1;
  a.role[0] = make_role(a, {q, s->q_stride, 1}, {k, s->k_stride, g}, {v, s->v_stride, g}, o, (int)s->key_width,
                        (int)s->value_width, false);
  a.role[0].a = a.role[0].r = s->scale;
  a.role[0].first = initial;
  a.role[0].last = final_state;
  if (!work && trnfft_decay_attention_work_bytes(s, 0)) return bad(TRNFFT_INVALID_VALUE, "%s: null work area", fn);
  if (work && misaligned(work, 16)) return bad(TRNFFT_INVALID_VALUE, "%s: misaligned work area", fn);
  OnDevice d(device);
  if (!d.ok) return bad(TRNFFT_CUDA_ERROR, "%s: cannot select device %d", fn, device);
  cudaError_t e = launch_decay_attention((ElemType)s->dtype, a, work, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TRNFFT_SUCCESS : cuda_bad(e, fn);
}

int trnfft_decay_attention_backward(const trnfft_decay_shape* s, const void* q, const void* k, const void* v,
                                    const float* log_decay, const float* initial, const void* d_o, const float* d_final,
                                    void* dq, void* dk, void* dv, float* d_initial, void* work, int device,
                                    void* stream) {
  const char* fn = "decay_attention_backward";
  int rc = check_shape(fn, s);
  if (rc) return rc;
  DecayArgs a = base_args(s, log_decay);
  const bool rows = s->batch > 0 && s->tokens > 0;
  if (!rows && (a.nseq == 0 || !d_initial)) return TRNFFT_SUCCESS;
  if (!log_decay || (rows && (!q || !k || !v || !d_o)))
    return bad(TRNFFT_INVALID_VALUE, "%s: null pointer", fn);
  if (!work && trnfft_decay_attention_work_bytes(s, 1)) return bad(TRNFFT_INVALID_VALUE, "%s: null work area", fn);
  rc = check_operands(fn, s, {q, k, v, d_o, dq, dk, dv}, {log_decay, initial, d_final, d_initial});
  if (rc) return rc;
  if (work && misaligned(work, 16)) return bad(TRNFFT_INVALID_VALUE, "%s: misaligned work area", fn);
  const int g = (int)(s->heads / s->kv_heads), wk = (int)s->key_width, wv = (int)s->value_width;
  const Operand Q{q, s->q_stride, 1}, K{k, s->k_stride, g}, V{v, s->v_stride, g}, dO{d_o, s->o_stride, 1};
  const bool grouped = g > 1;
  float* dv_heads = static_cast<float*>(work);
  float* dk_heads = grouped ? dv_heads + s->batch * s->tokens * s->heads * wv : nullptr;
  if (dq) {  // dq = F(dO, v, k), its state S^T
    DecayRole& r = a.role[a.roles++];
    r = make_role(a, dO, V, K, dq, wv, wk, false);
    r.a = r.r = s->scale;
    r.first = initial;
    r.first_sk = 1;
    r.first_sv = wv;
  }
  if (dv || d_initial) {  // dv = F_back(k, q, dO), its state the gradient of S
    DecayRole& r = a.role[a.roles++];
    r = make_role(a, K, Q, dO, dv ? (grouped ? dv_heads : dv) : nullptr, wk, wv, grouped);
    r.back = 1;
    r.a = r.c = s->scale;
    r.first = d_final;
    r.last = d_initial;
  }
  if (dk) {  // dk = F_back(v, dO, q), its state the gradient of S^T
    DecayRole& r = a.role[a.roles++];
    r = make_role(a, V, dO, Q, grouped ? dk_heads : dk, wv, wk, grouped);
    r.back = 1;
    r.a = r.c = s->scale;
    r.first = d_final;
    r.first_sk = 1;
    r.first_sv = wv;
  }
  if (a.roles == 0) return TRNFFT_SUCCESS;
  OnDevice d(device);
  if (!d.ok) return bad(TRNFFT_CUDA_ERROR, "%s: cannot select device %d", fn, device);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = launch_decay_attention((ElemType)s->dtype, a, static_cast<char*>(work) + head_grad_bytes(s), st);
  if (e == cudaSuccess && grouped && rows) {
    const long long n = s->batch * s->tokens;
    if (dv) e = launch_sum_heads((ElemType)s->dtype, dv_heads, dv, n, (int)s->kv_heads, g, wv, st);
    if (e == cudaSuccess && dk) e = launch_sum_heads((ElemType)s->dtype, dk_heads, dk, n, (int)s->kv_heads, g, wk, st);
  }
  return e == cudaSuccess ? TRNFFT_SUCCESS : cuda_bad(e, fn);
}

int trnfft_decay_attention_step(const trnfft_decay_step_shape* s, const void* q, const void* k, const void* v,
                                const float* log_decay, const float* state, float* new_state, void* o, int device,
                                void* stream) {
  const char* fn = "decay_attention_step";
  if (!s) return bad(TRNFFT_INVALID_VALUE, "%s: null shape", fn);
  if (s->dtype < TRNFFT_F32 || s->dtype > TRNFFT_F16) return bad(TRNFFT_INVALID_VALUE, "%s: unknown dtype %d", fn, s->dtype);
  if (s->batch < 0 || s->heads < 1 || s->kv_heads < 1 || s->heads % s->kv_heads || s->key_width < 1 || s->value_width < 1)
    return bad(TRNFFT_INVALID_VALUE, "%s: bad sizes", fn);
  if (s->key_width > 128 || s->value_width > 128)
    return bad(TRNFFT_UNSUPPORTED, "%s: head widths %lld and %lld (up to 128)", fn, (long long)s->key_width,
               (long long)s->value_width);
  if (s->heads > 65535 || s->batch > INT_MAX / 2 / s->heads)
    return bad(TRNFFT_UNSUPPORTED, "%s: more than 65535 heads or 2^30 states", fn);
  if (s->batch == 0) return TRNFFT_SUCCESS;
  if (!q || !k || !v || !log_decay || !state || !new_state || !o) return bad(TRNFFT_INVALID_VALUE, "%s: null pointer", fn);
  const int64_t one = s->heads * s->key_width * s->value_width;
  if (s->state_stride < one || s->new_state_stride < one)
    return bad(TRNFFT_INVALID_VALUE, "%s: the states of two streams overlap", fn);
  if (misaligned(state, 4) || misaligned(new_state, 4) || misaligned(log_decay, 4))
    return bad(TRNFFT_INVALID_VALUE, "%s: misaligned float pointer", fn);
  const char* a0 = reinterpret_cast<const char*>(state);
  const char* b0 = reinterpret_cast<const char*>(new_state);
  const int64_t an = 4 * ((s->batch - 1) * s->state_stride + one), bn = 4 * ((s->batch - 1) * s->new_state_stride + one);
  bool apart = a0 >= b0 + bn || b0 >= a0 + an;
  if (s->state_stride == s->new_state_stride) {  // each new state between two old ones, or in the place of one's own
    const int64_t step = 4 * s->state_stride, off = ((b0 - a0) % step + step) % step;
    apart = apart || a0 == b0 || (off >= 4 * one && off <= step - 4 * one);
  }
  if (!apart)
    return bad(TRNFFT_INVALID_VALUE, "%s: the new state overlaps the old one without being it", fn);
  DecayStepArgs a;
  std::memset(&a, 0, sizeof a);
  a.q = q;
  a.k = k;
  a.v = v;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = s->q_stride[i];
    a.ks[i] = s->k_stride[i];
    a.vs[i] = s->v_stride[i];
  }
  a.o = o;
  a.state = state;
  a.next = new_state;
  a.state_s = s->state_stride;
  a.next_s = s->new_state_stride;
  a.log_decay = log_decay;
  a.batch = (int)s->batch;
  a.heads = (int)s->heads;
  a.group = (int)(s->heads / s->kv_heads);
  a.dk = (int)s->key_width;
  a.dv = (int)s->value_width;
  a.scale = s->scale;
  OnDevice d(device);
  if (!d.ok) return bad(TRNFFT_CUDA_ERROR, "%s: cannot select device %d", fn, device);
  cudaError_t e = launch_decay_step((ElemType)s->dtype, a, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TRNFFT_SUCCESS : cuda_bad(e, fn);
}

static int norm_args(const char* fn, GroupNormArgs& a, int64_t batch, int64_t spots, int64_t channels, int64_t groups,
                     int activation, int dtype) {
  if (dtype < TRNFFT_F32 || dtype > TRNFFT_F16) return bad(TRNFFT_INVALID_VALUE, "%s: unknown dtype %d", fn, dtype);
  if (activation < TRNFFT_ACT_NONE || activation > TRNFFT_ACT_GELU)
    return bad(TRNFFT_INVALID_VALUE, "%s: unknown activation %d", fn, activation);
  if (batch < 0 || spots < 0 || channels < 1 || groups < 1 || channels % groups)
    return bad(TRNFFT_INVALID_VALUE, "%s: bad sizes (%lld channels in %lld groups)", fn, (long long)channels,
               (long long)groups);
  if (channels > (1 << 24) || batch > INT_MAX / groups || spots > INT_MAX)
    return bad(TRNFFT_UNSUPPORTED, "%s: more than 2^24 channels, 2^31 groups or 2^31 spots", fn);
  std::memset(&a, 0, sizeof a);
  a.batch = batch;
  a.spots = spots;
  a.channels = (int)channels;
  a.groups = (int)groups;
  a.act = activation;
  return TRNFFT_SUCCESS;
}

int64_t trnfft_group_norm_work_bytes(int64_t batch, int64_t spots, int64_t channels, int64_t groups, int dtype,
                                     int backward) {
  GroupNormArgs a;
  if (norm_args("group_norm_work_bytes", a, batch, spots, channels, groups, 0, dtype)) return -1;
  return group_norm_work_bytes((ElemType)dtype, a, backward != 0);
}

int trnfft_group_norm(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                      int64_t batch, int64_t spots, int64_t channels, int64_t groups, float eps, int activation, int dtype,
                      void* work, int device, void* stream) {
  const char* fn = "group_norm";
  GroupNormArgs a;
  int rc = norm_args(fn, a, batch, spots, channels, groups, activation, dtype);
  if (rc) return rc;
  if (batch == 0 || spots == 0) return TRNFFT_SUCCESS;
  if (!x || !y || (!mean) != (!rstd)) return bad(TRNFFT_INVALID_VALUE, "%s: null pointer", fn);
  if (misaligned(x, elem_size(dtype)) || misaligned(y, elem_size(dtype)) || misaligned(weight, 4) || misaligned(bias, 4) ||
      misaligned(mean, 4) || misaligned(rstd, 4))
    return bad(TRNFFT_INVALID_VALUE, "%s: misaligned pointer", fn);
  if (!work && group_norm_work_bytes((ElemType)dtype, a, false))
    return bad(TRNFFT_INVALID_VALUE, "%s: null work area", fn);
  if (misaligned(work, 16)) return bad(TRNFFT_INVALID_VALUE, "%s: misaligned work area", fn);
  a.x = x;
  a.y = y;
  a.weight = weight;
  a.bias = bias;
  a.mean = mean;
  a.rstd = rstd;
  a.eps = eps;
  a.work = static_cast<float*>(work);
  OnDevice d(device);
  if (!d.ok) return bad(TRNFFT_CUDA_ERROR, "%s: cannot select device %d", fn, device);
  cudaError_t e = launch_group_norm((ElemType)dtype, a, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TRNFFT_SUCCESS : cuda_bad(e, fn);
}

int trnfft_group_norm_backward(const void* x, const void* dy, const float* weight, const float* bias, const float* mean,
                               const float* rstd, void* dx, float* dw, float* db, int64_t batch, int64_t spots,
                               int64_t channels, int64_t groups, int activation, int dtype, void* work, int device,
                               void* stream) {
  const char* fn = "group_norm_backward";
  GroupNormArgs a;
  int rc = norm_args(fn, a, batch, spots, channels, groups, activation, dtype);
  if (rc) return rc;
  if (misaligned(work, 16)) return bad(TRNFFT_INVALID_VALUE, "%s: misaligned work area", fn);
  OnDevice d(device);
  if (!d.ok) return bad(TRNFFT_CUDA_ERROR, "%s: cannot select device %d", fn, device);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (batch == 0 || spots == 0) {  // sums of nothing
    if (dw) e = cudaMemsetAsync(dw, 0, 4 * channels, st);
    if (e == cudaSuccess && db) e = cudaMemsetAsync(db, 0, 4 * channels, st);
    return e == cudaSuccess ? TRNFFT_SUCCESS : cuda_bad(e, fn);
  }
  if (!x || !dy || !mean || !rstd) return bad(TRNFFT_INVALID_VALUE, "%s: null pointer", fn);
  if (misaligned(x, elem_size(dtype)) || misaligned(dy, elem_size(dtype)) || misaligned(dx, elem_size(dtype)) ||
      misaligned(weight, 4) || misaligned(bias, 4) || misaligned(mean, 4) || misaligned(rstd, 4) || misaligned(dw, 4) ||
      misaligned(db, 4))
    return bad(TRNFFT_INVALID_VALUE, "%s: misaligned pointer", fn);
  if (!work && group_norm_work_bytes((ElemType)dtype, a, true)) return bad(TRNFFT_INVALID_VALUE, "%s: null work area", fn);
  a.x = x;
  a.dy = dy;
  a.y = dx;
  a.weight = weight;
  a.bias = bias;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dw = dw;
  a.db = db;
  a.work = static_cast<float*>(work);
  e = launch_group_norm_backward((ElemType)dtype, a, st);
  return e == cudaSuccess ? TRNFFT_SUCCESS : cuda_bad(e, fn);
}

}  // extern "C"
