// Decayed linear attention in chunks of 64 tokens, on the warp-level tensor
// core instructions: every type, head widths up to 128 and any decay.
//
// With C the state carried into a chunk of n tokens, row i of it:
//   P_ij = a g^{i-j} (q_i . k_j)  for j <= i, else 0
//   o    = P v + r g^{i+1-back} (q C)
//   C'   = g^n C + sum_j (c g^{n-1-j+back} k_j) v_j^T
// One block of 8 warps walks the chunks of one (segment, head, role).  A warp
// owns 16 rows of P, which stay in its registers as the A operand of P v, and
// a block of C, which stays in its registers in float32; C goes to shared
// memory once per chunk as the B operand of q C.
//
// Precision.  float32 operands are split in two TF32 parts each and multiplied
// as hi hi + hi lo + lo hi (2^-22).  16-bit operands are exact in TF32 (and
// q . k runs on their own type); P, C and the scaled k are multiplied in two
// parts (P and C: the parts cut off, 2^-20; one part, rounded, would lose
// 2^-11, as much as the rounding of a float16 o).  The tensor core
// truncates as it accumulates, so C never is an accumulator over chunks: a
// chunk's sum starts from 0 and is added to the scaled C in round-to-nearest,
// with g^n as the sum of two float32 (decay_state.cuh).
//
// Bound by instruction issue and the tensor pipe together (55 and 46 % of
// their cycles with two blocks of 8 warps per SM, 64 x 64 float16): 112501
// tokens of 8 such heads take 531 us in segments (501 us with one part of P and
// C), a packed float32 call of 2517 rows 72-77 us.
#pragma once

#include <type_traits>

#include "decay_attn.h"
#include "decay_state.cuh"
#include "elem.cuh"
#include "tma.cuh"

namespace tfb {
namespace chunk {

constexpr int kC = 64;
constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// The same in two integer instructions, for finite x: NaN may become 0.
__device__ __forceinline__ uint32_t tf32_finite(float x) { return (__float_as_uint(x) + 0x1000u) & 0xffffe000u; }

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A TF32 operand in PARTS parts: hi, and what is left of it.
template <int N, int PARTS>
struct Frag {
  uint32_t p[PARTS][N];
  // (Both parts are rounded: a first part that is merely cut off leaves a second one of the same sign
  // always, and the products of second parts, which are left out, would add up to 1e-6.  Of NaN the
  // first part may be 0, and the second is NaN.)
  __device__ __forceinline__ void set(int i, float x) {
    if constexpr (PARTS > 1) {
      p[0][i] = tf32_finite(x);
      p[1][i] = tf32(x - __uint_as_float(p[0][i]));
    } else {
      p[0][i] = tf32(x);
    }
  }
  // Both parts cut off, in three instructions: for products with a factor that is exact, where no
  // product of two second parts is left out.
  __device__ __forceinline__ void cut(int i, float x) {
    static_assert(PARTS == 2, "two parts");
    p[0][i] = __float_as_uint(x) & 0xffffe000u;
    p[1][i] = __float_as_uint(x - __uint_as_float(p[0][i])) & 0xffffe000u;
  }
  // a value that TF32 holds exactly
  __device__ __forceinline__ void exact(int i, float x) {
    static_assert(PARTS == 1, "one part");
    p[0][i] = __float_as_uint(x);
  }
};
template <int PA, int PB>
__device__ __forceinline__ void mma_parts(float (&d)[4], const Frag<4, PA>& a, const Frag<2, PB>& b) {
  if constexpr (PB > 1) mma_tf32(d, a.p[0], b.p[1][0], b.p[1][1]);
  if constexpr (PA > 1) mma_tf32(d, a.p[1], b.p[0][0], b.p[0][1]);
  mma_tf32(d, a.p[0], b.p[0][0], b.p[0][1]);
}

// The same with the products of a second part in a sum of their own, so that the first parts' sum is
// truncated once, not three times, for each 8 terms (o of 64 x 64 heads: 1.3e-6 -> 6e-7 off; the packed
// call above: 66 -> 71 us).
__device__ __forceinline__ void mma_apart(float (&d)[4], float (&rest)[4], const Frag<4, 2>& a, const Frag<2, 2>& b) {
  mma_tf32(rest, a.p[0], b.p[1][0], b.p[1][1]);
  mma_tf32(rest, a.p[1], b.p[0][0], b.p[0][1]);
  mma_tf32(d, a.p[0], b.p[0][0], b.p[0][1]);
}

// N (1, 2 or 4) blocks of 8 x 8 16-bit elements from shared memory, block i's row r at the address that
// lane 8 i + r gives: a thread gets elements (row lane/4, columns 2 (lane%4) and the next), or, with
// kTrans, (rows 2 (lane%4) and the next, column lane/4).
template <int N, bool kTrans>
__device__ __forceinline__ void load_blocks(uint32_t (&r)[N], const void* at) {
  const uint32_t p = smem_u32(at);
  if constexpr (N == 4 && kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
  else if constexpr (N == 4)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
  else if constexpr (N == 2)
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(p) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x1.trans.shared.b16 {%0}, [%1];" : "=r"(r[0]) : "r"(p) : "memory");
}
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t x) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// d[j] += A B_j for TILES neighbouring blocks of 8 columns, B the 8 rows of v from `rows` on, of which
// A's slot t holds row 2t and its slot t + 4 row 2t + 1.
template <typename T, int TILES, int PA, int PITCH>
__device__ __forceinline__ void mma_rows(float (&d)[TILES][4], const Frag<4, PA>& a, const T* rows) {
  const int lane = threadIdx.x & 31;
  if constexpr (sizeof(T) == 4) {
    const T* p = rows + lane % 4 * 2 * PITCH + lane / 4;
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
      Frag<2, 2> b;
      b.set(0, p[j * 8]);
      b.set(1, p[PITCH + j * 8]);
      mma_parts(d[j], a, b);
    }
  } else {
    constexpr int N = TILES % 4 == 0 ? 4 : TILES % 2 == 0 ? 2 : 1;
    const T* p = rows + lane % 8 * PITCH + lane / 8 % N * 8;
#pragma unroll
    for (int j = 0; j < TILES; j += N) {
      uint32_t r[N];
      load_blocks<N, true>(r, p + j * 8);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float2 x = unpack<T>(r[i]);
        Frag<2, 1> b;
        b.exact(0, x.x);
        b.exact(1, x.y);
        mma_parts(d[j + i], a, b);
      }
    }
  }
}

template <int TILES, int PITCH>
__device__ __forceinline__ void mma_rows_apart(float (&d)[TILES][4], float (&rest)[TILES][4], const Frag<4, 2>& a,
                                               const float* rows) {
  const int lane = threadIdx.x & 31;
  const float* p = rows + lane % 4 * 2 * PITCH + lane / 4;
#pragma unroll
  for (int j = 0; j < TILES; ++j) {
    Frag<2, 2> b;
    b.set(0, p[j * 8]);
    b.set(1, p[PITCH + j * 8]);
    mma_apart(d[j], rest[j], a, b);
  }
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
constexpr int pitch(int d) { return d + 16 / (int)sizeof(T); }  // 4 words past a multiple of 32: conflict-free columns

template <typename T, int DK, int DV>
struct Shape {
  static constexpr bool kSplit = sizeof(T) == 4;          // float32: every operand in two parts
  static constexpr int kPK = pitch<T>(DK), kPV = pitch<T>(DV), kPS = DV + 4;
  static constexpr int kTile = kC * (2 * kPK + kPV) * sizeof(T);  // q, k, v of one chunk
  static constexpr int kState = DK * kPS * 4;
  static constexpr int kTable = 3 * (kC + 1) * 4 + 24;
  static constexpr int kStages = 2 * kTile + kState + kTable <= 113 * 1024 || sizeof(T) == 2 ? 2 : 1;
  static constexpr int kSmem = kStages * kTile + kState + kTable;
  static constexpr int kBlocks = kSmem <= 113 * 1024 && DK * DV <= 64 * 64 ? 2 : 1;  // per SM
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert(4 * (DK * DV + 8 * (2 * DK + DV + kThreads)) <= kStages * kTile + kState, "walk_with_care");
  // state: warps tile DK in blocks of 16 rows, the rest of them the columns
  static constexpr int kSRows = DK / 16 < 8 ? DK / 16 : 8, kSCols = 8 / kSRows;
  static constexpr int kSTiles = DV / 8 / kSCols;          // 8-column tiles of a warp
  static_assert(DK / 16 <= 8 && kSTiles >= 1, "state layout");
  // output: 4 blocks of 16 rows, two halves of the columns
  static constexpr int kOTiles = DV / 16;
};

// The rows of one chunk of one operand into shared memory, zeros behind its width and length.
template <typename T, int D, int P>
__device__ __forceinline__ void load_rows(T* dst, const T* src, long long row_stride, int rows, int width, bool back,
                                          bool wide) {
  constexpr int V = 16 / sizeof(T), PER = D / V;
  if (wide) {
    for (int i = threadIdx.x; i < kC * PER; i += kThreads) {
      const int r = i / PER, c = i % PER * V;
      const bool in = r < rows && c < width;
      const T* p = src + (in ? (long long)(back ? -r : r) * row_stride + c : 0);
      cp_async16(dst + r * P + c, p, in ? 16 : 0);
    }
  } else {
    for (int i = threadIdx.x; i < kC * D; i += kThreads) {
      const int r = i / D, c = i % D;
      dst[r * P + c] = r < rows && c < width ? src[(long long)(back ? -r : r) * row_stride + c] : from_f32<T>(0.f);
    }
  }
}

__device__ __forceinline__ long long cu_value(const DecayArgs& a, int i) {
  const long long x = a.cu64 ? static_cast<const long long*>(a.cu)[i] : (long long)static_cast<const int*>(a.cu)[i];
  return x < 0 ? 0 : (x > a.tokens ? a.tokens : x);  // no value of cu leads outside the tensors
}

// The segment of a unit: its sequence, first token and length, whether it is the sequence's last,
// and how long the sequence is.  seq < 0: none.
struct Segment {
  long long first, len, start, total;  // of the segment; of its sequence
  int seq;
};

// Called by warp 0.
__device__ __forceinline__ Segment find_segment(const DecayArgs& a, int unit) {
  Segment s;
  s.seq = -1;
  s.first = s.len = s.start = s.total = 0;
  if (!a.cu) {
    s.seq = unit / a.segs;
    s.total = a.tokens;
    s.first = (long long)(unit % a.segs) * a.seg_len;
    s.len = min((long long)a.seg_len, a.tokens - s.first);
    return s;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 32) {
    const int i = i0 + lane;
    long long lo = 0, n = 0;
    int count = 0;
    if (i < a.nseq) {
      lo = cu_value(a, i);
      n = cu_value(a, i + 1) - lo;
      if (n < 0) n = 0;
      count = max(1, (int)((n + a.seg_len - 1) / a.seg_len));
    }
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    const bool here = i < a.nseq && unit >= before + upto - count && unit < before + upto;
    const unsigned who = __ballot_sync(~0u, here);
    if (who) {
      const int l = __ffs(who) - 1;
      lo = __shfl_sync(~0u, lo, l);
      n = __shfl_sync(~0u, n, l);
      const int k = unit - before - __shfl_sync(~0u, upto - count, l);
      s.seq = i0 + l;
      s.start = lo;
      s.total = n;
      s.first = (long long)k * a.seg_len;
      s.len = min((long long)a.seg_len, n - s.first);
      return s;
    }
    before += __shfl_sync(~0u, upto, 31);
  }
  return s;
}

// What a launch does: whole sequences, the segments' own final states (from 0), or the segments'
// outputs from the states carried into them.
enum Pass { kWhole, kLocal, kCarried };

// The start of a pass over a segment: its (sequence, head)'s place in the tensors.
struct Place {
  long long row0;   // row i of the segment is token row0 + i, or row0 - i from the sequence's end
  long long batch, sbase;
  float* seg_state;
  __device__ __forceinline__ Place(const DecayArgs& a, const DecayRole& R, const Segment& seg, int unit, int h) {
    row0 = seg.start + (R.back ? seg.total - 1 - seg.first : seg.first);
    batch = a.cu ? 0 : seg.seq;
    sbase = ((long long)seg.seq * a.heads + h) * R.wk * R.wv;
    seg_state = R.seg ? R.seg + ((long long)unit * a.heads + h) * R.wk * R.wv : nullptr;
  }
};

// The same segment token by token, one product at a time, where the walk's states do not end finite.  In
// the walk an infinite factor in two parts makes NaN of sums that are infinite, and keys behind a row
// have weight 0 in P, but 0 times an infinite or NaN value is NaN.  All roles have a = r c, so here
//   forwards   S = g S + c k v^T,  o = r q S        backwards   S = S + c k v^T,  o = r q S,  S = g S
// from S = C, and C' = S.  kCare tokens at a time: their rows in shared memory as float32, and a thread
// takes each of its elements of S through all of them (8 x 4096 tokens of 16 heads of 128,
// every head with a NaN: 9 ms).
constexpr int kCare = 8;
template <typename T>
__device__ __forceinline__ void walk_with_care(const DecayArgs& a, const DecayRole& R, int pass, const Segment& seg,
                                               const DecayFactor& factor, float* sm) {
  const int h = blockIdx.x % a.heads, unit = blockIdx.x / a.heads, tid = threadIdx.x;
  const Place at(a, R, seg, unit, h);
  const bool want_o = R.o && pass != kLocal, back = R.back;
  float *S = sm, *sk = S + (R.wk * R.wv + 3) / 4 * 4, *sq = sk + kCare * R.wk, *sv = sq + kCare * R.wk, *red = sv + kCare * R.wv;
  const DecayFactor f = factor;
  // a thread has one column and every `step`-th row
  int columns = 1;
  while (columns < R.wv) columns *= 2;
  const int col = tid % columns, step = kThreads / columns;
  const bool mine = col < R.wv;
  __syncthreads();
#pragma unroll 1
  for (int d = tid / columns; mine && d < R.wk; d += step) {
    float x = 0.f;
    if (pass == kCarried) x = at.seg_state[d * R.wv + col];
    if (pass == kWhole && R.first) x = R.first[at.sbase + d * R.first_sk + col * R.first_sv];
    S[d * R.wv + col] = x;
  }
#pragma unroll 1
  for (long long i = 0; i < seg.len; i += kCare) {
    const int rows = (int)min((long long)kCare, seg.len - i);
    const long long token = R.back ? at.row0 - i : at.row0 + i;  // of row 0; the others follow in time
    auto stage = [&](float* to, const void* from, const long long* stride, int div, int width) {
      const T* p = static_cast<const T*>(from) + at.batch * stride[0] + (long long)(h / div) * stride[2];
#pragma unroll 1
      for (int e = tid; e < rows * width; e += kThreads) {
        const int r = e / width, x = e % width;
        to[x * kCare + r] = to_f32(p[(token + (R.back ? -r : r)) * stride[1] + x]);
      }
    };
    stage(sk, R.k, R.ks, R.kdiv, R.wk);
    stage(sv, R.v, R.vs, R.vdiv, R.wv);
    if (want_o) stage(sq, R.q, R.qs, R.qdiv, R.wk);
    __syncthreads();
    float v[kCare], o[kCare];
#pragma unroll
    for (int r = 0; r < kCare; ++r) {
      v[r] = mine && r < rows ? R.c * sv[col * kCare + r] : 0.f;
      o[r] = 0.f;
    }
#pragma unroll 1
    for (int d = tid / columns; mine && d < R.wk; d += step) {
      float x = S[d * R.wv + col], k[kCare], q[kCare];
#pragma unroll
      for (int r = 0; r < kCare; r += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(sk + d * kCare + r), q4 = *reinterpret_cast<const float4*>(sq + d * kCare + r);
        k[r] = k4.x, k[r + 1] = k4.y, k[r + 2] = k4.z, k[r + 3] = k4.w;
        q[r] = q4.x, q[r + 1] = q4.y, q[r + 2] = q4.z, q[r + 3] = q4.w;
      }
      if (back) {
#pragma unroll
        for (int r = 0; r < kCare; ++r)
          if (r < rows) {
            x += k[r] * v[r];
            o[r] = fmaf(q[r], x, o[r]);
            x = f.step(x, 0.f);
          }
      } else {
#pragma unroll
        for (int r = 0; r < kCare; ++r)
          if (r < rows) {
            x = f.step(x, k[r] * v[r]);
            o[r] = fmaf(q[r], x, o[r]);
          }
      }
      S[d * R.wv + col] = x;
    }
    if (want_o) {
#pragma unroll
      for (int r = 0; r < kCare; ++r) red[r * kThreads + tid] = o[r];
    }
    __syncthreads();
    if (!want_o) continue;
#pragma unroll 1
    for (int e = tid; e < rows * R.wv; e += kThreads) {
      const int r = e / R.wv, x = e % R.wv;
      float sum = 0.f;
#pragma unroll 1
      for (int j = 0; j < step; ++j) sum += red[r * kThreads + j * columns + x];
      const long long to = at.batch * R.os[0] + (long long)h * R.os[2] + (token + (R.back ? -r : r)) * R.os[1] + x;
      if (R.o_f32) static_cast<float*>(R.o)[to] = R.r * sum;
      else static_cast<T*>(R.o)[to] = from_f32<T>(R.r * sum);
    }
  }
  float* to = pass == kLocal ? at.seg_state : (pass == kWhole && R.last ? R.last + at.sbase : nullptr);
  if (!to) return;
#pragma unroll 1
  for (int d = tid / columns; mine && d < R.wk; d += step) to[d * R.wv + col] = S[d * R.wv + col];
}

template <typename T, int DK, int DV>
__device__ __forceinline__ void walk(const DecayArgs& a, const DecayRole& R, int pass, unsigned char* sm) {
  using S = Shape<T, DK, DV>;
  constexpr int PK = S::kPK, PV = S::kPV, PS = S::kPS, STAGES = S::kStages;
  float* state = reinterpret_cast<float*>(sm + STAGES * S::kTile);
  float* dec = state + DK * PS;  // g^n, n <= 64, and the same as factors of a state
  DecayFactor* factor = reinterpret_cast<DecayFactor*>(dec + kC + 1);
  __shared__ Segment seg_shared;

  const int h = blockIdx.x % a.heads, unit = blockIdx.x / a.heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;

  // (with flags: only what an earlier kernel left to this one)
  if (a.flags && (unit == a.units || !a.flags[((long long)blockIdx.z * a.units + unit) * a.heads + h])) return;
  if (a.cu && unit == a.units) {  // the rows of no sequence
    if (!R.o || pass == kLocal) return;
    const long long lo = cu_value(a, 0), hi = max(lo, cu_value(a, a.nseq));
    for (long long r = warp; r < lo + (a.tokens - hi); r += 8) {
      const long long at = (long long)h * R.os[2] + (r < lo ? r : hi + r - lo) * R.os[1];
      for (int c = lane; c < R.wv; c += 32) {
        if (R.o_f32)
          static_cast<float*>(R.o)[at + c] = 0.f;
        else
          static_cast<T*>(R.o)[at + c] = from_f32<T>(0.f);
      }
    }
    return;
  }
  if (warp == 0) {
    const Segment s = find_segment(a, unit);
    if (lane == 0) seg_shared = s;
  }
  {
    const float ld = a.log_decay[h];
    for (int n = threadIdx.x; n <= kC; n += kThreads) {
      const double x = n ? exp((double)ld * n) : 1.0;
      dec[n] = (float)x;
      factor[n] = DecayFactor(x, ld);
    }
  }
  __syncthreads();
  const Segment seg = seg_shared;
  if (seg.seq < 0) return;
  const int back = R.back, len = (int)seg.len;
  const bool want_o = R.o && pass != kLocal;
  const Place place(a, R, seg, unit, h);
  const long long row0 = place.row0, batch = place.batch, sbase = place.sbase;
  const T* q = static_cast<const T*>(R.q) + batch * R.qs[0] + (long long)(h / R.qdiv) * R.qs[2] + row0 * R.qs[1];
  const T* k = static_cast<const T*>(R.k) + batch * R.ks[0] + (long long)(h / R.kdiv) * R.ks[2] + row0 * R.ks[1];
  const T* v = static_cast<const T*>(R.v) + batch * R.vs[0] + (long long)(h / R.vdiv) * R.vs[2] + row0 * R.vs[1];
  const long long obase = batch * R.os[0] + (long long)h * R.os[2] + row0 * R.os[1];
  float* seg_state = place.seg_state;
  // a kLocal pass of a sequence's last segment serves its final state alone
  if (pass == kLocal && !R.last && seg.first + seg.len >= seg.total) return;

  auto load = [&](int c, int stage) {
    T* dst = reinterpret_cast<T*>(sm + stage * S::kTile);
    const int rows = min(kC, len - c * kC);
    const long long skip = (long long)(back ? -c : c) * kC;
    if (want_o) load_rows<T, DK, PK>(dst, q + skip * R.qs[1], R.qs[1], rows, R.wk, back, R.wide & 1);
    load_rows<T, DK, PK>(dst + kC * PK, k + skip * R.ks[1], R.ks[1], rows, R.wk, back, R.wide & 2);
    load_rows<T, DV, PV>(dst + 2 * kC * PK, v + skip * R.vs[1], R.vs[1], rows, R.wv, back, R.wide & 4);
    cp_commit();
  };
  const int chunks = a.flags ? 0 : (len + kC - 1) / kC;  // (what is left to this kernel is walked with care)

  // the state: rows sr + g (+ 8), columns sc + 8 j + 2 t (+ 1)
  const int sr = warp % S::kSRows * 16, sc = warp / S::kSRows * (S::kSTiles * 8);
  float st[S::kSTiles][4];
  if (chunks > 0) load(0, 0);
  {
    const float* from = pass == kCarried ? seg_state : (pass == kWhole ? R.first : nullptr);
    const long long sk = pass == kCarried ? R.wv : R.first_sk, sv = pass == kCarried ? 1 : R.first_sv;
    const long long base = pass == kCarried ? 0 : sbase;
#pragma unroll
    for (int j = 0; j < S::kSTiles; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = sr + g + (e >> 1) * 8, col = sc + j * 8 + 2 * t + (e & 1);
        st[j][e] = from && row < R.wk && col < R.wv ? from[base + row * sk + col * sv] : 0.f;
      }
  }
  auto put_state = [&] {
#pragma unroll
    for (int j = 0; j < S::kSTiles; ++j)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        *reinterpret_cast<float2*>(state + (sr + g + (e >> 1) * 8) * PS + sc + j * 8 + 2 * t) =
            make_float2(st[j][e], st[j][e + 1]);
      }
  };
  if (want_o) put_state();

  // rows of P and o: two of the warps that share a scheduler have 5 blocks of 16 keys together
  const int mi = warp < 4 ? warp : 7 - warp, oc = warp / 4 * (DV / 2);
  // Weights a g^d of this thread's places in a block of 8 keys, d tokens from the key to the row: in the
  // row's own block, in the one before, and (as products with cf) in those before that.
  const float own0 = R.a * dec[max(g - 2 * t, 0)], own1 = R.a * dec[max(g - 2 * t - 1, 0)];
  const float next0 = R.a * dec[g + 8 - 2 * t], next1 = R.a * dec[g + 7 - 2 * t];
  const float rf0 = R.a * dec[g + 1], rf1 = R.a * dec[g + 9], cf0 = dec[7 - 2 * t], cf1 = dec[6 - 2 * t], g8 = dec[8];

  for (int c = 0; c < chunks; ++c) {
    const int stage = STAGES == 2 ? c & 1 : 0, rows = min(kC, len - c * kC);
    if (STAGES == 2 && c + 1 < chunks) {
      load(c + 1, stage ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    const T* sq = reinterpret_cast<const T*>(sm + stage * S::kTile);
    const T* sk = sq + kC * PK;
    const T* sv = sk + kC * PK;
    if (want_o && mi * 16 < rows) {
      float acc[S::kOTiles][4], pr[8][4];
#pragma unroll
      for (int j = 0; j < S::kOTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[n][e] = 0.f;
      constexpr int kRest = S::kSplit ? 8 : 1, kRestO = S::kSplit ? S::kOTiles : 1;
      float pr_rest[kRest][4], acc_rest[kRestO][4];
#pragma unroll
      for (int n = 0; n < kRest; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) pr_rest[n][e] = 0.f;
#pragma unroll
      for (int j = 0; j < kRestO; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc_rest[j][e] = 0.f;
      // q k^T, for the 8-key blocks n that are not behind all rows, and q C, from the same parts of q
      if constexpr (S::kSplit) {
        // (one after the other: the sums of both at once do not fit the registers of two blocks per SM)
        const T* qrow = sq + (mi * 16 + g) * PK;
        auto q_parts = [&](int kk) {
          Frag<4, 2> fa;
          const int at = kk * 8 + 2 * t;
#pragma unroll
          for (int e = 0; e < 4; ++e) fa.set(e, to_f32(qrow[at + (e & 1) * 8 * PK + (e >> 1)]));
          return fa;
        };
#pragma unroll 1
        for (int kk = 0; kk < DK / 8; ++kk) {
          const Frag<4, 2> fa = q_parts(kk);
          const T* krow = sk + g * PK + kk * 8 + 2 * t;
#pragma unroll
          for (int n = 0; n < 8; ++n)
            if (n < 2 * mi + 2) {
              Frag<2, 2> fb;
              fb.set(0, to_f32(krow[n * 8 * PK]));
              fb.set(1, to_f32(krow[n * 8 * PK + 1]));
              mma_apart(pr[n], pr_rest[n], fa, fb);
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[n][e] += pr_rest[n][e];
#pragma unroll 1
        for (int kk = 0; kk < DK / 8; ++kk)
          mma_rows_apart<S::kOTiles, PS>(acc, acc_rest, q_parts(kk), state + kk * 8 * PS + oc);
      } else {
        const T* qp = sq + (mi * 16 + lane % 16) * PK + lane / 16 * 8;
        const T* kp = sk + (lane / 16 * 8 + lane % 8) * PK + lane / 8 % 2 * 8;
#pragma unroll 2
        for (int kb = 0; kb < DK / 16; ++kb) {
          uint32_t fq[4];
          load_blocks<4, false>(fq, qp + kb * 16);
#pragma unroll
          for (int n = 0; n < 8; n += 2)
            if (n < 2 * mi + 2) {
              uint32_t fk[4];
              load_blocks<4, false>(fk, kp + n * 8 * PK + kb * 16);
              mma_16<T>(pr[n], fq, fk[0], fk[1]);
              mma_16<T>(pr[n + 1], fq, fk[2], fk[3]);
            }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 x = unpack<T>(fq[2 * half]), y = unpack<T>(fq[2 * half + 1]);
            Frag<4, 1> fa;
            fa.exact(0, x.x);
            fa.exact(1, y.x);
            fa.exact(2, x.y);
            fa.exact(3, y.y);
            const float* sp = state + (kb * 16 + half * 8 + 2 * t) * PS + oc + g;
#pragma unroll
            for (int j = 0; j < S::kOTiles; ++j) {
              Frag<2, 2> fb;
              fb.cut(0, sp[j * 8]);
              fb.cut(1, sp[PS + j * 8]);
              mma_parts(acc[j], fa, fb);
            }
          }
        }
      }
      const int i0 = mi * 16 + g;
      const float f0 = R.r * dec[i0 + 1 - back], f1 = R.r * dec[i0 + 9 - back];
#pragma unroll
      for (int j = 0; j < S::kOTiles; ++j) {
        acc[j][0] *= f0;
        acc[j][1] *= f0;
        acc[j][2] *= f1;
        acc[j][3] *= f1;
        if constexpr (S::kSplit) {
          acc_rest[j][0] *= f0;
          acc_rest[j][1] *= f0;
          acc_rest[j][2] *= f1;
          acc_rest[j][3] *= f1;
        }
      }
      // + P v, from the diagonal on to the first keys: there the weights shrink by g^8 a block
      float near0 = rf0, near1 = rf1;
#pragma unroll
      for (int n = 7; n >= 0; --n)
        if (n < 2 * mi + 2) {
          float w[4];
          if (n == 2 * mi + 1) {
            w[0] = w[1] = 0.f;
            w[2] = own0;
            w[3] = own1;
          } else if (n == 2 * mi) {
            w[0] = own0;
            w[1] = own1;
            w[2] = next0;
            w[3] = next1;
          } else {
            w[0] = near0 * cf0;
            w[1] = near0 * cf1;
            w[2] = near1 * cf0;
            w[3] = near1 * cf1;
            near0 *= g8;
            near1 *= g8;
          }
          Frag<4, 2> fp;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool behind = (n == 2 * mi + 1 && e < 2) || (n >= 2 * mi && (e >> 1) == n - 2 * mi && 2 * t + (e & 1) > g);
            // C layout (row, 2t + e&1) to A layout (row, slot t + 4 (e&1)): key 2t + s sits in slot t + 4 s
            const float x = behind ? 0.f : pr[n][e] * w[e];
            if constexpr (S::kSplit) fp.set((e >> 1) + (e & 1) * 2, x);
            else fp.cut((e >> 1) + (e & 1) * 2, x);
          }
          if constexpr (S::kSplit)
            mma_rows_apart<S::kOTiles, PV>(acc, acc_rest, fp, sv + n * 8 * PV + oc);
          else
            mma_rows<T, S::kOTiles, 2, PV>(acc, fp, sv + n * 8 * PV + oc);
        }
      if constexpr (S::kSplit) {
#pragma unroll
        for (int j = 0; j < S::kOTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] += acc_rest[j][e];
      }
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int i = i0 + (e >> 1) * 8;
        if (i >= rows) continue;
        const long long at = obase + (long long)(back ? -(c * kC + i) : c * kC + i) * R.os[1] + oc + 2 * t;
        const int w = R.wv - oc - 2 * t;  // columns from here on
#pragma unroll
        for (int j = 0; j < S::kOTiles; ++j) {
          const float x = acc[j][e], y = acc[j][e + 1];
          if (R.o_f32) {
            float* o = static_cast<float*>(R.o) + at + j * 8;
            if (R.wide & 8) {
              if (j * 8 + 1 < w) *reinterpret_cast<float2*>(o) = make_float2(x, y);
            } else {
              if (j * 8 < w) o[0] = x;
              if (j * 8 + 1 < w) o[1] = y;
            }
          } else {
            T* o = static_cast<T*>(R.o) + at + j * 8;
            if (R.wide & 8) {
              if (j * 8 + 1 < w) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(o) = make_float2(x, y);
                else from_f32_pair(x, y, o);
              }
            } else {
              if (j * 8 < w) o[0] = from_f32<T>(x);
              if (j * 8 + 1 < w) o[1] = from_f32<T>(y);
            }
          }
        }
      }
    }
    // C' = g^n C + (scaled k)^T v
    {
      float d[S::kSTiles][4];
#pragma unroll
      for (int j = 0; j < S::kSTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[j][e] = 0.f;
      const int blocks = (rows + 15) / 16;
#pragma unroll 1
      for (int kb = 0; kb < blocks; ++kb) {
        uint32_t fk[4];
        if constexpr (!S::kSplit) load_blocks<4, true>(fk, sk + (kb * 16 + lane / 16 * 8 + lane % 8) * PK + sr + lane / 8 % 2 * 8);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int j0 = kb * 16 + half * 8 + 2 * t;
          const float w0 = R.c * dec[max(rows - 1 - j0 + back, 0)], w1 = R.c * dec[max(rows - 2 - j0 + back, 0)];
          Frag<4, 2> fa;
          if constexpr (S::kSplit) {
            const T* p = sk + j0 * PK + sr + g;
            fa.set(0, to_f32(p[0]) * w0);
            fa.set(1, to_f32(p[8]) * w0);
            fa.set(2, to_f32(p[PK]) * w1);
            fa.set(3, to_f32(p[PK + 8]) * w1);
          } else {
            const float2 x = unpack<T>(fk[2 * half]), y = unpack<T>(fk[2 * half + 1]);
            fa.set(0, x.x * w0);
            fa.set(1, y.x * w0);
            fa.set(2, x.y * w1);
            fa.set(3, y.y * w1);
          }
          mma_rows<T, S::kSTiles, 2, PV>(d, fa, sv + (kb * 16 + half * 8) * PV + sc);
        }
      }
      const DecayFactor f = factor[rows];
#pragma unroll
      for (int j = 0; j < S::kSTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[j][e] = f.step(st[j][e], d[j][e]);
    }
    if (c + 1 < chunks) {
      __syncthreads();  // all have read the stage and the state
      if (want_o) put_state();
      if (STAGES == 1) load(c + 1, 0);
    }
  }
  float bad = 0.f;
#pragma unroll
  for (int j = 0; j < S::kSTiles; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) bad = fmaf(st[j][e], 0.f, bad);
  if (__syncthreads_or(bad != 0.f || a.flags)) return walk_with_care<T>(a, R, pass, seg_shared, factor[1], reinterpret_cast<float*>(sm));
  float* to = pass == kLocal ? seg_state : (pass == kWhole && R.last ? R.last + sbase : nullptr);
  if (to) {
#pragma unroll
    for (int j = 0; j < S::kSTiles; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = sr + g + (e >> 1) * 8, col = sc + j * 8 + 2 * t + (e & 1);
        if (row < R.wk && col < R.wv) to[row * R.wv + col] = st[j][e];
      }
  }
}

// Widths padded to D0 <= D1: the roles of one call have both orders (the gradients of q and k have
// keys of the values' width), and run in one launch.
template <typename T, int D0, int D1>
__global__ void __launch_bounds__(kThreads, (Shape<T, D0, D1>::kBlocks))
    k_decay_chunk(const __grid_constant__ DecayArgs a, int pass) {
  extern __shared__ __align__(128) unsigned char sm[];
  const DecayRole& R = a.role[blockIdx.z];
  if (D0 == D1 || R.wk <= D0)
    walk<T, D0, D1>(a, R, pass, sm);
  else if constexpr (D0 != D1)
    walk<T, D1, D0>(a, R, pass, sm);
}

template <typename T, int D0, int D1>
static cudaError_t run_widths(const DecayArgs& a, Pass pass, cudaStream_t st) {
  constexpr int smem = Shape<T, D0, D1>::kSmem > Shape<T, D1, D0>::kSmem ? Shape<T, D0, D1>::kSmem : Shape<T, D1, D0>::kSmem;
  const cudaError_t e = allow_shared<k_decay_chunk<T, D0, D1>>(smem);
  if (e != cudaSuccess) return e;
  const unsigned units = (unsigned)a.units + (a.cu && pass != kLocal ? 1 : 0);
  k_decay_chunk<T, D0, D1><<<dim3(units * a.heads, 1, a.roles), kThreads, smem, st>>>(a, pass);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_chunks(const DecayArgs& a, Pass pass, cudaStream_t st) {
  const int lo = padded_width(min(a.role[0].wk, a.role[0].wv)), hi = padded_width(max(a.role[0].wk, a.role[0].wv));
  if (hi == 32) return run_widths<T, 32, 32>(a, pass, st);
  if (hi == 64) return lo == 32 ? run_widths<T, 32, 64>(a, pass, st) : run_widths<T, 64, 64>(a, pass, st);
  if (lo == 32) return run_widths<T, 32, 128>(a, pass, st);
  return lo == 64 ? run_widths<T, 64, 128>(a, pass, st) : run_widths<T, 128, 128>(a, pass, st);
}

template <typename T>
cudaError_t run_all(const DecayArgs& a, cudaStream_t st) {
  if (!a.split) return run_chunks<T>(a, kWhole, st);
  cudaError_t e = run_chunks<T>(a, kLocal, st);
  if (e == cudaSuccess) e = launch_decay_scan(a, st);
  return e == cudaSuccess ? run_chunks<T>(a, kCarried, st) : e;
}

}  // namespace chunk
}  // namespace tfb
