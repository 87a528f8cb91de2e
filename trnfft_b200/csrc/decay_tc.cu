// Decayed linear attention for bfloat16 operands on the 5th-generation tensor
// cores (tcgen05, accumulators in TMEM), in chunks of 128 tokens.
//
// The same walk as decay_chunk.cuh, with P_ij = a g^{i-j} (q_i . k_j):
//   P = q k^T     M = tokens, N = tokens      A, B: rows of the width (K-major)
//   X = q C       M = tokens, N = values      B: C, rows of keys (MN-major)
//   O = P v       M = tokens, N = values      A: P from TMEM; B: v (MN-major)
//   E = k'^T v    M = keys,   N = values      A: k' = c g^{n-1-j} k (MN-major); B: v
//   o = O + r g^{i+1} X,   C' = g^n C + E
// Every operand tile in shared memory is [columns/64][rows][64 columns of 2
// bytes], its 16-byte pieces swizzled by the row (SWIZZLE_128B): the same bytes
// serve as K-major and, with rows as K, as MN-major operand.
//
// Precision: q k^T is exact up to float32 sums.  P and C are multiplied in two
// bfloat16 parts each (2^-17), k' in three (2^-25): with one part each, rounding
// P and C alone would double the error that the rounding of o makes, and the
// state, a float32 result, would be off by 2^-9.  C itself stays in float32
// registers and is scaled by g^n as a sum of two float32.
//
// One block per (segment, head, role), 13 warps:
//   0-3   P: read from TMEM, weigh, split, write back as the A operand of P v
//   4-7   k': in place of k, and its other two parts beside it
//   0-7   o, half of the columns each; the state, likewise
//   8     one thread issues every product
//   9-12  loads: cp.async, row by row (any strides, either direction, zeros
//         behind a sequence's end); q as soon as X is done, k and v after E
// What bounds it: at 128 x 128 a chunk's products take 4096 cycles of the
// tensor pipe, its bytes 5700 at 1/148 of the measured bandwidth.
//
// A masked P is 0, and 0 times an infinite or NaN value is NaN: blocks whose o
// is not finite somewhere say so, and the walk of decay_chunk.cuh, which looks
// at such rows one by one, takes them again.
#include "decay_attn.h"
#include "decay_chunk.cuh"

namespace tfb {
namespace tc {

constexpr int kC = 128;
constexpr int kComputeWarps = 8, kMmaWarp = 8;
constexpr uint32_t kBlockBytes = kC * 128;  // 64 columns of a tile

template <int D>
struct Shape {
  static constexpr int kLoadWarps = D == 128 ? 4 : 2;
  static constexpr int kThreads = 32 * (kComputeWarps + 1 + kLoadWarps);
  static constexpr int kTile = kC * D * 2, kState = D * D * 2;
  static constexpr int kQ = 0, kK = kTile, kV = 2 * kTile, kMid = 3 * kTile, kLo = 4 * kTile;
  static constexpr int kSHi = 5 * kTile, kSLo = kSHi + kState, kTable = kSLo + kState;
  static constexpr int kSmem = kTable + 2 * (kC + 1) * 4 + 56 + 10 * 8 + 64 + 48;
  // TMEM columns: P (also in two bfloat16 parts), O, X, E.  With D = 64, E shares X's, so that two
  // blocks fit on an SM; X is then read before E is issued.
  static constexpr int kP = 0, kO = 128, kX = 128 + D, kE = D == 64 ? kX : kX + D;
  static constexpr int kColumns = D == 64 ? 256 : 512;
  static constexpr bool kShared = D == 64;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

enum Bar { kFull, kQK, kQS, kPV, kKV, kPDone, kKDone, kSReady, kXRead, kBars };

__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;  // MN-major: from 64 columns to the next 64
  d |= (uint64_t)(1024 >> 4) << 32;            // from 8 rows to the next 8
  d |= (uint64_t)1 << 46;                      // descriptor version
  d |= (uint64_t)2 << 61;                      // SWIZZLE_128B
  return d;
}
// D float32, A and B bfloat16; ta / tb: operand is MN-major
constexpr uint32_t idesc(int n, bool ta, bool tb) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((ta ? 1u : 0u) << 15) | ((tb ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(add)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A bounded wait; false once any wait of the block has given up.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  bool ok = false;
  for (int i = 0; i < (1 << 22) && !*gave_up; ++i)
    if ((ok = mbar_try_wait(bar, parity))) break;
  if (!ok) *gave_up = 1;
  return ok;
}
// The same for a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  return __all_sync(~0u, wait(bar, parity, gave_up));
}

__device__ __forceinline__ void tmem_ld32(uint32_t (&v)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&v)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
      "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two neighbours as bfloat16 (the first in the lower half), and what that loses of them.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
__device__ __forceinline__ float low_f32(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_f32(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

template <int D>
__global__ void __launch_bounds__(Shape<D>::kThreads, D == 64 ? 2 : 1)
    k_decay_tc(const __grid_constant__ DecayArgs a, int pass) {
  using S = Shape<D>;
  using chunk::kCarried;
  using chunk::kLocal;
  using chunk::kWhole;
  extern __shared__ __align__(1024) unsigned char sm[];
  float* dec = reinterpret_cast<float*>(sm + S::kTable);
  float* dec_lo = dec + kC + 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + ((S::kTable + 2 * (kC + 1) * 4 + 7) & ~7));
  chunk::Segment* seg_shared = reinterpret_cast<chunk::Segment*>(bars + 10);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(seg_shared + 1);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* odd = reinterpret_cast<int*>(tmem_slot + 2);

  const DecayRole& R = a.role[blockIdx.z];
  const int h = blockIdx.x % a.heads, unit = blockIdx.x / a.heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (a.cu && unit == a.units) {  // the rows of no sequence
    if (!R.o || pass == kLocal) return;
    const long long lo = chunk::cu_value(a, 0), hi = max(lo, chunk::cu_value(a, a.nseq));
    for (long long r = warp; r < lo + (a.tokens - hi); r += S::kThreads / 32) {
      const long long at = (long long)h * R.os[2] + (r < lo ? r : hi + r - lo) * R.os[1];
      for (int c = lane; c < R.wv; c += 32) {
        if (R.o_f32) static_cast<float*>(R.o)[at + c] = 0.f;
        else static_cast<__nv_bfloat16*>(R.o)[at + c] = from_f32<__nv_bfloat16>(0.f);
      }
    }
    return;
  }
  if (warp == 0) {
    const chunk::Segment s = chunk::find_segment(a, unit);
    if (lane == 0) *seg_shared = s;
  }
  {
    const double ld = a.log_decay[h];
    for (int n = threadIdx.x; n <= kC; n += S::kThreads) {
      const double x = n ? exp(ld * n) : 1.0, rest = x - (double)(float)x;
      dec[n] = (float)x;
      dec_lo[n] = rest == rest ? (float)rest : 0.f;
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBars; ++i) {
      const int count = i == kFull ? 32 * S::kLoadWarps
                                   : (i == kPDone || i == kKDone ? 128 : (i == kSReady || i == kXRead ? 256 : 1));
      mbar_init(&bars[i], count);
    }
    *gave_up = 0;
    *odd = 0;
    mbar_init_fence();
  }
  __syncthreads();
  const chunk::Segment seg = *seg_shared;
  const int len = (int)seg.len, back = R.back;
  const long long size = (long long)R.wk * R.wv;
  int* flag = a.flags ? a.flags + ((long long)blockIdx.z * a.units + unit) * a.heads + h : nullptr;
  // a kLocal pass of a sequence's last segment serves its final state alone
  if (seg.seq < 0 || (pass == kLocal && !R.last && seg.first + seg.len >= seg.total)) {
    if (threadIdx.x == 0 && flag) *flag = 0;
    return;
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot, base = smem_u32(sm);
  const bool want_o = R.o && pass != kLocal;
  const long long row0 = seg.start + (back ? seg.total - 1 - seg.first : seg.first);
  const long long batch = a.cu ? 0 : seg.seq;
  const int chunks = (len + kC - 1) / kC;

  if (warp > kMmaWarp) {
    // ---------------- loads
    const int t = threadIdx.x - 32 * (kMmaWarp + 1);
    constexpr int kLoaders = 32 * S::kLoadWarps, kVecs = D / 8;
    const int sign = back ? -1 : 1;
    auto rows_in = [&](int tile, const void* p, const long long* stride, int div, int width, int c) {
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p) + batch * stride[0] + (long long)(h / div) * stride[2] +
                                 (row0 + (long long)sign * c * kC) * stride[1];
      const int rows = min(kC, len - c * kC);
      const long long step = sign * stride[1];
      // a thread keeps its column and walks down the rows
      const int cc = t % kVecs, r0 = t / kVecs;
      const bool in = cc * 8 < width;
      const __nv_bfloat16* from = src + cc * 8;
      unsigned char* to = sm + tile + cc / 8 * kBlockBytes;
#pragma unroll 4
      for (int r = r0; r < kC; r += kLoaders / kVecs) {
        const bool live = in && r < rows;
        chunk::cp_async16(to + r * 128 + ((cc % 8) ^ (r & 7)) * 16, live ? from + r * step : src, live ? 16 : 0);
      }
    };
    auto touch = [&](const void* p, const long long* stride, int div, int width, int c) {  // into L2
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p) + batch * stride[0] + (long long)(h / div) * stride[2] +
                                 (row0 + (long long)sign * c * kC) * stride[1];
      const int rows = min(kC, len - c * kC);
      for (int r = t; r < rows; r += kLoaders)
        for (int x = 0; x < width; x += 64)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(src + (long long)sign * r * stride[1] + x));
    };
    for (int c = 0; c < chunks; ++c) {
      if (want_o) {
        if (c > 0 && !wait_warp(&bars[kQS], (c - 1) & 1, gave_up)) break;
        rows_in(S::kQ, R.q, R.qs, R.qdiv, R.wk, c);
      }
      if (c > 0 && !wait_warp(&bars[kKV], (c - 1) & 1, gave_up)) break;
      rows_in(S::kK, R.k, R.ks, R.kdiv, R.wk, c);
      rows_in(S::kV, R.v, R.vs, R.vdiv, R.wv, c);
      chunk::cp_commit();
      if (c + 1 < chunks) {
        touch(R.k, R.ks, R.kdiv, R.wk, c + 1);
        touch(R.v, R.vs, R.vdiv, R.wv, c + 1);
      }
      chunk::cp_wait<0>();
      fence_proxy_async();
      arrive(&bars[kFull]);
    }
    chunk::cp_wait<0>();
  } else if (warp == kMmaWarp) {
    // ---------------- products
    if (lane == 0) {
      constexpr uint32_t kQKId = idesc(128, false, false), kQSId = idesc(D, false, true), kPVId = idesc(D, false, true),
                         kKVId = idesc(D, true, true);
      for (int c = 0; c < chunks; ++c) {
        const uint32_t ph = c & 1;
        if (!wait(&bars[kFull], ph, gave_up)) break;
        fence_after();
        if (want_o) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = k / 4 * kBlockBytes + k % 4 * 32;
            mma_ss(tmem + S::kP, desc(base + S::kQ + at, 16), desc(base + S::kK + at, 16), kQKId, k > 0);
          }
          commit(&bars[kQK]);
          if (!wait(&bars[kSReady], ph, gave_up)) break;
          fence_after();
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_ss(tmem + S::kX, desc(base + S::kQ + k / 4 * kBlockBytes + k % 4 * 32, 16),
                     desc(base + (part ? S::kSLo : S::kSHi) + k * 2048, D * 128), kQSId, part + k > 0);
          commit(&bars[kQS]);
          if (!wait(&bars[kPDone], ph, gave_up)) break;
          fence_after();
#pragma unroll
          for (int k = 0; k < kC / 16; ++k) {
            const uint64_t v = desc(base + S::kV + k * 2048, kBlockBytes);
            mma_ts(tmem + S::kO, tmem + S::kP + k / 2 * 32 + k % 2 * 8, v, kPVId, k > 0);
            mma_ts(tmem + S::kO, tmem + S::kP + k / 2 * 32 + 16 + k % 2 * 8, v, kPVId, 1);
          }
          commit(&bars[kPV]);
        }
        if (!wait(&bars[kKDone], ph, gave_up)) break;
        if (!want_o && !wait(&bars[kSReady], ph, gave_up)) break;
        if (want_o && S::kShared && !wait(&bars[kXRead], ph, gave_up)) break;
        fence_after();
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) {
          const uint64_t v = desc(base + S::kV + k * 2048, kBlockBytes);
          mma_ss(tmem + S::kE, desc(base + S::kLo + k * 2048, kBlockBytes), v, kKVId, k > 0);
          mma_ss(tmem + S::kE, desc(base + S::kMid + k * 2048, kBlockBytes), v, kKVId, 1);
          mma_ss(tmem + S::kE, desc(base + S::kK + k * 2048, kBlockBytes), v, kKVId, 1);
        }
        commit(&bars[kKV]);
      }
    }
  } else {
    // ---------------- P, k', o and the state
    const int group = warp / 4, row = warp % 4 * 32 + lane, c0 = group * (D / 2);
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;  // TMEM lanes of this warp
    const long long sbase = ((long long)seg.seq * a.heads + h) * size;
    float* seg_state = R.seg ? R.seg + ((long long)unit * a.heads + h) * size : nullptr;
    float st[D / 2];
    {
      const float* from = pass == kCarried ? seg_state : (pass == kWhole && R.first ? R.first + sbase : nullptr);
      const long long sk = pass == kCarried ? R.wv : R.first_sk, sv = pass == kCarried ? 1 : R.first_sv;
#pragma unroll
      for (int j = 0; j < D / 2; ++j) st[j] = from && row < R.wk && c0 + j < R.wv ? from[row * sk + (c0 + j) * sv] : 0.f;
    }
    auto put_state = [&] {
      if (row < D) {
#pragma unroll
        for (int j = 0; j < D / 2; j += 8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = st[j + 2 * e], y = st[j + 2 * e + 1];
            hi[e] = pack_bf16(x, y);
            lo[e] = pack_bf16(x - low_f32(hi[e]), y - high_f32(hi[e]));
          }
          const uint32_t at = (c0 + j) / 64 * (D * 128) + row * 128 + ((((c0 + j) % 64) / 8) ^ (row & 7)) * 16;
          *reinterpret_cast<uint4*>(sm + S::kSHi + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(sm + S::kSLo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      fence_proxy_async();
      fence_before();
      arrive(&bars[kSReady]);
    };
    // kSReady: C is in shared memory for the products of the next chunk, and E has been read
    if (chunks > 0) {
      if (want_o) put_state();
      else arrive(&bars[kSReady]);
    }
    bool strange = false;
    for (int c = 0; c < chunks; ++c) {
      const uint32_t ph = c & 1;
      const int rows = min(kC, len - c * kC);
      if (group == 0) {
        if (want_o) {
          if (!wait_warp(&bars[kQK], ph, gave_up)) break;
          fence_after();
#pragma unroll 1
          for (int p = 0; p < 4; ++p) {
            uint32_t v[32];
            const uint32_t at = tmem + S::kP + p * 32 + lanes;
            if (p <= warp) {
              tmem_ld32(v, at);
              tmem_ld_wait();
              uint32_t out[32];
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                const int d = row - p * 32 - j;
                const float x = d >= 0 ? __uint_as_float(v[j]) * (R.a * dec[max(d, 0)]) : 0.f;
                const float y = d >= 1 ? __uint_as_float(v[j + 1]) * (R.a * dec[max(d - 1, 0)]) : 0.f;
                out[j / 2] = pack_bf16(x, y);
                out[16 + j / 2] = pack_bf16(x - low_f32(out[j / 2]), y - high_f32(out[j / 2]));
              }
              tmem_st32(at, out);
            } else {  // keys behind all of this warp's rows
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0;
              tmem_st32(at, v);
            }
          }
          tmem_st_wait();
          fence_before();
          arrive(&bars[kPDone]);
        }
      } else {
        if (!wait_warp(want_o ? &bars[kQK] : &bars[kFull], ph, gave_up)) break;
        const int t = threadIdx.x - 128;
#pragma unroll 2
        for (int i = t; i < S::kTile / 16; i += 128) {
          const int j = i / 8 % kC;
          const float w = R.c * dec[max(rows - 1 - j + back, 0)];
          uint4* at = reinterpret_cast<uint4*>(sm + S::kK) + i;
          const uint4 k = *at;
          const uint32_t in[4] = {k.x, k.y, k.z, k.w};
          uint32_t hi[4], mid[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = low_f32(in[e]) * w, y = high_f32(in[e]) * w;
            hi[e] = pack_bf16(x, y);
            x -= low_f32(hi[e]);
            y -= high_f32(hi[e]);
            mid[e] = pack_bf16(x, y);
            lo[e] = pack_bf16(x - low_f32(mid[e]), y - high_f32(mid[e]));
          }
          *at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          reinterpret_cast<uint4*>(sm + S::kMid)[i] = make_uint4(mid[0], mid[1], mid[2], mid[3]);
          reinterpret_cast<uint4*>(sm + S::kLo)[i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async();
        arrive(&bars[kKDone]);
      }
      if (want_o) {
        // o: row `row` of the chunk, columns c0 .. c0 + D/2
        constexpr int kW = 16;
        float x_kept[S::kShared ? D / 2 : 1];
        if (!wait_warp(&bars[kQS], ph, gave_up)) break;
        fence_after();
        if constexpr (S::kShared) {
#pragma unroll
          for (int j = 0; j < D / 2; j += kW) {
            uint32_t v[kW];
            tmem_ld16(v, tmem + S::kX + c0 + j + lanes);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < kW; ++e) x_kept[j + e] = __uint_as_float(v[e]);
          }
          fence_before();
          arrive(&bars[kXRead]);
        }
        if (!wait_warp(&bars[kPV], ph, gave_up)) break;
        fence_after();
        const float f = R.r * dec[row + 1 - back];
        const long long at = batch * R.os[0] + (long long)h * R.os[2] +
                             (row0 + (long long)(back ? -(c * kC + row) : c * kC + row)) * R.os[1] + c0;
        float bad = 0.f;
#pragma unroll
        for (int j = 0; j < D / 2; j += kW) {
          uint32_t o[kW], x[kW];
          __syncwarp();
          tmem_ld16(o, tmem + S::kO + c0 + j + lanes);
          if constexpr (!S::kShared) tmem_ld16(x, tmem + S::kX + c0 + j + lanes);
          tmem_ld_wait();
          float y[kW];
#pragma unroll
          for (int e = 0; e < kW; ++e) {
            const float xe = S::kShared ? x_kept[S::kShared ? j + e : 0] : __uint_as_float(x[e]);
            y[e] = fmaf(xe, f, __uint_as_float(o[e]));
            bad = fmaf(y[e], 0.f, bad);
          }
          if (row < rows) {
            if (R.o_f32) {
#pragma unroll
              for (int e = 0; e < kW; e += 4)
                if (c0 + j + e < R.wv)
                  *reinterpret_cast<float4*>(static_cast<float*>(R.o) + at + j + e) =
                      make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < kW; e += 8)
                if (c0 + j + e < R.wv)
                  *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(R.o) + at + j + e) =
                      make_uint4(pack_bf16(y[e], y[e + 1]), pack_bf16(y[e + 2], y[e + 3]), pack_bf16(y[e + 4], y[e + 5]),
                                 pack_bf16(y[e + 6], y[e + 7]));
            }
          }
        }
        strange = strange || (row < rows && bad != 0.f);
      }
      if (!wait_warp(&bars[kKV], ph, gave_up)) break;
      fence_after();
      const float hi = dec[rows], lo = dec_lo[rows];
      __syncwarp();
#pragma unroll
      for (int j = 0; j < D / 2; j += 16) {
        uint32_t v[16];
        tmem_ld16(v, tmem + S::kE + c0 + j + lanes);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) st[j + e] = fmaf(st[j + e], hi, fmaf(st[j + e], lo, __uint_as_float(v[e])));
      }
      if (c + 1 < chunks) {
        if (want_o) {
          put_state();
        } else {
          fence_before();
          arrive(&bars[kSReady]);
        }
      }
    }
    if (strange) *odd = 1;
    float* to = pass == kLocal ? seg_state : (pass == kWhole && R.last ? R.last + sbase : nullptr);
    if (to && row < R.wk) {
#pragma unroll
      for (int j = 0; j < D / 2; ++j)
        if (c0 + j < R.wv) to[row * R.wv + c0 + j] = st[j];
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
  }
  if (threadIdx.x == 0) {
    if (*gave_up) atomicExch(&g_dev_status, kStatusWaitTimeout);
    if (flag) *flag = *odd;
  }
}

template <int D>
static cudaError_t run_tc(const DecayArgs& a, chunk::Pass pass, cudaStream_t st) {
  using S = Shape<D>;
  cudaError_t e = cudaFuncSetAttribute(k_decay_tc<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned units = (unsigned)a.units + (a.cu && pass != chunk::kLocal ? 1 : 0);
  k_decay_tc<D><<<dim3(units * a.heads, 1, a.roles), S::kThreads, S::kSmem, st>>>(a, pass);
  return cudaGetLastError();
}

}  // namespace tc

cudaError_t launch_decay_tc(const DecayArgs& a, cudaStream_t st) {
  int wide = 0;
  for (int i = 0; i < a.roles; ++i) wide = max(wide, max(a.role[i].wk, a.role[i].wv));
  const chunk::Pass last = a.split ? chunk::kCarried : chunk::kWhole;
  cudaError_t e = cudaSuccess;
  DecayArgs b = a;
  if (a.split) {
    b.flags = nullptr;
    e = wide <= 64 ? tc::run_tc<64>(b, chunk::kLocal, st) : tc::run_tc<128>(b, chunk::kLocal, st);
    if (e == cudaSuccess) e = chunk::run_scan(a, st);
    if (e != cudaSuccess) return e;
  }
  e = wide <= 64 ? tc::run_tc<64>(a, last, st) : tc::run_tc<128>(a, last, st);
  if (e != cudaSuccess) return e;
  return chunk::run_chunks<__nv_bfloat16>(a, last, st);  // the blocks that said so, and no others
}

}  // namespace tfb
