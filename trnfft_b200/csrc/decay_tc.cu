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
// bfloat16 parts each (2^-16: the first is cut off, which leaves up to 2^-7, and
// the rest rounded to 8 bits), k' in three (2^-24): with one part each, rounding
// P and C alone would double the error that the rounding of o makes, and the
// state, a float32 result, would be off by 2^-8.  C itself stays in float32
// registers and is scaled by g^n as a sum of two float32.
//
// One block per (segment, head, role), 12 warps:
//   0-7   P: read from TMEM, weigh, split, write back as the A operand of P v;
//         k': in place of k, and its other two parts beside it;
//         o, through the state's place in shared memory to whole lines of
//         global memory; the state.  Two warps share 32 rows and split the columns.
//   8     one thread issues every product
//   9     loads by TMA; q as soon as X is done, k after the first
//         part of E, v after all of it.  Packed
//         sequences (a box would reach into a neighbour) and operands that no
//         tensor map describes are loaded row by row by warps 9-11 (cp.async).
// Tiles hold tokens in their natural order for either direction; backwards in
// time the mask and the weights are those of the mirrored row.
// What bounds it: at 128 x 128 a chunk's products take 4096 cycles of the
// tensor pipe, its bytes 5700 at 1/148 of the measured bandwidth, the operands,
// parts and staging in shared memory 6250 at 128 bytes a cycle; k and v have one
// buffer (227 KB are full), so their load is not hidden.  Measured: 8500 cycles
// a chunk; 8 x 4096 tokens, 16 heads (4 for k and v): 206-211 us, 1.6 TB/s (2 %
// of it for a bounded wait, not a barrier, before the state goes where o was).
//
// A masked P is 0, and 0 times an infinite or NaN value is NaN; so is an infinite
// value in parts.  Blocks whose o or last state is not finite somewhere say so,
// and decay_chunk.cuh takes them again one product at a time; a segment's own
// state is summed again in place.
#include <cuda.h>

#include "decay_attn.h"
#include "decay_chunk.cuh"

namespace tfb {
namespace tc {

constexpr int kC = 128;
constexpr int kMmaWarp = 8, kLoadWarp = 9, kLoaders = 96;
constexpr int kThreads = 384;
constexpr uint32_t kBlockBytes = kC * 128;  // 64 columns of a tile

template <int D>
struct Shape {
  static constexpr int kTile = kC * D * 2, kState = D * D * 2;
  static constexpr int kQ = 0, kK = kTile, kV = 2 * kTile, kMid = 3 * kTile, kLo = 4 * kTile;
  static constexpr int kSHi = 5 * kTile, kSLo = kSHi + kState, kTable = kSLo + kState;
  static constexpr int kSmem = kTable + (int)sizeof(float) * 3 * 132 + 14 * 8 + 64;
  // TMEM columns: P (also in two bfloat16 parts), O, X, E.  With D = 64, E shares X's (256 columns
  // in all); X is then read before E is issued.  That and the shared memory would let two blocks share
  // an SM, but at 80 registers a thread they spill: 8 x 4096 tokens of 16 heads of 64 take 177 us with
  // two blocks, 153 us with one, which leaves the other half of both unused.
  static constexpr int kP = 0, kO = 128, kX = 128 + D, kE = D == 64 ? kX : kX + D;
  static constexpr int kColumns = D == 64 ? 256 : 512;
  static constexpr bool kShared = D == 64;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert(8 * 32 * D <= 2 * kState, "o is staged in the state's place");
};

// Tensor maps of the roles' q, k and v: (width, tokens, heads, batch), boxes of 64 columns by 128 tokens.
struct Maps {
  CUtensorMap m[kMaxRoles][3];
  int used;
};

enum Bar { kFull, kVFull, kQK, kQS, kPV, kKFree, kKV, kDrained, kPDone, kKDone, kSReady, kXRead, kOTaken, kBars };

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

// A bounded wait; false once any wait of the block has given up.  Between the roles of a block there is
// no other kind of barrier, so that all of them come to the end of the kernel.
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

// Two neighbours as bfloat16, the first in the lower half.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
__device__ __forceinline__ float low_f32(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_f32(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }
// Their leading 8 bits as bfloat16, which they lose: the parts before the last are cut off, not
// rounded (what is cut goes into the next part exactly), which takes a byte permutation for two.
__device__ __forceinline__ uint32_t take_bf16(float& x, float& y) {
  const uint32_t r = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
  return r;
}

// Weighs 32 neighbouring values of a row of P by a g^d, d tokens from the key to the row, by steps of
// one token in registers: the products keep shared memory busy.  kDiagonal: the row's own key is
// number `own` of them; else w is the weight of the nearest.
template <bool kBack, bool kDiagonal>
__device__ __forceinline__ void weigh(uint32_t (&v)[32], float w, float a, float g, int own) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int j = kBack ? i : 31 - i;
    if (kDiagonal) {
      w = j == own ? a : w;
      const float x = __uint_as_float(v[j]) * w;
      v[j] = __float_as_uint((kBack ? j < own : j > own) ? 0.f : x);
    } else {
      v[j] = __float_as_uint(__uint_as_float(v[j]) * w);
    }
    w *= g;
  }
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int token, int head, int batch,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(token), "r"(head), "r"(batch), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map, int x, int token, int head, int batch) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(x), "r"(token),
               "r"(head), "r"(batch)
               : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    k_decay_tc(const __grid_constant__ DecayArgs a, const __grid_constant__ Maps maps, int pass) {
  using S = Shape<D>;
  using chunk::kCarried;
  using chunk::kLocal;
  using chunk::kWhole;
  extern __shared__ __align__(1024) unsigned char sm[];
  float* dec = reinterpret_cast<float*>(sm + S::kTable);
  DecayFactor* factor = reinterpret_cast<DecayFactor*>(dec + 132);
  uint64_t* bars = reinterpret_cast<uint64_t*>(factor + 132);
  chunk::Segment* seg_shared = reinterpret_cast<chunk::Segment*>(bars + 14);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(seg_shared + 1);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* odd = reinterpret_cast<int*>(tmem_slot + 2);

  const DecayRole& R = a.role[blockIdx.z];
  const int h = blockIdx.x % a.heads, unit = blockIdx.x / a.heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool want_o = R.o && pass != kLocal;
  static_assert(kBars <= 14, "barriers");

  if (a.cu && unit == a.units) {  // the rows of no sequence
    if (!R.o || pass == kLocal) return;
    const long long lo = chunk::cu_value(a, 0), hi = max(lo, chunk::cu_value(a, a.nseq));
    for (long long r = warp; r < lo + (a.tokens - hi); r += kThreads / 32) {
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
    const float ld = a.log_decay[h];
    for (int n = threadIdx.x; n <= kC; n += kThreads) {
      const double x = n ? exp((double)ld * n) : 1.0;
      dec[n] = (float)x;
      factor[n] = DecayFactor(x, ld);
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBars; ++i) {
      int count = i == kOTaken ? 8 : (i >= kPDone ? 256 : 1);
      if (i == kFull || i == kVFull) count = !maps.used ? kLoaders : (i == kFull && want_o ? 2 : 1);
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
  const long long batch = a.cu ? 0 : seg.seq;
  const int chunks = (len + kC - 1) / kC;
  // token of row 0 of chunk c (backwards it may lie before the sequence), and the rows that belong to it
  auto first_token = [&](int c) {
    return seg.start + (back ? seg.total - seg.first - (long long)(c + 1) * kC : seg.first + (long long)c * kC);
  };

  if (warp > kMmaWarp) {
    // ---------------- loads
    if (maps.used) {
      if (warp == kLoadWarp && lane == 0) {
        const CUtensorMap *mq = &maps.m[blockIdx.z][0], *mk = &maps.m[blockIdx.z][1], *mv = &maps.m[blockIdx.z][2];
        const int hq = h / R.qdiv, hk = h / R.kdiv, hv = h / R.vdiv, b = (int)batch;
        int last = -1, last_v = -1;  // chunks whose loads have been issued
        for (int c = 0; c < chunks; ++c) {
          const int token = (int)first_token(c);
          if (want_o) {
            if (c > 0 && !wait(&bars[kQS], (c - 1) & 1, gave_up)) break;
            mbar_arrive_expect_tx(&bars[kFull], S::kTile);
            for (int x = 0; x < D; x += 64) tma_load(base + S::kQ + x / 64 * kBlockBytes, mq, x, token, hq, b, &bars[kFull]);
          }
          last = c;
          if (c > 0 && !wait(&bars[kKFree], (c - 1) & 1, gave_up)) {
            if (want_o) arrive(&bars[kFull]);  // in k's place: q is on its way
            else --last;
            break;
          }
          mbar_arrive_expect_tx(&bars[kFull], S::kTile);
          for (int x = 0; x < D; x += 64) tma_load(base + S::kK + x / 64 * kBlockBytes, mk, x, token, hk, b, &bars[kFull]);
          if (c > 0 && !wait(&bars[kKV], (c - 1) & 1, gave_up)) break;
          last_v = c;
          mbar_arrive_expect_tx(&bars[kVFull], S::kTile);
          for (int x = 0; x < D; x += 64) tma_load(base + S::kV + x / 64 * kBlockBytes, mv, x, token, hv, b, &bars[kVFull]);
          if (c + 1 < chunks) {
            const int next = (int)first_token(c + 1);
            for (int x = 0; x < D; x += 64) tma_prefetch(mk, x, next, hk, b);
            for (int x = 0; x < D; x += 64) tma_prefetch(mv, x, next, hv, b);
          }
        }
        // nothing is on its way to shared memory when the block ends, however the loop did
        if (last >= 0 && !mbar_wait_bounded(&bars[kFull], last & 1)) *gave_up = 1;
        if (last_v >= 0 && !mbar_wait_bounded(&bars[kVFull], last_v & 1)) *gave_up = 1;
      }
    } else {
      const int t = threadIdx.x - 32 * kLoadWarp;
      constexpr int kVecs = D / 8;
      auto rows_in = [&](int tile, const void* p, const long long* stride, int div, int width, int c) {
        const long long token = first_token(c);
        const __nv_bfloat16* src =
            static_cast<const __nv_bfloat16*>(p) + batch * stride[0] + (long long)(h / div) * stride[2];
        const int rows = min(kC, len - c * kC), lo = back ? kC - rows : 0, hi = back ? kC : rows;
        // a thread keeps its column and walks down the rows
        const int cc = t % kVecs;
        unsigned char* to = sm + tile + cc / 8 * kBlockBytes;
#pragma unroll 4
        for (int r = t / kVecs; r < kC; r += kLoaders / kVecs) {
          const bool live = cc * 8 < width && r >= lo && r < hi;
          chunk::cp_async16(to + r * 128 + ((cc % 8) ^ (r & 7)) * 16, live ? src + (token + r) * stride[1] + cc * 8 : src,
                            live ? 16 : 0);
        }
      };
      for (int c = 0; c < chunks; ++c) {
        if (want_o) {
          if (c > 0 && !wait_warp(&bars[kQS], (c - 1) & 1, gave_up)) break;
          rows_in(S::kQ, R.q, R.qs, R.qdiv, R.wk, c);
        }
        if (c > 0 && !wait_warp(&bars[kKFree], (c - 1) & 1, gave_up)) break;
        rows_in(S::kK, R.k, R.ks, R.kdiv, R.wk, c);
        chunk::cp_commit();
        if (c > 0 && !wait_warp(&bars[kKV], (c - 1) & 1, gave_up)) break;
        rows_in(S::kV, R.v, R.vs, R.vdiv, R.wv, c);
        chunk::cp_commit();
        chunk::cp_wait<1>();
        fence_proxy_async();
        arrive(&bars[kFull]);
        chunk::cp_wait<0>();
        fence_proxy_async();
        arrive(&bars[kVFull]);
      }
      chunk::cp_wait<0>();
    }
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
          if (!wait(&bars[kVFull], ph, gave_up) || !wait(&bars[kPDone], ph, gave_up)) break;
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
        if (!want_o && (!wait(&bars[kVFull], ph, gave_up) || !wait(&bars[kSReady], ph, gave_up))) break;
        if (want_o && S::kShared && !wait(&bars[kXRead], ph, gave_up)) break;
        fence_after();
#pragma unroll
        for (int part = 0; part < 3; ++part) {
#pragma unroll
          for (int k = 0; k < kC / 16; ++k)
            mma_ss(tmem + S::kE, desc(base + (part == 0 ? S::kK : (part == 1 ? S::kMid : S::kLo)) + k * 2048, kBlockBytes),
                   desc(base + S::kV + k * 2048, kBlockBytes), kKVId, part + k > 0);
          if (part == 0) commit(&bars[kKFree]);
        }
        commit(&bars[kKV]);
      }
      commit(&bars[kDrained]);  // no product reads shared memory or writes TMEM when the block ends
      if (!mbar_wait_bounded(&bars[kDrained], 0)) *gave_up = 1;
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
            float x = st[j + 2 * e], y = st[j + 2 * e + 1];
            hi[e] = take_bf16(x, y);
            lo[e] = pack_bf16(x, y);
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
    const float g = dec[1];
    for (int c = 0; c < chunks; ++c) {
      const uint32_t ph = c & 1;
      const int rows = min(kC, len - c * kC);
      if (!wait_warp(want_o ? &bars[kQK] : &bars[kFull], ph, gave_up)) break;
      if (want_o) {
        fence_after();
        // the row's 4 pieces of 32 keys, every other one for each of the two warps that have the row
#pragma unroll 1
        for (int p = group; p < 4; p += 2) {
          const uint32_t at = tmem + S::kP + p * 32 + lanes;
          uint32_t v[32], out[32];
          const bool diagonal = p == warp % 4;
          if (diagonal || (p < warp % 4) != (back != 0)) {
            tmem_ld32(v, at);
            const float w = diagonal ? 0.f : R.a * dec[back ? p * 32 - row : row - p * 32 - 31];
            tmem_ld_wait();
            if (diagonal) {
              if (back) weigh<true, true>(v, w, R.a, g, lane);
              else weigh<false, true>(v, w, R.a, g, lane);
            } else {
              if (back) weigh<true, false>(v, w, R.a, g, 0);
              else weigh<false, false>(v, w, R.a, g, 0);
            }
          } else {  // keys behind all of this warp's rows
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x = __uint_as_float(v[2 * j]), y = __uint_as_float(v[2 * j + 1]);
            out[j] = take_bf16(x, y);
            out[16 + j] = pack_bf16(x, y);
          }
          tmem_st32(at, out);
        }
        tmem_st_wait();
        fence_before();
        arrive(&bars[kPDone]);
      }
#pragma unroll 4
      for (int i = threadIdx.x; i < S::kTile / 16; i += 256) {
        const int j = i / 8 % kC;  // rows that belong to no token are zero
        const float w = R.c * dec[max(back ? rows - (kC - 1) + j : rows - 1 - j, 0)];
        uint4* at = reinterpret_cast<uint4*>(sm + S::kK) + i;
        const uint4 k = *at;
        const uint32_t in[4] = {k.x, k.y, k.z, k.w};
        uint32_t hi[4], mid[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = low_f32(in[e]) * w, y = high_f32(in[e]) * w;
          hi[e] = take_bf16(x, y);
          mid[e] = take_bf16(x, y);
          lo[e] = pack_bf16(x, y);
        }
        *at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        reinterpret_cast<uint4*>(sm + S::kMid)[i] = make_uint4(mid[0], mid[1], mid[2], mid[3]);
        reinterpret_cast<uint4*>(sm + S::kLo)[i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async();
      arrive(&bars[kKDone]);
      if (want_o) {
        // o: row `row` of the chunk, columns c0 .. c0 + D/2
        constexpr int kW = D == 128 ? 32 : 16;
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
        const float f = R.r * dec[back ? kC - 1 - row : row + 1];
        const bool mine = back ? row >= kC - rows : row < rows;
        const long long to = batch * R.os[0] + (long long)h * R.os[2] + first_token(c) * R.os[1] + c0;
        // o goes through this warp's part of the state's place: X has been taken from it
        unsigned char* stage = sm + S::kSHi + warp * (32 * D);
        const int twist = D == 128 ? lane & 7 : lane >> 1 & 3;
        float bad = 0.f;
#pragma unroll
        for (int j = 0; j < D / 2; j += kW) {
          uint32_t o[kW], x[kW];
          __syncwarp();
          if constexpr (S::kShared) {
            tmem_ld16(o, tmem + S::kO + c0 + j + lanes);
          } else {
            tmem_ld32(o, tmem + S::kO + c0 + j + lanes);
            tmem_ld32(x, tmem + S::kX + c0 + j + lanes);
          }
          tmem_ld_wait();
          float y[kW];
#pragma unroll
          for (int e = 0; e < kW; ++e) {
            const float xe = S::kShared ? x_kept[S::kShared ? j + e : 0] : __uint_as_float(x[e]);
            y[e] = fmaf(xe, f, __uint_as_float(o[e]));
            bad = fmaf(y[e], 0.f, bad);
          }
          if (R.o_f32) {
            if (mine) {
#pragma unroll
              for (int e = 0; e < kW; e += 4)
                if (c0 + j + e < R.wv)
                  *reinterpret_cast<float4*>(static_cast<float*>(R.o) + to + row * R.os[1] + j + e) =
                      make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < kW; e += 8)
              *reinterpret_cast<uint4*>(stage + lane * D + (((j + e) / 8) ^ twist) * 16) =
                  make_uint4(pack_bf16(y[e], y[e + 1]), pack_bf16(y[e + 2], y[e + 3]), pack_bf16(y[e + 4], y[e + 5]),
                             pack_bf16(y[e + 6], y[e + 7]));
          }
        }
        strange = strange || (mine && bad != 0.f);
        if (!R.o_f32) {
          __syncwarp();
          constexpr int kPer = D / 16, kRows = 32 / kPer;  // 16-byte pieces of a row's half; rows of one access
          const int piece = lane % kPer;
          __nv_bfloat16* from_row = static_cast<__nv_bfloat16*>(R.o) + to + piece * 8;
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int r = i * kRows + lane / kPer, all = warp % 4 * 32 + r;
            const uint4 x = *reinterpret_cast<const uint4*>(stage + r * D + (piece ^ (D == 128 ? r & 7 : r >> 1 & 3)) * 16);
            if ((back ? all >= kC - rows : all < rows) && c0 + piece * 8 < R.wv)
              *reinterpret_cast<uint4*>(from_row + all * R.os[1]) = x;
          }
        }
      }
      if (!wait_warp(&bars[kKV], ph, gave_up)) break;
      fence_after();
      const DecayFactor f = factor[rows];
      __syncwarp();
#pragma unroll
      for (int j = 0; j < D / 2; j += 32) {
        uint32_t v[32];
        tmem_ld32(v, tmem + S::kE + c0 + j + lanes);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) st[j + e] = f.step(st[j + e], __uint_as_float(v[e]));
      }
      if (c + 1 < chunks) {
        if (want_o) {
          __syncwarp();
          if (lane == 0) arrive(&bars[kOTaken]);
          if (!wait_warp(&bars[kOTaken], ph, gave_up)) break;  // all warps have taken their o from there
          put_state();
        } else {
          fence_before();
          arrive(&bars[kSReady]);
        }
      }
    }
    float* to = pass == kLocal ? seg_state : (pass == kWhole && R.last ? R.last + sbase : nullptr);
    if (to && row < R.wk) {
      float bad = 0.f;
#pragma unroll
      for (int j = 0; j < D / 2; ++j)
        if (c0 + j < R.wv) {
          to[row * R.wv + c0 + j] = st[j];
          bad = fmaf(st[j], 0.f, bad);
        }
      if (bad != 0.f) {
        strange = true;
        if (pass == kLocal) {  // here, from the operands themselves, one product at a time
          const __nv_bfloat16* kh = static_cast<const __nv_bfloat16*>(R.k) + batch * R.ks[0] + (long long)(h / R.kdiv) * R.ks[2];
          const __nv_bfloat16* vh = static_cast<const __nv_bfloat16*>(R.v) + batch * R.vs[0] + (long long)(h / R.vdiv) * R.vs[2];
#pragma unroll 1
          for (int j = 0; j < D / 2 && c0 + j < R.wv; j += 8) {  // (widths are multiples of 8)
            float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
              const int rows = min(kC, len - c * kC);
              const long long token = first_token(c) + (back ? kC - rows : 0);
              float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
              for (int i = 0; i < rows; ++i) {
                const float w = dec[back ? i + 1 : rows - 1 - i], x = to_f32(kh[(token + i) * R.ks[1] + row]);
                const uint4 raw = *reinterpret_cast<const uint4*>(vh + (token + i) * R.vs[1] + c0 + j);
                const uint32_t two[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float y = e % 2 ? high_f32(two[e / 2]) : low_f32(two[e / 2]);
                  sum[e] = fmaf(R.c * (finite(x) && finite(y) ? w : above_zero(w, a.log_decay[h])) * x, y, sum[e]);
                }
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) s[e] = factor[rows].step(s[e], sum[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) to[row * R.wv + c0 + j + e] = s[e];
          }
        }
      }
    }
    if (strange) *odd = 1;
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

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (EncodeTiled) nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// (width, tokens, heads, batch) of one operand; false where no map describes it (rows shared by tokens,
// heads or sequences, or distances past a map's range).
static bool operand_map(CUtensorMap* m, const void* p, const long long* stride, int width, long long tokens, int heads,
                        long long batch) {
  const long long sizes[3] = {tokens, heads, batch}, steps[3] = {stride[1], stride[2], stride[0]};
  cuuint64_t dims[4] = {(cuuint64_t)width, 1, 1, 1}, strides[3];
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = (cuuint64_t)sizes[i];
    const long long bytes = sizes[i] > 1 ? 2 * steps[i] : 2LL * width;
    if (bytes <= 0 || bytes % 16 || bytes >= (1LL << 40) || sizes[i] < 1) return false;
    strides[i] = (cuuint64_t)bytes;
  }
  const cuuint32_t box[4] = {64, kC, 1, 1}, each[4] = {1, 1, 1, 1};
  EncodeTiled fn = encoder();
  return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, each,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
static cudaError_t run_tc(const DecayArgs& a, const Maps& maps, chunk::Pass pass, cudaStream_t st) {
  using S = Shape<D>;
  const cudaError_t e = allow_shared<k_decay_tc<D>>(S::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned units = (unsigned)a.units + (a.cu && pass != chunk::kLocal ? 1 : 0);
  k_decay_tc<D><<<dim3(units * a.heads, 1, a.roles), kThreads, S::kSmem, st>>>(a, maps, pass);
  return cudaGetLastError();
}

}  // namespace tc

cudaError_t launch_decay_tc(const DecayArgs& a, cudaStream_t st) {
  int wide = 0;
  tc::Maps maps;
  maps.used = a.cu == nullptr && a.tokens > 0;
  for (int i = 0; i < a.roles; ++i) {
    const DecayRole& r = a.role[i];
    wide = max(wide, max(r.wk, r.wv));
    maps.used = maps.used && tc::operand_map(&maps.m[i][0], r.q, r.qs, r.wk, a.tokens, a.heads / r.qdiv, a.nseq) &&
                tc::operand_map(&maps.m[i][1], r.k, r.ks, r.wk, a.tokens, a.heads / r.kdiv, a.nseq) &&
                tc::operand_map(&maps.m[i][2], r.v, r.vs, r.wv, a.tokens, a.heads / r.vdiv, a.nseq);
  }
  const chunk::Pass last = a.split ? chunk::kCarried : chunk::kWhole;
  cudaError_t e = cudaSuccess;
  if (a.split) {
    DecayArgs b = a;
    b.flags = nullptr;
    e = wide <= 64 ? tc::run_tc<64>(b, maps, chunk::kLocal, st) : tc::run_tc<128>(b, maps, chunk::kLocal, st);
    if (e == cudaSuccess) e = launch_decay_scan(a, st);
    if (e != cudaSuccess) return e;
  }
  e = wide <= 64 ? tc::run_tc<64>(a, maps, last, st) : tc::run_tc<128>(a, maps, last, st);
  if (e != cudaSuccess) return e;
  return launch_decay_flagged_bf16(a, last, st);  // the blocks that said so, and no others
}

}  // namespace tfb
