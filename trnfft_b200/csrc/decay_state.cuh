// The factor of a decayed state, shared by the kernels of decayed linear attention.
#pragma once

#include <cuda_runtime.h>
#include <math.h>

namespace tfb {

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// A power of g as the factor of a value that is not finite: above 0 where g is, however small.
__device__ __forceinline__ float above_zero(float power, float log_decay) {
  return log_decay > -INFINITY ? fmaxf(power, 1e-30f) : power;
}

// g as the sum hi + lo, of a state's step s -> s hi + (s lo + x).  Both parts are above 0 where g is: with
// a lo of 0 or of the other sign an infinite s would become NaN.  The smallest float32 in the place of
// 0 changes no finite s, half a step of which is more.
struct DecayFactor {
  float hi, lo;
  __device__ __forceinline__ DecayFactor(double g, float log_decay) {
    hi = __double2float_rz(g);
    const float rest = (float)(g - (double)hi);
    const float least = __uint_as_float(1u);
    const bool above = log_decay > -INFINITY;  // (not of NaN, which both parts keep)
    hi = above ? fmaxf(hi, least) : hi;
    lo = above ? fmaxf(rest, least) : rest;  // (of an infinite g the rest is NaN, and lo the least)
  }
  __device__ __forceinline__ float step(float s, float x) const { return fmaf(s, hi, fmaf(s, lo, x)); }
};

}  // namespace tfb
