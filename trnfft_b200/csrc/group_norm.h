// Internal interface of the group normalisation kernels (group_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "decay_attn.h"

namespace tfb {

enum Activation { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// x, y, dy, dx: (batch, spots, channels) contiguous; weight, bias (may be
// null), dw, db: (channels) float32; mean, rstd: (batch, groups) float32.
struct GroupNormArgs {
  const void* x;
  const void* dy;   // backward
  void* y;          // forward: y, backward: dx
  const float* weight;
  const float* bias;
  float* mean;
  float* rstd;
  float* dw;
  float* db;
  float* work;
  long long batch, spots;
  int channels, groups;
  float eps;
  int act;
};

int64_t group_norm_work_bytes(ElemType t, const GroupNormArgs& a, bool backward);
cudaError_t launch_group_norm(ElemType t, const GroupNormArgs& a, cudaStream_t st);
cudaError_t launch_group_norm_backward(ElemType t, const GroupNormArgs& a, cudaStream_t st);

}  // namespace tfb
