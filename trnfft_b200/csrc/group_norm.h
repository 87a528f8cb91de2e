// Internal interface of the group normalisation kernels (group_norm.cu,
// group_norm_bwd.cu).
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
  void* y;          // forward: y, backward: dx (may be null)
  const float* weight;
  const float* bias;
  float* mean;
  float* rstd;
  float* dw;
  float* db;
  void* work;
  long long batch, spots;
  int channels, groups;
  float eps;
  int act;
};

// How a call is run; it depends on the sizes, the element size and the alignment alone.
struct GroupNormPlan {
  enum Kind { kSmall, kSplit, kAny } kind;
  int vec;         // elements of one access
  // kSmall: one group of `lanes` threads per (sample, group), nv accesses each
  int lanes, nv;
  // kSplit: `parts` blocks of `part_rows` rows per sample, `slots` rows of `cols` threads per block
  int parts, part_rows, slots, cols, tiles, threads, smem;
  int stage_rows;      // parts > 1: rows of a buffer of a block's stream; 0: rows are loaded by their threads
  int sample_buffers;  // parts == 1: buffers of a block's stream of samples; 0: rows are loaded by their threads
  int glanes, planes;  // threads that join a group's sets within a block, across the parts
  int grid;
  // work area, in bytes from its start (all 16-byte aligned); the parts' sets come first
  long long off_result, off_channels, channel_rows, off_sync, bytes;
};

constexpr int kNormThreads = 256;
constexpr int kMaxSplitSmem = 200 * 1024;
constexpr int kSms = 148;
constexpr int kStages = 4, kStreamBytes = 64 * 1024;  // buffers of a block's stream of rows
// Rows of `bytes` that a thread of kSplit has on their way at a time.
constexpr int rows_ahead(int bytes) { return 64 / bytes < 4 ? 64 / bytes : 4; }

// align: what all of x, y and dy are multiples of (16, 8, 4 or 2 bytes)
GroupNormPlan plan_group_norm(ElemType t, const GroupNormArgs& a, bool backward, int align);
int group_norm_align(const GroupNormArgs& a);
int64_t group_norm_work_bytes(ElemType t, const GroupNormArgs& a, bool backward);
cudaError_t launch_group_norm(ElemType t, const GroupNormArgs& a, cudaStream_t st);
cudaError_t launch_group_norm_backward(ElemType t, const GroupNormArgs& a, cudaStream_t st);

}  // namespace tfb
