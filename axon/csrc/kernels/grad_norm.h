// Launch interface of the multi-tensor gradient norm (grad_norm.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace axon {

// Up to kGradTensors tensors of one type, passed by value in the kernel's
// arguments (under 4 KiB): a call captured into a graph then owns its table,
// and no copy to the device is needed.
constexpr int kGradTensors = 192;
constexpr int64_t kGradChunk = 16384;  // values that a block takes at a time

struct GradTable {
  void* ptr[kGradTensors];
  int64_t n[kGradTensors];
  int32_t first[kGradTensors + 1];  // chunks before this tensor's
  int32_t count;
};

// Blocks (and partial sums) that the norm of a table takes.
int grad_norm_blocks(const GradTable& t);
// partial[block] = sum of |g| (type 1), g^2 (type 2) or max |g| (type 0)
// over the block's chunks.
void launch_grad_partial(const GradTable& t, int dtype, int type,
                         double* partial, hipStream_t stream);
// out[0] = the norm, out[1] = min(1, max_norm / (norm + 1e-6)).
void launch_grad_finish(const double* partial, int blocks, int type,
                        float max_norm, float* out, hipStream_t stream);
// g *= *factor; nothing is read or written where *factor is 1.
void launch_grad_scale(const GradTable& t, int dtype, const float* factor,
                       hipStream_t stream);
// Both in one launch for each table, where all partial sums are few (each
// block joins them): out as above, written by each of the launches alike.
bool grad_clip_folds(int blocks);
void launch_grad_clip(const GradTable& t, int dtype, int type,
                      const double* partial, int blocks, float max_norm,
                      float* out, hipStream_t stream);

}  // namespace axon
