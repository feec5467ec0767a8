// Global norm of a list of gradient tensors, and their scaling to a largest norm.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace paralia {

// Blocks of the norm kernel at most: three of 512 threads for each of 148 SMs.
constexpr int GL_NORM_BLOCKS = 148 * 3;
// Tensors whose description fits into the parameters of one launch. A longer list takes more.
constexpr int GL_MAX_TENSORS = 960;
// Elements of a unit, the grain in which a list is dealt out to the blocks.
constexpr int GL_UNIT = 2048;

// One tensor of a launch. Its first unit also holds the `head` elements in front of the first
// 16-byte boundary.
struct GradEntry {
  const void* src;
  void* dst;
  int64_t n;
  int32_t unit0;      // number of the tensor's first unit in the list
  uint8_t src_type;   // PARALIA_F32 / F16 / BF16
  uint8_t dst_type;
  uint8_t head;
  uint8_t flags;      // GL_*
};
constexpr uint8_t GL_DST_VEC = 1;    // groups of eight lie on 16-byte boundaries in dst too
constexpr uint8_t GL_IN_PLACE = 2;   // dst is src, of the same type

struct GradList {
  int count;                 // tensors with elements
  GradEntry* entries;        // unit0 counts over the whole list
  int64_t units;
  uintptr_t lo, hi;          // all tensors and outputs lie between these addresses
};

// Number of partial sums the norm of a list of `count` tensors may leave at most.
int64_t grad_partials(int64_t count);

// partials[0 .. *used) <- sums of squares.
cudaError_t launch_grad_sumsq(const GradList& l, double* partials, int* used, cudaStream_t stream);
// *sumsq <- sum of the partials, *norm <- its square root (either may be null).
cudaError_t launch_grad_norm_final(const double* partials, int used, double* sumsq, float* norm, cudaStream_t stream);
// dst <- src * (norm > max_norm ? max_norm / norm : 1), norm^2 = sum of the `used` partials;
// writes *sumsq and *norm too (either may be null). May put the sum in partials[0] if used > 1.
cudaError_t launch_grad_scale(const GradList& l, double* partials, int used, float max_norm, double* sumsq,
                              float* norm, cudaStream_t stream);

}  // namespace paralia
