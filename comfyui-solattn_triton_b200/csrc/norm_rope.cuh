// Head norms with the position rotation (solb200_qk_norm_rope and its gradient): the
// parameters shared by the kernels (norm_rope.cu) and the entry points (layer_api.cu).
#pragma once

#include <stdint.h>

#include <cuda_runtime.h>

namespace solb200 {

enum { kDtypeBF16 = 0, kDtypeF16 = 1, kDtypeF32 = 2 };

// One of the two tensors (q or k) of a call: [B, T, heads, D], element strides {batch, token,
// head}, head_dim contiguous; outputs and gradients are dense.
struct RopeTensor {
  const void* x;
  const void* dy;       // backward only: the gradient of the output
  void* out;            // forward: the output; backward: the gradient of x
  const void* weight;   // [D]
  void* dweight;        // [D], backward only
  int64_t xs[3], dys[3];
  int heads;
};

struct RopeParams {
  RopeTensor t[2];      // q, k
  const float *cos, *sin;
  int64_t ts[2];        // table strides {batch, token}; a row holds R / 2 floats
  int B, T, D, R;
  float eps;
  int rows[2];          // B * T * heads
  int ctas[2];          // CTAs that walk q's rows, then those that walk k's
  float* partial;       // backward: [ctas[0] + ctas[1], D] sums of the weight gradients
};

cudaError_t launch_norm_rope(RopeParams p, int dtype, int wdtype, bool interleaved, cudaStream_t st);
cudaError_t launch_norm_rope_backward(RopeParams p, int dtype, int wdtype, bool interleaved, cudaStream_t st);
// Most CTAs that the backward pass of any element type takes for this geometry (the lines of
// RopeParams::partial)
int norm_rope_backward_ctas(int64_t B, int64_t T, int64_t H, int64_t Hk, int D);

}  // namespace solb200
