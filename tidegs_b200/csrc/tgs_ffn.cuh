// Shared by the two implementations of the gated feed-forward block.
#pragma once

#include "tgs_common.cuh"
#include "tgs_vec.cuh"

namespace tgs {

struct FfnParams {
  const void *x, *dy, *wg, *wu, *wd;
  void* y;  // dx in the backward
  void *dwg, *dwu, *dwd;
  float* scratch;
  int32_t* err;
  int64_t n, x_stride, dy_stride;
  int d, h, o;
};

// bf16 on the tensor cores (tgs_ffn_tc.cu).
int ffn_tc_forward(const FfnParams& p, cudaStream_t s);
int64_t ffn_tc_scratch_floats(int64_t n, int d, int h, int o, bool backward);
int ffn_tc_backward(const FfnParams& p, cudaStream_t s);

// fp32 on the tensor cores (tgs_ffn_tc32.cu): Y or dX, and partial weights'
// gradients in `tc32_slices` slices [dWg [H, D] | dWu [H, D] | dWd^T [H, O]] at
// the start of the scratch.
int ffn_tc32_run(const FfnParams& p, bool backward, cudaStream_t s);
int tc32_slices(int64_t n, int d, int h, int o);
int64_t tc32_scratch_floats(int64_t n, int d, int h, int o, bool backward);

}  // namespace tgs
