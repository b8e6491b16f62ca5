// Norms before and after a block, its gate and residual scale, in one pass (residual_norm.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "activation8.h"

namespace soapb200 {

// h = x + scale * gate * branch', branch' = branch or norm(branch) * branch_weight; y = norm(h) * weight.
struct NormProblem {
  int type;                       // of x, branch and the results (ValueType)
  int vector_type;                // of weight, branch_weight and gate: `type` or fp32
  int64_t rows;
  int dim;
  float scale, eps;
  Rows x;
  Rows branch;                    // null: h = x
  const void *weight, *branch_weight, *gate;      // any may be null
  float *rms, *branch_rms;        // [rows]: 1 / sqrt(mean of squares + eps), of h and of the branch
  int* status;
};

// h (null: not written) and y (null where there is no weight), rows `ld` elements apart.
void residual_norm_forward(const NormProblem& p, void* h, void* y, int64_t ld, cudaStream_t stream);

// Gradients.  `grad_h`, `grad_y`, d_x and d_branch may be null.  `partials`: blocks x 2 x dim floats,
// of which d_weight, d_branch_weight and d_gate (vector_type; any may be null) are made.
struct NormGradients {
  Rows grad_h, grad_y;
  void *d_x, *d_branch;
  int64_t ld;
  float* partials;
  int blocks;
  void *d_weight, *d_branch_weight, *d_gate;
};
void residual_norm_backward(const NormProblem& p, const NormGradients& g, cudaStream_t stream);
// How many blocks a backward pass uses (`g` but for partials and blocks).
int residual_norm_blocks(const NormProblem& p, const NormGradients& g);

}  // namespace soapb200
