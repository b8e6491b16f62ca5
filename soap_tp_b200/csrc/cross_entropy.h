// Softmax cross entropy of hidden @ weight^T without the logits (cross_entropy.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm16.h"

namespace soapb200 {

enum LossReduction : int { kLossNone = 0, kLossSum = 1, kLossMean = 2 };

// Hidden states [tokens][depth], this rank's words [words][depth], and where its first word stands in the whole vocabulary.
struct HeadProblem {
  Matrix16 hidden, weight;
  int tokens, depth, words;
  bool bf16;
  const int64_t* targets;
  int64_t ignore_index, first_word, vocabulary;
};

// lse[i] = log sum_j exp(l_ij) over this rank's words, picked[i] = l_i,t_i where the target is one of them and 0 elsewhere.
// `parts`: ceil(words / 128) x tokens pairs.
void head_statistics(const HeadProblem& p, float2* parts, float* lse, float* picked, int* status, cudaStream_t stream);

// losses[i] = lse - picked; 0 for tokens that do not count, NaN for targets outside the vocabulary.  With a reduction the
// result goes to `loss`, and how many tokens count to `counted`.
void head_losses(const HeadProblem& p, const float* lse, const float* picked, LossReduction reduction, float* loss, float* counted,
                 cudaStream_t stream);

// What the gradient of the loss multiplies row i by: factor[i] * *alpha.  `grad_loss` has one value per token, or one.
void head_factors(const HeadProblem& p, LossReduction reduction, const float* grad_loss, const float* counted, float* factor,
                  float* alpha, cudaStream_t stream);

// Gradients of the hidden states and the weight (either may be null), `rows` tokens at a time through `logits`, rows x pitch 16-bit values.
// `sum`: words x ld_sum floats, needed where the tokens take more than one turn.
struct HeadGradients {
  void* hidden;
  int64_t ld_hidden;
  void* weight;
  int64_t ld_weight;
  void* logits;
  int64_t ld_logits;
  int rows;
  float* sum;
  int64_t ld_sum;
};
void head_gradients(const HeadProblem& p, const float* lse, const float* factor, const float* alpha, const HeadGradients& g, int* status,
                    cudaStream_t stream);

}  // namespace soapb200
