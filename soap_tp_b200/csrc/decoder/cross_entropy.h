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
  // The tokens that count, one after another: how many there are, which token each is, the column that is its target here (kElsewhere: another
  // rank's, kUnknown: none's), and their hidden states, unless all tokens count.
  int* count;               // [1]
  int* where;               // [tokens]
  int* column;              // [tokens]
  int* split_counters;      // [kSplitCounters], cleared with them
  Matrix16 packed;          // [tokens][depth]
};
constexpr int kElsewhere = -1, kUnknown = -2;

// Fills count, where, column, split_counters and packed; with `d_hidden`, clears the rows of the tokens that do not count.
// With `factor` (bf16, sum or mean) what head_factors leaves for a gradient of one as well.
void head_prepare(const HeadProblem& p, void* d_hidden, int64_t ld_hidden, LossReduction reduction, float* factor, float* alpha, cudaStream_t stream);

// What the loss and its gradient need of each token that counts, by its number among them.
struct TokenResults {
  float* lse;               // log sum_j exp(l_ij)
  float* loss;              // lse - l_i,t_i
};

// For tokens first .. first + rows of those that count.  `whole`: this rank has all words, and lse and loss are filled.  Otherwise `lse` gets that of
// this rank's words but for the target, and `loss` the target's logit where this rank has it and 0 elsewhere; joined over the
// ranks, rest and logit, they give loss = log(1 + exp(rest - logit)) and lse = logit + loss.
// `parts`: ceil(words / kLogitPart) x rows pairs.  With `logits` (bf16) the exponentials stay there as fp16, 2^15 times those relative to the
// largest of their part.
struct LogitRows {
  int first, rows;
  void* logits;
  int64_t ld_logits;
  float2* parts;
  int64_t second;           // columns from the logits' gradient to what its rounding left, or 0 (Gemm16Problem)
};
// Up to so many tokens the logits' gradient has two terms: there the roundings of a few large values, a target's above all, are most of a
// gradient's error, where over many tokens they average out.  (15 tokens x 228 x 2011: 0.0029 of the gradient, 0.0016 with two; 8192 x
// 4096 x 128256: 0.0019.)  The two products that read it have twice the K: with gradients 1 to 64 tokens x 4096 x 128256 take 955 us for 813, 128
// tokens 1000 for 795, 256 tokens 1200 to 1240 for 930 to 950.  It goes by all tokens of a call, padding included: where the second term lies
// is settled before the device counts.
constexpr int kFewTokens = 256;
void head_statistics(const HeadProblem& p, const LogitRows& r, const TokenResults& t, bool whole, int* status, cudaStream_t stream);

// The losses by token; 0 for tokens that do not count, NaN for targets outside the vocabulary.  With a reduction one number.
void head_losses(const HeadProblem& p, const TokenResults& t, LossReduction reduction, float* loss, cudaStream_t stream);

// What the gradient of the loss multiplies the row of a token that counts by: factor[i] * *alpha.  `grad_loss` has one value per token,
// or one.
void head_factors(const HeadProblem& p, LossReduction reduction, const float* grad_loss, float* factor, float* alpha, cudaStream_t stream);

// The exponentials that head_statistics left become the logits' gradient, factor (exp(l - lse) - [target]).
void head_rescale(const HeadProblem& p, const LogitRows& r, const TokenResults& t, const float* factor, cudaStream_t stream);
// The logits' gradient from the logits anew.
void head_logit_gradient(const HeadProblem& p, const LogitRows& r, const TokenResults& t, const float* factor, int* status, cudaStream_t stream);

// Gradients of the hidden states and the weight (either may be null) from the logits' gradient of these rows.  The weight's is summed over
// the turns in `sum`, words x ld_sum floats, where one does not take all tokens.
struct HeadGradients {
  void* hidden;
  int64_t ld_hidden;
  void* weight;
  int64_t ld_weight;
  float* sum;
  int64_t ld_sum;
  float* split_parts;       // kSplitScratch floats
};
void head_gradients(const HeadProblem& p, const LogitRows& r, const float* alpha, const HeadGradients& g, int* status, cudaStream_t stream);

// Two contiguous bf16 matrices times *factor, in place; nothing where it is one.
void scale_gradients(const float* factor, void* a, int64_t count_a, void* b, int64_t count_b, cudaStream_t stream);

}  // namespace soapb200
