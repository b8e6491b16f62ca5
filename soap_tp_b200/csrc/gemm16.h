// Products of bf16 or fp16 matrices on CTA pairs (gemm16.cu), and what becomes of their tiles.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace soapb200 {

// A matrix of 16-bit elements, `ld` elements between rows.  As an operand either K runs along its rows ([M][K], `k_major`) or
// M (N) does ([K][M]).  Base 16-byte aligned, `ld` a multiple of 8.
struct Matrix16 {
  const void* data;
  int64_t ld;
  bool k_major;
};

enum Gemm16Epilogue : int {
  kLogitStatistics = 0,     // largest logit and sum of exponentials per row and 128 columns, and the logit of each row's target
  kLogitGradient = 1,       // softmax minus target, times the row's factor, as a 16-bit matrix
  kStore16 = 2,             // the product itself
};

constexpr int kLogitPart = 128;      // columns that share one partial maximum and sum

struct Gemm16Problem {
  int M, N, K;
  // logits: row i is a token, column j a word; the token's target counts from this matrix's first column
  const int64_t* targets;
  int64_t first_word;
  float2* parts;            // [ceil(N / kLogitPart)][M]: largest logit, sum of exp(logit - largest)
  float* picked;            // [M]: the target's logit, written where the target is a column
  const float* lse;         // [M]
  const float* factor;      // [M]
  // kLogitGradient, kStore16: 16-bit result [M][ldc]
  void* C;
  int64_t ldc;
  // kStore16: alpha * (product + accumulator); without `C` the sum goes back into the accumulator [M][ld_accumulator]
  const float* alpha;       // on the device; null: 1
  float* accumulator;
  int64_t ld_accumulator;
  bool add;                 // whether the accumulator holds something
};

// acc[m, n] = sum_k A(m, k) B(n, k) and its epilogue.  `bf16`: both operands and the 16-bit result are bf16, otherwise fp16.
void gemm16(Gemm16Epilogue epilogue, bool bf16, const Matrix16& a, const Matrix16& b, const Gemm16Problem& problem, int* status,
            cudaStream_t stream);

}  // namespace soapb200
