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
  kLogitStatistics = 0,     // largest logit and sum of exponentials, but for the row's target, per row and 64 columns
  kLogitExponential = 1,    // the same, and the exponentials themselves, relative to the largest of their part, times 2^15 in fp16
  kLogitGradient = 2,       // softmax minus target, times the row's factor, as a 16-bit matrix
  kStore16 = 3,             // the product itself
};

constexpr int kLogitPart = 64;      // columns that share one partial maximum and sum

struct Gemm16Problem {
  int M, N, K;
  // How many tokens there are is known on the device: `*count` in all, of which this product starts with number `first`.  They are
  // A's rows (logits, and kStore16 with A K-major), or K.  Null: M and K hold as they are.
  const int* count;
  int first;
  // logits: row i is a token, column j a word
  const int* targets;       // [M]: the column that is the token's target; negative where none of them is
  float2* parts;            // [ceil(N / kLogitPart)][ld_parts]: largest logit, sum of exp(logit - largest) over all but the target
  int64_t ld_parts;
  int drain;                // of K, a multiple of 64: the accumulator is drained into fp32 sums that often;
  int drain_few, few;       // drain_few where there are at most `few` tokens in all (`count`)
  const float* lse;         // [M]
  const float* loss;        // [M]: lse - the target's logit
  const float* factor;      // [M]
  // 16-bit result [M][ldc]
  void* C;
  int64_t ldc;
  // What is left of the gradient's values when they are rounded, in 16 bits `second` columns further on, zeros up to the next multiple of 64
  // words in both; as A (kStore16) both terms are multiplied by B.  0: there is none.
  int64_t second;
  // kStore16: alpha * (product + accumulator), row i of it in row where[i] of C; without `C` the sum goes back into the accumulator
  const int* where;         // null: rows stay where they are
  const float* alpha;       // on the device; null: 1
  float* accumulator;       // [M][ld_accumulator]
  int64_t ld_accumulator;
  bool add;                 // whether the accumulator holds something
  // kStore16: where tiles whose K is split leave their parts (kSplitScratch floats), and how many have (kSplitCounters zeros, left as
  // zeros); null: no tile is split
  float* split_parts;
  int* split_counters;
};
constexpr int kSplitUnits = 80;                       // parts of tiles at most: one for each CTA pair of the device
constexpr int64_t kSplitScratch = kSplitUnits * int64_t{256} * 256;
constexpr int kSplitCounters = kSplitUnits * 16;

// The hidden states in two places: the tokens that count one after another, and all of them (`all`, of `tokens` rows), which is where
// they are read from when every token counts.
struct Hidden16 {
  Matrix16 packed, all;
  int tokens;
};

// acc[m, n] = sum_k A(m, k) B(n, k) and its epilogue.  `bf16`: both operands and the 16-bit result are bf16, otherwise fp16.
// `hidden` (or null) stands for the operand that the tokens' states are: A of logits, B of kStore16 otherwise.
void gemm16(Gemm16Epilogue epilogue, bool bf16, const Matrix16& a, const Matrix16& b, const Gemm16Problem& problem, int* status,
            cudaStream_t stream, const Hidden16* hidden = nullptr);

}  // namespace soapb200
