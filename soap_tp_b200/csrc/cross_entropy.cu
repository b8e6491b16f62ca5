// Softmax cross entropy of hidden @ weight^T and its gradients, without ever holding the logits of all tokens.
//
//   l_ij = h_i . w_j     lse_i = log sum_j exp l_ij     loss_i = lse_i - l_i,t_i
//   d_ij = f_i (exp(l_ij - lse_i) - [j = t_i])          dH = alpha D W      dW = alpha D^T H
//
// Forward: one product (gemm16.cu) whose epilogue leaves, per token and 128 words, the largest logit and the sum of
// exponentials relative to it; head_join_kernel joins these parts.  Backward: the logits once more, this time leaving D in 16 bits
// for a bounded number of tokens at a time, then the two products that read D in both directions.
//
// What multiplies a row is split into a factor in [-1, 1] that goes into D and a number on the device that the products' epilogues
// multiply by: mean's 1 / count never touches D, where -1 (the target of a token that the model does not know) is exact, and
// fp16 keeps probabilities down to 2^-29 as normal numbers (D is stored times 2^15 there).
#include <cuda_runtime.h>

#include <stdexcept>
#include <string>

#include "cross_entropy.h"
#include "launch_util.h"

namespace soapb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kJoinSlices = 16;
constexpr int kSingleThreads = 1024;

void check(cudaError_t err, const char* what) {
  if (err != cudaSuccess) throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(err));
}

// 32 tokens a block, lanes along tokens, the parts dealt to 16 warps and joined in a fixed order.
__global__ void __launch_bounds__(32 * kJoinSlices)
head_join_kernel(const float2* __restrict__ parts, int count, int tokens, const int64_t* __restrict__ targets, int64_t first_word, int words,
                 float* __restrict__ lse, float* __restrict__ picked) {
  __shared__ float2 shared[kJoinSlices][32];
  wait_for_predecessor();
  let_successor_start();
  const int token = blockIdx.x * 32 + threadIdx.x;
  float largest = -INFINITY, sum = 0.f;
  if (token < tokens) {
#pragma unroll 4
    for (int i = threadIdx.y; i < count; i += kJoinSlices) {
      const float2 part = parts[static_cast<int64_t>(i) * tokens + token];
      const float most = fmaxf(largest, part.x);
      const float base = most == -INFINITY ? 0.f : most;
      sum = sum * exp2f((largest - base) * kLog2e) + part.y * exp2f((part.x - base) * kLog2e);
      largest = most;
    }
  }
  shared[threadIdx.y][threadIdx.x] = make_float2(largest, sum);
  __syncthreads();
  if (threadIdx.y == 0 && token < tokens) {
#pragma unroll
    for (int s = 1; s < kJoinSlices; ++s) {
      const float2 part = shared[s][threadIdx.x];
      const float most = fmaxf(largest, part.x);
      const float base = most == -INFINITY ? 0.f : most;
      sum = sum * exp2f((largest - base) * kLog2e) + part.y * exp2f((part.x - base) * kLog2e);
      largest = most;
    }
    lse[token] = logf(sum) + (largest == -INFINITY ? 0.f : largest);
    const int64_t target = targets[token] - first_word;
    if (target < 0 || target >= words) picked[token] = 0.f;
  }
}

struct Targets {
  const int64_t* at;
  int64_t ignored, vocabulary;
  __device__ __forceinline__ bool counts(int i) const { return at[i] != ignored; }
  __device__ __forceinline__ bool known(int i) const { return at[i] >= 0 && at[i] < vocabulary; }
};

__global__ void head_token_losses_kernel(Targets targets, int tokens, const float* __restrict__ lse, const float* __restrict__ picked,
                                         float* __restrict__ losses) {
  wait_for_predecessor();
  let_successor_start();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < tokens) losses[i] = !targets.counts(i) ? 0.f : targets.known(i) ? lse[i] - picked[i] : nanf("");
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = shared[threadIdx.x];
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (threadIdx.x == 0) shared[0] = v;
  }
  __syncthreads();
  v = shared[0];
  __syncthreads();
  return v;
}

// One block: the sum does not depend on the order in which blocks end.
__global__ void __launch_bounds__(kSingleThreads)
head_reduced_loss_kernel(Targets targets, int tokens, const float* __restrict__ lse, const float* __restrict__ picked, bool mean,
                         float* __restrict__ loss, float* __restrict__ counted) {
  __shared__ double shared[32];
  wait_for_predecessor();
  let_successor_start();
  double sum = 0.0, count = 0.0;
  for (int i = threadIdx.x; i < tokens; i += kSingleThreads) {
    if (targets.counts(i)) {
      count += 1.0;
      sum += targets.known(i) ? lse[i] - picked[i] : nanf("");
    }
  }
  auto add = [](double a, double b) { return a + b; };
  sum = block_reduce(sum, add, shared);
  count = block_reduce(count, add, shared);
  if (threadIdx.x == 0) {
    *loss = static_cast<float>(mean ? (count > 0.0 ? sum / count : 0.0) : sum);
    *counted = static_cast<float>(count);
  }
}

__global__ void __launch_bounds__(kSingleThreads)
head_factors_kernel(Targets targets, int tokens, int reduction, float stored, const float* __restrict__ grad_loss,
                    const float* __restrict__ counted, float* __restrict__ factor, float* __restrict__ alpha) {
  __shared__ float shared[32];
  wait_for_predecessor();
  let_successor_start();
  float common = 1.f, relative = 1.f;      // the gradient is common * factor; factor = stored * relative * (the row's own)
  if (reduction == kLossNone) {
    float most = 0.f;
    for (int i = threadIdx.x; i < tokens; i += kSingleThreads)
      if (targets.counts(i)) most = fmaxf(most, fabsf(grad_loss[i]));
    most = block_reduce(most, [](float a, float b) { return fmaxf(a, b); }, shared);
    // a power of two, so that no factor is rounded; none where the largest is zero or not finite
    if (most > 0.f && most < INFINITY) {
      const int exponent = min(120, max(-120, ilogbf(most) + 1));
      common = ldexpf(1.f, exponent);
      relative = ldexpf(1.f, -exponent);
    }
  } else {
    common = *grad_loss;
    if (reduction == kLossMean) common = *counted > 0.f ? common / *counted : 0.f;
  }
  for (int i = threadIdx.x; i < tokens; i += kSingleThreads) {
    const float own = reduction == kLossNone ? grad_loss[i] : 1.f;
    factor[i] = !targets.counts(i) ? 0.f : targets.known(i) ? stored * relative * own : nanf("");
  }
  if (threadIdx.x == 0) *alpha = common / stored;
}

Targets targets_of(const HeadProblem& p) { return Targets{p.targets, p.ignore_index, p.vocabulary}; }

}  // namespace

void head_statistics(const HeadProblem& p, float2* parts, float* lse, float* picked, int* status, cudaStream_t stream) {
  Gemm16Problem g{};
  g.M = p.tokens; g.N = p.words; g.K = p.depth;
  g.targets = p.targets; g.first_word = p.first_word;
  g.parts = parts; g.picked = picked;
  gemm16(kLogitStatistics, p.bf16, p.hidden, p.weight, g, status, stream);
  check(launch_dependent(head_join_kernel, dim3((p.tokens + 31) / 32), dim3(32, kJoinSlices), 0, stream, parts,
                         (p.words + kLogitPart - 1) / kLogitPart, p.tokens, p.targets, p.first_word, p.words, lse, picked),
        "head_join");
}

void head_losses(const HeadProblem& p, const float* lse, const float* picked, LossReduction reduction, float* loss, float* counted,
                 cudaStream_t stream) {
  if (reduction == kLossNone)
    check(launch_dependent(head_token_losses_kernel, dim3((p.tokens + 255) / 256), dim3(256), 0, stream, targets_of(p), p.tokens, lse,
                           picked, loss),
          "head_token_losses");
  else
    check(launch_dependent(head_reduced_loss_kernel, dim3(1), dim3(kSingleThreads), 0, stream, targets_of(p), p.tokens, lse, picked,
                           reduction == kLossMean, loss, counted),
          "head_reduced_loss");
}

void head_factors(const HeadProblem& p, LossReduction reduction, const float* grad_loss, const float* counted, float* factor,
                  float* alpha, cudaStream_t stream) {
  check(launch_dependent(head_factors_kernel, dim3(1), dim3(kSingleThreads), 0, stream, targets_of(p), p.tokens,
                         static_cast<int>(reduction), p.bf16 ? 1.f : 32768.f, grad_loss, counted, factor, alpha),
        "head_factors");
}

void head_gradients(const HeadProblem& p, const float* lse, const float* factor, const float* alpha, const HeadGradients& out, int* status,
                    cudaStream_t stream) {
  if (out.rows < 1) throw std::invalid_argument("head_gradients: no room for logits");
  if (out.weight && p.tokens > out.rows && !out.sum) throw std::invalid_argument("head_gradients: several turns need a sum");
  for (int first = 0; first < p.tokens; first += out.rows) {
    const int rows = p.tokens - first < out.rows ? p.tokens - first : out.rows;
    const Matrix16 hidden{static_cast<const uint16_t*>(p.hidden.data) + first * p.hidden.ld, p.hidden.ld, true};
    Gemm16Problem g{};
    g.M = rows; g.N = p.words; g.K = p.depth;
    g.targets = p.targets + first; g.first_word = p.first_word;
    g.lse = lse + first; g.factor = factor + first;
    g.C = out.logits; g.ldc = out.ld_logits;
    gemm16(kLogitGradient, p.bf16, hidden, p.weight, g, status, stream);
    if (out.hidden) {
      Gemm16Problem d{};
      d.M = rows; d.N = p.depth; d.K = p.words;
      d.C = static_cast<uint16_t*>(out.hidden) + first * out.ld_hidden; d.ldc = out.ld_hidden;
      d.alpha = alpha;
      gemm16(kStore16, p.bf16, Matrix16{out.logits, out.ld_logits, true}, Matrix16{p.weight.data, p.weight.ld, false}, d, status, stream);
    }
    if (out.weight) {
      Gemm16Problem d{};
      d.M = p.words; d.N = p.depth; d.K = rows;
      d.alpha = alpha;
      d.accumulator = out.sum; d.ld_accumulator = out.ld_sum; d.add = first > 0;
      if (first + rows == p.tokens) {
        d.C = out.weight; d.ldc = out.ld_weight;
      }
      gemm16(kStore16, p.bf16, Matrix16{out.logits, out.ld_logits, false}, Matrix16{hidden.data, hidden.ld, false}, d, status, stream);
    }
  }
}

}  // namespace soapb200
