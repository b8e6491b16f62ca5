// Softmax cross entropy of hidden @ weight^T and its gradients, without ever holding the logits of all tokens.
//
//   l_ij = h_i . w_j     lse_i = log sum_j exp l_ij     loss_i = lse_i - l_i,t_i
//   d_ij = f_i (exp(l_ij - lse_i) - [j = t_i])          dH = alpha D W      dW = alpha D^T H
//
// Tokens that do not count are left out from the start: the others' numbers, targets and hidden states are put one after another, every
// product runs over those alone (their number stays on the device), and what the padding holds, NaN included, reaches nothing.
//
// The loss: one product (gemm16.cu) whose epilogue leaves, per token and 64 words, the largest logit and the sum of exponentials relative to
// it of all words but the target; head_join_kernel joins these parts to r = log sum over those words.  The target's logit t comes from an fp32
// product of its own, and loss = log(1 + exp(r - t)), lse = t + loss, p_t - 1 = exp(-loss) - 1: a token that the model knows has a loss of 1e-4 and
// less, of which a difference of lse and t in fp32 would leave two digits.  D goes through memory in 16 bits for a bounded number of tokens at a time, then
// two products read it in both directions.  It comes about in one of two ways:
//   * bf16 and one gradient of the loss for all tokens (mean, sum): the first product leaves the exponentials as well (in fp16 times 2^15, which
//     rounds them an eighth as much as D is rounded then, or to 2^-40 of the largest of their 64 words), one pass over them makes D of them
//     once lse is known, and the gradients come with the loss, 6 N V K operations for N tokens.  The pass moves 4 N V bytes: 44 us at
//     4096 x 4096 x 16032, where a product takes 357 to 373.
//   * fp16, whose gradients want the loss's scale before they are rounded, a gradient for each token, or a second backward pass: the logits
//     are computed again once these are known, 8 N V K operations (4096 x 4096 x 16032: 1.70 to 1.74 ms for 1.25).  The exponentials, which no
//     factor is in, could stay until then instead, for 2 N V bytes between the passes.
//
// What multiplies a row is split into a factor in [-1, 1] that goes into D and a number on the device that the products' epilogues
// multiply by: mean's 1 / count never touches D, where -1 (the target of a token that the model does not know) is exact, and
// fp16 keeps probabilities down to 2^-29 as normal numbers (D is stored times 2^15 there).
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "cross_entropy.h"
#include "launch_util.h"
#include "value16.cuh"

namespace soapb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSingleThreads = 1024;

void check(cudaError_t err, const char* what) {
  if (err != cudaSuccess) throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(err));
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  return v;
}

// One block, 8192 tokens at a time: a thread takes eight neighbouring ones, counts, learns how many come before, and writes.  With `factor`
// what the gradient of a reduced loss multiplies rows by is left as well (head_factors).
constexpr int kCountTokens = 8;
__global__ void __launch_bounds__(kSingleThreads)
head_count_kernel(const int64_t* __restrict__ targets, int tokens, int64_t ignored, int64_t first_word, int words, int64_t vocabulary,
                  int* __restrict__ count, int* __restrict__ where, int* __restrict__ column, int* __restrict__ split_counters, bool mean,
                  float* __restrict__ factor, float* __restrict__ alpha) {
  __shared__ int warps[32];
  wait_for_predecessor();
  let_successor_start();
  for (int i = threadIdx.x; i < kSplitCounters; i += kSingleThreads) split_counters[i] = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int counted = 0;
  for (int64_t base = 0; base < tokens; base += kSingleThreads * kCountTokens) {
    const int64_t begin = base + threadIdx.x * kCountTokens;
    int64_t target[kCountTokens];
#pragma unroll
    for (int i = 0; i < kCountTokens; ++i) target[i] = begin + i < tokens ? targets[begin + i] : ignored;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kCountTokens; ++i) mine += target[i] != ignored;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += other;
    }
    if (lane == 31) warps[warp] = before;
    __syncthreads();
    int sum = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += other;
    }
    const int ahead = __shfl_sync(0xffffffffu, sum, max(warp - 1, 0));      // in the warps before this one
    int at = counted + before - mine + (warp ? ahead : 0);
#pragma unroll
    for (int i = 0; i < kCountTokens; ++i) {
      if (target[i] == ignored) continue;
      const int64_t here = target[i] - first_word;
      const int c = target[i] < 0 || target[i] >= vocabulary ? kUnknown : here < 0 || here >= words ? kElsewhere : static_cast<int>(here);
      where[at] = static_cast<int>(begin + i);
      column[at] = c;
      if (factor) factor[at] = c == kUnknown ? nanf("") : 1.f;
      ++at;
    }
    counted += __shfl_sync(0xffffffffu, sum, 31);
    __syncthreads();      // before `warps` is written again
  }
  if (threadIdx.x == 0) {
    *count = counted;
    if (factor) *alpha = !mean ? 1.f : counted ? 1.f / static_cast<float>(counted) : 0.f;
  }
}

// Where not every token counts: the hidden states of those that do, one after another, zeros up to the next multiple of 64, and
// zeros in the gradients of the others.  A warp takes a row.
__global__ void head_gather_kernel(const uint16_t* __restrict__ hidden, int64_t ld, int tokens, int depth, const int64_t* __restrict__ targets, int64_t ignored,
                                   const int* __restrict__ count, const int* __restrict__ where, uint16_t* __restrict__ packed, int64_t ld_packed,
                                   uint16_t* __restrict__ d_hidden, int64_t ld_d) {
  wait_for_predecessor();
  let_successor_start();
  const int counted = *count;
  if (counted == tokens) return;
  const int lane = threadIdx.x & 31;
  const int rows_to_fill = min(tokens, (counted + 63) / 64 * 64);
  for (int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); row < tokens; row += gridDim.x * (blockDim.x >> 5)) {
    if (row < rows_to_fill) {
      const uint16_t* from = row < counted ? hidden + where[row] * ld : nullptr;
      uint16_t* to = packed + row * ld_packed;
      for (int i = lane; i < depth / 8; i += 32)      // (both pitches are multiples of 8)
        reinterpret_cast<uint4*>(to)[i] = from ? reinterpret_cast<const uint4*>(from)[i] : make_uint4(0, 0, 0, 0);
      for (int i = depth / 8 * 8 + lane; i < depth; i += 32) to[i] = from ? from[i] : 0;
    }
    if (d_hidden && targets[row] == ignored)
      for (int i = lane; i < depth; i += 32) d_hidden[row * ld_d + i] = 0;
  }
}

// Eight tokens a block, their parts dealt to 64 threads each and joined in a fixed order.  The target's logit is computed in fp32, a warp to a token:
// the tensor core's truncation makes all large logits a little too small (5e-6 of themselves at K = 4096).
constexpr int kJoinTokens = 8, kJoinWarps = 16, kJoinSlices = kJoinWarps * 32 / kJoinTokens;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps)
head_join_kernel(const float2* __restrict__ parts, int64_t ld_parts, int number, const int* __restrict__ count, int first, int rows,
                 const int* __restrict__ column, const T* __restrict__ all, int64_t ld_all, int tokens, const T* __restrict__ packed, int64_t ld_packed,
                 const T* __restrict__ weight, int64_t ld_weight, int depth, bool whole, TokenResults results) {
  __shared__ float2 shared[kJoinWarps][kJoinTokens];
  __shared__ float exact[kJoinTokens];
  wait_for_predecessor();
  let_successor_start();
  const int counted = *count;
  const int valid = min(rows, counted - first);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kJoinTokens + lane % kJoinTokens;
  float largest = -INFINITY, sum = 0.f;
  auto join = [&](const float2 part) {
    const float most = fmaxf(largest, part.x);
    const float base = most == -INFINITY ? 0.f : most;
    sum = sum * exp2f((largest - base) * kLog2e) + part.y * exp2f((part.x - base) * kLog2e);
    largest = most;
  };
  if (token < valid) {
#pragma unroll 4
    for (int i = warp * (32 / kJoinTokens) + lane / kJoinTokens; i < number; i += kJoinSlices) join(parts[i * ld_parts + token]);
  }
#pragma unroll
  for (int o = kJoinTokens; o < 32; o <<= 1)
    join(make_float2(__shfl_xor_sync(0xffffffffu, largest, o), __shfl_xor_sync(0xffffffffu, sum, o)));
  if (lane < kJoinTokens) shared[warp][lane] = make_float2(largest, sum);
  const int other = blockIdx.x * kJoinTokens + warp;
  const int word = warp < kJoinTokens && other < valid ? column[first + other] : -1;
  if (word >= 0) {                         // (the whole warp)
    const T* h = counted == tokens ? all + (first + other) * ld_all : packed + (first + other) * ld_packed;
    const T* w = weight + word * ld_weight;
    float dot = 0.f;
#pragma unroll 4
    for (int run = lane; run < depth / 8; run += 32) {      // (rows lie on 16-byte boundaries)
      Eight<T> a, b;
      a.load(h + 8 * run);
      b.load(w + 8 * run);
      float u[8], v[8];
      a.get(u);
      b.get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) dot = fmaf(u[j], v[j], dot);
    }
    for (int j = depth / 8 * 8 + lane; j < depth; j += 32) dot = fmaf(to_float(h[j]), to_float(w[j]), dot);
#pragma unroll
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0) exact[warp] = dot;
  }
  __syncthreads();
  if (threadIdx.x < kJoinTokens && token < valid) {
#pragma unroll
    for (int s = 1; s < kJoinWarps; ++s) join(shared[s][lane]);
    const float rest = logf(sum) + (largest == -INFINITY ? 0.f : largest);
    const int at = first + token;
    const bool known = column[at] >= 0;
    const float target = known ? exact[lane] : 0.f;
    if (whole && known) {
      const float over = rest - target, by = log1pf(expf(-fabsf(over)));
      results.loss[at] = over > 0.f ? over + by : by;
      results.lse[at] = over > 0.f ? rest + by : target + by;
    } else {
      results.loss[at] = target;
      results.lse[at] = rest;
    }
  }
}

__device__ __forceinline__ float token_loss(int column, float loss) { return column == kUnknown ? nanf("") : loss; }

// (the losses of tokens that do not count are cleared first)
__global__ void head_token_losses_kernel(const int* __restrict__ count, const int* __restrict__ where, const int* __restrict__ column,
                                         const float* __restrict__ of_token, float* __restrict__ losses) {
  wait_for_predecessor();
  let_successor_start();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < *count) losses[where[i]] = token_loss(column[i], of_token[i]);
}

// One block: the sum does not depend on the order in which blocks end.
__global__ void __launch_bounds__(kSingleThreads)
head_reduced_loss_kernel(const int* __restrict__ count, const int* __restrict__ column, const float* __restrict__ of_token, bool mean,
                         float* __restrict__ loss) {
  __shared__ double shared[32];
  wait_for_predecessor();
  let_successor_start();
  const int counted = *count;
  double sum = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < counted; i += kSingleThreads) sum += token_loss(column[i], of_token[i]);
  sum = block_reduce(sum, [](double a, double b) { return a + b; }, shared);
  if (threadIdx.x == 0) *loss = static_cast<float>(mean && counted ? sum / counted : sum);
}

__global__ void __launch_bounds__(kSingleThreads)
head_factors_kernel(const int* __restrict__ count, const int* __restrict__ where, const int* __restrict__ column, int reduction, float stored,
                    const float* __restrict__ grad_loss, float* __restrict__ factor, float* __restrict__ alpha) {
  __shared__ float shared[32];
  wait_for_predecessor();
  let_successor_start();
  const int counted = *count;
  float common = 1.f, relative = 1.f;      // the gradient is common * factor; factor = stored * relative * (the row's own)
  if (reduction == kLossNone) {
    float most = 0.f;
    for (int i = threadIdx.x; i < counted; i += kSingleThreads) most = fmaxf(most, fabsf(grad_loss[where[i]]));
    most = block_reduce(most, [](float a, float b) { return fmaxf(a, b); }, shared);
    // a power of two, so that no factor is rounded; none where the largest is zero or not finite
    if (most > 0.f && most < INFINITY) {
      const int exponent = min(120, max(-120, ilogbf(most) + 1));
      common = ldexpf(1.f, exponent);
      relative = ldexpf(1.f, -exponent);
    }
  } else {
    common = *grad_loss;
    if (reduction == kLossMean) common = counted ? common / static_cast<float>(counted) : 0.f;
  }
#pragma unroll 4
  for (int i = threadIdx.x; i < counted; i += kSingleThreads) {
    const float own = reduction == kLossNone ? grad_loss[where[i]] : 1.f;
    factor[i] = column[i] == kUnknown ? nanf("") : stored * relative * own;
  }
  if (threadIdx.x == 0) *alpha = common / stored;
}

// A row of exponentials, relative to the largest of their parts, becomes the row of D.  Rows up to the next multiple of 64 are cleared: they
// are read as part of K.
constexpr int kRescaleThreads = 256, kRescaleRuns = 4;
__global__ void __launch_bounds__(kRescaleThreads)
head_rescale_kernel(__nv_bfloat16* __restrict__ logits, int64_t ld, int64_t second, int words, const int* __restrict__ count, int first, int rows,
                    const float2* __restrict__ parts, int64_t ld_parts, const int* __restrict__ column, const float* __restrict__ lse,
                    const float* __restrict__ loss, const float* __restrict__ factor) {
  wait_for_predecessor();
  let_successor_start();
  const int row = blockIdx.y;
  const int counted = min(rows, *count - first);
  if (row >= min(rows, (counted + 63) / 64 * 64)) return;
  const bool here = row < counted;
  const float l = here ? lse[first + row] : 0.f, f = here ? factor[first + row] : 0.f;
  const int target = here ? column[first + row] : -1;
  __nv_bfloat16* line = logits + row * ld;
  const int run0 = blockIdx.x * kRescaleThreads * kRescaleRuns + threadIdx.x;
  // (the pitch is a multiple of 64; with a second term both are cleared up to the next multiple)
  const int runs = second ? (words + 63) / 64 * 8 : (words + 7) / 8;
  Eight<__half> e[kRescaleRuns];
  float largest[kRescaleRuns];
#pragma unroll
  for (int i = 0; i < kRescaleRuns; ++i) {
    const int run = run0 + i * kRescaleThreads;
    if (here && run < runs) {
      e[i].load(reinterpret_cast<const __half*>(line + 8 * run));
      largest[i] = parts[(run / (kLogitPart / 8)) * ld_parts + row].x;
    }
  }
#pragma unroll
  for (int i = 0; i < kRescaleRuns; ++i) {
    const int run = run0 + i * kRescaleThreads;
    if (run >= runs) break;
    Eight<__nv_bfloat16> d, left;
    if (here) {
      float v[8];
      e[i].get(v);
      const float by = exp2f((largest[i] - l) * kLog2e) * (f * (1.f / 32768.f));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 8 * run + j < words ? v[j] * by : 0.f;
      if (target >= 8 * run && target < 8 * run + 8) {
        const float of_target = expm1f(-loss[first + row]) * f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (target == 8 * run + j) v[j] = of_target;
      }
      d.set(v);
      float back[8];
      d.get(back);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] -= back[j];
      left.set(v);
    } else {
      d.clear();
      left.clear();
    }
    d.store(line + 8 * run);
    if (second) left.store(line + second + 8 * run);
  }
}

constexpr int kScaleThreads = 256;
__global__ void __launch_bounds__(kScaleThreads)
scale_gradients_kernel(const float* __restrict__ factor, __nv_bfloat16* __restrict__ a, int64_t count_a, __nv_bfloat16* __restrict__ b, int64_t count_b) {
  wait_for_predecessor();
  let_successor_start();
  const float f = *factor;
  if (f == 1.f) return;
  const int64_t runs_a = (count_a + 7) / 8, runs = runs_a + (count_b + 7) / 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kScaleThreads + threadIdx.x; i < runs; i += static_cast<int64_t>(gridDim.x) * kScaleThreads) {
    __nv_bfloat16* at = i < runs_a ? a + 8 * i : b + 8 * (i - runs_a);
    const int valid = static_cast<int>(min(static_cast<int64_t>(8), i < runs_a ? count_a - 8 * i : count_b - 8 * (i - runs_a)));
    if (valid == 8) {
      Eight<__nv_bfloat16> e;
      float v[8];
      e.load(at);
      e.get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
      e.set(v);
      e.store(at);
    } else {
      for (int j = 0; j < valid; ++j) at[j] = __float2bfloat16_rn(__bfloat162float(at[j]) * f);
    }
  }
}

// Where at most so many tokens count, logits are drained every 256 of K instead of 2048: an addition of the tensor core truncates up to 2^-23 of the
// running sum for each 16 of K, always towards zero, so that a logit is off by 16 or by 128 of these at most, and of a few tokens one
// such logit is most of the loss (of 400 drawn cases, six of one to six tokens had a loss 1.0e-6 to 2.8e-6 off with 2048, of 400 others the worst 1.2e-6
// with 256).  How many tokens count decides, not how many there are: padding changes no loss.  At 4096 x 128256 the loss of one token
// takes 290 us for 279; of 256 tokens, where no loss was as far off, it would be 275 for 236.
constexpr int kExactTokens = 64;

Hidden16 hidden_of(const HeadProblem& p, int first) {
  const int64_t at = static_cast<int64_t>(first);
  return Hidden16{Matrix16{static_cast<const uint16_t*>(p.packed.data) + at * p.packed.ld, p.packed.ld, true},
                  Matrix16{static_cast<const uint16_t*>(p.hidden.data) + at * p.hidden.ld, p.hidden.ld, true}, p.tokens};
}

Gemm16Problem logits_of(const HeadProblem& p, const LogitRows& r) {
  if (r.rows < 1 || r.first < 0 || r.first + r.rows > p.tokens) throw std::invalid_argument("cross entropy: rows outside the tokens");
  Gemm16Problem g{};
  g.M = r.rows; g.N = p.words; g.K = p.depth;
  g.drain = 2048; g.drain_few = 256; g.few = kExactTokens;
  g.count = p.count; g.first = r.first;
  g.targets = p.column + r.first;
  g.parts = r.parts; g.ld_parts = r.rows;
  g.C = r.logits; g.ldc = r.ld_logits;
  return g;
}

}  // namespace

void head_prepare(const HeadProblem& p, void* d_hidden, int64_t ld_hidden, LossReduction reduction, float* factor, float* alpha, cudaStream_t stream) {
  if (factor && (reduction == kLossNone || !p.bf16)) throw std::invalid_argument("head_prepare: these factors want the loss's gradient");
  check(launch_dependent(head_count_kernel, dim3(1), dim3(kSingleThreads), 0, stream, p.targets, p.tokens, p.ignore_index, p.first_word,
                         p.words, p.vocabulary, p.count, p.where, p.column, p.split_counters, reduction == kLossMean, factor, alpha),
        "head_count");
  const int blocks = std::min((p.tokens + 7) / 8, 8 * multiprocessors());
  check(launch_dependent(head_gather_kernel, dim3(blocks), dim3(256), 0, stream, static_cast<const uint16_t*>(p.hidden.data), p.hidden.ld,
                         p.tokens, p.depth, p.targets, p.ignore_index, p.count, p.where,
                         static_cast<uint16_t*>(const_cast<void*>(p.packed.data)), p.packed.ld, static_cast<uint16_t*>(d_hidden), ld_hidden),
        "head_gather");
}

void head_statistics(const HeadProblem& p, const LogitRows& r, const TokenResults& t, bool whole, int* status, cudaStream_t stream) {
  const Gemm16Problem g = logits_of(p, r);
  const Hidden16 hidden = hidden_of(p, r.first);
  gemm16(r.logits ? kLogitExponential : kLogitStatistics, p.bf16, hidden.packed, p.weight, g, status, stream, &hidden);
  auto join = [&](auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    check(launch_dependent(head_join_kernel<T>, dim3((r.rows + kJoinTokens - 1) / kJoinTokens), dim3(32 * kJoinWarps), 0, stream, r.parts,
                           static_cast<int64_t>(r.rows), (p.words + kLogitPart - 1) / kLogitPart, p.count, r.first, r.rows, p.column,
                           static_cast<const T*>(p.hidden.data), p.hidden.ld, p.tokens, static_cast<const T*>(p.packed.data), p.packed.ld,
                           static_cast<const T*>(p.weight.data), p.weight.ld, p.depth, whole, t),
          "head_join");
  };
  if (p.bf16) join(static_cast<__nv_bfloat16*>(nullptr));
  else join(static_cast<__half*>(nullptr));
}

void head_losses(const HeadProblem& p, const TokenResults& t, LossReduction reduction, float* loss, cudaStream_t stream) {
  if (reduction == kLossNone) {
    const cudaError_t err = cudaMemsetAsync(loss, 0, sizeof(float) * p.tokens, stream);
    if (err != cudaSuccess) throw std::runtime_error(std::string("head_losses: ") + cudaGetErrorString(err));
    check(launch_dependent(head_token_losses_kernel, dim3((p.tokens + 255) / 256), dim3(256), 0, stream, p.count, p.where, p.column, t.loss, loss),
          "head_token_losses");
  } else {
    check(launch_dependent(head_reduced_loss_kernel, dim3(1), dim3(kSingleThreads), 0, stream, p.count, p.column, t.loss,
                           reduction == kLossMean, loss),
          "head_reduced_loss");
  }
}

void head_factors(const HeadProblem& p, LossReduction reduction, const float* grad_loss, float* factor, float* alpha, cudaStream_t stream) {
  check(launch_dependent(head_factors_kernel, dim3(1), dim3(kSingleThreads), 0, stream, p.count, p.where, p.column,
                         static_cast<int>(reduction), p.bf16 ? 1.f : 32768.f, grad_loss, factor, alpha),
        "head_factors");
}

void head_rescale(const HeadProblem& p, const LogitRows& r, const TokenResults& t, const float* factor, cudaStream_t stream) {
  const Gemm16Problem g = logits_of(p, r);
  constexpr int kWords = 8 * kRescaleThreads * kRescaleRuns;
  if (r.second % 64 != 0 || r.ld_logits < r.second + (p.words + 63) / 64 * 64) throw std::invalid_argument("head_rescale: no room for both terms");
  // (the grid's second extent is at most 65535)
  for (int begin = 0; begin < r.rows; begin += 65472) {
    const int rows = std::min(r.rows - begin, 65472);
    check(launch_dependent(head_rescale_kernel, dim3((p.words + kWords - 1) / kWords, rows), dim3(kRescaleThreads), 0, stream,
                           static_cast<__nv_bfloat16*>(g.C) + begin * g.ldc, g.ldc, r.second, p.words, p.count, r.first + begin, rows, r.parts + begin,
                           g.ld_parts, p.column, t.lse, t.loss, factor),
          "head_rescale");
  }
}

void head_logit_gradient(const HeadProblem& p, const LogitRows& r, const TokenResults& t, const float* factor, int* status, cudaStream_t stream) {
  Gemm16Problem g = logits_of(p, r);
  g.second = r.second;
  g.lse = t.lse + r.first; g.loss = t.loss + r.first; g.factor = factor + r.first;
  const Hidden16 hidden = hidden_of(p, r.first);
  gemm16(kLogitGradient, p.bf16, hidden.packed, p.weight, g, status, stream, &hidden);
}

void head_gradients(const HeadProblem& p, const LogitRows& r, const float* alpha, const HeadGradients& out, int* status, cudaStream_t stream) {
  const bool last = r.first + r.rows == p.tokens;
  if (out.weight && !(r.first == 0 && last) && !out.sum) throw std::invalid_argument("head_gradients: several turns need a sum");
  if (out.hidden) {
    Gemm16Problem d{};
    d.M = r.rows; d.N = p.depth; d.K = p.words;
    d.count = p.count; d.first = r.first;
    d.C = out.hidden; d.ldc = out.ld_hidden; d.where = p.where + r.first;
    d.alpha = alpha; d.second = r.second;
    d.split_parts = out.split_parts; d.split_counters = p.split_counters;
    gemm16(kStore16, p.bf16, Matrix16{r.logits, r.ld_logits, true}, Matrix16{p.weight.data, p.weight.ld, false}, d, status, stream);
  }
  if (out.weight) {
    Gemm16Problem d{};
    d.M = p.words; d.N = p.depth; d.K = r.rows;
    d.count = p.count; d.first = r.first;
    d.alpha = alpha; d.second = r.second;
    d.accumulator = out.sum; d.ld_accumulator = out.ld_sum; d.add = r.first > 0;
    d.split_parts = out.split_parts; d.split_counters = p.split_counters;
    if (last) {
      d.C = out.weight; d.ldc = out.ld_weight;
    }
    Hidden16 hidden = hidden_of(p, r.first);
    hidden.packed.k_major = hidden.all.k_major = false;
    gemm16(kStore16, p.bf16, Matrix16{r.logits, r.ld_logits, false}, hidden.packed, d, status, stream, &hidden);
  }
}

void scale_gradients(const float* factor, void* a, int64_t count_a, void* b, int64_t count_b, cudaStream_t stream) {
  if ((reinterpret_cast<uintptr_t>(a) & 15) != 0 || (reinterpret_cast<uintptr_t>(b) & 15) != 0)
    throw std::invalid_argument("scale_gradients: matrices lie on 16-byte boundaries");
  const int64_t runs = (count_a + 7) / 8 + (count_b + 7) / 8;
  if (runs == 0) return;
  const int blocks = static_cast<int>(std::min<int64_t>((runs + kScaleThreads - 1) / kScaleThreads, 8 * multiprocessors()));
  check(launch_dependent(scale_gradients_kernel, dim3(blocks), dim3(kScaleThreads), 0, stream, factor, static_cast<__nv_bfloat16*>(a), count_a,
                         static_cast<__nv_bfloat16*>(b), count_b),
        "scale_gradients");
}

}  // namespace soapb200
