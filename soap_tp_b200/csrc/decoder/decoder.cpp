// The operators of a decoder's training step as torch operators with gradients (module soap_tp_b200._decoder).
//
// The launches of an optimizer step are issued from Python with raw pointers (bindings.cpp); a model calls these operators some hundred times a
// step, forward and backward, and autograd functions written in Python cost 25 to 130 us more of host time for a forward and a
// backward pass (packing 44 -> 19 us, cross entropy 223 -> 134, a gated activation 172 -> 80, a norm 229 -> 100), as much as an ordinary layer's kernels.  So their autograd nodes are native: they allocate what they return and their scratch with
// torch's allocator on the current stream, and launch.
//
// Arguments are checked in Python (soap_tp_b200/ops); what a kernel relies on is checked again where it is launched.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <pybind11/functional.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <functional>
#include <optional>
#include <vector>

#include "activation8.h"
#include "cross_entropy.h"
#include "residual_norm.h"

namespace py = pybind11;
using namespace soapb200;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

std::atomic<int64_t> g_launches{0};
void count(int64_t launches) { g_launches += launches; }

cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
int64_t round_up(int64_t value, int64_t multiple) { return (value + multiple - 1) / multiple * multiple; }

int size_as_int(int64_t value, const char* what) {
  TORCH_CHECK_VALUE(value <= INT32_MAX, what, " must be below 2**31, got ", value, ".");
  return static_cast<int>(value);
}

int type_of(at::ScalarType type) {
  switch (type) {
    case at::kBFloat16: return kBf16;
    case at::kHalf: return kFp16;
    case at::kFloat: return kFp32;
    default: TORCH_CHECK_TYPE(false, "decoder operators take bfloat16, float16 and float32, got ", type, ".");
  }
}

// Where a graph of the backward pass is asked for (`graph`), differentiating it is an error, raised when that happens.
variable_list once(variable_list gradients, bool graph) {
  if (!graph) return gradients;
  variable_list defined;
  for (const auto& g : gradients)
    if (g.defined()) defined.push_back(g.requires_grad() ? g : g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once", static_cast<int64_t>(defined.size()));
  defined = (*error)(std::move(defined));
  size_t at = 0;
  for (auto& g : gradients)
    if (g.defined()) g = defined[at++];
  return gradients;
}

// `x` as rows of its last dimension, without copying where they are evenly spaced; values of a row are neighbours.
Tensor rows_of(const Tensor& x) {
  const int64_t dim = x.size(-1);
  Tensor rows = x.dim() == 2 ? x : x.reshape({-1, dim});
  return dim == 1 || rows.stride(1) == 1 ? rows : rows.contiguous();
}
Rows address(const Tensor& rows) { return rows.defined() ? Rows{rows.data_ptr(), rows.stride(0)} : Rows{nullptr, 0}; }
void* pointer(const Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; }
Tensor like_rows(const Tensor& x) { return at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous); }

int64_t bits_of(double value) {
  int64_t bits;
  std::memcpy(&bits, &value, sizeof bits);
  return bits;
}
double double_of(int64_t bits) {
  double value;
  std::memcpy(&value, &bits, sizeof value);
  return value;
}

// The linear layer's products are in the type of their operands, forward and backward, whatever autocast says around the one or the other.
struct NoAutocast {
  c10::impl::ExcludeDispatchKeyGuard guard{c10::autocast_dispatch_keyset};
};

Tensor given(const std::optional<Tensor>& x) { return x ? *x : Tensor(); }

// ---- norms --------------------------------------------------------------------------------------------------------------
struct Vectors {
  Tensor weight, branch_weight, gate;
};

NormProblem norm_problem(const Tensor& rows, const Tensor& branch, const Vectors& v, double scale, double eps, const Tensor& rms, int64_t status) {
  NormProblem p{};
  p.type = type_of(rows.scalar_type());
  p.vector_type = p.type;
  for (const Tensor* t : {&v.weight, &v.branch_weight, &v.gate})
    if (t->defined()) p.vector_type = type_of(t->scalar_type());
  p.rows = rows.size(0);
  p.dim = size_as_int(rows.size(1), "a row's length");
  p.scale = static_cast<float>(scale);
  p.eps = static_cast<float>(eps);
  p.x = address(rows);
  p.branch = address(branch);
  p.weight = pointer(v.weight); p.branch_weight = pointer(v.branch_weight); p.gate = pointer(v.gate);
  p.rms = rms.data_ptr<float>();
  p.branch_rms = p.rms + p.rows;
  p.status = reinterpret_cast<int*>(static_cast<uintptr_t>(status));
  return p;
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  // h, if there is a branch, and y, if there is a weight
  using Maybe = std::optional<Tensor>;
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& branch_, const Maybe& weight_, const Maybe& branch_weight_,
                               const Maybe& gate_, double scale, double eps, int64_t status, std::vector<int64_t> want) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor branch = given(branch_), weight = given(weight_), branch_weight = given(branch_weight_), gate = given(gate_);
    const Vectors v{weight, branch_weight, gate};
    const Tensor x_rows = rows_of(x), branch_rows = branch.defined() ? rows_of(branch) : Tensor();
    Tensor h = branch.defined() ? like_rows(x) : Tensor(), y = weight.defined() ? like_rows(x) : Tensor();
    const Tensor rms = at::empty({2, x_rows.size(0)}, x.options().dtype(at::kFloat));
    const NormProblem p = norm_problem(x_rows, branch_rows, v, scale, eps, rms, status);
    residual_norm_forward(p, pointer(h), pointer(y), p.dim, current_stream());
    count(1);
    ctx->save_for_backward({x, branch, weight, branch_weight, gate, rms});
    want.insert(want.end(), {branch.defined(), status, bits_of(scale), bits_of(eps)});      // (one look-up in the backward pass)
    ctx->saved_data["numbers"] = std::move(want);
    ctx->set_materialize_grads(false);
    variable_list out;
    for (const Tensor* t : {&h, &y})
      if (t->defined()) out.push_back(*t);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    const auto saved = ctx->get_saved_variables();
    const auto numbers = ctx->saved_data["numbers"].toIntVector();
    const int64_t* want = numbers.data();
    const bool graph = at::GradMode::is_enabled(), with_branch = numbers[5];
    const Tensor grad_h = with_branch ? grads[0] : Tensor(), grad_y = saved[2].defined() ? grads[with_branch ? 1 : 0] : Tensor();
    if (!grad_h.defined() && !grad_y.defined()) return out;
    const Vectors v{saved[2], saved[3], saved[4]};
    const c10::cuda::CUDAGuard guard(saved[0].device());
    const at::NoGradGuard no_grad;
    const Tensor x = rows_of(saved[0]), branch = saved[1].defined() ? rows_of(saved[1]) : Tensor();
    const Tensor gh = grad_h.defined() ? rows_of(grad_h) : Tensor(), gy = grad_y.defined() ? rows_of(grad_y) : Tensor();
    NormProblem p = norm_problem(x, branch, v, double_of(numbers[7]), double_of(numbers[8]), saved[5], numbers[6]);
    // each gradient in memory of its own: where x and the branch are views of leaves, torch accumulates into what it is handed
    for (int i = 0; i < 2; ++i)
      if (want[i]) out[i] = like_rows(saved[0]);
    for (int i = 2; i < 5; ++i)
      if (want[i] && (i != 2 || grad_y.defined())) out[i] = at::empty_like(saved[i]);
    NormGradients g{};
    g.grad_h = address(gh); g.grad_y = address(gy);
    g.d_x = pointer(out[0]); g.d_branch = pointer(out[1]); g.ld = p.dim;
    g.d_weight = pointer(out[2]); g.d_branch_weight = pointer(out[3]); g.d_gate = pointer(out[4]);
    g.blocks = residual_norm_blocks(p, g);
    Tensor partials;
    if (g.d_weight || g.d_branch_weight || g.d_gate) {
      partials = at::empty({g.blocks, 2, p.dim}, x.options().dtype(at::kFloat));
      g.partials = partials.data_ptr<float>();
      count(1);
    }
    residual_norm_backward(p, g, current_stream());
    count(1);
    return once(std::move(out), graph);
  }
};

// ---- activations in 8 bits ------------------------------------------------------------------------------------------------
std::vector<Tensor> empty_kept(int64_t rows, int64_t dim, const Tensor& like) {
  return {at::empty({rows, round_up(dim, 8)}, like.options().dtype(at::kChar)),
          at::empty({rows, (dim + kScaleGroup - 1) / kScaleGroup}, like.options().dtype(at::kFloat))};
}
Kept8 kept(const Tensor& values, const Tensor& scales) { return Kept8{values.data_ptr<int8_t>(), values.size(1), scales.data_ptr<float>()}; }

std::vector<Tensor> pack(const Tensor& x) {
  const c10::cuda::CUDAGuard guard(x.device());
  const at::NoGradGuard no_grad;
  const Tensor rows = rows_of(x);
  auto out = empty_kept(rows.size(0), rows.size(1), rows);
  pack8(type_of(x.scalar_type()), address(rows), rows.size(0), size_as_int(rows.size(1), "a row's length"), kept(out[0], out[1]), current_stream());
  count(1);
  return out;
}

Tensor unpack(const Tensor& values, const Tensor& scales, std::vector<int64_t> shape, at::ScalarType type) {
  const c10::cuda::CUDAGuard guard(values.device());
  Tensor out = at::empty(shape, values.options().dtype(type));
  const int dim = size_as_int(shape.back(), "a row's length");
  unpack8(type_of(type), kept(values, scales), values.size(0), dim, out.data_ptr(), dim, current_stream());
  count(1);
  return out;
}

// y, and what keeps gate and up where `keep` says so
std::vector<Tensor> swiglu_forward(const Tensor& gate, const Tensor& up, bool keep) {
  const Tensor g = rows_of(gate), u = rows_of(up);
  const int64_t rows = g.size(0);
  const int dim = size_as_int(g.size(1), "a row's length");
  std::vector<Tensor> out{like_rows(gate)};
  Kept8 gate8{}, up8{};
  if (keep) {
    for (int i = 0; i < 2; ++i)
      for (auto& t : empty_kept(rows, dim, g)) out.push_back(t);
    gate8 = kept(out[1], out[2]);
    up8 = kept(out[3], out[4]);
  }
  swiglu8_forward(type_of(gate.scalar_type()), address(g), address(u), rows, dim, out[0].data_ptr(), dim, keep ? &gate8 : nullptr,
                  keep ? &up8 : nullptr, current_stream());
  count(1);
  return out;
}

// gradients of gate and up, and y at the kept values where it is asked for
std::vector<Tensor> swiglu_backward(const Tensor& grad, const Tensor* kept8, bool with_y) {
  const Tensor d = rows_of(grad);
  const int dim = size_as_int(d.size(1), "a row's length");
  std::vector<Tensor> out{like_rows(grad), like_rows(grad), with_y ? like_rows(grad) : Tensor()};
  swiglu8_backward(type_of(grad.scalar_type()), address(d), kept(kept8[0], kept8[1]), kept(kept8[2], kept8[3]), d.size(0), dim,
                   out[0].data_ptr(), out[1].data_ptr(), pointer(out[2]), dim, current_stream());
  count(1);
  return out;
}

struct SwiGLU8 : torch::autograd::Function<SwiGLU8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up) {
    const c10::cuda::CUDAGuard guard(gate.device());
    auto out = swiglu_forward(gate, up, true);
    ctx->save_for_backward({out[1], out[2], out[3], out[4]});
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    auto out = swiglu_backward(grads[0], saved.data(), false);
    return once({out[0], out[1]}, graph);
  }
};

struct SwiGLULinear8 : torch::autograd::Function<SwiGLULinear8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up, const Tensor& weight, bool want_weight) {
    const c10::cuda::CUDAGuard guard(gate.device());
    auto out = swiglu_forward(gate, up, true);
    ctx->save_for_backward({out[1], out[2], out[3], out[4], weight});
    ctx->saved_data["want_weight"] = want_weight;
    const NoAutocast own_type;
    return at::linear(out[0], weight);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    const bool want_weight = ctx->saved_data["want_weight"].toBool();
    variable_list result(4);
    const bool graph = at::GradMode::is_enabled();
    {
      const at::NoGradGuard no_grad;
      const NoAutocast own_type;
      const Tensor grad = grads[0].reshape({-1, grads[0].size(-1)});
      auto out = swiglu_backward(at::matmul(grads[0], saved[4]), saved.data(), want_weight);
      result[0] = out[0];
      result[1] = out[1];
      if (want_weight) result[2] = at::mm(grad.t(), out[2].reshape({-1, out[2].size(-1)}));
    }
    return once(std::move(result), graph);
  }
};

// ---- cross entropy --------------------------------------------------------------------------------------------------------
// `x` (rows, depth) as the tensor cores' loads take it: unit stride along depth, rows a multiple of 16 bytes apart.  Anything else is
// copied once.
Tensor rows16(const Tensor& x) {
  const bool lies = x.stride(1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  if (lies && x.stride(0) % 8 == 0 && x.stride(0) >= x.size(1)) return x;
  Tensor padded = at::empty({x.size(0), round_up(x.size(1), 8)}, x.options()).narrow(1, 0, x.size(1));
  padded.copy_(x);
  return padded;
}

// One call's hidden states, this rank's words and the targets, ready for the kernels, with the scratch they share.
struct Head {
  Tensor hidden, weight, targets, numbers, packed;
  HeadProblem problem{};
  int* status;

  Head(const Tensor& hidden_, const Tensor& weight_, const Tensor& targets_, int64_t ignore_index, int64_t first_word, int64_t vocabulary, int64_t status_)
      : hidden(rows16(hidden_)), weight(rows16(weight_)), targets(targets_.to(at::kLong).contiguous()),
        status(reinterpret_cast<int*>(static_cast<uintptr_t>(status_))) {
    HeadProblem& p = problem;
    p.tokens = size_as_int(hidden.size(0), "the number of tokens");
    p.depth = size_as_int(hidden.size(1), "depth");
    p.words = size_as_int(weight.size(0), "the number of words");
    p.hidden = Matrix16{hidden.data_ptr(), hidden.stride(0), true};
    p.weight = Matrix16{weight.data_ptr(), weight.stride(0), true};
    p.bf16 = hidden.scalar_type() == at::kBFloat16;
    p.targets = targets.data_ptr<int64_t>();
    p.ignore_index = ignore_index; p.first_word = first_word; p.vocabulary = vocabulary;
    numbers = at::empty({1 + 2 * int64_t{p.tokens} + kSplitCounters}, hidden.options().dtype(at::kInt));
    p.count = numbers.data_ptr<int>();
    p.where = p.count + 1;
    p.column = p.where + p.tokens;
    p.split_counters = p.column + p.tokens;
    packed = at::empty({p.tokens, round_up(p.depth, 8)}, hidden.options());
    p.packed = Matrix16{packed.data_ptr(), packed.size(1), true};
  }
  Tensor parts(int64_t rows) const {
    return at::empty({(problem.words + kLogitPart - 1) / kLogitPart, rows, 2}, hidden.options().dtype(at::kFloat));
  }
};

// The gradients that are wanted, made turn by turn from the softmax of as many tokens as the workspace holds (256 at least).
struct Gradients {
  Tensor hidden, weight, logits, sum, factor, split_parts;
  int rows;
  int64_t second;
  HeadGradients made{};

  Gradients(const Head& head, bool want_hidden, bool want_weight, int64_t workspace_bytes) {
    const HeadProblem& p = head.problem;
    const int64_t pitch = round_up(p.words, 64);
    rows = static_cast<int>(std::min<int64_t>(p.tokens, std::max<int64_t>(256, workspace_bytes / (2 * pitch) / 256 * 256)));
    const auto options = head.hidden.options(), floats = options.dtype(at::kFloat);
    second = p.tokens <= kFewTokens ? pitch : 0;
    logits = at::empty({rows, pitch + second}, options);
    if (want_hidden) hidden = at::empty({p.tokens, p.depth}, options);
    if (want_weight) weight = at::empty({p.words, p.depth}, options);
    if (want_weight && rows < p.tokens) sum = at::empty({p.words, round_up(p.depth, 32)}, floats);
    factor = at::empty({1 + int64_t{p.tokens}}, floats);      // alpha, then a factor for each token
    split_parts = at::empty({kSplitScratch}, floats);
    made.hidden = pointer(hidden); made.ld_hidden = p.depth;
    made.weight = pointer(weight); made.ld_weight = p.depth;
    made.sum = static_cast<float*>(pointer(sum)); made.ld_sum = sum.defined() ? sum.size(1) : 0;
    made.split_parts = split_parts.data_ptr<float>();
  }
  float* alpha() const { return factor.data_ptr<float>(); }
  float* factors() const { return alpha() + 1; }
  LogitRows turn(const Head& head, int first, float2* parts) const {
    return LogitRows{first, std::min(rows, head.problem.tokens - first), logits.data_ptr(), logits.size(1), parts, second};
  }
  int products() const { return (hidden.defined() ? 1 : 0) + (weight.defined() ? 1 : 0); }
};

float2* pairs(const Tensor& parts) { return reinterpret_cast<float2*>(parts.data_ptr<float>()); }

struct LossOptions {
  int64_t reduction, ignore_index, first_word, vocabulary, workspace_bytes, status;
  bool want_hidden, want_weight;
  std::function<void(const Tensor&, const Tensor&)> join;      // makes lse and loss of what several ranks have (head_statistics), in place
  std::vector<int64_t> numbers() const {
    return {reduction, ignore_index, first_word, vocabulary, workspace_bytes, status, want_hidden, want_weight};
  }
};

// Which capture the current stream is part of; 0: none.
int64_t capture_id() {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return 0;
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(current_stream(), &status, &id));
  return static_cast<int64_t>(id);
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets, const LossOptions& o) {
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Head head(hidden.reshape({-1, hidden.size(-1)}), weight, targets.reshape({-1}), o.ignore_index, o.first_word, o.vocabulary, o.status);
    const HeadProblem& p = head.problem;
    const auto stream = current_stream();
    const auto reduction = static_cast<LossReduction>(o.reduction);
    const auto floats = hidden.options().dtype(at::kFloat);
    const Tensor both = at::empty({2, p.tokens}, floats);
    const Tensor lse = both.select(0, 0), losses = both.select(0, 1);
    const TokenResults t{lse.data_ptr<float>(), losses.data_ptr<float>()};
    const bool whole = !o.join;
    // bf16 only: fp16 gradients are rounded after the loss's scale, which the backward pass brings, has been multiplied in
    const bool with_loss = (o.want_hidden || o.want_weight) && reduction != kLossNone && p.bf16;
    if (with_loss) {
      const Gradients g(head, o.want_hidden, o.want_weight, o.workspace_bytes);
      head_prepare(p, pointer(g.hidden), p.depth, reduction, g.factors(), g.alpha(), stream);
      const Tensor parts = head.parts(g.rows);
      for (int first = 0; first < p.tokens; first += g.rows) {
        const LogitRows r = g.turn(head, first, pairs(parts));
        head_statistics(p, r, t, whole, head.status, stream);
        if (o.join) o.join(lse.narrow(0, first, r.rows), losses.narrow(0, first, r.rows));
        head_rescale(p, r, t, g.factors(), stream);
        head_gradients(p, r, g.alpha(), g.made, head.status, stream);
        count(3 + g.products());
      }
      ctx->saved_data["hidden"] = g.hidden;
      ctx->saved_data["weight"] = g.weight;
    } else {
      head_prepare(p, nullptr, 0, reduction, nullptr, nullptr, stream);
      const int64_t parts_of_token = 8 * ((p.words + kLogitPart - 1) / kLogitPart);
      const int rows = static_cast<int>(std::min<int64_t>(p.tokens, std::max<int64_t>(256, o.workspace_bytes / parts_of_token / 256 * 256)));
      const Tensor parts = head.parts(rows);
      for (int first = 0; first < p.tokens; first += rows) {
        head_statistics(p, LogitRows{first, std::min(rows, p.tokens - first), nullptr, 0, pairs(parts)}, t, whole, head.status, stream);
        count(2);
      }
      if (o.join) o.join(lse, losses);
    }
    count(2);
    Tensor loss = reduction == kLossNone ? at::empty(targets.sizes(), floats) : at::empty({}, floats);
    head_losses(p, t, reduction, loss.data_ptr<float>(), stream);
    count(1);
    ctx->save_for_backward({hidden, weight, targets, both});
    ctx->saved_data["numbers"] = o.numbers();
    ctx->saved_data["made"] = with_loss;
    ctx->saved_data["capture"] = capture_id();
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &hidden = saved[0], &weight = saved[1], &targets = saved[2], &both = saved[3];
    const c10::cuda::CUDAGuard guard(hidden.device());
    variable_list result(4);
    const bool graph = at::GradMode::is_enabled();
    {
      const at::NoGradGuard no_grad;
      const auto stream = current_stream();
      const auto o = ctx->saved_data["numbers"].toIntVector();
      const Tensor grad_loss = grads[0].to(at::kFloat).contiguous();
      Tensor d_hidden, d_weight;
      // Handed over once: they are the caller's from then on.  A graph without the forward pass would scale them again at every replay.
      const bool made = ctx->saved_data["made"].toBool() && ctx->saved_data["capture"].toInt() == capture_id();
      if (ctx->saved_data["made"].toBool()) {
        if (made) {
          if (o[6]) d_hidden = ctx->saved_data["hidden"].toTensor();
          if (o[7]) d_weight = ctx->saved_data["weight"].toTensor();
          scale_gradients(grad_loss.data_ptr<float>(), pointer(d_hidden), d_hidden.defined() ? d_hidden.numel() : 0, pointer(d_weight),
                          d_weight.defined() ? d_weight.numel() : 0, stream);
          count(1);
        }
        ctx->saved_data["hidden"] = ctx->saved_data["weight"] = Tensor();
        ctx->saved_data["made"] = false;
      }
      if (!made) {
        const Head head(hidden.reshape({-1, hidden.size(-1)}), weight, targets.reshape({-1}), o[1], o[2], o[3], o[5]);
        const HeadProblem& p = head.problem;
        const Gradients g(head, o[6], o[7], o[4]);
        head_prepare(p, pointer(g.hidden), p.depth, static_cast<LossReduction>(o[0]), nullptr, nullptr, stream);
        head_factors(p, static_cast<LossReduction>(o[0]), grad_loss.data_ptr<float>(), g.factors(), g.alpha(), stream);
        for (int first = 0; first < p.tokens; first += g.rows) {
          const LogitRows r = g.turn(head, first, nullptr);
          head_logit_gradient(p, r, TokenResults{both.data_ptr<float>(), both.data_ptr<float>() + p.tokens}, g.factors(), head.status, stream);
          head_gradients(p, r, g.alpha(), g.made, head.status, stream);
          count(1 + g.products());
        }
        count(3);
        d_hidden = g.hidden;
        d_weight = g.weight;
      }
      if (d_hidden.defined()) result[0] = d_hidden.view(hidden.sizes());
      result[1] = d_weight;
    }
    return once(std::move(result), graph);
  }
};

// ---- entry points -----------------------------------------------------------------------------------------------------------
bool wanted(const Tensor& x) { return x.defined() && at::GradMode::is_enabled() && x.requires_grad(); }
// Whether a call goes through its autograd function: for gradients, and where an input has a tangent (of forward mode, which needs neither
// requires_grad nor grad mode), so that torch refuses it instead of getting a result without one.
bool differentiated(const Tensor& x) { return wanted(x) || x._fw_grad(0).defined(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Operators of a decoder's training step, with gradients, on CUDA tensors";
  m.def("residual_norm", [](const Tensor& x, const std::optional<Tensor>& branch, const std::optional<Tensor>& weight,
                            const std::optional<Tensor>& branch_weight, const std::optional<Tensor>& gate, double scale, double eps, int64_t status) {
    using Maybe = std::optional<Tensor>;
    auto vector = [](const Maybe& v) { return v ? Maybe(v->contiguous()) : Maybe(); };
    const Maybe w = vector(weight), wb = vector(branch_weight), g = vector(gate);
    std::vector<int64_t> want{wanted(x), wanted(given(branch)), wanted(given(w)), wanted(given(wb)), wanted(given(g))};
    return ResidualNorm::apply(x, branch, w, wb, g, scale, eps, status, std::move(want));
  });
  m.def("pack8", &pack);
  m.def("unpack8", [](const Tensor& values, const Tensor& scales, std::vector<int64_t> shape, at::ScalarType type) {
    return unpack(values, scales, std::move(shape), type);
  });
  m.def("swiglu8", [](const Tensor& gate, const Tensor& up) {
    if (differentiated(gate) || differentiated(up)) return SwiGLU8::apply(gate, up);
    const c10::cuda::CUDAGuard guard(gate.device());
    const at::NoGradGuard no_grad;
    return swiglu_forward(gate, up, false)[0];
  });
  m.def("swiglu_linear8", [](const Tensor& gate, const Tensor& up, const Tensor& weight) {
    if (differentiated(gate) || differentiated(up) || differentiated(weight)) return SwiGLULinear8::apply(gate, up, weight, wanted(weight));
    const c10::cuda::CUDAGuard guard(gate.device());
    const at::NoGradGuard no_grad;
    const NoAutocast own_type;
    return at::linear(swiglu_forward(gate, up, false)[0], weight);
  });
  m.def("linear_cross_entropy", [](const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t reduction, int64_t ignore_index,
                                   int64_t first_word, int64_t vocabulary, int64_t workspace_bytes, int64_t status,
                                   std::optional<std::function<void(const Tensor&, const Tensor&)>> join) {
    LossOptions o{reduction, ignore_index, first_word, vocabulary, workspace_bytes, status, wanted(hidden), wanted(weight), nullptr};
    if (join) o.join = *join;
    return LinearCrossEntropy::apply(hidden, weight, targets, o);
  });
  // A plain product, C[m, n] = sum_k A(m, k) B(n, k): `a` is (m, k) or with `turned` (k, m), `b` (k, n), both with 16-byte rows.
  m.def("gemm16", [](const Tensor& a, const Tensor& b, const Tensor& out, bool turned, int64_t status, const std::optional<Tensor>& split_parts,
                     const std::optional<Tensor>& split_counters) {
    for (const Tensor* t : {&a, &b, &out}) {
      TORCH_CHECK_VALUE(t->dim() == 2 && t->numel() > 0 && t->stride(1) == 1 && t->stride(0) >= t->size(1), "gemm16 takes matrices whose rows lie in memory one by one.");
      TORCH_CHECK_TYPE(t->scalar_type() == a.scalar_type() && (a.scalar_type() == at::kBFloat16 || a.scalar_type() == at::kHalf),
                       "gemm16 takes bfloat16 or float16, all of one type.");
    }
    TORCH_CHECK_VALUE(a.size(turned ? 0 : 1) == b.size(0) && out.size(0) >= a.size(turned ? 1 : 0) && out.size(1) >= b.size(1),
                      "gemm16: sizes do not match, or the result has no room: ", a.sizes(), ", ", b.sizes(), " and ", out.sizes(), ".");
    TORCH_CHECK_VALUE(split_parts.has_value() == split_counters.has_value(), "gemm16: split_parts and split_counters go together.");
    if (split_parts) {
      TORCH_CHECK_TYPE(split_parts->scalar_type() == at::kFloat && split_counters->scalar_type() == at::kInt, "gemm16: split_parts are float32, split_counters int32.");
      TORCH_CHECK_VALUE(split_parts->is_contiguous() && split_parts->numel() >= kSplitScratch && split_counters->is_contiguous() &&
                        split_counters->numel() >= kSplitCounters, "gemm16: split_parts or split_counters are too small.");
      TORCH_CHECK_VALUE(split_parts->device() == a.device() && split_counters->device() == a.device(), "gemm16: scratch is on another device.");
    }
    TORCH_CHECK_VALUE(a.is_cuda() && b.device() == a.device() && out.device() == a.device(), "gemm16 takes tensors of one CUDA device.");
    const c10::cuda::CUDAGuard guard(a.device());
    Gemm16Problem p{};
    p.M = size_as_int(turned ? a.size(1) : a.size(0), "m");
    p.N = size_as_int(b.size(1), "n");
    p.K = size_as_int(b.size(0), "k");
    p.C = out.data_ptr();
    p.ldc = out.stride(0);
    p.split_parts = split_parts ? split_parts->data_ptr<float>() : nullptr;
    p.split_counters = split_counters ? split_counters->data_ptr<int>() : nullptr;
    gemm16(kStore16, a.scalar_type() == at::kBFloat16, Matrix16{a.data_ptr(), a.stride(0), !turned}, Matrix16{b.data_ptr(), b.stride(0), false}, p,
           reinterpret_cast<int*>(static_cast<uintptr_t>(status)), current_stream());
    count(1);
  }, py::arg("a"), py::arg("b"), py::arg("out"), py::arg("turned"), py::arg("status"), py::arg("split_parts") = py::none(),
     py::arg("split_counters") = py::none());
  m.def("launches", [] { return g_launches.load(); });
  m.def("compiled_arch", [] { return std::string("sm_100a"); });
  m.attr("SPLIT_COUNTERS") = kSplitCounters;
  m.attr("SPLIT_SCRATCH") = kSplitScratch;
}
