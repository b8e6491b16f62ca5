// Python bindings of the operators of a decoder's training step: addresses, pitches and sizes as integers, as in bindings.cpp.
#include "decoder.h"

#include <pybind11/stl.h>

#include <cstdint>
#include <stdexcept>
#include <vector>

#include "activation8.h"
#include "cross_entropy.h"
#include "residual_norm.h"

namespace py = pybind11;
using namespace soapb200;

namespace {
// A flat list of integers read in order (one list costs the interpreter a third of as many arguments).
class Reader {
 public:
  explicit Reader(const std::vector<int64_t>& values) : values_(values) {}
  int64_t next() {
    if (at_ >= values_.size()) throw std::invalid_argument("too few integers for this call");
    return values_[at_++];
  }
  int size() {
    const int64_t v = next();
    if (v < 0 || v > INT32_MAX) throw std::invalid_argument("a size is negative or above 2^31 - 1");
    return static_cast<int>(v);
  }
  template <typename T>
  T* pointer() { return reinterpret_cast<T*>(static_cast<uintptr_t>(next())); }
  cudaStream_t stream() { return pointer<CUstream_st>(); }
  bool done() const { return at_ == values_.size(); }
  void finish() const {
    if (at_ != values_.size()) throw std::invalid_argument("too many integers for this call");
  }

 private:
  const std::vector<int64_t>& values_;
  size_t at_ = 0;
};

Kept8 kept_of(Reader& in) {
  Kept8 kept{};
  kept.values = in.pointer<int8_t>(); kept.pitch = in.next(); kept.scales = in.pointer<float>();
  return kept;
}
Rows rows_of(Reader& in) {
  Rows rows{};
  rows.data = in.pointer<void>(); rows.ld = in.next();
  return rows;
}

NormProblem norm_problem(Reader& in, double scale, double eps) {
  NormProblem p{};
  p.type = in.size(); p.vector_type = in.size(); p.rows = in.next(); p.dim = in.size();
  p.scale = static_cast<float>(scale); p.eps = static_cast<float>(eps);
  p.x = rows_of(in); p.branch = rows_of(in);
  p.weight = in.pointer<void>(); p.branch_weight = in.pointer<void>(); p.gate = in.pointer<void>();
  p.rms = in.pointer<float>(); p.branch_rms = in.pointer<float>();
  return p;
}

HeadProblem head_problem(Reader& in) {
  HeadProblem p{};
  p.hidden.data = in.pointer<void>(); p.hidden.ld = in.next(); p.hidden.k_major = true;
  p.weight.data = in.pointer<void>(); p.weight.ld = in.next(); p.weight.k_major = true;
  p.tokens = in.size(); p.depth = in.size(); p.words = in.size();
  p.bf16 = in.next() != 0;
  p.targets = in.pointer<int64_t>();
  p.ignore_index = in.next(); p.first_word = in.next(); p.vocabulary = in.next();
  p.count = in.pointer<int>(); p.where = p.count + 1; p.column = p.where + p.tokens;
  p.split_counters = p.column + p.tokens;      // 1 + 2 * tokens + kSplitCounters integers
  p.packed.data = in.pointer<void>(); p.packed.ld = in.next(); p.packed.k_major = true;
  return p;
}

LogitRows logit_rows(Reader& in) {
  LogitRows r{};
  r.first = in.size(); r.rows = in.size();
  r.logits = in.pointer<void>(); r.ld_logits = in.next();
  r.parts = in.pointer<float2>();
  return r;
}
}  // namespace

void register_decoder(py::module_& m) {
  // Each call: the problem, then what this step adds (addresses, pitches, sizes), the status word where it is needed, the stream.
  m.def("head_prepare", [](const std::vector<int64_t>& problem, const std::vector<int64_t>& more) {
    Reader first(problem), in(more);
    const HeadProblem p = head_problem(first);
    first.finish();
    auto* d_hidden = in.pointer<void>();
    const int64_t ld = in.next();
    auto stream = in.stream();
    in.finish();
    head_prepare(p, d_hidden, ld, stream);
  });
  m.def("head_statistics", [](const std::vector<int64_t>& problem, const std::vector<int64_t>& more) {
    Reader first(problem), in(more);
    const HeadProblem p = head_problem(first);
    first.finish();
    const LogitRows r = logit_rows(in);
    auto* lse = in.pointer<float>(); auto* picked = in.pointer<float>();
    auto* status = in.pointer<int>(); auto stream = in.stream();
    in.finish();
    head_statistics(p, r, lse, picked, status, stream);
  });
  m.def("head_losses", [](const std::vector<int64_t>& problem, const std::vector<int64_t>& more) {
    Reader first(problem), in(more);
    const HeadProblem p = head_problem(first);
    first.finish();
    auto* lse = in.pointer<float>(); auto* picked = in.pointer<float>();
    const auto reduction = static_cast<LossReduction>(in.next());
    auto* loss = in.pointer<float>(); auto stream = in.stream();
    in.finish();
    head_losses(p, lse, picked, reduction, loss, stream);
  });
  m.def("head_factors", [](const std::vector<int64_t>& problem, const std::vector<int64_t>& more) {
    Reader first(problem), in(more);
    const HeadProblem p = head_problem(first);
    first.finish();
    const auto reduction = static_cast<LossReduction>(in.next());
    auto* grad_loss = in.pointer<float>(); auto* factor = in.pointer<float>(); auto* alpha = in.pointer<float>();
    auto stream = in.stream();
    in.finish();
    head_factors(p, reduction, grad_loss, factor, alpha, stream);
  });
  // The gradients of one turn.  With `picked` the logits are the exponentials that head_statistics left, otherwise they are computed anew.
  m.def("head_gradients", [](const std::vector<int64_t>& problem, const std::vector<int64_t>& more) {
    Reader first(problem), in(more);
    const HeadProblem p = head_problem(first);
    first.finish();
    const LogitRows r = logit_rows(in);
    auto* lse = in.pointer<float>(); auto* picked = in.pointer<float>();
    auto* factor = in.pointer<float>(); auto* alpha = in.pointer<float>();
    HeadGradients g{};
    g.hidden = in.pointer<void>(); g.ld_hidden = in.next();
    g.weight = in.pointer<void>(); g.ld_weight = in.next();
    g.sum = in.pointer<float>(); g.ld_sum = in.next();
    g.split_parts = in.pointer<float>();
    auto* status = in.pointer<int>(); auto stream = in.stream();
    in.finish();
    if (picked) head_rescale(p, r, lse, picked, factor, stream);
    else head_logit_gradient(p, r, lse, factor, status, stream);
    head_gradients(p, r, alpha, g, status, stream);
  });
  m.def("scale_gradients", [](const std::vector<int64_t>& values) {
    Reader in(values);
    auto* factor = in.pointer<float>();
    auto* a = in.pointer<void>();
    const int64_t count_a = in.next();
    auto* b = in.pointer<void>();
    const int64_t count_b = in.next();
    auto stream = in.stream();
    in.finish();
    scale_gradients(factor, a, count_a, b, count_b, stream);
  });
  // A plain product, C[m, n] = sum_k A(m, k) B(n, k), B with N along its rows and A in either order (tests, kernel cases).
  m.def("gemm16_store", [](bool bf16, bool a_k_major, const std::vector<int64_t>& values) {
    Reader in(values);
    Matrix16 a{in.pointer<void>(), in.next(), a_k_major};
    Matrix16 b{in.pointer<void>(), in.next(), false};
    Gemm16Problem p{};
    p.M = in.size(); p.N = in.size(); p.K = in.size();
    p.C = in.pointer<void>(); p.ldc = in.next();
    p.split_parts = in.pointer<float>(); p.split_counters = in.pointer<int>();
    auto* status = in.pointer<int>(); auto stream = in.stream();
    in.finish();
    gemm16(kStore16, bf16, a, b, p, status, stream);
  });
  m.def("pack8", [](int type, const std::vector<int64_t>& values) {
    Reader in(values);
    const Rows x = rows_of(in);
    const int64_t rows = in.next();
    const int dim = in.size();
    const Kept8 kept = kept_of(in);
    auto stream = in.stream();
    in.finish();
    pack8(type, x, rows, dim, kept, stream);
  });
  m.def("unpack8", [](int type, const std::vector<int64_t>& values) {
    Reader in(values);
    const Kept8 kept = kept_of(in);
    const int64_t rows = in.next();
    const int dim = in.size();
    auto* out = in.pointer<void>();
    const int64_t ld = in.next();
    auto stream = in.stream();
    in.finish();
    unpack8(type, kept, rows, dim, out, ld, stream);
  });
  // gate, up, rows, dim, y and its pitch, stream, then what keeps both (or nothing)
  m.def("swiglu8_forward", [](int type, const std::vector<int64_t>& values) {
    Reader in(values);
    const Rows gate = rows_of(in), up = rows_of(in);
    const int64_t rows = in.next();
    const int dim = in.size();
    auto* y = in.pointer<void>();
    const int64_t ld = in.next();
    auto stream = in.stream();
    if (in.done()) {
      swiglu8_forward(type, gate, up, rows, dim, y, ld, nullptr, nullptr, stream);
      return;
    }
    const Kept8 gate8 = kept_of(in), up8 = kept_of(in);
    in.finish();
    swiglu8_forward(type, gate, up, rows, dim, y, ld, &gate8, &up8, stream);
  });
  m.def("swiglu8_backward", [](int type, const std::vector<int64_t>& values) {
    Reader in(values);
    const Rows grad = rows_of(in);
    const Kept8 gate8 = kept_of(in), up8 = kept_of(in);
    const int64_t rows = in.next();
    const int dim = in.size();
    auto* d_gate = in.pointer<void>(); auto* d_up = in.pointer<void>(); auto* y = in.pointer<void>();
    const int64_t ld = in.next();
    auto stream = in.stream();
    in.finish();
    swiglu8_backward(type, grad, gate8, up8, rows, dim, d_gate, d_up, y, ld, stream);
  });
  m.def("residual_norm_forward", [](double scale, double eps, const std::vector<int64_t>& values) {
    Reader in(values);
    const NormProblem p = norm_problem(in, scale, eps);
    auto* h = in.pointer<void>(); auto* y = in.pointer<void>();
    const int64_t ld = in.next();
    auto stream = in.stream();
    in.finish();
    residual_norm_forward(p, h, y, ld, stream);
  });
  m.def("residual_norm_backward", [](double scale, double eps, const std::vector<int64_t>& values) {
    Reader in(values);
    const NormProblem p = norm_problem(in, scale, eps);
    NormGradients g{};
    g.grad_h = rows_of(in); g.grad_y = rows_of(in);
    g.d_x = in.pointer<void>(); g.d_branch = in.pointer<void>(); g.ld = in.next();
    g.partials = in.pointer<float>(); g.blocks = in.size();
    g.d_weight = in.pointer<void>(); g.d_branch_weight = in.pointer<void>(); g.d_gate = in.pointer<void>();
    auto stream = in.stream();
    in.finish();
    residual_norm_backward(p, g, stream);
  });
  m.def("residual_norm_blocks", &residual_norm_blocks);
  m.attr("SCALE_GROUP") = kScaleGroup;
  m.attr("LOGIT_PART") = kLogitPart;
  m.attr("SPLIT_COUNTERS") = kSplitCounters;
  m.attr("SPLIT_SCRATCH") = kSplitScratch;
}
