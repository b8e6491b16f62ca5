// h = x + s g * b',  b' = b or r_b b w_b;  y = r h w   with r = 1 / sqrt(mean(h^2) + eps), r_b the same of b.
//
// Backward, from the gradients of h and y, at the h that was stored and the r that was computed:
//   t = dy w             dh = dh' + r (t - h r^2 mean(t h))          dw  = sum over rows of dy h r
//   db' = s g dh         dg = sum of s dh b'                         dx  = dh
//   t_b = db' w_b        db = r_b (t_b - b r_b^2 mean(t_b b))        dw_b = sum of db' b r_b
// All sums in fp32, h and y rounded once, y from the unrounded h.
//
// Memory bounds it: a row is read once into registers (a warp for short rows, a block for long ones), the means are block sums, and
// everything leaves in one pass.  The backward pass runs a fixed number of blocks over all rows; each thread keeps its columns' sums for the
// vectors' gradients in registers, and a second kernel adds the blocks' sums in a fixed order.
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "launch_util.h"
#include "residual_norm.h"
#include "value16.cuh"

namespace soapb200 {
namespace {

// A thread's E values of a row that start at `column`, as fp32.  E = 8: a run that lies on 16-byte boundaries; E = 1: any row.
template <typename T, int E>
struct Run {
  static __device__ __forceinline__ void read(const T* p, float (&v)[E]) {
    if constexpr (E == 8) {
      Eight<T> e;
      e.load(p);
      e.get(v);
    } else {
      v[0] = to_float(*p);
    }
  }
  static __device__ __forceinline__ void write(T* p, const float (&v)[E]) {
    if constexpr (E == 8) {
      Eight<T> e;
      e.set(v);
      e.store(p);
    } else {
      *p = from_float<T>(v[0]);
    }
  }
};

template <int E>
__device__ __forceinline__ void read_vector(const void* p, bool fp32, const __nv_bfloat16*, int column, float (&v)[E]) {
  if (fp32) Run<float, E>::read(static_cast<const float*>(p) + column, v);
  else Run<__nv_bfloat16, E>::read(static_cast<const __nv_bfloat16*>(p) + column, v);
}
template <int E>
__device__ __forceinline__ void read_vector(const void* p, bool fp32, const __half*, int column, float (&v)[E]) {
  if (fp32) Run<float, E>::read(static_cast<const float*>(p) + column, v);
  else Run<__half, E>::read(static_cast<const __half*>(p) + column, v);
}
template <int E>
__device__ __forceinline__ void read_vector(const void* p, bool, const float*, int column, float (&v)[E]) {
  Run<float, E>::read(static_cast<const float*>(p) + column, v);
}

// Sum over the threads of a row: a warp (blockDim.x = 32), or the block.  `shared`: 33 floats; `turn` alternates so that one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, float* shared, int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (blockDim.x == 32) return v;
  float* slot = shared + 32 * turn;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = (threadIdx.x & 31) < warps ? slot[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int E, int N, int THREADS, bool AFTER>
__global__ void __launch_bounds__(THREADS) residual_norm_forward_kernel(NormProblem p, T* __restrict__ h_out, T* __restrict__ y_out, int64_t ld, int runs) {
  __shared__ float shared[64];
  int turn = 0;
  wait_for_predecessor();
  let_successor_start();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;             // (a whole warp, or no one: blockDim.y > 1 only with rows of a warp)
  const bool fp32 = p.vector_type == kFp32;
  const T* x = static_cast<const T*>(p.x.data) + row * p.x.ld;
  const T* b = static_cast<const T*>(p.branch.data) + row * p.branch.ld;
  const T* tag = nullptr;
  float h[N][E];
  const bool with_branch = p.branch.data != nullptr;
  if (with_branch) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int run = threadIdx.x + i * blockDim.x;
      if (run < runs) {
        Run<T, E>::read(b + run * E, h[i]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] = 0.f;
      }
    }
    float r_b = 1.f;
    if (AFTER) {
      float squares = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) squares = fmaf(h[i][e], h[i][e], squares);
      r_b = 1.f / sqrtf(row_sum(squares, shared, turn) / static_cast<float>(p.dim) + p.eps);
      if (threadIdx.x == 0) p.branch_rms[row] = r_b;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int run = threadIdx.x + i * blockDim.x;
      if (run < runs) {
        float v[E];
        if (AFTER) {
          read_vector<E>(p.branch_weight, fp32, tag, run * E, v);
#pragma unroll
          for (int e = 0; e < E; ++e) h[i][e] *= r_b * v[e];
        }
        if (p.gate) {
          read_vector<E>(p.gate, fp32, tag, run * E, v);
#pragma unroll
          for (int e = 0; e < E; ++e) h[i][e] *= v[e];
        }
        Run<T, E>::read(x + run * E, v);
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] = fmaf(p.scale, h[i][e], v[e]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int run = threadIdx.x + i * blockDim.x;
      if (run < runs) {
        Run<T, E>::read(x + run * E, h[i]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] = 0.f;
      }
    }
  }
  if (h_out) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int run = threadIdx.x + i * blockDim.x;
      if (run < runs) Run<T, E>::write(h_out + row * ld + run * E, h[i]);
    }
  }
  if (!y_out) return;
  float squares = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (static_cast<int>(threadIdx.x + i * blockDim.x) < runs) {
#pragma unroll
      for (int e = 0; e < E; ++e) squares = fmaf(h[i][e], h[i][e], squares);
    }
  }
  const float r = 1.f / sqrtf(row_sum(squares, shared, turn) / static_cast<float>(p.dim) + p.eps);
  if (threadIdx.x == 0) p.rms[row] = r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int run = threadIdx.x + i * blockDim.x;
    if (run < runs) {
      float w[E];
      read_vector<E>(p.weight, fp32, tag, run * E, w);
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] *= h[i][e] * r;
      Run<T, E>::write(y_out + row * ld + run * E, w);
    }
  }
}

// Blocks of blockDim.y rows at a time, over all rows.  N runs of E values a thread.  SCALED: the branch has a norm or a gate.
template <typename T, int E, int N, int THREADS, bool SCALED>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1)
residual_norm_backward_kernel(NormProblem p, NormGradients g, int runs) {
  __shared__ float shared[64];
  extern __shared__ float joined[];      // dim floats where several rows share a block
  int turn = 0;
  wait_for_predecessor();
  let_successor_start();
  const bool fp32 = p.vector_type == kFp32;
  const T* tag = nullptr;
  const float inverse_dim = 1.f / static_cast<float>(p.dim);
  const bool after = SCALED && p.branch_weight, gated = SCALED && p.gate;
  float d_w[N][E], d_wb[SCALED ? N : 1][E], d_g[SCALED ? N : 1][E];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      d_w[i][e] = 0.f;
      if (SCALED) d_wb[i][e] = d_g[i][e] = 0.f;
    }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; row < p.rows; row += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    float dh[N][E];
    const T* gh = static_cast<const T*>(g.grad_h.data) + row * g.grad_h.ld;
    const T* gy = static_cast<const T*>(g.grad_y.data) + row * g.grad_y.ld;
    const T* h = static_cast<const T*>(p.x.data) + row * p.x.ld;
    const T* b = static_cast<const T*>(p.branch.data) + row * p.branch.ld;
    if (g.grad_y.data) {
      const float r = p.rms[row];
      float hv[N][E], dot = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int run = threadIdx.x + i * blockDim.x;
        if (run < runs) {
          float w[E];
          Run<T, E>::read(gy + run * E, dh[i]);
          Run<T, E>::read(h + run * E, hv[i]);
          read_vector<E>(p.weight, fp32, tag, run * E, w);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            d_w[i][e] = fmaf(dh[i][e], hv[i][e] * r, d_w[i][e]);
            dh[i][e] *= w[e];
            dot = fmaf(dh[i][e], hv[i][e], dot);
          }
        }
      }
      const float c = row_sum(dot, shared, turn) * inverse_dim * r * r;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) dh[i][e] = r * (dh[i][e] - hv[i][e] * c);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) dh[i][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int run = threadIdx.x + i * blockDim.x;
      if (run < runs) {
        if (g.grad_h.data) {
          float v[E];
          Run<T, E>::read(gh + run * E, v);
#pragma unroll
          for (int e = 0; e < E; ++e) dh[i][e] += v[e];
        }
        if (g.d_x) Run<T, E>::write(static_cast<T*>(g.d_x) + row * g.ld + run * E, dh[i]);
      }
    }
    if constexpr (!SCALED) {
      if (g.d_branch) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int run = threadIdx.x + i * blockDim.x;
          if (run < runs) {
#pragma unroll
            for (int e = 0; e < E; ++e) dh[i][e] *= p.scale;
            Run<T, E>::write(static_cast<T*>(g.d_branch) + row * g.ld + run * E, dh[i]);
          }
        }
      }
    } else {
      const float r_b = after ? p.branch_rms[row] : 1.f;
      float bv[N][E], dot = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int run = threadIdx.x + i * blockDim.x;
        if (run < runs) {
          float wb[E], gate[E];
          Run<T, E>::read(b + run * E, bv[i]);
#pragma unroll
          for (int e = 0; e < E; ++e) wb[e] = gate[e] = 1.f;
          if (after) read_vector<E>(p.branch_weight, fp32, tag, run * E, wb);
          if (gated) read_vector<E>(p.gate, fp32, tag, run * E, gate);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float normed = bv[i][e] * r_b;
            dh[i][e] *= p.scale;
            d_g[i][e] = fmaf(dh[i][e], normed * wb[e], d_g[i][e]);
            dh[i][e] *= gate[e];
            d_wb[i][e] = fmaf(dh[i][e], normed, d_wb[i][e]);
            dh[i][e] *= wb[e];
            dot = fmaf(dh[i][e], bv[i][e], dot);
          }
        }
      }
      const float c = after ? row_sum(dot, shared, turn) * inverse_dim * r_b * r_b : 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int run = threadIdx.x + i * blockDim.x;
        if (run < runs) {
          if (after) {
#pragma unroll
            for (int e = 0; e < E; ++e) dh[i][e] = r_b * (dh[i][e] - bv[i][e] * c);
          }
          if (g.d_branch) Run<T, E>::write(static_cast<T*>(g.d_branch) + row * g.ld + run * E, dh[i]);
        }
      }
    }
  }
  // this block's sums: rows that share the block are added one after another
  auto leave = [&](float (&sums)[N][E], int which) {
    float* out = g.partials + (static_cast<int64_t>(blockIdx.x) * 3 + which) * p.dim;
    if (blockDim.y == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int run = threadIdx.x + i * blockDim.x;
        if (run < runs) {
#pragma unroll
          for (int e = 0; e < E; ++e) out[run * E + e] = sums[i][e];
        }
      }
      return;
    }
    for (int y = 0; y < static_cast<int>(blockDim.y); ++y) {
      __syncthreads();
      if (static_cast<int>(threadIdx.y) == y) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int run = threadIdx.x + i * blockDim.x;
          if (run < runs) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float before = y ? joined[run * E + e] : 0.f;
              if (y + 1 < static_cast<int>(blockDim.y)) joined[run * E + e] = before + sums[i][e];
              else out[run * E + e] = before + sums[i][e];
            }
          }
        }
      }
    }
  };
  if (g.d_weight) leave(d_w, 0);
  if constexpr (SCALED) {
    if (g.d_branch_weight) leave(d_wb, 1);
    if (g.d_gate) leave(d_g, 2);
  }
}

constexpr int kSumSlices = 8;
// 32 columns a block, the blocks' sums dealt to eight warps.
__global__ void __launch_bounds__(32 * kSumSlices) norm_vectors_kernel(NormProblem p, NormGradients g) {
  __shared__ float shared[kSumSlices][32];
  wait_for_predecessor();
  let_successor_start();
  const int which = blockIdx.y;
  void* out = which == 0 ? g.d_weight : which == 1 ? g.d_branch_weight : g.d_gate;
  if (!out) return;
  const int column = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (column < p.dim) {
#pragma unroll 8
    for (int i = threadIdx.y; i < g.blocks; i += kSumSlices) sum += g.partials[(static_cast<int64_t>(i) * 3 + which) * p.dim + column];
  }
  shared[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && column < p.dim) {
#pragma unroll
    for (int s = 1; s < kSumSlices; ++s) sum += shared[s][threadIdx.x];
    if (p.vector_type == kFp32) static_cast<float*>(out)[column] = sum;
    else if (p.vector_type == kFp16) static_cast<__half*>(out)[column] = __float2half_rn(sum);
    else static_cast<__nv_bfloat16*>(out)[column] = __float2bfloat16_rn(sum);
  }
}

// How a row is dealt to threads: runs of eight values where everything lies on 16-byte boundaries, single values otherwise; a warp
// for up to 512 or 256 values, otherwise as many warps as 16 or 8 values a thread ask for.  `bound`: what the kernel is compiled for.
struct Deal {
  int run, per_thread, threads, rows, runs, bound;
};
constexpr int kShortRow = 256;      // values of a row that one warp takes, whatever the run
Deal deal_of(bool wide, int dim) {
  Deal d{};
  d.run = wide ? 8 : 1;
  d.runs = (dim + d.run - 1) / d.run;
  d.per_thread = wide ? 2 : 8;
  if (dim <= kShortRow) {
    d.threads = 32;
    d.rows = 8;
    d.bound = 256;
    return d;
  }
  d.rows = 1;
  if (d.runs > 1024 * d.per_thread) d.per_thread = wide ? 4 : 32;
  if (d.runs > 1024 * d.per_thread) throw std::invalid_argument("residual_norm: rows of more than 32768 values are not supported");
  d.threads = ((d.runs + d.per_thread - 1) / d.per_thread + 31) / 32 * 32;
  d.bound = d.threads <= 256 ? 256 : d.threads <= 512 ? 512 : 1024;
  return d;
}

bool on_16(const void* data, int64_t ld, int size) { return (reinterpret_cast<uintptr_t>(data) & 15) == 0 && (ld * size) % 16 == 0; }
int size_of(int type) { return type == kFp32 ? 4 : 2; }

bool wide_problem(const NormProblem& p) {
  const int size = size_of(p.type);
  return p.dim % 8 == 0 && on_16(p.x.data, p.x.ld, size) && on_16(p.branch.data, p.branch.ld, size) && on_16(p.weight, 0, 1) &&
         on_16(p.branch_weight, 0, 1) && on_16(p.gate, 0, 1);
}

void check_problem(const NormProblem& p) {
  if (p.dim < 1 || p.rows < 1) throw std::invalid_argument("residual_norm: empty");
  if (p.vector_type != p.type && p.vector_type != kFp32) throw std::invalid_argument("residual_norm: vectors have the rows' type or fp32");
  if (!p.branch.data && (p.branch_weight || p.gate)) throw std::invalid_argument("residual_norm: a norm or gate without a branch");
}

void check(cudaError_t err, const char* what) {
  if (err != cudaSuccess) throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(err));
}

template <typename F>
void for_type(int type, F f) {
  if (type == kBf16) f(static_cast<__nv_bfloat16*>(nullptr));
  else if (type == kFp16) f(static_cast<__half*>(nullptr));
  else if (type == kFp32) f(static_cast<float*>(nullptr));
  else throw std::invalid_argument("residual_norm: unknown type");
}

template <int E_, int N_, int THREADS_>
struct Form {
  static constexpr int E = E_, N = N_, THREADS = THREADS_;
};
template <typename F>
void for_deal(const Deal& d, F f) {
  if (d.run == 8) {
    if (d.per_thread == 4) f(Form<8, 4, 1024>{});
    else if (d.bound == 256) f(Form<8, 2, 256>{});
    else if (d.bound == 512) f(Form<8, 2, 512>{});
    else f(Form<8, 2, 1024>{});
  } else {
    if (d.per_thread == 32) f(Form<1, 32, 1024>{});
    else if (d.bound == 256) f(Form<1, 8, 256>{});
    else f(Form<1, 8, 1024>{});
  }
}

}  // namespace

int residual_norm_blocks(int64_t rows, int dim) {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    throw std::runtime_error("residual_norm: no device");
  const int at_once = dim <= kShortRow ? 8 : 1;
  return static_cast<int>(std::min<int64_t>((rows + at_once - 1) / at_once, 2 * sms));
}

void residual_norm_forward(const NormProblem& p, void* h, void* y, int64_t ld, cudaStream_t stream) {
  check_problem(p);
  const int size = size_of(p.type);
  const Deal d = deal_of(wide_problem(p) && on_16(h, ld, size) && on_16(y, ld, size), p.dim);
  const int64_t blocks = (p.rows + d.rows - 1) / d.rows;
  if (blocks > 0x7fffffff) throw std::invalid_argument("residual_norm: too many rows");
  for_type(p.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    for_deal(d, [&](auto form) {
      using F = decltype(form);
      auto kernel = p.branch_weight ? residual_norm_forward_kernel<T, F::E, F::N, F::THREADS, true>
                                    : residual_norm_forward_kernel<T, F::E, F::N, F::THREADS, false>;
      check(launch_dependent(kernel, dim3(static_cast<unsigned>(blocks)), dim3(d.threads, d.rows), 0, stream, p, static_cast<T*>(h),
                             static_cast<T*>(y), ld, d.runs),
            "residual_norm_forward");
    });
  });
}

void residual_norm_backward(const NormProblem& p, const NormGradients& g, cudaStream_t stream) {
  check_problem(p);
  const int size = size_of(p.type);
  const Deal d = deal_of(wide_problem(p) && on_16(g.grad_h.data, g.grad_h.ld, size) && on_16(g.grad_y.data, g.grad_y.ld, size) &&
                             on_16(g.d_x, g.ld, size) && on_16(g.d_branch, g.ld, size),
                         p.dim);
  if (g.blocks < 1) throw std::invalid_argument("residual_norm: no blocks");
  for_type(p.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    for_deal(d, [&](auto form) {
      using F = decltype(form);
      auto kernel = p.branch_weight || p.gate ? residual_norm_backward_kernel<T, F::E, F::N, F::THREADS, true>
                                              : residual_norm_backward_kernel<T, F::E, F::N, F::THREADS, false>;
      check(launch_dependent(kernel, dim3(g.blocks), dim3(d.threads, d.rows), d.rows > 1 ? p.dim * sizeof(float) : 0, stream, p, g, d.runs),
            "residual_norm_backward");
    });
  });
  if (g.d_weight || g.d_branch_weight || g.d_gate)
    check(launch_dependent(norm_vectors_kernel, dim3((p.dim + 31) / 32, 3), dim3(32, kSumSlices), 0, stream, p, g), "norm_vectors");
}

}  // namespace soapb200
