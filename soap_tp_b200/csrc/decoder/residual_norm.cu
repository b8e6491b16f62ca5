// h = x + s g * b',  b' = b or r_b b w_b;  y = r h w   with r = 1 / sqrt(mean(h^2) + eps), r_b the same of b.
//
// Backward, from the gradients of h and y; h comes from x and b once more (as it was stored it has 2^-9 less, and dw with it):
//   t = dy w             dh = dh' + r (t - h r^2 mean(t h))          dw  = sum over rows of dy h r
//   db' = s g dh         dg = sum of s dh b'                         dx  = dh
//   t_b = db' w_b        db = r_b (t_b - b r_b^2 mean(t_b b))        dw_b = sum of db' b r_b
// dg and dw_b are one sum, of s dh b r_b, times w_b and g.
// All sums in fp32, h and y rounded once, y from the unrounded h.
//
// Memory bounds it.  A fixed number of blocks goes over all rows; in a block one to sixteen warps share a row (16 values a thread), and
// groups of warps take rows of their own.  Each group keeps a ring of rows in shared memory, which untiled bulk copies fill ahead of their use: the
// means are sums over a group that everything else of a row waits for, and what must be under way meanwhile (some 40 KB an SM) does
// not fit in registers next to the sums of the vectors' gradients.  Those stay in registers until a block's last row; a second kernel adds the
// blocks' sums in a fixed order.  The vectors stay in registers as well, as fp32, and arithmetic goes two values at a time: with 40 instructions a value,
// converted and multiplied anew for every row, issue bounded it.  Rows that do not lie on 16-byte boundaries are copied from the boundary before them and read shifted (fp32:
// value by value); rows too long for two of them in shared memory are read straight into registers.
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "launch_util.h"
#include "ptx.cuh"
#include "residual_norm.h"
#include "value16.cuh"

namespace soapb200 {
namespace {

// A thread's 2 P values of a row, as pairs of fp32.  kWhole: runs of eight neighbouring values on 16-byte boundaries, blockDim.x runs apart;
// kShifted: the same anywhere (16-bit types); kSingle: single values, blockDim.x apart.  Values beyond the row are zero and are not written.
enum Access : int { kWhole, kShifted, kSingle };
template <int A, int P>
struct Lane {
  uint64_t v[P];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const { return pair_element(v[i / 2], i & 1); }
  static __device__ __forceinline__ int column_of(int run) { return 8 * (threadIdx.x + run * blockDim.x); }

  template <typename T>
  __device__ __forceinline__ void load(const T* row, int dim) {
    if constexpr (A == kSingle) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int first = threadIdx.x + 2 * i * blockDim.x, second = first + blockDim.x;
        v[i] = pack_floats(first < dim ? to_float(row[first]) : 0.f, second < dim ? to_float(row[second]) : 0.f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < P / 4; ++i) {
        const int column = column_of(i);
        float f[8];
        if constexpr (A == kShifted && sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = column + j < dim ? to_float(row[column + j]) : 0.f;
        } else {
          Eight<T> e;
          if constexpr (A == kShifted) e = load8_shifted(row + column, min(8, dim - column));
          else if (column < dim) e.load(row + column);
          else e.clear();
          e.get(f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = pack_floats(f[2 * j], f[2 * j + 1]);
      }
    }
  }
  // (with kShifted all lanes of a warp call)
  template <typename T>
  __device__ __forceinline__ void store(T* row, int dim) const {
    if constexpr (A == kSingle) {
#pragma unroll
      for (int i = 0; i < 2 * P; ++i) {
        const int column = threadIdx.x + i * blockDim.x;
        if (column < dim) row[column] = from_float<T>(get(i));
      }
    } else {
#pragma unroll
      for (int i = 0; i < P / 4; ++i) {
        const int column = column_of(i);
        const float f[8] = {get(8 * i), get(8 * i + 1), get(8 * i + 2), get(8 * i + 3), get(8 * i + 4), get(8 * i + 5), get(8 * i + 6), get(8 * i + 7)};
        if constexpr (A == kShifted && sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (column + j < dim) row[column + j] = from_float<T>(f[j]);
        } else {
          Eight<T> e;
          e.set(f);
          if constexpr (A == kShifted) store8_shifted(row + column, e, min(8, dim - column), true);
          else if (column < dim) e.store(row + column);
        }
      }
    }
  }
  // A vector of type T or fp32; ones where there is none.
  template <typename T>
  __device__ __forceinline__ void load_vector(const void* vector, bool fp32, int dim) {
    if (!vector) {
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = pack_floats(1.f, 1.f);
    } else if (fp32) {
      load(static_cast<const float*>(vector), dim);
    } else {
      load(static_cast<const T*>(vector), dim);
    }
  }
};

__device__ __forceinline__ float sum_of(uint64_t pair) { return pair_element(pair, 0) + pair_element(pair, 1); }
__device__ __forceinline__ uint64_t twice(float v) { return pack_floats(v, v); }

// The threads of a row wait for one another: a warp, or blockDim.x threads at a barrier of their own.
__device__ __forceinline__ void row_sync() {
  if (blockDim.x == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.y), "r"(blockDim.x) : "memory");
}

// Sum over the threads of a row.  `shared`: 64 floats of the row's own; `turn` alternates so that one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, float* shared, int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (blockDim.x == 32) return v;
  float* slot = shared + 32 * turn;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  row_sync();
  const int warps = blockDim.x >> 5;
  if (warps == 8) {      // (rows of 2049 to 4096 values: two wide loads are sooner done than another round of shuffles; not measured for other rows)
    const float4 a = *reinterpret_cast<const float4*>(slot), b = *reinterpret_cast<const float4*>(slot + 4);
    return ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
  }
  v = (threadIdx.x & 31) < warps ? slot[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kMostGroups = 8, kMostStages = 8, kMostInputs = 4;

// How a row is dealt to threads, and what a group of them keeps ahead.
struct Deal {
  bool ring;
  int access, values, threads, groups, bound;             // values a thread, threads a row, rows at once, threads the kernel is compiled for
  int stages, row_bytes;                                  // of the ring
  int smem, blocks;
};

// The rows of up to four matrices, one row of each a stage.  INPUTS that are absent have a null base.
template <typename T, int INPUTS, int A>
struct Ring {
  Rows inputs[INPUTS];
  uint8_t* data;
  uint64_t* full;
  int stages, row_bytes, dim;
  int stage = 0;
  uint32_t parity = 0;

  __device__ __forceinline__ uintptr_t address(int i, int64_t row) const {
    return reinterpret_cast<uintptr_t>(inputs[i].data) + row * inputs[i].ld * static_cast<int64_t>(sizeof(T));
  }
  // One thread: row's copies into stage `s`, from the 16-byte boundary before it to the one behind.
  __device__ __forceinline__ void fetch(int s, int64_t row) {
    uint32_t bytes[INPUTS], sum = 0;
#pragma unroll
    for (int i = 0; i < INPUTS; ++i) {
      bytes[i] = 0;
      if (inputs[i].data) {
        const uintptr_t from = address(i, row);
        bytes[i] = static_cast<uint32_t>(((from + dim * sizeof(T) + 15) & ~uintptr_t(15)) - (from & ~uintptr_t(15)));
        sum += bytes[i];
      }
    }
    mbar_expect_tx(&full[s], sum);
#pragma unroll
    for (int i = 0; i < INPUTS; ++i)
      if (bytes[i]) bulk_load(data + (s * INPUTS + i) * row_bytes, reinterpret_cast<const void*>(address(i, row) & ~uintptr_t(15)), bytes[i], &full[s]);
  }
  // Input `i` of the current row.
  __device__ __forceinline__ const T* at(int i, int64_t row) const {
    return reinterpret_cast<const T*>(data + (stage * INPUTS + i) * row_bytes + (A == kWhole ? 0 : address(i, row) & 15));
  }
  template <bool RING>
  __device__ __forceinline__ const T* row_at(int i, int64_t row) const {
    return RING ? at(i, row) : reinterpret_cast<const T*>(address(i, row));
  }
  // (a copy of this GPU's own memory always arrives; where it should not have in time, that is recorded, and the results are wrong)
  __device__ __forceinline__ void wait(int* status) {
    for (uint32_t it = 0; it < (1u << 24); ++it)
      if (mbar_try_wait(&full[stage], parity)) return;
    if (status) atomicCAS(status, 0, kStatusRowWaitTimeout);
  }
  // The group is done with the current row; the row `stages` further on takes its place.
  __device__ __forceinline__ void next(int64_t row, int64_t step, int64_t rows) {
    row_sync();
    if (threadIdx.x == 0 && row + stages * step < rows) fetch(stage, row + stages * step);
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  }
  __device__ __forceinline__ void start(int64_t row, int64_t step, int64_t rows) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < stages && row + s * step < rows; ++s) fetch(s, row + s * step);
    }
  }
};

template <typename T, int INPUTS, int A, bool RING>
__device__ __forceinline__ Ring<T, INPUTS, A> make_ring(const Deal& d, int dim, uint8_t* dynamic, uint64_t (&bars)[kMostGroups][kMostStages]) {
  Ring<T, INPUTS, A> ring;
  ring.stages = d.stages; ring.row_bytes = d.row_bytes; ring.dim = dim;
  ring.data = dynamic + static_cast<int64_t>(threadIdx.y) * d.stages * INPUTS * d.row_bytes;
  ring.full = bars[threadIdx.y];
  if constexpr (RING) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < d.stages; ++s) mbar_init(&ring.full[s], 1);
      mbar_fence_init();
    }
    __syncthreads();
  }
  return ring;
}

// Products of a row's vectors: `weight` that y is multiplied by, and scale * gate * branch_weight, which the branch is.
template <typename T, int A, int P>
__device__ __forceinline__ void load_vectors(const NormProblem& p, Lane<A, P>& weight, Lane<A, P>& branch) {
  const bool fp32 = p.vector_type == kFp32;
  weight.template load_vector<T>(p.weight, fp32, p.dim);
  branch.template load_vector<T>(p.branch_weight, fp32, p.dim);
  Lane<A, P> gate;
  gate.template load_vector<T>(p.gate, fp32, p.dim);
#pragma unroll
  for (int i = 0; i < P; ++i) branch.v[i] = mul_pair(mul_pair(branch.v[i], gate.v[i]), twice(p.scale));
}

template <typename T, int A, int P, int THREADS, bool RING, bool AFTER>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1) residual_norm_forward_kernel(NormProblem p, T* __restrict__ h_out, T* __restrict__ y_out, int64_t ld, Deal d) {
  __shared__ __align__(16) float sums[kMostGroups][64];
  __shared__ uint64_t bars[kMostGroups][kMostStages];
  extern __shared__ __align__(128) uint8_t dynamic[];
  float* shared = sums[threadIdx.y];
  int turn = 0;
  Ring<T, 2, A> ring = make_ring<T, 2, A, RING>(d, p.dim, dynamic, bars);
  ring.inputs[0] = p.x; ring.inputs[1] = p.branch;
  wait_for_predecessor();
  let_successor_start();
  const bool with_branch = p.branch.data != nullptr;
  const float inverse_dim = 1.f / static_cast<float>(p.dim);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if constexpr (RING) ring.start(row, step, p.rows);
  Lane<A, P> weight, branch_factor;
  load_vectors<T>(p, weight, branch_factor);
  for (; row < p.rows; row += step) {
    if constexpr (RING) ring.wait(p.status);
    Lane<A, P> h;
    h.load(ring.template row_at<RING>(0, row), p.dim);
    if (with_branch) {
      Lane<A, P> b;
      b.load(ring.template row_at<RING>(1, row), p.dim);
      float r_b = 1.f;
      if (AFTER) {
        uint64_t squares = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) fma_pair(squares, b.v[i], b.v[i]);
        r_b = rsqrtf(row_sum(sum_of(squares), shared, turn) * inverse_dim + p.eps);
        if (threadIdx.x == 0) p.branch_rms[row] = r_b;
      }
#pragma unroll
      for (int i = 0; i < P; ++i) fma_pair(h.v[i], AFTER ? mul_pair(b.v[i], twice(r_b)) : b.v[i], branch_factor.v[i]);
    }
    if (h_out) h.store(h_out + row * ld, p.dim);
    if (y_out) {
      uint64_t squares = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) fma_pair(squares, h.v[i], h.v[i]);
      const float r = rsqrtf(row_sum(sum_of(squares), shared, turn) * inverse_dim + p.eps);
      if (threadIdx.x == 0) p.rms[row] = r;
#pragma unroll
      for (int i = 0; i < P; ++i) h.v[i] = mul_pair(mul_pair(h.v[i], twice(r)), weight.v[i]);
      h.store(y_out + row * ld, p.dim);
    }
    if constexpr (RING) ring.next(row, step, p.rows);
  }
}

// SCALED: the branch has a norm or a gate.
template <typename T, int A, int P, int THREADS, bool RING, bool SCALED>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1)
residual_norm_backward_kernel(NormProblem p, NormGradients g, Deal d) {
  __shared__ __align__(16) float sums[kMostGroups][64];
  __shared__ uint64_t bars[kMostGroups][kMostStages];
  extern __shared__ __align__(128) uint8_t dynamic[];
  float* shared = sums[threadIdx.y];
  int turn = 0;
  Ring<T, 4, A> ring = make_ring<T, 4, A, RING>(d, p.dim, dynamic, bars);
  const bool with_branch = p.branch.data != nullptr;
  ring.inputs[0] = g.grad_y; ring.inputs[1] = g.grad_y.data ? p.x : Rows{nullptr, 0};
  ring.inputs[2] = g.grad_h; ring.inputs[3] = SCALED || g.grad_y.data ? p.branch : Rows{nullptr, 0};
  wait_for_predecessor();
  let_successor_start();
  const float inverse_dim = 1.f / static_cast<float>(p.dim);
  const bool after = SCALED && p.branch_weight;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if constexpr (RING) ring.start(row, step, p.rows);
  Lane<A, P> weight, branch_factor, d_weight, d_branch;      // the last: the sum that both of the branch's vectors' gradients are made of
  load_vectors<T>(p, weight, branch_factor);
  d_weight.clear();
  d_branch.clear();
  // (a row's reciprocal root mean squares travel while the row before it is worked on)
  float r_next = 0.f, r_b_next = 1.f;
  auto look_up = [&](int64_t of) {
    if (of < p.rows) {
      if (g.grad_y.data) r_next = p.rms[of];
      if (after) r_b_next = p.branch_rms[of];
    }
  };
  look_up(row);
  for (; row < p.rows; row += step) {
    const float r = r_next, r_b = r_b_next;
    look_up(row + step);
    if constexpr (RING) ring.wait(p.status);
    Lane<A, P> dh;
    if (g.grad_y.data) {
      Lane<A, P> h;
      h.load(ring.template row_at<RING>(1, row), p.dim);
      if (with_branch) {
        dh.load(ring.template row_at<RING>(3, row), p.dim);
#pragma unroll
        for (int i = 0; i < P; ++i) fma_pair(h.v[i], SCALED ? mul_pair(dh.v[i], twice(r_b)) : dh.v[i], branch_factor.v[i]);
      }
      dh.load(ring.template row_at<RING>(0, row), p.dim);
      uint64_t dot = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint64_t product = mul_pair(dh.v[i], h.v[i]);
        fma_pair(d_weight.v[i], product, twice(r));
        fma_pair(dot, product, weight.v[i]);
        dh.v[i] = mul_pair(dh.v[i], weight.v[i]);
      }
      const float c = row_sum(sum_of(dot), shared, turn) * inverse_dim * r * r;
#pragma unroll
      for (int i = 0; i < P; ++i) dh.v[i] = mul_pair(fma_pair_of(h.v[i], twice(-c), dh.v[i]), twice(r));
    } else {
      dh.clear();
    }
    if (g.grad_h.data) {
      Lane<A, P> gh;
      gh.load(ring.template row_at<RING>(2, row), p.dim);
#pragma unroll
      for (int i = 0; i < P; ++i) add_pair(dh.v[i], gh.v[i]);
    }
    if (g.d_x) dh.store(static_cast<T*>(g.d_x) + row * g.ld, p.dim);
    if constexpr (SCALED) {
      Lane<A, P> b;
      b.load(ring.template row_at<RING>(3, row), p.dim);
      const float by = p.scale * r_b;
      uint64_t dot = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        fma_pair(d_branch.v[i], mul_pair(dh.v[i], b.v[i]), twice(by));
        dh.v[i] = mul_pair(dh.v[i], branch_factor.v[i]);
        fma_pair(dot, dh.v[i], b.v[i]);
      }
      if (after) {
        const float c = row_sum(sum_of(dot), shared, turn) * inverse_dim * r_b * r_b;
#pragma unroll
        for (int i = 0; i < P; ++i) dh.v[i] = mul_pair(fma_pair_of(b.v[i], twice(-c), dh.v[i]), twice(r_b));
      }
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) dh.v[i] = mul_pair(dh.v[i], twice(p.scale));
    }
    if (g.d_branch) dh.store(static_cast<T*>(g.d_branch) + row * g.ld, p.dim);
    if constexpr (RING) ring.next(row, step, p.rows);
  }
  // this block's sums: rows that share the block are added one after another, where the ring was
  float* joined = reinterpret_cast<float*>(dynamic);
  auto leave = [&](const Lane<A, P>& values, int which) {
    float* out = g.partials + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.dim;
    for (int y = 0; y < static_cast<int>(blockDim.y); ++y) {
      if (blockDim.y > 1) __syncthreads();
      if (static_cast<int>(threadIdx.y) == y) {
        Lane<A, P> sum = values;
        if (y) {
          Lane<A, P> before;
          before.load(static_cast<const float*>(joined), p.dim);
#pragma unroll
          for (int i = 0; i < P; ++i) add_pair(sum.v[i], before.v[i]);
        }
        sum.store(y + 1 < static_cast<int>(blockDim.y) ? joined : out, p.dim);
      }
    }
  };
  if (g.d_weight) leave(d_weight, 0);
  if constexpr (SCALED) {
    if (g.d_branch_weight || g.d_gate) leave(d_branch, 1);
  }
}

constexpr int kSumSlices = 8;
// 32 columns a block, the blocks' sums dealt to eight warps.
__global__ void __launch_bounds__(32 * kSumSlices) norm_vectors_kernel(NormProblem p, NormGradients g) {
  __shared__ float shared[kSumSlices][32];
  wait_for_predecessor();
  let_successor_start();
  const int which = blockIdx.y;
  if (which == 0 ? !g.d_weight : !g.d_branch_weight && !g.d_gate) return;
  const int column = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (column < p.dim) {
#pragma unroll 8
    for (int i = threadIdx.y; i < g.blocks; i += kSumSlices) sum += g.partials[(static_cast<int64_t>(i) * 2 + which) * p.dim + column];
  }
  shared[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && column < p.dim) {
#pragma unroll
    for (int s = 1; s < kSumSlices; ++s) sum += shared[s][threadIdx.x];
    auto vector = [&](const void* v) {
      if (!v) return 1.f;
      return p.vector_type == kFp32 ? static_cast<const float*>(v)[column]
                                    : p.vector_type == kFp16 ? __half2float(static_cast<const __half*>(v)[column])
                                                             : __bfloat162float(static_cast<const __nv_bfloat16*>(v)[column]);
    };
    auto write = [&](void* out, float value) {
      if (!out) return;
      if (p.vector_type == kFp32) static_cast<float*>(out)[column] = value;
      else if (p.vector_type == kFp16) static_cast<__half*>(out)[column] = __float2half_rn(value);
      else static_cast<__nv_bfloat16*>(out)[column] = __float2bfloat16_rn(value);
    };
    if (which == 0) {
      write(g.d_weight, sum);
    } else {
      write(g.d_branch_weight, sum * vector(p.gate));
      write(g.d_gate, sum * vector(p.branch_weight));
    }
  }
}

// A warp for every 512 values, rounded up to a power of two, with 16 values a thread: rows of 5120 leave three eighths of the threads without any
// (16384 x 5120 with norm and gate, forward and backward, in 501 us where its bytes take 256; 16384 x 4096 in 260 for 205).  Blocks of eight warps share an SM's shared memory by
// twos or threes (a backward pass's registers allow two).
constexpr int kRingBytes = 216 * 1024;      // of an SM's 227 KB
Deal deal_of(bool wide, int64_t rows, int dim, int size, int inputs, int resident) {
  Deal d{};
  const int warps_of = (dim + 511) / 512;
  int warps = 1;
  while (warps < warps_of) warps *= 2;
  d.access = wide ? kWhole : size == 2 ? kShifted : kSingle;
  d.values = 16;
  d.threads = 32 * warps;
  d.groups = warps < 8 ? 8 / warps : 1;
  d.bound = warps <= 8 ? 256 : 512;
  d.row_bytes = (dim * size + (wide ? 0 : 15) + 15) / 16 * 16;
  const int64_t stage = static_cast<int64_t>(d.groups) * inputs * d.row_bytes;
  for (int ctas = warps <= 8 ? resident : 1; ctas >= 1 && !d.ring; --ctas) {
    d.stages = static_cast<int>(std::min<int64_t>(kMostStages, (kRingBytes / ctas - 4096) / stage));      // (what else a block has is under 4 KB)
    if (d.stages < 2 || warps > 16) continue;
    d.ring = true;
    d.smem = static_cast<int>(d.stages * stage);
    d.blocks = static_cast<int>(std::min<int64_t>((rows + d.groups - 1) / d.groups, int64_t{ctas} * multiprocessors()));
  }
  if (d.ring) return d;
  d.stages = d.row_bytes = 0;
  d.groups = 1;
  if (!wide) d.access = kSingle;
  if (!wide || dim > 1024 * 16) d.values = 32;
  if (dim > 1024 * d.values) throw std::invalid_argument("residual_norm: rows of more than 32768 values are not supported");
  d.threads = ((dim + d.values - 1) / d.values + 31) / 32 * 32;
  d.bound = 1024;
  d.blocks = static_cast<int>(std::min<int64_t>(rows, 2 * multiprocessors()));
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

template <int A_, int P_, int THREADS_, bool RING_>
struct Form {
  static constexpr int A = A_, P = P_, THREADS = THREADS_;
  static constexpr bool RING = RING_;
};
template <typename T, typename F>
void for_deal(const Deal& d, F f) {
  constexpr int kOdd = sizeof(T) == 2 ? kShifted : kSingle;
  if (d.ring) {
    if (d.access == kWhole && d.bound == 256) f(Form<kWhole, 8, 256, true>{});
    else if (d.access == kWhole) f(Form<kWhole, 8, 512, true>{});
    else if (d.bound == 256) f(Form<kOdd, 8, 256, true>{});
    else f(Form<kOdd, 8, 512, true>{});
  } else if (d.access == kWhole) {
    if (d.values == 32) f(Form<kWhole, 16, 1024, false>{});
    else f(Form<kWhole, 8, 1024, false>{});
  } else {
    f(Form<kSingle, 16, 1024, false>{});
  }
}

Deal forward_deal(const NormProblem& p, const void* h, const void* y, int64_t ld) {
  const int size = size_of(p.type);
  return deal_of(wide_problem(p) && on_16(h, ld, size) && on_16(y, ld, size), p.rows, p.dim, size, 2, 2);
}
Deal backward_deal(const NormProblem& p, const NormGradients& g) {
  const int size = size_of(p.type);
  const bool wide = wide_problem(p) && on_16(g.grad_h.data, g.grad_h.ld, size) && on_16(g.grad_y.data, g.grad_y.ld, size) &&
                    on_16(g.d_x, g.ld, size) && on_16(g.d_branch, g.ld, size);
  return deal_of(wide, p.rows, p.dim, size, 4, 2);
}

template <typename Kernel, typename... Arguments>
void start(const char* what, Kernel kernel, const Deal& d, PerDeviceOnce& once, cudaStream_t stream, Arguments&&... arguments) {
  allow_dynamic_smem(reinterpret_cast<const void*>(kernel), kRingBytes, once, what);
  check(launch_dependent(kernel, dim3(d.blocks), dim3(d.threads, d.groups), d.smem, stream, std::forward<Arguments>(arguments)...), what);
}

}  // namespace

int residual_norm_blocks(const NormProblem& p, const NormGradients& g) { return backward_deal(p, g).blocks; }

void residual_norm_forward(const NormProblem& p, void* h, void* y, int64_t ld, cudaStream_t stream) {
  check_problem(p);
  const Deal d = forward_deal(p, h, y, ld);
  for_type(p.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    for_deal<T>(d, [&](auto form) {
      using F = decltype(form);
      static PerDeviceOnce plain, after;
      if (p.branch_weight)
        start("residual_norm_forward", residual_norm_forward_kernel<T, F::A, F::P, F::THREADS, F::RING, true>, d, after, stream, p,
              static_cast<T*>(h), static_cast<T*>(y), ld, d);
      else
        start("residual_norm_forward", residual_norm_forward_kernel<T, F::A, F::P, F::THREADS, F::RING, false>, d, plain, stream, p,
              static_cast<T*>(h), static_cast<T*>(y), ld, d);
    });
  });
}

void residual_norm_backward(const NormProblem& p, const NormGradients& g, cudaStream_t stream) {
  check_problem(p);
  const Deal d = backward_deal(p, g);
  if (g.blocks != d.blocks) throw std::invalid_argument("residual_norm: as many blocks as residual_norm_blocks says");
  for_type(p.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    for_deal<T>(d, [&](auto form) {
      using F = decltype(form);
      static PerDeviceOnce plain, scaled;
      if (p.branch_weight || p.gate)
        start("residual_norm_backward", residual_norm_backward_kernel<T, F::A, F::P, F::THREADS, F::RING, true>, d, scaled, stream, p, g, d);
      else
        start("residual_norm_backward", residual_norm_backward_kernel<T, F::A, F::P, F::THREADS, F::RING, false>, d, plain, stream, p, g, d);
    });
  });
  if (g.d_weight || g.d_branch_weight || g.d_gate)
    check(launch_dependent(norm_vectors_kernel, dim3((p.dim + 31) / 32, 2), dim3(32, kSumSlices), 0, stream, p, g), "norm_vectors");
}

}  // namespace soapb200
