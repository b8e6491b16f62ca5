// Activations kept in 8 bits for the backward pass: what a block or a gated MLP would keep in 16, at 8.5 bits a value.
//
//   scale = max |x| / 127 over 64 neighbouring features of a row      q = round(x / scale)      x' = q scale
//
// so |x - x'| is at most half a step, max |x| / 254.  A scale is not less than 2^-126, so that its reciprocal is finite; a group with
// an infinity or a NaN in it gets a NaN as its scale and comes back as NaN: nothing that went wrong is lost.
//
// y = silu(g) u keeps g and u this way, and its backward pass works from them: dg = dy u' s (1 + g' (1 - s)), du = dy g' s with
// s = sigmoid(g').
//
// Memory bounds all four: eight threads take a group, eight values each (16-byte loads and stores of 16-bit types, 8-byte ones of
// the kept values), and the group's maximum goes round with three shuffles.
#include <cuda_runtime.h>

#include <stdexcept>
#include <string>

#include "activation8.h"
#include "launch_util.h"
#include "value16.cuh"

namespace soapb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 8;
constexpr int kGroupThreads = kScaleGroup / kPerThread;
constexpr float kSmallestScale = 1.17549435e-38f;      // 2^-126

// Where this thread's eight values are.
struct Place {
  int64_t row;
  int group, column, valid;      // valid <= 0: beyond the row
};

struct Shape {
  int64_t rows;
  int dim, groups;               // groups of a row
  __device__ __forceinline__ bool place(int64_t group, int lane8, Place& p) const {
    if (group >= rows * groups) return false;
    if (rows * groups <= 0x7fffffff) {
      p.row = static_cast<uint32_t>(group) / static_cast<uint32_t>(groups);
      p.group = static_cast<int>(static_cast<uint32_t>(group) - static_cast<uint32_t>(p.row) * static_cast<uint32_t>(groups));
    } else {
      p.row = group / groups;
      p.group = static_cast<int>(group - p.row * groups);
    }
    p.column = p.group * kScaleGroup + lane8 * kPerThread;
    p.valid = min(kPerThread, dim - p.column);
    return true;
  }
};

__device__ __forceinline__ int64_t first_group() {
  return (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kGroupThreads;
}

// The scale of a group whose eight threads hold its values; all 32 lanes call.
__device__ __forceinline__ float group_scale(const float (&v)[8]) {
  uint32_t most = 0;                       // of the magnitudes' bits: infinities and NaN come out above all numbers
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < kGroupThreads; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  return most >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fmaxf(__uint_as_float(most) / 127.f, kSmallestScale);
}

// 16-bit values are multiplied by the reciprocal, whose rounding can move what lies within 2^-16 of a step from a tie to the other side;
// fp32 values, which come back exactly but for their step, are divided.
template <typename T>
__device__ __forceinline__ uint2 quantise(const float (&v)[8], float scale) {
  const float inverse = 1.f / scale;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float quotient = std::is_same<T, float>::value ? v[i] / scale : v[i] * inverse;
    w[i / 4] |= (static_cast<uint32_t>(__float2int_rn(quotient)) & 0xffu) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void dequantise(uint2 q, float scale, float (&v)[8]) {
  const uint32_t w[2] = {q.x, q.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i & 3)))) * scale;
}

template <typename T>
__device__ __forceinline__ void keep(const Kept8& kept, const Shape& shape, const Place& p, bool here, int lane8, const float (&v)[8]) {
  const float scale = group_scale(v);
  if (!here) return;
  if (p.valid > 0) *reinterpret_cast<uint2*>(kept.values + p.row * kept.pitch + p.column) = quantise<T>(v, scale);
  if (lane8 == 0) kept.scales[p.row * shape.groups + p.group] = scale;
}

__device__ __forceinline__ void kept_values(const Kept8& kept, const Shape& shape, const Place& p, float (&v)[8]) {
  dequantise(*reinterpret_cast<const uint2*>(kept.values + p.row * kept.pitch + p.column),
             kept.scales[p.row * shape.groups + p.group], v);
}

template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (std::is_same<T, float>::value) {
    return 1.f / (1.f + expf(-x));
  } else {
    return __fdividef(1.f, 1.f + __expf(-x));      // off by some 2^-20 where the result is rounded to 2^-9 or 2^-12
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pack8_kernel(const T* __restrict__ x, int64_t ld, Shape shape, Kept8 kept, bool wide) {
  wait_for_predecessor();
  let_successor_start();
  const int lane8 = threadIdx.x % kGroupThreads;
  Place p{};
  const bool here = shape.place(first_group(), lane8, p);
  float v[8];
  read_eight(x + p.row * ld + p.column, here ? p.valid : 0, wide, v);
  keep<T>(kept, shape, p, here, lane8, v);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack8_kernel(Kept8 kept, Shape shape, T* __restrict__ out, int64_t ld, bool wide) {
  wait_for_predecessor();
  let_successor_start();
  Place p{};
  if (!shape.place(first_group(), threadIdx.x % kGroupThreads, p) || p.valid <= 0) return;
  float v[8];
  kept_values(kept, shape, p, v);
  write_eight(out + p.row * ld + p.column, p.valid, wide, v);
}

template <typename T, bool KEEP>
__global__ void __launch_bounds__(kThreads)
swiglu8_forward_kernel(const T* __restrict__ gate, int64_t ld_gate, const T* __restrict__ up, int64_t ld_up, Shape shape,
                       T* __restrict__ y, int64_t ld, Kept8 gate8, Kept8 up8, bool wide) {
  wait_for_predecessor();
  let_successor_start();
  const int lane8 = threadIdx.x % kGroupThreads;
  Place p{};
  const bool here = shape.place(first_group(), lane8, p);
  const int valid = here ? p.valid : 0;
  float g[8], u[8];
  read_eight(gate + p.row * ld_gate + p.column, valid, wide, g);
  read_eight(up + p.row * ld_up + p.column, valid, wide, u);
  if (KEEP) {
    keep<T>(gate8, shape, p, here, lane8, g);
    keep<T>(up8, shape, p, here, lane8, u);
  }
  if (valid <= 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] *= g[i] * sigmoid<T>(g[i]);
  write_eight(y + p.row * ld + p.column, valid, wide, u);
}

template <typename T, bool WITH_Y>
__global__ void __launch_bounds__(kThreads)
swiglu8_backward_kernel(const T* __restrict__ grad, int64_t ld_grad, Kept8 gate8, Kept8 up8, Shape shape, T* __restrict__ d_gate,
                        T* __restrict__ d_up, T* __restrict__ y, int64_t ld, bool wide) {
  wait_for_predecessor();
  let_successor_start();
  Place p{};
  if (!shape.place(first_group(), threadIdx.x % kGroupThreads, p) || p.valid <= 0) return;
  float d[8], g[8], u[8], out_g[8], out_u[8];
  read_eight(grad + p.row * ld_grad + p.column, p.valid, wide, d);
  kept_values(gate8, shape, p, g);
  kept_values(up8, shape, p, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = sigmoid<T>(g[i]), silu = g[i] * s;
    out_u[i] = d[i] * silu;
    out_g[i] = d[i] * u[i] * (s + silu * (1.f - s));
    if (WITH_Y) u[i] *= silu;
  }
  const int64_t at = p.row * ld + p.column;
  write_eight(d_gate + at, p.valid, wide, out_g);
  write_eight(d_up + at, p.valid, wide, out_u);
  if (WITH_Y) write_eight(y + at, p.valid, wide, u);
}

bool on_16(const void* data, int64_t ld, int size) { return (reinterpret_cast<uintptr_t>(data) & 15) == 0 && (ld * size) % 16 == 0; }

Shape shape_of(int64_t rows, int dim) {
  if (rows < 0 || dim < 1) throw std::invalid_argument("activation8: bad shape");
  return Shape{rows, dim, (dim + kScaleGroup - 1) / kScaleGroup};
}

void check_kept(const Kept8& kept, int dim) {
  if (kept.pitch % 8 != 0 || kept.pitch < dim || (reinterpret_cast<uintptr_t>(kept.values) & 7) != 0)
    throw std::invalid_argument("activation8: kept rows lie on 8-byte boundaries");
}

dim3 grid_of(const Shape& s) {
  const int64_t blocks = (s.rows * s.groups * kGroupThreads + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) throw std::invalid_argument("activation8: too many values");
  return dim3(static_cast<unsigned>(blocks));
}

template <typename... P, typename... A>
void start(const char* what, void (*kernel)(P...), const Shape& shape, cudaStream_t stream, A&&... arguments) {
  const cudaError_t err = launch_dependent(kernel, grid_of(shape), dim3(kThreads), 0, stream, std::forward<A>(arguments)...);
  if (err != cudaSuccess) throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(err));
}

template <typename F>
void for_type(int type, F f) {
  if (type == kBf16) f(static_cast<__nv_bfloat16*>(nullptr));
  else if (type == kFp16) f(static_cast<__half*>(nullptr));
  else if (type == kFp32) f(static_cast<float*>(nullptr));
  else throw std::invalid_argument("activation8: unknown type");
}

}  // namespace

void pack8(int type, const Rows& x, int64_t rows, int dim, const Kept8& kept, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  check_kept(kept, dim);
  if (rows == 0) return;
  for_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    start("pack8", pack8_kernel<T>, shape, stream, static_cast<const T*>(x.data), x.ld, shape, kept, on_16(x.data, x.ld, sizeof(T)));
  });
}

void unpack8(int type, const Kept8& kept, int64_t rows, int dim, void* out, int64_t ld, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  check_kept(kept, dim);
  if (rows == 0) return;
  for_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    start("unpack8", unpack8_kernel<T>, shape, stream, kept, shape, static_cast<T*>(out), ld, on_16(out, ld, sizeof(T)));
  });
}

void swiglu8_forward(int type, const Rows& gate, const Rows& up, int64_t rows, int dim, void* y, int64_t ld, const Kept8* gate8,
                     const Kept8* up8, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  if (gate8) {
    check_kept(*gate8, dim);
    check_kept(*up8, dim);
  }
  if (rows == 0) return;
  for_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool wide = on_16(gate.data, gate.ld, sizeof(T)) && on_16(up.data, up.ld, sizeof(T)) && on_16(y, ld, sizeof(T));
    start("swiglu8_forward", gate8 ? swiglu8_forward_kernel<T, true> : swiglu8_forward_kernel<T, false>, shape, stream,
          static_cast<const T*>(gate.data), gate.ld, static_cast<const T*>(up.data), up.ld, shape, static_cast<T*>(y), ld,
          gate8 ? *gate8 : Kept8{}, gate8 ? *up8 : Kept8{}, wide);
  });
}

void swiglu8_backward(int type, const Rows& grad, const Kept8& gate8, const Kept8& up8, int64_t rows, int dim, void* d_gate, void* d_up,
                      void* y, int64_t ld, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  check_kept(gate8, dim);
  check_kept(up8, dim);
  if (rows == 0) return;
  for_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool wide = on_16(grad.data, grad.ld, sizeof(T)) && on_16(d_gate, ld, sizeof(T)) && on_16(d_up, ld, sizeof(T)) &&
                      (!y || on_16(y, ld, sizeof(T)));
    start("swiglu8_backward", y ? swiglu8_backward_kernel<T, true> : swiglu8_backward_kernel<T, false>, shape, stream,
          static_cast<const T*>(grad.data), grad.ld, gate8, up8, shape, static_cast<T*>(d_gate), static_cast<T*>(d_up),
          static_cast<T*>(y), ld, wide);
  });
}

}  // namespace soapb200
