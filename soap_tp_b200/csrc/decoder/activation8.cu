// Activations kept in 8 bits for the backward pass: what a block or a gated MLP would keep in 16, at 8.5 bits a value.
//
//   scale = max |x| / 127 over 64 neighbouring features of a row      q = round(x / scale)      x' = q scale
//
// so |x - x'| is at most half a step, max |x| / 254.  A scale is not less than 2^-126, so that its reciprocal is finite, nor so large that 127 of it
// are not: fp32's largest number, rounded up as a quotient, would come back as an infinity.  A group with an infinity or a NaN in it gets a NaN as its scale and comes back as NaN: nothing that went wrong is lost.
//
// y = silu(g) u keeps g and u this way, and its backward pass works from them: dg = dy u' s (1 + g' (1 - s)), du = dy g' s with
// s = sigmoid(g').
//
// Memory bounds all four, once instructions do not: eight threads take a group, eight values each (16-byte loads and stores of 16-bit types,
// 8-byte ones of the kept values), and the group's maximum goes round with three shuffles.  Magnitudes of 16-bit values are compared two at a
// time as they lie; a value becomes its whole number by a multiply-add and an addition that leave it in the low byte of 1.5 * 2^23 + q, and comes back
// as the low byte of 2^23 + q + 128.  (Conversion instructions, at a quarter of the rate, and a division for each address made 19
// instructions a value and bounded packing at 32768 x 4096: 112 us where its bytes take 63.)
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
constexpr int kTurns = 2;        // runs of eight values that a thread packs or unpacks
constexpr int kGroupThreads = kScaleGroup / kPerThread;
constexpr float kSmallestScale = 1.17549435e-38f;      // 2^-126
constexpr float kLargestScale = 0x1.020406p+121f;      // 127 of it round to a number just below the largest

// Division of numbers below 2^31 by a number that is known before the launch: (n m) >> (32 + s) with m = ceil(2^(32 + s) / d), s =
// ceil(log2 d) - 1 (Granlund and Montgomery, 1994; d = 1 apart).
struct Divisor {
  uint32_t d, multiplier, shift;
  explicit Divisor(uint32_t divisor) : d(divisor), multiplier(0), shift(0) {
    if (d == 1) return;
    while ((uint64_t{1} << (shift + 1)) < d) ++shift;
    multiplier = static_cast<uint32_t>(((uint64_t{1} << (32 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1 ? n : __umulhi(n, multiplier) >> shift; }
};

struct Shape {
  uint32_t count;                // groups in all
  int dim;
  Divisor groups;                // of a row
};

// Where this thread's eight values are.
struct Place {
  uint32_t group;                // of all
  int64_t row;
  int column, valid;             // valid <= 0: beyond the row
  __device__ __forceinline__ explicit Place(const Shape& s, uint32_t block = blockIdx.x) {
    group = block * static_cast<uint32_t>(kThreads / kGroupThreads) + threadIdx.x / kGroupThreads;
    row = s.groups.of(group);
    column = static_cast<int>(group - static_cast<uint32_t>(row) * s.groups.d) * kScaleGroup + (threadIdx.x % kGroupThreads) * kPerThread;
    valid = group < s.count ? min(kPerThread, s.dim - column) : 0;
  }
};

// WIDE: all rows lie on 16-byte boundaries and are multiples of eight values long.  Otherwise 16-bit rows are shifted as they are moved, and fp32
// values go one by one.
template <bool WIDE, typename T>
__device__ __forceinline__ Eight<T> load8(const T* p, int valid) {
  Eight<T> e;
  if constexpr (WIDE) {
    if (valid > 0) e.load(p);
    else e.clear();
  } else if constexpr (sizeof(T) == 2) {
    e = load8_shifted(p, valid);
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? p[i] : 0.f;
    e.set(v);
  }
  return e;
}
// All 32 lanes call.
template <bool WIDE, typename T>
__device__ __forceinline__ void store8(T* p, const Place& place, const float (&v)[8]) {
  Eight<T> e;
  e.set(v);
  if constexpr (WIDE) {
    if (place.valid > 0) e.store(p);
  } else if constexpr (sizeof(T) == 2) {
    store8_shifted(p, e, place.valid, place.column != 0);      // (lanes go along rows)
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < place.valid) p[i] = v[i];
  }
}

// The largest magnitude of a group whose eight threads hold its values, as bits of fp32; all 32 lanes call.  Magnitudes are compared as whole numbers: infinities and NaN
// come out above all others.
template <typename T>
__device__ __forceinline__ uint32_t group_most(const Eight<T>& e) {
  uint32_t most;
  if constexpr (sizeof(T) == 4) {
    const uint32_t w[8] = {e.words[0].x, e.words[0].y, e.words[0].z, e.words[0].w, e.words[1].x, e.words[1].y, e.words[1].z, e.words[1].w};
    most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, w[i] & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < kGroupThreads; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  } else {
    constexpr uint32_t kMagnitude = 0x7fff7fffu;
    most = __vmaxu2(__vmaxu2(e.words[0].x & kMagnitude, e.words[0].y & kMagnitude), __vmaxu2(e.words[0].z & kMagnitude, e.words[0].w & kMagnitude));
#pragma unroll
    for (int o = 1; o < kGroupThreads; o <<= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
    most = max(most & 0xffffu, most >> 16);
    if constexpr (std::is_same<T, __half>::value) most = __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(most))));
    else most <<= 16;
  }
  return most;
}
__device__ __forceinline__ float scale_of(uint32_t most) {
  return most >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fminf(fmaxf(__uint_as_float(most) / 127.f, kSmallestScale), kLargestScale);
}

// 127 x / max of 16-bit values is often a tie, which a rounded reciprocal would move to either side (2e-4 of fp16 values, 1e-3 of bf16 ones).  So
// x (127 / max) is first rounded to multiples of 2^-15, by adding it to 384: it is off by 127 2^-24 at most, less than half of 2^-15, and every tie is
// such a multiple.  What is not a tie but within 2^-16 + 127 2^-24 of one may become it (1e-6 of fp16 values).
// At 32768 x 4096, there and back, it costs 3 to 6 us of 142 to 145.  fp32 values are divided by their scale.
template <typename T>
__device__ __forceinline__ uint2 quantise(const Eight<T>& e, uint32_t most, float scale) {
  constexpr float kShift = 12582912.f;       // 1.5 * 2^23: its neighbours are whole numbers, in two's complement in the low byte
  constexpr float kGrid = 384.f;             // sums with -127 to 127 lie between 2^8 and 2^9
  float v[8];
  e.get(v);
  uint32_t bits[8];
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bits[i] = __float_as_uint(v[i] / scale + kShift);
  } else {
    const float steps = 127.f / fmaxf(__uint_as_float(most), 127.f * kSmallestScale);
#pragma unroll
    for (int i = 0; i < 8; ++i) bits[i] = __float_as_uint(fmaf(v[i], steps, kGrid) + (kShift - kGrid));
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(bits[4 * i], bits[4 * i + 1], 0x0040), __byte_perm(bits[4 * i + 2], bits[4 * i + 3], 0x0040), 0x5410);
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void dequantise(uint2 q, float scale, float (&v)[8]) {
  constexpr uint32_t kBits = 0x4b000000u;    // 2^23
  const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (__uint_as_float(__byte_perm(w[i / 4], kBits, 0x7650 | (i & 3))) - 8388736.f) * scale;
}

// All 32 lanes call.
template <typename T>
__device__ __forceinline__ void keep(const Kept8& kept, const Shape& shape, const Place& p, const Eight<T>& e) {
  const uint32_t most = group_most(e);
  const float scale = scale_of(most);
  if (p.valid > 0) *reinterpret_cast<uint2*>(kept.values + p.row * kept.pitch + p.column) = quantise(e, most, scale);
  if (threadIdx.x % kGroupThreads == 0 && p.group < shape.count) kept.scales[p.group] = scale;
}

__device__ __forceinline__ void kept_values(const Kept8& kept, const Place& p, float (&v)[8]) {
  if (p.valid <= 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    return;
  }
  dequantise(*reinterpret_cast<const uint2*>(kept.values + p.row * kept.pitch + p.column), kept.scales[p.group], v);
}

// 1 / (1 + e^-x), down to 2^-150: where 1 + e^-x itself is the divisor, silu is 0 below -87.3 or -88.7, though 1e37 silu(-88) is -0.5.
// fp32: t / (1 + t) or 1 / (1 + t) with t = e^-|x|, whose divisor is at most 2.
// 16 bits: 2^-24 / (2^-24 + 2^(-x log2 e - 24)), whose divisor overflows at x = -105 and is no more work.  The exponent's rounding makes it off by 2^-20
// near zero and by |x| 2^-23 far from it, where results are rounded to 2^-9 or 2^-12.
template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (std::is_same<T, float>::value) {
    const float t = expf(-fabsf(x));
    return (x < 0.f ? t : 1.f) / (1.f + t);
  } else {
    constexpr float kLog2e = 1.4426950408889634f, kDown = 5.9604644775390625e-8f;      // 2^-24
    float power, reciprocal;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(fmaf(x, -kLog2e, -24.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(reciprocal) : "f"(kDown + power));
    return reciprocal * kDown;
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) pack8_kernel(const T* __restrict__ x, int64_t ld, Shape shape, Kept8 kept) {
  wait_for_predecessor();
  let_successor_start();
  // (two loads under way in a thread: 32768 x 4096 values there and back in 129 us, one 154, four 132, before ties were rounded as ties)
  Eight<T> e[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const Place p(shape, blockIdx.x * kTurns + i);
    e[i] = load8<WIDE>(x + p.row * ld + p.column, p.valid);
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) keep(kept, shape, Place(shape, blockIdx.x * kTurns + i), e[i]);
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) unpack8_kernel(Kept8 kept, Shape shape, T* __restrict__ out, int64_t ld) {
  wait_for_predecessor();
  let_successor_start();
  uint2 q[kTurns];
  float scale[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const Place p(shape, blockIdx.x * kTurns + i);
    q[i] = p.valid > 0 ? *reinterpret_cast<const uint2*>(kept.values + p.row * kept.pitch + p.column) : make_uint2(0, 0);
    scale[i] = p.valid > 0 ? kept.scales[p.group] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const Place p(shape, blockIdx.x * kTurns + i);
    float v[8];
    dequantise(q[i], scale[i], v);
    store8<WIDE>(out + p.row * ld + p.column, p, v);
  }
}

template <typename T, bool WIDE, bool KEEP>
__global__ void __launch_bounds__(kThreads)
swiglu8_forward_kernel(const T* __restrict__ gate, int64_t ld_gate, const T* __restrict__ up, int64_t ld_up, Shape shape,
                       T* __restrict__ y, int64_t ld, Kept8 gate8, Kept8 up8) {
  wait_for_predecessor();
  let_successor_start();
  const Place p(shape);
  const Eight<T> g8 = load8<WIDE>(gate + p.row * ld_gate + p.column, p.valid);
  const Eight<T> u8 = load8<WIDE>(up + p.row * ld_up + p.column, p.valid);
  if (KEEP) {
    keep(gate8, shape, p, g8);
    keep(up8, shape, p, u8);
  }
  float g[8], u[8];
  g8.get(g);
  u8.get(u);
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] *= g[i] * sigmoid<T>(g[i]);
  store8<WIDE>(y + p.row * ld + p.column, p, u);
}

template <typename T, bool WIDE, bool WITH_Y>
__global__ void __launch_bounds__(kThreads)
swiglu8_backward_kernel(const T* __restrict__ grad, int64_t ld_grad, Kept8 gate8, Kept8 up8, Shape shape, T* __restrict__ d_gate,
                        T* __restrict__ d_up, T* __restrict__ y, int64_t ld) {
  wait_for_predecessor();
  let_successor_start();
  const Place p(shape);
  float d[8], g[8], u[8], out_g[8], out_u[8];
  const Eight<T> d8 = load8<WIDE>(grad + p.row * ld_grad + p.column, p.valid);
  kept_values(gate8, p, g);
  kept_values(up8, p, u);
  d8.get(d);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = sigmoid<T>(g[i]), silu = g[i] * s;
    out_u[i] = d[i] * silu;
    out_g[i] = d[i] * u[i] * fmaf(silu, 1.f - s, s);
    if (WITH_Y) u[i] *= silu;
  }
  const int64_t at = p.row * ld + p.column;
  store8<WIDE>(d_gate + at, p, out_g);
  store8<WIDE>(d_up + at, p, out_u);
  if (WITH_Y) store8<WIDE>(y + at, p, u);
}

bool on_16(const void* data, int64_t ld, int size) { return (reinterpret_cast<uintptr_t>(data) & 15) == 0 && (ld * size) % 16 == 0; }

Shape shape_of(int64_t rows, int dim) {
  if (rows < 0 || dim < 1) throw std::invalid_argument("activation8: bad shape");
  const int64_t groups = (static_cast<int64_t>(dim) + kScaleGroup - 1) / kScaleGroup;
  if (rows * groups > INT32_MAX) throw std::invalid_argument("activation8: more than 2^31 - 1 groups of 64 values");
  return Shape{static_cast<uint32_t>(rows * groups), dim, Divisor(static_cast<uint32_t>(groups))};
}

void check_kept(const Kept8& kept, int dim) {
  if (kept.pitch % 8 != 0 || kept.pitch < dim || (reinterpret_cast<uintptr_t>(kept.values) & 7) != 0)
    throw std::invalid_argument("activation8: kept rows lie on 8-byte boundaries");
}

template <typename... P, typename... A>
void start(const char* what, void (*kernel)(P...), const Shape& shape, int turns, cudaStream_t stream, A&&... arguments) {
  const uint32_t groups = turns * (kThreads / kGroupThreads);      // of a block
  const dim3 grid((shape.count + groups - 1) / groups);
  const cudaError_t err = launch_dependent(kernel, grid, dim3(kThreads), 0, stream, std::forward<A>(arguments)...);
  if (err != cudaSuccess) throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(err));
}

// f(type, whether rows are wide)
template <typename F>
void for_type(int type, bool wide, F f) {
  auto with = [&](auto* t) {
    if (wide) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (type == kBf16) with(static_cast<__nv_bfloat16*>(nullptr));
  else if (type == kFp16) with(static_cast<__half*>(nullptr));
  else if (type == kFp32) with(static_cast<float*>(nullptr));
  else throw std::invalid_argument("activation8: unknown type");
}

int size_of(int type) { return type == kFp32 ? 4 : 2; }

}  // namespace

void pack8(int type, const Rows& x, int64_t rows, int dim, const Kept8& kept, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  check_kept(kept, dim);
  if (rows == 0) return;
  for_type(type, dim % 8 == 0 && on_16(x.data, x.ld, size_of(type)), [&](auto* t, auto wide) {
    using T = std::remove_pointer_t<decltype(t)>;
    start("pack8", pack8_kernel<T, decltype(wide)::value>, shape, kTurns, stream, static_cast<const T*>(x.data), x.ld, shape, kept);
  });
}

void unpack8(int type, const Kept8& kept, int64_t rows, int dim, void* out, int64_t ld, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  check_kept(kept, dim);
  if (rows == 0) return;
  for_type(type, dim % 8 == 0 && on_16(out, ld, size_of(type)), [&](auto* t, auto wide) {
    using T = std::remove_pointer_t<decltype(t)>;
    start("unpack8", unpack8_kernel<T, decltype(wide)::value>, shape, kTurns, stream, kept, shape, static_cast<T*>(out), ld);
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
  const int size = size_of(type);
  for_type(type, dim % 8 == 0 && on_16(gate.data, gate.ld, size) && on_16(up.data, up.ld, size) && on_16(y, ld, size), [&](auto* t, auto wide) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr bool kWide = decltype(wide)::value;
    start("swiglu8_forward", gate8 ? swiglu8_forward_kernel<T, kWide, true> : swiglu8_forward_kernel<T, kWide, false>, shape, 1, stream,
          static_cast<const T*>(gate.data), gate.ld, static_cast<const T*>(up.data), up.ld, shape, static_cast<T*>(y), ld,
          gate8 ? *gate8 : Kept8{}, gate8 ? *up8 : Kept8{});
  });
}

void swiglu8_backward(int type, const Rows& grad, const Kept8& gate8, const Kept8& up8, int64_t rows, int dim, void* d_gate, void* d_up,
                      void* y, int64_t ld, cudaStream_t stream) {
  const Shape shape = shape_of(rows, dim);
  check_kept(gate8, dim);
  check_kept(up8, dim);
  if (rows == 0) return;
  const int size = size_of(type);
  for_type(type, dim % 8 == 0 && on_16(grad.data, grad.ld, size) && on_16(d_gate, ld, size) && on_16(d_up, ld, size) && (!y || on_16(y, ld, size)),
           [&](auto* t, auto wide) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr bool kWide = decltype(wide)::value;
    start("swiglu8_backward", y ? swiglu8_backward_kernel<T, kWide, true> : swiglu8_backward_kernel<T, kWide, false>, shape, 1, stream,
          static_cast<const T*>(grad.data), grad.ld, gate8, up8, shape, static_cast<T*>(d_gate), static_cast<T*>(d_up),
          static_cast<T*>(y), ld);
  });
}

}  // namespace soapb200
