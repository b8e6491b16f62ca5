// Reading and writing runs of eight values of any floating type as fp32 (elementwise kernels of the decoder's operators).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace soapb200 {

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float low, float high) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Eight values as they lie in memory.
template <typename T>
struct Eight {
  uint4 words[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) words[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = words[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) words[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[4 * i] = __uint_as_float(words[i].x); v[4 * i + 1] = __uint_as_float(words[i].y);
        v[4 * i + 2] = __uint_as_float(words[i].z); v[4 * i + 3] = __uint_as_float(words[i].w);
      }
    } else {
      const uint32_t w[4] = {words[0].x, words[0].y, words[0].z, words[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        words[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
    } else {
      words[0] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  }
};

// ---- rows that do not lie on 16-byte boundaries (16-bit types) ----------------------------------------------------------
// A row of odd length puts every other row off the boundary.  Value by value, eight to a thread, such rows moved at a third of the speed
// of others (30000 x 1333 unpacked in 110 us, 30000 x 1344 in 24); so they too go in whole 16-byte words, moved along by `s` values.

// Words `s` 16-bit values (0 to 8) on in two neighbouring 16-byte words.
__device__ __forceinline__ uint4 window(const uint4& low, const uint4& high, int s) {
  uint32_t w[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
  if (s & 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = w[i + 4];
  }
  if (s & 4) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (s & 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (s & 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The first `valid` (at most 8) values from `p` on, zeros for the others.  What is read are the 16-byte words that hold one of them.
template <typename T>
__device__ __forceinline__ Eight<T> load8_shifted(const T* p, int valid) {
  static_assert(sizeof(T) == 2, "16-bit values");
  Eight<T> e;
  e.clear();
  if (valid <= 0) return e;
  const int s = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) >> 1);
  const uint4* words = reinterpret_cast<const uint4*>(p - s);
  const uint4 low = words[0];
  const uint4 high = s + valid > 8 ? words[1] : low;
  e.words[0] = window(low, high, s);
  if (valid < 8) {
    uint32_t w[4] = {e.words[0].x, e.words[0].y, e.words[0].z, e.words[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i + 1 < valid ? w[i] : 2 * i < valid ? w[i] & 0xffffu : 0u;
    e.words[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return e;
}

// The first `valid` of eight values to `p` on.  All 32 lanes call; `follows`: the lane before has the eight values before these, all
// valid.  A lane stores the 16-byte word that ends with its values, the first of which it has from the lane before; what no such word holds, at
// the ends of rows and of warps, is stored value by value.
template <typename T>
__device__ __forceinline__ void store8_shifted(T* p, const Eight<T>& e, int valid, bool follows) {
  static_assert(sizeof(T) == 2, "16-bit values");
  const int s = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) >> 1);
  const uint4 mine = e.words[0];
  const uint4 before = make_uint4(__shfl_up_sync(0xffffffffu, mine.x, 1), __shfl_up_sync(0xffffffffu, mine.y, 1),
                                  __shfl_up_sync(0xffffffffu, mine.z, 1), __shfl_up_sync(0xffffffffu, mine.w, 1));
  const bool takes = valid >= 8 - s && valid > 0 && (s == 0 || (follows && (threadIdx.x & 31) != 0));
  const bool next_takes = __shfl_down_sync(0xffffffffu, takes && follows, 1) && (threadIdx.x & 31) != 31;
  if (takes) *reinterpret_cast<uint4*>(p - s) = window(before, mine, 8 - s);
  const int head = takes ? 8 - s : 0, tail = next_takes ? 8 - s : 8;      // (a lane that follows has the same shift)
  if (head < min(tail, valid)) {
    const uint32_t w[4] = {mine.x, mine.y, mine.z, mine.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= head && i < tail && i < valid) reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
  }
}

}  // namespace soapb200
