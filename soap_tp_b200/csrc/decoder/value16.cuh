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
  __device__ __forceinline__ void load_streamed(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) words[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
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

// The first `valid` of eight values, element by element where `wide` does not say that all eight lie on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void read_eight(const T* p, int valid, bool wide, float (&v)[8]) {
  if (wide && valid >= 8) {
    Eight<T> e;
    e.load(p);
    e.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_float(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void write_eight(T* p, int valid, bool wide, const float (&v)[8]) {
  if (wide && valid >= 8) {
    Eight<T> e;
    e.set(v);
    e.store(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = from_float<T>(v[i]);
  }
}

}  // namespace soapb200
