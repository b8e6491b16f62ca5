// Activations kept in 8 bits (activation8.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace soapb200 {

enum ValueType : int { kBf16 = 0, kFp16 = 1, kFp32 = 2 };
constexpr int kScaleGroup = 64;      // neighbouring features that share a scale

// rows x dim values as 8-bit whole numbers, `pitch` (a multiple of 8) bytes between rows, and one scale per row and group of 64.
struct Kept8 {
  int8_t* values;
  int64_t pitch;
  float* scales;      // [rows][ceil(dim / 64)]
};
struct Rows {
  const void* data;
  int64_t ld;         // elements between rows
};

void pack8(int type, const Rows& x, int64_t rows, int dim, const Kept8& kept, cudaStream_t stream);
void unpack8(int type, const Kept8& kept, int64_t rows, int dim, void* out, int64_t ld, cudaStream_t stream);
// y = silu(gate) * up; with `gate8` both are kept as well.
void swiglu8_forward(int type, const Rows& gate, const Rows& up, int64_t rows, int dim, void* y, int64_t ld, const Kept8* gate8,
                     const Kept8* up8, cudaStream_t stream);
// Gradients of gate and up at the kept values; `y` (or null): silu(gate) * up of them.
void swiglu8_backward(int type, const Rows& grad, const Kept8& gate8, const Kept8& up8, int64_t rows, int dim, void* d_gate, void* d_up,
                      void* y, int64_t ld, cudaStream_t stream);

}  // namespace soapb200
