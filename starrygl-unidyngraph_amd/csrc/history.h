// Shared pieces of the history operators (gated scan, cross attention, gated
// norm): element types, vector access at any alignment, MFMA fragments over
// the three types, and the sum of per-workgroup partial rows.
#pragma once

#include <cstdint>

#include "common.h"
#include "mfma.h"

namespace sgl {

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;

// One 16-byte vector of a type (8 or 4 elements).
template <typename T>
struct Vec16 {
  static constexpr int E = 16 / int(sizeof(T));
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};

// N consecutive elements at the element type's own alignment (the hardware
// takes a global vector access at any address that is a multiple of four
// bytes or not; the compiler emits one wide load or store).
template <typename T, int N>
__device__ __forceinline__ void load_n(T (&r)[N], const T *__restrict__ p) {
  __builtin_memcpy(r, p, sizeof(r));
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T *__restrict__ p, const T (&r)[N]) {
  __builtin_memcpy(p, r, sizeof(r));
}

// s(x) and s(-x) without cancellation at either end: t = exp(-|x|).
__device__ __forceinline__ void sigmoid_pair(float x, float &s, float &sn) {
  const float t = __expf(-fabsf(x));
  const float big = __builtin_amdgcn_rcpf(1.f + t), small = t * big;
  s = x >= 0.f ? big : small;
  sn = x >= 0.f ? small : big;
}

// out[c] = sum over rows of part[row][c], c < width, in double and in one
// order. A workgroup takes 8 columns (32 bytes of each row), a thread every
// 128th row of one, 8 loads in flight: narrow matrices of many rows still
// give every CU something (4,000 x 172: 20 us with 64 columns a workgroup).
constexpr int kSumCols = 8, kSumRows = 128;
static __global__ __launch_bounds__(kSumCols * kSumRows) void k_sum_rows(const float *__restrict__ part, int64_t rows,
                                                                         int width, float *__restrict__ out) {
  __shared__ double s[kSumRows][kSumCols];
  const int col = threadIdx.x % kSumCols, w = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + col;
  double a = 0.0;
  if (c < width) {
    int64_t r = w;
    for (; r + 7 * kSumRows < rows; r += 8 * kSumRows) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = part[(r + u * kSumRows) * width + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) a += double(v[u]);
    }
    for (; r < rows; r += kSumRows) a += double(part[r * width + c]);
  }
  s[w][col] = a;
  __syncthreads();
  for (int d = kSumRows / 2; d > 0; d >>= 1) {
    if (w < d) s[w][col] += s[w + d][col];
    __syncthreads();
  }
  if (w == 0 && c < width) out[c] = float(s[0][col]);
}

inline void sum_rows(const float *part, int64_t rows, int width, float *out, hipStream_t stream) {
  launch(&k_sum_rows, dim3(unsigned((width + kSumCols - 1) / kSumCols)), dim3(kSumCols * kSumRows), 0, stream, part,
         rows, width, out);
}

}  // namespace sgl
