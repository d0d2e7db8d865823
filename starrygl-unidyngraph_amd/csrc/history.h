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
// order: 16 waves of a workgroup take rows w, w + 16, ... of 64 columns each.
// blockIdx.y selects one of several such matrices.
constexpr int kSumWaves = 16;
static __global__ __launch_bounds__(kSumWaves * 64) void k_sum_rows(const float *__restrict__ part, int64_t rows,
                                                                    int width, int64_t part_y,
                                                                    float *__restrict__ out, int64_t out_y) {
  __shared__ double s[kSumWaves][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  part += int64_t(blockIdx.y) * part_y;
  double a = 0.0;
  if (c < width) {
    int64_t r = w;
    for (; r + 7 * kSumWaves < rows; r += 8 * kSumWaves) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = part[(r + u * kSumWaves) * width + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) a += double(v[u]);
    }
    for (; r < rows; r += kSumWaves) a += double(part[r * width + c]);
  }
  s[w][lane] = a;
  __syncthreads();
  if (w == 0 && c < width) {
    for (int i = 1; i < kSumWaves; ++i) a += s[i][lane];
    out[int64_t(blockIdx.y) * out_y + c] = float(a);
  }
}

inline void sum_rows(const float *part, int64_t rows, int width, float *out, hipStream_t stream, int count = 1,
                     int64_t part_y = 0, int64_t out_y = 0) {
  launch(&k_sum_rows, dim3(unsigned((width + 63) / 64), unsigned(count)), dim3(kSumWaves * 64), 0, stream, part, rows,
         width, part_y, out, out_y);
}

}  // namespace sgl
