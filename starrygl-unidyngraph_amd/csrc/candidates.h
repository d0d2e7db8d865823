// What the kernels over all candidates share: the problem, 32 x 32 matrix
// products over the three types, row tiles in LDS.
//
// One engine serves the forward and the table's gradient. A wave keeps 32 or
// 64 outer rows x (as the columns of its products) and walks over inner rows y
// in tiles that the workgroup shares:
//   S^T[y, x] = <y, x>      (reduction over the channels)
//   P^T[y, x] = f(S^T)      (elementwise, in the accumulators)
//   O^T[d, x] += y[d] P^T   (reduction over y)
// An accumulator of S^T holds, in a lane of column x, four consecutive y of
// each eight: in that order it is the second product's operand as it stands,
// and the tile is read down its columns in the same order. The forward takes x
// from the rows and y from the table with the running maximum and sum of a
// softmax; the gradient takes x from the table and y from the rows.
#pragma once

#include "cross_attention.h"

namespace sgl {
namespace cand {

using attn::fix;
using attn::FragOf;
using attn::zero_frag;

constexpr int kBlock = 256, kWaves = kBlock / kWave;
constexpr int kMaxDim = 256, kMaxTargets = 1024;
constexpr int64_t kMaxRows = (1 << 24) - 1;
constexpr float kLog2e = attn::kLog2e;
constexpr float kLn2 = 0.693147180559945309f;

typedef float f32x16 __attribute__((ext_vector_type(16)));

// A fragment holds E consecutive k of a lane's row: lane l's row is l % 32, its
// k values (l / 32) * E + e of a step of KS = 2 E.
template <typename T>
struct Mma32;
template <>
struct Mma32<float> {
  static constexpr int E = 4, KS = 8;
  static __device__ __forceinline__ f32x16 mma(FragOf<float> a, FragOf<float> b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};
template <>
struct Mma32<bf16_t> {
  static constexpr int E = 8, KS = 16;
  static __device__ __forceinline__ f32x16 mma(FragOf<bf16_t> a, FragOf<bf16_t> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma32<fp16_t> {
  static constexpr int E = 8, KS = 16;
  static __device__ __forceinline__ f32x16 mma(FragOf<fp16_t> a, FragOf<fp16_t> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// The place of accumulator r of a lane in its block of 32: 8 (r / 4) + 4 (lane
// / 32) + r % 4.
__device__ __forceinline__ int half_of_wave() { return (threadIdx.x >> 5) & 1; }

// Accumulators [4 B s, 4 B (s + 1)) as the operand of reduction step s.
template <typename T>
__device__ __forceinline__ FragOf<T> frag_of16(const f32x16 &p, int s) {
  FragOf<T> f;
  constexpr int E = Mma32<T>::E;
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = T(p[s * E + e]);
  return f;
}

// Row-major tiles of DP columns, 16 bytes of padding a row.
template <typename T, int DP>
struct Tile32 {
  static constexpr int E = Mma32<T>::E, LD = DP + E, UPR = DP / E;
  static __device__ __forceinline__ FragOf<T> frag(const T *s, int row0, int k0) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const FragOf<T> *>(s + (row0 + (lane & 31)) * LD + k0 + (lane >> 5) * E);
  }
  // Column d = lane % 32 of step s of the rows from row0, in the accumulators'
  // order (16-bit types by the transposing LDS read: 16 lanes take 4 rows of
  // 16 columns).
  static __device__ __forceinline__ FragOf<T> frag_t(const T *s, int col0, int row0, int step) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    FragOf<T> f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = s[(row0 + 8 * step + 4 * h + e) * LD + col0 + (lane & 31)];
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 *Lds;
      const int i = lane & 15, q = (lane >> 4) & 1;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const T *p = s + (row0 + 16 * step + 8 * b + 4 * h + (i >> 2)) * LD + col0 + 16 * q + 4 * (i & 3);
        const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(const_cast<T *>(p)));
#pragma unroll
        for (int v = 0; v < 4; ++v) f[4 * b + v] = __builtin_bit_cast(T, short(t[v]));
      }
    }
    return f;
  }
};

// A tile's YT rows on their way from memory to LDS: 16 bytes a load, a row's
// partial last one taken from D - E (it writes what its neighbour writes, with
// the same values; columns past D are cleared once). Loads and stores are then
// all whole and unconditional. Rows past `rows` are read as the last one and
// written as zeros, as are those with `out` set: they may hold anything.
template <typename T, int DP, int YT>
struct Stage {
  using Tl = Tile32<T, DP>;
  static constexpr int E = Tl::E, UPR = Tl::UPR, NL = YT * UPR / kBlock;
  static_assert(YT * UPR % kBlock == 0, "whole rounds of the workgroup");
  FragOf<T> f[NL];
  bool out[NL];
  static __device__ __forceinline__ int row(int i) { return (int(threadIdx.x) + i * kBlock) / UPR; }
  static __device__ __forceinline__ int col(int i, int D) {
    return min((int(threadIdx.x) + i * kBlock) % UPR * E, D - E);
  }
  // base: the tile's first row
  __device__ __forceinline__ void fetch(const T *base, int64_t stride, int64_t rows, int D) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = int(min(int64_t(row(i)), rows - 1));
      out[i] = row(i) >= rows;
      __builtin_memcpy(&f[i], base + r * stride + col(i, D), sizeof(f[i]));
    }
  }
  __device__ __forceinline__ void put(T *tile, int D) const {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const FragOf<T> g = out[i] ? zero_frag<T>() : f[i];
      __builtin_memcpy(tile + row(i) * Tl::LD + col(i, D), &g, sizeof(g));
    }
  }
  static __device__ __forceinline__ void clear(T *tile) {
    for (int u = threadIdx.x; u < YT * UPR; u += kBlock)
      *reinterpret_cast<FragOf<T> *>(tile + u / UPR * Tl::LD + u % UPR * E) = zero_frag<T>();
  }
};
// A lane's fragments of an outer row (zeros past D and for `out`).
template <typename T, int NK>
__device__ __forceinline__ void load_outer(FragOf<T> (&f)[NK], const T *row, bool out, int D) {
  constexpr int E = Mma32<T>::E, KS = Mma32<T>::KS;
#pragma unroll
  for (int k = 0; k < NK; ++k) __builtin_memcpy(&f[k], row + min(k * KS + half_of_wave() * E, D - E), sizeof(f[k]));
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int d = k * KS + half_of_wave() * E;
    f[k] = out || d >= D ? zero_frag<T>() : fix<T>(f[k], d, D);
  }
}

// Sum, maximum over the two lanes of a column.
__device__ __forceinline__ float pair_sum(float v) {
  auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}
__device__ __forceinline__ float pair_max(float v) {
  auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float sum16(const f32x16 &p) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = p[i] + p[i + 8];
#pragma unroll
  for (int d = 4; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) a[i] += a[i + d];
  return a[0];
}
__device__ __forceinline__ float max16(const f32x16 &p) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = fmaxf(p[i], p[i + 8]);
#pragma unroll
  for (int d = 4; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) a[i] = fmaxf(a[i], a[i + d]);
  return a[0];
}
// Accumulator blocks times a factor, in place in the matrix unit's registers.
// Written out because a rescale that seldom runs sits behind a branch, where
// the compiler otherwise keeps the blocks in two places and moves all of them
// on the path that does nothing (256 moves a block of 32 rows). The waits are a
// matrix product's before its result is read and a write's before the next one.
template <int NB>
__device__ __forceinline__ void scale_blocks(f32x16 (&o)[NB], float by) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = o[d][r], t;
      asm volatile("v_accvgpr_read_b32 %1, %0\n\ts_nop 1\n\tv_mul_f32 %1, %1, %2\n\ts_nop 1\n\tv_accvgpr_write_b32 %0, %1"
                   : "+a"(x), "=&v"(t)
                   : "v"(by));
      o[d][r] = x;
    }
  asm volatile("s_nop 7" ::: "memory");
}
// 2^x by the hardware instruction (1 ulp; results under 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The problem as the kernels take it. Scores are to base 2: c <h, w> + cb bias.
struct Problem {
  const void *h, *table;
  int64_t hs, ts;        // row strides, elements
  const float *bias;     // or NULL
  int64_t N, V;
  int D;
  float c, cb, scale, temperature;
};
// A candidate's bias to base 2. Finite ones stay finite.
__device__ __forceinline__ float bias2(const Problem &p, int64_t v) {
  const float b = p.bias[v], t = b * p.cb;
  return fabsf(t) == INFINITY && fabsf(b) != INFINITY ? copysignf(FLT_MAX, b) : t;
}

// ------------------------------------------------------------------ launches
// What a forward leaves for each split of the table and row (its own maximum
// as used, its sum) and, with `dir`, sum_v p_v w_v at that maximum.
struct Partials {
  float *m, *l, *o;   // [splits][N], [splits][N], [splits][N][dp]
  int64_t splits;
  int dp;
};
int64_t forward_splits(int32_t dtype, const Problem &p, bool dir);
int padded_dim(int D);
void forward_partials(int32_t dtype, const Problem &p, const Partials &out, bool dir, hipStream_t stream);

struct RowCoef {
  const float *nm, *gl, *gq;   // [N]: minus the maximum, g T / l, g T (dead rows: -inf, 0, 0)
  const int32_t *ids;          // [N][K], -1: none; no candidate twice in a row
  const float *weight;         // [N][K] or NULL: 1
  int K;
};
int64_t table_grad_splits(int32_t dtype, const Problem &p);
// dtable (type of the table, contiguous) and dbias (or NULL); part: with more
// than one split fp32 [splits][V][dp + 1].
void table_grad(int32_t dtype, const Problem &p, const RowCoef &r, void *dtable, float *dbias, float *part,
                int64_t splits, hipStream_t stream);

}  // namespace cand
}  // namespace sgl
