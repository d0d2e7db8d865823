// What the kernels over all candidates share: the problem, 32 x 32 matrix
// products over the three types, row tiles in LDS.
//
// One engine serves the forward and the table's gradient. A wave keeps 32
// outer rows x (as the columns of its products) and walks over inner rows y
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

#include <utility>

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
template <typename T, typename V>
__device__ __forceinline__ FragOf<T> frag_of16(const V &p, int s, float by = 1.f) {
  FragOf<T> f;
  constexpr int E = Mma32<T>::E;
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = T(p[s * E + e] * by);
  return f;
}

// Sum of a fragment's values as a product takes them: bf16 by the two-element
// dot product with ones (within 3 x 2^-24 of each of its four sums, measured), fp16 by
// additions that take 16 bits (its dot product is off by 2^-21).
__device__ __forceinline__ float frag_sum(FragOf<bf16_t> f) {
  typedef __bf16 Two __attribute__((ext_vector_type(2)));
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    a = __builtin_amdgcn_fdot2_f32_bf16(Two{f[e], f[e + 1]}, Two{1.f, 1.f}, a, false);
    b = __builtin_amdgcn_fdot2_f32_bf16(Two{f[e + 2], f[e + 3]}, Two{1.f, 1.f}, b, false);
  }
  return a + b;
}
__device__ __forceinline__ float frag_sum(FragOf<fp16_t> f) {
  float a[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = float(f[e]) + float(f[e + 4]);
  return (a[0] + a[1]) + (a[2] + a[3]);
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

// A tile's YT rows on their way from memory to LDS: 16 bytes a load, eight
// lanes a row and 128 bytes of it, BLOCK / 8 rows a step. A row's partial last load is
// taken from D - E (it writes what its neighbour writes, with the same values;
// columns past D are cleared once), so that loads and stores are all whole.
// Rows past the tensor's end are read as the last one and written as zeros, as
// are those marked -inf: they may hold anything.
constexpr int64_t kMaxStride = 1 << 22;   // of a row: a tile's offsets stay in 32 bits
template <typename T, int DP, int YT, int BLOCK = kBlock>
struct Stage {
  using Tl = Tile32<T, DP>;
  static constexpr int E = Tl::E, CB = Tl::UPR / 8, ROWS = BLOCK / 8, RB = YT / ROWS, SZ = int(sizeof(T));
  static_assert(YT % ROWS == 0 && Tl::UPR % 8 == 0, "eight lanes a row");
  FragOf<T> f[RB][CB];
  float mark[RB];      // a value that may still be on its way
  uint32_t from[CB];   // bytes from the tile's first row
  int to[CB];          // elements of the tile
  int stride;          // bytes
  __device__ __forceinline__ Stage(int64_t row_stride, int D) : stride(int(row_stride) * SZ) {
    const int r = threadIdx.x >> 3;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const int col = min((c * 8 + int(threadIdx.x & 7)) * E, D - E);
      from[c] = uint32_t(r * stride + col * SZ);
      to[c] = r * Tl::LD + col;
    }
  }
  // base: the tile's first row, of `rows` to the end; marks (or NULL): a value of each
  __device__ __forceinline__ void fetch(const T *base, int rows, const float *marks) {
    const char *b = reinterpret_cast<const char *>(base);
    const int r = threadIdx.x >> 3;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      // (rows past the end: back to the last one)
      const int back = rows >= YT ? 0 : max(ROWS * i + r - (rows - 1), 0);
#pragma unroll
      for (int c = 0; c < CB; ++c)
        __builtin_memcpy(&f[i][c], b + (from[c] + uint32_t((ROWS * i - back) * stride)), sizeof(f[i][c]));
      if (marks != nullptr) mark[i] = marks[ROWS * i + r - back];
    }
  }
  __device__ __forceinline__ void put(T *tile, int rows, bool marked) const {
    const int r = threadIdx.x >> 3;
    if (!marked && rows >= YT) {
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int c = 0; c < CB; ++c) __builtin_memcpy(tile + to[c] + ROWS * i * Tl::LD, &f[i][c], sizeof(f[i][c]));
    } else {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const bool out = ROWS * i + r >= rows || (marked && mark[i] == -INFINITY);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
          const FragOf<T> g = out ? zero_frag<T>() : f[i][c];
          __builtin_memcpy(tile + to[c] + ROWS * i * Tl::LD, &g, sizeof(g));
        }
      }
    }
  }
  // zeros, and ones in column `one` (at or past D, where put leaves them; -1: none)
  static __device__ __forceinline__ void clear(T *tile, int one = -1) {
    for (int u = threadIdx.x; u < YT * Tl::UPR; u += BLOCK) {
      FragOf<T> f = zero_frag<T>();
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (u % Tl::UPR * E + e == one) f[e] = T(1.f);
      *reinterpret_cast<FragOf<T> *>(tile + u / Tl::UPR * Tl::LD + u % Tl::UPR * E) = f;
    }
  }
};
// A value that the compiler takes as new: what is formed from it inside a loop
// is not formed before it and kept (masks and addresses of a piece's start and
// end otherwise fill the registers of the loop between).
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+s"(x));
  return x;
}
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
template <typename V>
__device__ __forceinline__ float sum16(const V &p) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = p[i] + p[i + 8];
#pragma unroll
  for (int d = 4; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) a[i] += a[i + d];
  return a[0];
}
template <typename V>
__device__ __forceinline__ float max16(const V &p) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = fmaxf(p[i], p[i + 8]);
#pragma unroll
  for (int d = 4; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) a[i] = fmaxf(a[i], a[i + d]);
  return a[0];
}
// Every block an operand of what stands between: no product of theirs is moved
// across it in either direction.
template <int NB>
__device__ __forceinline__ void settle_blocks(f32x16 (&o)[NB]) {
  static_assert(NB <= 8, "operands of one statement");
  if constexpr (NB == 8)
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]),
                 "+a"(o[6]), "+a"(o[7]));
  else if constexpr (NB == 6)
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]));
  else static_assert(NB == 6, "blocks of rows of 192 and 256 channels");
}
// Accumulator blocks times a factor. With one wave a SIMD (ALONE) they lie in
// the matrix unit's own registers, and the factor is applied in place by hand:
// behind a branch that is seldom taken the compiler otherwise keeps the blocks
// in two places and moves all of them on the path that does nothing (128 moves
// a step of 256 channels). The waits before and behind it are a matrix product's
// before its result is read (19 of the 32 wait states after one of 16 passes) and a
// write's before the next one; the blocks pass through them, so that no product
// stands between a wait and what it is for.
template <bool ALONE, int NB>
__device__ __forceinline__ void scale_blocks(f32x16 (&o)[NB], float by) {
  if constexpr (!ALONE) {
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= by;
  } else {
    settle_blocks(o);
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        float x[4], t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = o[d][r + i];
        asm volatile("v_accvgpr_read_b32 %4, %0\n\tv_accvgpr_read_b32 %5, %1\n\t"
                     "v_accvgpr_read_b32 %6, %2\n\tv_accvgpr_read_b32 %7, %3\n\t"
                     "v_mul_f32 %4, %4, %8\n\tv_mul_f32 %5, %5, %8\n\t"
                     "v_mul_f32 %6, %6, %8\n\tv_mul_f32 %7, %7, %8\n\t"
                     "v_accvgpr_write_b32 %0, %4\n\tv_accvgpr_write_b32 %1, %5\n\t"
                     "v_accvgpr_write_b32 %2, %6\n\tv_accvgpr_write_b32 %3, %7"
                     : "+a"(x[0]), "+a"(x[1]), "+a"(x[2]), "+a"(x[3]), "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]),
                       "=&v"(t[3])
                     : "v"(by));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][r + i] = x[i];
      }
    settle_blocks(o);
  }
}
template <typename V>
__device__ __forceinline__ float abs_max16(const V &p) {   // (three operands an instruction)
  float a = fabsf(p[0]);
#pragma unroll
  for (int i = 1; i < 15; i += 2) a = fmaxf(fmaxf(a, fabsf(p[i])), fabsf(p[i + 1]));
  return fmaxf(a, fabsf(p[15]));
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
// A bias to base 2. Finite ones stay finite.
__device__ __forceinline__ float bias2_of(const Problem &p, float b) {
  const float t = b * p.cb;
  return fabsf(t) == INFINITY && fabsf(b) != INFINITY ? copysignf(FLT_MAX, b) : t;
}
__device__ __forceinline__ float bias2(const Problem &p, int64_t v) { return bias2_of(p, p.bias[v]); }

// Outer tiles x inner tiles in one line, outer first, shared out evenly: a
// workgroup w takes units [b_w, b_(w+1)) of it, b_w = w units / groups, and so
// pieces of one or more outer tiles; the piece of outer tile x of workgroup w is
// number w + x (each step along the line raises one of the two or both).
// Whole rounds of the GPU then cost nothing, whatever the numbers of tiles are
// (600 rows are three tiles of 256 over 256 workgroups).
struct Line {
  int64_t units;
  int inner, groups;
  __host__ __device__ Line(int64_t outer, int64_t in, int most)
      : units(outer * in), inner(int(in)), groups(units < most ? int(units) : most) {}
  __device__ __forceinline__ int64_t begin(int64_t w) const { return w * units / groups; }
  __device__ __forceinline__ int64_t group_of(int64_t unit) const { return ((unit + 1) * groups - 1) / units; }
};

// How the work is cut: waves of a workgroup (32 outer rows each), steps of 32
// inner rows a tile, workgroups of a launch (all resident) and waves a SIMD.
// Two waves a SIMD: one's vector work and LDS reads run beside the other's
// matrix instructions (one wave of 64 rows reads half as much from LDS and took
// longer: forward and gradient 357 + 502 us for 310 + 402, 768 x 570,074 x 172 bf16). 16-bit
// types have them in one workgroup, so that a tile is read once for 256 rows;
// fp32, whose matrix instructions take 16 times as long, in two of 128 rows,
// which fill up ragged numbers of rows better. fp32 rows of more than 128
// channels have one wave a SIMD: 172 channels in half the registers take 419 + 382 us
// for 400 + 380 at 600 x 100,000 and 514 + 465 for 508 + 478 at 4,000 x 20,000, and 256
// channels' tiles of two workgroups do not fit a CU's LDS. A step a tile in fp32:
// more even shares of small problems (200 x 1,000 x 100 16 us for 20 with two, 600 x
// 20,000 71 for 75, 4,000 x 100,000 1,473 for 1,454).
template <typename T, int DB>
struct Plan {
  static constexpr bool WIDE = sizeof(T) == 4 && DB >= 6;
  static constexpr int WAVES = sizeof(T) == 4 ? 4 : 8, SUB = sizeof(T) == 4 ? 1 : 2;
  static constexpr int PER_SIMD = WIDE ? 1 : 2, GROUPS_PER_TWO = sizeof(T) == 4 && !WIDE ? 1 : 2;   // CUs of two
  static constexpr int GROUPS = 512 / GROUPS_PER_TWO;
};
// Steps of a product along the channels that are left out by a branch where a
// row ends before them (DB counts rows in 64 channels). fp32 alone: 100 channels
// of 128 270 -> 250 us; in 16 bits the branch costs what the step does (pick_dim's
// constants).
template <typename T>
constexpr int kTrim = sizeof(T) == 4 ? 64 / Mma32<T>::KS - 1 : 0;
// f(a value of the element type, the row's blocks of 32 as a constant, and of
// its last 64 channels the steps of 16 past its end that are left out: up to 2, in 16
// bits; 768 x 570,074 in bf16, forward and gradient: 160 channels of 192 307 + 381 us,
// 281 + 349 without two, 172 317 + 389 and 308 + 379 without one).
template <typename F>
auto pick_dim(int32_t dtype, int D, F &&f) {
  auto cuts = [&](auto t, auto db) {
    const int past = sizeof(t) == 4 ? 0 : (32 * db.value - D) / 16;
    if constexpr (sizeof(t) == 2) {
      if (past == 1) return f(t, db, std::integral_constant<int, 1>{});
      if (past >= 2) return f(t, db, std::integral_constant<int, 2>{});
    }
    return f(t, db, std::integral_constant<int, 0>{});
  };
  auto dims = [&](auto t) {
    switch ((D + 63) / 64) {
      case 1: return cuts(t, std::integral_constant<int, 2>{});
      case 2: return cuts(t, std::integral_constant<int, 4>{});
      case 3: return cuts(t, std::integral_constant<int, 6>{});
      default: return cuts(t, std::integral_constant<int, 8>{});
    }
  };
  if (dtype == SGL_FP32) return dims(float{});
  if (dtype == SGL_BF16) return dims(bf16_t{});
  return dims(fp16_t{});
}

// ------------------------------------------------------------------ launches
// Rows in the order that they are worked on: those with a target first.
// order, live NULL: all, as they are.
struct Order {
  const int32_t *order;   // [N]
  const int32_t *live;    // [1]: how many have one
  __device__ __forceinline__ int64_t row(int64_t at) const { return order != nullptr ? order[at] : at; }
  __device__ __forceinline__ int64_t count(int64_t N) const { return live != nullptr ? int64_t(*live) : N; }
};
// What a forward leaves for each piece (Line) and wave along the table: its
// own maximum as used, its sum and, with a direction, sum_v p_v w_v at that maximum
// and the sum of the p_v as rounded there (16-bit types; fp32: the sum itself): in
// column `ones` of o, where the tiles hold ones, or in r (no column is free: -1).
struct Partials {
  float *m, *l, *r, *o;   // [pieces][wy][rows], the same twice, [pieces][wy][rows][dp]
  int64_t ytiles;
  int rows, wy, dp, groups, ones;
};
Partials forward_shape(int32_t dtype, const Problem &p);   // (without its arrays)
void forward_partials(int32_t dtype, const Problem &p, const Order &order, const Partials &out, hipStream_t stream);

// The rows as the table's gradient takes them: tiles that are copied to LDS as
// they lie. A tile: its rows, `ld` elements apart, zeros past the last channel,
// then for each row minus the maximum, g T / l, g T and the candidate wanted of
// labels (-1: none); rows without a gradient and past the last one: zeros, -inf, 0, 0, -1.
struct Image {
  int rows, ld;    // of a tile, elements of a row
  int64_t bytes;   // of a tile
};
Image grad_image(int32_t dtype, int D);

struct RowCoef {
  const char *image;
  const int32_t *live;     // [1] or NULL: rows that count (the first ones)
  const int32_t *index;    // NULL: labels; else [tiles][vblocks + 1]: a tile's entries by candidate block
  const int2 *entries;     // [N K], a tile's first at tile * rows * K: candidate of the block * 64 + row of the
                           // tile, weight
  int64_t vblocks;
  int K;
};
void route_targets(int32_t dtype, const Problem &p, int K, const int32_t *ids, const float *weight, int32_t *index,
                   int2 *entries, hipStream_t stream);
constexpr int kGradBlock = 32;   // candidates of a wave
// fp32 elements of `part`: whatever the table's size, two pieces a workgroup.
int64_t table_grad_part(int32_t dtype, const Problem &p);
void table_grad(int32_t dtype, const Problem &p, const RowCoef &r, void *dtable, float *dbias, float *part,
                hipStream_t stream);

}  // namespace cand
}  // namespace sgl
