// What the cross attention's kernels share: the problem, MFMA fragments over
// the three types, row tiles in LDS, distances to bias columns.
#pragma once

#include "history.h"

namespace sgl {
namespace attn {

constexpr int kBlock = 256, kWaves = kBlock / kWave;
constexpr int kMaxDim = 128, kMaxCols = 64;
constexpr int kKeys = 64;   // keys of a tile: one a lane where a wave looks at a tile's keys
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ MFMA over the types
// A fragment holds E consecutive k of a lane's row: lane l's row is l % 16, its
// k values (l / 16) * E + e of a step of KS = 4 E.
template <typename T>
struct Mma;
template <>
struct Mma<float> {
  static constexpr int E = 4, KS = 16;
  typedef f32x4 Frag;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};
template <>
struct Mma<sgl::bf16_t> {
  static constexpr int E = 8, KS = 32;
  typedef sgl::bf16_t Frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<sgl::fp16_t> {
  static constexpr int E = 8, KS = 32;
  typedef sgl::fp16_t Frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

template <typename T>
using FragOf = typename Mma<T>::Frag;

// The accumulator blocks (16 reduction indexes each, lane group g holding 4g +
// v of a block) that make the fragment of step s: one block (fp32) or two.
// Blocks past the NB that are given are 0.
template <typename T, int NB>
__device__ __forceinline__ FragOf<T> frag_of(const float (&x)[NB][4], int s) {
  FragOf<T> f;
  constexpr int B = Mma<T>::KS / 16;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) f[4 * b + v] = s * B + b < NB ? T(x[s * B + b][v]) : T(0.f);
  return f;
}

// ------------------------------------------------------------------ rows in memory
// Elements [d, d + E) of a row of dh, 0 past it, from one 16-byte load at any
// alignment: the last, partial vector is loaded from dh - E and moved down
// (`fix`, after the load has landed, so that a tile's loads are issued
// together). Rows shorter than a vector are read by their elements.
template <typename T>
__device__ __forceinline__ FragOf<T> zero_frag() {
  FragOf<T> f;
#pragma unroll
  for (int e = 0; e < Mma<T>::E; ++e) f[e] = T(0.f);
  return f;
}
template <typename T>
__device__ __forceinline__ FragOf<T> load_raw(const T *row, bool ok, int d, int dh) {
  constexpr int E = Mma<T>::E;
  FragOf<T> f = zero_frag<T>();
  if (ok && d < dh) {
    if (dh >= E) {
      __builtin_memcpy(&f, row + min(d, dh - E), sizeof(f));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < dh) f[e] = row[e];
    }
  }
  return f;
}
template <typename T>
__device__ __forceinline__ FragOf<T> fix(FragOf<T> f, int d, int dh) {
  constexpr int E = Mma<T>::E;
  if (dh % E == 0 || dh < E) return f;   // uniform
  const int by = (d + E - dh) * 8 * int(sizeof(T));   // bits past the row's end
  if (by <= 0 || d >= dh) return f;
  typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
  u64x2 u = __builtin_bit_cast(u64x2, f);
  u[0] = by >= 64 ? u[1] >> (by - 64) : (u[0] >> by) | (u[1] << (64 - by));
  u[1] = by >= 64 ? 0 : u[1] >> by;
  return __builtin_bit_cast(FragOf<T>, u);
}
template <typename T>
__device__ __forceinline__ FragOf<T> load_row(const T *row, bool ok, int d, int dh) {
  return fix<T>(load_raw<T>(row, ok, d, dh), d, dh);
}

// A column block (4 consecutive d of 16 db + 4 g) of a lane into its row.
template <typename T>
__device__ __forceinline__ void store4(T *row, int d, int dh, f32x4 x) {
  if (d + 4 <= dh) {
    T t[4] = {T(x[0]), T(x[1]), T(x[2]), T(x[3])};
    store_n(row + d, t);
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (d + v < dh) row[d + v] = T(x[v]);
  }
}

// ------------------------------------------------------------------ rows in LDS
// Row-major tiles of DP columns with 16 bytes of padding. `frag`: a fragment
// along the row. `frag_t`: a fragment down the columns (column = lane % 16, the
// reduction index the row, in the accumulators' order), by the transposing LDS
// read for 16-bit types: no transposed copy of a tile is kept.
template <typename T, int DP>
struct Tile {
  static constexpr int E = Mma<T>::E, LD = DP + E, UPR = DP / E;
  static __device__ __forceinline__ FragOf<T> frag(const T *s, int row0, int k0) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const FragOf<T> *>(s + (row0 + (lane & 15)) * LD + k0 + (lane >> 4) * E);
  }
  // ROWS: rows that exist (a step past them is 0)
  template <int ROWS>
  static __device__ __forceinline__ FragOf<T> frag_t(const T *s, int col0, int row0) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    FragOf<T> f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = s[(row0 + 4 * g + e) * LD + col0 + i];
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 *Lds;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s16x4 t = {0, 0, 0, 0};
        if (ROWS >= 32 || b == 0) {
          const T *p = s + (row0 + 16 * b + 4 * g + (i >> 2)) * LD + col0 + (i & 3) * 4;
          t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(const_cast<T *>(p)));
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) f[4 * b + v] = __builtin_bit_cast(T, short(t[v]));
      }
    }
    return f;
  }
};

// ------------------------------------------------------------------ the problem
struct Args {
  sgl_attention p;
  int G, cols;       // query heads a key head; columns of the bias table
  int64_t rows;      // lq * G
};

template <typename T>
struct Seq {   // one (sequence, key head)
  const T *q, *k, *v;
  int64_t qlen, klen;
  const uint8_t *mask;
  const int64_t *qpos, *kpos;
};
template <typename T>
__device__ __forceinline__ Seq<T> seq_of(const sgl_attention &p, int64_t n, int hk, int G) {
  Seq<T> s;
  s.q = static_cast<const T *>(p.q) + n * p.q_n + int64_t(hk) * G * p.q_h;
  s.k = static_cast<const T *>(p.k) + n * p.k_n + hk * p.k_h;
  s.v = static_cast<const T *>(p.v) + n * p.v_n + hk * p.v_h;
  s.qlen = p.q_lens != nullptr ? min(max(int64_t(p.q_lens[n]), int64_t(0)), p.lq) : p.lq;
  s.klen = p.k_lens != nullptr ? min(max(int64_t(p.k_lens[n]), int64_t(0)), p.lk) : p.lk;
  s.mask = p.key_mask != nullptr ? p.key_mask + n * p.mask_n : nullptr;
  s.qpos = p.q_pos != nullptr ? p.q_pos + n * p.qpos_n : nullptr;
  s.kpos = p.k_pos != nullptr ? p.k_pos + n * p.kpos_n : nullptr;
  return s;
}
template <typename T>
__device__ __forceinline__ bool key_live(const Seq<T> &s, const sgl_attention &p, int64_t j) {
  return j < s.klen && (s.mask == nullptr || s.mask[j * p.mask_t] != 0);
}

// Where query row (i, head qh of the key head's G) lies in o, do and dq.
__device__ __forceinline__ int64_t out_row(const Args &a, int64_t n, int hk, int64_t i, int qh) {
  return ((n * a.p.lq + i) * a.p.heads_q + int64_t(hk) * a.G + qh) * a.p.head_dim;
}

// Row blocks of 16 (one row a lane of 16). SHARE (G even): the blocks 0 and 1
// of a pair are two heads of the same 16 queries, so that a distance is
// turned into its column once for both; t counts (query, head pair). Else t
// counts the rows i G + h and the blocks follow each other.
struct RowAt {
  int64_t i;
  int h;
};
template <bool SHARE>
__device__ __forceinline__ RowAt row_at(int64_t t, int block, int G) {
  RowAt r;
  if constexpr (SHARE) {
    const int half = G >> 1;
    r.i = half == 1 ? t : t / half;
    r.h = int(t - r.i * half) * 2 + block;
  } else {
    r.i = G == 1 ? t : t / G;
    r.h = int(t - r.i * G);
  }
  return r;
}

// ------------------------------------------------------------------ the bias
// Distances are taken from a base position of the workgroup's, in 32 bits
// where every position of a tile lies within 2^30 of it (`Near`, uniform) and
// in 64 else.
__device__ __forceinline__ bool is_near(int64_t rel) { return rel >= -(1ll << 30) && rel < (1ll << 30); }

struct Buckets {
  int last, m, add;   // last bucket, resolution, the second half's offset (0: one-sided)
};
__device__ __forceinline__ Buckets buckets_of(const sgl_attention &p) {
  return Buckets{p.buckets - 1, p.resolution, p.two_sided ? p.buckets : 0};
}
__device__ __forceinline__ int bucket_of(uint32_t n, const Buckets &k) {
  const int sh = (31 - k.m) - __builtin_clz(n | (1u << k.m));
  return min(int(n >> sh) + (sh << k.m), k.last);
}
__device__ __forceinline__ int column(int d, const Buckets &k) {   // |d| < 2^31
  if (k.add == 0) return bucket_of(uint32_t(max(d, 0)), k);        // uniform
  return bucket_of(uint32_t(max(d, -d)), k) + ((d >> 31) & k.add);
}
__device__ __forceinline__ int column64(int64_t d, const Buckets &k) {
  const bool neg = d < 0;
  const uint64_t n64 = neg ? (k.add != 0 ? uint64_t(0) - uint64_t(d) : 0) : uint64_t(d);
  const uint32_t n = n64 > 0xFFFFFFFFull ? 0xFFFFFFFFu : uint32_t(n64);
  return bucket_of(n, k) + (neg ? k.add : 0);
}

// A tile's positions in LDS, by the lanes that see one key (or row) each.
template <int N>
struct PosTile {
  int rel[N];
  int64_t pos[N];
};
// The columns of 4 consecutive keys (or rows) of a tile against one position;
// `sign` -1 where the tile holds the query positions.
template <int N>
__device__ __forceinline__ void columns4(int (&col)[4], const PosTile<N> &t, int at, int rel, int64_t pos, bool near_,
                                         int sign, const Buckets &k) {
  if (near_) {
    int r[4];
    __builtin_memcpy(r, t.rel + at, sizeof(r));
#pragma unroll
    for (int v = 0; v < 4; ++v) col[v] = column(sign > 0 ? rel - r[v] : r[v] - rel, k);
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v) col[v] = column64(sign > 0 ? pos - t.pos[at + v] : t.pos[at + v] - pos, k);
  }
}

// ------------------------------------------------------------------ small things
__host__ __device__ constexpr size_t align_bytes(size_t n) { return (n + 15) & ~size_t(15); }   // a wave's LDS area
// Sum or maximum over the four lane groups that hold one column.
__device__ __forceinline__ float groups_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ float groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
// LDS of one wave: its accesses are in order; nothing moves across this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// The bias table of a key head's G heads, times log2 e.
__device__ __forceinline__ void stage_bias(float *table, const Args &a, int hk, int tid, int threads) {
  for (int c = tid; c < a.G * a.cols; c += threads) table[c] = a.p.bias[int64_t(hk) * a.G * a.cols + c] * kLog2e;
}

// A power of two near 1 / most (1 for 0 and what is not finite).
__device__ __forceinline__ float unit_scale(float most) {
  return most > 0.f && most < INFINITY ? ldexpf(1.f, -max(ilogbf(most), -126)) : 1.f;
}

// fp16 gradients: a power of two that brings the largest |do| near one, so
// that ds keeps fp16's digits whatever the loss is scaled by.
template <typename T>
__device__ __forceinline__ float grad_scale(float most) {
  return std::is_same_v<T, fp16_t> ? unit_scale(most) : 1.f;
}
// fp16: p goes into a product as 2^10 p, away from the subnormals.
template <typename T>
constexpr float kProbUp = std::is_same_v<T, fp16_t> ? 1024.f : 1.f;

// The bias gradient's cells in LDS: [column][16] sums of ds for a set of row
// blocks whose row c has one head, in fixed point (34 fractional bits in an
// int64, relative to a power of two near the largest |do|): integer adds give
// the same sum in any order, and the LDS adds them at 7 to 8 clocks an
// instruction, four lanes a cell included, where float adds take 194 (3 a
// lane; a read, an add and a write 11, in cells of a lane's own). A value
// holds to 2^29 times that power; `seen`, the sum of magnitudes, tells beyond
// it (and of NaN and infinities), and the gradient is NaN then.
constexpr int kCellBits = 34;
constexpr float kCellMax = 536870912.f;   // 2^29
typedef unsigned long long Cell;
__device__ __forceinline__ void clear_cells(Cell *cells, int n, int tid, int threads) {
  for (int i = tid; i < n; i += threads) cells[i] = 0;
}
template <int N>
__device__ __forceinline__ void add_cells(Cell *cells, const int (&col)[N][4], const float (&x)[N][4], float up,
                                          float &seen) {
  const int c = threadIdx.x & 15;
  const float f = up * 4.f;   // 2^34 = 2^2 2^32
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float t = x[k][v] * f, hi = floorf(t);
      seen += fabsf(t);
      const Cell val = (Cell(uint32_t(int(hi))) << 32) | uint32_t((t - hi) * 4294967296.f);
      __hip_atomic_fetch_add(cells + col[k][v] * 16 + c, val, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
}
__device__ __forceinline__ bool cells_hold(float seen) { return seen < 4.f * kCellMax; }
// ------------------------------------------------------------------ launches
int run_forward(const Args &a, void *o, void *rest, float *lse, void *workspace, hipStream_t s);
size_t forward_bytes(const Args &a);
int run_backward(const Args &a, const void *o, const void *rest, const float *lse, const void *go, void *dq, void *dk,
                 void *dv, float *dbias, void *workspace, hipStream_t s);
size_t backward_bytes(const Args &a);
// One wave a (sequence, key head): rows and keys in a few blocks.
constexpr int kSmallRows = 32, kSmallKeys = 64;
inline bool is_small(const Args &a) { return a.rows <= kSmallRows && a.p.lk <= kSmallKeys; }
int run_small_backward(const Args &a, const void *go, void *dq, void *dk, void *dv, float *dbias, void *workspace,
                       hipStream_t s);
size_t small_backward_bytes(const Args &a);

template <typename F>
int by_instance(const sgl_attention &p, F f) {
  auto dims = [&](auto t) {
    if (p.head_dim <= 32) return f(t, std::integral_constant<int, 32>{});
    if (p.head_dim <= 64) return f(t, std::integral_constant<int, 64>{});
    return f(t, std::integral_constant<int, 128>{});
  };
  if (p.dtype == SGL_FP32) return dims(float{});
  if (p.dtype == SGL_BF16) return dims(bf16_t{});
  return dims(fp16_t{});
}

}  // namespace attn
}  // namespace sgl
