// What the cross attention's kernels share: the problem, MFMA fragments over
// the three types, row tiles in LDS, distances to bias columns.
#pragma once

#include <cfloat>

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

// The same in parts that together hold 22 bits (fp16: two) or 24 (bf16: three)
// of a value, each the rounding of what those before it left.
template <typename T>
constexpr int kParts = std::is_same_v<T, fp16_t> ? 2 : 3;
template <typename T, int NB>
__device__ __forceinline__ void split_frag_of(const float (&x)[NB][4], int s, FragOf<T> (&f)[kParts<T>]) {
  constexpr int B = Mma<T>::KS / 16;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float e = s * B + b < NB ? x[s * B + b][v] : 0.f;
#pragma unroll
      for (int i = 0; i < kParts<T>; ++i) {
        f[i][4 * b + v] = T(e);
        e -= float(T(e));
      }
    }
}

// ------------------------------------------------------------------ rows in memory
// Elements [d, d + E) of a row of dh, 0 past it, from one 16-byte load at any
// alignment: the last, partial vector is loaded from dh - E and moved down
// (`fix`, after the load has landed, so that a tile's loads are issued
// together). dh >= E.
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
  if (ok && d < dh) __builtin_memcpy(&f, row + min(d, dh - E), sizeof(f));
  return f;
}
template <typename T>
__device__ __forceinline__ FragOf<T> fix(FragOf<T> f, int d, int dh) {
  constexpr int E = Mma<T>::E;
  if (dh % E == 0) return f;   // uniform
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

// What rounding x to o left, kept in 16 bits beside o, and x of the two. bf16:
// the low half of x's bits as a signed number (a tie that was rounded down is
// one unit of 2^-24 off), so that o and rest are x; fp16: the difference, 2^11
// as large so that it stays normal where o does (22 bits of x).
template <typename T>
__device__ __forceinline__ T rest_of(float x, T o) {
  if constexpr (std::is_same_v<T, bf16_t>) {
    const int low = int(__float_as_uint(x) - (uint32_t(__builtin_bit_cast(uint16_t, o)) << 16));
    return __builtin_bit_cast(T, int16_t(min(low, 32767)));
  } else {
    return T((x - float(o)) * 2048.f);
  }
}

template <typename T>
__device__ __forceinline__ float whole_of(T o, T rest) {
  if constexpr (std::is_same_v<T, bf16_t>)
    return __uint_as_float((uint32_t(__builtin_bit_cast(uint16_t, o)) << 16) + int(__builtin_bit_cast(int16_t, rest)));
  else
    return float(o) + float(rest) * (1.f / 2048.f);
}

// store4 of what it rounds away.
template <typename T>
__device__ __forceinline__ void store_rest(T *row, int d, int dh, f32x4 x) {
  T t[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) t[v] = rest_of<T>(x[v], T(x[v]));
  if (d + 4 <= dh) {
    store_n(row + d, t);
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (d + v < dh) row[d + v] = t[v];
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

// A value at a uniform address that no kernel here writes: a scalar load.
template <typename V>
__device__ __forceinline__ V scalar_load(const V *p) {
  typedef const __attribute__((address_space(4))) V *Const;
  return *(Const)(p);
}

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
  s.qlen = p.q_lens != nullptr ? min(max(int64_t(scalar_load(p.q_lens + n)), int64_t(0)), p.lq) : p.lq;
  s.klen = p.k_lens != nullptr ? min(max(int64_t(scalar_load(p.k_lens + n)), int64_t(0)), p.lk) : p.lk;
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
// Rows and queries are counted in 32 bits (divisions are long in 64).
struct RowAt {
  uint32_t i;
  int h;
};
template <bool SHARE>
__device__ __forceinline__ RowAt row_at(uint32_t t, int block, int G) {
  RowAt r;
  if constexpr (SHARE) {
    const uint32_t half = uint32_t(G) >> 1;
    r.i = half == 1 ? t : t / half;
    r.h = int(t - r.i * half) * 2 + block;
  } else {
    r.i = G == 1 ? t : t / uint32_t(G);
    r.h = int(t - r.i * uint32_t(G));
  }
  return r;
}
// A workgroup's tile of a (sequence, key head).
struct TileAt {
  int64_t n;
  int hk;
  uint32_t tile;
};
__device__ __forceinline__ TileAt tile_at(uint32_t id, uint32_t tiles, int heads) {
  TileAt t;
  const uint32_t item = tiles == 1 ? id : __builtin_amdgcn_readfirstlane(id / tiles);   // (uniform: id is)
  t.tile = id - item * tiles;
  const uint32_t n = heads == 1 ? item : __builtin_amdgcn_readfirstlane(item / uint32_t(heads));
  t.n = n;
  t.hk = int(item - n * uint32_t(heads));
  return t;
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
// The columns of NB blocks of 16 keys (or rows) of a tile from `at` (4 of each
// a lane) against one position; `sign` -1 where the tile holds the query
// positions. One uniform branch for all of them, so that their steps overlap.
template <int NB, int N>
__device__ __forceinline__ void columns(int (&col)[NB][4], const PosTile<N> &t, int at, int rel, int64_t pos,
                                        bool near_, int sign, const Buckets &k) {
  if (near_) {
    int d[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      int r[4];
      __builtin_memcpy(r, t.rel + at + 16 * b, sizeof(r));
#pragma unroll
      for (int v = 0; v < 4; ++v) d[b][v] = sign > 0 ? rel - r[v] : r[v] - rel;
    }
    if (k.add == 0) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int v = 0; v < 4; ++v) col[b][v] = bucket_of(uint32_t(max(d[b][v], 0)), k);
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          col[b][v] = bucket_of(uint32_t(max(d[b][v], -d[b][v])), k) + ((d[b][v] >> 31) & k.add);
    }
  } else {
#pragma unroll 1
    for (int b = 0; b < NB; ++b) {
      int c[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int64_t p = t.pos[at + 16 * b + v];
        c[v] = column64(sign > 0 ? pos - p : p - pos, k);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i)   // (static places)
#pragma unroll
        for (int v = 0; v < 4; ++v) col[i][v] = i == b ? c[v] : col[i][v];
    }
  }
}

// ------------------------------------------------------------------ small things
__host__ __device__ constexpr size_t align_bytes(size_t n) { return (n + 15) & ~size_t(15); }   // a wave's LDS area
// Sum or maximum over the four lane groups that hold one column, by swapping
// rows of 16 lanes and halves of the wave between two copies of the register.
__device__ __forceinline__ float groups_sum(float v) {
  auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
__device__ __forceinline__ float groups_max(float v) {
  auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
  auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
// The largest magnitude of what is put in, over the lane and then the wave. By
// the bits without the sign, which order as the magnitudes do (two 16-bit
// elements an operation) and put NaN last, so that it is not passed over.
template <typename T>
struct Largest {
  uint32_t bits = 0;
  __device__ __forceinline__ void add(FragOf<T> f) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        bits = max(bits, w[i] & 0x7FFFFFFFu);
      else
        bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, bits),
                                                                      __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu)));
    }
  }
  __device__ __forceinline__ float wave() const {
    uint32_t m = sizeof(T) == 4 ? bits : max(bits & 0xFFFFu, bits >> 16);
    // rows of 16 lanes rotated by 8, 4, 2 and 1, then rows and halves of the wave swapped
    m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x128, 0xF, 0xF, true)));
    m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x124, 0xF, 0xF, true)));
    m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x122, 0xF, 0xF, true)));
    m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x121, 0xF, 0xF, true)));
    auto h = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = max(h[0], h[1]);
    auto q = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(q[0], q[1]);
    if constexpr (sizeof(T) == 4) return __uint_as_float(m);
    else return float(__builtin_bit_cast(T, uint16_t(m)));
  }
};
// The wave's index in its workgroup, as a scalar: what depends on it alone is
// then uniform to the compiler too (scalar loads, addresses and branches).
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// LDS of one wave: its accesses are in order; nothing moves across this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// The bias table of a key head's G heads in LDS, times log2 e; an odd stride,
// so that two heads' values of a column lie in different banks. A finite value
// stays finite: rows whose keys all have the type's lowest one are rows of
// equal scores, as in a softmax that is not taken to base 2.
__host__ __device__ __forceinline__ int table_ld(const Args &a) { return a.cols | 1; }
__host__ __device__ __forceinline__ size_t table_bytes(const Args &a) {
  return a.cols == 0 ? 0 : sizeof(float) * size_t(a.G) * size_t(table_ld(a));
}
__device__ __forceinline__ float base2(float b) {
  const float t = b * kLog2e;
  return fabsf(t) == INFINITY && fabsf(b) != INFINITY ? copysignf(FLT_MAX, b) : t;
}
__device__ __forceinline__ void stage_bias(float *table, const Args &a, int hk, int tid, int threads) {
  for (int c = tid; c < a.G * a.cols; c += threads) {
    const int h = c / a.cols;
    table[h * table_ld(a) + c - h * a.cols] = base2(a.p.bias[int64_t(hk) * a.G * a.cols + c]);
  }
}
// x = x c + shift (+ the bias of each column) over blocks
template <int NB>
__device__ __forceinline__ void scale_scores(float (&x)[NB][4], float c, float shift, const float *row,
                                             const int (&col)[NB][4], bool biased) {
  if (biased) {
    float t[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int v = 0; v < 4; ++v) t[b][v] = row[col[b][v]];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int v = 0; v < 4; ++v) x[b][v] = fmaf(x[b][v], c, shift) + t[b][v];
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int v = 0; v < 4; ++v) x[b][v] = fmaf(x[b][v], c, shift);
  }
}

// fp16: ds goes into a product times a power of two that follows its largest
// magnitude so far, whatever do, v and p are of: from a start that any value
// passes, ds beyond 2^15 (the type ends at 2^16) brings the largest to 2^10, and
// what was summed at the old power is rescaled. The normal numbers then reach
// 2^24 below the largest term of a sum.
constexpr float kFirstScale = 0x1p100f, kMostHalf = 32768.f;
__device__ __forceinline__ float half_scale(float most) {   // (1 for what is not finite)
  return most < INFINITY ? ldexpf(1.f, min(10 - ilogbf(most), 100)) : 1.f;
}
// Blocks' y = ds of a lane's column (a row or key that four lane groups share)
// times that power, the accumulators with it.
template <int NB, int DB>
__device__ __forceinline__ void follow_scale(float (&y)[NB][4], float &scale, f32x4 (&acc)[DB]) {
  float most = 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) most = fmaxf(most, fabsf(y[b][v]));
  if (__any(most * scale > kMostHalf)) {   // (uniform over the wave; the first terms, then seldom)
    most = groups_max(most);
    const float now = most * scale > kMostHalf ? half_scale(most) : scale;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] *= now / scale;
    scale = now;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) y[b][v] *= scale;
}
// fp16: p goes into a product as 2^10 p, away from the subnormals.
template <typename T>
constexpr float kProbUp = std::is_same_v<T, fp16_t> ? 1024.f : 1.f;

// The bias gradient's cells in LDS: [column][slots] sums of ds for a set of row
// blocks whose row c has one head, in fixed point: integer adds give
// the same sum in any order, and the LDS adds them at 7 to 8 clocks an
// instruction, four lanes a cell included, where float adds take 194 (3 a
// lane; a read, an add and a write 11, in cells of a lane's own). The unit is
// 2^-62 of a bound on everything that is added: |ds_ij| <= p_ij (|dp_ij| +
// |D_i|), |dp_ij| and |D_i| are at most |do_i|_1 times the largest |v|, and a
// row's p sum to one, so no sum of any of the terms exceeds 2 max|v| sum |do|
// (twice which a cell holds). A term 2^38 times smaller than that still has the
// 24 bits of a float.
constexpr int kCellBits = 32;   // fractional bits of a term times the power of two
typedef unsigned long long Cell;
// Cells a column: lane c of 16 adds into cell c mod slots; 8 where they
// keep the heads apart (row c has head c mod heads), else 16.
__host__ __device__ __forceinline__ int cell_slots(int heads) { return heads <= 8 && 16 % heads == 0 ? 8 : 16; }
__device__ __forceinline__ void clear_cells(Cell *cells, int n, int tid, int threads) {
  for (int i = tid; i < n; i += threads) cells[i] = 0;
}
// The cells' power of two for sums of magnitudes up to `most`: below 2^30 (1
// for 0 and what is not finite).
__device__ __forceinline__ float cell_scale(float most) {
  return most > 0.f && most < INFINITY ? ldexpf(1.f, min(29 - ilogbf(most), 127)) : 1.f;
}
template <int N>
__device__ __forceinline__ void add_cells(Cell *cells, const int (&col)[N][4], const float (&x)[N][4], int slots,
                                          float up) {
  const int c = threadIdx.x & (slots - 1);
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      // the nearest integer and a signed rest, which is exact (from the integer below, a small negative value's
      // rest lies next to one and has lost its digits)
      const float t = x[k][v] * up, hi = rintf(t);
      const int lo = int((t - hi) * 2147483648.f);   // in units of 2^-31 of t, so two of a cell's
      const Cell val = (Cell(uint32_t(int(hi) + (lo >> 31))) << 32) | (uint32_t(lo) << 1);
      __hip_atomic_fetch_add(cells + col[k][v] * slots + c, val, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
}
// What the cells' sum t is worth.
__device__ __forceinline__ float cell_value(long long t, float up) {
  return float(double(t) * (1.0 / double(1ll << kCellBits)) / double(up));
}
// Waves a SIMD that a kernel's registers leave room for (512 of them): asked of
// the compiler, which otherwise spends registers on loads it could not issue
// earlier anyway (two 8-wave workgroups a CU need 4).
template <typename T, int DP>
__host__ __device__ constexpr int simd_waves(int narrow, int wide) {   // heads up to 64 in 16 bits, or wider
  return sizeof(T) == 2 && DP <= 64 ? narrow : wide;
}

// ------------------------------------------------------------------ key tiles of a workgroup
// Keys of a tile that KW waves share, 32 each (fp32 with four waves: 16).
template <typename T>
constexpr int tile_keys(int kw) {
  return sizeof(T) == 2 ? 32 * kw : 64;
}
__device__ __forceinline__ constexpr uint32_t full_mask(int n) { return n >= 32 ? ~0u : (1u << n) - 1; }

// Tiles in LDS: two where both leave room for a second workgroup (one barrier
// a tile), else one.
template <typename S>
__host__ __device__ constexpr int buffers() {
  return sizeof(S) <= 24 * 1024 ? 2 : 1;
}

// The first n of 64 (n any sign)
__device__ __forceinline__ uint64_t first_bits(int64_t n) { return n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1; }

// A tile of TK keys on its way from memory to LDS, by 16-byte units over the
// workgroup. A thread's row offset and column are the same in every tile, so
// its addresses are a uniform pointer and an offset kept. `load` only issues
// loads (of every row inside the length: what it fetched is looked at in
// `store`, a tile later, so that no wave waits for memory in between): there
// the mask's bytes, one key a lane, become bits and dead rows 0, and the first
// wave, which fetched the positions, tells whether all are near.
template <int TK>
struct KeyInfo {
  PosTile<TK> pos;
  int near_;
};
template <typename T, int DP, int TK, int BLOCK>
struct KeyTile {
  using L = Tile<T, DP>;
  static constexpr int W = TK / 64, PER = (TK * L::UPR + BLOCK - 1) / BLOCK, E = Mma<T>::E, RSTEP = BLOCK / L::UPR;
  static_assert(BLOCK % L::UPR == 0 && (PER == 1 || TK % RSTEP == 0), "units of a thread share their column");
  FragOf<T> kr[PER], vr[PER];
  uint64_t live[W];
  int64_t pos[W], koff, voff;
  int byte[W], r0, d;
  __device__ __forceinline__ KeyTile(const Args &a) {
    r0 = threadIdx.x / L::UPR;
    d = (threadIdx.x % L::UPR) * E;
    const int at = min(d, a.p.head_dim - E);
    koff = r0 * a.p.k_t + at;
    voff = r0 * a.p.v_t + at;
  }
  __device__ __forceinline__ uint32_t live_of(int first, int n) const {   // first: a multiple of 16, uniform
    return uint32_t(live[W == 1 ? 0 : first >> 6] >> (first & 63)) & full_mask(n);
  }
  __device__ __forceinline__ void load(const Seq<T> &q, const Args &a, int64_t j0) {
    const int lane = threadIdx.x & 63;
    const sgl_attention &p = a.p;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      live[i] = first_bits(q.klen - j0 - 64 * i);
      const bool in = (live[i] >> lane) & 1;
      byte[i] = 0;
      pos[i] = 0;
      if (q.mask != nullptr && in) byte[i] = q.mask[(j0 + 64 * i + lane) * p.mask_t];
      if (p.bias != nullptr && threadIdx.x < 64 && in) pos[i] = q.kpos[(j0 + 64 * i + lane) * p.kpos_t];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = r0 + i * RSTEP;
      kr[i] = zero_frag<T>();
      vr[i] = zero_frag<T>();
      if (r < TK && d < p.head_dim && j0 + r < q.klen) {
        __builtin_memcpy(&kr[i], q.k + (j0 + i * RSTEP) * p.k_t + koff, 16);
        __builtin_memcpy(&vr[i], q.v + (j0 + i * RSTEP) * p.v_t + voff, 16);
      }
    }
  }
  __device__ __forceinline__ void store(T *k, T *v, KeyInfo<TK> &t, const Seq<T> &q, const Args &a, int64_t base) {
    const int dh = a.p.head_dim, lane = threadIdx.x & 63;
    if (q.mask != nullptr) {   // uniform
#pragma unroll
      for (int i = 0; i < W; ++i) live[i] = __ballot(byte[i] != 0);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = r0 + i * RSTEP;
      if (TK * L::UPR % BLOCK == 0 || r < TK) {
        FragOf<T> kk = fix<T>(kr[i], d, dh), vv = fix<T>(vr[i], d, dh);
        if (q.mask != nullptr && !((live[W == 1 ? 0 : r >> 6] >> (r & 63)) & 1)) kk = vv = zero_frag<T>();
        *reinterpret_cast<FragOf<T> *>(k + r * L::LD + d) = kk;
        *reinterpret_cast<FragOf<T> *>(v + r * L::LD + d) = vv;
      }
    }
    if (a.p.bias != nullptr && threadIdx.x < 64) {
      bool near_ = true;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int64_t at = (live[i] >> lane) & 1 ? pos[i] : base;
        near_ = near_ && is_near(at - base);
        t.pos.pos[64 * i + lane] = at;
        t.pos.rel[64 * i + lane] = int(at - base);
      }
      near_ = __all(near_);
      if (lane == 0) t.near_ = near_;
    }
  }
};

// The KW waves of each row block (wave w: block w / KW) joined into the first
// of them: the maximum, the sum and the products of NB accumulators a block.
// The workgroup's LDS is free for it (every wave calls this).
inline size_t join_bytes(int rw, int kw, int nq, int dp) {
  return sizeof(float2) * 16 * size_t(rw * kw * nq) + sizeof(float) * 16 * size_t(rw * (kw - 1) * nq * dp);
}
// rows of products: wave w (its part above 0) and block b, [value][16]
template <int KW, int NQ, int NB>
__device__ __forceinline__ float *join_slot(float *pr, int w, int b) {
  return pr + ((w / KW * (KW - 1) + w % KW - 1) * NQ + b) * (NB * 16 * 16);
}
template <int KW, int NQ, int NB>
__device__ __forceinline__ void put_join(float *pr, const f32x4 (&acc)[NQ][NB]) {
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15;
  if (w % KW == 0) return;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    float *t = join_slot<KW, NQ, NB>(pr, w, b);
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int v = 0; v < 4; ++v) t[(d * 16 + 4 * g + v) * 16 + cl] = acc[b][d][v];
  }
}
template <int KW, int NQ, int NB>
__device__ __forceinline__ void take_join(float *pr, f32x4 (&acc)[NQ][NB]) {
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15;
  if (w % KW != 0) return;
#pragma unroll
  for (int k = 1; k < KW; ++k)
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      const float *t = join_slot<KW, NQ, NB>(pr, w + k, b);
#pragma unroll
      for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[b][d][v] += t[(d * 16 + 4 * g + v) * 16 + cl];
    }
}
template <int RW, int KW, int NQ, int NB>
__device__ __forceinline__ void join_waves(char *smem, float (&m)[NQ], float (&l)[NQ], f32x4 (&acc)[NQ][NB]) {
  if constexpr (KW > 1) {
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15, w0 = w / KW * KW;
    float2 *ml = reinterpret_cast<float2 *>(smem);
    float *pr = reinterpret_cast<float *>(smem + sizeof(float2) * 16 * RW * KW * NQ);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NQ; ++b)
      if (g == 0) ml[(w * NQ + b) * 16 + cl] = make_float2(m[b], l[b]);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < KW; ++i) top = fmaxf(top, ml[((w0 + i) * NQ + b) * 16 + cl].x);
      const float at = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        const float2 e = ml[((w0 + i) * NQ + b) * 16 + cl];
        sum += e.y * __builtin_amdgcn_exp2f(e.x - at);
      }
      const float f = __builtin_amdgcn_exp2f(m[b] - at);
#pragma unroll
      for (int d = 0; d < NB; ++d) acc[b][d] *= f;
      m[b] = top;
      l[b] = sum;
    }
    put_join<KW, NQ, NB>(pr, acc);
    __syncthreads();
    take_join<KW, NQ, NB>(pr, acc);
  }
}

// ------------------------------------------------------------------ launches
// Two blocks a wave where their registers fit (fp32 heads above 64 would spill).
template <typename T, int DP>
constexpr bool two_blocks() {
  return sizeof(T) == 2 || DP <= 64;
}
// Row tiles of a (sequence, key head), RW x NQ blocks each (SHARE: pairs).
inline int64_t row_tiles(const Args &a, int nq, bool share, int rw) {
  const int64_t count = share ? a.rows / 2 : a.rows, per = share ? 16 * rw : 16 * rw * nq;
  return (count + per - 1) / per;
}
// Whether tiles of 128 rows fill the GPU: two blocks a wave then (each key
// fragment read from LDS, and with an even G each column, serves two), eight
// waves a workgroup; else 16 rows a workgroup, its four waves along the keys.
inline bool many_rows(const Args &a) { return a.p.n * a.p.heads_kv * ((a.rows + 127) / 128) >= 192; }

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
