// Attention of query rows over another sequence's states with a bias learned
// by time distance, forward and backward.
//
// For sequence n and query head h (G = Hq / Hkv query heads share a key head):
//   s_ij = scale <q_i, k_j> + bias[h][bucket(q_pos_i - k_pos_j)]
//   p_ij = exp(s_ij) / sum over the live keys, o_i = sum_j p_ij v_j
// A key is live if it lies inside the sequence's length and its mask is set;
// rows without a live key, and rows past the query length, are 0. Backward,
// with D_i = <do_i, o_i>:
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (<do_i, v_j> - D_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
//   dbias[h][b] = sum of ds_ij over the pairs in bucket b.
//
// bucket(d): n = |d| (one-sided: max(d, 0)), at most 2^32 - 1. With 2^m
// buckets an octave, n < 2^m is its own bucket and otherwise, e = floor(log2 n),
// (e - m) 2^m + (n >> (e - m)); the last bucket takes what lies beyond it, and
// negative distances of a two-sided table its second half. Integers only, so
// a distance next to a border falls on its own side.
//
// The rows of a key head's G query heads are one list of rows r = i G + g, so
// that they share each key tile and their sums into dk and dv are one loop
// over r (no atomics: every result is the same each time). Products run on
// MFMA, fp32 accumulation (fp32 inputs: v_mfma_f32_16x16x4_f32). The score
// blocks come out of the MFMA with the reduction index of the product that
// follows in a lane's own registers (key x row blocks for o and dq, row x
// key blocks for dk and dv), so p and ds go from one product to the next
// without leaving the registers; the other operand is read from a transposed
// tile whose columns are permuted to that order.
#include <climits>

#include "history.h"

namespace {

using sgl::f32x4;
using sgl::kWave;

constexpr int kBlock = 256, kWaves = kBlock / kWave;
constexpr int kMaxDim = 128, kMaxCols = 64;
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

// The accumulator blocks (16 reduction indexes each, lane group g holding 4g +
// v of a block) that make the fragment of step s: one block (fp32) or two.
template <typename T, int NB>
__device__ __forceinline__ typename Mma<T>::Frag frag_of(const float (&x)[NB][4], int s) {
  typename Mma<T>::Frag f;
  constexpr int B = Mma<T>::KS / 16;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) f[4 * b + v] = T(x[s * B + b][v]);
  return f;
}
// Place of reduction index i in a transposed tile's rows, so that a lane
// group's indexes of a step are consecutive.
template <typename T>
__device__ __forceinline__ int place(int i) {
  constexpr int KS = Mma<T>::KS;
  const int r = i % KS;
  return i - r + (r % 16) / 4 * Mma<T>::E + r / 16 * 4 + r % 4;
}

template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag zero_frag() {
  typename Mma<T>::Frag f;
#pragma unroll
  for (int e = 0; e < Mma<T>::E; ++e) f[e] = T(0.f);
  return f;
}

// Elements [d, d + E) of a row of dh (0 past it; a NULL row is 0).
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag load_row(const T *row, int d, int dh) {
  constexpr int E = Mma<T>::E;
  typename Mma<T>::Frag f = zero_frag<T>();
  if (row != nullptr && d < dh) {
    if (d + E <= dh) {
      __builtin_memcpy(&f, row + d, sizeof(f));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (d + e < dh) f[e] = row[d + e];
    }
  }
  return f;
}

template <typename T, int DP>
struct Tile {
  static constexpr int E = Mma<T>::E, LD = DP + E, UPR = DP / E;   // row-major rows: 16 bytes of padding
  static constexpr int ldt(int rows) { return rows + E; }
  // fragment of rows [row0, row0 + 16) at k0
  static __device__ __forceinline__ typename Mma<T>::Frag frag(const T *s, int ld, int row0, int k0) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const typename Mma<T>::Frag *>(s + (row0 + (lane & 15)) * ld + k0 + (lane >> 4) * E);
  }
  // NR rows into LDS, row-major (rm) and / or transposed (tr); row_of(r): the
  // row's address or NULL.
  template <int NR, bool RM, bool TR, typename F>
  static __device__ __forceinline__ void stage(T *rm, T *tr, int dh, F row_of) {
    constexpr int UNITS = NR / 2 * UPR;
    for (int u = threadIdx.x; u < UNITS; u += kBlock) {
      const int r = 2 * (u / UPR), d = (u % UPR) * E;
      const auto a = load_row<T>(row_of(r), d, dh), b = load_row<T>(row_of(r + 1), d, dh);
      if constexpr (RM) {
        *reinterpret_cast<typename Mma<T>::Frag *>(rm + r * LD + d) = a;
        *reinterpret_cast<typename Mma<T>::Frag *>(rm + (r + 1) * LD + d) = b;
      }
      if constexpr (TR) {
        typedef T Pair __attribute__((ext_vector_type(2)));
        const int at = place<T>(r);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          Pair p;
          p[0] = a[e];
          p[1] = b[e];
          *reinterpret_cast<Pair *>(tr + (d + e) * ldt(NR) + at) = p;
        }
      }
    }
  }
};

// ------------------------------------------------------------------ the problem
struct Args {
  sgl_attention p;
  int G, cols;       // query heads a key head; columns of the bias table
  int64_t rows;      // lq * G
  int64_t row_tiles, key_tiles;
};

// Column of the bias table for a distance.
__device__ __forceinline__ int bucket_col(int64_t d, int buckets, int m, bool two) {
  const bool neg = d < 0;
  const uint64_t n64 = neg ? (two ? uint64_t(-d) : 0) : uint64_t(d);
  const uint32_t n = n64 > 0xFFFFFFFFull ? 0xFFFFFFFFu : uint32_t(n64);
  const int sh = (31 - m) - __builtin_clz(n | (1u << m));
  const int b = min(int(n >> sh) + (sh << m), buckets - 1);
  return two && neg ? b + buckets : b;
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

// Sum or maximum over the four lane groups that hold one column.
__device__ __forceinline__ float groups_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ float groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}

// The bias table of this key head's G heads, times log2 e, and the keys of a
// tile: positions and liveness.
__device__ __forceinline__ void stage_bias(float *table, const sgl_attention &p, int hk, int G, int cols) {
  for (int c = threadIdx.x; c < G * cols; c += kBlock) table[c] = p.bias[int64_t(hk) * G * cols + c] * kLog2e;
}

// A column block (4 consecutive d of 16 db + 4 g) of a lane into its row.
template <typename T>
__device__ __forceinline__ void store4(T *row, int d, int dh, f32x4 x) {
  if (d + 4 <= dh) {
    T t[4] = {T(x[0]), T(x[1]), T(x[2]), T(x[3])};
    sgl::store_n(row + d, t);
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (d + v < dh) row[d + v] = T(x[v]);
  }
}

// ------------------------------------------------------------------ forward
// A workgroup takes 64 rows (16 a wave, one a lane of 16) of a (sequence, key
// head) and walks its keys 64 at a time with the running maximum and sum.
constexpr int kKeys = 64;

template <typename T, int DP>
struct FwdLds {
  T k[kKeys * Tile<T, DP>::LD];
  T vt[DP * Tile<T, DP>::ldt(kKeys)];
  int64_t pos[kKeys];
  float live[kKeys];   // 0, or -inf at a dead key
};

template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_fwd(Args a, T *__restrict__ o, float *__restrict__ lse) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  extern __shared__ __align__(16) char smem[];
  FwdLds<T, DP> &s = *reinterpret_cast<FwdLds<T, DP> *>(smem);
  float *table = reinterpret_cast<float *>(smem + sizeof(s));
  const sgl_attention &p = a.p;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  int64_t id = blockIdx.x;
  const int64_t rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int hk = int(id % p.heads_kv);
  const int64_t n = id / p.heads_kv;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const int64_t r = rt * 64 + w * 16 + (lane & 15);   // this lane's row
  const int64_t qi = r / a.G;
  const int qh = int(r - qi * a.G);
  const bool row_ok = r < a.rows && qi < q.qlen;
  const bool any = rt * 64 < q.qlen * a.G;   // uniform: a live row in the tile
  const bool biased = p.bias != nullptr;
  if (biased) stage_bias(table, p, hk, a.G, a.cols);
  typename M::Frag qf[DP / M::KS];
  const T *qrow = row_ok ? q.q + qi * p.q_t + qh * p.q_h : nullptr;
#pragma unroll
  for (int st = 0; st < DP / M::KS; ++st) qf[st] = load_row<T>(qrow, st * M::KS + g * M::E, p.head_dim);
  const int64_t qp = biased && row_ok ? q.qpos[qi * p.qpos_t] : 0;
  const float c = p.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  f32x4 acc[DP / 16];
#pragma unroll
  for (int b = 0; b < DP / 16; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int64_t j0 = 0; any && j0 < q.klen; j0 += kKeys) {
    __syncthreads();
    L::template stage<kKeys, true, false>(s.k, nullptr, p.head_dim, [&](int j) {
      return key_live(q, p, j0 + j) ? q.k + (j0 + j) * p.k_t : nullptr;
    });
    L::template stage<kKeys, false, true>(nullptr, s.vt, p.head_dim, [&](int j) {
      return key_live(q, p, j0 + j) ? q.v + (j0 + j) * p.v_t : nullptr;
    });
    if (threadIdx.x < kKeys) {
      const int64_t j = j0 + threadIdx.x;
      s.live[threadIdx.x] = key_live(q, p, j) ? 0.f : -INFINITY;
      s.pos[threadIdx.x] = biased && j < q.klen ? q.kpos[j * p.kpos_t] : 0;
    }
    __syncthreads();
    float x[kKeys / 16][4];
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < kKeys / 16; ++kb) {
      f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < DP / M::KS; ++st) sc = M::mma(L::frag(s.k, L::LD, kb * 16, st * M::KS), qf[st], sc);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int j = kb * 16 + 4 * g + v;
        float t = sc[v] * c;
        if (biased) t += table[qh * a.cols + bucket_col(qp - s.pos[j], p.buckets, p.resolution, p.two_sided)];
        t = s.live[j] < 0.f ? -INFINITY : t;
        x[kb][v] = t;
        mx = fmaxf(mx, t);
      }
    }
    mx = groups_max(mx);
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < kKeys / 16; ++kb)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        x[kb][v] = __builtin_amdgcn_exp2f(x[kb][v] - base);
        sum += x[kb][v];
      }
    l = l * alpha + sum;
    m = mn;
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) acc[b] *= alpha;
#pragma unroll
    for (int st = 0; st < kKeys / M::KS; ++st) {
      const typename M::Frag pf = frag_of<T>(x, st);
#pragma unroll
      for (int b = 0; b < DP / 16; ++b)
        acc[b] = M::mma(L::frag(s.vt, L::ldt(kKeys), b * 16, st * M::KS), pf, acc[b]);
    }
  }
  l = groups_sum(l);
  if (r >= a.rows) return;
  const float inv = row_ok && l > 0.f ? 1.f / l : 0.f;
  T *orow = o + ((n * p.lq + qi) * p.heads_q + int64_t(hk) * a.G + qh) * p.head_dim;
#pragma unroll
  for (int b = 0; b < DP / 16; ++b) store4(orow, b * 16 + 4 * g, p.head_dim, acc[b] * inv);
  // log2 of the sum of exp(s); +inf where no key is live, so that p is 0 there
  if (g == 0) lse[(n * p.heads_kv + hk) * a.rows + r] = row_ok && l > 0.f ? m + __log2f(l) : INFINITY;
}

// ------------------------------------------------------------------ backward: dq, dbias, D
// As the forward: 64 rows a workgroup over the keys. bias gradients: a lane
// adds its ds into cells of its own (one a column of the table), so nothing
// depends on the order of atomics; the lanes' cells are summed once at the
// end into one row of partial sums a workgroup.
template <typename T, int DP>
struct DqLds {
  static constexpr int N = sizeof(T) == 2 ? 64 : 32;   // keys a tile
  T k[N * Tile<T, DP>::LD], v[N * Tile<T, DP>::LD];
  T kt[DP * Tile<T, DP>::ldt(N)];
  int64_t pos[N];
  float live[N];
};

// fp16 gradients: a power of two that brings the largest |do| near one, so
// that ds keeps fp16's digits whatever the loss is scaled by.
template <typename T>
__device__ __forceinline__ float grad_scale(float most) {
  if constexpr (std::is_same_v<T, sgl::fp16_t>) {
    return most > 0.f && most < INFINITY ? ldexpf(1.f, -ilogbf(most)) : 1.f;
  } else {
    return 1.f;
  }
}

template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_dq(Args a, const T *__restrict__ o, const float *__restrict__ lse,
                                                    const T *__restrict__ go, T *__restrict__ dq,
                                                    float2 *__restrict__ rowstat, float *__restrict__ part) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using S = DqLds<T, DP>;
  extern __shared__ __align__(16) char smem[];
  S &s = *reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + sizeof(s));
  float *cells = table + a.G * a.cols;
  const sgl_attention &p = a.p;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  int64_t id = blockIdx.x;
  const int64_t rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int hk = int(id % p.heads_kv);
  const int64_t n = id / p.heads_kv;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const int64_t r = rt * 64 + w * 16 + (lane & 15);
  const int64_t qi = r / a.G;
  const int qh = int(r - qi * a.G);
  const bool row_ok = r < a.rows && qi < q.qlen;
  const bool any = rt * 64 < q.qlen * a.G;
  const bool biased = p.bias != nullptr;
  if (biased) stage_bias(table, p, hk, a.G, a.cols);
  float *mine = cells + w * a.cols * 64;
  if (part != nullptr)
    for (int cidx = 0; cidx < a.cols; ++cidx) mine[cidx * 64 + lane] = 0.f;
  typename M::Frag qf[DP / M::KS], gf[DP / M::KS];
  const T *qrow = row_ok ? q.q + qi * p.q_t + qh * p.q_h : nullptr;
  const int64_t orow = ((n * p.lq + qi) * p.heads_q + int64_t(hk) * a.G + qh) * p.head_dim;
  float delta = 0.f, most = 0.f;
#pragma unroll
  for (int st = 0; st < DP / M::KS; ++st) {
    const int d = st * M::KS + g * M::E;
    qf[st] = load_row<T>(qrow, d, p.head_dim);
    gf[st] = load_row<T>(row_ok ? go + orow : nullptr, d, p.head_dim);
    const typename M::Frag of = load_row<T>(row_ok ? o + orow : nullptr, d, p.head_dim);
#pragma unroll
    for (int e = 0; e < M::E; ++e) {
      delta += float(gf[st][e]) * float(of[e]);
      most = fmaxf(most, fabsf(float(gf[st][e])));
    }
  }
  delta = groups_sum(delta);
  most = groups_max(most);
  const float gs = grad_scale<T>(most);
  const float ls = row_ok ? lse[(n * p.heads_kv + hk) * a.rows + r] : INFINITY;
  if (g == 0 && r < a.rows) rowstat[(n * p.heads_kv + hk) * a.rows + r] = make_float2(delta, most);
  const int64_t qp = biased && row_ok ? q.qpos[qi * p.qpos_t] : 0;
  const float c = p.scale * kLog2e;
  f32x4 acc[DP / 16];
#pragma unroll
  for (int b = 0; b < DP / 16; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int64_t j0 = 0; any && j0 < q.klen; j0 += S::N) {
    __syncthreads();
    L::template stage<S::N, true, true>(s.k, s.kt, p.head_dim, [&](int j) {
      return key_live(q, p, j0 + j) ? q.k + (j0 + j) * p.k_t : nullptr;
    });
    L::template stage<S::N, true, false>(s.v, nullptr, p.head_dim, [&](int j) {
      return key_live(q, p, j0 + j) ? q.v + (j0 + j) * p.v_t : nullptr;
    });
    if (threadIdx.x < S::N) {
      const int64_t j = j0 + threadIdx.x;
      s.live[threadIdx.x] = key_live(q, p, j) ? 0.f : -INFINITY;
      s.pos[threadIdx.x] = biased && j < q.klen ? q.kpos[j * p.kpos_t] : 0;
    }
    __syncthreads();
    float x[S::N / 16][4];
#pragma unroll
    for (int kb = 0; kb < S::N / 16; ++kb) {
      f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < DP / M::KS; ++st) {
        sc = M::mma(L::frag(s.k, L::LD, kb * 16, st * M::KS), qf[st], sc);
        dp = M::mma(L::frag(s.v, L::LD, kb * 16, st * M::KS), gf[st], dp);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int j = kb * 16 + 4 * g + v;
        float t = sc[v] * c;
        int col = 0;
        if (biased) {
          col = bucket_col(qp - s.pos[j], p.buckets, p.resolution, p.two_sided);
          t += table[qh * a.cols + col];
        }
        const float pr = s.live[j] < 0.f ? 0.f : __builtin_amdgcn_exp2f(t - ls);
        const float ds = pr * (dp[v] - delta);
        if (part != nullptr) mine[col * 64 + (lane ^ col)] += ds;
        x[kb][v] = ds * gs;
      }
    }
#pragma unroll
    for (int st = 0; st < S::N / M::KS; ++st) {
      const typename M::Frag df = frag_of<T>(x, st);
#pragma unroll
      for (int b = 0; b < DP / 16; ++b)
        acc[b] = M::mma(L::frag(s.kt, L::ldt(S::N), b * 16, st * M::KS), df, acc[b]);
    }
  }
  if (r < a.rows) {
    const float f = p.scale / gs;
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) store4(dq + orow, b * 16 + 4 * g, p.head_dim, acc[b] * f);
  }
  if (part != nullptr) {
    // wave w's lanes take the columns: the sum of column `lane`'s cells by
    // head (the cell of lane i sits at i ^ column: no bank conflicts), then
    // the waves' sums in order
    __syncthreads();
    float *out = part + ((n * a.row_tiles + rt) * p.heads_kv + hk) * a.G * a.cols;
    const int h0 = int((rt * 64 + w * 16) % a.G);
    for (int h = 0; h < a.G; ++h) {
      float t = 0.f;
      if (lane < a.cols)
        for (int i = 0; i < 16; ++i)
          if ((h0 + i) % a.G == h)
#pragma unroll
            for (int k = 0; k < 4; ++k) t += mine[lane * 64 + ((k * 16 + i) ^ lane)];
      float *sums = reinterpret_cast<float *>(smem);   // (the tiles are done)
      __syncthreads();
      sums[w * 64 + lane] = t;
      __syncthreads();
      if (w == 0 && lane < a.cols)
        out[h * a.cols + lane] = (sums[lane] + sums[64 + lane]) + (sums[128 + lane] + sums[192 + lane]);
    }
  }
}

// ------------------------------------------------------------------ backward: dk, dv
// A workgroup takes 64 keys (16 a wave, one a lane of 16) and walks the rows
// of all G heads, 32 at a time.
constexpr int kRows = 32;

template <typename T, int DP>
struct DkvLds {
  T q[kRows * Tile<T, DP>::LD], go[kRows * Tile<T, DP>::LD];
  T qt[DP * Tile<T, DP>::ldt(kRows)], got[DP * Tile<T, DP>::ldt(kRows)];
  int64_t pos[kRows];
  float lse[kRows], delta[kRows];
  int head[kRows];
  float red[kWaves];
};

template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_dkv(Args a, const float *__restrict__ lse, const T *__restrict__ go,
                                                     const float2 *__restrict__ rowstat, T *__restrict__ dk,
                                                     T *__restrict__ dv) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using S = DkvLds<T, DP>;
  constexpr bool kHalf = std::is_same_v<T, sgl::fp16_t>;
  constexpr float kUp = kHalf ? 10.f : 0.f;   // fp16: p carried as 2^10 p, away from the subnormals
  extern __shared__ __align__(16) char smem[];
  S &s = *reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + sizeof(s));
  const sgl_attention &p = a.p;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  int64_t id = blockIdx.x;
  const int64_t kt = id % a.key_tiles;
  id /= a.key_tiles;
  const int hk = int(id % p.heads_kv);
  const int64_t n = id / p.heads_kv;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const int64_t j = kt * kKeys + w * 16 + (lane & 15);   // this lane's key
  const bool live = key_live(q, p, j);
  const bool biased = p.bias != nullptr;
  if (biased) stage_bias(table, p, hk, a.G, a.cols);
  const int64_t live_rows = kt * kKeys < q.klen ? q.qlen * a.G : 0;
  const int64_t stat0 = (n * p.heads_kv + hk) * a.rows;
  float gs = 1.f;
  if constexpr (kHalf) {
    float most = 0.f;
    for (int64_t r = threadIdx.x; r < live_rows; r += kBlock) most = fmaxf(most, rowstat[stat0 + r].y);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, kWave));
    if (lane == 0) s.red[w] = most;
    __syncthreads();
    gs = grad_scale<T>(fmaxf(fmaxf(s.red[0], s.red[1]), fmaxf(s.red[2], s.red[3])));
  }
  typename M::Frag kf[DP / M::KS], vf[DP / M::KS];
#pragma unroll
  for (int st = 0; st < DP / M::KS; ++st) {
    const int d = st * M::KS + g * M::E;
    kf[st] = load_row<T>(live ? q.k + j * p.k_t : nullptr, d, p.head_dim);
    vf[st] = load_row<T>(live ? q.v + j * p.v_t : nullptr, d, p.head_dim);
  }
  const int64_t kp = biased && live ? q.kpos[j * p.kpos_t] : 0;
  const float c = p.scale * kLog2e;
  const float dsf = kHalf ? gs * 0x1p-10f : 1.f;
  f32x4 ak[DP / 16], av[DP / 16];
#pragma unroll
  for (int b = 0; b < DP / 16; ++b) ak[b] = av[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int64_t r0 = 0; r0 < live_rows; r0 += kRows) {
    __syncthreads();
    L::template stage<kRows, true, true>(s.q, s.qt, p.head_dim, [&](int i) {
      const int64_t r = r0 + i, qi = r / a.G;
      return r < live_rows ? q.q + qi * p.q_t + (r - qi * a.G) * p.q_h : nullptr;
    });
    L::template stage<kRows, true, true>(s.go, s.got, p.head_dim, [&](int i) {
      const int64_t r = r0 + i, qi = r / a.G;
      return r < live_rows ? go + ((n * p.lq + qi) * p.heads_q + int64_t(hk) * a.G + (r - qi * a.G)) * p.head_dim
                           : nullptr;
    });
    if (threadIdx.x < kRows) {
      const int i = threadIdx.x;
      const int64_t r = r0 + i, qi = r / a.G;
      const bool ok = r < live_rows;
      s.lse[i] = ok ? lse[stat0 + r] : INFINITY;
      s.delta[i] = ok ? rowstat[stat0 + r].x : 0.f;
      s.pos[i] = biased && ok ? q.qpos[qi * p.qpos_t] : 0;
      s.head[i] = int(r - qi * a.G);
    }
    __syncthreads();
    float x[kRows / 16][4], y[kRows / 16][4];   // p and ds, rows x this lane's key
#pragma unroll
    for (int rb = 0; rb < kRows / 16; ++rb) {
      f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < DP / M::KS; ++st) {
        sc = M::mma(L::frag(s.q, L::LD, rb * 16, st * M::KS), kf[st], sc);
        dp = M::mma(L::frag(s.go, L::LD, rb * 16, st * M::KS), vf[st], dp);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int i = rb * 16 + 4 * g + v;
        float t = sc[v] * c;
        if (biased) t += table[s.head[i] * a.cols + bucket_col(s.pos[i] - kp, p.buckets, p.resolution, p.two_sided)];
        const float pr = live ? __builtin_amdgcn_exp2f(t - s.lse[i] + kUp) : 0.f;
        x[rb][v] = pr;
        y[rb][v] = pr * ((dp[v] - s.delta[i]) * dsf);
      }
    }
#pragma unroll
    for (int st = 0; st < kRows / M::KS; ++st) {
      const typename M::Frag pf = frag_of<T>(x, st), df = frag_of<T>(y, st);
#pragma unroll
      for (int b = 0; b < DP / 16; ++b) {
        av[b] = M::mma(L::frag(s.got, L::ldt(kRows), b * 16, st * M::KS), pf, av[b]);
        ak[b] = M::mma(L::frag(s.qt, L::ldt(kRows), b * 16, st * M::KS), df, ak[b]);
      }
    }
  }
  if (j >= p.lk) return;
  const int64_t row = ((n * p.lk + j) * p.heads_kv + hk) * p.head_dim;
  const float fk = p.scale / gs, fv = kHalf ? 0x1p-10f : 1.f;
#pragma unroll
  for (int b = 0; b < DP / 16; ++b) {
    store4(dk + row, b * 16 + 4 * g, p.head_dim, ak[b] * fk);
    store4(dv + row, b * 16 + 4 * g, p.head_dim, av[b] * fv);
  }
}

// ------------------------------------------------------------------ host
Args args_of(const sgl_attention *p) {
  Args a;
  a.p = *p;
  a.G = p->heads_q / p->heads_kv;
  a.cols = p->bias != nullptr ? p->buckets * (p->two_sided ? 2 : 1) : 0;
  a.rows = p->lq * a.G;
  a.row_tiles = (a.rows + 63) / 64;
  a.key_tiles = (p->lk + kKeys - 1) / kKeys;
  return a;
}

int check_attn(const sgl_attention *p) {
  SGL_REQUIRE(p != nullptr, "cross_attention: NULL problem");
  SGL_REQUIRE(p->dtype >= 0 && p->dtype <= SGL_FP16, "cross_attention: unknown element type %d", p->dtype);
  SGL_REQUIRE(p->n >= 0 && p->lq >= 0 && p->lk >= 0 && p->n < INT_MAX && p->lq < INT_MAX && p->lk < INT_MAX,
              "cross_attention: bad sizes");
  SGL_REQUIRE(p->heads_q > 0 && p->heads_kv > 0 && p->heads_q % p->heads_kv == 0,
              "cross_attention: %d query heads over %d key heads", p->heads_q, p->heads_kv);
  SGL_REQUIRE(p->head_dim > 0 && p->head_dim <= kMaxDim, "cross_attention: head size %d (1 to %d)", p->head_dim,
              kMaxDim);
  SGL_REQUIRE(p->heads_q / p->heads_kv <= 64, "cross_attention: more than 64 query heads to a key head");
  if (p->bias != nullptr) {
    SGL_REQUIRE(p->buckets > 0 && p->buckets * (p->two_sided ? 2 : 1) <= kMaxCols,
                "cross_attention: a bias table of %d buckets (at most %d columns)", p->buckets, kMaxCols);
    SGL_REQUIRE(p->resolution >= 0 && p->resolution <= 4, "cross_attention: bias resolution %d (0 to 4)",
                p->resolution);
    SGL_REQUIRE(p->n == 0 || ((p->lq == 0 || p->q_pos) && (p->lk == 0 || p->k_pos)),
                "cross_attention: a bias needs positions");
  }
  SGL_REQUIRE(p->n == 0 || ((p->lq == 0 || p->q) && (p->lk == 0 || (p->k && p->v))), "cross_attention: NULL array");
  const Args a = args_of(p);
  SGL_REQUIRE(p->n * p->heads_kv < INT_MAX && p->n * p->heads_kv * std::max(a.row_tiles, a.key_tiles) < INT_MAX,
              "cross_attention: too many rows for one call");
  return SGL_OK;
}

size_t stat_bytes(const Args &a) { return sgl::align_up(sizeof(float2) * size_t(a.p.n * a.p.heads_kv * a.rows)); }

template <typename T, int DP>
int attn_fwd(const Args &a, void *o, float *lse, hipStream_t s) {
  const size_t lds = sizeof(FwdLds<T, DP>) + sizeof(float) * size_t(a.G) * a.cols;
  SGL_CHECK_HIP(sgl::ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_fwd<T, DP>), lds));
  sgl::launch(&k_attn_fwd<T, DP>, dim3(unsigned(a.p.n * a.p.heads_kv * a.row_tiles)), dim3(kBlock), lds, s, a,
              static_cast<T *>(o), lse);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

template <typename T, int DP>
int attn_bwd(const Args &a, const void *o, const float *lse, const void *go, void *dq, void *dk, void *dv,
             float *dbias, float2 *stat, float *part, hipStream_t s) {
  if (a.row_tiles > 0) {
    const size_t lds = sizeof(DqLds<T, DP>) + sizeof(float) * size_t(a.G) * a.cols +
                       (dbias != nullptr ? sizeof(float) * kBlock * size_t(a.cols) : 0);
    SGL_REQUIRE(lds <= 160 * 1024, "cross_attention_backward: %zu bytes of LDS", lds);
    SGL_CHECK_HIP(sgl::ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dq<T, DP>), lds));
    sgl::launch(&k_attn_dq<T, DP>, dim3(unsigned(a.p.n * a.p.heads_kv * a.row_tiles)), dim3(kBlock), lds, s, a,
                static_cast<const T *>(o), lse, static_cast<const T *>(go), static_cast<T *>(dq), stat,
                dbias != nullptr ? part : nullptr);
    SGL_CHECK_LAUNCH();
  }
  if (dbias != nullptr)
    sgl::sum_rows(part, a.p.n * a.row_tiles, a.p.heads_q * a.cols, dbias, s);
  if (a.key_tiles > 0) {
    const size_t lds = sizeof(DkvLds<T, DP>) + sizeof(float) * size_t(a.G) * a.cols;
    SGL_CHECK_HIP(sgl::ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dkv<T, DP>), lds));
    sgl::launch(&k_attn_dkv<T, DP>, dim3(unsigned(a.p.n * a.p.heads_kv * a.key_tiles)), dim3(kBlock), lds, s, a, lse,
                static_cast<const T *>(go), static_cast<const float2 *>(stat), static_cast<T *>(dk),
                static_cast<T *>(dv));
  }
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

template <typename F>
int by_instance(const sgl_attention *p, F f) {
  auto dims = [&](auto t) {
    if (p->head_dim <= 32) return f(t, std::integral_constant<int, 32>{});
    if (p->head_dim <= 64) return f(t, std::integral_constant<int, 64>{});
    return f(t, std::integral_constant<int, 128>{});
  };
  if (p->dtype == SGL_FP32) return dims(float{});
  if (p->dtype == SGL_BF16) return dims(sgl::bf16_t{});
  return dims(sgl::fp16_t{});
}

}  // namespace

extern "C" size_t sgl_cross_attention_workspace_bytes(const sgl_attention *p, int32_t backward) {
  if (check_attn(p) != SGL_OK || p->n == 0 || !backward) return 0;
  const Args a = args_of(p);
  return stat_bytes(a) + sizeof(float) * size_t(p->n * a.row_tiles) * p->heads_q * a.cols;
}

extern "C" int sgl_cross_attention_forward(const sgl_attention *p, void *o, float *lse, void *workspace,
                                           size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_attn(p)) return rc;
  if (p->n == 0 || p->lq == 0) return SGL_OK;
  SGL_REQUIRE(o && lse, "cross_attention: NULL array");
  if (workspace_bytes < sgl_cross_attention_workspace_bytes(p, 0)) {
    sgl::set_error("cross_attention: workspace of %zu bytes, %zu needed", workspace_bytes,
                   sgl_cross_attention_workspace_bytes(p, 0));
    return SGL_ERR_WORKSPACE;
  }
  const Args a = args_of(p);
  return by_instance(p, [&](auto t, auto dp) {
    return attn_fwd<decltype(t), decltype(dp)::value>(a, o, lse, stream);
  });
}

extern "C" int sgl_cross_attention_backward(const sgl_attention *p, const void *o, const float *lse, const void *go,
                                            void *dq, void *dk, void *dv, float *dbias, void *workspace,
                                            size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_attn(p)) return rc;
  SGL_REQUIRE(dbias == nullptr || p->bias != nullptr, "cross_attention_backward: a bias gradient without a bias");
  if (p->n == 0) {
    if (dbias != nullptr) {
      const Args z = args_of(p);
      sgl::sum_rows(nullptr, 0, p->heads_q * z.cols, dbias, stream);
      SGL_CHECK_LAUNCH();
    }
    return SGL_OK;
  }
  SGL_REQUIRE((p->lq == 0 || (o && lse && go && dq)) && (p->lk == 0 || (dk && dv)),
              "cross_attention_backward: NULL array");
  const size_t need = sgl_cross_attention_workspace_bytes(p, 1);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    sgl::set_error("cross_attention_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  const Args a = args_of(p);
  float2 *stat = static_cast<float2 *>(workspace);
  float *part = reinterpret_cast<float *>(static_cast<char *>(workspace) + stat_bytes(a));
  return by_instance(p, [&](auto t, auto dp) {
    return attn_bwd<decltype(t), decltype(dp)::value>(a, o, lse, go, dq, dk, dv, dbias, stat, part, stream);
  });
}
