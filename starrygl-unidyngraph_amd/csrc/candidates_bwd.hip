// The gradient of the table (and of a bias): dw_v = scale sum_n (gl_n e_nv -
// gq_n q_nv) h_n over the rows, e the forward's exponentials, formed again.
#include "candidates.h"

namespace {

using namespace sgl;
using namespace sgl::cand;

struct BwdArgs {
  Problem p;
  RowCoef r;
  void *dtable;
  float *dbias, *part;
  int64_t xtiles, ytiles, splits;
};

// fp16: a coefficient goes into the product times a power of two a candidate
// that follows its largest magnitude so far (from a start that any value
// passes: beyond 2^15 the largest is brought to 2^10), so that terms keep their
// digits down to 2^-24 of the largest whatever the gradients and p are of.
constexpr float kFirstScale = 0x1p100f, kMostHalf = 32768.f;
__device__ __forceinline__ float half_scale(float most) {   // (1 for what is not finite)
  const int e = int(__float_as_uint(most) >> 23);           // most >= 0
  return e >= 255 ? 1.f : __uint_as_float(uint32_t(min(max(264 - e, 1), 254)) << 23);
}

// XB blocks of 32 candidates a wave, four waves along the candidates.
template <typename T, int DB, int XB>
__global__ __launch_bounds__(kBlock, 1) void k_table_grad(BwdArgs a) {
  using M = Mma32<T>;
  constexpr int KS = M::KS, DP = 32 * DB, NK = DP / KS;
  using Tl = Tile32<T, DP>;
  constexpr int LD = Tl::LD;
  constexpr int YT = sizeof(T) == 4 ? 32 : 64, YS = YT / 32, XT = 32 * XB * kWaves, QL = YT + 4;
  constexpr bool HALF = std::is_same_v<T, fp16_t>;
  extern __shared__ __align__(16) char lds[];
  T *tiles = reinterpret_cast<T *>(lds);
  float *coef = reinterpret_cast<float *>(lds + size_t(2) * YT * LD * sizeof(T));   // [2][3][YT]
  float *q = coef + 2 * 3 * YT;   // [XT][QL]: what the tile's rows want of the candidates; zero between uses
  int *hit = reinterpret_cast<int *>(q + XT * QL);   // [waves]: whether any of a wave's is wanted

  const Problem &p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, col = lane & 31;
  const int wave = attn::wave_index();
  const int64_t xt = int64_t(blockIdx.x) / a.splits, split = int64_t(blockIdx.x) % a.splits;
  const int64_t t0 = split * a.ytiles / a.splits, t1 = (split + 1) * a.ytiles / a.splits;
  const int64_t v0 = xt * XT;
  const T *rows_h = static_cast<const T *>(p.h);

  FragOf<T> xf[XB][NK];
  float b2[XB], db[XB], sc[XB];
  const int64_t x0 = v0 + wave * (32 * XB) + col;
#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    const int64_t x = min(x0 + 32 * xb, p.V - 1);
    b2[xb] = p.bias != nullptr ? bias2(p, x) : 0.f;
    load_outer<T>(xf[xb], static_cast<const T *>(p.table) + x * p.ts, b2[xb] == -INFINITY, p.D);
    db[xb] = 0.f;
    sc[xb] = kFirstScale;
  }
  f32x16 o[XB][DB];
#pragma unroll
  for (int xb = 0; xb < XB; ++xb)
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[xb][d][r] = 0.f;

  Stage<T, DP, YT> next;
  float nc[3] = {-INFINITY, 0.f, 0.f};
  auto fetch = [&](int64_t t) {
    const int64_t y0 = t * YT, rows = p.N - y0;
    next.fetch(rows_h + y0 * p.hs, p.hs, rows, p.D);
    // rows without a gradient may hold anything
#pragma unroll
    for (int i = 0; i < next.NL; ++i)
      next.out[i] |= a.r.nm[y0 + min(int64_t(next.row(i)), rows - 1)] == -INFINITY;
    if (tid < YT) {
      const bool ok = tid < rows;
      const int64_t n = y0 + (ok ? tid : 0);
      nc[0] = ok ? a.r.nm[n] : -INFINITY;
      nc[1] = ok ? a.r.gl[n] : 0.f;
      nc[2] = ok ? a.r.gq[n] : 0.f;
    }
  };
  for (int i = tid; i < XT * QL; i += kBlock) q[i] = 0.f;
  if (tid < kWaves) hit[tid] = 0;
  Stage<T, DP, YT>::clear(tiles);
  Stage<T, DP, YT>::clear(tiles + YT * LD);
  __syncthreads();
  if (t0 < t1) fetch(t0);

  const int K = a.r.K;
#pragma unroll 1
  for (int64_t t = t0; t < t1; ++t) {
    const int buf = int(t - t0) & 1;
    T *tile = tiles + buf * YT * LD;
    float *cf = coef + buf * 3 * YT;
    next.put(tile, p.D);
    if (tid < YT) cf[tid] = nc[0], cf[YT + tid] = nc[1], cf[2 * YT + tid] = nc[2];
    // the tile's targets among the workgroup's candidates
    const int64_t y0 = t * YT, e0 = y0 * K;
    const int ne = int(min(int64_t(YT), p.N - y0)) * K;
    bool any = false;
    for (int e = tid; e < ne; e += kBlock) any |= uint64_t(int64_t(a.r.ids[e0 + e]) - v0) < uint64_t(XT);
    if (__syncthreads_or(any)) {   // (the waves are done with the tile before: q is clear)
      for (int e = tid; e < ne; e += kBlock) {
        const int64_t x = int64_t(a.r.ids[e0 + e]) - v0;
        if (uint64_t(x) < uint64_t(XT)) {   // each place at most once: a row has a candidate once
          q[x * QL + e / K] = a.r.weight != nullptr ? a.r.weight[e0 + e] : 1.f;
          hit[int(x) / (32 * XB)] = 1;
        }
      }
      __syncthreads();
    }
    if (t + 1 < t1) fetch(t + 1);
    const bool wanted = hit[wave] != 0;
#pragma unroll 1
    for (int ys = 0; ys < YS; ++ys) {
      const int row0 = ys * 32;
      f32x16 s[XB];
#pragma unroll
      for (int xb = 0; xb < XB; ++xb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[xb][r] = 0.f;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const FragOf<T> f = Tl::frag(tile, row0, k * KS);
#pragma unroll
        for (int xb = 0; xb < XB; ++xb) s[xb] = M::mma(f, xf[xb][k], s[xb]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float nm[4], gl[4];
        __builtin_memcpy(nm, cf + row0 + 8 * i + 4 * h, sizeof(nm));
        __builtin_memcpy(gl, cf + YT + row0 + 8 * i + 4 * h, sizeof(gl));
#pragma unroll
        for (int xb = 0; xb < XB; ++xb)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            s[xb][4 * i + v] = exp2_fast(fmaf(s[xb][4 * i + v], p.c, b2[xb]) + nm[v]) * gl[v];
      }
      if (wanted) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float gq[4];
          __builtin_memcpy(gq, cf + 2 * YT + row0 + 8 * i + 4 * h, sizeof(gq));
#pragma unroll
          for (int xb = 0; xb < XB; ++xb) {
            float w[4];
            __builtin_memcpy(w, q + (wave * (32 * XB) + 32 * xb + col) * QL + row0 + 8 * i + 4 * h, sizeof(w));
#pragma unroll
            for (int v = 0; v < 4; ++v) s[xb][4 * i + v] = fmaf(-gq[v], w[v], s[xb][4 * i + v]);
          }
        }
      }
      if (a.dbias != nullptr) {
#pragma unroll
        for (int xb = 0; xb < XB; ++xb) db[xb] += sum16(s[xb]);
      }
      if constexpr (HALF) {
        float most[XB];
        bool over = false;
#pragma unroll
        for (int xb = 0; xb < XB; ++xb) {
          float m[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) m[r] = fabsf(s[xb][r]);
#pragma unroll
          for (int d = 8; d > 0; d >>= 1)
#pragma unroll
            for (int r = 0; r < d; ++r) m[r] = fmaxf(m[r], m[r + d]);
          most[xb] = pair_max(m[0]);
          over |= most[xb] * sc[xb] > kMostHalf;
        }
        if (__any(over)) {
#pragma unroll
          for (int xb = 0; xb < XB; ++xb) {
            const float to = most[xb] * sc[xb] > kMostHalf ? half_scale(most[xb]) : sc[xb];
            const float by = to / sc[xb];
            sc[xb] = to;
            scale_blocks(o[xb], by);
          }
        }
#pragma unroll
        for (int xb = 0; xb < XB; ++xb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[xb][r] *= sc[xb];
      }
#pragma unroll
      for (int st = 0; st < 32 / KS; ++st) {
        FragOf<T> pf[XB];
#pragma unroll
        for (int xb = 0; xb < XB; ++xb) pf[xb] = frag_of16<T>(s[xb], st);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const FragOf<T> f = Tl::frag_t(tile, 32 * d, row0, st);
#pragma unroll
          for (int xb = 0; xb < XB; ++xb) o[xb][d] = M::mma(f, pf[xb], o[xb][d]);
        }
      }
    }
    if (wanted) {   // the wave's own part: clear before the next tile's targets come
      for (int i = lane; i < 32 * XB * QL; i += kWave) q[wave * 32 * XB * QL + i] = 0.f;
      if (lane == 0) hit[wave] = 0;
    }
  }

#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    const int64_t x = x0 + 32 * xb;
    const float sum = pair_sum(db[xb]);
    if (x >= p.V) continue;
    const float by = HALF ? p.scale / sc[xb] : p.scale;
    if (a.part != nullptr) {
      float *row = a.part + (split * p.V + x) * (DP + 1);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float w[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) w[v] = o[xb][d][4 * i + v] * by;
          store_n(row + 32 * d + 8 * i + 4 * h, w);
        }
      if (h == 0) row[DP] = sum;
    } else {
      T *row = static_cast<T *>(a.dtable) + x * p.D;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 w;
#pragma unroll
          for (int v = 0; v < 4; ++v) w[v] = o[xb][d][4 * i + v] * by;
          attn::store4<T>(row, 32 * d + 8 * i + 4 * h, p.D, w);
        }
      if (a.dbias != nullptr && h == 0) a.dbias[x] = sum;
    }
  }
}

// The splits' sums in their order, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void k_join_grad(const float *part, int64_t splits, int64_t V, int D, int dp,
                                                   T *dtable, float *dbias) {
  const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= V * (D + 1)) return;
  const int64_t v = at / (D + 1);
  const int d = int(at - v * (D + 1));
  if (d == D && dbias == nullptr) return;
  const float *src = part + v * (dp + 1) + (d == D ? dp : d);
  float x = 0.f;
  int64_t s = 0;
  for (; s + 8 <= splits; s += 8) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = src[(s + i) * V * (dp + 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) x += y[i];
  }
  for (; s < splits; ++s) x += src[s * V * (dp + 1)];
  if (d == D) dbias[v] = x;
  else dtable[v * D + d] = T(x);
}

// Which form: candidates of a workgroup, rows of a tile.
template <typename T>
constexpr int kXTile = sizeof(T) == 4 ? 128 : 256;
template <typename T>
constexpr int kYTile = sizeof(T) == 4 ? 32 : 64;

template <typename T>
int64_t pieces_of(const Problem &p) {
  const int64_t xt = (p.V + kXTile<T> - 1) / kXTile<T>, yt = (p.N + kYTile<T> - 1) / kYTile<T>;
  int64_t best = 1;
  double cost = 1e300;
  for (int64_t s = 1; s <= std::min<int64_t>(yt, 256); ++s) {
    const int64_t per = (yt + s - 1) / s, rounds = (xt * s + 255) / 256;
    const double t = double(rounds) * (double(per) + 4.0) + (s > 1 ? 4.0 + 0.02 * double(s * xt) : 0.0);
    if (t < cost) cost = t, best = s;
  }
  return best;
}

template <typename T, int DB>
void run(const BwdArgs &a, hipStream_t stream) {
  constexpr int XB = sizeof(T) == 4 ? 1 : 2;
  constexpr int LD = Tile32<T, 32 * DB>::LD, YT = kYTile<T>, XT = kXTile<T>;
  static_assert(XT == 32 * XB * kWaves, "");
  constexpr size_t bytes = size_t(2) * YT * LD * sizeof(T) + sizeof(float) * (6 * YT + XT * (YT + 4) + kWaves);
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  auto *k = &k_table_grad<T, DB, XB>;
  (void)ensure_dynamic_lds(reinterpret_cast<const void *>(k), bytes);
  launch(k, dim3(unsigned(a.xtiles * a.splits)), dim3(kBlock), bytes, stream, a);
}
template <typename T>
void pick(const Problem &p, const RowCoef &r, void *dtable, float *dbias, float *part, int64_t splits,
          hipStream_t stream) {
  const BwdArgs a{p, r, dtable, dbias, splits > 1 ? part : nullptr, (p.V + kXTile<T> - 1) / kXTile<T>,
                  (p.N + kYTile<T> - 1) / kYTile<T>, splits};
  const int dp = padded_dim(p.D);
  if (dp == 64) run<T, 2>(a, stream);
  else if (dp == 128) run<T, 4>(a, stream);
  else if (dp == 192) run<T, 6>(a, stream);
  else run<T, 8>(a, stream);
  if (splits > 1) {
    const int64_t n = p.V * (p.D + 1);
    launch(&k_join_grad<T>, dim3(unsigned((n + 255) / 256)), dim3(256), 0, stream, static_cast<const float *>(part),
           splits, p.V, p.D, dp, static_cast<T *>(dtable), dbias);
  }
}

}  // namespace

namespace sgl {
namespace cand {

int64_t table_grad_splits(int32_t dtype, const Problem &p) {
  return dtype == SGL_FP32 ? pieces_of<float>(p) : pieces_of<bf16_t>(p);
}

void table_grad(int32_t dtype, const Problem &p, const RowCoef &r, void *dtable, float *dbias, float *part,
                int64_t splits, hipStream_t stream) {
  if (dtype == SGL_FP32) return pick<float>(p, r, dtable, dbias, part, splits, stream);
  if (dtype == SGL_BF16) return pick<bf16_t>(p, r, dtable, dbias, part, splits, stream);
  return pick<fp16_t>(p, r, dtable, dbias, part, splits, stream);
}

}  // namespace cand
}  // namespace sgl
