// Softmax over all candidates: each row's maximum and sum over a piece of the
// table and, for training, sum_v p_v w_v of that piece.
#include "candidates.h"

namespace {

using namespace sgl;
using namespace sgl::cand;

struct FwdArgs {
  Problem p;
  Order order;
  Partials out;
};

// fp16: p lies in 2^-24 .. 2^16, so the row's maximum is put at 2^7 (with the
// slack below it stays under 2^15) and terms keep digits down to 2^-21 of it.
template <typename T>
constexpr float kTop = std::is_same_v<T, fp16_t> ? 7.f : 0.f;
// A maximum is replaced (and what was summed rescaled) once it has grown by
// this many powers of two: exact whichever maximum is used, and most tiles
// then rescale nothing.
constexpr float kSlack = 8.f;

constexpr int64_t kFewRows = 32;   // up to here a workgroup's waves share them and split the table

// Blocks of 32 candidates of a wave in a tile: two for fewer barriers, one
// where the tile on its way would not fit in the registers.
template <typename T, int DB, int WX>
constexpr int kSubTiles = WX == kWaves && DB < 8 ? 2 : 1;

// XB blocks of 32 rows a wave; WX waves along the rows, 4 / WX along the table.
template <typename T, int DB, int XB, int WX, bool DIR>
__global__ __launch_bounds__(kBlock, 1) void k_forward(FwdArgs a) {
  using M = Mma32<T>;
  constexpr int KS = M::KS, DP = 32 * DB, NK = DP / KS;
  using Tl = Tile32<T, DP>;
  constexpr int LD = Tl::LD;
  constexpr int WY = kWaves / WX, YS = kSubTiles<T, DB, WX>, YT = 32 * YS * WY;
  constexpr int NBUF = 2 * YT * LD * int(sizeof(T)) <= 140 * 1024 ? 2 : 1;
  extern __shared__ __align__(16) char lds[];
  T *tiles = reinterpret_cast<T *>(lds);
  float *b2s = reinterpret_cast<float *>(lds + size_t(NBUF) * YT * LD * sizeof(T));

  const Problem &p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = attn::wave_index(), wx = wave % WX, wy = wave / WX;
  constexpr int XT = 32 * XB * WX;
  const int64_t N = a.order.count(p.N);
  const Line line((N + XT - 1) / XT, (p.V + YT - 1) / YT, kGroups);
  const int w = blockIdx.x;
  if (w >= line.groups) return;
  const int64_t u1 = line.begin(w + 1);
  const T *table = static_cast<const T *>(p.table);
  const bool biased = p.bias != nullptr;

  Stage<T, DP, YT> next(p.ts, p.D);
  float nb = 0.f;   // the bias of the next tile's row tid
  auto rows_of = [&](int t) { return int(min(p.V - int64_t(t) * YT, int64_t(YT))); };
  auto fetch = [&](int t) {
    const int64_t y0 = int64_t(t) * YT;
    const int rows = rows_of(t);
    next.fetch(table + y0 * p.ts, rows, biased ? p.bias + y0 : nullptr);
    if (biased && tid < YT) nb = p.bias[y0 + min(tid, rows - 1)];
  };
#pragma unroll
  for (int i = 0; i < NBUF; ++i) Stage<T, DP, YT>::clear(tiles + i * YT * LD);
  int64_t u = line.begin(w);
  int xt = int(u / line.inner), t = int(u - int64_t(xt) * line.inner), buf = 0;
  fetch(t);
  __syncthreads();

#pragma unroll 1
  for (; u < u1; ++xt) {   // an outer tile's piece
  FragOf<T> xf[XB][NK];
  const int D = fresh(p.D);
  const int64_t x0 = (int64_t(xt) * WX + wx) * (32 * XB) + (lane & 31);
#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    const int64_t x = x0 + 32 * xb, row = a.order.row(min(x, N - 1));
    load_outer<T>(xf[xb], static_cast<const T *>(p.h) + row * p.hs, x >= N, D);
  }
  float m[XB], mu[XB], l[XB], lc[XB];
  f32x16 o[XB][DIR ? DB : 1];
#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    m[xb] = -INFINITY;
    mu[xb] = -kTop<T>;
    l[xb] = lc[xb] = 0.f;
#pragma unroll
    for (int d = 0; d < (DIR ? DB : 1); ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[xb][d][r] = 0.f;
  }
  const int end = int(min(int64_t(line.inner), t + (u1 - u)));
  u += end - t;
#pragma unroll 1
  for (; t < end; ++t) {
    T *tile = tiles + buf * YT * LD;
    float *b2 = b2s + buf * YT;
    if (NBUF == 1) __syncthreads();
    const int rows = rows_of(t);
    next.put(tile, rows, biased);
    if (tid < YT) b2[tid] = tid >= rows ? -INFINITY : biased ? bias2_of(p, nb) : 0.f;
    __syncthreads();
    if (t + 1 < end || u < u1) fetch(t + 1 < end ? t + 1 : 0);   // (the next outer tile's first)
    if (NBUF == 2) buf ^= 1;
#pragma unroll 1
    for (int ys = 0; ys < YS; ++ys) {
      const int row0 = (wy * YS + ys) * 32;
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
      float top[XB];
      bool grow = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float b[4];
        __builtin_memcpy(b, b2 + row0 + 8 * i + 4 * h, sizeof(b));
#pragma unroll
        for (int xb = 0; xb < XB; ++xb)
#pragma unroll
          for (int v = 0; v < 4; ++v) s[xb][4 * i + v] = fmaf(s[xb][4 * i + v], p.c, b[v]);
      }
#pragma unroll
      for (int xb = 0; xb < XB; ++xb) {
        top[xb] = pair_max(max16(s[xb]));
        grow |= top[xb] > m[xb] + kSlack;
      }
      if (__any(grow)) {
#pragma unroll
        for (int xb = 0; xb < XB; ++xb) {
          const float mn = fmaxf(m[xb], top[xb]);
          const float by = mn == m[xb] ? 1.f : exp2_fast(m[xb] - mn);
          m[xb] = mn;
          mu[xb] = (mn == -INFINITY ? 0.f : mn) - kTop<T>;
          l[xb] *= by;
          lc[xb] *= by;
          if constexpr (DIR) scale_blocks(o[xb], by);
        }
      }
#pragma unroll
      for (int xb = 0; xb < XB; ++xb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[xb][r] = exp2_fast(s[xb][r] - mu[xb]);
        // a compensated sum of the blocks' sums: a row's sum has up to 2^15 of them
        const float add = sum16(s[xb]) - lc[xb], sum = l[xb] + add;
        lc[xb] = (sum - l[xb]) - add;
        l[xb] = sum;
      }
      if constexpr (DIR) {
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
    }
  }

  const int64_t part = int64_t(w + xt) * WY + wy;
#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    const int at = wx * (32 * XB) + 32 * xb + (lane & 31);
    const float sum = pair_sum(l[xb]);
    if (x0 + 32 * xb >= N) continue;
    if (h == 0) {
      a.out.m[part * XT + at] = m[xb] == -INFINITY ? -INFINITY : mu[xb];
      a.out.l[part * XT + at] = sum;
    }
    if constexpr (DIR) {
      float *row = a.out.o + (part * XT + at) * DP;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float q[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) q[v] = o[xb][d][4 * i + v];
          store_n(row + 32 * d + 8 * i + 4 * h, q);
        }
    }
  }
  t = 0;
  }
}

// Which form: by the rows.
template <typename T, int DB, int XB, int WX, bool DIR>
void run(const FwdArgs &a, hipStream_t stream) {
  constexpr int DP = 32 * DB, LD = Tile32<T, DP>::LD, YS = kSubTiles<T, DB, WX>, YT = 32 * YS * (kWaves / WX);
  constexpr int NBUF = 2 * YT * LD * int(sizeof(T)) <= 140 * 1024 ? 2 : 1;
  constexpr size_t bytes = size_t(NBUF) * YT * (LD * sizeof(T) + sizeof(float));
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  auto *k = &k_forward<T, DB, XB, WX, DIR>;
  (void)ensure_dynamic_lds(reinterpret_cast<const void *>(k), bytes);
  const Line line((a.p.N + 32 * XB * WX - 1) / (32 * XB * WX), (a.p.V + YT - 1) / YT, kGroups);
  launch(k, dim3(unsigned(line.groups)), dim3(kBlock), bytes, stream, a);
}
template <typename T, int DB, bool DIR>
void pick_form(const FwdArgs &a, hipStream_t stream) {
  constexpr int XB = sizeof(T) == 4 ? 1 : 2;
  if (a.p.N <= kFewRows)
    run<T, DB, 1, 1, DIR>(a, stream);
  else
    run<T, DB, XB, 4, DIR>(a, stream);
}
template <typename T, bool DIR>
void pick_dim(const FwdArgs &a, hipStream_t stream) {
  switch (padded_dim(a.p.D)) {
    case 64: return pick_form<T, 2, DIR>(a, stream);
    case 128: return pick_form<T, 4, DIR>(a, stream);
    case 192: return pick_form<T, 6, DIR>(a, stream);
    default: return pick_form<T, 8, DIR>(a, stream);
  }
}
template <typename T>
void pick_dir(const FwdArgs &a, hipStream_t stream) {
  if (a.out.o != nullptr) pick_dim<T, true>(a, stream);
  else pick_dim<T, false>(a, stream);
}

}  // namespace

namespace sgl {
namespace cand {

int padded_dim(int D) { return (D + 63) / 64 * 64; }

Partials forward_shape(int32_t dtype, const Problem &p) {
  Partials s{};
  const bool few = p.N <= kFewRows;
  s.rows = few ? 32 : dtype == SGL_FP32 ? 128 : 256;
  s.wy = few ? 4 : 1;
  s.dp = padded_dim(p.D);
  const int64_t ytile = few ? 128 : s.dp == 256 ? 32 : 64;
  s.ytiles = (p.V + ytile - 1) / ytile;
  return s;
}

void forward_partials(int32_t dtype, const Problem &p, const Order &order, const Partials &out, hipStream_t stream) {
  const FwdArgs a{p, order, out};
  if (dtype == SGL_FP32) return pick_dir<float>(a, stream);
  if (dtype == SGL_BF16) return pick_dir<bf16_t>(a, stream);
  return pick_dir<fp16_t>(a, stream);
}

}  // namespace cand
}  // namespace sgl
