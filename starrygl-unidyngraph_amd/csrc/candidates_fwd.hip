// Softmax over all candidates: each row's maximum and sum over a piece of the
// table and, for training, sum_v p_v w_v of that piece.
#include "candidates.h"

namespace {

using namespace sgl;
using namespace sgl::cand;

struct FwdArgs {
  Problem p;
  Partials out;
  int64_t xtiles, ytiles, splits, deal;   // splits: pieces of the table (each WY partials), dealt to `deal` XCDs
};

// fp16: p lies in 2^-24 .. 2^16, so the row's maximum is put at 2^7 (with the
// slack below it stays under 2^15) and terms keep digits down to 2^-21 of it.
template <typename T>
constexpr float kTop = std::is_same_v<T, fp16_t> ? 7.f : 0.f;
// A maximum is replaced (and what was summed rescaled) once it has grown by
// this many powers of two: exact whichever maximum is used, and most tiles
// then rescale nothing.
constexpr float kSlack = 8.f;

// XB blocks of 32 rows a wave; WX waves along the rows, 4 / WX along the table.
template <typename T, int DB, int XB, int WX, bool DIR>
__global__ __launch_bounds__(kBlock, 1) void k_forward(FwdArgs a) {
  using M = Mma32<T>;
  constexpr int KS = M::KS, DP = 32 * DB, NK = DP / KS;
  using Tl = Tile32<T, DP>;
  constexpr int LD = Tl::LD;
  constexpr int WY = kWaves / WX, YS = WX == kWaves ? 2 : 1, YT = 32 * YS * WY;
  constexpr int NBUF = 2 * YT * LD * int(sizeof(T)) <= 140 * 1024 ? 2 : 1;
  extern __shared__ __align__(16) char lds[];
  T *tiles = reinterpret_cast<T *>(lds);
  float *b2s = reinterpret_cast<float *>(lds + size_t(NBUF) * YT * LD * sizeof(T));

  const Problem &p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = attn::wave_index(), wx = wave % WX, wy = wave / WX;
  // workgroups of one piece of the table are dealt to one XCD: they share its L2
  const int64_t id = blockIdx.x, j = id / a.deal;
  const int64_t split = id % a.deal + a.deal * (j / a.xtiles), xt = j % a.xtiles;
  if (split >= a.splits) return;
  const int64_t t0 = split * a.ytiles / a.splits, t1 = (split + 1) * a.ytiles / a.splits;
  const T *table = static_cast<const T *>(p.table);

  FragOf<T> xf[XB][NK];
  const int64_t x0 = (xt * WX + wx) * (32 * XB) + (lane & 31);
#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    const int64_t x = x0 + 32 * xb;
    load_outer<T>(xf[xb], static_cast<const T *>(p.h) + min(x, p.N - 1) * p.hs, x >= p.N, p.D);
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

  Stage<T, DP, YT> next;
  float nb = 0.f;   // the bias of the next tile's row tid, to base 2
  auto fetch = [&](int64_t t) {
    const int64_t y0 = t * YT, rows = p.V - y0;
    next.fetch(table + y0 * p.ts, p.ts, rows, p.D);
    if (p.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < next.NL; ++i) next.out[i] |= p.bias[y0 + min(int64_t(next.row(i)), rows - 1)] == -INFINITY;
    }
    if (tid < YT) nb = tid >= rows ? -INFINITY : p.bias != nullptr ? bias2(p, y0 + tid) : 0.f;
  };
#pragma unroll
  for (int i = 0; i < NBUF; ++i) Stage<T, DP, YT>::clear(tiles + i * YT * LD);
  __syncthreads();
  if (t0 < t1) fetch(t0);
#pragma unroll 1
  for (int64_t t = t0; t < t1; ++t) {
    const int buf = NBUF == 2 ? int(t - t0) & 1 : 0;
    T *tile = tiles + buf * YT * LD;
    float *b2 = b2s + buf * YT;
    if (NBUF == 1 && t > t0) __syncthreads();
    next.put(tile, p.D);
    if (tid < YT) b2[tid] = nb;
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
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

  const int64_t part = split * WY + wy;
#pragma unroll
  for (int xb = 0; xb < XB; ++xb) {
    const int64_t x = x0 + 32 * xb;
    const float sum = pair_sum(l[xb]);
    if (x >= p.N) continue;
    if (h == 0) {
      a.out.m[part * p.N + x] = m[xb] == -INFINITY ? -INFINITY : mu[xb];
      a.out.l[part * p.N + x] = sum;
    }
    if constexpr (DIR) {
      float *row = a.out.o + (part * p.N + x) * DP;
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
}

// Which form: rows of a workgroup, waves along the rows.
struct Form {
  int rows, waves_y, ytile;
};
template <typename T>
Form form_of(int64_t N) {
  if (N <= 32) return Form{32, 4, 128};
  return Form{sizeof(T) == 4 ? 128 : 256, 1, 64};
}

template <typename T>
int64_t pieces_of(const Problem &p) {
  const Form f = form_of<T>(p.N);
  const int64_t xt = (p.N + f.rows - 1) / f.rows, yt = (p.V + f.ytile - 1) / f.ytile;
  // one workgroup a CU at a time: whole rounds of 256, the fewest that come near it
  int64_t best = 1;
  double cost = 1e300;
  for (int64_t s = 1; s <= std::min<int64_t>(yt, 512); ++s) {
    const int64_t per = (yt + s - 1) / s, rounds = (xt * s + 255) / 256;
    const double t = double(rounds) * (double(per) + 4.0) + 0.02 * double(s * xt);
    if (t < cost) cost = t, best = s;
  }
  return best;
}

template <typename T, int DB, int XB, int WX, bool DIR>
void run(const FwdArgs &a, hipStream_t stream) {
  constexpr int DP = 32 * DB, LD = Tile32<T, DP>::LD, YS = WX == kWaves ? 2 : 1, YT = 32 * YS * (kWaves / WX);
  constexpr int NBUF = 2 * YT * LD * int(sizeof(T)) <= 140 * 1024 ? 2 : 1;
  constexpr size_t bytes = size_t(NBUF) * YT * (LD * sizeof(T) + sizeof(float));
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  auto *k = &k_forward<T, DB, XB, WX, DIR>;
  (void)ensure_dynamic_lds(reinterpret_cast<const void *>(k), bytes);
  const int64_t grid = a.deal * a.xtiles * ((a.splits + a.deal - 1) / a.deal);
  launch(k, dim3(unsigned(grid)), dim3(kBlock), bytes, stream, a);
}
template <typename T, int DB, bool DIR>
void pick_form(const FwdArgs &a, hipStream_t stream) {
  constexpr int XB = sizeof(T) == 4 ? 1 : 2;
  if (a.p.N <= 32)
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
void pick_dir(const Problem &p, const Partials &out, bool dir, hipStream_t stream) {
  const Form f = form_of<T>(p.N);
  const int64_t splits = out.splits / f.waves_y;
  const FwdArgs a{p, out, (p.N + f.rows - 1) / f.rows, (p.V + f.ytile - 1) / f.ytile, splits,
                  std::min<int64_t>(splits, 8)};
  if (dir) pick_dim<T, true>(a, stream);
  else pick_dim<T, false>(a, stream);
}

}  // namespace

namespace sgl {
namespace cand {

int padded_dim(int D) { return (D + 63) / 64 * 64; }

int64_t forward_splits(int32_t dtype, const Problem &p, bool) {
  const int wy = p.N <= 32 ? 4 : 1;
  if (dtype == SGL_FP32) return pieces_of<float>(p) * wy;
  return pieces_of<bf16_t>(p) * wy;
}

void forward_partials(int32_t dtype, const Problem &p, const Partials &out, bool dir, hipStream_t stream) {
  if (dtype == SGL_FP32) return pick_dir<float>(p, out, dir, stream);
  if (dtype == SGL_BF16) return pick_dir<bf16_t>(p, out, dir, stream);
  return pick_dir<fp16_t>(p, out, dir, stream);
}

}  // namespace cand
}  // namespace sgl
