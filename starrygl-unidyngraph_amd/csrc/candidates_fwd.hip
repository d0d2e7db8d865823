// Softmax over all candidates: each row's maximum and sum over a piece of the
// table and, for training, sum_v p_v w_v of that piece.
//
// One pass over the table: a tile of it gives scores, the running maximum and
// sum (what was summed is rescaled when the maximum has grown), and the tile's
// share of sum p w. 2 N V D operations, 4 with sum p w: the matrix unit
// and the vector unit (exponentials, maxima) bound it together, at the clock that
// the card's power leaves: 4,096 x 570,074 x 172 in bf16 1,558 us, 1,031 TFLOP/s, the
// matrix unit busy for half and the vector unit for 0.44 of the cycles, at 1.95 GHz of
// 2.4 (a large library product 1,099 TFLOP/s, 0.7 of the cycles at 1.5 to 1.9 GHz);
// rows of 100 channels 786 TFLOP/s (7 and 8 steps of 16 are run for 6.25); 600 x 100,000
// x 172 in fp32 400 us, 103 of 152. A few rows: the table's bytes, 1 x 1,140,149 x 172
// in 72 us, 5.4 TB/s.
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

// Two tiles in LDS, one being filled while the other is read, or one where two
// do not fit.
template <typename T, int DB, int YT>
constexpr int kBuffers = 2 * YT * Tile32<T, 32 * DB>::LD * int(sizeof(T)) <= 140 * 1024 ? 2 : 1;

// A wave has 32 rows; WX waves lie along the rows, WY along the table (few rows:
// each has 32 candidates of a tile of its own, and leaves a partial of its
// own). SUB steps of 32 candidates a tile. COUNT: no column of the tiles is free
// to sum p as rounded (a branch in the loop cost the products 2.6 %).
template <typename T, int DB, int CUT, int WX, int WY, int SUB, int PER_SIMD, bool DIR, bool COUNT>
__global__ __launch_bounds__(64 * WX * WY, PER_SIMD) void k_forward(FwdArgs a) {
  using M = Mma32<T>;
  constexpr int BLOCK = 64 * WX * WY, KS = M::KS, DP = 32 * DB, NK = DP / KS - CUT, TRIM = kTrim<T>, OB = DB - CUT / 2;
  static_assert(!COUNT || (DIR && sizeof(T) == 2), "p is rounded");
  using Tl = Tile32<T, DP>;
  constexpr int LD = Tl::LD, YT = 32 * SUB * WY, XT = 32 * WX, NBUF = kBuffers<T, DB, YT>;
  extern __shared__ __align__(16) char lds[];
  T *tiles = reinterpret_cast<T *>(lds);
  float *b2s = reinterpret_cast<float *>(lds + size_t(NBUF) * YT * LD * sizeof(T));

  const Problem &p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = attn::wave_index(), wx = wave % WX, wy = wave / WX;
  const int64_t N = a.order.count(p.N);
  const Line line((N + XT - 1) / XT, (p.V + YT - 1) / YT, a.out.groups);
  const int w = blockIdx.x;
  if (w >= line.groups) return;
  const int64_t u1 = line.begin(w + 1);
  const T *table = static_cast<const T *>(p.table);
  const bool biased = p.bias != nullptr;

  Stage<T, DP, YT, BLOCK> next(p.ts, p.D);
  float nb = 0.f;   // the bias of the next tile's row tid
  auto rows_of = [&](int t) { return int(min(p.V - int64_t(t) * YT, int64_t(YT))); };
  auto fetch = [&](int t) {
    const int64_t y0 = int64_t(t) * YT;
    const int rows = rows_of(t);
    next.fetch(table + y0 * p.ts, rows, biased ? p.bias + y0 : nullptr);
    if (biased && tid < YT) nb = p.bias[y0 + min(tid, rows - 1)];
  };
#pragma unroll
  for (int i = 0; i < NBUF; ++i) Stage<T, DP, YT, BLOCK>::clear(tiles + i * YT * LD, DIR ? a.out.ones : -1);
  int64_t u = line.begin(w);
  int xt = int(u / line.inner), t = int(u - int64_t(xt) * line.inner), buf = 0;
  fetch(t);
  __syncthreads();

#pragma unroll 1
  for (; u < u1; ++xt) {   // an outer tile's piece
    FragOf<T> xf[NK];
    const int D = fresh(p.D);
    const int64_t x = (int64_t(xt) * WX + wx) * 32 + (lane & 31);
    load_outer<T>(xf, static_cast<const T *>(p.h) + a.order.row(min(x, N - 1)) * p.hs, x >= N, D);
    // the maximum, as used, the sum and its compensation (a row's sum has up to 2^15 terms)
    float m = -INFINITY, mu = -kTop<T>, l = 0.f, lc = 0.f;
    // What the sum of p as rounded for sum p w has beyond l (COUNT). Where a tile has a column to spare it holds
    // ones, and the product sums them: 4,000 x 1,140,149 x 172 in bf16, both passes, 6,582 us with the vector unit's
    // sums, 6,366 so, 6,328 with none; 4,000 x 50,001 x 256 in fp16, no column to spare, 665 for 652.
    float off = 0.f;
    f32x16 o[DIR ? OB : 1];
#pragma unroll
    for (int d = 0; d < (DIR ? OB : 1); ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
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
      // The loss alone, bound by vector work: in whole tiles without a bias scores get their factor as their
      // exponentials are taken (4,096 x 570,074 in bf16, 172 channels 950 us for 1,085, 64 635 for 650; 4,000 x 50,001
      // x 100 in fp32 369 for 385; beside sum p w it gains nothing).
      const bool plain = !DIR && !biased && rows >= YT && p.c > 0.f;
      const float by_c = plain ? p.c : 1.f;
#pragma unroll 1
      for (int ys = 0; ys < SUB; ++ys) {
        const int row0 = (wy * SUB + ys) * 32;
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k)
          if (k < NK - TRIM || k * KS < p.D) s = M::mma(Tl::frag(tile, row0, k * KS), xf[k], s);
        if (!plain) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float b[4];
            __builtin_memcpy(b, b2 + row0 + 8 * i + 4 * h, sizeof(b));
#pragma unroll
            for (int v = 0; v < 4; ++v) s[4 * i + v] = fmaf(s[4 * i + v], p.c, b[v]);
          }
        }
        const float top = DIR ? pair_max(max16(s)) : pair_max(max16(s)) * by_c;
        if (__any(top > m + kSlack)) {
          const float mn = fmaxf(m, top);
          const float by = mn == m ? 1.f : exp2_fast(m - mn);
          m = mn;
          mu = (mn == -INFINITY ? 0.f : mn) - kTop<T>;
          l *= by;
          lc *= by;
          if constexpr (COUNT) off *= by;
          if constexpr (DIR) scale_blocks<PER_SIMD == 1>(o, by);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = exp2_fast(DIR ? s[r] - mu : fmaf(s[r], by_c, -mu));
        const float here = sum16(s), add = here - lc, sum = l + add;
        lc = (sum - l) - add;
        l = sum;
        if constexpr (COUNT) off -= here;
        if constexpr (DIR) {
#pragma unroll
          for (int st = 0; st < 32 / KS; ++st) {
            const FragOf<T> pf = frag_of16<T>(s, st);
            if constexpr (COUNT) off += frag_sum(pf);
#pragma unroll
            for (int d = 0; d < OB; ++d) o[d] = M::mma(Tl::frag_t(tile, 32 * d, row0, st), pf, o[d]);
          }
        }
      }
    }

    const int64_t at = (int64_t(w + xt) * WY + wy) * XT + wx * 32 + (lane & 31);
    const float sum = pair_sum(l), rounded = COUNT ? pair_sum(l + off) : 0.f;
    if (x < N) {
      if (h == 0) {
        a.out.m[at] = m == -INFINITY ? -INFINITY : mu;
        a.out.l[at] = sum;
        if constexpr (COUNT) a.out.r[at] = rounded;
      }
      if constexpr (DIR) {
        float *row = a.out.o + at * DP;
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float q[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) q[v] = o[d][4 * i + v];
            store_n(row + 32 * d + 8 * i + 4 * h, q);
          }
      }
    }
    t = 0;
  }
}

// Steps of 16 channels left out: 7 of 8 are slower than 8 (768 x 570,074 x 104 in
// bf16 262 us for 239), 6 faster, as 11 of 12 are.
template <int DB, int CUT>
constexpr int kForwardCut = DB == 4 && CUT == 1 ? 0 : CUT;
// Up to here a workgroup's waves share the rows and split the table.
constexpr int64_t kFewRows = 32;
constexpr int kFewWaves = 4;
// 16-bit rows in two workgroups a CU of four waves, where tiles of 128 rows
// leave out a sixth of what tiles of 256 take (600 rows: 640 of 768). Each
// then reads the table for half as many rows. 570,074 x 172 in bf16, 256 / 128: 100
// rows 110 / 84 us, 384 202 / 184, 600 299 / 283, 512 218 / 233, 1,200 512 / 548; not
// beyond 192 channels (their registers spill there: 600 x 256 499 / 825).
template <typename T, int DB>
struct Half {
  static constexpr bool AT_ALL = sizeof(T) == 2 && DB <= 6;
  static constexpr int WAVES = 4, GROUPS = 512;
  static bool takes(int64_t N) {
    const int64_t whole = (N + 255) / 256 * 256, halves = (N + 127) / 128 * 128;
    return AT_ALL && 6 * halves <= 5 * whole;
  }
};
template <typename T, int DB, int CUT>
Partials shape_of(const Problem &p) {
  using P = Plan<T, DB>;
  Partials s{};
  const bool few = p.N <= kFewRows, half = !few && Half<T, DB>::takes(p.N);
  s.rows = few ? 32 : 32 * (half ? Half<T, DB>::WAVES : P::WAVES);
  s.wy = few ? kFewWaves : 1;
  s.dp = 32 * DB;
  s.ones = sizeof(T) == 2 && p.D < 32 * (few ? DB : DB - CUT / 2) ? p.D : -1;
  s.groups = few ? 256 : half ? Half<T, DB>::GROUPS : P::GROUPS;
  const int ytile = few ? 32 * kFewWaves : 32 * P::SUB;
  s.ytiles = (p.V + ytile - 1) / ytile;
  return s;
}
template <typename T, int DB, int CUT, bool DIR, bool COUNT>
void run(const FwdArgs &a, hipStream_t stream) {
  using P = Plan<T, DB>;
  using H = Half<T, DB>;
  const Line line((a.p.N + a.out.rows - 1) / a.out.rows, a.out.ytiles, a.out.groups);
  auto go = [&](auto *k, int threads, size_t bytes) {
    (void)ensure_dynamic_lds(reinterpret_cast<const void *>(k), bytes);
    launch(k, dim3(unsigned(line.groups)), dim3(unsigned(threads)), bytes, stream, a);
  };
  constexpr size_t row = Tile32<T, 32 * DB>::LD * sizeof(T) + sizeof(float);
  constexpr int few = 32 * kFewWaves, many = 32 * P::SUB;
  constexpr size_t few_bytes = kBuffers<T, DB, few> * few * row, many_bytes = kBuffers<T, DB, many> * many * row;
  static_assert(few_bytes <= 160 * 1024 && many_bytes <= 160 * 1024 * P::GROUPS_PER_TWO / 2, "LDS of a CU");
  static_assert(!H::AT_ALL || many_bytes <= 80 * 1024, "two workgroups a CU");
  if (a.p.N <= kFewRows) {
    if constexpr (!COUNT || CUT == 0)   // (these tiles keep all columns: one is free where steps are left out)
      go(&k_forward<T, DB, 0, 1, kFewWaves, 1, P::PER_SIMD, DIR, COUNT>, 64 * kFewWaves, few_bytes);
    return;
  }
  if constexpr (H::AT_ALL)
    if (H::takes(a.p.N)) {
      go(&k_forward<T, DB, CUT, H::WAVES, 1, P::SUB, P::PER_SIMD, DIR, COUNT>, 64 * H::WAVES, many_bytes);
      return;
    }
  go(&k_forward<T, DB, CUT, P::WAVES, 1, P::SUB, P::PER_SIMD, DIR, COUNT>, 64 * P::WAVES, many_bytes);
}
template <typename T, int DB, int CUT>
void pick(const FwdArgs &a, hipStream_t stream) {
  if (a.out.o == nullptr) run<T, DB, CUT, false, false>(a, stream);
  else if (a.out.r == nullptr) run<T, DB, CUT, true, false>(a, stream);
  else if constexpr (sizeof(T) == 2 && CUT != 1) run<T, DB, CUT, true, true>(a, stream);   // (a column is free with 1)
}

}  // namespace

namespace sgl {
namespace cand {

Partials forward_shape(int32_t dtype, const Problem &p) {
  return pick_dim(dtype, p.D, [&](auto t, auto db, auto cut) {
    return shape_of<decltype(t), db.value, kForwardCut<db.value, cut.value>>(p);
  });
}

void forward_partials(int32_t dtype, const Problem &p, const Order &order, const Partials &out, hipStream_t stream) {
  const FwdArgs a{p, order, out};
  pick_dim(dtype, p.D, [&](auto t, auto db, auto cut) {
    pick<decltype(t), db.value, kForwardCut<db.value, cut.value>>(a, stream);
  });
}

}  // namespace cand
}  // namespace sgl
