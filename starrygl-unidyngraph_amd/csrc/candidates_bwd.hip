// The gradient of the table (and of a bias): dw_v = scale sum_n (gl_n e_nv -
// gq_n q_nv) h_n over the rows, e the forward's exponentials, formed again.
//
// 4 N V D operations, bound as the forward is: 4,096 x 570,074 x 172 in bf16 1,600
// us, 1,000 TFLOP/s; 600 x 100,000 x 172 in fp32 380 us, 109. Few rows: reading the
// candidates and writing their gradients, 128 x 570,074 x 172 177 us for 392 MB, which
// the products of a workgroup's next candidates do not cover (two workgroups of
// half the size a CU: 3 to 7 % less up to 600 rows, 3 to 5 % more from 1,200).
#include "candidates.h"

namespace {

using namespace sgl;
using namespace sgl::cand;

struct BwdArgs {
  Problem p;
  RowCoef r;
  void *dtable;
  float *dbias, *part;   // part: [pieces][candidates of a workgroup][dp + 4]
};
// Pieces of tiles that are shared out, the only ones that are kept apart: a
// workgroup has two at most, one of a tile begun earlier (2 w) and one of a tile
// that it begins and leaves (2 w + 1).
__device__ __forceinline__ int64_t shared_piece(int64_t w, bool begins) { return 2 * w + (begins ? 1 : 0); }

// fp16: a coefficient goes into the product times a power of two a candidate
// that follows its largest magnitude so far (from a start that any value
// passes: beyond 2^15 the largest is brought to 2^4, far enough below that a
// target after many small p does not do it again), so that terms keep their
// digits down to 2^-18 of the largest, and some of them to 2^-28, whatever the
// gradients and p are of.
constexpr float kFirstScale = 0x1p100f, kMostHalf = 32768.f;
__device__ __forceinline__ float half_scale(float most) {   // (1 for what is not finite)
  const int e = int(__float_as_uint(most) >> 23);           // most >= 0
  return e >= 255 ? 1.f : __uint_as_float(uint32_t(min(max(258 - e, 1), 254)) << 23);
}

// A tile in memory and in LDS (Image): steps of 32 rows. (Rows of 256 16-bit
// channels one step a tile: two take 634 us for 603, 768 x 570,074 in bf16.)
template <typename T, int DB>
struct Tiles {
  static constexpr int SUB = sizeof(T) == 4 || DB == 8 ? 1 : 2;
  static constexpr int YT = 32 * SUB, LD = Tile32<T, 32 * DB>::LD;
  static constexpr int ROWS = YT * LD * int(sizeof(T)), BYTES = ROWS + 16 * YT;
  static constexpr int XT = 32 * Plan<T, DB>::WAVES;   // candidates of a workgroup
  static constexpr int QL = 32 + 4;
  static_assert(BYTES % 1024 == 0, "whole loads of a wave");
};

// A wave has 32 candidates. What the tile's rows want of them is added behind
// the scores: a label a row, in the image (TEACHER false), or a teacher's
// entries, which are asked for before the scores and land while these are formed
// (1,200 x 1,140,149 x 172 in bf16, 64 entries a row: 1,309 us with their loads
// where they are used, 1,178 so).
template <typename T, int DB, int CUT, int WAVES, int PER_SIMD, bool TEACHER>
__global__ __launch_bounds__(64 * WAVES, PER_SIMD) void k_table_grad(BwdArgs a) {
  using M = Mma32<T>;
  using Im = Tiles<T, DB>;
  constexpr int BLOCK = 64 * WAVES;
  constexpr int KS = M::KS, DP = 32 * DB, NK = DP / KS - CUT, TRIM = kTrim<T>, OB = DB - CUT / 2;
  constexpr int YT = Im::YT, XT = Im::XT, QL = Im::QL;
  using Tl = Tile32<T, DP>;
  constexpr bool HALF = std::is_same_v<T, fp16_t>;
  extern __shared__ __align__(16) char lds[];
  // [XT][QL]: what 32 rows want of the candidates; zero between uses. A wave writes, reads and clears its
  // own candidates' part.
  float *q_all = reinterpret_cast<float *>(lds + 2 * Im::BYTES);

  const Problem &p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, col = lane & 31;
  const int wave = attn::wave_index();
  float *q = q_all + wave * 32 * QL;
  const int64_t N = a.r.live != nullptr ? int64_t(*a.r.live) : p.N;
  const Line line((p.V + XT - 1) / XT, max((N + YT - 1) / YT, int64_t(1)), Plan<T, DB>::GROUPS);
  const int w = blockIdx.x;
  if (w >= line.groups) return;
  const int64_t u1 = line.begin(w + 1);

  constexpr int NL = (Im::BYTES + 16 * BLOCK - 1) / (16 * BLOCK);
  typedef __attribute__((address_space(1))) const void *Global;
  typedef __attribute__((address_space(3))) void *Lds;
  int ne0 = 0, ne1 = 0;
  auto loads = [&](int i) { return (i + 1) * 16 * BLOCK <= Im::BYTES || (i * WAVES + wave) * 1024 < Im::BYTES; };
  // tile t into buffer `to`: straight to LDS, 1,024 bytes a wave and load (by way of registers 768 x 570,074 x 256 in
  // bf16 730 us for 603, x 172 411 for 398)
  auto fetch = [&](int t, int xt, int to) {
    const char *src = a.r.image + int64_t(t) * Im::BYTES + tid * 16;
    char *dst = lds + to * Im::BYTES + wave * 1024;
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (loads(i))
        __builtin_amdgcn_global_load_lds((Global)(src + i * 16 * BLOCK), (Lds)(dst + i * 16 * BLOCK), 16, 0, 0);
    if constexpr (TEACHER) {
      const int64_t vb = int64_t(xt) * WAVES + wave;
      const int32_t *at = a.r.index + int64_t(t) * (a.r.vblocks + 1) + min(vb, a.r.vblocks - 1);
      ne0 = attn::scalar_load(at);
      ne1 = vb < a.r.vblocks ? attn::scalar_load(at + 1) : ne0;
    }
  };
  for (int i = tid; i < XT * QL / 4; i += BLOCK) reinterpret_cast<f32x4 *>(q_all)[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  int64_t u = line.begin(w);
  int xt = int(u / line.inner), t = int(u - int64_t(xt) * line.inner), buf = 0;
  fetch(t, xt, buf);

#pragma unroll 1
  for (; u < u1; ++xt) {   // an outer tile's piece
    FragOf<T> xf[NK];
    const int D = fresh(p.D);
    const int64_t x = int64_t(xt) * XT + wave * 32 + col, xr = min(x, p.V - 1);
    const float b2 = p.bias != nullptr ? bias2(p, xr) : 0.f;
    const bool out = b2 == -INFINITY;
    load_outer<T>(xf, static_cast<const T *>(p.table) + xr * p.ts, out, D);
    float db = 0.f, sc = kFirstScale;
    f32x16 o[OB];
#pragma unroll
    for (int d = 0; d < OB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    const int first = t, end = int(min(int64_t(line.inner), t + (u1 - u)));
    u += end - t;
#pragma unroll 1
    for (; t < end; ++t) {
      char *image = lds + buf * Im::BYTES;
      const T *tile = reinterpret_cast<const T *>(image);
      const float *cf = reinterpret_cast<const float *>(image + Im::ROWS);
      buf ^= 1;
      const int e0 = ne0, e1 = ne1;
      const int2 *entries = a.r.entries + int64_t(t) * YT * a.r.K;
      __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's part of the tile has landed
      __syncthreads();
      // what the tile's rows want of the wave's candidates: a row has a candidate once, so each place once
      const int id = !TEACHER && lane < YT ? reinterpret_cast<const int *>(cf)[3 * YT + lane] : -1;
      const int mine = id - (xt * XT + wave * 32);
      const bool one = id >= 0 && uint32_t(mine) < 32u;
      const bool wanted = TEACHER ? e0 < e1 : __any(one);
      int2 entry = make_int2(-1, 0);   // the lane's of the first 64: on its way while the scores are formed
      if (TEACHER && e0 + lane < e1) entry = entries[e0 + lane];
      if (t + 1 < end || u < u1) fetch(t + 1 < end ? t + 1 : 0, t + 1 < end ? xt : xt + 1, buf);
#pragma unroll 1
      for (int ys = 0; ys < Im::SUB; ++ys) {
        const int row0 = ys * 32;
        if (!TEACHER && wanted) {
          if (one && (lane >> 5) == ys) q[mine * QL + (lane & 31)] = 1.f;
          attn::wave_sync();
        }
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k)
          if (k < NK - TRIM || k * KS < p.D) s = M::mma(Tl::frag(tile, row0, k * KS), xf[k], s);
        float c[16];   // (numbers of their own: as the product's block they would be moved between the register files)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float nm[4], gl[4];
          __builtin_memcpy(nm, cf + row0 + 8 * i + 4 * h, sizeof(nm));
          __builtin_memcpy(gl, cf + YT + row0 + 8 * i + 4 * h, sizeof(gl));
#pragma unroll
          for (int v = 0; v < 4; ++v) c[4 * i + v] = exp2_fast(fmaf(s[4 * i + v], p.c, b2) + nm[v]) * gl[v];
        }
        if (wanted) {
          const bool first = entry.x >= 0 && ((entry.x >> 5) & 1) == ys;
          float *to = q + (entry.x >> 6) * QL + (entry.x & 31);
          if constexpr (TEACHER) {
            if (first) *to = __int_as_float(entry.y);
            for (int k = e0 + kWave + lane; k < e1; k += kWave) {
              const int2 e = entries[k];
              if (((e.x >> 5) & 1) == ys) q[(e.x >> 6) * QL + (e.x & 31)] = __int_as_float(e.y);
            }
            attn::wave_sync();
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float gq[4], y[4];
            __builtin_memcpy(gq, cf + 2 * YT + row0 + 8 * i + 4 * h, sizeof(gq));
            __builtin_memcpy(y, q + col * QL + 8 * i + 4 * h, sizeof(y));
#pragma unroll
            for (int v = 0; v < 4; ++v) c[4 * i + v] = fmaf(-gq[v], y[v], c[4 * i + v]);
          }
          attn::wave_sync();
          if constexpr (TEACHER) {
            if (first) *to = 0.f;
            for (int k = e0 + kWave + lane; k < e1; k += kWave) {
              const int e = entries[k].x;
              if (((e >> 5) & 1) == ys) q[(e >> 6) * QL + (e & 31)] = 0.f;
            }
          } else if (one && (lane >> 5) == ys) {
            q[mine * QL + (lane & 31)] = 0.f;
          }
        }
        if constexpr (HALF) {
          const float most = pair_max(abs_max16(c));
          const bool over = most * sc > kMostHalf;
          if (__any(over)) {
            const float to = over ? half_scale(most) : sc;
            scale_blocks<PER_SIMD == 1>(o, to / sc);
            sc = to;
          }
        }
#pragma unroll
        for (int st = 0; st < 32 / KS; ++st) {
          const FragOf<T> pf = frag_of16<T>(c, st, HALF ? sc : 1.f);
#pragma unroll
          for (int d = 0; d < OB; ++d) o[d] = M::mma(Tl::frag_t(tile, 32 * d, row0, st), pf, o[d]);
        }
        if (a.dbias != nullptr) db += sum16(c);
      }
    }

    const int width = fresh(p.D);
    const bool whole = first == 0 && end == line.inner;
    const float sum = out ? 0.f : pair_sum(db), by = HALF ? p.scale / sc : p.scale;
    // (a row that is not finite makes NaN of every candidate that is in, and of those only)
    if (x < p.V) {
      if (!whole) {
        float *row = a.part + (shared_piece(w, first == 0) * XT + wave * 32 + col) * (DP + 4);
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = out ? 0.f : o[d][4 * i + v] * by;
            store_n(row + 32 * d + 8 * i + 4 * h, y);
          }
        if (h == 0) row[DP] = sum;
      } else {
        T *row = static_cast<T *>(a.dtable) + x * width;
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4 y;
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = out ? 0.f : o[d][4 * i + v] * by;
            attn::store4<T>(row, 32 * d + 8 * i + 4 * h, width, y);
          }
        if (a.dbias != nullptr && h == 0) a.dbias[x] = sum;
      }
    }
    t = 0;
  }
}

// Outer tiles whose rows were shared out: the pieces' sums in their order,
// rounded once. Workgroup b of kJoin parts looks after the tile that workgroup
// b / kJoin + 1 begins inside of, unless an earlier one does.
constexpr int kJoin = 8;
template <typename T>
__global__ __launch_bounds__(kBlock) void k_join_grad(BwdArgs a, int xtile, int ytile, int dp, int groups) {
  const Problem &p = a.p;
  const int64_t N = a.r.live != nullptr ? int64_t(*a.r.live) : p.N;
  const Line line((p.V + xtile - 1) / xtile, max((N + ytile - 1) / ytile, int64_t(1)), groups);
  const int w = blockIdx.x / kJoin + 1, part = blockIdx.x % kJoin;
  if (w >= line.groups) return;
  const int64_t u = line.begin(w), xt = u / line.inner;
  if (u == xt * line.inner || line.begin(w - 1) > xt * line.inner) return;
  const int64_t w0 = w - 1, w1 = line.group_of((xt + 1) * line.inner - 1);
  const int ld = dp + 4, n = int(w1 - w0), units = (p.D + 3) / 4 + 1;   // four columns a thread, and the bias
  const int64_t step = int64_t(xtile) * ld;
  // (the tile's first piece begins it, the others are of tiles begun earlier)
  const float *first = a.part + shared_piece(w0, true) * step, *rest = a.part + shared_piece(w, false) * step;
  const int rows = int(min(int64_t(xtile), p.V - xt * xtile));
  const int r0 = rows * part / kJoin, r1 = rows * (part + 1) / kJoin;
  for (int i = threadIdx.x; i < (r1 - r0) * units; i += kBlock) {
    const int r = r0 + i / units, c = i % units, d = c == units - 1 ? dp : 4 * c;
    const int64_t v = xt * xtile + r;
    const int64_t at = int64_t(r) * ld + d;
    f32x4 x = *reinterpret_cast<const f32x4 *>(first + at);
#pragma unroll 4
    for (int s = 0; s < n; ++s) x += *reinterpret_cast<const f32x4 *>(rest + 2 * s * step + at);
    if (d == dp) {
      if (a.dbias != nullptr) a.dbias[v] = x[0];
    } else {
      attn::store4<T>(static_cast<T *>(a.dtable) + v * p.D, d, p.D, x);
    }
  }
}

// ------------------------------------------------------------------ several targets a row
// A row tile's entries in the order of the candidates' blocks (those of a
// wave), with the place where each block begins: a workgroup a row tile and
// kBins blocks counts, sums and places the entries of its blocks in LDS, behind
// those of earlier ones. (The order of a block's entries varies; each is a
// place of its own.) 64 x 64 entries over 35,630 blocks: 28 us with one workgroup
// a row tile, 12 so.
constexpr int kRouteBlock = 1024, kBins = 12 * kRouteBlock;
struct RouteArgs {
  const int32_t *ids;     // [N][K]
  const float *weight;
  int64_t N, vblocks;
  int K, ytile, vblock;
  int32_t *index;
  int2 *entries;
};
__global__ __launch_bounds__(kRouteBlock) void k_route(RouteArgs a) {
  __shared__ int bins[kBins];
  __shared__ int waves[kRouteBlock / kWave];
  const int tid = threadIdx.x;
  const int64_t y0 = int64_t(blockIdx.x) * a.ytile, e0 = y0 * a.K, b0 = int64_t(blockIdx.y) * kBins;
  const int n = int(min(int64_t(a.ytile), a.N - y0)) * a.K;
  int32_t *index = a.index + int64_t(blockIdx.x) * (a.vblocks + 1);
  int2 *entries = a.entries + int64_t(blockIdx.x) * a.ytile * a.K;
  for (int i = tid; i < kBins; i += kRouteBlock) bins[i] = 0;
  __syncthreads();
  int earlier = 0;
  for (int e = tid; e < n; e += kRouteBlock) {
    const int id = a.ids[e0 + e];
    const int64_t b = id / a.vblock - b0;
    if (id >= 0 && b < 0) ++earlier;
    if (id >= 0 && b >= 0 && b < kBins) atomicAdd(&bins[b], 1);
  }
  int base, total;
  block_exclusive_scan<int, kRouteBlock>(earlier, waves, base);
  constexpr int PER = kBins / kRouteBlock;
  int c[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = sum;
    sum += bins[tid * PER + i];
  }
  const int before = base + block_exclusive_scan<int, kRouteBlock>(sum, waves, total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    bins[tid * PER + i] = before + c[i];
    if (b0 + tid * PER + i < a.vblocks) index[b0 + tid * PER + i] = before + c[i];
  }
  if (tid == 0 && blockIdx.y == gridDim.y - 1) index[a.vblocks] = base + total;
  __syncthreads();
  for (int e = tid; e < n; e += kRouteBlock) {
    const int id = a.ids[e0 + e];
    const int64_t b = id / a.vblock - b0;
    if (id >= 0 && b >= 0 && b < kBins)
      entries[atomicAdd(&bins[b], 1)] =
          make_int2((id - int(b0 + b) * a.vblock) * 64 + e / a.K, __float_as_int(a.weight[e0 + e]));
  }
}

template <typename T, int DB, int CUT>
void run(const BwdArgs &a, hipStream_t stream) {
  using P = Plan<T, DB>;
  using Im = Tiles<T, DB>;
  constexpr size_t bytes = size_t(2) * Im::BYTES + sizeof(float) * Im::XT * Im::QL;
  static_assert(bytes <= 160 * 1024 * P::GROUPS_PER_TWO / 2, "LDS of a CU");
  auto *k = a.r.index != nullptr ? &k_table_grad<T, DB, CUT, P::WAVES, P::PER_SIMD, true>
                                 : &k_table_grad<T, DB, CUT, P::WAVES, P::PER_SIMD, false>;
  (void)ensure_dynamic_lds(reinterpret_cast<const void *>(k), bytes);
  const Line line((a.p.V + Im::XT - 1) / Im::XT, (a.p.N + Im::YT - 1) / Im::YT, P::GROUPS);
  launch(k, dim3(unsigned(line.groups)), dim3(64 * P::WAVES), bytes, stream, a);
  if (line.groups > 1)
    launch(&k_join_grad<T>, dim3(unsigned(line.groups - 1) * kJoin), dim3(kBlock), 0, stream, a, int(Im::XT),
           int(Im::YT), 32 * DB, int(P::GROUPS));
}

}  // namespace

namespace sgl {
namespace cand {

Image grad_image(int32_t dtype, int D) {
  return pick_dim(dtype, D, [](auto t, auto db, auto) {
    using Im = Tiles<decltype(t), db.value>;
    return Image{Im::YT, Im::LD, Im::BYTES};
  });
}
int64_t table_grad_part(int32_t dtype, const Problem &p) {
  return pick_dim(dtype, p.D, [&](auto t, auto db, auto) {
    using P = Plan<decltype(t), db.value>;
    constexpr int64_t xtile = 32 * P::WAVES, ytile = Tiles<decltype(t), db.value>::YT;
    const Line line((p.V + xtile - 1) / xtile, (p.N + ytile - 1) / ytile, P::GROUPS);
    return 2 * int64_t(line.groups) * xtile * (32 * db.value + 4);
  });
}

void route_targets(int32_t dtype, const Problem &p, int K, const int32_t *ids, const float *weight, int32_t *index,
                   int2 *entries, hipStream_t stream) {
  const int yt = grad_image(dtype, p.D).rows;
  const RouteArgs a{ids, weight, p.N, (p.V + kGradBlock - 1) / kGradBlock, K, yt, kGradBlock, index, entries};
  launch(&k_route, dim3(unsigned((p.N + yt - 1) / yt), unsigned((a.vblocks + kBins - 1) / kBins)), dim3(kRouteBlock), 0,
         stream, a);
}

void table_grad(int32_t dtype, const Problem &p, const RowCoef &r, void *dtable, float *dbias, float *part,
                hipStream_t stream) {
  const BwdArgs a{p, r, dtable, dbias, part};
  pick_dim(dtype, p.D, [&](auto t, auto db, auto cut) { run<decltype(t), db.value, cut.value>(a, stream); });
}

}  // namespace cand
}  // namespace sgl
