// Forward kernels of the cross attention.
#include "cross_attention.h"

namespace sgl {
namespace attn {
namespace {

// ------------------------------------------------------------------ many rows
// A workgroup takes RW x NQ blocks of 16 rows of a (sequence, key head) and
// walks its keys a tile at a time with the running maximum and sum of the
// softmax (base 2); KW waves share each row block, each with its part of every
// tile, and are joined at the end: two to four waves a SIMD, whose chains of
// dependent steps (position, column, table, exp) fill each other's gaps, from
// grids of one or two workgroups a CU. The next tile's keys and values are in
// flight while the current one is worked on. The products are computed as
// (keys x rows) and (head size x rows): a lane keeps one row a block, so its
// maximum, sum and rescale are its own, joined over four lanes only. The
// accumulators are rescaled only when the maximum has grown by more than 2^6:
// p stays below 2^6, and the sum and the products carry the same factor.
// p is rounded to the operands' type for its product. Where a backward will
// follow, what that rounding leaves is multiplied too (kParts in all), so that o
// and `rest` together hold o as float32 would: D = <do, o> meets p dp in sums
// of a column over all rows and keys that nearly cancel, where an error in D,
// the same for a whole row, does not. In bf16 with p in one part the bias
// table's gradient of 8 sequences, 8 heads of 64 (2 key heads), 1000 x 2049 was
// 2.6e-3 off, in two 4.6e-6, in three 3.9e-6 (the formula in float32 throughout:
// 2.9e-6); of 4 sequences of one row and 444 keys 6.4e-5 in two, 9e-6 in three
// (5e-6). The first takes 119, 149 or 177 us forward (21 GFLOP). A block of
// rows at a time then, its values' fragments read again: kept in registers for
// all blocks they spill (220 us).
constexpr float kSlack = 6.f;

// What the backward reads of a row's softmax: the maximum m that the sum is
// relative to and log2 of the sum, so that p = 2^((x - m) - log2 l). The two
// apart: in one number log2 l is lost beside a large m (all of a row's buckets
// at -1e9, say), and p is 1 at every key. Infinite without a live key: p is 0
// there. A NaN score's row keeps its NaN.
__device__ __forceinline__ float2 row_sum(float m, float l, bool ok) {
  return ok && l != 0.f ? make_float2(m, __log2f(l)) : make_float2(INFINITY, 0.f);
}

template <typename T, int DP, int TK>
struct alignas(16) FwdLds {
  T k[TK * Tile<T, DP>::LD], v[TK * Tile<T, DP>::LD];
  KeyInfo<TK> info;
};

template <typename T, int DP, int NQ, bool SHARE, int RW, int KW, bool SPLIT>
__global__ __launch_bounds__(RW * KW * 64, (simd_waves<T, DP>(4, 2))) void k_attn_fwd(Args a, int64_t tiles, T *__restrict__ o,
                                                           T *__restrict__ rest, float2 *__restrict__ lse) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  constexpr int TK = tile_keys<T>(KW), BLOCK = RW * KW * 64;
  constexpr int ST = DP / M::KS, DB = DP / 16, KB = TK / 16 / KW;
  constexpr int NP = SHARE ? 1 : NQ;   // positions a lane holds
  extern __shared__ __align__(16) char smem[];
  using S = FwdLds<T, DP, TK>;
  constexpr int NB = buffers<S>();
  S *const bufs = reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + NB * sizeof(S));
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15;
  const int wr = w / KW, k0 = (w % KW) * KB * 16;   // this wave's row blocks, and its first key of a tile
  const TileAt at_ = tile_at(blockIdx.x, uint32_t(tiles), p.heads_kv);
  const uint32_t rt = at_.tile;
  const int hk = at_.hk;
  const int64_t n = at_.n;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  // the workgroup's first query; nothing to do past the length
  const uint32_t t0 = rt * (SHARE ? RW * 16 : RW * 16 * NQ);
  const uint32_t i0 = __builtin_amdgcn_readfirstlane(row_at<SHARE>(t0, 0, a.G).i);
  const bool any = i0 < q.qlen;
  if (biased) stage_bias(table, a, hk, threadIdx.x, BLOCK);
  RowAt row[NQ];
  bool in[NQ], ok[NQ];
  FragOf<T> qf[NQ][ST];
  int64_t qpos[NP];
  int qrel[NP];
  const int64_t base = biased && any ? scalar_load(q.qpos + int64_t(i0) * p.qpos_t) : 0;
  bool qnear = true;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    const uint32_t t = SHARE ? t0 + wr * 16 + cl : t0 + (wr * NQ + b) * 16 + cl;
    row[b] = row_at<SHARE>(t, b, a.G);
    in[b] = row[b].i < p.lq;
    ok[b] = row[b].i < q.qlen;
#pragma unroll
    for (int st = 0; st < ST; ++st)
      qf[b][st] = load_row<T>(q.q + int64_t(row[b].i) * p.q_t + row[b].h * p.q_h, ok[b], st * M::KS + g * M::E, dh);
    if (b < NP) {
      qpos[b] = biased && ok[b] ? q.qpos[int64_t(row[b].i) * p.qpos_t] : base;
      qnear = qnear && is_near(qpos[b] - base);
      qrel[b] = int(qpos[b] - base);
    }
  }
  qnear = __all(qnear);
  const float c = p.scale * kLog2e;
  float m[NQ], l[NQ];
  f32x4 acc[NQ][DB];
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  KeyTile<T, DP, TK, BLOCK> tile(a);
  if (any && q.klen > 0) tile.load(q, a, 0);
  int buf = 0;
  for (int64_t j0 = 0; any && j0 < q.klen; j0 += TK) {
    S &s = bufs[buf];
    if constexpr (NB == 1) __syncthreads();
    else buf ^= 1;
    tile.store(s.k, s.v, s.info, q, a, base);
    const uint32_t on = tile.live_of(k0, KB * 16);   // this wave's keys
    __syncthreads();
    if (j0 + TK < q.klen) tile.load(q, a, j0 + TK);
    float x[NQ][KB][4], mx[NQ];
    int col[NP][KB][4];
    if (biased) {
      const bool near_now = qnear && s.info.near_ != 0;
#pragma unroll
      for (int b = 0; b < NP; ++b) columns(col[b], s.info.pos, k0 + 4 * g, qrel[b], qpos[b], near_now, 1, bk);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      FragOf<T> kf[ST];
#pragma unroll
      for (int st = 0; st < ST; ++st) kf[st] = L::frag(s.k, k0 + kb * 16, st * M::KS);
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) sc = M::mma(kf[st], qf[b][st], sc);
#pragma unroll
        for (int v = 0; v < 4; ++v) x[b][kb][v] = sc[v];
      }
    }
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      mx[b] = -INFINITY;
      scale_scores(x[b], c, 0.f, table + row[b].h * table_ld(a), col[b < NP ? b : 0], biased);
    }
    if (on != full_mask(KB * 16)) {   // uniform
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const bool dead = !((on >> (kb * 16 + 4 * g + v)) & 1);
#pragma unroll
          for (int b = 0; b < NQ; ++b) x[b][kb][v] = dead ? -INFINITY : x[b][kb][v];
        }
    }
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) mx[b] = fmaxf(mx[b], x[b][kb][v]);
      if (__any(mx[b] > m[b] + kSlack)) {   // (uniform over the wave; also the first live tile)
        const float mn = fmaxf(m[b], groups_max(mx[b]));
        const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[b] - mn);
        l[b] *= alpha;
        m[b] = mn;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[b][d] *= alpha;
      }
      const float at = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = __builtin_amdgcn_exp2f(x[b][kb][v] - at);
          l[b] += x[b][kb][v];
        }
    }
    if constexpr (!SPLIT) {
#pragma unroll
      for (int st = 0; st < KB * 16 / M::KS; ++st) {
        FragOf<T> pf[NQ];
#pragma unroll
        for (int b = 0; b < NQ; ++b) pf[b] = frag_of<T>(x[b], st);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const FragOf<T> vf = L::template frag_t<TK>(s.v, d * 16, k0 + st * M::KS);
#pragma unroll
          for (int b = 0; b < NQ; ++b) acc[b][d] = M::mma(vf, pf[b], acc[b][d]);
        }
      }
    } else {   // a block at a time, the values' fragments read again: no registers to keep them
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int st = 0; st < KB * 16 / M::KS; ++st) {
          FragOf<T> pf[kParts<T>];
          split_frag_of<T>(x[b], st, pf);
          asm volatile("" ::: "memory");
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const FragOf<T> vf = L::template frag_t<TK>(s.v, d * 16, k0 + st * M::KS);
#pragma unroll
            for (int i = 0; i < kParts<T>; ++i) acc[b][d] = M::mma(vf, pf[i], acc[b][d]);
          }
        }
    }
  }
#pragma unroll
  for (int b = 0; b < NQ; ++b) l[b] = groups_sum(l[b]);
  join_waves<RW, KW, NQ, DB>(smem, m, l, acc);
  if (w % KW != 0) return;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    if (!in[b]) continue;
    const float inv = ok[b] && l[b] != 0.f ? 1.f / l[b] : 0.f;
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const f32x4 v = acc[b][d] * inv;
      store4(o + at, d * 16 + 4 * g, dh, v);
      if (rest != nullptr) store_rest(rest + at, d * 16 + 4 * g, dh, v);   // for the backward's D
    }
    if (lse != nullptr && g == 0)
      lse[(n * p.heads_kv + hk) * a.rows + int64_t(row[b].i) * a.G + row[b].h] = row_sum(m[b], l[b], ok[b]);
  }
}

// ------------------------------------------------------------------ few rows
// Up to 16 NQ rows a (sequence, key head): there is no reuse of a key beyond a
// wave, so the waves work apart: keys go from memory straight into fragments,
// values through the wave's own LDS tile for the transposed read, 32 keys at
// a time, the next ones in flight. One wave takes a short sequence (`parts` 0);
// long ones are split over the four waves of `parts` workgroups, whose
// (maximum, sum, products) are joined in LDS and, with several workgroups, by
// a second kernel. Bound by the chain of loads of a wave (counts, then keys and
// positions, then the values' LDS tile) at three waves a SIMD: 32 x 8192 keys,
// 2 heads of 64 in bf16, 28 us and 4 joined (105 MB: 3.7 TB/s in the first);
// 4000 windows of 20 x 32, 4 heads of 43: 67 us (1.9 TB/s).
constexpr int kStep = 32;

template <typename T, int DP, int NQ>
struct alignas(16) FewLds {
  T v[kStep * Tile<T, DP>::LD];
  PosTile<kStep> pos;
};

template <typename T, int DP, int NQ, bool SPLIT>
__global__ __launch_bounds__(kBlock, (simd_waves<T, DP>(3, DP <= 64 ? 2 : 1))) void k_attn_few(Args a, int parts, int64_t part_keys, T *__restrict__ o,
                                                     T *__restrict__ rest, float2 *__restrict__ lse,
                                                     float *__restrict__ pacc, float2 *__restrict__ pml) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  constexpr int ST = DP / M::KS, DB = DP / 16, KB = kStep / 16;
  extern __shared__ __align__(16) char smem[];
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15;
  using Lds = FewLds<T, DP, NQ>;
  const size_t per = align_bytes(sizeof(Lds) + table_bytes(a));
  Lds &s = *reinterpret_cast<Lds *>(smem + w * per);
  float *table = reinterpret_cast<float *>(smem + w * per + sizeof(Lds));
  const TileAt at_ = parts == 0 ? tile_at(blockIdx.x * kWaves + w, 1, p.heads_kv)
                                : tile_at(blockIdx.x, uint32_t(parts), p.heads_kv);
  const int hk = at_.hk, part = int(at_.tile);
  const int64_t n = at_.n, item = n * p.heads_kv + hk;
  if (n >= p.n) return;   // (whole waves of the form without barriers)
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  if (biased) {
    stage_bias(table, a, hk, lane, kWave);
    wave_sync();
  }
  RowAt row[NQ];
  bool in[NQ], ok[NQ];
  FragOf<T> qf[NQ][ST];
  int64_t qpos[NQ];
  int qrel[NQ];
  const int64_t base = biased && q.qlen > 0 ? scalar_load(q.qpos) : 0;
  bool qnear = true;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    row[b] = row_at<false>(uint32_t(b * 16 + cl), b, a.G);
    in[b] = row[b].i < p.lq;
    ok[b] = row[b].i < q.qlen;
#pragma unroll
    for (int st = 0; st < ST; ++st)
      qf[b][st] = load_row<T>(q.q + int64_t(row[b].i) * p.q_t + row[b].h * p.q_h, ok[b], st * M::KS + g * M::E, dh);
    qpos[b] = biased && ok[b] ? q.qpos[int64_t(row[b].i) * p.qpos_t] : base;
    qnear = qnear && is_near(qpos[b] - base);
    qrel[b] = int(qpos[b] - base);
  }
  qnear = __all(qnear);
  const float c = p.scale * kLog2e;
  float m[NQ], l[NQ];
  f32x4 acc[NQ][DB];
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t stride = parts == 0 ? kStep : kStep * kWaves;
  const int64_t end = q.qlen > 0 ? (parts == 0 ? q.klen : min(q.klen, (part + 1) * part_keys)) : 0;
  int64_t j0 = parts == 0 ? 0 : part * part_keys + w * kStep;
  constexpr int PER = kStep * L::UPR / kWave;
  FragOf<T> kr[KB][ST], vr[PER];
  int64_t kpos = 0;
  int byte = 0;
  auto load_tile = [&](int64_t j) {   // (only issues loads: what they bring is looked at a step later)
    const bool in = lane < kStep && j + lane < q.klen;
    byte = 0;
    kpos = 0;
    if (q.mask != nullptr && in) byte = q.mask[(j + lane) * p.mask_t];
    if (biased && in) kpos = q.kpos[(j + lane) * p.kpos_t];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int st = 0; st < ST; ++st)
        kr[kb][st] = load_raw<T>(q.k + (j + kb * 16 + cl) * p.k_t, j + kb * 16 + cl < q.klen, st * M::KS + g * M::E, dh);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = lane + i * kWave, r = u / L::UPR, d = (u % L::UPR) * M::E;
      vr[i] = load_raw<T>(q.v + (j + r) * p.v_t, j + r < q.klen, d, dh);
    }
  };
  if (j0 < end) load_tile(j0);
  for (; j0 < end; j0 += stride) {
    uint32_t on = uint32_t(first_bits(q.klen - j0));
    if (q.mask != nullptr) on &= uint32_t(__ballot(byte != 0));
    FragOf<T> kf[KB][ST];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        kf[kb][st] = fix<T>(kr[kb][st], st * M::KS + g * M::E, dh);
        if (q.mask != nullptr && !((on >> (kb * 16 + cl)) & 1)) kf[kb][st] = zero_frag<T>();
      }
    const int64_t kp = lane < kStep && ((on >> (lane & 31)) & 1) ? kpos : base;
    const bool near_now = qnear && __all(is_near(kp - base));
    wave_sync();   // the reads of the tile before are done
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = lane + i * kWave, r = u / L::UPR, d = (u % L::UPR) * M::E;
      FragOf<T> vv = fix<T>(vr[i], d, dh);
      if (q.mask != nullptr && !((on >> r) & 1)) vv = zero_frag<T>();
      *reinterpret_cast<FragOf<T> *>(s.v + r * L::LD + d) = vv;
    }
    if (biased && lane < kStep) {
      s.pos.pos[lane] = kp;
      s.pos.rel[lane] = int(kp - base);
    }
    wave_sync();
    if (j0 + stride < end) load_tile(j0 + stride);
    float x[NQ][KB][4];
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      float mx = -INFINITY;
      int col[KB][4];
      if (biased) columns(col, s.pos, 4 * g, qrel[b], qpos[b], near_now, 1, bk);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) sc = M::mma(kf[kb][st], qf[b][st], sc);
#pragma unroll
        for (int v = 0; v < 4; ++v) x[b][kb][v] = sc[v];
      }
      scale_scores(x[b], c, 0.f, table + row[b].h * table_ld(a), col, biased);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = (on >> (kb * 16 + 4 * g + v)) & 1 ? x[b][kb][v] : -INFINITY;
          mx = fmaxf(mx, x[b][kb][v]);
        }
      if (__any(mx > m[b] + kSlack)) {
        const float mn = fmaxf(m[b], groups_max(mx));
        const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[b] - mn);
        l[b] *= alpha;
        m[b] = mn;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[b][d] *= alpha;
      }
      const float at = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = __builtin_amdgcn_exp2f(x[b][kb][v] - at);
          l[b] += x[b][kb][v];
        }
    }
    if constexpr (!SPLIT) {
#pragma unroll
      for (int st = 0; st < kStep / M::KS; ++st) {
        FragOf<T> pf[NQ];
#pragma unroll
        for (int b = 0; b < NQ; ++b) pf[b] = frag_of<T>(x[b], st);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const FragOf<T> vf = L::template frag_t<kStep>(s.v, d * 16, st * M::KS);
#pragma unroll
          for (int b = 0; b < NQ; ++b) acc[b][d] = M::mma(vf, pf[b], acc[b][d]);
        }
      }
    } else {   // a block at a time, the values' fragments read again: no registers to keep them
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int st = 0; st < kStep / M::KS; ++st) {
          FragOf<T> pf[kParts<T>];
          split_frag_of<T>(x[b], st, pf);
          asm volatile("" ::: "memory");
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const FragOf<T> vf = L::template frag_t<kStep>(s.v, d * 16, st * M::KS);
#pragma unroll
            for (int i = 0; i < kParts<T>; ++i) acc[b][d] = M::mma(vf, pf[i], acc[b][d]);
          }
        }
    }
  }
#pragma unroll
  for (int b = 0; b < NQ; ++b) l[b] = groups_sum(l[b]);
  if (parts != 0) {
    join_waves<1, kWaves, NQ, DB>(smem, m, l, acc);
    if (w != 0) return;
  }
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    if (!in[b]) continue;
    if (parts > 1) {
      const int64_t r = (item * parts + part) * a.rows + int64_t(row[b].i) * a.G + row[b].h;
#pragma unroll
      for (int d = 0; d < DB; ++d) store4(pacc + r * dh, d * 16 + 4 * g, dh, acc[b][d]);
      if (g == 0) pml[r] = make_float2(m[b], l[b]);
      continue;
    }
    const float inv = ok[b] && l[b] != 0.f ? 1.f / l[b] : 0.f;
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const f32x4 v = acc[b][d] * inv;
      store4(o + at, d * 16 + 4 * g, dh, v);
      if (rest != nullptr) store_rest(rest + at, d * 16 + 4 * g, dh, v);
    }
    if (lse != nullptr && g == 0)
      lse[item * a.rows + int64_t(row[b].i) * a.G + row[b].h] = row_sum(m[b], l[b], ok[b]);
  }
}

// The parts of a row joined: one wave a row, a lane two neighbouring values. All
// loads of sixteen parts go out at once: 256 rows of 64 from 16 parts take 4 us,
// where a pass over the maxima first took 11.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_attn_join(Args a, int parts, const float *__restrict__ pacc,
                                                      const float2 *__restrict__ pml, T *__restrict__ o,
                                                      T *__restrict__ rest, float2 *__restrict__ lse) {
  const sgl_attention &p = a.p;
  const int lane = threadIdx.x & 63, dh = p.head_dim;
  const uint32_t x = blockIdx.x * kWaves + wave_index();   // (item, row)
  const uint32_t rows = uint32_t(a.rows), all = uint32_t(p.n * p.heads_kv) * rows;
  if (x >= all) return;
  const uint32_t item = x / rows, r = x - item * rows;
  const int64_t n = item / uint32_t(p.heads_kv), i = r / uint32_t(a.G);
  const int hk = int(item - uint32_t(n) * p.heads_kv), h = int(r - uint32_t(i) * a.G);
  const bool ok = p.q_lens == nullptr || i < p.q_lens[n];
  // a group of parts at a time, its sums rescaled where its maximum is larger
  constexpr int U = 16;
  float top = -INFINITY, sum = 0.f, v0 = 0.f, v1 = 0.f;
  const int d = 2 * lane;
  for (int k0 = 0; k0 < parts; k0 += U) {
    float2 e[U];
    float w0[U], w1[U];
    float most = top;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t row = (int64_t(item) * parts + min(k0 + k, parts - 1)) * rows + r;
      e[k] = pml[row];
      w0[k] = d < dh ? pacc[row * dh + d] : 0.f;
      w1[k] = d + 1 < dh ? pacc[row * dh + d + 1] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) most = fmaxf(most, e[k].x);
    const float at = most == -INFINITY ? 0.f : most, f0 = __builtin_amdgcn_exp2f(top - at);
    sum *= f0;
    v0 *= f0;
    v1 *= f0;
    top = most;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float f = k0 + k < parts ? __builtin_amdgcn_exp2f(e[k].x - at) : 0.f;
      sum += e[k].y * f;
      v0 += f * w0[k];
      v1 += f * w1[k];
    }
  }
  const float inv = ok && sum != 0.f ? 1.f / sum : 0.f;
  const int64_t to = out_row(a, n, hk, i, h);
  v0 *= inv;
  v1 *= inv;
  if (d < dh) o[to + d] = T(v0);
  if (d + 1 < dh) o[to + d + 1] = T(v1);
  if (rest != nullptr) {
    if (d < dh) rest[to + d] = rest_of<T>(v0, T(v0));
    if (d + 1 < dh) rest[to + d + 1] = rest_of<T>(v1, T(v1));
  }
  if (lse != nullptr && lane == 0) lse[x] = row_sum(top, sum, ok);
}

// ------------------------------------------------------------------ host
constexpr int kFewRows = 32;

// Workgroups a (sequence, key head) whose rows are few: 0 (a wave alone) up to
// 4 steps of keys, else as many as bring 1,024 workgroups, of at least 4 steps
// a wave each.
int few_parts(const Args &a) {
  if (a.p.lk <= 4 * kStep) return 0;
  const int64_t items = a.p.n * a.p.heads_kv, most = (a.p.lk + 4 * kStep * kWaves - 1) / (4 * kStep * kWaves);
  return int(std::max<int64_t>(1, std::min<int64_t>({(1024 + items - 1) / items, most, int64_t(256)})));
}
int64_t few_keys(const Args &a, int parts) {
  const int64_t k = (a.p.lk + parts - 1) / parts;
  return (k + kStep * kWaves - 1) / (kStep * kWaves) * (kStep * kWaves);
}
size_t ml_bytes(const Args &a, int parts) {
  return align_up(sizeof(float2) * size_t(a.p.n * a.p.heads_kv) * size_t(parts) * size_t(a.rows));
}

template <typename T, int DP, int NQ, bool SPLIT>
int launch_few(const Args &a, T *o, T *rest, float2 *lse, void *ws, hipStream_t s) {
  const int parts = few_parts(a);
  const int64_t items = a.p.n * a.p.heads_kv, keys = parts > 0 ? few_keys(a, parts) : 0;
  const size_t per = align_bytes(sizeof(FewLds<T, DP, NQ>) + table_bytes(a));
  size_t lds = per * kWaves;
  if (parts > 0)
    lds = std::max(lds, join_bytes(1, kWaves, NQ, DP));
  float2 *ml = static_cast<float2 *>(ws);
  float *acc = reinterpret_cast<float *>(static_cast<char *>(ws) + (parts > 1 ? ml_bytes(a, parts) : 0));
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_few<T, DP, NQ, SPLIT>), lds));
  const int64_t grid = parts == 0 ? (items + kWaves - 1) / kWaves : items * parts;
  launch(&k_attn_few<T, DP, NQ, SPLIT>, dim3(unsigned(grid)), dim3(kBlock), lds, s, a, parts, keys, o, rest, lse, acc, ml);
  if (parts > 1)
    launch(&k_attn_join<T>, dim3(unsigned((items * a.rows + kWaves - 1) / kWaves)), dim3(kBlock), 0, s, a, parts,
           static_cast<const float *>(acc), static_cast<const float2 *>(ml), o, rest, lse);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

template <typename T, int DP, int NQ, bool SHARE, int RW, int KW, bool SPLIT>
int launch_fwd(const Args &a, T *o, T *rest, float2 *lse, hipStream_t s) {
  const int64_t tiles = row_tiles(a, NQ, SHARE, RW);
  const size_t lds = std::max(buffers<FwdLds<T, DP, tile_keys<T>(KW)>>() * sizeof(FwdLds<T, DP, tile_keys<T>(KW)>) + table_bytes(a),
                              join_bytes(RW, KW, NQ, DP));
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_fwd<T, DP, NQ, SHARE, RW, KW, SPLIT>), lds));
  launch(&k_attn_fwd<T, DP, NQ, SHARE, RW, KW, SPLIT>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(RW * KW * kWave),
         lds, s, a, tiles, o, rest, lse);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

}  // namespace

size_t forward_bytes(const Args &a) {
  if (a.rows > kFewRows) return 0;
  const int parts = few_parts(a);
  if (parts <= 1) return 0;
  return ml_bytes(a, parts) +
         sizeof(float) * size_t(a.p.n * a.p.heads_kv) * size_t(parts) * size_t(a.rows) * size_t(a.p.head_dim);
}

int run_forward(const Args &a, void *o, void *rest, float *stats, void *ws, hipStream_t s) {
  float2 *lse = reinterpret_cast<float2 *>(stats);
  return by_instance(a.p, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    T *to = static_cast<T *>(o), *tr = static_cast<T *>(rest);
    auto run = [&](auto split) -> int {
      constexpr bool S = decltype(split)::value;
      if (a.rows <= 16) return launch_few<T, DP, 1, S>(a, to, tr, lse, ws, s);
      if (a.rows <= kFewRows) return launch_few<T, DP, 2, S>(a, to, tr, lse, ws, s);
      if (!many_rows(a)) return launch_fwd<T, DP, 1, false, 1, 4, S>(a, to, tr, lse, s);
      if constexpr (two_blocks<T, DP>()) {
        if (a.G % 2 == 0) return launch_fwd<T, DP, 2, true, 4, 2, S>(a, to, tr, lse, s);
        return launch_fwd<T, DP, 2, false, 4, 2, S>(a, to, tr, lse, s);
      } else {
        return launch_fwd<T, DP, 1, false, 4, 2, S>(a, to, tr, lse, s);
      }
    };
    if constexpr (sizeof(T) == 2)
      if (rest != nullptr) return run(std::true_type{});
    return run(std::false_type{});
  });
}

}  // namespace attn
}  // namespace sgl
