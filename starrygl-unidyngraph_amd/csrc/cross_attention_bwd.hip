// Backward kernels of the cross attention: dq, the bias' gradient and D from
// one walk of each row block over the keys, dk and dv from one walk of each
// key block over the rows. The scores are formed again in both.
#include "cross_attention.h"

namespace sgl {
namespace attn {
namespace {

// ------------------------------------------------------------------ dq, dbias, D
// As the forward with many rows. D = <do, o> takes o with what its rounding
// left (rest), so that the sums that should cancel do; where all keys lie in
// one tile it is the sum of p dp itself, which cancels exactly (a single key
// has no gradient).
template <typename T, int DP, int TK>
struct DqLds {
  T k[TK * Tile<T, DP>::LD], v[TK * Tile<T, DP>::LD];
  PosTile<TK> pos;
};
template <int ROWS>
struct DqSums {
  float red[8], delta[ROWS];
};

// Sets of cells a workgroup needs: where 16 rows hold every head the same
// number of times, row c of every block has the same head (SHARE: of every
// first block, and of every second one), and the waves share their cells.
template <int NQ, bool SHARE, int RW>
__host__ __device__ __forceinline__ int cell_sets(int G) {
  return 16 % (SHARE ? G / 2 : G) == 0 ? (SHARE ? 2 : 1) : RW * NQ;
}

template <typename T, int DP, int NQ, bool SHARE, int RW, int KW>
__global__ __launch_bounds__(RW * KW * 64) void k_attn_dq(Args a, int64_t tiles, const T *__restrict__ o,
                                                          const T *__restrict__ rest, const float *__restrict__ lse,
                                                          const T *__restrict__ go, T *__restrict__ dq,
                                                          float2 *__restrict__ rowstat, float *__restrict__ part) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  constexpr int TK = tile_keys<T>(KW), BLOCK = RW * KW * 64, WAVES = RW * KW;
  using S = DqLds<T, DP, TK>;
  using X = DqSums<WAVES * NQ * 16>;
  constexpr int NB = buffers<S>();
  constexpr int ST = DP / M::KS, DB = DP / 16, KB = TK / 16 / KW;
  constexpr int NP = SHARE ? 1 : NQ;
  extern __shared__ __align__(16) char smem[];
  S *const bufs = reinterpret_cast<S *>(smem);
  X &sx = *reinterpret_cast<X *>(smem + NB * sizeof(S));
  float *table = reinterpret_cast<float *>(smem + NB * sizeof(S) + sizeof(X));
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, cl = lane & 15;
  const int wr = w / KW, k0 = (w % KW) * KB * 16;
  const int sets = cell_sets<NQ, SHARE, RW>(a.G);
  Cell *cells = reinterpret_cast<Cell *>(smem + align_bytes(NB * sizeof(S) + sizeof(X) + table_bytes(a)));
  const TileAt at_ = tile_at(blockIdx.x, uint32_t(tiles), p.heads_kv);
  const uint32_t rt = at_.tile;
  const int hk = at_.hk;
  const int64_t n = at_.n;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  const uint32_t t0 = rt * (SHARE ? RW * 16 : RW * 16 * NQ);
  const uint32_t i0 = row_at<SHARE>(t0, 0, a.G).i;
  const bool any = i0 < q.qlen;
  const bool one_tile = q.klen <= kKeys;
  if (biased) stage_bias(table, a, hk, threadIdx.x, BLOCK);
  if (part != nullptr) clear_cells(cells, sets * a.cols * 16, threadIdx.x, BLOCK);
  RowAt row[NQ];
  bool in[NQ], ok[NQ];
  FragOf<T> qf[NQ][ST], gf[NQ][ST];
  int64_t qpos[NP];
  int qrel[NP];
  float delta[NQ], ls[NQ], gs[NQ], top = 0.f;
  const int64_t base = biased && any ? q.qpos[int64_t(i0) * p.qpos_t] : 0;
  const int64_t stat0 = (n * p.heads_kv + hk) * a.rows;
  bool qnear = true;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    const uint32_t t = SHARE ? t0 + wr * 16 + cl : t0 + (wr * NQ + b) * 16 + cl;
    row[b] = row_at<SHARE>(t, b, a.G);
    in[b] = row[b].i < p.lq;
    ok[b] = row[b].i < q.qlen;
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
    float most = 0.f;
    delta[b] = 0.f;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      const int d = st * M::KS + g * M::E;
      qf[b][st] = load_row<T>(q.q + int64_t(row[b].i) * p.q_t + row[b].h * p.q_h, ok[b], d, dh);
      gf[b][st] = load_row<T>(go + at, ok[b], d, dh);
#pragma unroll
      for (int e = 0; e < M::E; ++e) most = fmaxf(most, fabsf(float(gf[b][st][e])));
      if (!one_tile) {
        const FragOf<T> of = load_row<T>(o + at, ok[b], d, dh);
        FragOf<T> rf = zero_frag<T>();
        if (rest != nullptr) rf = load_row<T>(rest + at, ok[b], d, dh);
#pragma unroll
        for (int e = 0; e < M::E; ++e) delta[b] += float(gf[b][st][e]) * (float(of[e]) + float(rf[e]));
      }
    }
    delta[b] = groups_sum(delta[b]);
    most = groups_max(most);
    top = fmaxf(top, most);
    gs[b] = grad_scale<T>(most);
    const int64_t r = stat0 + int64_t(row[b].i) * a.G + row[b].h;
    ls[b] = ok[b] ? lse[r] : INFINITY;
    if (g == 0 && in[b] && w % KW == 0) rowstat[r] = make_float2(delta[b], most);
    if (b < NP) {
      qpos[b] = biased && ok[b] ? q.qpos[int64_t(row[b].i) * p.qpos_t] : base;
      qnear = qnear && is_near(qpos[b] - base);
      qrel[b] = int(qpos[b] - base);
    }
  }
  qnear = __all(qnear);
  const float c = p.scale * kLog2e;
  float up = 1.f, seen = 0.f;   // the cells' power of two, for the whole workgroup
  if (part != nullptr) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
    if (lane == 0) sx.red[w] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = fmaxf(top, sx.red[i]);
    up = unit_scale(top);
  }
  f32x4 acc[NQ][DB];
#pragma unroll
  for (int b = 0; b < NQ; ++b)
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  KeyTile<T, DP, TK, BLOCK> tile;
  if (any && q.klen > 0) tile.load(q, a, 0, base, qnear);
  int buf = 0;
  for (int64_t j0 = 0; any && j0 < q.klen; j0 += TK) {
    S &s = bufs[buf];
    if constexpr (NB == 1) __syncthreads();
    else buf ^= 1;
    tile.store(s.k, s.v, s.pos, a, base);
    const uint32_t on = tile.live_of(k0, KB * 16);
    const bool near_now = tile.near_;
    __syncthreads();
    if (j0 + TK < q.klen) tile.load(q, a, j0 + TK, base, qnear);
    float x[NQ][KB][4], y[NQ][KB][4];   // p and dp, then ds
    int col[NP][KB][4];
    if (biased) {
#pragma unroll
      for (int b = 0; b < NP; ++b) columns(col[b], s.pos, k0 + 4 * g, qrel[b], qpos[b], near_now, 1, bk);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      FragOf<T> kf[ST], vf[ST];
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        kf[st] = L::frag(s.k, k0 + kb * 16, st * M::KS);
        vf[st] = L::frag(s.v, k0 + kb * 16, st * M::KS);
      }
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          sc = M::mma(kf[st], qf[b][st], sc);
          dp = M::mma(vf[st], gf[b][st], dp);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = sc[v];
          y[b][kb][v] = dp[v];
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      scale_scores(x[b], c, -ls[b], table + row[b].h * table_ld(a), col[b < NP ? b : 0], biased);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) x[b][kb][v] = __builtin_amdgcn_exp2f(x[b][kb][v]);
    }
    if (on != full_mask(KB * 16)) {   // uniform
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const bool dead = !((on >> (kb * 16 + 4 * g + v)) & 1);
#pragma unroll
          for (int b = 0; b < NQ; ++b) x[b][kb][v] = dead ? 0.f : x[b][kb][v];
        }
    }
    if (one_tile) {   // uniform over the workgroup; the sums of a row's KW waves in one order
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        float t = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) t += x[b][kb][v] * y[b][kb][v];
        t = groups_sum(t);
        if (g == 0) sx.delta[(w * NQ + b) * 16 + cl] = t;
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        delta[b] = 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) delta[b] += sx.delta[((wr * KW + i) * NQ + b) * 16 + cl];
        if (g == 0 && in[b] && w % KW == 0) rowstat[stat0 + int64_t(row[b].i) * a.G + row[b].h].x = delta[b];
      }
    }
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) y[b][kb][v] = x[b][kb][v] * (y[b][kb][v] - delta[b]);
    if (part != nullptr) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        const int set = sets == RW * NQ ? wr * NQ + b : SHARE ? b : 0;
        add_cells(cells + set * a.cols * 16, col[b < NP ? b : 0], y[b], up, seen);
      }
    }
    if constexpr (std::is_same_v<T, fp16_t>) {
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) y[b][kb][v] *= gs[b];
    }
#pragma unroll
    for (int st = 0; st < KB * 16 / M::KS; ++st) {
      FragOf<T> df[NQ];
#pragma unroll
      for (int b = 0; b < NQ; ++b) df[b] = frag_of<T>(y[b], st);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const FragOf<T> kt = L::template frag_t<TK>(s.k, d * 16, k0 + st * M::KS);
#pragma unroll
        for (int b = 0; b < NQ; ++b) acc[b][d] = M::mma(kt, df[b], acc[b][d]);
      }
    }
  }
  if (part != nullptr) {
    // cell (set, column, c) belongs to the head of its blocks' row c: a thread
    // sums a (head, column) over them
    const bool held = __all(cells_hold(seen));
    __syncthreads();
    if (lane == 0) sx.red[w] = held ? 0.f : NAN;
    __syncthreads();
    float bad = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) bad += sx.red[i];
    const bool own = sets == RW * NQ;
    float *out = part + ((n * tiles + rt) * p.heads_kv + hk) * a.G * a.cols;
    for (int x = threadIdx.x; x < a.G * a.cols; x += BLOCK) {
      const int h = x / a.cols, cidx = x - h * a.cols;
      long long t = 0;
      for (int set = 0; set < sets; ++set) {
        const int ww = own ? set / NQ : 0, b = own ? set % NQ : SHARE ? set : 0;
        const int h0 = row_at<SHARE>(SHARE ? t0 + ww * 16 : t0 + (own ? set : 0) * 16, b, a.G).h;   // of c = 0
        for (int i = 0; i < 16; ++i) {
          const int e = (i + cidx) & 15;   // (rotated: neighbouring columns in different banks)
          if ((h0 + (SHARE ? 2 : 1) * e) % a.G == h) t += static_cast<long long>(cells[(set * a.cols + cidx) * 16 + e]);
        }
      }
      out[x] = float(double(t) * (1.0 / double(1ll << kCellBits)) / double(up)) + bad;
    }
  }
  if constexpr (KW > 1) {
    float *pr = reinterpret_cast<float *>(smem);
    __syncthreads();
    put_join<KW, NQ, DB>(pr, acc);
    __syncthreads();
    take_join<KW, NQ, DB>(pr, acc);
    if (w % KW != 0) return;
  }
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    if (!in[b]) continue;
    const float f = p.scale / gs[b];
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
    for (int d = 0; d < DB; ++d) store4(dq + at, d * 16 + 4 * g, dh, acc[b][d] * f);
  }
}

// ------------------------------------------------------------------ dk, dv
// A workgroup takes CW blocks of 16 keys (one a lane of 16) and walks the rows
// of all G heads; RS waves share a key block, each with 32 rows of every tile,
// and are joined at the end. With an even G the 32 are two heads of 16 queries
// (SHARE). The next tile's rows are in flight while one is worked on.
constexpr int kRows = 32;

template <typename T, int DP, int TR>
struct DkvLds {
  T q[TR * Tile<T, DP>::LD], go[TR * Tile<T, DP>::LD];
  PosTile<TR> pos;
  float lse[TR], delta[TR];
  int head[TR];
  float red[8];
};

template <typename T, int DP, bool SHARE, int CW, int RS>
__global__ __launch_bounds__(CW * RS * 64) void k_attn_dkv(Args a, int64_t tiles, const float *__restrict__ lse,
                                                     const T *__restrict__ go, const float2 *__restrict__ rowstat,
                                                     T *__restrict__ dk, T *__restrict__ dv) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  constexpr int TR = kRows * RS, BLOCK = CW * RS * 64, WAVES = CW * RS;
  using S = DkvLds<T, DP, TR>;
  constexpr int ST = DP / M::KS, DB = DP / 16, RB = kRows / 16, NP = SHARE ? 1 : RB;
  constexpr bool kHalf = std::is_same_v<T, fp16_t>;
  extern __shared__ __align__(16) char smem[];
  S &s = *reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + sizeof(s));
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  const TileAt at_ = tile_at(blockIdx.x, uint32_t(tiles), p.heads_kv);
  const int64_t kt = at_.tile;
  const int hk = at_.hk;
  const int64_t n = at_.n;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const int64_t j = (kt * CW + w / RS) * 16 + (lane & 15);   // this lane's key
  const int x0 = (w % RS) * kRows;                           // this wave's rows of a tile
  const bool on = key_live(q, p, j);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  if (biased) stage_bias(table, a, hk, threadIdx.x, BLOCK);
  const int64_t stat0 = (n * p.heads_kv + hk) * a.rows;
  // steps of 32 rows (blocks of 16 queries x head pairs, or 32 rows in order), RS of them a tile
  const int pairs = a.G >> 1;
  const bool any = kt * CW * 16 < q.klen;
  const uint32_t qlen = uint32_t(q.qlen);
  const uint32_t steps = !any ? 0 : SHARE ? (qlen + 15) / 16 * uint32_t(pairs) : (qlen * a.G + kRows - 1) / kRows;
  float gs = 1.f;
  if constexpr (kHalf) {
    float most = 0.f;
    if (any)
      for (uint32_t r = threadIdx.x; r < qlen * a.G; r += BLOCK) most = fmaxf(most, rowstat[stat0 + r].y);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, kWave));
    if (lane == 0) s.red[w] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) most = fmaxf(most, s.red[i]);
    gs = grad_scale<T>(most);
  }
  FragOf<T> kf[ST], vf[ST];
#pragma unroll
  for (int st = 0; st < ST; ++st) {
    const int d = st * M::KS + g * M::E;
    kf[st] = load_row<T>(q.k + j * p.k_t, on, d, dh);
    vf[st] = load_row<T>(q.v + j * p.v_t, on, d, dh);
  }
  const int64_t base = biased && steps > 0 ? q.qpos[0] : 0;
  const int64_t kp = biased && on ? q.kpos[j * p.kpos_t] : base;
  const int krel = int(kp - base);
  const bool knear = __all(is_near(kp - base));
  const float c = p.scale * kLog2e;
  const float dsf = gs / kProbUp<T>;
  f32x4 acc[2][DB];   // dk, dv
#pragma unroll
  for (int b = 0; b < DB; ++b) acc[0][b] = acc[1][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int PER = (TR * L::UPR + BLOCK - 1) / BLOCK;
  FragOf<T> qr[PER], gr[PER];
  constexpr int RL = (TR + 63) / 64;   // rows a lane looks at (every wave sees the whole tile)
  int64_t qp[RL];
  float ls[RL], de[RL];
  int he[RL];
  bool near_ = true;
  auto row_of = [&](uint32_t step, int i) {   // row i of a step's 32
    if constexpr (SHARE) {
      const uint32_t ib = pairs == 1 ? step : step / uint32_t(pairs);
      return RowAt{ib * 16 + (i & 15), int(step - ib * pairs) * 2 + (i >> 4)};
    } else {
      return row_at<false>(step * kRows + i, 0, a.G);
    }
  };
  auto load_step = [&](uint32_t step) {
    near_ = knear;
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      const int rr = i * 64 + lane;
      const RowAt r = row_of(step + rr / kRows, rr % kRows);
      const bool ok = rr < TR && r.i < qlen;
      ls[i] = ok ? lse[stat0 + int64_t(r.i) * a.G + r.h] : INFINITY;
      de[i] = ok ? rowstat[stat0 + int64_t(r.i) * a.G + r.h].x : 0.f;
      he[i] = r.h;
      qp[i] = base;
      if (biased) {
        if (ok) qp[i] = q.qpos[int64_t(r.i) * p.qpos_t];
        near_ = near_ && __all(is_near(qp[i] - base));
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * BLOCK, rr = u / L::UPR, d = (u % L::UPR) * M::E;
      // (a wave's units lie in one step of 32 rows: its division is a scalar one)
      const RowAt t = row_of(step + uint32_t(__builtin_amdgcn_readfirstlane(rr / kRows)), rr % kRows);
      const bool okr = rr < TR && t.i < qlen;
      qr[i] = load_raw<T>(q.q + int64_t(t.i) * p.q_t + t.h * p.q_h, okr, d, dh);
      gr[i] = load_raw<T>(go + out_row(a, n, hk, t.i, t.h), okr, d, dh);
    }
  };
  if (steps > 0) load_step(0);
  for (uint32_t step = 0; step < steps; step += RS) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * BLOCK, rr = u / L::UPR, d = (u % L::UPR) * M::E;
      if (rr < TR) {
        *reinterpret_cast<FragOf<T> *>(s.q + rr * L::LD + d) = fix<T>(qr[i], d, dh);
        *reinterpret_cast<FragOf<T> *>(s.go + rr * L::LD + d) = fix<T>(gr[i], d, dh);
      }
    }
    if (w == 0) {
#pragma unroll
      for (int i = 0; i < RL; ++i) {
        const int rr = i * 64 + lane;
        if (rr < TR) {
          s.lse[rr] = ls[i];
          s.delta[rr] = de[i];
          s.head[rr] = he[i] * table_ld(a);
          s.pos.pos[rr] = qp[i];
          s.pos.rel[rr] = int(qp[i] - base);
        }
      }
    }
    const bool near_now = near_;
    __syncthreads();
    if (step + RS < steps) load_step(step + RS);
    float x[RB][4], y[RB][4];   // p and ds, rows x this lane's key
    int col[RB][4];
    if (biased) {
      int own[NP][4];
      columns(own, s.pos, x0 + 4 * g, krel, kp, near_now, -1, bk);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int v = 0; v < 4; ++v) col[rb][v] = own[rb < NP ? rb : 0][v] + s.head[x0 + rb * 16 + 4 * g + v];
    }
    float lsv[RB][4], dev[RB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      __builtin_memcpy(lsv[rb], s.lse + x0 + rb * 16 + 4 * g, sizeof(lsv[rb]));
      __builtin_memcpy(dev[rb], s.delta + x0 + rb * 16 + 4 * g, sizeof(dev[rb]));
      f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        sc = M::mma(L::frag(s.q, x0 + rb * 16, st * M::KS), kf[st], sc);
        dp = M::mma(L::frag(s.go, x0 + rb * 16, st * M::KS), vf[st], dp);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        x[rb][v] = sc[v];
        y[rb][v] = dp[v];
      }
    }
    scale_scores(x, c, 0.f, table, col, biased);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float pr = on ? __builtin_amdgcn_exp2f(x[rb][v] - lsv[rb][v]) * kProbUp<T> : 0.f;
        x[rb][v] = pr;
        y[rb][v] = pr * ((y[rb][v] - dev[rb][v]) * dsf);
      }
#pragma unroll
    for (int st = 0; st < kRows / M::KS; ++st) {
      const FragOf<T> pf = frag_of<T>(x, st), df = frag_of<T>(y, st);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        acc[0][b] = M::mma(L::template frag_t<kRows>(s.q, b * 16, x0 + st * M::KS), df, acc[0][b]);
        acc[1][b] = M::mma(L::template frag_t<kRows>(s.go, b * 16, x0 + st * M::KS), pf, acc[1][b]);
      }
    }
  }
  if constexpr (RS > 1) {
    float *pr = reinterpret_cast<float *>(smem);
    __syncthreads();
    put_join<RS, 2, DB>(pr, acc);
    __syncthreads();
    take_join<RS, 2, DB>(pr, acc);
    if (w % RS != 0) return;
  }
  if (j >= p.lk) return;
  const int64_t row = ((n * p.lk + j) * p.heads_kv + hk) * dh;
  const float fk = p.scale / gs, fv = 1.f / kProbUp<T>;
#pragma unroll
  for (int b = 0; b < DB; ++b) {
    store4(dk + row, b * 16 + 4 * g, dh, acc[0][b] * fk);
    store4(dv + row, b * 16 + 4 * g, dh, acc[1][b] * fv);
  }
}

// ------------------------------------------------------------------ host
size_t stat_bytes(const Args &a) { return align_up(sizeof(float2) * size_t(a.p.n * a.p.heads_kv * a.rows)); }
int64_t dq_tiles(const Args &a) {
  return many_rows(a) ? row_tiles(a, 2, a.G % 2 == 0, 4) : row_tiles(a, 1, false, 1);
}

template <typename T, int DP, int NQ, bool SHARE, int RW, int KW>
int launch_dq(const Args &a, int64_t tiles, const void *o, const void *rest, const float *lse, const void *go, void *dq,
              float2 *stat, float *part, hipStream_t s) {
  const size_t lds = std::max(
      align_bytes(buffers<DqLds<T, DP, tile_keys<T>(KW)>>() * sizeof(DqLds<T, DP, tile_keys<T>(KW)>) +
                  sizeof(DqSums<RW * KW * NQ * 16>) + table_bytes(a)) +
          (part != nullptr ? sizeof(Cell) * cell_sets<NQ, SHARE, RW>(a.G) * 16 * size_t(a.cols) : 0),
      join_bytes(RW, KW, NQ, DP));
  SGL_REQUIRE(lds <= 160 * 1024, "cross_attention_backward: %zu bytes of LDS", lds);
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dq<T, DP, NQ, SHARE, RW, KW>), lds));
  launch(&k_attn_dq<T, DP, NQ, SHARE, RW, KW>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(RW * KW * kWave), lds,
         s, a, tiles, static_cast<const T *>(o), static_cast<const T *>(rest), lse, static_cast<const T *>(go),
         static_cast<T *>(dq), stat, part);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

template <typename T, int DP, bool SHARE, int CW, int RS>
int launch_dkv(const Args &a, const float *lse, const void *go, const float2 *stat, void *dk, void *dv,
               hipStream_t s) {
  const int64_t tiles = (a.p.lk + 16 * CW - 1) / (16 * CW);
  const size_t lds = std::max(sizeof(DkvLds<T, DP, kRows * RS>) + table_bytes(a),
                              join_bytes(CW, RS, 2, DP));
  SGL_REQUIRE(lds <= 160 * 1024, "cross_attention_backward: %zu bytes of LDS", lds);
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dkv<T, DP, SHARE, CW, RS>), lds));
  launch(&k_attn_dkv<T, DP, SHARE, CW, RS>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(CW * RS * kWave), lds, s,
         a, tiles, lse, static_cast<const T *>(go), stat, static_cast<T *>(dk), static_cast<T *>(dv));
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

}  // namespace

size_t backward_bytes(const Args &a) {
  return stat_bytes(a) + sizeof(float) * size_t(a.p.n * dq_tiles(a)) * a.p.heads_q * a.cols;
}

int run_backward(const Args &a, const void *o, const void *rest, const float *lse, const void *go, void *dq, void *dk,
                 void *dv, float *dbias, void *ws, hipStream_t s) {
  float2 *stat = static_cast<float2 *>(ws);
  float *part = dbias != nullptr ? reinterpret_cast<float *>(static_cast<char *>(ws) + stat_bytes(a)) : nullptr;
  const int64_t tiles = dq_tiles(a);
  return by_instance(a.p, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (tiles > 0) {
      int rc;
      if (!many_rows(a)) rc = launch_dq<T, DP, 1, false, 1, 4>(a, tiles, o, rest, lse, go, dq, stat, part, s);
      else if (a.G % 2 == 0) rc = launch_dq<T, DP, 2, true, 4, 2>(a, tiles, o, rest, lse, go, dq, stat, part, s);
      else rc = launch_dq<T, DP, 2, false, 4, 2>(a, tiles, o, rest, lse, go, dq, stat, part, s);
      if (rc != SGL_OK) return rc;
    }
    if (dbias != nullptr) sum_rows(part, a.p.n * tiles, a.p.heads_q * a.cols, dbias, s);
    if (a.p.lk == 0) {
      SGL_CHECK_LAUNCH();
      return int(SGL_OK);
    }
    // 64 keys a workgroup where that fills the GPU, else 16, its four waves along the rows
    const bool wide = a.p.n * a.p.heads_kv * ((a.p.lk + 63) / 64) >= 192;
    if (a.G % 2 == 0)
      return wide ? launch_dkv<T, DP, true, 4, 2>(a, lse, go, stat, dk, dv, s)
                  : launch_dkv<T, DP, true, 1, 4>(a, lse, go, stat, dk, dv, s);
    return wide ? launch_dkv<T, DP, false, 4, 2>(a, lse, go, stat, dk, dv, s)
                : launch_dkv<T, DP, false, 1, 4>(a, lse, go, stat, dk, dv, s);
  });
}

}  // namespace attn
}  // namespace sgl
