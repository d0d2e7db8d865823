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
template <typename T, int DP>
struct DqLds {
  T k[kKeys * Tile<T, DP>::LD], v[kKeys * Tile<T, DP>::LD];
  PosTile<kKeys> pos;
  float red[kWaves];
};

// Sets of cells a workgroup needs: where 16 rows hold every head the same
// number of times, row c of every block has the same head (SHARE: of every
// first block, and of every second one), and the waves share their cells.
template <int NQ, bool SHARE>
__host__ __device__ __forceinline__ int cell_sets(int G) {
  return 16 % (SHARE ? G / 2 : G) == 0 ? (SHARE ? 2 : 1) : kWaves * NQ;
}

template <typename T, int DP, int NQ, bool SHARE>
__global__ __launch_bounds__(kBlock) void k_attn_dq(Args a, int64_t tiles, const T *__restrict__ o,
                                                    const T *__restrict__ rest, const float *__restrict__ lse,
                                                    const T *__restrict__ go, T *__restrict__ dq,
                                                    float2 *__restrict__ rowstat, float *__restrict__ part) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using S = DqLds<T, DP>;
  constexpr int ST = DP / M::KS, DB = DP / 16, KB = kKeys / 16;
  constexpr int NP = SHARE ? 1 : NQ;
  extern __shared__ __align__(16) char smem[];
  S &s = *reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + sizeof(s));
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, cl = lane & 15;
  const int sets = cell_sets<NQ, SHARE>(a.G);
  Cell *cells = reinterpret_cast<Cell *>(smem + align_bytes(sizeof(s) + sizeof(float) * a.G * a.cols));
  int64_t id = blockIdx.x;
  const int64_t rt = id % tiles;
  id /= tiles;
  const int hk = int(id % p.heads_kv);
  const int64_t n = id / p.heads_kv;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  const int64_t t0 = rt * (SHARE ? 64 : 64 * NQ);
  const int64_t i0 = row_at<SHARE>(t0, 0, a.G).i;
  const bool any = i0 < q.qlen;
  const bool one_tile = q.klen <= kKeys;
  if (biased) stage_bias(table, a, hk, threadIdx.x, kBlock);
  if (part != nullptr) clear_cells(cells, sets * a.cols * 16, threadIdx.x, kBlock);
  RowAt row[NQ];
  bool in[NQ], ok[NQ];
  FragOf<T> qf[NQ][ST], gf[NQ][ST];
  int64_t qpos[NP];
  int qrel[NP];
  float delta[NQ], ls[NQ], gs[NQ], top = 0.f;
  const int64_t base = biased && any ? q.qpos[i0 * p.qpos_t] : 0;
  const int64_t stat0 = (n * p.heads_kv + hk) * a.rows;
  bool qnear = true;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    const int64_t t = SHARE ? t0 + w * 16 + cl : t0 + (w * NQ + b) * 16 + cl;
    row[b] = row_at<SHARE>(t, b, a.G);
    in[b] = row[b].i < p.lq;
    ok[b] = row[b].i < q.qlen;
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
    float most = 0.f;
    delta[b] = 0.f;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      const int d = st * M::KS + g * M::E;
      qf[b][st] = load_row<T>(q.q + row[b].i * p.q_t + row[b].h * p.q_h, ok[b], d, dh);
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
    const int64_t r = stat0 + row[b].i * a.G + row[b].h;
    ls[b] = ok[b] ? lse[r] : INFINITY;
    if (g == 0 && in[b]) rowstat[r] = make_float2(delta[b], most);
    if (b < NP) {
      qpos[b] = biased && ok[b] ? q.qpos[row[b].i * p.qpos_t] : base;
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
    if (lane == 0) s.red[w] = top;
    __syncthreads();
    up = unit_scale(fmaxf(fmaxf(s.red[0], s.red[1]), fmaxf(s.red[2], s.red[3])));
  }
  f32x4 acc[NQ][DB];
#pragma unroll
  for (int b = 0; b < NQ; ++b)
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int PER = kKeys * L::UPR / kBlock;
  FragOf<T> kr[PER], vr[PER];
  uint64_t live = 0;
  bool near_ = true;
  int64_t kp = 0;
  auto load_tile = [&](int64_t j0) {
    const bool on = key_live(q, p, j0 + lane);
    live = __ballot(on);
    if (biased) {
      kp = on ? q.kpos[(j0 + lane) * p.kpos_t] : base;
      near_ = qnear && __all(is_near(kp - base));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * kBlock, r = u / L::UPR, d = (u % L::UPR) * M::E;
      const bool on_r = (live >> r) & 1;
      kr[i] = load_raw<T>(q.k + (j0 + r) * p.k_t, on_r, d, dh);
      vr[i] = load_raw<T>(q.v + (j0 + r) * p.v_t, on_r, d, dh);
    }
  };
  if (any && q.klen > 0) load_tile(0);
  for (int64_t j0 = 0; any && j0 < q.klen; j0 += kKeys) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * kBlock, r = u / L::UPR, d = (u % L::UPR) * M::E;
      *reinterpret_cast<FragOf<T> *>(s.k + r * L::LD + d) = fix<T>(kr[i], d, dh);
      *reinterpret_cast<FragOf<T> *>(s.v + r * L::LD + d) = fix<T>(vr[i], d, dh);
    }
    if (biased && w == 0) {
      s.pos.pos[lane] = kp;
      s.pos.rel[lane] = int(kp - base);
    }
    const uint64_t on = live;
    const bool near_now = near_;
    __syncthreads();
    if (j0 + kKeys < q.klen) load_tile(j0 + kKeys);
    float x[NQ][KB][4], y[NQ][KB][4];   // p and dp, then ds
    int col[NP][KB][4];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      FragOf<T> kf[ST], vf[ST];
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        kf[st] = L::frag(s.k, kb * 16, st * M::KS);
        vf[st] = L::frag(s.v, kb * 16, st * M::KS);
      }
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          sc = M::mma(kf[st], qf[b][st], sc);
          dp = M::mma(vf[st], gf[b][st], dp);
        }
        if (biased && b < NP)
          columns4(col[b < NP ? b : 0][kb], s.pos, kb * 16 + 4 * g, qrel[b < NP ? b : 0], qpos[b < NP ? b : 0],
                   near_now, 1, bk);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float t = sc[v] * c - ls[b];
          if (biased) t += table[row[b].h * a.cols + col[b < NP ? b : 0][kb][v]];
          x[b][kb][v] = __builtin_amdgcn_exp2f(t);
          y[b][kb][v] = dp[v];
        }
      }
    }
    if (on != ~0ull) {   // uniform
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const bool dead = !((on >> (kb * 16 + 4 * g + v)) & 1);
#pragma unroll
          for (int b = 0; b < NQ; ++b) x[b][kb][v] = dead ? 0.f : x[b][kb][v];
        }
    }
    if (one_tile) {   // uniform
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        float t = 0.f, u = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            t += x[b][kb][v] * y[b][kb][v];
            u = fmaxf(u, fabsf(y[b][kb][v]));
          }
        delta[b] = groups_sum(t);
        if (g == 0 && in[b]) rowstat[stat0 + row[b].i * a.G + row[b].h].x = delta[b];
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
        const int set = sets == kWaves * NQ ? w * NQ + b : SHARE ? b : 0;
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
    for (int st = 0; st < kKeys / M::KS; ++st) {
      FragOf<T> df[NQ];
#pragma unroll
      for (int b = 0; b < NQ; ++b) df[b] = frag_of<T>(y[b], st);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const FragOf<T> kt = L::template frag_t<kKeys>(s.k, d * 16, st * M::KS);
#pragma unroll
        for (int b = 0; b < NQ; ++b) acc[b][d] = M::mma(kt, df[b], acc[b][d]);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    if (!in[b]) continue;
    const float f = p.scale / gs[b];
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
    for (int d = 0; d < DB; ++d) store4(dq + at, d * 16 + 4 * g, dh, acc[b][d] * f);
  }
  if (part != nullptr) {
    // cell (set, column, c) belongs to the head of its blocks' row c: a thread
    // sums a (head, column) over them
    const bool held = __all(cells_hold(seen));
    __syncthreads();
    if (lane == 0) s.red[w] = held ? 0.f : NAN;
    __syncthreads();
    const float bad = s.red[0] + s.red[1] + s.red[2] + s.red[3];
    float *out = part + ((n * tiles + rt) * p.heads_kv + hk) * a.G * a.cols;
    for (int x = threadIdx.x; x < a.G * a.cols; x += kBlock) {
      const int h = x / a.cols, cidx = x - h * a.cols;
      long long t = 0;
      for (int set = 0; set < sets; ++set) {
        const bool own = sets == kWaves * NQ;
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
}

// ------------------------------------------------------------------ dk, dv
// A workgroup takes 64 keys (16 a wave, one a lane of 16) and walks the rows
// of all G heads, 32 at a time, the next ones in flight; with an even G the 32
// are two heads of 16 queries (SHARE).
constexpr int kRows = 32;

template <typename T, int DP>
struct DkvLds {
  T q[kRows * Tile<T, DP>::LD], go[kRows * Tile<T, DP>::LD];
  PosTile<kRows> pos;
  float lse[kRows], delta[kRows];
  int head[kRows];
  float red[kWaves];
};

template <typename T, int DP, bool SHARE>
__global__ __launch_bounds__(kBlock) void k_attn_dkv(Args a, int64_t tiles, const float *__restrict__ lse,
                                                     const T *__restrict__ go, const float2 *__restrict__ rowstat,
                                                     T *__restrict__ dk, T *__restrict__ dv) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using S = DkvLds<T, DP>;
  constexpr int ST = DP / M::KS, DB = DP / 16, RB = kRows / 16, NP = SHARE ? 1 : RB;
  constexpr bool kHalf = std::is_same_v<T, fp16_t>;
  extern __shared__ __align__(16) char smem[];
  S &s = *reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + sizeof(s));
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  int64_t id = blockIdx.x;
  const int64_t kt = id % tiles;
  id /= tiles;
  const int hk = int(id % p.heads_kv);
  const int64_t n = id / p.heads_kv;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const int64_t j = kt * kKeys + w * 16 + (lane & 15);   // this lane's key
  const bool on = key_live(q, p, j);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  if (biased) stage_bias(table, a, hk, threadIdx.x, kBlock);
  const int64_t stat0 = (n * p.heads_kv + hk) * a.rows;
  // steps of 32 rows: blocks of 16 queries x head pairs, or 32 rows in order
  const int pairs = a.G >> 1;
  const bool any = kt * kKeys < q.klen;
  const int64_t steps = !any ? 0 : SHARE ? (q.qlen + 15) / 16 * pairs : (q.qlen * a.G + kRows - 1) / kRows;
  float gs = 1.f;
  if constexpr (kHalf) {
    float most = 0.f;
    if (any)
      for (int64_t r = threadIdx.x; r < q.qlen * a.G; r += kBlock) most = fmaxf(most, rowstat[stat0 + r].y);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, kWave));
    if (lane == 0) s.red[w] = most;
    __syncthreads();
    gs = grad_scale<T>(fmaxf(fmaxf(s.red[0], s.red[1]), fmaxf(s.red[2], s.red[3])));
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
  f32x4 ak[DB], av[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) ak[b] = av[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int PER = (kRows * L::UPR + kBlock - 1) / kBlock;
  FragOf<T> qr[PER], gr[PER];
  int64_t qp = 0;
  float ls = INFINITY, de = 0.f;
  int he = 0;
  bool near_ = true;
  auto row_of = [&](int64_t step, int i) {   // row i of a step's 32
    if constexpr (SHARE) {
      const int64_t ib = pairs == 1 ? step : step / pairs;
      return RowAt{ib * 16 + (i & 15), int(step - ib * pairs) * 2 + (i >> 4)};
    } else {
      return row_at<false>(step * kRows + i, 0, a.G);
    }
  };
  auto load_step = [&](int64_t step) {
    const RowAt r = row_of(step, lane & (kRows - 1));   // every wave: a row a lane (twice)
    const bool ok = r.i < q.qlen;
    ls = ok ? lse[stat0 + r.i * a.G + r.h] : INFINITY;
    de = ok ? rowstat[stat0 + r.i * a.G + r.h].x : 0.f;
    he = r.h;
    if (biased) {
      qp = ok ? q.qpos[r.i * p.qpos_t] : base;
      near_ = knear && __all(is_near(qp - base));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * kBlock, rr = u / L::UPR, d = (u % L::UPR) * M::E;
      const RowAt t = row_of(step, rr);
      const bool okr = rr < kRows && t.i < q.qlen;
      qr[i] = load_raw<T>(q.q + t.i * p.q_t + t.h * p.q_h, okr, d, dh);
      gr[i] = load_raw<T>(go + out_row(a, n, hk, t.i, t.h), okr, d, dh);
    }
  };
  if (steps > 0) load_step(0);
  for (int64_t step = 0; step < steps; ++step) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * kBlock, rr = u / L::UPR, d = (u % L::UPR) * M::E;
      if (rr < kRows) {
        *reinterpret_cast<FragOf<T> *>(s.q + rr * L::LD + d) = fix<T>(qr[i], d, dh);
        *reinterpret_cast<FragOf<T> *>(s.go + rr * L::LD + d) = fix<T>(gr[i], d, dh);
      }
    }
    if (threadIdx.x < kRows) {
      s.lse[lane] = ls;
      s.delta[lane] = de;
      s.head[lane] = he * a.cols;
      s.pos.pos[lane] = qp;
      s.pos.rel[lane] = int(qp - base);
    }
    const bool near_now = near_;
    __syncthreads();
    if (step + 1 < steps) load_step(step + 1);
    float x[RB][4], y[RB][4];   // p and ds, rows x this lane's key
    int col[NP][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        sc = M::mma(L::frag(s.q, rb * 16, st * M::KS), kf[st], sc);
        dp = M::mma(L::frag(s.go, rb * 16, st * M::KS), vf[st], dp);
      }
      const int at = rb * 16 + 4 * g;
      if (biased && rb < NP) columns4(col[rb < NP ? rb : 0], s.pos, at, krel, kp, near_now, -1, bk);
      float lsv[4], dev[4];
      int hev[4];
      __builtin_memcpy(lsv, s.lse + at, sizeof(lsv));
      __builtin_memcpy(dev, s.delta + at, sizeof(dev));
      __builtin_memcpy(hev, s.head + at, sizeof(hev));
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float t = sc[v] * c - lsv[v];
        if (biased) t += table[hev[v] + col[rb < NP ? rb : 0][v]];
        const float pr = on ? __builtin_amdgcn_exp2f(t) * kProbUp<T> : 0.f;
        x[rb][v] = pr;
        y[rb][v] = pr * ((dp[v] - dev[v]) * dsf);
      }
    }
#pragma unroll
    for (int st = 0; st < kRows / M::KS; ++st) {
      const FragOf<T> pf = frag_of<T>(x, st), df = frag_of<T>(y, st);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        av[b] = M::mma(L::template frag_t<kRows>(s.go, b * 16, st * M::KS), pf, av[b]);
        ak[b] = M::mma(L::template frag_t<kRows>(s.q, b * 16, st * M::KS), df, ak[b]);
      }
    }
  }
  if (j >= p.lk) return;
  const int64_t row = ((n * p.lk + j) * p.heads_kv + hk) * dh;
  const float fk = p.scale / gs, fv = 1.f / kProbUp<T>;
#pragma unroll
  for (int b = 0; b < DB; ++b) {
    store4(dk + row, b * 16 + 4 * g, dh, ak[b] * fk);
    store4(dv + row, b * 16 + 4 * g, dh, av[b] * fv);
  }
}

// ------------------------------------------------------------------ host
// The form of dq: two blocks a wave where that fills the GPU (as the forward).
struct DqForm {
  int nq;
  bool share;
  int64_t tiles;
};
DqForm dq_form(const Args &a) {
  DqForm f;
  f.nq = a.p.n * a.p.heads_kv * ((a.rows + 127) / 128) < 256 ? 1 : 2;
  f.share = f.nq == 2 && a.G % 2 == 0;
  const int64_t count = f.share ? a.rows / 2 : a.rows, per = f.share ? 64 : 64 * f.nq;
  f.tiles = (count + per - 1) / per;
  return f;
}
size_t stat_bytes(const Args &a) { return align_up(sizeof(float2) * size_t(a.p.n * a.p.heads_kv * a.rows)); }

template <typename T, int DP, int NQ, bool SHARE>
int launch_dq(const Args &a, int64_t tiles, const void *o, const void *rest, const float *lse, const void *go, void *dq,
              float2 *stat, float *part, hipStream_t s) {
  const size_t lds = align_bytes(sizeof(DqLds<T, DP>) + sizeof(float) * size_t(a.G) * a.cols) +
                     (part != nullptr ? sizeof(Cell) * cell_sets<NQ, SHARE>(a.G) * 16 * size_t(a.cols) : 0);
  SGL_REQUIRE(lds <= 160 * 1024, "cross_attention_backward: %zu bytes of LDS", lds);
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dq<T, DP, NQ, SHARE>), lds));
  launch(&k_attn_dq<T, DP, NQ, SHARE>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(kBlock), lds, s, a, tiles,
         static_cast<const T *>(o), static_cast<const T *>(rest), lse, static_cast<const T *>(go),
         static_cast<T *>(dq), stat, part);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

template <typename T, int DP, bool SHARE>
int launch_dkv(const Args &a, const float *lse, const void *go, const float2 *stat, void *dk, void *dv,
               hipStream_t s) {
  const int64_t tiles = (a.p.lk + kKeys - 1) / kKeys;
  const size_t lds = sizeof(DkvLds<T, DP>) + sizeof(float) * size_t(a.G) * a.cols;
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dkv<T, DP, SHARE>), lds));
  launch(&k_attn_dkv<T, DP, SHARE>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(kBlock), lds, s, a, tiles, lse,
         static_cast<const T *>(go), stat, static_cast<T *>(dk), static_cast<T *>(dv));
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

}  // namespace

size_t backward_bytes(const Args &a) {
  return stat_bytes(a) + sizeof(float) * size_t(a.p.n * dq_form(a).tiles) * a.p.heads_q * a.cols;
}

int run_backward(const Args &a, const void *o, const void *rest, const float *lse, const void *go, void *dq, void *dk,
                 void *dv, float *dbias, void *ws, hipStream_t s) {
  float2 *stat = static_cast<float2 *>(ws);
  float *part = dbias != nullptr ? reinterpret_cast<float *>(static_cast<char *>(ws) + stat_bytes(a)) : nullptr;
  const DqForm f = dq_form(a);
  return by_instance(a.p, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (f.tiles > 0) {
      int rc;
      if (f.nq == 1) rc = launch_dq<T, DP, 1, false>(a, f.tiles, o, rest, lse, go, dq, stat, part, s);
      else if (f.share) rc = launch_dq<T, DP, 2, true>(a, f.tiles, o, rest, lse, go, dq, stat, part, s);
      else rc = launch_dq<T, DP, 2, false>(a, f.tiles, o, rest, lse, go, dq, stat, part, s);
      if (rc != SGL_OK) return rc;
    }
    if (dbias != nullptr) sum_rows(part, a.p.n * f.tiles, a.p.heads_q * a.cols, dbias, s);
    if (a.p.lk == 0) {
      SGL_CHECK_LAUNCH();
      return int(SGL_OK);
    }
    if (a.G % 2 == 0) return launch_dkv<T, DP, true>(a, lse, go, stat, dk, dv, s);
    return launch_dkv<T, DP, false>(a, lse, go, stat, dk, dv, s);
  });
}

}  // namespace attn
}  // namespace sgl
