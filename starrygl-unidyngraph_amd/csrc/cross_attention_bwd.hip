// Backward kernels of the cross attention: dq, the bias' gradient and D from
// one walk of each row block over the keys, dk and dv from one walk of each
// key block over the rows. The scores are formed again in both.
#include "cross_attention.h"

namespace sgl {
namespace attn {
namespace {

// ------------------------------------------------------------------ the largest |v|
// Of the live keys of a (sequence, key head), a part of its
// keys a workgroup: what bounds the cells. A kernel of its own, 5 us: it reads
// v once, where every row tile's workgroup would have to before its first cell.
inline int vmost_parts(const Args &a) {   // (a workgroup's four loads a thread, 64 workgroups at most)
  const int dp = a.p.head_dim <= 32 ? 32 : a.p.head_dim <= 64 ? 64 : 128, e = a.p.dtype == SGL_FP32 ? 4 : 8;
  const int64_t keys = 4 * kBlock * e / dp;
  return int(std::min<int64_t>(64, (a.p.lk + keys - 1) / keys));
}

template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_vmost(Args a, int parts, float *__restrict__ vmost) {
  using L = Tile<T, DP>;
  constexpr int E = Mma<T>::E, RPB = kBlock / L::UPR, U = 4;
  __shared__ uint32_t red[kWaves];
  const TileAt at_ = tile_at(blockIdx.x, uint32_t(parts), a.p.heads_kv);
  const Seq<T> q = seq_of<T>(a.p, at_.n, at_.hk, a.G);
  const int r0 = threadIdx.x / L::UPR, d = (threadIdx.x % L::UPR) * E, w = wave_index();
  Largest<T> most;
  for (int64_t j0 = int64_t(at_.tile) * (RPB * U); j0 < q.klen; j0 += int64_t(parts) * (RPB * U)) {
    FragOf<T> f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + u * RPB + r0;
      f[u] = load_raw<T>(q.v + j * a.p.v_t, key_live(q, a.p, j), d, a.p.head_dim);   // (a last vector's overlap is v too)
    }
#pragma unroll
    for (int u = 0; u < U; ++u) most.add(f[u]);
  }
  const float x = most.wave();
  if ((threadIdx.x & 63) == 0) red[w] = __float_as_uint(x);   // (as bits: NaN is the largest)
  __syncthreads();
  if (threadIdx.x == 0) vmost[blockIdx.x] = __uint_as_float(max(max(red[0], red[1]), max(red[2], red[3])));
}

// ------------------------------------------------------------------ dq, dbias, D
// As the forward with many rows. D = <do, o> takes o with what its rounding
// left (rest), so that the sums that should cancel do; where all keys lie in
// one tile it is the sum of p dp itself, which cancels exactly (a single key
// has no gradient). The table's gradient is summed in 64-bit cells of fixed
// point in LDS (a float atomic of LDS costs 194 clocks a wave, an integer one
// 8), relative to a bound on their sum; where that is not finite (a do, v or
// score that is not, or magnitudes whose product overflows) the workgroup's
// part is NaN. 8 sequences, 8 heads of 64, 1000 x 2049 in bf16: 195
// us; of workgroups of 4 waves instead of 8 a tenth more.
template <typename T, int DP, int TK>
struct alignas(16) DqLds {
  T k[TK * Tile<T, DP>::LD], v[TK * Tile<T, DP>::LD];
  KeyInfo<TK> info;
};
template <int ROWS>
struct alignas(16) DqSums {
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
__global__ __launch_bounds__(RW * KW * 64, (2)) void k_attn_dq(Args a, int64_t tiles, const T *__restrict__ o,
                                                          const T *__restrict__ rest, const float2 *__restrict__ lse,
                                                          const T *__restrict__ go, T *__restrict__ dq,
                                                          float *__restrict__ rowdelta, float *__restrict__ part,
                                                          const float *__restrict__ vmost, int vparts) {
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
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15;
  const int wr = w / KW, k0 = (w % KW) * KB * 16;
  const int sets = cell_sets<NQ, SHARE, RW>(a.G), slots = cell_slots(SHARE ? a.G / 2 : a.G);
  Cell *cells = reinterpret_cast<Cell *>(smem + align_bytes(NB * sizeof(S) + sizeof(X) + table_bytes(a)));
  const TileAt at_ = tile_at(blockIdx.x, uint32_t(tiles), p.heads_kv);
  const uint32_t rt = at_.tile;
  const int hk = at_.hk;
  const int64_t n = at_.n;
  const Seq<T> q = seq_of<T>(p, n, hk, a.G);
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  const uint32_t t0 = rt * (SHARE ? RW * 16 : RW * 16 * NQ);
  const uint32_t i0 = __builtin_amdgcn_readfirstlane(row_at<SHARE>(t0, 0, a.G).i);
  const bool any = i0 < q.qlen;
  const bool one_tile = q.klen <= kKeys;
  if (biased) stage_bias(table, a, hk, threadIdx.x, BLOCK);
  if (part != nullptr) clear_cells(cells, sets * a.cols * slots, threadIdx.x, BLOCK);
  RowAt row[NQ];
  bool in[NQ], ok[NQ];
  FragOf<T> qf[NQ][ST], gf[NQ][ST];
  int64_t qpos[NP];
  int qrel[NP];
  float delta[NQ], size = 0.f;   // size: this lane's share of the rows' |do|_1
  float2 ls[NQ];
  const int64_t base = biased && any ? scalar_load(q.qpos + int64_t(i0) * p.qpos_t) : 0;
  const int64_t stat0 = (n * p.heads_kv + hk) * a.rows;
  bool qnear = true;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    const uint32_t t = SHARE ? t0 + wr * 16 + cl : t0 + (wr * NQ + b) * 16 + cl;
    row[b] = row_at<SHARE>(t, b, a.G);
    in[b] = row[b].i < p.lq;
    ok[b] = row[b].i < q.qlen;
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
    float sum = 0.f;
    delta[b] = 0.f;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      const int d = st * M::KS + g * M::E;
      qf[b][st] = load_row<T>(q.q + int64_t(row[b].i) * p.q_t + row[b].h * p.q_h, ok[b], d, dh);
      gf[b][st] = load_row<T>(go + at, ok[b], d, dh);
#pragma unroll
      for (int e = 0; e < M::E; ++e) sum += fabsf(float(gf[b][st][e]));
      if (!one_tile) {
        const FragOf<T> of = load_row<T>(o + at, ok[b], d, dh);
        FragOf<T> rf = zero_frag<T>();
        if (rest != nullptr) rf = load_row<T>(rest + at, ok[b], d, dh);
#pragma unroll
        for (int e = 0; e < M::E; ++e) delta[b] += float(gf[b][st][e]) * whole_of<T>(of[e], rf[e]);
      }
    }
    delta[b] = groups_sum(delta[b]);
    const int64_t r = stat0 + int64_t(row[b].i) * a.G + row[b].h;
    ls[b] = ok[b] ? lse[r] : make_float2(INFINITY, 0.f);
    // (rows without p count for nothing, whatever their do; a NaN score for NaN)
    if (w % KW == 0) size += ls[b].y != ls[b].y ? NAN : ls[b].x == INFINITY ? 0.f : sum;
    if (g == 0 && in[b] && w % KW == 0) rowdelta[r] = delta[b];   // for dk and dv
    if (b < NP) {
      qpos[b] = biased && ok[b] ? q.qpos[int64_t(row[b].i) * p.qpos_t] : base;
      qnear = qnear && is_near(qpos[b] - base);
      qrel[b] = int(qpos[b] - base);
    }
  }
  qnear = __all(qnear);
  const float c = p.scale * kLog2e;
  float up = 1.f, bad = 0.f;   // the cells' power of two, for the whole workgroup; NaN if they cannot hold
  if (part != nullptr) {
    Largest<float> vm;
    if (lane < vparts) vm.bits = __float_as_uint(vmost[(n * p.heads_kv + hk) * vparts + lane]);
    size = wave_reduce_sum(size);
    if (lane == 0) sx.red[w] = size;
    __syncthreads();
    size = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) size += sx.red[i];
    const float most = 2.f * vm.wave() * size;
    up = cell_scale(most);
    bad = most < INFINITY ? 0.f : NAN;
  }
  f32x4 acc[NQ][DB];
  float gs[NQ];   // (fp16) what ds of this wave's rows is multiplied by
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    gs[b] = kFirstScale;
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
    const uint32_t on = tile.live_of(k0, KB * 16);
    __syncthreads();
    if (j0 + TK < q.klen) tile.load(q, a, j0 + TK);
    float x[NQ][KB][4], y[NQ][KB][4];   // p and dp, then ds
    int col[NP][KB][4];
    if (biased) {
      const bool near_now = qnear && s.info.near_ != 0;
#pragma unroll
      for (int b = 0; b < NP; ++b) columns(col[b], s.info.pos, k0 + 4 * g, qrel[b], qpos[b], near_now, 1, bk);
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
      // (the forward's scores to the bit, then less the row's maximum and sum: taken off within the fma, its rounding
      // is one error for a row and column, which the table's gradient keeps; and a single key's p is 1)
      scale_scores(x[b], c, 0.f, table + row[b].h * table_ld(a), col[b < NP ? b : 0], biased);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) x[b][kb][v] = __builtin_amdgcn_exp2f((x[b][kb][v] - ls[b].x) - ls[b].y);
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
        if (g == 0 && in[b] && w % KW == 0) rowdelta[stat0 + int64_t(row[b].i) * a.G + row[b].h] = delta[b];
      }
    }
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) y[b][kb][v] = x[b][kb][v] * (y[b][kb][v] - delta[b]);
    if (on != full_mask(KB * 16)) {   // (0 too where do, and with it D, is not finite)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const bool dead = !((on >> (kb * 16 + 4 * g + v)) & 1);
#pragma unroll
          for (int b = 0; b < NQ; ++b) y[b][kb][v] = dead ? 0.f : y[b][kb][v];
        }
    }
    if (part != nullptr) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        const int set = sets == RW * NQ ? wr * NQ + b : SHARE ? b : 0;
        add_cells(cells + set * a.cols * slots, col[b < NP ? b : 0], y[b], slots, up);
      }
    }
    if constexpr (std::is_same_v<T, fp16_t>) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) follow_scale(y[b], gs[b], acc[b]);
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
    // cell (set, column, slot) belongs to the head of its blocks' row `slot`: a
    // thread sums a (head, column) over them
    __syncthreads();
    const bool own = sets == RW * NQ;
    float *out = part + ((n * tiles + rt) * p.heads_kv + hk) * a.G * a.cols;
    for (int x = threadIdx.x; x < a.G * a.cols; x += BLOCK) {
      const int h = x / a.cols, cidx = x - h * a.cols;
      long long t = 0;
      for (int set = 0; set < sets; ++set) {
        const int ww = own ? set / NQ : 0, b = own ? set % NQ : SHARE ? set : 0;
        const int h0 = row_at<SHARE>(SHARE ? t0 + ww * 16 : t0 + (own ? set : 0) * 16, b, a.G).h;   // of c = 0
        for (int i = 0; i < slots; ++i) {
          const int e = (i + cidx) & (slots - 1);   // (rotated: neighbouring columns in different banks)
          if ((h0 + (SHARE ? 2 : 1) * e) % a.G == h)
            t += static_cast<long long>(cells[(set * a.cols + cidx) * slots + e]);
        }
      }
      out[x] = cell_value(t, up) + bad;
    }
  }
  if constexpr (std::is_same_v<T, fp16_t>) {
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[b][d] *= 1.f / gs[b];
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
    const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
    for (int d = 0; d < DB; ++d) store4(dq + at, d * 16 + 4 * g, dh, acc[b][d] * p.scale);
  }
}

// ------------------------------------------------------------------ dk, dv
// A workgroup takes CW blocks of 16 keys (one a lane of 16) and walks the rows
// of all G heads; RS waves share a key block, each with 32 rows of every tile,
// and are joined at the end. The 32 rows of a step are two heads of 16
// queries (SHARE, an even G) or 32 rows in order. The next tile's rows are in
// flight while one is worked on: a thread's unit of a step lies at a uniform
// pointer and an offset that it keeps (an odd G above one divides instead);
// the first wave fetches what belongs to a row (D, maximum, sum, position). Bound by
// what a SIMD issues and LDS together (24 fragment reads and 8 table reads a
// step of 512 scores) at two waves a SIMD: at the same size 245 us; with 32 keys
// and 64 rows a workgroup the same, with 8 waves of it a tenth more.
constexpr int kRows = 32;

template <typename T, int DP, int TR>
struct alignas(16) DkvLds {
  T q[TR * Tile<T, DP>::LD], go[TR * Tile<T, DP>::LD];
  KeyInfo<TR> info;   // (of the rows)
  float most[TR], sum[TR], delta[TR];
  int head[TR];
};

template <typename T, int DP, bool SHARE, int CW, int RS>
__global__ __launch_bounds__(CW * RS * 64, (RS == 4 ? 1 : simd_waves<T, DP>(3, 2))) void k_attn_dkv(Args a, int64_t tiles, const T *__restrict__ go,
                                                           const float2 *__restrict__ lse,
                                                           const float *__restrict__ rowdelta,
                                                           T *__restrict__ dk, T *__restrict__ dv) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  constexpr int TR = kRows * RS, BLOCK = CW * RS * 64;
  using S = DkvLds<T, DP, TR>;
  constexpr int NB = buffers<S>();
  constexpr int ST = DP / M::KS, DB = DP / 16, RB = kRows / 16, NP = SHARE ? 1 : RB;
  constexpr bool kHalf = std::is_same_v<T, fp16_t>;
  extern __shared__ __align__(16) char smem[];
  S *const bufs = reinterpret_cast<S *>(smem);
  float *table = reinterpret_cast<float *>(smem + NB * sizeof(S));
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4;
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
  const uint32_t pairs = uint32_t(a.G) >> 1, qlen = uint32_t(q.qlen);
  const bool any = kt * CW * 16 < q.klen;
  const uint32_t steps = !any ? 0 : SHARE ? (qlen + 15) / 16 * pairs : (qlen * a.G + kRows - 1) / kRows;
  FragOf<T> kf[ST], vf[ST];
#pragma unroll
  for (int st = 0; st < ST; ++st) {
    const int d = st * M::KS + g * M::E;
    kf[st] = load_row<T>(q.k + j * p.k_t, on, d, dh);
    vf[st] = load_row<T>(q.v + j * p.v_t, on, d, dh);
  }
  const int64_t base = biased && steps > 0 ? scalar_load(q.qpos) : 0;
  const int64_t kp = biased && on ? q.kpos[j * p.kpos_t] : base;
  const int krel = int(kp - base);
  const bool knear = __all(is_near(kp - base));
  const float c = p.scale * kLog2e;
  float gs = kFirstScale;   // (fp16) what ds of this wave's keys is multiplied by
  f32x4 acc[2][DB];   // dk, dv
#pragma unroll
  for (int b = 0; b < DB; ++b) acc[0][b] = acc[1][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int RSTEP = BLOCK / L::UPR, PER = (TR + RSTEP - 1) / RSTEP, RL = (TR + 63) / 64;
  static_assert(RSTEP % kRows == 0 || kRows % RSTEP == 0, "a pass of the workgroup keeps a thread's place in a step");
  FragOf<T> qr[PER], gr[PER];
  // a step's first row (i, h) and a thread's row x of its 32 from there
  const bool flat = SHARE || a.G == 1;
  auto first_of = [&](uint32_t step) {
    if constexpr (SHARE) {
      const uint32_t ib = pairs == 1 ? step : step / pairs;
      return RowAt{ib * 16, int(step - ib * pairs) * 2};
    } else {
      return row_at<false>(step * kRows, 0, a.G);
    }
  };
  auto row_of = [&](const RowAt &f, uint32_t step, int x) {
    if constexpr (SHARE) return RowAt{f.i + (x & 15), f.h + (x >> 4)};
    else return flat ? RowAt{f.i + x, 0} : row_at<false>(step * kRows + x, 0, a.G);
  };
  const int r0 = threadIdx.x / L::UPR, d0 = (threadIdx.x % L::UPR) * M::E, at0 = min(d0, dh - M::E);
  const int64_t go_t = int64_t(p.heads_q) * dh;
  auto offset = [&](int x, int64_t t, int64_t h) { return SHARE ? (x & 15) * t + (x >> 4) * h : x * t; };
  constexpr int PLACES = RSTEP < kRows ? kRows / RSTEP : 1;
  static_assert(PLACES <= 8, "places of a thread in a step");
  int64_t qo[PLACES], gofs[PLACES];
#pragma unroll
  for (int i = 0; i < PLACES; ++i) {
    qo[i] = offset(r0 % kRows + i * RSTEP, p.q_t, p.q_h) + at0;
    gofs[i] = offset(r0 % kRows + i * RSTEP, go_t, dh) + at0;
  }
  int64_t qp[RL];
  float2 st_[RL];
  float de_[RL];
  int he[RL] = {};
  auto load_step = [&](uint32_t step) {
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      st_[i] = make_float2(INFINITY, 0.f);
      de_[i] = 0.f;
      qp[i] = 0;
      if (w == 0) {
        const int x = i * 64 + lane;
        const uint32_t sub = step + x / kRows;
        const RowAt r = row_of(first_of(sub), sub, x % kRows);
        he[i] = r.h;
        if (x < TR && r.i < qlen) {
          st_[i] = lse[stat0 + int64_t(r.i) * a.G + r.h];
          de_[i] = rowdelta[stat0 + int64_t(r.i) * a.G + r.h];
          if (biased) qp[i] = q.qpos[int64_t(r.i) * p.qpos_t];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int x = r0 + i * RSTEP;
      // (a wave's rows lie in one step of 32)
      const uint32_t sub = step + uint32_t(__builtin_amdgcn_readfirstlane(x / kRows));
      const RowAt f = first_of(sub), t = row_of(f, sub, x % kRows);
      qr[i] = zero_frag<T>();
      gr[i] = zero_frag<T>();
      if (x < TR && t.i < qlen && d0 < dh) {
        if (flat) {
          const T *qb = q.q + int64_t(f.i) * p.q_t + f.h * p.q_h;
          const T *gb = go + out_row(a, n, hk, f.i, f.h);
          __builtin_memcpy(&qr[i], qb + qo[i % PLACES], 16);
          __builtin_memcpy(&gr[i], gb + gofs[i % PLACES], 16);
        } else {
          __builtin_memcpy(&qr[i], q.q + int64_t(t.i) * p.q_t + t.h * p.q_h + at0, 16);
          __builtin_memcpy(&gr[i], go + out_row(a, n, hk, t.i, t.h) + at0, 16);
        }
      }
    }
  };
  if (steps > 0) load_step(0);
  int buf = 0;
  for (uint32_t step = 0; step < steps; step += RS) {
    S &s = bufs[buf];
    if constexpr (NB == 1) __syncthreads();
    else buf ^= 1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int x = r0 + i * RSTEP;
      if (TR % RSTEP == 0 || x < TR) {
        *reinterpret_cast<FragOf<T> *>(s.q + x * L::LD + d0) = fix<T>(qr[i], d0, dh);
        *reinterpret_cast<FragOf<T> *>(s.go + x * L::LD + d0) = fix<T>(gr[i], d0, dh);
      }
    }
    if (w == 0) {
      bool near_ = true;   // (looked at here, a tile after its load)
#pragma unroll
      for (int i = 0; i < RL; ++i) {
        const int x = i * 64 + lane;
        const int64_t at = st_[i].x == INFINITY ? base : qp[i];   // (no row, or one without p)
        near_ = near_ && is_near(at - base);
        if (x < TR) {
          s.most[x] = st_[i].x;
          s.sum[x] = st_[i].y;
          s.delta[x] = de_[i];
          s.head[x] = he[i] * table_ld(a);
          s.info.pos.pos[x] = at;
          s.info.pos.rel[x] = int(at - base);
        }
      }
      near_ = __all(near_);
      if (lane == 0) s.info.near_ = near_;
    }
    __syncthreads();
    if (step + RS < steps) load_step(step + RS);
    float x[RB][4], y[RB][4];   // p and ds, rows x this lane's key
    int col[RB][4];
    if (biased) {
      int own[NP][4];
      columns(own, s.info.pos, x0 + 4 * g, krel, kp, knear && s.info.near_ != 0, -1, bk);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int v = 0; v < 4; ++v) col[rb][v] = own[rb < NP ? rb : 0][v] + s.head[x0 + rb * 16 + 4 * g + v];
    }
    float mov[RB][4], suv[RB][4], dev[RB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      __builtin_memcpy(mov[rb], s.most + x0 + rb * 16 + 4 * g, sizeof(mov[rb]));
      __builtin_memcpy(suv[rb], s.sum + x0 + rb * 16 + 4 * g, sizeof(suv[rb]));
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
        const float pr = on ? __builtin_amdgcn_exp2f((x[rb][v] - mov[rb][v]) - suv[rb][v]) : 0.f;
        x[rb][v] = pr * kProbUp<T>;
        y[rb][v] = pr * (y[rb][v] - dev[rb][v]);
      }
    if constexpr (kHalf) follow_scale(y, gs, acc[0]);
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
  if constexpr (kHalf) {
#pragma unroll
    for (int b = 0; b < DB; ++b) acc[0][b] *= 1.f / gs;
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
  const float fk = p.scale, fv = 1.f / kProbUp<T>;
#pragma unroll
  for (int b = 0; b < DB; ++b) {
    // (a dead key's sums are of p = 0, which an infinity in do or q makes NaN)
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    store4(dk + row, b * 16 + 4 * g, dh, on ? acc[0][b] * fk : zero);
    store4(dv + row, b * 16 + 4 * g, dh, on ? acc[1][b] * fv : zero);
  }
}

// ------------------------------------------------------------------ host
size_t stat_bytes(const Args &a) { return align_up(sizeof(float) * size_t(a.p.n * a.p.heads_kv * a.rows)); }
int64_t dq_tiles(const Args &a) {
  if (!many_rows(a)) return row_tiles(a, 1, false, 1);
  const bool two = a.p.dtype != SGL_FP32 || a.p.head_dim <= 64;   // two_blocks
  return two ? row_tiles(a, 2, a.G % 2 == 0, 4) : row_tiles(a, 1, false, 4);
}

template <typename T, int DP, int NQ, bool SHARE, int RW, int KW>
int launch_dq(const Args &a, int64_t tiles, const void *o, const void *rest, const float2 *lse, const void *go, void *dq,
              float *stat, float *part, float *vmost, hipStream_t s) {
  const int vparts = vmost_parts(a);
  if (part != nullptr && vparts > 0)
    launch(&k_attn_vmost<T, DP>, dim3(unsigned(a.p.n * a.p.heads_kv * vparts)), dim3(kBlock), 0, s, a, vparts, vmost);
  const size_t lds = std::max(
      align_bytes(buffers<DqLds<T, DP, tile_keys<T>(KW)>>() * sizeof(DqLds<T, DP, tile_keys<T>(KW)>) +
                  sizeof(DqSums<RW * KW * NQ * 16>) + table_bytes(a)) +
          (part != nullptr ? sizeof(Cell) * cell_sets<NQ, SHARE, RW>(a.G) * cell_slots(SHARE ? a.G / 2 : a.G) * size_t(a.cols) : 0),
      join_bytes(RW, KW, NQ, DP));
  SGL_REQUIRE(lds <= 160 * 1024, "cross_attention_backward: %zu bytes of LDS", lds);
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dq<T, DP, NQ, SHARE, RW, KW>), lds));
  launch(&k_attn_dq<T, DP, NQ, SHARE, RW, KW>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(RW * KW * kWave), lds,
         s, a, tiles, static_cast<const T *>(o), static_cast<const T *>(rest), lse, static_cast<const T *>(go),
         static_cast<T *>(dq), stat, part, static_cast<const float *>(vmost), vparts);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

template <typename T, int DP, bool SHARE, int CW, int RS>
int launch_dkv(const Args &a, const float2 *lse, const void *go, float *stat, void *dk, void *dv, hipStream_t s) {
  const int64_t tiles = (a.p.lk + 16 * CW - 1) / (16 * CW);
  using S = DkvLds<T, DP, kRows * RS>;
  const size_t lds = std::max(buffers<S>() * sizeof(S) + table_bytes(a),
                              join_bytes(CW, RS, 2, DP));
  SGL_REQUIRE(lds <= 160 * 1024, "cross_attention_backward: %zu bytes of LDS", lds);
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_dkv<T, DP, SHARE, CW, RS>), lds));
  launch(&k_attn_dkv<T, DP, SHARE, CW, RS>, dim3(unsigned(a.p.n * a.p.heads_kv * tiles)), dim3(CW * RS * kWave), lds, s,
         a, tiles, static_cast<const T *>(go), lse, static_cast<const float *>(stat),
         static_cast<T *>(dk), static_cast<T *>(dv));
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

size_t part_bytes(const Args &a) {
  return align_up(sizeof(float) * size_t(a.p.n * dq_tiles(a)) * a.p.heads_q * a.cols);
}

}  // namespace

size_t backward_bytes(const Args &a) {
  return stat_bytes(a) + part_bytes(a) + (a.cols > 0 ? sizeof(float) * size_t(a.p.n * a.p.heads_kv) * vmost_parts(a) : 0);
}

int run_backward(const Args &a, const void *o, const void *rest, const float *stats, const void *go, void *dq, void *dk,
                 void *dv, float *dbias, void *ws, hipStream_t s) {
  const float2 *lse = reinterpret_cast<const float2 *>(stats);
  float *stat = static_cast<float *>(ws);
  float *part = dbias != nullptr ? reinterpret_cast<float *>(static_cast<char *>(ws) + stat_bytes(a)) : nullptr;
  float *vmost = dbias != nullptr ? reinterpret_cast<float *>(static_cast<char *>(ws) + stat_bytes(a) + part_bytes(a)) : nullptr;
  const int64_t tiles = dq_tiles(a);
  return by_instance(a.p, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (tiles > 0) {
      int rc;
      if (!many_rows(a)) rc = launch_dq<T, DP, 1, false, 1, 4>(a, tiles, o, rest, lse, go, dq, stat, part, vmost, s);
      else if constexpr (!two_blocks<T, DP>()) rc = launch_dq<T, DP, 1, false, 4, 2>(a, tiles, o, rest, lse, go, dq, stat, part, vmost, s);
      else if (a.G % 2 == 0) rc = launch_dq<T, DP, 2, true, 4, 2>(a, tiles, o, rest, lse, go, dq, stat, part, vmost, s);
      else rc = launch_dq<T, DP, 2, false, 4, 2>(a, tiles, o, rest, lse, go, dq, stat, part, vmost, s);
      if (rc != SGL_OK) return rc;
    }
    if (dbias != nullptr) sum_rows(part, a.p.n * tiles, a.p.heads_q * a.cols, dbias, s);
    if (a.p.lk == 0) {
      SGL_CHECK_LAUNCH();
      return int(SGL_OK);
    }
    // 64 keys a workgroup where that fills the GPU, else 16, its four waves along the rows
    const bool wide = a.p.n * a.p.heads_kv * ((a.p.lk + 63) / 64) >= 192;
    constexpr int RS = two_blocks<T, DP>() && DP <= 64 ? 1 : 2;   // (three 4-wave workgroups a CU, or one of 8)
    if (a.G % 2 == 0)
      return wide ? launch_dkv<T, DP, true, 4, RS>(a, lse, go, stat, dk, dv, s)
                  : launch_dkv<T, DP, true, 1, 4>(a, lse, go, stat, dk, dv, s);
    return wide ? launch_dkv<T, DP, false, 4, RS>(a, lse, go, stat, dk, dv, s)
                : launch_dkv<T, DP, false, 1, 4>(a, lse, go, stat, dk, dv, s);
  });
}

}  // namespace attn
}  // namespace sgl
