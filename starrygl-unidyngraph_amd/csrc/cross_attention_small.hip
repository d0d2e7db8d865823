// The cross attention's backward for windows: up to 32 rows (queries x heads
// of a key head) and 64 keys, one wave a (sequence, key head) and no barriers.
//
// Everything of an item is on chip at once, so the softmax is formed again
// with its own maximum and sum, D is the sum of p dp, and nothing of the
// forward is read but its inputs. q, k, v and do are read once, straight into
// fragments; k, do and q pass through the wave's LDS for the products down
// their columns, p and ds to be read with the rows as the reduction index. A
// wave walks items of one key head, so that the bias' gradient is one row of
// partial sums a wave. 4000 windows of 20 x 32, 4 heads of 43 in bf16: 118 us,
// bound by a wave's chain of loads and products at two waves a SIMD (a pass of
// both directions went from 1313 to 323 us when this form and one wave an item
// in the forward took over from the tiled kernels; 186 to 190 now).
#include "cross_attention.h"

namespace sgl {
namespace attn {
namespace {

template <typename T, int DP, int NQ, int NK>
struct alignas(16) SmallLds {
  static constexpr int R = 16 * NQ, K = 16 * NK;
  static constexpr int kKeyTile = K * Tile<T, DP>::LD, kProbTile = R * Tile<T, K>::LD;
  // k, then p and ds in its place; do, then q in its place
  T a[kKeyTile > 2 * kProbTile ? kKeyTile : 2 * kProbTile];
  T b[R * Tile<T, DP>::LD];
  PosTile<K> pos;
};

template <typename Lds>
__host__ __device__ __forceinline__ size_t small_lds(const Args &a, int nq, bool cells) {   // bytes a wave
  return align_bytes(sizeof(Lds) + table_bytes(a)) +
         (cells ? sizeof(Cell) * size_t(16 % a.G == 0 ? 1 : nq) * cell_slots(a.G) * a.cols : 0);
}

template <typename T, int DP, int NQ, int NK>
__global__ __launch_bounds__(kBlock, (DP <= 64 ? 2 : 1)) void k_attn_small_bwd(Args a, int64_t each, const T *__restrict__ go,
                                                           T *__restrict__ dq, T *__restrict__ dk,
                                                           T *__restrict__ dv, float *__restrict__ part) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using Lds = SmallLds<T, DP, NQ, NK>;
  using P = Tile<T, Lds::K>;
  constexpr int ST = DP / M::KS, DB = DP / 16, R = Lds::R, K = Lds::K;
  extern __shared__ __align__(16) char smem[];
  const sgl_attention &p = a.p;
  const int dh = p.head_dim;
  const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, cl = lane & 15;
  const size_t per = small_lds<Lds>(a, NQ, part != nullptr);
  Lds &s = *reinterpret_cast<Lds *>(smem + w * per);
  float *table = reinterpret_cast<float *>(smem + w * per + sizeof(Lds));
  Cell *cells = reinterpret_cast<Cell *>(smem + w * per + align_bytes(sizeof(Lds) + table_bytes(a)));
  const int sets = 16 % a.G == 0 ? 1 : NQ, slots = cell_slots(a.G);   // (one set: row c of either block has the same head)
  const TileAt at_ = tile_at(blockIdx.x * (blockDim.x / kWave) + w, 1, p.heads_kv);
  const int hk = at_.hk;
  const int64_t first = at_.n;
  if (first >= each) return;   // (whole waves; there are no barriers)
  const bool biased = p.bias != nullptr;
  const Buckets bk = buckets_of(p);
  if (biased) stage_bias(table, a, hk, lane, kWave);
  if (part != nullptr) clear_cells(cells, sets * slots * a.cols, lane, kWave);
  // the cells' power of two (0: nothing in them yet), the bound on all that was added, NaN if they cannot hold
  float up = 0.f, reach = 0.f, bad = 0.f;
  wave_sync();
  RowAt row[NQ];
#pragma unroll
  for (int b = 0; b < NQ; ++b) row[b] = row_at<false>(uint32_t(b * 16 + cl), b, a.G);
  const float c = p.scale * kLog2e;
  for (int64_t n = first; n < p.n; n += each) {
    const Seq<T> q = seq_of<T>(p, n, hk, a.G);
    const int64_t base = biased && q.qlen > 0 ? scalar_load(q.qpos) : 0;
    // every load of the item is issued before anything is looked at
    const bool in_key = lane < K && q.qlen > 0 && lane < q.klen;
    int64_t kpos = 0;
    int byte = 0;
    if (biased && in_key) kpos = q.kpos[lane * p.kpos_t];
    if (q.mask != nullptr && in_key) byte = q.mask[lane * p.mask_t];
    FragOf<T> kf[NK][ST], vf[NK][ST];
#pragma unroll
    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int d = st * M::KS + g * M::E;
        const int64_t j = kb * 16 + cl;
        kf[kb][st] = load_raw<T>(q.k + j * p.k_t, q.qlen > 0 && j < q.klen, d, dh);
        vf[kb][st] = load_raw<T>(q.v + j * p.v_t, q.qlen > 0 && j < q.klen, d, dh);
      }
    FragOf<T> qf[NQ][ST], gf[NQ][ST];
    int64_t qpos[NQ];
    int qrel[NQ];
    bool ok[NQ];
    Largest<T> gm, vm;   // |do|, |v|
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      ok[b] = row[b].i < q.qlen;
      const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int d = st * M::KS + g * M::E;
        qf[b][st] = load_raw<T>(q.q + int64_t(row[b].i) * p.q_t + row[b].h * p.q_h, ok[b], d, dh);
        gf[b][st] = load_raw<T>(go + at, ok[b], d, dh);
      }
      qpos[b] = 0;
      if (biased && ok[b]) qpos[b] = q.qpos[int64_t(row[b].i) * p.qpos_t];
    }
    uint64_t live = q.qlen > 0 ? first_bits(q.klen) : 0;
    if (q.mask != nullptr) live = __ballot(byte != 0);
    const int64_t kp = lane < K && ((live >> lane) & 1) ? kpos : base;
    bool near_ = is_near(kp - base);
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      if (!ok[b]) qpos[b] = base;
      near_ = near_ && is_near(qpos[b] - base);
      qrel[b] = int(qpos[b] - base);
    }
    near_ = __all(near_);
    wave_sync();   // the item before is done with the LDS
    if (biased && lane < K) {
      s.pos.pos[lane] = kp;
      s.pos.rel[lane] = int(kp - base);
    }
    wave_sync();
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int d = st * M::KS + g * M::E;
        qf[b][st] = fix<T>(qf[b][st], d, dh);
        gf[b][st] = fix<T>(gf[b][st], d, dh);
        gm.add(gf[b][st]);
        *reinterpret_cast<FragOf<T> *>(s.b + (b * 16 + cl) * L::LD + d) = gf[b][st];
      }
    // scores and dp, (keys x rows)
    float x[NQ][NK][4], y[NQ][NK][4];
    int col[NQ][NK][4];
    if (biased) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) columns(col[b], s.pos, 4 * g, qrel[b], qpos[b], near_, 1, bk);
    }
#pragma unroll
    for (int kb = 0; kb < NK; ++kb) {
      const bool on_r = (live >> (kb * 16 + cl)) & 1;
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int d = st * M::KS + g * M::E;
        kf[kb][st] = fix<T>(kf[kb][st], d, dh);
        vf[kb][st] = fix<T>(vf[kb][st], d, dh);
        if (q.mask != nullptr && !on_r) kf[kb][st] = vf[kb][st] = zero_frag<T>();
        vm.add(vf[kb][st]);
        *reinterpret_cast<FragOf<T> *>(s.a + (kb * 16 + cl) * L::LD + d) = kf[kb][st];
      }
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        f32x4 sc = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          sc = M::mma(kf[kb][st], qf[b][st], sc);
          dp = M::mma(vf[kb][st], gf[b][st], dp);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = sc[v];
          y[b][kb][v] = dp[v];
        }
      }
    }
    if (part != nullptr && live != 0) {   // (uniform) beyond what the cells' power is for: cells shifted
      // (each row's |do|_1 by dh times the largest |do|)
      reach += 2.f * vm.wave() * (gm.wave() * float(a.rows * dh));
      const float want = cell_scale(reach);
      if (!(reach < INFINITY)) {
        bad = NAN;
      } else if (up == 0.f) {
        up = reach > 0.f ? want : 0.f;
      } else if (want < up) {
        const int by = min(ilogbf(up) - ilogbf(want), 63);
        for (int i = lane; i < sets * slots * a.cols; i += kWave)
          cells[i] = Cell(static_cast<long long>(cells[i]) >> by);
        up = want;
        wave_sync();
      }
    }
    // p, D and ds
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      float mx = -INFINITY, sum = 0.f, de = 0.f;
      scale_scores(x[b], c, 0.f, table + row[b].h * table_ld(a), col[b], biased);
#pragma unroll
      for (int kb = 0; kb < NK; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = (live >> (kb * 16 + 4 * g + v)) & 1 ? x[b][kb][v] : -INFINITY;
          mx = fmaxf(mx, x[b][kb][v]);
        }
      mx = groups_max(mx);
      const float at = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int kb = 0; kb < NK; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] = __builtin_amdgcn_exp2f(x[b][kb][v] - at);
          sum += x[b][kb][v];
        }
      sum = groups_sum(sum);
      const float inv = ok[b] && sum != 0.f ? 1.f / sum : 0.f;   // (NaN stays)
      if (ok[b] && sum != sum) bad = NAN;
#pragma unroll
      for (int kb = 0; kb < NK; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[b][kb][v] *= inv;
          de += x[b][kb][v] * y[b][kb][v];
        }
      de = groups_sum(de);
#pragma unroll
      for (int kb = 0; kb < NK; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v)   // (0 at a dead key also where do, and with it D, is not finite)
          y[b][kb][v] = (live >> (kb * 16 + 4 * g + v)) & 1 ? x[b][kb][v] * (y[b][kb][v] - de) : 0.f;
      if (part != nullptr) add_cells(cells + (sets == 1 ? 0 : b) * slots * a.cols, col[b], y[b], slots, up);
    }
    float fk = p.scale;
    if constexpr (std::is_same_v<T, fp16_t>) {   // one power of two for the item's ds
      Largest<float> dm;
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) dm.add(f32x4{y[b][kb][0], y[b][kb][1], y[b][kb][2], y[b][kb][3]});
      const float most = dm.wave(), gs = most > 0.f ? half_scale(most) : 1.f;
      fk = p.scale / gs;
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            y[b][kb][v] *= gs;
            x[b][kb][v] *= kProbUp<T>;
          }
    }
    // dq (head size x rows)
    wave_sync();
    {
      f32x4 acc[NQ][DB];
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < K / M::KS; ++st) {
        FragOf<T> df[NQ];
#pragma unroll
        for (int b = 0; b < NQ; ++b) df[b] = frag_of<T>(y[b], st);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const FragOf<T> kt = L::template frag_t<K>(s.a, d * 16, st * M::KS);
#pragma unroll
          for (int b = 0; b < NQ; ++b) acc[b][d] = M::mma(kt, df[b], acc[b][d]);
        }
      }
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        if (row[b].i < p.lq) {
          const int64_t at = out_row(a, n, hk, row[b].i, row[b].h);
#pragma unroll
          for (int d = 0; d < DB; ++d) store4(dq + at, d * 16 + 4 * g, dh, acc[b][d] * fk);
        }
      }
    }
    // p and ds as [row][key], over k
    T *ps = s.a, *ds = s.a + R * P::LD;
    wave_sync();
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int kb = 0; kb < NK; ++kb) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 pv, dvv;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          pv[v] = T(x[b][kb][v]);
          dvv[v] = T(y[b][kb][v]);
        }
        const int at = (b * 16 + cl) * P::LD + kb * 16 + 4 * g;
        *reinterpret_cast<T4 *>(ps + at) = pv;
        *reinterpret_cast<T4 *>(ds + at) = dvv;
      }
    wave_sync();
    // dv, then dk (head size x keys), do and then q in s.b
    constexpr int RS = (R + M::KS - 1) / M::KS;   // steps over the rows
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 1) {
        wave_sync();
#pragma unroll
        for (int b = 0; b < NQ; ++b)
#pragma unroll
          for (int st = 0; st < ST; ++st)
            *reinterpret_cast<FragOf<T> *>(s.b + (b * 16 + cl) * L::LD + st * M::KS + g * M::E) = qf[b][st];
        wave_sync();
      }
      T *out = which == 0 ? dv : dk;
      const T *src = which == 0 ? ps : ds;
      const float f = which == 0 ? 1.f / kProbUp<T> : fk;
#pragma unroll
      for (int kb = 0; kb < NK; ++kb) {
        FragOf<T> pf[RS];
#pragma unroll
        for (int st = 0; st < RS; ++st) pf[st] = P::template frag_t<R>(src, kb * 16, st * M::KS);
        const int64_t j = kb * 16 + cl;
        const int64_t at = ((n * p.lk + j) * p.heads_kv + hk) * dh;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < RS; ++st)
            acc = M::mma(L::template frag_t<R>(s.b, d * 16, st * M::KS), pf[st], acc);
          // (a dead key's sum is of p = 0, which an infinity in do or q makes NaN)
          if (j < p.lk) store4(out + at, d * 16 + 4 * g, dh, (live >> j) & 1 ? acc * f : f32x4{0.f, 0.f, 0.f, 0.f});
        }
      }
    }
  }
  if (part != nullptr) {
    wave_sync();
    const bool held = __all(bad == 0.f);
    float *out = part + (first * p.heads_kv + hk) * a.G * a.cols;
    for (int x = lane; x < a.G * a.cols; x += kWave) {
      const int h = x / a.cols, cidx = x - h * a.cols;
      long long t = 0;
      for (int set = 0; set < sets; ++set)
        for (int i = 0; i < slots; ++i) {
          const int e = (i + cidx) & (slots - 1);
          if ((set * 16 + e) % a.G == h) t += static_cast<long long>(cells[(set * a.cols + cidx) * slots + e]);
        }
      out[x] = held ? cell_value(t, up == 0.f ? 1.f : up) : NAN;
    }
  }
}

// Waves a key head: enough to fill the GPU four waves a SIMD deep, the
// sequences in equal numbers.
int64_t small_each(const Args &a) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(a.p.n, 4096 / a.p.heads_kv));
  const int64_t per = (a.p.n + most - 1) / most;
  return (a.p.n + per - 1) / per;
}

template <typename T, int DP, int NQ, int NK>
int launch_small(const Args &a, const void *go, void *dq, void *dk, void *dv, float *part, hipStream_t s) {
  const size_t per = small_lds<SmallLds<T, DP, NQ, NK>>(a, NQ, part != nullptr);
  const int64_t wpb = std::min<int64_t>(kWaves, 160 * 1024 / int64_t(per));   // waves a workgroup
  SGL_REQUIRE(wpb > 0, "cross_attention_backward: %zu bytes of LDS", per);
  const size_t lds = per * size_t(wpb);
  SGL_CHECK_HIP(ensure_dynamic_lds(reinterpret_cast<const void *>(&k_attn_small_bwd<T, DP, NQ, NK>), lds));
  const int64_t each = small_each(a), waves = each * a.p.heads_kv;
  launch(&k_attn_small_bwd<T, DP, NQ, NK>, dim3(unsigned((waves + wpb - 1) / wpb)), dim3(unsigned(wpb) * kWave), lds, s, a, each,
         static_cast<const T *>(go), static_cast<T *>(dq), static_cast<T *>(dk), static_cast<T *>(dv), part);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

}  // namespace

size_t small_backward_bytes(const Args &a) { return sizeof(float) * size_t(small_each(a)) * a.p.heads_q * a.cols; }

int run_small_backward(const Args &a, const void *go, void *dq, void *dk, void *dv, float *dbias, void *ws,
                       hipStream_t s) {
  float *part = dbias != nullptr ? static_cast<float *>(ws) : nullptr;
  const int rc = by_instance(a.p, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (a.rows <= 16) {
      if (a.p.lk <= 32) return launch_small<T, DP, 1, 2>(a, go, dq, dk, dv, part, s);
      return launch_small<T, DP, 1, 4>(a, go, dq, dk, dv, part, s);
    }
    if (a.p.lk <= 32) return launch_small<T, DP, 2, 2>(a, go, dq, dk, dv, part, s);
    return launch_small<T, DP, 2, 4>(a, go, dq, dk, dv, part, s);
  });
  if (rc != SGL_OK) return rc;
  if (dbias != nullptr) sum_rows(part, small_each(a), a.p.heads_q * a.cols, dbias, s);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

}  // namespace attn
}  // namespace sgl
