// Losses over all candidates: what joins the pieces of the forward, a
// teacher's distribution, the rows' coefficients for the gradients, and the
// entry points.
#include "candidates.h"

namespace {

using namespace sgl;
using namespace sgl::cand;

// Sum, maximum over the wave, the same in every lane: rows of 16 lanes rotated
// by 8, 4, 2 and 1, then rows and halves of the wave swapped.
template <int CTRL>
__device__ __forceinline__ float turned(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += turned<0x128>(v);
  v += turned<0x124>(v);
  v += turned<0x122>(v);
  v += turned<0x121>(v);
  return attn::groups_sum(v);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, turned<0x128>(v));
  v = fmaxf(v, turned<0x124>(v));
  v = fmaxf(v, turned<0x122>(v));
  v = fmaxf(v, turned<0x121>(v));
  return attn::groups_max(v);
}

// ------------------------------------------------------------------ a teacher's distribution
// q = softmax(z / T) over a row's live entries, one wave a row (the maximum is
// taken off before the division, which may pass float32's range). Entries of the
// same candidate are put together in the first of them (the sums over entries
// are the same), so that a candidate is wanted once; the loss of such a row may be
// negative, down to `least`: sum q log q over the entries less that over the
// candidates. A row without a live
// entry has the constant 0 and no targets, one with an index past the table
// NaN and none.
struct TeacherArgs {
  const int64_t *ids;
  const float *logits;
  int64_t N, V;
  int K;
  float temperature;
  int32_t *ids_out;
  float *weight, *konst, *least;
};
__global__ __launch_bounds__(kBlock) void k_teacher(TeacherArgs a) {
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = attn::wave_index();
  int *ids = reinterpret_cast<int *>(lds) + wave * 2 * a.K;
  float *q = reinterpret_cast<float *>(ids + a.K);
  const int64_t n = int64_t(blockIdx.x) * kWaves + wave;
  if (n >= a.N) return;   // (the wave works alone)
  float most = -INFINITY;
  bool past = false;
  for (int k = lane; k < a.K; k += kWave) {
    const int64_t id = a.ids[n * a.K + k];
    const float z = a.logits[n * a.K + k];
    const bool live = id >= 0 && !(z == -INFINITY);
    past |= live && id >= a.V;
    ids[k] = live ? int(min(id, a.V)) : -1;
    q[k] = z;
    if (live) most = fmaxf(most, z);
  }
  most = wave_max(most);
  const bool bad = __any(past);
  float total = 0.f;
  bool any = false;
  for (int k = lane; k < a.K; k += kWave) {
    if (ids[k] < 0) continue;
    any = true;
    total += expf((q[k] - most) / a.temperature);
  }
  total = wave_sum(total);
  const bool live_row = __any(any) && !bad;
  const float log_total = logf(total);
  float konst = 0.f;
  for (int k = lane; k < a.K; k += kWave) {
    if (ids[k] < 0) continue;
    const float z = (q[k] - most) / a.temperature, w = expf(z) / total;
    if (!(w == 0.f)) konst += w * (z - log_total);
    else ids[k] = -1;   // (nothing wanted of it)
    q[k] = w;
  }
  konst = wave_sum(konst);
  attn::wave_sync();
  float together = 0.f;   // sum q log q over the candidates
  bool twice = false;
  for (int k = lane; k < a.K; k += kWave) {
    int id = live_row ? ids[k] : -1;
    float w = 0.f;
    for (int i = 0; i < a.K; ++i) {
      if (ids[i] != id) continue;
      if (i < k) id = -2;   // put together in an earlier entry (no index is -2)
      else w += q[i];
    }
    twice |= id == -2 && ids[k] >= 0;
    if (id >= 0) together += w * logf(w);
    a.ids_out[n * a.K + k] = id < 0 ? -1 : id;
    a.weight[n * a.K + k] = id < 0 ? 0.f : w;
  }
  together = wave_sum(together);
  twice = __any(twice);
  if (lane == 0) {
    a.konst[n] = bad ? NAN : live_row ? konst : 0.f;
    a.least[n] = twice ? konst - together : 0.f;
  }
}

// ------------------------------------------------------------------ the rows with a target first
// order[]: the rows with a target in their order, then the others; live[0]: how
// many have one. A workgroup counts the targets before its 1,024 rows itself
// (8 us for 24,000 rows; two megabytes a workgroup at kOrderMost, beyond which the rows stay as they are).
constexpr int kOrderRows = 1024;
constexpr int64_t kOrderLeast = 1024, kOrderMost = 1 << 18;
__global__ __launch_bounds__(kOrderRows) void k_order(const int64_t *target, int64_t N, int64_t V, int32_t *order,
                                                      int32_t *live) {
  __shared__ int waves[kOrderRows / kWave];
  const int tid = threadIdx.x;
  const int64_t n0 = int64_t(blockIdx.x) * kOrderRows, n = n0 + tid;
  auto has = [&](int64_t at) { return uint64_t(target[at]) < uint64_t(V); };
  int count = 0, total = 0;
#pragma unroll 8
  for (int64_t i = tid; i < N; i += kOrderRows) {
    const int on = has(i) ? 1 : 0;
    total += on;
    if (i < n0) count += on;
  }
  int before, all;
  block_exclusive_scan<int, kOrderRows>(count, waves, before);
  block_exclusive_scan<int, kOrderRows>(total, waves, all);
  const bool here = n < N, on = here && has(n);
  int ignored;
  const int at = before + block_exclusive_scan<int, kOrderRows>(on ? 1 : 0, waves, ignored);
  if (here) order[on ? at : all + (n - at)] = int32_t(n);
  if (n == 0) *live = all;
}

// ------------------------------------------------------------------ joining the pieces
struct FinishArgs {
  Problem p;
  Order order;
  Partials in;
  const int64_t *target;   // [N], or NULL:
  const int32_t *ids;      // [N][K]
  const float *weight, *konst, *least;
  int K;
  float *loss, *stat, *dir;   // stat: [2][N] the maximum and 1 / sum (0: no gradient)
  int32_t *ids_out;           // of `target`
};
constexpr int kAhead = 4;     // partials of a lane

// A lane's four columns of a row of D: 4 lane on, the last lane's the row's
// last four (some of them its neighbour's too: `own` marks those that are not).
struct Cols {
  int d;
  bool here, own[4];
  __device__ __forceinline__ explicit Cols(int D) {
    const int at = 4 * int(threadIdx.x & 63);
    here = at < D;
    d = min(at, D - 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) own[j] = here && d + j >= at;
  }
};

// The row's maximum, sum and direction from its pieces', its targets' scores
// (formed again, in fp32), the loss and what the backward reads. Latency bounds
// it: a row's partials, its own values and its targets' rows are asked for at
// once. W waves a row, 4 / W rows a workgroup; targets in batches of BATCH. One row
// with four waves 8 us (21 with one), 24,000 rows 21 us (33 one load after the other),
// 4,000 rows of 100 targets of 512 bytes 51 us, 4 TB/s.
template <typename T, int W, int BATCH, bool DIR>
__global__ __launch_bounds__(kBlock) void k_finish(FinishArgs a) {
  __shared__ float parts[kWaves][DIR && W > 1 ? kMaxDim : 1];
  __shared__ float sums[2][kWaves][4];
  const Problem &p = a.p;
  const int lane = threadIdx.x & 63, wave = attn::wave_index(), w = wave % W;
  const int64_t at = int64_t(blockIdx.x) * (kWaves / W) + wave / W;
  const bool here = at < p.N;
  const int64_t pos = here ? at : p.N - 1;   // (a row past the end joins the barriers)
  const int64_t row = a.order.row(pos), live_rows = a.order.count(p.N);
  const int64_t target = a.target != nullptr ? a.target[row] : 0;
  const Cols c(p.D);
  T raw[4];
  load_n(raw, static_cast<const T *>(p.h) + row * p.hs + c.d);

  // the row's partials: the waves along the table of consecutive pieces, shared by the row's waves
  int n = 0;
  int64_t first = 0;
  if (pos < live_rows) {
    const Line line((live_rows + a.in.rows - 1) / a.in.rows, a.in.ytiles, a.in.groups);
    const int64_t xt = pos / a.in.rows, w0 = line.group_of(xt * line.inner);
    n = int(line.group_of((xt + 1) * line.inner - 1) - w0 + 1) * a.in.wy;
    first = (w0 + xt) * a.in.wy * a.in.rows + (pos - xt * a.in.rows);
  }
  constexpr bool ROUNDED = DIR && sizeof(T) == 2;
  const float *pm = a.in.m + first, *pl = a.in.l + first, *pr = nullptr;
  int step_r = a.in.rows;   // of the rounded sums
  if constexpr (ROUNDED) {
    if (a.in.ones >= 0) step_r *= a.in.dp;
    pr = a.in.ones >= 0 ? a.in.o + first * a.in.dp + a.in.ones : a.in.r + first;
  }
  // (the first of them at once: their loads, the row's and the targets' overlap)
  float m[kAhead], s[kAhead], rs[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int k = w * kWave + lane + i * (W * kWave);
    m[i] = k < n ? pm[k * a.in.rows] : -INFINITY;
    s[i] = k < n ? pl[k * a.in.rows] : 0.f;
    rs[i] = ROUNDED && k < n ? pr[k * step_r] : 0.f;
  }
  // the first targets' rows
  int id = -1;
  float q = 0.f, b = 0.f, want = 0.f, out = 0.f;
  T y[BATCH][4];
  auto ask = [&](int k0) {
    id = -1;
    q = b = 0.f;
    if (lane < BATCH && k0 + lane < a.K) {
      if (a.target != nullptr) {
        id = uint64_t(target) < uint64_t(p.V) ? int(target) : -1;
        q = 1.f;
      } else {
        id = a.ids[row * a.K + k0 + lane];
        q = a.weight[row * a.K + k0 + lane];
      }
      if (id < 0) q = 0.f;
      else if (p.bias != nullptr) b = bias2(p, id);
    }
    want += q;
    if (b == -INFINITY) {   // left out: its row is not read
      out = 1.f;
      id = -1;
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int v = __builtin_amdgcn_readlane(id, i);
      if (v >= 0) load_n(y[i], static_cast<const T *>(p.table) + int64_t(v) * p.ts + c.d);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j) y[i][j] = T(0.f);
    }
  };
  int k0 = w * BATCH;
  ask(k0);

  // the maximum and the sum of all partials (a piece without a live candidate has sum 0)
  float mx = -INFINITY, l = 0.f, lr = 0.f;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) mx = fmaxf(mx, m[i]);
  for (int k = w * kWave + lane + kAhead * W * kWave; k < n; k += W * kWave) mx = fmaxf(mx, pm[k * a.in.rows]);
  mx = wave_max(mx);
  auto at_max = [&](float y, float z) { return y == -INFINITY ? z : z * exp2_fast(y - mx); };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    l += at_max(m[i], s[i]);
    if constexpr (ROUNDED) lr += at_max(m[i], rs[i]);
  }
  for (int k = w * kWave + lane + kAhead * W * kWave; k < n; k += W * kWave) {
    l += at_max(pm[k * a.in.rows], pl[k * a.in.rows]);
    if constexpr (ROUNDED) lr += at_max(pm[k * a.in.rows], pr[k * step_r]);
  }
  l = wave_sum(l);
  if constexpr (ROUNDED) lr = wave_sum(lr);
  if constexpr (W > 1) {
    if (lane == 0) sums[0][wave][0] = mx, sums[0][wave][1] = l, sums[0][wave][2] = lr;
    __syncthreads();
    mx = -INFINITY;
    l = lr = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) mx = fmaxf(mx, sums[0][i][0]);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      l += at_max(sums[0][i][0], sums[0][i][1]);
      if constexpr (ROUNDED) lr += at_max(sums[0][i][0], sums[0][i][2]);
    }
  }
  if constexpr (!ROUNDED) lr = l;

  // the targets: sum of q (mx - s), of q, of q w; a bias that base 2 takes past float32's range (a mask of its
  // lowest value) goes into a sum of its own, as it is
  float x[4], tw[4], far = 0.f, low = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = c.own[j] ? float(raw[j]) : 0.f;
    tw[j] = 0.f;
  }
  while (true) {
    float dot[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float qi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q), i));
      dot[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float z = c.own[j] ? float(y[i][j]) : 0.f;   // (not 0 times a neighbour's NaN)
        dot[i] = fmaf(x[j], z, dot[i]);
        tw[j] = fmaf(qi, float(y[i][j]), tw[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) dot[i] = wave_sum(dot[i]);
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (lane == i && id >= 0) {
        const bool past = b == -FLT_MAX && mx > -0.99f * FLT_MAX;   // (of rows where it is not every candidate's)
        far += q * (mx - fmaf(dot[i], p.c, past ? 0.f : b));
        if (past) low -= q * p.bias[id];
      }
    k0 += W * BATCH;
    if (k0 >= a.K) break;
    ask(k0);
  }
  far = wave_sum(far);
  low = wave_sum(low);
  want = wave_sum(want);
  out = wave_max(out);
  if constexpr (W > 1) {
    if (lane == 0) sums[1][wave][0] = far, sums[1][wave][1] = want, sums[1][wave][2] = out, sums[1][wave][3] = low;
    __syncthreads();
    far = want = out = low = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i)
      far += sums[1][i][0], want += sums[1][i][1], out = fmaxf(out, sums[1][i][2]), low += sums[1][i][3];
  }
  const bool wanted = !(want == 0.f);   // (NaN: a row that its teacher spoils)
  const bool spoilt = mx == -INFINITY && !(l == 0.f);   // (no score but NaN)
  const bool grad = wanted && out == 0.f;
  if (here && w == 0 && lane == 0) {
    float loss;
    if (!wanted) {
      loss = a.target != nullptr ? (target >= p.V ? NAN : 0.f) : a.konst[row];
    } else if (mx == -INFINITY) {   // no live candidate, or one is wanted whose score is -inf as every other's is
      loss = spoilt || out == 0.f ? NAN : 0.f;
    } else if (out != 0.f) {
      loss = INFINITY;
    } else {
      const float konst = a.target != nullptr ? 0.f : a.konst[row], least = a.target != nullptr ? 0.f : a.least[row];
      loss = konst + kLn2 * (far + want * __builtin_amdgcn_logf(l));
      loss = p.temperature * (p.temperature * loss + low);   // (T^2 may be 0)
      const float bound = p.temperature * (p.temperature * least);
      loss = loss < bound ? bound : loss;   // (rounding: it is not under it)
    }
    a.loss[row] = loss;
    if (a.stat != nullptr) {
      a.stat[row] = grad ? mx : 0.f;
      a.stat[p.N + row] = grad ? 1.f / l : 0.f;
    }
    if (a.ids_out != nullptr) a.ids_out[row] = uint64_t(target) < uint64_t(p.V) ? int32_t(target) : -1;
  }
  if constexpr (DIR) {
    if (W == 1 && !grad) return;   // (not read)
    float o[4] = {};
    const float *src = a.in.o + first * a.in.dp + c.d;
    const int64_t step = int64_t(a.in.rows) * a.in.dp;
#pragma unroll 4
    for (int k = w; k < n; k += W) {
      const float f = at_max(pm[k * a.in.rows], 1.f);
      float z[4];
      load_n(z, src + k * step);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(z[j], f, o[j]);
    }
    float e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = o[j] / lr - tw[j];
    if constexpr (W > 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) parts[wave][4 * lane + j] = e[j];
      __syncthreads();
      if (w != 0) return;
#pragma unroll
      for (int i = 1; i < W; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] += parts[i][4 * lane + j];
    }
    if (here && c.here && grad) store_n(a.dir + row * p.D + c.d, e);
  }
}

// ------------------------------------------------------------------ the gradients' rows
// dh, and the rows' image for the table's gradient, in its order: with `order`
// those that have a target, then tiles filled up.
struct RowArgs {
  Problem p;
  Order order;
  const float *stat, *dir, *g;
  const int32_t *ids;        // [N] of labels, or NULL
  void *dh;                  // or NULL
  char *image;               // or NULL
  Image im;
};
template <typename T>
__global__ __launch_bounds__(kBlock) void k_rows(RowArgs a) {
  const Problem &p = a.p;
  const int lane = threadIdx.x & 63;
  const int64_t pos = int64_t(blockIdx.x) * kWaves + attn::wave_index();
  const bool here = pos < p.N;
  const int64_t n = here ? a.order.row(pos) : 0;
  const float m = here ? a.stat[n] : 0.f, il = here ? a.stat[p.N + n] : 0.f;
  const bool live = !(il == 0.f);
  const float g = live ? a.g[n] * p.temperature : 0.f;
  if (a.image != nullptr) {
    const int64_t tile = pos / a.im.rows;
    const int r = int(pos - tile * a.im.rows);
    char *image = a.image + tile * a.im.bytes;
    T *row = reinterpret_cast<T *>(image) + r * a.im.ld;
    const T *h = static_cast<const T *>(p.h) + n * p.hs;
    const int width = a.im.ld - 16 / int(sizeof(T));   // (the padding is not read)
    if (4 * lane < width) {
      T x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = live && 4 * lane + j < p.D ? h[4 * lane + j] : T(0.f);
      store_n(row + 4 * lane, x);
    }
    if (lane == 0) {
      float *c = reinterpret_cast<float *>(image + a.im.rows * a.im.ld * int(sizeof(T))) + r;
      c[0] = !live ? -INFINITY : m == INFINITY ? NAN : -m;
      c[a.im.rows] = g * il;
      c[2 * a.im.rows] = g;
      reinterpret_cast<int32_t *>(c)[3 * a.im.rows] = live && a.ids != nullptr ? a.ids[n] : -1;
    }
  }
  const Cols c(p.D);
  if (a.dh != nullptr && here && c.here) {
    float e[4] = {};
    if (live) load_n(e, a.dir + n * p.D + c.d);
    T x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = T(live ? g * p.scale * e[j] : 0.f);
    store_n(static_cast<T *>(a.dh) + n * p.D + c.d, x);
  }
}

// ------------------------------------------------------------------ entry points
int make_problem(const sgl_candidates *c, Problem &p) {
  SGL_REQUIRE(c != nullptr, "candidates: NULL problem");
  SGL_REQUIRE(c->dtype >= 0 && c->dtype <= SGL_FP16, "candidates: unknown element type %d", c->dtype);
  const int least = c->dtype == SGL_FP32 ? 4 : 8;
  SGL_REQUIRE(c->dim >= least && c->dim <= kMaxDim, "candidates: rows of %d values (%d to %d)", c->dim, least, kMaxDim);
  // (a workgroup a row where four waves share one: 2^24 of 256 threads make a launch)
  SGL_REQUIRE(c->n >= 0 && c->n <= kMaxRows && c->v > 0 && c->v < INT32_MAX - 512,
              "candidates: %lld rows over %lld candidates are too many (or none)", (long long)c->n, (long long)c->v);
  SGL_REQUIRE(c->h_stride >= 0 && c->table_stride >= 0 && c->h_stride <= kMaxStride && c->table_stride <= kMaxStride,
              "candidates: row strides of %lld and %lld elements (0 to %lld)", (long long)c->h_stride,
              (long long)c->table_stride, (long long)kMaxStride);
  SGL_REQUIRE(c->n == 0 || (c->h != nullptr && c->table != nullptr), "candidates: NULL array");
  SGL_REQUIRE(c->temperature > 0.f && c->temperature < INFINITY && c->scale - c->scale == 0.f,
              "candidates: scale %g, temperature %g", double(c->scale), double(c->temperature));
  p.h = c->h;
  p.table = c->table;
  p.hs = c->h_stride;
  p.ts = c->table_stride;
  p.bias = c->bias;
  p.N = c->n;
  p.V = c->v;
  p.D = c->dim;
  p.scale = c->scale;
  p.temperature = c->temperature;
  p.c = float(double(c->scale) * 1.4426950408889634 / double(c->temperature));
  p.cb = float(1.4426950408889634 / double(c->temperature));
  SGL_REQUIRE(p.c - p.c == 0.f && p.cb < INFINITY && p.temperature * p.temperature < INFINITY,
              "candidates: scale %g over temperature %g is out of range", double(c->scale), double(c->temperature));
  return SGL_OK;
}

Partials carve_forward(void *ws, int32_t dtype, const Problem &p, bool dir, size_t *bytes) {
  Carver c(ws);
  Partials out = forward_shape(dtype, p);
  const size_t pieces = size_t((p.N + out.rows - 1) / out.rows + out.groups) * size_t(out.wy) * size_t(out.rows);
  out.m = c.take<float>(pieces);
  out.l = c.take<float>(pieces);
  out.r = dir && dtype != SGL_FP32 && out.ones < 0 ? c.take<float>(pieces) : nullptr;
  out.o = dir ? c.take<float>(pieces * size_t(out.dp)) : nullptr;
  *bytes = c.used;
  return out;
}

// Rows without a target are set aside where there are rows enough to gain more
// than the launch that orders them costs.
bool orders(int64_t N) { return N >= kOrderLeast && N <= kOrderMost; }

// What the backward reads of the forward (and the forward's own steps of each other).
struct Keep {
  float *stat, *dir, *weight, *konst, *least;
  int32_t *ids, *order;
};
constexpr int32_t kNeedRows = 1, kNeedTable = 2;
Keep carve_keep(void *keep, const Problem &p, int K, bool teacher, int32_t need, size_t *bytes) {
  Carver c(keep);
  Keep k{};
  const size_t n = size_t(p.N), e = n * size_t(K);
  if (need != 0) k.stat = c.take<float>(2 * n);
  if (need & kNeedRows) k.dir = c.take<float>(n * size_t(p.D));
  if (teacher || (need & kNeedTable)) k.ids = c.take<int32_t>(e);
  if (teacher) {
    k.weight = c.take<float>(e);
    k.konst = c.take<float>(n);
    k.least = c.take<float>(n);
  } else if (orders(p.N)) {
    k.order = c.take<int32_t>(n + 1);
  }
  *bytes = c.used;
  return k;
}

struct Grad {
  char *image;
  float *part;
  int32_t *index;
  int2 *entries;
};
Grad carve_backward(void *ws, int32_t dtype, const Problem &p, int K, bool teacher, size_t *bytes) {
  Carver c(ws);
  Grad g{};
  const Image im = grad_image(dtype, p.D);
  const size_t tiles = size_t((p.N + im.rows - 1) / im.rows);
  g.image = c.take<char>(tiles * size_t(im.bytes));
  if (teacher) {
    g.index = c.take<int32_t>(tiles * size_t((p.V + kGradBlock - 1) / kGradBlock + 1));
    g.entries = c.take<int2>(tiles * size_t(im.rows) * size_t(K));
  }
  g.part = c.take<float>(size_t(table_grad_part(dtype, p)));
  *bytes = c.used;
  return g;
}

int check_room(const char *what, const void *room, size_t bytes, size_t need) {
  if (need == 0 || (room != nullptr && bytes >= need)) return SGL_OK;
  sgl::set_error("candidates: %s of %zu bytes, %zu needed", what, room != nullptr ? bytes : 0, need);
  return SGL_ERR_WORKSPACE;
}

template <typename T>
void finish(const FinishArgs &a, hipStream_t stream) {
  // four waves a row where they have partials or targets enough to share
  const bool wide = a.K >= 16 || a.in.wy > 1 || a.p.N <= 16 * a.in.rows;
  const dim3 grid(unsigned(wide ? a.p.N : (a.p.N + kWaves - 1) / kWaves));
  auto go = [&](auto *k) { launch(k, grid, dim3(kBlock), 0, stream, a); };
  auto pick = [&](auto batch) {
    constexpr int B = batch.value;
    if (a.dir != nullptr) wide ? go(&k_finish<T, kWaves, B, true>) : go(&k_finish<T, 1, B, true>);
    else wide ? go(&k_finish<T, kWaves, B, false>) : go(&k_finish<T, 1, B, false>);
  };
  if (a.K == 1) pick(std::integral_constant<int, 1>{});
  else pick(std::integral_constant<int, 8>{});
}

}  // namespace

extern "C" size_t sgl_candidates_keep_bytes(const sgl_candidates *problem, int32_t k, int32_t teacher, int32_t need) {
  Problem p;
  size_t bytes = 0;
  if (make_problem(problem, p) != SGL_OK || k <= 0 || k > kMaxTargets) return 0;
  carve_keep(nullptr, p, k, teacher != 0, need, &bytes);
  return bytes;
}

extern "C" size_t sgl_candidates_workspace_bytes(const sgl_candidates *problem, int32_t k, int32_t teacher,
                                                 int32_t need, int32_t backward) {
  Problem p;
  size_t bytes = 0;
  if (make_problem(problem, p) != SGL_OK || k <= 0 || k > kMaxTargets) return 0;
  if (backward == 0) carve_forward(nullptr, problem->dtype, p, (need & kNeedRows) != 0, &bytes);
  else if (need & kNeedTable) carve_backward(nullptr, problem->dtype, p, k, teacher != 0, &bytes);
  return bytes;
}

extern "C" int sgl_candidates_forward(const sgl_candidates *problem, const int64_t *target, const int64_t *ids,
                                      const float *logits, int32_t k, int32_t need, float *loss, void *keep,
                                      size_t keep_bytes, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  Problem p;
  if (const int rc = make_problem(problem, p)) return rc;
  SGL_REQUIRE(k > 0 && k <= kMaxTargets && (target == nullptr || k == 1), "candidates: %d targets a row", k);
  SGL_REQUIRE(need >= 0 && need <= (kNeedRows | kNeedTable), "candidates: need %d", need);
  if (p.N == 0) return SGL_OK;
  SGL_REQUIRE(loss && (target != nullptr ? ids == nullptr && logits == nullptr : ids != nullptr && logits != nullptr),
              "candidates: NULL array, or labels and a teacher's entries at once");
  const bool teacher = target == nullptr;
  size_t room = 0;
  const Keep kept = carve_keep(keep, p, k, teacher, need, &room);
  if (const int rc = check_room("memory for the backward", keep, keep_bytes, room)) return rc;
  const Partials part = carve_forward(workspace, problem->dtype, p, (need & kNeedRows) != 0, &room);
  if (const int rc = check_room("workspace", workspace, workspace_bytes, room)) return rc;
  if (teacher) {
    const TeacherArgs a{ids, logits, p.N, p.V, k, p.temperature, kept.ids, kept.weight, kept.konst,
                        kept.least};
    sgl::launch(&k_teacher, dim3(unsigned((p.N + kWaves - 1) / kWaves)), dim3(kBlock), size_t(kWaves) * 8 * size_t(k),
                stream, a);
  } else if (kept.order != nullptr) {
    sgl::launch(&k_order, dim3(unsigned((p.N + kOrderRows - 1) / kOrderRows)), dim3(kOrderRows), 0, stream, target, p.N,
                p.V, kept.order, kept.order + p.N);
  }
  const Order o{kept.order, kept.order != nullptr ? kept.order + p.N : nullptr};
  forward_partials(problem->dtype, p, o, part, stream);
  const FinishArgs a{p,          o,          part,       target, teacher ? kept.ids : nullptr,
                     kept.weight, kept.konst, kept.least, k,      loss,
                     kept.stat,   kept.dir,   teacher ? nullptr : kept.ids};
  if (problem->dtype == SGL_FP32) finish<float>(a, stream);
  else if (problem->dtype == SGL_BF16) finish<bf16_t>(a, stream);
  else finish<fp16_t>(a, stream);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

extern "C" int sgl_candidates_backward(const sgl_candidates *problem, int32_t k, int32_t teacher, int32_t need,
                                       const void *keep, size_t keep_bytes, const float *g, void *dh, void *dtable,
                                       float *dbias, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  Problem p;
  if (const int rc = make_problem(problem, p)) return rc;
  SGL_REQUIRE(k > 0 && k <= kMaxTargets && (teacher != 0 || k == 1), "candidates_backward: %d targets a row", k);
  SGL_REQUIRE(need > 0 && need <= (kNeedRows | kNeedTable) && p.N > 0, "candidates_backward: need %d of %lld rows",
              need, (long long)p.N);
  SGL_REQUIRE(g != nullptr && (dh == nullptr || (need & kNeedRows)) && (dtable == nullptr || (need & kNeedTable)) &&
              (dbias == nullptr || dtable != nullptr),
              "candidates_backward: a gradient that the forward did not prepare");
  size_t room = 0;
  const Keep kept = carve_keep(const_cast<void *>(keep), p, k, teacher != 0, need, &room);
  if (const int rc = check_room("memory for the backward", keep, keep_bytes, room)) return rc;
  Grad w{};
  if (dtable != nullptr) {
    w = carve_backward(workspace, problem->dtype, p, k, teacher != 0, &room);
    if (const int rc = check_room("workspace", workspace, workspace_bytes, room)) return rc;
  }
  const Order o{kept.order, kept.order != nullptr ? kept.order + p.N : nullptr};
  const Image im = grad_image(problem->dtype, p.D);
  const int64_t rows = dtable != nullptr ? (p.N + im.rows - 1) / im.rows * im.rows : p.N;
  const RowArgs a{p, o, kept.stat, kept.dir, g, teacher != 0 ? nullptr : kept.ids, dh, w.image, im};
  const dim3 grid(unsigned((rows + kWaves - 1) / kWaves));
  if (problem->dtype == SGL_FP32) sgl::launch(&k_rows<float>, grid, dim3(kBlock), 0, stream, a);
  else if (problem->dtype == SGL_BF16) sgl::launch(&k_rows<bf16_t>, grid, dim3(kBlock), 0, stream, a);
  else sgl::launch(&k_rows<fp16_t>, grid, dim3(kBlock), 0, stream, a);
  if (dtable != nullptr) {
    RowCoef r{w.image, o.live, w.index, w.entries, 0, k};
    if (teacher != 0) {
      r.vblocks = (p.V + kGradBlock - 1) / kGradBlock;
      route_targets(problem->dtype, p, k, kept.ids, kept.weight, w.index, w.entries, stream);
    }
    table_grad(problem->dtype, p, r, dtable, dbias, w.part, stream);
  }
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}
