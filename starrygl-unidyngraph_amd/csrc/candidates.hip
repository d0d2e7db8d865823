// Losses over all candidates: what joins the pieces of the forward, a
// teacher's distribution, the rows' coefficients for the gradients, and the
// entry points.
#include "candidates.h"

namespace {

using namespace sgl;
using namespace sgl::cand;

// Sum over the wave, the same in every lane.
__device__ __forceinline__ float wave_sum(float v) { return wave_reduce_sum(v); }
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
  return v;
}

// ------------------------------------------------------------------ a teacher's distribution
// q = softmax(z / T) over a row's live entries, one wave a row. Entries of the
// same candidate are put together in the first of them (the sums over entries
// are the same), so that a candidate is wanted once. A row without a live
// entry has the constant 0 and no targets, one with an index past the table
// NaN and none.
struct TeacherArgs {
  const int64_t *ids;
  const float *logits;
  int64_t N, V;
  int K;
  float temperature;
  int32_t *ids_out;
  float *weight, *konst;
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
    const float z = a.logits[n * a.K + k] / a.temperature;
    const bool live = id >= 0 && !(z == -INFINITY);
    past |= id >= a.V;
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
    total += expf(q[k] - most);
  }
  total = wave_sum(total);
  const bool live_row = __any(any) && !bad;
  const float log_total = logf(total);
  float konst = 0.f;
  for (int k = lane; k < a.K; k += kWave) {
    if (ids[k] < 0) continue;
    const float z = q[k] - most, w = expf(z) / total;
    if (!(w == 0.f)) konst += w * (z - log_total);
    else ids[k] = -1;   // (nothing wanted of it)
    q[k] = w;
  }
  konst = wave_sum(konst);
  attn::wave_sync();
  for (int k = lane; k < a.K; k += kWave) {
    int id = live_row ? ids[k] : -1;
    float w = 0.f;
    for (int i = 0; i < a.K; ++i) {
      if (ids[i] != id) continue;
      if (i < k) id = -2;   // put together in an earlier entry (no index is -2)
      else w += q[i];
    }
    a.ids_out[n * a.K + k] = id < 0 ? -1 : id;
    a.weight[n * a.K + k] = id < 0 ? 0.f : w;
  }
  if (lane == 0) a.konst[n] = bad ? NAN : live_row ? konst : 0.f;
}

// ------------------------------------------------------------------ joining the pieces
struct FinishArgs {
  Problem p;
  Partials in;
  const int64_t *target;   // [N], or NULL:
  const int32_t *ids;      // [N][K]
  const float *weight, *konst;
  int K;
  float *loss, *stat, *dir;   // stat: [2][N] the maximum and 1 / sum (0: no gradient)
  int32_t *ids_out;           // of `target`
};
constexpr int kCols = kMaxDim / kWave;   // columns of a lane

// W waves a row, 4 / W rows a workgroup.
template <typename T, int W, bool DIR>
__global__ __launch_bounds__(kBlock) void k_finish(FinishArgs a) {
  __shared__ float parts[kWaves][DIR ? kMaxDim : 1];
  __shared__ float sums[kWaves];
  __shared__ int outs[kWaves];
  const Problem &p = a.p;
  const int lane = threadIdx.x & 63, wave = attn::wave_index(), w = wave % W;
  const int64_t n = int64_t(blockIdx.x) * (kWaves / W) + wave / W;
  const bool here = n < p.N;
  const int64_t row = here ? n : p.N - 1;   // (a row past the end joins the barriers)
  const T *h = static_cast<const T *>(p.h) + row * p.hs;

  float mx = -INFINITY;
  for (int64_t s = lane; s < a.in.splits; s += kWave) mx = fmaxf(mx, a.in.m[s * p.N + row]);
  mx = wave_max(mx);
  float l = 0.f;
  for (int64_t s = lane; s < a.in.splits; s += kWave) {
    const float m = a.in.m[s * p.N + row];
    // (a piece without a live candidate has sum 0)
    l += m == -INFINITY ? a.in.l[s * p.N + row] : a.in.l[s * p.N + row] * exp2_fast(m - mx);
  }
  l = wave_sum(l);

  // the targets: sum of q (mx - s), and of q w
  float x[kCols], tw[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    const int d = lane + kWave * j;
    x[j] = d < p.D ? float(h[d]) : 0.f;
    tw[j] = 0.f;
  }
  float far = 0.f, want = 0.f;
  bool out = false;
  for (int k = w; k < a.K; k += W) {
    int64_t id;
    float q = 1.f;
    if (a.target != nullptr) {
      id = a.target[row];
      if (id >= p.V) id = -1;
    } else {
      id = a.ids[row * a.K + k];
      q = a.weight[row * a.K + k];
    }
    if (id < 0) continue;
    const float b = p.bias != nullptr ? bias2(p, id) : 0.f;
    want += q;
    if (b == -INFINITY) {   // left out: its row is not read
      out = true;
      continue;
    }
    const T *t = static_cast<const T *>(p.table) + id * p.ts;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int d = lane + kWave * j;
      const float y = d < p.D ? float(t[d]) : 0.f;
      dot = fmaf(x[j], y, dot);
      tw[j] = fmaf(q, y, tw[j]);
    }
    far += q * (mx - fmaf(wave_sum(dot), p.c, b));
  }
  if constexpr (W > 1) {
    if (lane == 0) sums[wave] = far, outs[wave] = out;
    __syncthreads();
    far = 0.f;
    out = false;
#pragma unroll
    for (int i = 0; i < W; ++i) far += sums[i], out |= outs[i] != 0;
    __syncthreads();
    if (lane == 0) sums[wave] = want;
    __syncthreads();
    want = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) want += sums[i];
  }
  const bool wanted = !(want == 0.f);   // (NaN: a row that its teacher spoils)
  const bool live = wanted && !out && mx > -INFINITY;
  if (here && w == 0 && lane == 0) {
    float loss;
    if (!wanted) {
      loss = a.target != nullptr ? (a.target[n] >= p.V ? NAN : 0.f) : a.konst[n];
    } else if (mx == -INFINITY) {
      loss = l == 0.f ? 0.f : NAN;   // no live candidate (or only NaN)
    } else if (out) {
      loss = INFINITY;
    } else {
      const float konst = a.target != nullptr ? 0.f : a.konst[n];
      loss = p.temperature * p.temperature * (konst + kLn2 * (far + want * __builtin_amdgcn_logf(l)));
      loss = loss < 0.f ? 0.f : loss;   // (rounding: it is not negative)
    }
    a.loss[n] = loss;
    if (a.stat != nullptr) {
      const bool grad = live || (wanted && !out && l != 0.f);   // (NaN scores alone: NaN gradients)
      a.stat[n] = grad ? mx : 0.f;
      a.stat[p.N + n] = grad ? 1.f / l : 0.f;
    }
    if (a.ids_out != nullptr) {
      const int64_t t = a.target[n];
      a.ids_out[n] = t >= 0 && t < p.V ? int32_t(t) : -1;
    }
  }
  if constexpr (DIR) {
    float o[kCols] = {};
    const int64_t step = p.N * a.in.dp;
    const float *src = a.in.o + row * a.in.dp;
    for (int64_t s = w; s < a.in.splits; s += W) {
      const float m = a.in.m[s * p.N + row];
      const float f = m == -INFINITY ? 1.f : exp2_fast(m - mx);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int d = lane + kWave * j;
        if (d < p.D) o[j] = fmaf(src[s * step + d], f, o[j]);
      }
    }
    const bool grad = live || (wanted && !out && l != 0.f);
    if constexpr (W > 1) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) parts[wave][lane + kWave * j] = o[j] / l - tw[j];
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int d = lane + kWave * j;
      float e = o[j] / l - tw[j];
      if constexpr (W > 1) {
        if (w != 0) continue;
#pragma unroll
        for (int i = 1; i < W; ++i) e += parts[i][d];
      }
      if (here && d < p.D) a.dir[n * p.D + d] = grad ? e : 0.f;
    }
  }
}

// ------------------------------------------------------------------ the gradients' rows
struct RowArgs {
  Problem p;
  const float *stat, *dir, *g;
  void *dh;                  // or NULL
  float *nm, *gl, *gq;       // or NULL
};
template <typename T>
__global__ __launch_bounds__(kBlock) void k_rows(RowArgs a) {
  const Problem &p = a.p;
  const int lane = threadIdx.x & 63;
  const int64_t n = int64_t(blockIdx.x) * kWaves + attn::wave_index();
  if (n >= p.N) return;
  const float m = a.stat[n], il = a.stat[p.N + n];
  const bool live = !(il == 0.f);
  const float g = live ? a.g[n] * p.temperature : 0.f;
  if (a.nm != nullptr && lane == 0) {
    a.nm[n] = !live ? -INFINITY : m == INFINITY ? NAN : -m;
    a.gl[n] = g * il;
    a.gq[n] = g;
  }
  if (a.dh != nullptr)
    for (int d = lane; d < p.D; d += kWave)
      static_cast<T *>(a.dh)[n * p.D + d] = T(live ? g * p.scale * a.dir[n * p.D + d] : 0.f);
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
  SGL_REQUIRE(c->h_stride >= 0 && c->table_stride >= 0, "candidates: negative row stride");
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
  return SGL_OK;
}

Partials carve_forward(void *ws, int32_t dtype, const Problem &p, bool dir, size_t *bytes) {
  Carver c(ws);
  Partials out{};
  out.splits = forward_splits(dtype, p, dir);
  out.dp = padded_dim(p.D);
  out.m = c.take<float>(size_t(out.splits) * size_t(p.N));
  out.l = c.take<float>(size_t(out.splits) * size_t(p.N));
  out.o = dir ? c.take<float>(size_t(out.splits) * size_t(p.N) * size_t(out.dp)) : nullptr;
  *bytes = c.used;
  return out;
}

struct Grad {
  float *nm, *gl, *gq, *part;
  int64_t splits;
};
Grad carve_backward(void *ws, int32_t dtype, const Problem &p, size_t *bytes) {
  Carver c(ws);
  Grad g{};
  g.nm = c.take<float>(size_t(p.N));
  g.gl = c.take<float>(size_t(p.N));
  g.gq = c.take<float>(size_t(p.N));
  g.splits = table_grad_splits(dtype, p);
  g.part = g.splits > 1 ? c.take<float>(size_t(g.splits) * size_t(p.V) * size_t(padded_dim(p.D) + 1)) : nullptr;
  *bytes = c.used;
  return g;
}

template <typename T>
void finish(const FinishArgs &a, hipStream_t stream) {
  // four waves a row where they have pieces or targets enough to share
  const bool wide = a.in.splits >= 16 || a.K >= 16;
  const dim3 grid(unsigned(wide ? a.p.N : (a.p.N + kWaves - 1) / kWaves));
  if (a.dir != nullptr) {
    if (wide) launch(&k_finish<T, kWaves, true>, grid, dim3(kBlock), 0, stream, a);
    else launch(&k_finish<T, 1, true>, grid, dim3(kBlock), 0, stream, a);
  } else {
    if (wide) launch(&k_finish<T, kWaves, false>, grid, dim3(kBlock), 0, stream, a);
    else launch(&k_finish<T, 1, false>, grid, dim3(kBlock), 0, stream, a);
  }
}

}  // namespace

extern "C" int sgl_candidates_teacher(int64_t n, int32_t k, int64_t v, const int64_t *ids, const float *logits,
                                      float temperature, int32_t *ids_out, float *weight, float *konst,
                                      hipStream_t stream) {
  SGL_REQUIRE(n >= 0 && n <= kMaxRows && v > 0 && v < INT32_MAX - 512 && k > 0 && k <= kMaxTargets,
              "candidates_teacher: %lld rows of %d entries (1 to %d)", (long long)n, k, kMaxTargets);
  SGL_REQUIRE(temperature > 0.f && temperature < INFINITY, "candidates_teacher: temperature %g", double(temperature));
  if (n == 0) return SGL_OK;
  SGL_REQUIRE(ids && logits && ids_out && weight && konst, "candidates_teacher: NULL array");
  const TeacherArgs a{ids, logits, n, v, k, temperature, ids_out, weight, konst};
  sgl::launch(&k_teacher, dim3(unsigned((n + kWaves - 1) / kWaves)), dim3(kBlock), size_t(kWaves) * 8 * size_t(k), stream,
         a);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

extern "C" size_t sgl_candidates_workspace_bytes(const sgl_candidates *problem, int32_t what) {
  Problem p;
  if (make_problem(problem, p) != SGL_OK || p.N == 0) return 0;
  size_t bytes = 0;
  if (what == 2) carve_backward(nullptr, problem->dtype, p, &bytes);
  else carve_forward(nullptr, problem->dtype, p, what == 1, &bytes);
  return bytes;
}

extern "C" int sgl_candidates_forward(const sgl_candidates *problem, const int64_t *target, const int32_t *ids,
                                      const float *weight, const float *konst, int32_t k, float *loss, float *stat,
                                      float *dir, int32_t *ids_out, void *workspace, size_t workspace_bytes,
                                      hipStream_t stream) {
  Problem p;
  if (const int rc = make_problem(problem, p)) return rc;
  SGL_REQUIRE(k > 0 && k <= kMaxTargets && (target == nullptr || k == 1), "candidates_forward: %d targets a row", k);
  if (p.N == 0) return SGL_OK;
  SGL_REQUIRE(loss && (target != nullptr ? ids == nullptr : ids && weight && konst && !ids_out),
              "candidates_forward: NULL array, or labels and a teacher's entries at once");
  SGL_REQUIRE(dir == nullptr || stat != nullptr, "candidates_forward: dir without stat");
  size_t need = 0;
  const Partials part = carve_forward(workspace, problem->dtype, p, dir != nullptr, &need);
  if (workspace == nullptr || workspace_bytes < need) {
    sgl::set_error("candidates_forward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  forward_partials(problem->dtype, p, part, dir != nullptr, stream);
  const FinishArgs a{p, part, target, ids, weight, konst, k, loss, stat, dir, ids_out};
  if (problem->dtype == SGL_FP32) finish<float>(a, stream);
  else if (problem->dtype == SGL_BF16) finish<bf16_t>(a, stream);
  else finish<fp16_t>(a, stream);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

extern "C" int sgl_candidates_backward(const sgl_candidates *problem, const float *stat, const int32_t *ids,
                                       const float *weight, int32_t k, const float *dir, const float *g, void *dh,
                                       void *dtable, float *dbias, void *workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
  Problem p;
  if (const int rc = make_problem(problem, p)) return rc;
  SGL_REQUIRE(k > 0 && k <= kMaxTargets, "candidates_backward: %d targets a row", k);
  SGL_REQUIRE(p.N > 0, "candidates_backward: no rows");
  SGL_REQUIRE(stat && g && (dh == nullptr || dir) && (dtable == nullptr || ids), "candidates_backward: NULL array");
  SGL_REQUIRE(dbias == nullptr || dtable != nullptr, "candidates_backward: dbias without dtable");
  Grad w{};
  if (dtable != nullptr) {
    size_t need = 0;
    w = carve_backward(workspace, problem->dtype, p, &need);
    if (workspace == nullptr || workspace_bytes < need) {
      sgl::set_error("candidates_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
      return SGL_ERR_WORKSPACE;
    }
  }
  const RowArgs a{p, stat, dir, g, dh, w.nm, w.gl, w.gq};
  const dim3 grid(unsigned((p.N + kWaves - 1) / kWaves));
  if (problem->dtype == SGL_FP32) sgl::launch(&k_rows<float>, grid, dim3(kBlock), 0, stream, a);
  else if (problem->dtype == SGL_BF16) sgl::launch(&k_rows<bf16_t>, grid, dim3(kBlock), 0, stream, a);
  else sgl::launch(&k_rows<fp16_t>, grid, dim3(kBlock), 0, stream, a);
  if (dtable != nullptr) {
    const RowCoef r{w.nm, w.gl, w.gq, ids, weight, k};
    table_grad(problem->dtype, p, r, dtable, dbias, w.part, w.splits, stream);
  }
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}
