// The gated residual between two norms, forward and backward.
//
//   y = x + scale * s(gate) * Norm(z; post),   n = Norm(y; pre)
//
// per row of D values: Norm is (t - mean) / sqrt(var + eps) * weight + bias,
// or with rms t / sqrt(mean(t^2) + eps) * weight + bias. The residual stream
// y and the next block's input n come from one pass over x, z and gate.
//
// Bound by its bytes: 5 tensors forward, 8 backward. A row stays in the
// registers of its lanes from the first load to the last store (the
// statistics are two sums over it each, the variance about the mean held in
// fp32), so every tensor is read or written once; n is taken from the fp32 y,
// and each output rounds once. The backward computes the statistics again
// from the tensors it reads anyway, so the forward stores none. The weights'
// gradients are sums over rows: a lane keeps its columns' sums over the rows
// its workgroup walks, and the workgroups' rows of sums are added by
// k_sum_rows in one order. The next row's values are in flight while a row is
// worked on.
//
// Measured: 131073 rows of 512 in fp16, rms: 131 us forward, 208 backward, 5.1
// TB/s both (a copy of 2 GiB reaches 4.9); 24000 rows of 172 in bf16: 19 and 27
// us, 2.4 TB/s, two or three rows a wave; 400 rows of 100 in fp32: 4 us.
#include <climits>

#include "history.h"

namespace {

using sgl::kWave;

constexpr int kMaxD = 8192;

struct NormArgs {
  const void *x, *z, *gate;
  int64_t sx, sz, sg;   // row strides (elements)
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;
  float eps;
  int rms, D;
  int64_t rows;
};

// Sum over the LPR lanes that hold a row, returned to each of them. LPR > 64:
// the whole workgroup, through LDS (every wave calls it).
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float *s_red, int &slot) {
  if constexpr (LPR <= kWave) {
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
  } else {
    constexpr int W = LPR / kWave;
    v = sgl::wave_reduce_sum(v);
    float *s = s_red + slot * W;
    slot ^= 1;   // two areas in turn: one barrier a sum
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) t += s[i];
    return t;
  }
}

// A row's values: vector i of a lane starts at column (i * LPR + lane) * V.
template <typename T, int V, int NV, int LPR>
struct Row {
  static constexpr int E = V * NV;
  static constexpr int RPB = LPR > kWave ? 1 : 256 / LPR;   // rows of a workgroup at a time
  static constexpr int BLOCK = LPR > kWave ? LPR : 256;

  struct Raw {   // as loaded (the next row's, in flight)
    T t[NV][V];
  };
  static __device__ __forceinline__ void load(Raw &r, const T *p, int lane, int D) {   // (NULL reads as 0)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) r.t[i][j] = T(0.f);
      if (p != nullptr && c < D) sgl::load_n(r.t[i], p + c);
    }
  }
  static __device__ __forceinline__ void widen(float (&r)[E], const Raw &x) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) r[i * V + j] = float(x.t[i][j]);
  }
  static __device__ __forceinline__ void store(T *p, const float (&r)[E], int lane, int D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + lane) * V;
      if (c < D) {
        T t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = T(r[i * V + j]);
        sgl::store_n(p + c, t);
      }
    }
  }
  // a weight row (fp32; NULL reads as `none`)
  static __device__ __forceinline__ void weight(float (&r)[E], const float *p, float none, int lane, int D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) r[i * V + j] = p != nullptr && c < D ? p[c + j] : none;
    }
  }
  // t -> its standardised values (columns past D: 0), returns 1 / sqrt(var + eps)
  static __device__ __forceinline__ float standard(float (&t)[E], int lane, int D, float inv, float eps, int rms,
                                                   float *s_red, int &slot) {
    if (!rms) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += t[e];
      const float mean = row_sum<LPR>(s, s_red, slot) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) t[i * V + j] = (i * LPR + lane) * V < D ? t[i * V + j] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) q += t[e] * t[e];
    const float r = rsqrtf(row_sum<LPR>(q, s_red, slot) * inv + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] *= r;
    return r;
  }
  // g (the gradient of the standardised t) -> the gradient of the values
  static __device__ __forceinline__ void through(float (&g)[E], const float (&t)[E], float r, float inv, int rms,
                                                 float *s_red, int &slot) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) b += g[e] * t[e];
    b = row_sum<LPR>(b, s_red, slot) * inv;
    if (!rms) {
#pragma unroll
      for (int e = 0; e < E; ++e) a += g[e];
      a = row_sum<LPR>(a, s_red, slot) * inv;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = r * (g[e] - a - t[e] * b);
  }
};

template <typename T, int V, int NV, int LPR>
__global__ __launch_bounds__((Row<T, V, NV, LPR>::BLOCK)) void k_norm_fwd(NormArgs a, T *__restrict__ y,
                                                                          T *__restrict__ n) {
  using R = Row<T, V, NV, LPR>;
  constexpr int E = R::E;
  __shared__ float s_red[LPR > 64 ? 2 * LPR / 64 : 1];
  int slot = 0;
  const int lane = threadIdx.x % LPR;
  const float inv = 1.f / float(a.D);
  float al[E], pw[E], pb[E], nw[E], nb[E];
  R::weight(al, a.scale, 0.f, lane, a.D);
  R::weight(pw, a.post_w, 1.f, lane, a.D);
  R::weight(pb, a.post_b, 0.f, lane, a.D);
  R::weight(nw, a.pre_w, 1.f, lane, a.D);
  R::weight(nb, a.pre_b, 0.f, lane, a.D);
  const int64_t step = int64_t(gridDim.x) * R::RPB;
  typename R::Raw rx, rz, rg;
  auto fetch = [&](int64_t r) {
    R::load(rz, static_cast<const T *>(a.z) + r * a.sz, lane, a.D);
    R::load(rx, static_cast<const T *>(a.x) + r * a.sx, lane, a.D);
    R::load(rg, static_cast<const T *>(a.gate) + r * a.sg, lane, a.D);
  };
  int64_t r = int64_t(blockIdx.x) * R::RPB + threadIdx.x / LPR;
  if (r < a.rows) fetch(r);
  for (; r < a.rows; r += step) {
    float x[E], z[E], g[E];
    R::widen(z, rz);
    R::widen(x, rx);
    R::widen(g, rg);
    if (r + step < a.rows) fetch(r + step);
    R::standard(z, lane, a.D, inv, a.eps, a.rms, s_red, slot);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float s, sn;
      sgl::sigmoid_pair(g[e], s, sn);
      x[e] += al[e] * s * (z[e] * pw[e] + pb[e]);
    }
    R::store(y + r * a.D, x, lane, a.D);
    R::standard(x, lane, a.D, inv, a.eps, a.rms, s_red, slot);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * nw[e] + nb[e];
    R::store(n + r * a.D, x, lane, a.D);
  }
}

// part: this workgroup's sums, [5][D]: scale, post weight, pre weight, post
// bias, pre bias (the biases' rows only with biases).
// (three waves a SIMD where a lane holds 8 columns: 168 registers, a few of them
// spilled, 206 us where two waves take 230 at 131073 x 512)
template <typename T, int V, int NV, int LPR, bool BIAS>
__global__ __launch_bounds__((Row<T, V, NV, LPR>::BLOCK), (LPR <= 256 && V * NV == 8 && !BIAS ? 3 : 1)) void k_norm_bwd(NormArgs a, const T *__restrict__ gy,
                                                                          const T *__restrict__ gn,
                                                                          T *__restrict__ dx, T *__restrict__ dz,
                                                                          T *__restrict__ dgate,
                                                                          float *__restrict__ part) {
  using R = Row<T, V, NV, LPR>;
  constexpr int E = R::E;
  __shared__ float s_red[LPR > 64 ? 2 * LPR / 64 : 1];
  int slot = 0;
  const int lane = threadIdx.x % LPR;
  const float inv = 1.f / float(a.D);
  constexpr int NS = BIAS ? 5 : 3;   // sums kept
  float al[E], pw[E], pb[E], nw[E];
  R::weight(al, a.scale, 0.f, lane, a.D);
  R::weight(pw, a.post_w, 1.f, lane, a.D);
  R::weight(pb, BIAS ? a.post_b : nullptr, 0.f, lane, a.D);
  R::weight(nw, a.pre_w, 1.f, lane, a.D);
  float sums[NS][E];
#pragma unroll
  for (int k = 0; k < NS; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) sums[k][e] = 0.f;
  const int64_t step = int64_t(gridDim.x) * R::RPB;
  typename R::Raw rx, rz, rg, ru, rq;
  auto fetch = [&](int64_t r) {
    R::load(rx, static_cast<const T *>(a.x) + r * a.sx, lane, a.D);
    R::load(rz, static_cast<const T *>(a.z) + r * a.sz, lane, a.D);
    R::load(rg, static_cast<const T *>(a.gate) + r * a.sg, lane, a.D);
    R::load(ru, gn != nullptr ? gn + r * a.D : nullptr, lane, a.D);
    R::load(rq, gy != nullptr ? gy + r * a.D : nullptr, lane, a.D);
  };
  int64_t r = int64_t(blockIdx.x) * R::RPB + threadIdx.x / LPR;
  if (r < a.rows) fetch(r);
  for (; r < a.rows; r += step) {
    float x[E], z[E], g[E], q[E], u[E];
    R::widen(x, rx);
    R::widen(z, rz);
    R::widen(g, rg);
    R::widen(u, ru);
    R::widen(q, rq);
    if (r + step < a.rows) fetch(r + step);
    // y again
    const float zr = R::standard(z, lane, a.D, inv, a.eps, a.rms, s_red, slot);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float s, sn;
      sgl::sigmoid_pair(g[e], s, sn);
      x[e] += al[e] * s * (z[e] * pw[e] + pb[e]);
    }
    const float yr = R::standard(x, lane, a.D, inv, a.eps, a.rms, s_red, slot);
    // the pre norm
#pragma unroll
    for (int e = 0; e < E; ++e) {
      sums[2][e] += u[e] * x[e];
      if constexpr (BIAS) sums[4][e] += u[e];
      u[e] *= nw[e];
    }
    R::through(u, x, yr, inv, a.rms, s_red, slot);
    // the residual, the gate and the scale
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] += u[e];
    R::store(dx + r * a.D, q, lane, a.D);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float s, sn;
      sgl::sigmoid_pair(g[e], s, sn);
      const float post = z[e] * pw[e] + pb[e], qs = q[e] * s;
      sums[0][e] += qs * post;
      const float dpost = qs * al[e];
      g[e] = dpost * post * sn;
      sums[1][e] += dpost * z[e];
      if constexpr (BIAS) sums[3][e] += dpost;
      u[e] = dpost * pw[e];
    }
    R::store(dgate + r * a.D, g, lane, a.D);
    R::through(u, z, zr, inv, a.rms, s_red, slot);
    R::store(dz + r * a.D, u, lane, a.D);
  }
  // the workgroup's rows (RPB of them at a time) into one row of sums
  if constexpr (R::RPB > 1) {
    __shared__ float s_sum[R::RPB * LPR * E];
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) s_sum[(threadIdx.x / LPR) * (LPR * E) + e * LPR + lane] = sums[k][e];
      __syncthreads();
      for (int c = threadIdx.x; c < LPR * E; c += R::BLOCK) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < R::RPB; ++g) t += s_sum[g * (LPR * E) + c];
        const int e = c / LPR, col = ((e / V) * LPR + c % LPR) * V + e % V;
        if (col < a.D) part[(int64_t(blockIdx.x) * NS + k) * a.D + col] = t;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (i * LPR + lane) * V + j;
          if (c < a.D) part[(int64_t(blockIdx.x) * NS + k) * a.D + c] = sums[k][i * V + j];
        }
    }
  }
}

constexpr unsigned kBwdGrid = 1024;   // most rows of partial sums

// As many workgroups as are resident at once (each walks rows at that stride):
// with more of them the last ones run alone (131073 rows of 512 in fp16: a
// grid of 1.5 times that takes 142 and 249 us, this one 128 and 207).
template <typename K>
unsigned norm_grid(K kernel, int block, int64_t rows, int rpb, unsigned most) {
  constexpr int kCUs = 256;
  int each = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, block, 0) != hipSuccess || each < 1) each = 2;
  return unsigned(std::max<int64_t>(1, std::min<int64_t>({(rows + rpb - 1) / rpb, int64_t(most), int64_t(each) * kCUs})));
}

template <typename T, int V, int NV, int LPR>
int run_norm(const NormArgs &a, const void *gy, const void *gn, void *o1, void *o2, void *o3, float *part, int nsum,
             bool back, hipStream_t s) {
  using R = Row<T, V, NV, LPR>;
  if (!back) {
    const unsigned most = norm_grid(&k_norm_fwd<T, V, NV, LPR>, R::BLOCK, a.rows, R::RPB, UINT_MAX);
    sgl::launch(&k_norm_fwd<T, V, NV, LPR>, dim3(most), dim3(R::BLOCK), 0, s, a, static_cast<T *>(o1),
                static_cast<T *>(o2));
    return 0;
  }
  const auto kernel = nsum == 5 ? &k_norm_bwd<T, V, NV, LPR, true> : &k_norm_bwd<T, V, NV, LPR, false>;
  const unsigned grid = norm_grid(kernel, R::BLOCK, a.rows, R::RPB, kBwdGrid);
  sgl::launch(kernel, dim3(grid), dim3(R::BLOCK), 0, s, a, static_cast<const T *>(gy), static_cast<const T *>(gn),
              static_cast<T *>(o1), static_cast<T *>(o2), static_cast<T *>(o3), part);
  return int(grid);
}

// Lanes a row: as few as hold it in one vector each; beyond 256 of them a
// workgroup of 1,024 threads. That is made for vectors of 4 and 8: a width of
// 257 that divides by neither leaves three quarters of it idle (93,385 rows in
// bf16: 642 us forward and 1,486 backward, where 256 columns take 49 and 99; 1,001
// columns 195 and 433, 1,000 57 and 141).
template <typename T, int V>
int pick_norm(const NormArgs &a, const void *gy, const void *gn, void *o1, void *o2, void *o3, float *part, int nsum,
              bool back, hipStream_t s) {
  const int u = (a.D + V - 1) / V;
  if (u <= 16) return run_norm<T, V, 1, 16>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (u <= 32) return run_norm<T, V, 1, 32>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (u <= 64) return run_norm<T, V, 1, 64>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (u <= 128) return run_norm<T, V, 1, 128>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (u <= 256) return run_norm<T, V, 1, 256>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (u <= 1024) return run_norm<T, V, 1, 1024>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (V > 1 || u <= 2048) return run_norm<T, V, 2, 1024>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  return run_norm<T, V, V == 1 ? 8 : 2, 1024>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
}

// 16 bytes (fp32: 4 elements) a lane where the columns divide, else 4 or 1
// elements; any row stride and alignment.
template <typename T>
int pick_vec(const NormArgs &a, const void *gy, const void *gn, void *o1, void *o2, void *o3, float *part, int nsum,
             bool back, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (a.D % 8 == 0) return pick_norm<T, 8>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  }
  if (a.D % 4 == 0) return pick_norm<T, 4>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  return pick_norm<T, 1>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
}

int pick_type(int dtype, const NormArgs &a, const void *gy, const void *gn, void *o1, void *o2, void *o3, float *part,
              int nsum, bool back, hipStream_t s) {
  if (dtype == SGL_FP32) return pick_vec<float>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  if (dtype == SGL_BF16) return pick_vec<sgl::bf16_t>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
  return pick_vec<sgl::fp16_t>(a, gy, gn, o1, o2, o3, part, nsum, back, s);
}

int check_norm(int32_t dtype, int64_t rows, int32_t D, const NormArgs &a) {
  SGL_REQUIRE(dtype >= 0 && dtype <= SGL_FP16, "gated_norm: unknown element type %d", dtype);
  SGL_REQUIRE(rows >= 0 && D > 0 && D <= kMaxD, "gated_norm: %lld rows of %d values (1 to %d)", (long long)rows, D,
              kMaxD);
  SGL_REQUIRE(a.sx >= 0 && a.sz >= 0 && a.sg >= 0, "gated_norm: negative row stride");
  SGL_REQUIRE(rows == 0 || (a.x && a.z && a.gate && a.scale), "gated_norm: NULL array");
  return SGL_OK;
}

}  // namespace

extern "C" size_t sgl_gated_norm_workspace_bytes(int64_t rows, int32_t D) {
  if (rows <= 0 || D <= 0) return 0;
  return sizeof(float) * 5 * size_t(D) * std::min<size_t>(size_t(rows), kBwdGrid);
}

extern "C" int sgl_gated_norm_forward(int32_t dtype, int64_t rows, int32_t D, const void *x, int64_t sx,
                                      const void *z, int64_t sz, const void *gate, int64_t sg, const float *scale,
                                      const float *post_w, const float *post_b, const float *pre_w,
                                      const float *pre_b, float eps, int32_t rms, void *y, void *n,
                                      hipStream_t stream) {
  const NormArgs a{x, z, gate, sx, sz, sg, scale, post_w, post_b, pre_w, pre_b, eps, rms, D, rows};
  if (const int rc = check_norm(dtype, rows, D, a)) return rc;
  if (rows == 0) return SGL_OK;
  SGL_REQUIRE(y && n, "gated_norm: NULL array");
  pick_type(dtype, a, nullptr, nullptr, y, n, nullptr, nullptr, 0, false, stream);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

extern "C" int sgl_gated_norm_backward(int32_t dtype, int64_t rows, int32_t D, const void *x, int64_t sx,
                                       const void *z, int64_t sz, const void *gate, int64_t sg, const float *scale,
                                       const float *post_w, const float *post_b, const float *pre_w,
                                       const float *pre_b, float eps, int32_t rms, const void *gy, const void *gn,
                                       void *dx, void *dz, void *dgate, float *dparams, int32_t nsum,
                                       void *workspace, size_t workspace_bytes, hipStream_t stream) {
  const NormArgs a{x, z, gate, sx, sz, sg, scale, post_w, post_b, pre_w, pre_b, eps, rms, D, rows};
  if (const int rc = check_norm(dtype, rows, D, a)) return rc;
  SGL_REQUIRE(nsum == 3 || nsum == 5, "gated_norm_backward: %d parameter gradients (3 or 5)", nsum);
  // (the form of 3 has no biases in its y)
  SGL_REQUIRE(nsum == 5 || (post_b == nullptr && pre_b == nullptr), "gated_norm_backward: biases need 5 parameter gradients");
  SGL_REQUIRE(dparams != nullptr, "gated_norm_backward: NULL array");
  if (rows > 0) {
    SGL_REQUIRE(dx && dz && dgate, "gated_norm_backward: NULL array");
    if (workspace_bytes < sgl_gated_norm_workspace_bytes(rows, D) || workspace == nullptr) {
      sgl::set_error("gated_norm_backward: workspace of %zu bytes, %zu needed", workspace_bytes,
                     sgl_gated_norm_workspace_bytes(rows, D));
      return SGL_ERR_WORKSPACE;
    }
  }
  int grid = 0;
  if (rows > 0)
    grid = pick_type(dtype, a, gy, gn, dx, dz, dgate, static_cast<float *>(workspace), nsum, true, stream);
  sgl::sum_rows(static_cast<const float *>(workspace), grid, nsum * D, dparams, stream);   // (no rows: zeros)
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}
