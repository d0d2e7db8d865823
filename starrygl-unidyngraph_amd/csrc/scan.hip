// The gated linear recurrence over windows of events, forward and backward.
//
// Per channel d of sequence n, over its events t = 0 .. lens[n]-1:
//   a_t = s(gate_t) exp(-decay[d] gaps_t),   h_t = a_t h_{t-1} + (1 - a_t) value_t
// from h_{-1} = state (or 0); without decay a_t = s(gate_t). 1 - a_t is formed
// as s(-gate) + s(gate) (1 - exp(-u)), whose terms are both positive, so it
// keeps its digits where a_t is next to one.
//
// The adjoint runs the other way: lam_t = gh_t + a_{t+1} lam_{t+1}, and
//   dvalue = (1 - a) lam,  dlog = lam (h_{t-1} - value) a,
//   dgate = dlog s(-gate),  ddecay = -sum dlog gaps,  dstate = a_0 lam_0.
//
// Bound by its bytes (two tensors read, one written; backward three read, two
// written). A thread owns V neighbouring channels of one sequence, and the
// threads of a wave neighbouring channels, so each step is one contiguous
// access. States stay in fp32 registers. Both directions are chains in t, so
// a sequence is cut into chunks where there are too few channels to fill the
// GPU: a first kernel gives each chunk's composition (A, B) of h -> A h + B, and
// the second forms each chunk's starting state from those before it and
// walks its chunk. The forward keeps the state in fp32 at every kKeep-th
// step; the backward walks blocks of kKeep steps last to first, computing a
// block's states again in registers from the kept one, so it neither reads
// the (rounded) outputs nor differentiates through their rounding.
#include <climits>

#include "history.h"

namespace {

constexpr int kBlock = 256;
constexpr int kKeep = 16;            // steps between kept states
constexpr int64_t kFill = 1 << 18;   // threads that fill the GPU: 16 waves a CU
constexpr int kMaxChunks = 64;
constexpr int kMinChunk = 64;        // steps (a multiple of kKeep)

struct ScanArgs {
  const void *gate, *value;
  int64_t gate_n, gate_t, value_n, value_t;   // strides (elements)
  const int32_t *lens;
  const float *state;   // [N, D]
  const float *gaps;    // [N, L], strides gaps_n, gaps_t
  int64_t gaps_n, gaps_t;
  const float *decay;   // [D]
  int64_t N, L;
  int D, chunks;
  int64_t clen;         // steps a chunk (a multiple of kKeep)
};

// a and 1 - a of one step
template <bool DECAY>
__device__ __forceinline__ void step_gate(float f, float u, float &a, float &b, float &sn) {
  float s;
  sgl::sigmoid_pair(f, s, sn);
  if constexpr (DECAY) {
    // 1 - exp(-u): the series where exp(-u) is near one
    const float e = __expf(-u);
    const float p = u * (1.f - u * (0.5f - u * (1.f / 6 - u * (1.f / 24 - u * (1.f / 120 - u * (1.f / 720))))));
    const float less = fabsf(u) < 0.25f ? p : 1.f - e;
    a = s * e;
    b = sn + s * less;
  } else {
    a = s;
    b = sn;
  }
}

__device__ __forceinline__ int64_t seq_len(const ScanArgs &a, int64_t n) {
  if (a.lens == nullptr) return a.L;
  return min(max(int64_t(a.lens[n]), int64_t(0)), a.L);
}

// Units: (sequence, channel group, chunk), the channel group fastest, so that
// a wave's accesses are contiguous; chunks before sequences.
struct Unit {
  int64_t n;
  int d, chunk;
};
template <int V>
__device__ __forceinline__ Unit unit_of(const ScanArgs &a, int64_t i) {
  const int dv = (a.D + V - 1) / V;
  Unit u;
  const int64_t q = i / dv;
  u.d = int(i - q * dv) * V;
  u.n = q / a.chunks;
  u.chunk = int(q - u.n * a.chunks);
  return u;
}

// The compositions of each chunk: forward (A = prod a, B = the state it ends
// in from 0), or backward (B = a_0 lam_0 of the chunk from nothing after it).
template <typename T, int V, bool DECAY, bool BACK>
__global__ __launch_bounds__(kBlock) void k_scan_chunks(ScanArgs a, const T *__restrict__ gh, float *__restrict__ comp) {
  const int64_t units = a.N * a.chunks * ((a.D + V - 1) / V);
  const int64_t i = int64_t(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= units) return;
  const Unit u = unit_of<V>(a, i);
  const int64_t len = seq_len(a, u.n);
  const int64_t t0 = u.chunk * a.clen, t1 = min(t0 + a.clen, len);
  const T *gate = static_cast<const T *>(a.gate) + u.n * a.gate_n + u.d;
  const T *src = BACK ? gh + u.n * a.L * a.D + u.d : static_cast<const T *>(a.value) + u.n * a.value_n + u.d;
  const int64_t src_t = BACK ? a.D : a.value_t;
  float A[V], B[V], dec[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    A[j] = 1.f;
    B[j] = 0.f;
    dec[j] = DECAY ? a.decay[u.d + j] : 0.f;
  }
  constexpr int U = 8;
  for (int64_t t = t0; t < t1; t += U) {
    T f[U][V], x[U][V];
    float gap[U];
    const int m = int(min(int64_t(U), t1 - t));
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t at = BACK ? t1 - 1 - (t - t0) - min(k, m - 1) : t + min(k, m - 1);
      sgl::load_n(f[k], gate + at * a.gate_t);
      if (BACK && gh == nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[k][j] = T(0.f);
      } else {
        sgl::load_n(x[k], src + at * src_t);
      }
      gap[k] = DECAY ? a.gaps[u.n * a.gaps_n + at * a.gaps_t] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k < m) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float ga, gb, sn;
          step_gate<DECAY>(float(f[k][j]), dec[j] * gap[k], ga, gb, sn);
          A[j] *= ga;
          B[j] = BACK ? ga * (float(x[k][j]) + B[j]) : ga * B[j] + gb * float(x[k][j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float2 c = make_float2(A[j], B[j]);
    *reinterpret_cast<float2 *>(comp + 2 * ((u.n * a.chunks + u.chunk) * a.D + u.d + j)) = c;
  }
}

// Forward: h (all L steps; zero past the length), the last state, and the
// kept states (keep may be NULL).
template <typename T, int V, bool DECAY>
__global__ __launch_bounds__(kBlock) void k_scan_fwd(ScanArgs a, const float *__restrict__ comp, T *__restrict__ h,
                                                     float *__restrict__ last, float *__restrict__ keep) {
  const int64_t units = a.N * a.chunks * ((a.D + V - 1) / V);
  const int64_t i = int64_t(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= units) return;
  const Unit u = unit_of<V>(a, i);
  const int64_t len = seq_len(a, u.n);
  const int64_t t0 = u.chunk * a.clen, t1 = min(t0 + a.clen, a.L), live = min(t1, len);
  const T *gate = static_cast<const T *>(a.gate) + u.n * a.gate_n + u.d;
  const T *value = static_cast<const T *>(a.value) + u.n * a.value_n + u.d;
  T *out = h + u.n * a.L * a.D + u.d;
  const int64_t keeps = (a.L + kKeep - 1) / kKeep;
  float s[V], dec[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s[j] = a.state != nullptr ? a.state[u.n * a.D + u.d + j] : 0.f;
    dec[j] = DECAY ? a.decay[u.d + j] : 0.f;
  }
  for (int c = 0; c < u.chunk; ++c) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 p = *reinterpret_cast<const float2 *>(comp + 2 * ((u.n * a.chunks + c) * a.D + u.d + j));
      s[j] = p.x * s[j] + p.y;
    }
  }
  constexpr int U = 8;
  static_assert(kKeep % U == 0, "kept states fall on the first step of a group");
  for (int64_t t = t0; t < t1; t += U) {
    if (t < live) {
      if (keep != nullptr && t % kKeep == 0) sgl::store_n(keep + (u.n * keeps + t / kKeep) * a.D + u.d, s);
      T f[U][V], x[U][V];
      float gap[U];
      const int m = int(min(int64_t(U), live - t));
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t at = t + min(k, m - 1);
        sgl::load_n(f[k], gate + at * a.gate_t);
        sgl::load_n(x[k], value + at * a.value_t);
        gap[k] = DECAY ? a.gaps[u.n * a.gaps_n + at * a.gaps_t] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (t + k < t1) {
          T o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float ga, gb, sn;
            step_gate<DECAY>(float(f[k][j]), dec[j] * gap[k], ga, gb, sn);
            if (k < m) s[j] = ga * s[j] + gb * float(x[k][j]);
            o[j] = k < m ? T(s[j]) : T(0.f);
          }
          sgl::store_n(out + (t + k) * a.D, o);
        }
      }
    } else {
      T o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = T(0.f);
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (t + k < t1) sgl::store_n(out + (t + k) * a.D, o);
    }
  }
  // the chunk that holds the last event (the first one of an empty sequence)
  if (last != nullptr && (len > t0 ? len <= t0 + a.clen : len == 0 && u.chunk == 0))
    sgl::store_n(last + u.n * a.D + u.d, s);
}

// Backward: thread g of `groups` walks the sequences g, g + groups, ... of its
// channels (all its chunks' work units), so that decay's gradient is one row
// of partial sums a group.
template <typename T, int V, bool DECAY>
__global__ __launch_bounds__(kBlock) void k_scan_bwd(ScanArgs a, const float *__restrict__ comp,
                                                     const float *__restrict__ keep, const T *__restrict__ gh,
                                                     const float *__restrict__ glast, T *__restrict__ dgate,
                                                     T *__restrict__ dvalue, float *__restrict__ dstate,
                                                     float *__restrict__ part, int64_t groups) {
  const int dv = (a.D + V - 1) / V;
  const int64_t i = int64_t(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= groups * dv) return;
  const int64_t g = i / dv;
  const int d = int(i - g * dv) * V;
  const int64_t keeps = (a.L + kKeep - 1) / kKeep;
  float dec[V], dsum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    dec[j] = DECAY ? a.decay[d + j] : 0.f;
    dsum[j] = 0.f;
  }
  for (int64_t w = g; w < a.N * a.chunks; w += groups) {
    const int64_t n = w / a.chunks;
    const int chunk = int(w - n * a.chunks);
    const int64_t len = seq_len(a, n);
    const int64_t t0 = chunk * a.clen, t1 = min(t0 + a.clen, a.L), live = min(t1, len);
    const T *gate = static_cast<const T *>(a.gate) + n * a.gate_n + d;
    const T *value = static_cast<const T *>(a.value) + n * a.value_n + d;
    const int64_t row0 = n * a.L * a.D + d;
    float c[V];   // a_{t+1} lam_{t+1}
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = glast != nullptr ? glast[n * a.D + d + j] : 0.f;
    for (int k = a.chunks - 1; k > chunk; --k) {
      if (k * a.clen >= len) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 p = *reinterpret_cast<const float2 *>(comp + 2 * ((n * a.chunks + k) * a.D + d + j));
        c[j] = p.x * c[j] + p.y;
      }
    }
    T zero[V];
#pragma unroll
    for (int j = 0; j < V; ++j) zero[j] = T(0.f);
    for (int64_t t = max(t0, live); t < t1; ++t) {
      sgl::store_n(dgate + row0 + t * a.D, zero);
      sgl::store_n(dvalue + row0 + t * a.D, zero);
    }
    if (live > t0) {
      for (int64_t b = (live - 1) / kKeep * kKeep; b >= t0; b -= kKeep) {
        T f[kKeep][V], x[kKeep][V], gr[kKeep][V];
        float gap[kKeep], s[V];
        const int m = int(min(int64_t(kKeep), live - b));
        sgl::load_n(s, keep + (n * keeps + b / kKeep) * a.D + d);
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
          const int64_t at = b + min(k, m - 1);
          sgl::load_n(f[k], gate + at * a.gate_t);
          sgl::load_n(x[k], value + at * a.value_t);
          if (gh != nullptr) {
            sgl::load_n(gr[k], gh + row0 + at * a.D);
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) gr[k][j] = T(0.f);
          }
          gap[k] = DECAY ? a.gaps[n * a.gaps_n + at * a.gaps_t] : 0.f;
        }
        float before[kKeep][V];   // the state each step meets
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            before[k][j] = s[j];
            float ga, gb, sn;
            step_gate<DECAY>(float(f[k][j]), dec[j] * gap[k], ga, gb, sn);
            s[j] = ga * s[j] + gb * float(x[k][j]);
          }
#pragma unroll
        for (int k = kKeep - 1; k >= 0; --k) {
          if (k < m) {
            T og[V], ov[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              float ga, gb, sn;
              step_gate<DECAY>(float(f[k][j]), dec[j] * gap[k], ga, gb, sn);
              const float lam = float(gr[k][j]) + c[j];
              const float dlog = lam * (before[k][j] - float(x[k][j])) * ga;
              c[j] = ga * lam;
              og[j] = T(dlog * sn);
              ov[j] = T(gb * lam);
              if (DECAY) dsum[j] -= dlog * gap[k];
            }
            sgl::store_n(dgate + row0 + (b + k) * a.D, og);
            sgl::store_n(dvalue + row0 + (b + k) * a.D, ov);
          }
        }
      }
    }
    if (dstate != nullptr && chunk == 0) sgl::store_n(dstate + n * a.D + d, c);
  }
  if (DECAY) sgl::store_n(part + g * a.D + d, dsum);
}

// Chunks a sequence: one where the channels alone fill the GPU, else as many
// as do, of at least kMinChunk steps each.
int scan_chunks(int64_t N, int64_t L, int64_t dv) {
  const int64_t want = (kFill + N * dv - 1) / (N * dv);
  return int(std::max<int64_t>(1, std::min<int64_t>({want, L / kMinChunk, int64_t(kMaxChunks)})));
}
int64_t chunk_len(int64_t L, int chunks) {
  const int64_t c = (L + chunks - 1) / chunks;
  return (c + kKeep - 1) / kKeep * kKeep;
}
int scan_vec(int32_t dtype, int32_t D) { return dtype != SGL_FP32 && D % 2 == 0 ? 2 : 1; }

int64_t bwd_groups(int64_t N, int chunks, int64_t dv) {
  return std::max<int64_t>(1, std::min<int64_t>(N * chunks, (kFill + dv - 1) / dv));
}

struct ScanPlan {
  int vec, chunks;
  int64_t clen, comp, groups;   // comp: floats of the compositions
};
ScanPlan scan_plan(int32_t dtype, int64_t N, int64_t L, int32_t D) {
  ScanPlan p;
  p.vec = scan_vec(dtype, D);
  const int64_t dv = (D + p.vec - 1) / p.vec;
  p.chunks = scan_chunks(N, L, dv);
  p.clen = chunk_len(L, p.chunks);
  p.chunks = int((L + p.clen - 1) / p.clen);
  p.comp = p.chunks > 1 ? 2 * N * p.chunks * D : 0;
  p.groups = bwd_groups(N, p.chunks, dv);
  return p;
}

template <typename T, int V, bool DECAY>
void scan_fwd(const ScanArgs &a, float *comp, void *h, float *last, float *keep, hipStream_t s) {
  const int64_t units = a.N * a.chunks * ((a.D + V - 1) / V);
  const dim3 grid(unsigned((units + kBlock - 1) / kBlock));
  if (a.chunks > 1)
    sgl::launch(&k_scan_chunks<T, V, DECAY, false>, grid, dim3(kBlock), 0, s, a, static_cast<const T *>(nullptr), comp);
  sgl::launch(&k_scan_fwd<T, V, DECAY>, grid, dim3(kBlock), 0, s, a, static_cast<const float *>(comp),
              static_cast<T *>(h), last, keep);
}

template <typename T, int V, bool DECAY>
void scan_bwd(const ScanArgs &a, float *comp, const float *keep, const void *gh, const float *glast, void *dgate,
              void *dvalue, float *dstate, float *ddecay, float *part, int64_t groups, hipStream_t s) {
  const int64_t dv = (a.D + V - 1) / V, units = a.N * a.chunks * dv;
  if (a.chunks > 1)
    sgl::launch(&k_scan_chunks<T, V, DECAY, true>, dim3(unsigned((units + kBlock - 1) / kBlock)), dim3(kBlock), 0, s,
                a, static_cast<const T *>(gh), comp);
  sgl::launch(&k_scan_bwd<T, V, DECAY>, dim3(unsigned((groups * dv + kBlock - 1) / kBlock)), dim3(kBlock), 0, s, a,
              static_cast<const float *>(comp), keep, static_cast<const T *>(gh), glast, static_cast<T *>(dgate),
              static_cast<T *>(dvalue), dstate, part, groups);
  if (DECAY) sgl::sum_rows(part, groups, a.D, ddecay, s);
}

template <typename F>
void by_type(int32_t dtype, int vec, bool decay, F f) {
  auto go = [&](auto t, auto v) {
    if (decay) f(t, v, std::true_type{});
    else f(t, v, std::false_type{});
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  if (dtype == SGL_FP32) go(float{}, I1{});
  else if (dtype == SGL_BF16 && vec == 2) go(sgl::bf16_t{}, I2{});
  else if (dtype == SGL_BF16) go(sgl::bf16_t{}, I1{});
  else if (vec == 2) go(sgl::fp16_t{}, I2{});
  else go(sgl::fp16_t{}, I1{});
}

int check_scan(int32_t dtype, int64_t N, int64_t L, int32_t D, const ScanArgs &a) {
  SGL_REQUIRE(dtype >= 0 && dtype <= SGL_FP16, "gated_scan: unknown element type %d", dtype);
  SGL_REQUIRE(N >= 0 && L >= 0 && D > 0 && N < INT_MAX && L < INT_MAX, "gated_scan: bad sizes");
  SGL_REQUIRE(N * D < int64_t(INT_MAX) * (kBlock / 2), "gated_scan: %lld sequences of %d channels are too many",
              (long long)N, D);
  SGL_REQUIRE((a.gaps == nullptr) == (a.decay == nullptr), "gated_scan: give both gaps and decay or neither");
  SGL_REQUIRE(N == 0 || L == 0 || (a.gate && a.value), "gated_scan: NULL array");
  return SGL_OK;
}

}  // namespace

extern "C" int64_t sgl_gated_scan_keep_elems(int64_t N, int64_t L, int32_t D) {
  return N * ((L + kKeep - 1) / kKeep) * D;
}

extern "C" size_t sgl_gated_scan_workspace_bytes(int32_t dtype, int64_t N, int64_t L, int32_t D, int32_t backward,
                                                 int32_t decay) {
  if (N <= 0 || L <= 0 || D <= 0) return 0;
  const ScanPlan p = scan_plan(dtype, N, L, D);
  size_t b = sgl::align_up(sizeof(float) * size_t(p.comp));
  if (backward && decay) b += sizeof(float) * size_t(p.groups) * size_t(D);
  return b;
}

extern "C" int sgl_gated_scan_forward(int32_t dtype, int64_t N, int64_t L, int32_t D, const void *gate,
                                      int64_t gate_n, int64_t gate_t, const void *value, int64_t value_n,
                                      int64_t value_t, const int32_t *lens, const float *state, const float *gaps,
                                      int64_t gaps_n, int64_t gaps_t, const float *decay, void *h, float *last,
                                      float *keep, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  ScanArgs a{gate, value, gate_n, gate_t, value_n, value_t, lens, state, gaps, gaps_n, gaps_t, decay, N, L, D, 1, L};
  if (const int rc = check_scan(dtype, N, L, D, a)) return rc;
  if (N == 0 || L == 0) return SGL_OK;
  SGL_REQUIRE(h != nullptr, "gated_scan: NULL array");
  const ScanPlan p = scan_plan(dtype, N, L, D);
  const size_t need = sgl_gated_scan_workspace_bytes(dtype, N, L, D, 0, 0);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    sgl::set_error("gated_scan: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  a.chunks = p.chunks;
  a.clen = p.clen;
  by_type(dtype, p.vec, decay != nullptr, [&](auto t, auto v, auto dec) {
    scan_fwd<decltype(t), decltype(v)::value, decltype(dec)::value>(a, static_cast<float *>(workspace), h, last, keep,
                                                                    stream);
  });
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}

extern "C" int sgl_gated_scan_backward(int32_t dtype, int64_t N, int64_t L, int32_t D, const void *gate,
                                       int64_t gate_n, int64_t gate_t, const void *value, int64_t value_n,
                                       int64_t value_t, const int32_t *lens, const float *state, const float *gaps,
                                       int64_t gaps_n, int64_t gaps_t, const float *decay, const float *keep,
                                       const void *gh, const float *glast, void *dgate, void *dvalue, float *dstate,
                                       float *ddecay, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  ScanArgs a{gate, value, gate_n, gate_t, value_n, value_t, lens, state, gaps, gaps_n, gaps_t, decay, N, L, D, 1, L};
  if (const int rc = check_scan(dtype, N, L, D, a)) return rc;
  if (N == 0 || L == 0) return SGL_OK;
  SGL_REQUIRE(keep && dgate && dvalue && (decay == nullptr || ddecay != nullptr), "gated_scan_backward: NULL array");
  const ScanPlan p = scan_plan(dtype, N, L, D);
  const size_t need = sgl_gated_scan_workspace_bytes(dtype, N, L, D, 1, decay != nullptr);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    sgl::set_error("gated_scan_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  a.chunks = p.chunks;
  a.clen = p.clen;
  float *comp = static_cast<float *>(workspace);
  float *part = reinterpret_cast<float *>(static_cast<char *>(workspace) + sgl::align_up(sizeof(float) * size_t(p.comp)));
  by_type(dtype, p.vec, decay != nullptr, [&](auto t, auto v, auto dec) {
    scan_bwd<decltype(t), decltype(v)::value, decltype(dec)::value>(a, comp, keep, gh, glast, dgate, dvalue, dstate,
                                                                    ddecay, part, p.groups, stream);
  });
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}
