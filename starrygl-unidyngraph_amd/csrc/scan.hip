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
// where the channels alone are too few to fill the GPU a sequence is cut into
// up to kMaxSupers * kSubs pieces: a first kernel forms each piece's
// composition (A, B) of h -> A h + B and, in LDS, those of the pieces before
// it in its workgroup; the second kernel forms a piece's starting state from
// the workgroups' compositions and its own prefix, and walks its piece.
// The forward keeps the state in fp32 at every kKeep-th step; the backward
// walks blocks of kKeep steps last to first, computing a block's states again
// in registers from the kept one, so it neither reads the (rounded) outputs
// nor differentiates through their rounding; the block before is in flight
// meanwhile (without that 217 us where it is now 122).
//
// Measured, bf16: 8000 windows of up to 32 x 172 with decay 74 us forward and
// 122 backward (3.2 TB/s both; a copy reaches 4.9); 16 x 8191 x 256 25 + 37
// and 35 + 64 us (pieces + walk; the inputs are read twice). One event of 400
// x 100 in fp32: 4 us, a launch.
#include <climits>

#include "history.h"

namespace {

constexpr int kBlock = 256;
constexpr int kKeep = 8;             // steps between kept states
constexpr int64_t kFill = 1 << 18;   // threads that fill the GPU: 16 waves a CU (the backward holds 8 at a time)
// pieces x channel groups: two rounds of the backward's workgroups (16 x 8191 x
// 256 in bf16, both directions: 160 us; 1.25 kFill 170, 0.75 kFill 183)
constexpr int64_t kPieces = 2 * kFill;
constexpr int kSubs = 8;             // pieces a workgroup of the cut form: kLanes channel groups each
constexpr int kLanes = kBlock / kSubs;
constexpr int kMaxSupers = 32;
constexpr int kMinPiece = 32;        // steps (a multiple of kKeep)

struct ScanArgs {
  const void *gate, *value;
  int64_t gate_n, gate_t, value_n, value_t;   // strides (elements)
  const int32_t *lens;
  const float *state;   // [N, D]
  const float *gaps;    // [N, L], strides gaps_n, gaps_t
  int64_t gaps_n, gaps_t;
  const float *decay;   // [D]
  int64_t N, L;
  int D;
  int supers;           // workgroups along a sequence (0: sequences whole, channels side by side)
  int64_t piece;        // steps a piece (a multiple of kKeep)
  float2 *sup, *sub;    // compositions: [N][supers][D], [N][supers][kSubs][D] (those before it in its workgroup)
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

// What a thread walks: V channels from d of sequence n, steps [t0, t1) of it.
struct Unit {
  int64_t n, t0, t1;
  int d, super, sub;
  bool ok;
};
template <int V>
__device__ __forceinline__ Unit unit_of(const ScanArgs &a) {
  const int dv = (a.D + V - 1) / V;
  Unit u;
  if (a.supers == 0) {   // whole sequences: (n, d) side by side
    const int64_t i = int64_t(blockIdx.x) * kBlock + threadIdx.x;
    if (blockIdx.x < (1u << 24)) {   // (a 64-bit division is a long sequence of instructions)
      const uint32_t n = uint32_t(i) / uint32_t(dv);
      u.n = n;
      u.d = int(uint32_t(i) - n * uint32_t(dv)) * V;
    } else {
      u.n = i / dv;
      u.d = int(i - u.n * dv) * V;
    }
    u.super = u.sub = 0;
    u.t0 = 0;
    u.t1 = a.L;
    u.ok = u.n < a.N;
  } else {   // a workgroup: kLanes channel groups x kSubs pieces
    const int blocks = (dv + kLanes - 1) / kLanes;
    const uint32_t i = blockIdx.x / uint32_t(blocks), cb = blockIdx.x - i * uint32_t(blocks);
    const uint32_t n = i / uint32_t(a.supers);
    u.super = int(i - n * uint32_t(a.supers));
    u.n = n;
    u.sub = threadIdx.x / kLanes;
    u.d = int(cb * kLanes + threadIdx.x % kLanes) * V;
    u.t0 = min((int64_t(u.super) * kSubs + u.sub) * a.piece, a.L);
    u.t1 = min(u.t0 + a.piece, a.L);
    u.ok = u.d < a.D;
  }
  return u;
}
template <int V>
__device__ __forceinline__ int64_t comp_at(const ScanArgs &a, const Unit &u, int super) {
  return (u.n * a.supers + super) * a.D + u.d;
}
// s -> A s + B
template <int V>
__device__ __forceinline__ void compose(float (&s)[V], const float2 *__restrict__ p) {
  float2 c[V];
  __builtin_memcpy(c, p, sizeof(c));
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = c[j].x * s[j] + c[j].y;
}

// The address of one step after another: a pointer moved by a stride, or left
// (a step past the last one reads that again). A product a step of 64 bits cost
// more than the step's own arithmetic.
template <typename T>
struct Steps {
  const T *p;
  int64_t by;
  __device__ __forceinline__ Steps(const T *base, int64_t t, int64_t stride) : p(base + t * stride), by(stride) {}
  __device__ __forceinline__ void next(bool go) { p += go ? by : 0; }
};

// The compositions of the pieces: forward (A = prod a, B = the state a piece
// ends in from 0), or backward (B = a_0 lam_0 of the piece from nothing after
// it), combined over the pieces before it (forward) or after it (backward) in
// the workgroup; the workgroup's own into sup.
template <typename T, int V, bool DECAY, bool BACK>
__global__ __launch_bounds__(kBlock) void k_scan_pieces(ScanArgs a, const T *__restrict__ gh) {
  __shared__ float2 comp[kSubs][kLanes * V];
  const Unit u = unit_of<V>(a);
  float A[V], B[V], dec[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    A[j] = 1.f;
    B[j] = 0.f;
    dec[j] = DECAY && u.ok ? a.decay[u.d + j] : 0.f;
  }
  if (u.ok) {
    const int64_t t0 = u.t0, t1 = min(u.t1, seq_len(a, u.n));
    const T *gate = static_cast<const T *>(a.gate) + u.n * a.gate_n + u.d;
    const T *src = BACK ? (gh != nullptr ? gh + u.n * a.L * a.D + u.d : nullptr) : static_cast<const T *>(a.value) + u.n * a.value_n + u.d;
    const int64_t src_t = BACK ? a.D : a.value_t;
    constexpr int U = 8;
    Steps<T> pf(gate, t0, a.gate_t), px(src, t0, src_t);
    Steps<float> pg(DECAY ? a.gaps + u.n * a.gaps_n : nullptr, t0, a.gaps_t);
    for (int64_t t = t0; t < t1; t += U) {
      T f[U][V], x[U][V];
      float gap[U];
      const int m = int(min(int64_t(U), t1 - t));
#pragma unroll
      for (int k = 0; k < U; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[k][j] = T(0.f);
        sgl::load_n(f[k], pf.p);
        if (!BACK || gh != nullptr) sgl::load_n(x[k], px.p);
        gap[k] = DECAY ? *pg.p : 0.f;
        pf.next(k + 1 < m);
        if (!BACK || gh != nullptr) px.next(k + 1 < m);
        if (DECAY) pg.next(k + 1 < m);
      }
      pf.next(m == U);   // (a last short group is not followed)
      if (!BACK || gh != nullptr) px.next(m == U);
      if (DECAY) pg.next(m == U);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (k < m) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float ga, gb, sn;
            step_gate<DECAY>(float(f[k][j]), dec[j] * gap[k], ga, gb, sn);
            A[j] *= ga;
            // (backward too in the order of the steps: a step's gradient goes through every a before it)
            B[j] = BACK ? B[j] + A[j] * float(x[k][j]) : ga * B[j] + gb * float(x[k][j]);
          }
        }
      }
    }
  }
  const int l = (threadIdx.x % kLanes) * V;
#pragma unroll
  for (int j = 0; j < V; ++j) comp[u.sub][l + j] = make_float2(A[j], B[j]);
  __syncthreads();
  if (!u.ok) return;
  float pa[V], pb[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    pa[j] = 1.f;
    pb[j] = 0.f;
  }
  for (int i = 0; i < (BACK ? kSubs - 1 - u.sub : u.sub); ++i) {
    const int from = BACK ? kSubs - 1 - i : i;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 c = comp[from][l + j];
      pa[j] *= c.x;
      pb[j] = c.x * pb[j] + c.y;
    }
  }
  float2 o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = make_float2(pa[j], pb[j]);
  sgl::store_n(a.sub + ((u.n * a.supers + u.super) * kSubs + u.sub) * a.D + u.d, o);
  if (u.sub == (BACK ? 0 : kSubs - 1)) {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = make_float2(A[j] * pa[j], A[j] * pb[j] + B[j]);
    sgl::store_n(a.sup + comp_at<V>(a, u, u.super), o);
  }
}

// Forward: h (all L steps; zero past the length), the last state, and the
// kept states (keep may be NULL).
template <typename T, int V, bool DECAY>
__global__ __launch_bounds__(kBlock) void k_scan_fwd(ScanArgs a, T *__restrict__ h, float *__restrict__ last,
                                                     float *__restrict__ keep) {
  const Unit u = unit_of<V>(a);
  if (!u.ok) return;
  const int64_t len = seq_len(a, u.n);
  const int64_t t0 = u.t0, t1 = u.t1, live = min(t1, len);
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
  if (a.supers > 0) {
    for (int c = 0; c < u.super; ++c) compose(s, a.sup + comp_at<V>(a, u, c));
    compose(s, a.sub + ((u.n * a.supers + u.super) * kSubs + u.sub) * a.D + u.d);
  }
  constexpr int U = 8;
  static_assert(kKeep % U == 0, "kept states fall on the first step of a group");
  Steps<T> pf(gate, t0, a.gate_t), px(value, t0, a.value_t);
  Steps<float> pg(DECAY ? a.gaps + u.n * a.gaps_n : nullptr, t0, a.gaps_t);
  for (int64_t t = t0; t < t1; t += U) {
    if (t < live) {
      if (keep != nullptr && t % kKeep == 0) sgl::store_n(keep + (u.n * keeps + t / kKeep) * a.D + u.d, s);
      T f[U][V], x[U][V];
      float gap[U];
      const int m = int(min(int64_t(U), live - t));
#pragma unroll
      for (int k = 0; k < U; ++k) {
        sgl::load_n(f[k], pf.p);
        sgl::load_n(x[k], px.p);
        gap[k] = DECAY ? *pg.p : 0.f;
        pf.next(k + 1 < m);
        px.next(k + 1 < m);
        if (DECAY) pg.next(k + 1 < m);
      }
      pf.next(m == U);   // (a last short group is not followed)
      px.next(m == U);
      if (DECAY) pg.next(m == U);
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
  // the piece that holds the last event (the first one of an empty sequence)
  if (last != nullptr && (len > 0 ? len > t0 && len <= t1 : t0 == 0)) sgl::store_n(last + u.n * a.D + u.d, s);
}

// One piece's adjoint, from c = a_{t+1} lam_{t+1} after it; c becomes a_0 lam_0 of
// its first step, dsum gathers decay's gradient.
template <typename T, int V, bool DECAY>
__device__ __forceinline__ void walk_back(const ScanArgs &a, const Unit &u, int64_t len, const float (&dec)[V],
                                          const float *__restrict__ keep, const T *__restrict__ gh,
                                          T *__restrict__ dgate, T *__restrict__ dvalue, float (&c)[V],
                                          float (&dsum)[V]) {
  const int64_t t0 = u.t0, t1 = u.t1, live = min(t1, len);
  const int64_t keeps = (a.L + kKeep - 1) / kKeep;
  const T *gate = static_cast<const T *>(a.gate) + u.n * a.gate_n + u.d;
  const T *value = static_cast<const T *>(a.value) + u.n * a.value_n + u.d;
  const int64_t row0 = u.n * a.L * a.D + u.d;
  T zero[V];
#pragma unroll
  for (int j = 0; j < V; ++j) zero[j] = T(0.f);
  for (int64_t t = max(t0, live); t < t1; ++t) {
    sgl::store_n(dgate + row0 + t * a.D, zero);
    sgl::store_n(dvalue + row0 + t * a.D, zero);
  }
  if (live <= t0) return;
  // a block as loaded: the one before it is in flight while one is walked
  T f[kKeep][V], x[kKeep][V], gr[kKeep][V];
  float gap[kKeep], s[V];
  auto fetch = [&](int64_t b, int m) {
    Steps<T> pf(gate, b, a.gate_t), px(value, b, a.value_t), ph(gh != nullptr ? gh + row0 : nullptr, b, a.D);
    Steps<float> pg(DECAY ? a.gaps + u.n * a.gaps_n : nullptr, b, a.gaps_t);
    sgl::load_n(s, keep + (u.n * keeps + b / kKeep) * a.D + u.d);
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      sgl::load_n(f[k], pf.p);
      sgl::load_n(x[k], px.p);
#pragma unroll
      for (int j = 0; j < V; ++j) gr[k][j] = zero[j];
      if (gh != nullptr) sgl::load_n(gr[k], ph.p);
      gap[k] = DECAY ? *pg.p : 0.f;
      pf.next(k + 1 < m);
      px.next(k + 1 < m);
      if (gh != nullptr) ph.next(k + 1 < m);
      if (DECAY) pg.next(k + 1 < m);
    }
  };
  int64_t b = (live - 1) / kKeep * kKeep;
  int m = int(live - b);
  fetch(b, m);
  for (;;) {
    // forward through the block: a, 1 - a, and the factors lam meets
    float ga[kKeep][V], gb[kKeep][V], wl[kKeep][V], wg[kKeep][V], gn[kKeep];
    T gl[kKeep][V];
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float sn;
        step_gate<DECAY>(float(f[k][j]), dec[j] * gap[k], ga[k][j], gb[k][j], sn);
        const float xv = float(x[k][j]);
        wl[k][j] = (s[j] - xv) * ga[k][j];   // d log a
        wg[k][j] = wl[k][j] * sn;            // d gate
        s[j] = ga[k][j] * s[j] + gb[k][j] * xv;
        gl[k][j] = gr[k][j];
      }
      gn[k] = gap[k];
    }
    const int64_t at = row0 + b * a.D;
    const int now = m;
    const bool more = b - kKeep >= t0;
    if (more) {
      b -= kKeep;
      m = kKeep;
      fetch(b, m);
    }
#pragma unroll
    for (int k = kKeep - 1; k >= 0; --k) {
      if (k < now) {
        T og[V], ov[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float lam = float(gl[k][j]) + c[j];
          c[j] = ga[k][j] * lam;
          og[j] = T(lam * wg[k][j]);
          ov[j] = T(lam * gb[k][j]);
          if (DECAY) dsum[j] -= lam * wl[k][j] * gn[k];
        }
        sgl::store_n(dgate + at + k * a.D, og);
        sgl::store_n(dvalue + at + k * a.D, ov);
      }
    }
    if (!more) return;
  }
}

// Backward. Whole sequences: thread group g of `groups` walks the sequences g,
// g + groups, ... of its channels, so that decay's gradient is one row of
// partial sums a group. Cut: a workgroup's pieces, one row a workgroup.
template <typename T, int V, bool DECAY>
__global__ __launch_bounds__(kBlock) void k_scan_bwd(ScanArgs a, const float *__restrict__ keep,
                                                     const T *__restrict__ gh, const float *__restrict__ glast,
                                                     T *__restrict__ dgate, T *__restrict__ dvalue,
                                                     float *__restrict__ dstate, float *__restrict__ part,
                                                     int64_t groups) {
  Unit u = unit_of<V>(a);
  float dec[V], dsum[V], c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    dec[j] = DECAY && u.ok ? a.decay[u.d + j] : 0.f;
    dsum[j] = 0.f;
  }
  if (a.supers == 0) {
    const int64_t g = u.n;
    if (g >= groups) return;
    for (u.n = g; u.n < a.N; u.n += groups) {
#pragma unroll
      for (int j = 0; j < V; ++j) c[j] = glast != nullptr ? glast[u.n * a.D + u.d + j] : 0.f;
      walk_back<T, V, DECAY>(a, u, seq_len(a, u.n), dec, keep, gh, dgate, dvalue, c, dsum);
      if (dstate != nullptr) sgl::store_n(dstate + u.n * a.D + u.d, c);
    }
    if (DECAY) sgl::store_n(part + g * a.D + u.d, dsum);
    return;
  }
  if (u.ok) {
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = glast != nullptr ? glast[u.n * a.D + u.d + j] : 0.f;
    for (int k = a.supers - 1; k > u.super; --k) compose(c, a.sup + comp_at<V>(a, u, k));
    compose(c, a.sub + ((u.n * a.supers + u.super) * kSubs + u.sub) * a.D + u.d);
    walk_back<T, V, DECAY>(a, u, seq_len(a, u.n), dec, keep, gh, dgate, dvalue, c, dsum);
    if (dstate != nullptr && u.t0 == 0 && u.super == 0 && u.sub == 0) sgl::store_n(dstate + u.n * a.D + u.d, c);
  }
  if (DECAY) {
    __shared__ float sums[kSubs][kLanes * V];
    const int l = (threadIdx.x % kLanes) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) sums[u.sub][l + j] = dsum[j];
    __syncthreads();
    if (u.sub == 0 && u.ok) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        for (int i = 1; i < kSubs; ++i) dsum[j] += sums[i][l + j];
      sgl::store_n(part + comp_at<V>(a, u, u.super), dsum);
    }
  }
}

int scan_vec(int32_t dtype, int32_t D) { return dtype != SGL_FP32 && D % 2 == 0 ? 2 : 1; }

// Sequences whole where their channels fill half the GPU or a piece would be
// shorter than kMinPiece; else cut so that the pieces fill it.
struct ScanPlan {
  int vec, supers;
  int64_t piece, groups;       // groups: rows of decay's partial sums
  size_t sup, sub, part;       // bytes of the workspace's parts
};
ScanPlan scan_plan(int32_t dtype, int64_t N, int64_t L, int32_t D) {
  ScanPlan p;
  p.vec = scan_vec(dtype, D);
  const int64_t dv = (D + p.vec - 1) / p.vec, threads = N * dv;
  int64_t supers = 0;
  if (2 * threads < kFill) {
    const int64_t want = (kPieces + threads * kSubs - 1) / (threads * kSubs);
    supers = std::min<int64_t>({want, L / (kMinPiece * kSubs), int64_t(kMaxSupers)});
  }
  p.supers = 0;
  p.piece = L;
  if (supers > 0) {
    p.piece = (L + supers * kSubs - 1) / (supers * kSubs);
    p.piece = (p.piece + kKeep - 1) / kKeep * kKeep;
    p.supers = int((L + p.piece * kSubs - 1) / (p.piece * kSubs));
    p.groups = N * p.supers;
  } else {   // as many as fill the GPU, each with as many sequences
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(N, kFill / dv)), each = (N + most - 1) / most;
    p.groups = (N + each - 1) / each;
  }
  p.sup = sgl::align_up(sizeof(float2) * size_t(N * p.supers * D));
  p.sub = sgl::align_up(sizeof(float2) * size_t(N * p.supers * kSubs * D));
  p.part = sizeof(float) * size_t(p.groups) * size_t(D);
  return p;
}

unsigned scan_grid(const ScanArgs &a, int64_t rows, int V) {
  const int64_t dv = (a.D + V - 1) / V;
  if (a.supers > 0) return unsigned(a.N * a.supers * ((dv + kLanes - 1) / kLanes));
  return unsigned((rows * dv + kBlock - 1) / kBlock);
}

template <typename T, int V, bool DECAY>
void scan_fwd(const ScanArgs &a, void *h, float *last, float *keep, hipStream_t s) {
  const dim3 grid(scan_grid(a, a.N, V));
  if (a.supers > 0)
    sgl::launch(&k_scan_pieces<T, V, DECAY, false>, grid, dim3(kBlock), 0, s, a, static_cast<const T *>(nullptr));
  sgl::launch(&k_scan_fwd<T, V, DECAY>, grid, dim3(kBlock), 0, s, a, static_cast<T *>(h), last, keep);
}

template <typename T, int V, bool DECAY>
void scan_bwd(const ScanArgs &a, const float *keep, const void *gh, const float *glast, void *dgate, void *dvalue,
              float *dstate, float *ddecay, float *part, int64_t groups, hipStream_t s) {
  const dim3 grid(scan_grid(a, groups, V));
  if (a.supers > 0)
    sgl::launch(&k_scan_pieces<T, V, DECAY, true>, grid, dim3(kBlock), 0, s, a, static_cast<const T *>(gh));
  sgl::launch(&k_scan_bwd<T, V, DECAY>, grid, dim3(kBlock), 0, s, a, keep, static_cast<const T *>(gh), glast,
              static_cast<T *>(dgate), static_cast<T *>(dvalue), dstate, part, groups);
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

// The workspace's parts; returns decay's partial sums.
float *place_work(ScanArgs &a, const ScanPlan &p, void *workspace) {
  char *w = static_cast<char *>(workspace);
  a.supers = p.supers;
  a.piece = p.piece;
  a.sup = reinterpret_cast<float2 *>(w);
  a.sub = reinterpret_cast<float2 *>(w + p.sup);
  return reinterpret_cast<float *>(w + p.sup + p.sub);
}

int check_scan(int32_t dtype, int64_t N, int64_t L, int32_t D, const ScanArgs &a) {
  SGL_REQUIRE(dtype >= 0 && dtype <= SGL_FP16, "gated_scan: unknown element type %d", dtype);
  SGL_REQUIRE(N >= 0 && L >= 0 && D > 0 && N < INT_MAX && L < INT_MAX, "gated_scan: bad sizes");
  // (a launch has fewer than 2^32 threads: one for each channel)
  SGL_REQUIRE(N * D <= (int64_t(1) << 32) - kBlock, "gated_scan: %lld sequences of %d channels are too many",
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
  return p.sup + p.sub + (backward && decay ? p.part : 0);
}

extern "C" int sgl_gated_scan_forward(int32_t dtype, int64_t N, int64_t L, int32_t D, const void *gate,
                                      int64_t gate_n, int64_t gate_t, const void *value, int64_t value_n,
                                      int64_t value_t, const int32_t *lens, const float *state, const float *gaps,
                                      int64_t gaps_n, int64_t gaps_t, const float *decay, void *h, float *last,
                                      float *keep, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  ScanArgs a{gate, value, gate_n, gate_t, value_n, value_t, lens, state, gaps, gaps_n, gaps_t, decay, N, L, D,
             0, L, nullptr, nullptr};
  if (const int rc = check_scan(dtype, N, L, D, a)) return rc;
  if (N == 0 || L == 0) return SGL_OK;
  SGL_REQUIRE(h != nullptr, "gated_scan: NULL array");
  const ScanPlan p = scan_plan(dtype, N, L, D);
  const size_t need = sgl_gated_scan_workspace_bytes(dtype, N, L, D, 0, 0);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    sgl::set_error("gated_scan: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  place_work(a, p, workspace);
  by_type(dtype, p.vec, decay != nullptr, [&](auto t, auto v, auto dec) {
    scan_fwd<decltype(t), decltype(v)::value, decltype(dec)::value>(a, h, last, keep, stream);
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
  ScanArgs a{gate, value, gate_n, gate_t, value_n, value_t, lens, state, gaps, gaps_n, gaps_t, decay, N, L, D,
             0, L, nullptr, nullptr};
  if (const int rc = check_scan(dtype, N, L, D, a)) return rc;
  if (N == 0 || L == 0) return SGL_OK;
  SGL_REQUIRE(keep && dgate && dvalue && (decay == nullptr || ddecay != nullptr), "gated_scan_backward: NULL array");
  const ScanPlan p = scan_plan(dtype, N, L, D);
  const size_t need = sgl_gated_scan_workspace_bytes(dtype, N, L, D, 1, decay != nullptr);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    sgl::set_error("gated_scan_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  float *part = place_work(a, p, workspace);
  by_type(dtype, p.vec, decay != nullptr, [&](auto t, auto v, auto dec) {
    scan_bwd<decltype(t), decltype(v)::value, decltype(dec)::value>(a, keep, gh, glast, dgate, dvalue, dstate, ddecay,
                                                                    part, p.groups, stream);
  });
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}
