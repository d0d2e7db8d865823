// Rotary positions: pairs of a head's channels turned by an angle that grows
// with the row's position, for queries and keys in one launch.
//
// (a, b) -> gain (a cos t - b sin t, a sin t + b cos t), t = position * f_i.
// The angle is kept in turns, as a 64-bit fraction: position times f_i / 2 pi
// modulo 1 is one integer product, exact for every int64 position (a float
// angle of a position of 1e9 has no digits left of the turn). The gradient is
// the same rotation the other way round.
//
// Memory bounds it: every element is read and written once.
#include "history.h"

namespace {

using namespace sgl;

constexpr int kBlock = 256;

struct Side {
  const void *x;
  void *y;
  const int64_t *pos;
  int64_t sn, st, sh;    // strides of x (sequences, rows, heads), elements
  int64_t pn, pt;        // of pos
  int64_t L;
  int H;
  int64_t rows;          // N L
  int64_t first;         // this side's first workgroup
};
struct RotArgs {
  Side side[2];
  const double *freqs;   // angles a unit of position, [rot / 2]
  int dh, rot;
  float gain, way;       // way: 1, or -1 the other way round
};

// sin and cos of `turns` (a 64-bit fraction of a turn): the nearest quarter, and
// the series of both within an eighth of it (2e-9 off at its ends).
__device__ __forceinline__ void sincos_turns(uint64_t turns, float &s, float &c) {
  const uint64_t q = turns + (1ull << 61);
  const int quarter = int(q >> 62);
  const int64_t off = int64_t(q & ((1ull << 62) - 1)) - (1ll << 61);
  const float x = float(off) * float(6.283185307179586477 / 18446744073709551616.0);   // within pi / 4
  const float z = x * x;
  const float sn = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float cs = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
  const float u = (quarter & 1) != 0 ? cs : sn, v = (quarter & 1) != 0 ? sn : cs;
  s = (quarter & 2) != 0 ? -u : u;
  c = ((quarter + 1) & 2) != 0 ? -v : v;
}

// A frequency (angle a unit of position) in turns, modulo 1, as a 64-bit
// fraction: f / 2 pi to 106 bits (1 / 2 pi in two doubles), so that its fraction
// has them all.
__device__ __forceinline__ uint64_t turn_step(double f) {
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;
  const double hi = f * kHi, lo = fma(f, kLo, fma(f, kHi, -hi));
  auto fraction = [](double x) {   // x modulo 1, in 2^-64 (of the magnitude: its steps are exact)
    const double m = fabs(x), r = m - floor(m), up = floor(r * 4294967296.0);
    const uint64_t u = (uint64_t(up) << 32) + uint64_t((r * 4294967296.0 - up) * 4294967296.0);
    return x < 0.0 ? 0 - u : u;
  };
  return fraction(hi) + fraction(lo);
}

// A lane owns VEC consecutive channels of a row (both halves' in the half
// layout) for a range of its heads; the angle is formed once for all of them.
// The lanes past the rotated channels copy.
template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(kBlock) void k_rotate(RotArgs a) {
  const int sd = int64_t(blockIdx.x) >= a.side[1].first ? 1 : 0;
  const Side &s = a.side[sd];
  const int half = a.rot / 2;
  // units of a row: pairs of the rotated part, then the rest
  const int pairs = INTER ? VEC / 2 : VEC;                 // pairs a unit holds
  const int ru = (half + pairs - 1) / pairs, cu = (a.dh - a.rot + VEC - 1) / VEC, units = ru + cu;
  const int64_t at = (int64_t(blockIdx.x) - s.first) * kBlock + threadIdx.x;
  const int64_t row = at / units;
  if (row >= s.rows) return;
  const int u = int(at - row * units);
  const int64_t n = row / s.L, t = row - n * s.L;
  const T *x = static_cast<const T *>(s.x) + n * s.sn + t * s.st;
  T *y = static_cast<T *>(s.y) + row * s.H * a.dh;
  if (u >= ru) {   // what is not rotated
    const int d = a.rot + (u - ru) * VEC, w = min(VEC, a.dh - d);
    for (int h = 0; h < s.H; ++h, x += s.sh, y += a.dh) {
      if (w == VEC) {
        T v[VEC];
        load_n(v, x + d);
        store_n(y + d, v);
      } else {
        for (int i = 0; i < w; ++i) y[d + i] = x[d + i];
      }
    }
    return;
  }
  const int p0 = u * pairs, np = min(pairs, half - p0);
  const int64_t pos = s.pos[n * s.pn + t * s.pt];
  constexpr int PV = INTER ? VEC / 2 : VEC;
  float sn[PV], cs[PV];
#pragma unroll
  for (int i = 0; i < PV; ++i) {
    sincos_turns(uint64_t(pos) * turn_step(a.freqs[p0 + min(i, np - 1)]), sn[i], cs[i]);
    sn[i] *= a.gain * a.way;
    cs[i] *= a.gain;
  }
  for (int h = 0; h < s.H; ++h, x += s.sh, y += a.dh) {
    if constexpr (INTER) {
      T v[VEC];
      if (np == PV) {
        load_n(v, x + 2 * p0);
#pragma unroll
        for (int i = 0; i < PV; ++i) {
          const float p = float(v[2 * i]), q = float(v[2 * i + 1]);
          v[2 * i] = T(p * cs[i] - q * sn[i]);
          v[2 * i + 1] = T(p * sn[i] + q * cs[i]);
        }
        store_n(y + 2 * p0, v);
      } else {
#pragma unroll
        for (int i = 0; i < PV; ++i)
          if (i < np) {
            const float p = float(x[2 * (p0 + i)]), q = float(x[2 * (p0 + i) + 1]);
            y[2 * (p0 + i)] = T(p * cs[i] - q * sn[i]);
            y[2 * (p0 + i) + 1] = T(p * sn[i] + q * cs[i]);
          }
      }
    } else {
      if (np == PV) {
        T v[VEC], w[VEC];
        load_n(v, x + p0);
        load_n(w, x + half + p0);
#pragma unroll
        for (int i = 0; i < PV; ++i) {
          const float p = float(v[i]), q = float(w[i]);
          v[i] = T(p * cs[i] - q * sn[i]);
          w[i] = T(p * sn[i] + q * cs[i]);
        }
        store_n(y + p0, v);
        store_n(y + half + p0, w);
      } else {
#pragma unroll
        for (int i = 0; i < PV; ++i)
          if (i < np) {
            const float p = float(x[p0 + i]), q = float(x[half + p0 + i]);
            y[p0 + i] = T(p * cs[i] - q * sn[i]);
            y[half + p0 + i] = T(p * sn[i] + q * cs[i]);
          }
      }
    }
  }
}

template <typename T, bool INTER>
int run(RotArgs a, hipStream_t stream) {
  constexpr int VEC = 16 / int(sizeof(T));
  const int pairs = INTER ? VEC / 2 : VEC, half = a.rot / 2;
  const int64_t units = (half + pairs - 1) / pairs + (a.dh - a.rot + VEC - 1) / VEC;
  int64_t grid = 0;
  for (int i = 0; i < 2; ++i) {
    a.side[i].first = grid;
    grid += (a.side[i].rows * units + kBlock - 1) / kBlock;
  }
  if (a.side[1].rows == 0) a.side[1].first = INT64_MAX;
  SGL_REQUIRE(grid < (1 << 24), "rotary: too many rows");   // (a launch has 2^32 threads)
  if (grid == 0) return SGL_OK;
  launch(&k_rotate<T, VEC, INTER>, dim3(unsigned(grid)), dim3(kBlock), 0, stream, a);
  SGL_CHECK_LAUNCH();
  return SGL_OK;
}
template <typename T>
int pick(const RotArgs &a, bool interleaved, hipStream_t stream) {
  return interleaved ? run<T, true>(a, stream) : run<T, false>(a, stream);
}

}  // namespace

extern "C" int sgl_rotary(int32_t dtype, int64_t n, int32_t dh, int32_t rot, const sgl_rotary_side *q,
                          const sgl_rotary_side *k, const double *freqs, int32_t interleaved, float gain,
                          int32_t inverse, hipStream_t stream) {
  SGL_REQUIRE(dtype >= 0 && dtype <= SGL_FP16, "rotary: unknown element type %d", dtype);
  SGL_REQUIRE(n >= 0 && dh > 0 && dh <= 65536 && rot >= 0 && rot <= dh && rot % 2 == 0,
              "rotary: %d of %d channels", rot, dh);
  SGL_REQUIRE(rot == 0 || freqs != nullptr, "rotary: NULL frequencies");
  SGL_REQUIRE(q != nullptr, "rotary: NULL side");
  RotArgs a{};
  a.freqs = freqs;
  a.dh = dh;
  a.rot = rot;
  a.gain = gain;
  a.way = inverse != 0 ? -1.f : 1.f;
  for (int i = 0; i < 2; ++i) {
    const sgl_rotary_side *s = i == 0 ? q : k;
    if (s == nullptr) continue;
    SGL_REQUIRE(s->len >= 0 && s->heads >= 0 && s->len < (int64_t(1) << 40) / (n + 1), "rotary: %lld rows of %d heads",
                (long long)s->len, s->heads);
    Side &d = a.side[i];
    d.rows = s->heads > 0 ? n * s->len : 0;
    if (d.rows == 0) continue;
    SGL_REQUIRE(s->x && s->y && s->pos, "rotary: NULL array");
    d.x = s->x;
    d.y = s->y;
    d.pos = s->pos;
    d.sn = s->x_n;
    d.st = s->x_t;
    d.sh = s->x_h;
    d.pn = s->pos_n;
    d.pt = s->pos_t;
    d.L = s->len;
    d.H = s->heads;
  }
  for (int i = 0; i < 2; ++i)
    if (a.side[i].L == 0) a.side[i].L = 1;
  if (dtype == SGL_FP32) return pick<float>(a, interleaved != 0, stream);
  if (dtype == SGL_BF16) return pick<bf16_t>(a, interleaved != 0, stream);
  return pick<fp16_t>(a, interleaved != 0, stream);
}
