// Rotary positions: pairs of a head's channels turned by an angle that grows
// with the row's position, for queries and keys in one launch.
//
// (a, b) -> gain (a cos t - b sin t, a sin t + b cos t), t = position * f_i.
// The angle is kept in turns, as a 64-bit fraction: position times f_i / 2 pi
// modulo 1 is an integer product, and with f_i / 2 pi to 96 bits it is within
// 2^-32 of a turn (1.5e-9 rad) at every int64 position (a float angle of a position
// of 1e9 has no digits left of the turn, a 64-bit f_i / 2 pi is 0.6 rad off at
// nanosecond stamps of 1.7e18). The gradient is the same rotation the other way
// round.
//
// Memory bounds it, every element read and written once: 16 sequences of 8,191
// x (8 + 2) heads of 128 in fp16 123 us, 5.5 TB/s (a large copy: 5.1); 4,000 x
// (20 + 32) x 4 heads of 43 in bf16 34 us, 4.2 TB/s; 400 x 1 x 2 heads of 50, one
// new event each, 4 us, the launch.
#include "history.h"

namespace {

using namespace sgl;

constexpr int kBlock = 256, kSteps = 512;

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

// A frequency (angle a unit of position) in turns, modulo 1: (hi 2^32 + lo) / 2^96.
// The last bit marks one that has no angle (not finite, or 2^128 and more). (128 bits
// take two products more a pair: 4,000 x 52 x 4 heads of 43 in bf16 38.5 us for 37.3.)
struct Step {
  uint64_t hi;
  uint32_t lo;
};
struct Steps {   // a workgroup's, in LDS of kStepBytes for each
  uint64_t *hi;
  uint32_t *lo;
  __device__ __forceinline__ Steps(char *lds, int n)
      : hi(reinterpret_cast<uint64_t *>(lds)), lo(reinterpret_cast<uint32_t *>(hi + n)) {}
  __device__ __forceinline__ void put(int i, const Step &s) const { hi[i] = s.hi, lo[i] = s.lo; }
  __device__ __forceinline__ Step at(int i) const { return Step{hi[i], lo[i]}; }
};
constexpr size_t kStepBytes = sizeof(uint64_t) + sizeof(uint32_t);
// m 2^e / 2 pi of a double m 2^e, with 1 / 2 pi to 320 bits: enough behind the
// point of a turn for any frequency under 2^128.
__device__ __forceinline__ Step turn_step(double f) {
  constexpr uint64_t kInv[5] = {0x28be60db9391054aull, 0x7f09d5f47d4d3770ull, 0x36d8a5664f10e410ull,
                                0x7f9458eaf7aef158ull, 0x6dc91b8e909374b8ull};
  const uint64_t bits = uint64_t(__double_as_longlong(f));
  const int ex = int(bits >> 52) & 0x7FF, e = max(ex, 1) - 1075;
  const uint64_t m = (bits & ((1ull << 52) - 1)) | (ex != 0 ? 1ull << 52 : 0ull);
  uint64_t w0 = kInv[0], w1 = kInv[1], w2 = kInv[2];
  if (e > 0) {   // (whole turns of 2^e / 2 pi are left out)
    const int by = e & 63;
    const bool far = e >= 64;
    const uint64_t v0 = far ? kInv[1] : kInv[0], v1 = far ? kInv[2] : kInv[1], v2 = far ? kInv[3] : kInv[2],
                   v3 = far ? kInv[4] : kInv[3];
    w0 = by != 0 ? v0 << by | v1 >> (64 - by) : v0;
    w1 = by != 0 ? v1 << by | v2 >> (64 - by) : v1;
    w2 = by != 0 ? v2 << by | v3 >> (64 - by) : v2;
  }
  // m times it: p3 whole turns, then the fraction's words p2 and p1
  const uint64_t p1 = m * w1 + __umul64hi(m, w2), c1 = p1 < m * w1 ? 1 : 0;
  const uint64_t t = m * w0 + __umul64hi(m, w1), p2 = t + c1;
  const uint64_t p3 = __umul64hi(m, w0) + (t < m * w0 ? 1 : 0) + (p2 < t ? 1 : 0);
  uint64_t hi = p2, lo = p1;
  if (e < 0) {   // 2^e of it
    const int r = -e, by = r & 63;
    const uint64_t x0 = r < 64 ? p2 : r < 128 ? p3 : 0, up = r < 64 ? p3 : 0;
    const uint64_t x1 = r < 64 ? p1 : r < 128 ? p2 : r < 192 ? p3 : 0;
    hi = by != 0 ? x0 >> by | up << (64 - by) : x0;
    lo = by != 0 ? x1 >> by | x0 << (64 - by) : x1;
  }
  if (f < 0.0) {
    lo = 0 - lo;
    hi = 0 - hi - (lo != 0 ? 1 : 0);
  }
  return Step{hi, (uint32_t(lo >> 32) & ~1u) | (fabs(f) < 0x1p128 ? 0u : 1u)};
}
// The position's turns, modulo 1, as a 64-bit fraction, within 2^-32 of a turn.
__device__ __forceinline__ uint64_t turns_at(int64_t pos, const Step &s) {
  const uint64_t u = uint64_t(pos);
  const uint64_t low = (u >> 32) * s.lo + __umulhi(uint32_t(u), s.lo);   // u lo / 2^32
  return u * s.hi + low - (pos < 0 ? uint64_t(s.lo) << 32 : 0);
}
// gain times the angle's sine (way -1: the other way round) and cosine.
__device__ __forceinline__ void sincos_at(int64_t pos, const Step &step, float gain, float way, float &sn, float &cs) {
  sincos_turns(turns_at(pos, step), sn, cs);
  const float by = (step.lo & 1) != 0 ? NAN : gain;
  sn *= by * way;
  cs *= by;
}

// a cos - b sin and a sin + b cos, rounded to 32 bits before the type's (one
// rounding less in some places and not in others would give lanes that write the
// same channel different bits).
template <typename T>
__device__ __forceinline__ void turn(T &a, T &b, float sn, float cs) {
  const float p = float(a), q = float(b);
  float x = fmaf(p, cs, -(q * sn)), y = fmaf(p, sn, q * cs);
  asm("" : "+v"(x), "+v"(y));
  a = T(x);
  b = T(y);
}

// A workgroup forms the frequencies' steps once where they are few (SHARED: up
// to kSteps pairs; 64-bit floating point of every lane otherwise: one head of 172
// in fp16 38 us for 57, two of 100 with 64 turned 39 for 53).
// A lane owns VEC consecutive channels of a row (both halves' in the half
// layout) for all its heads; the angles are formed once for all of them. A
// part's last lane takes its last VEC channels, some of them its neighbour's
// too (it writes the same bits), so that loads and stores are all whole (4 heads
// of 44 in bf16: 123 us with the last ones one by one, 30 so); channels that are
// not rotated and fewer than VEC go one by one.
template <typename T, int VEC, bool INTER, bool SHARED>
__global__ __launch_bounds__(kBlock) void k_rotate(RotArgs a) {
  const int sd = int64_t(blockIdx.x) >= a.side[1].first ? 1 : 0;
  const Side &s = a.side[sd];
  const int half = a.rot / 2;
  constexpr int PV = INTER ? VEC / 2 : VEC;   // pairs of a lane
  const int ru = (half + PV - 1) / PV, cu = (a.dh - a.rot + VEC - 1) / VEC, units = ru + cu;
  const int64_t at = (int64_t(blockIdx.x) - s.first) * kBlock + threadIdx.x;
  const int64_t row = at / units;
  extern __shared__ __align__(16) char lds[];
  const Steps steps(lds, half);
  if constexpr (SHARED) {
    for (int i = threadIdx.x; i < half; i += kBlock) steps.put(i, turn_step(a.freqs[i]));
    __syncthreads();
  }
  if (row >= s.rows) return;
  const int u = int(at - row * units);
  const int64_t n = row / s.L, t = row - n * s.L;
  const T *x = static_cast<const T *>(s.x) + n * s.sn + t * s.st;
  T *y = static_cast<T *>(s.y) + row * s.H * a.dh;
  if (u >= ru) {   // what is not rotated
    const int rest = a.dh - a.rot;
    const int d = a.rot + max(min((u - ru) * VEC, rest - VEC), 0);
#pragma unroll 4
    for (int h = 0; h < s.H; ++h, x += s.sh, y += a.dh) {
      if (rest >= VEC) {
        T v[VEC];
        load_n(v, x + d);
        store_n(y + d, v);
      } else {
        for (int i = 0; i < rest; ++i) y[d + i] = x[d + i];
      }
    }
    return;
  }
  const int p0 = min(u * PV, half - PV);
  const int64_t pos = s.pos[n * s.pn + t * s.pt];
  float sn[PV], cs[PV];
#pragma unroll
  for (int i = 0; i < PV; ++i)
    sincos_at(pos, SHARED ? steps.at(p0 + i) : turn_step(a.freqs[p0 + i]), a.gain, a.way, sn[i], cs[i]);
  for (int h = 0; h < s.H; ++h, x += s.sh, y += a.dh) {
    if constexpr (INTER) {
      T v[VEC];
      load_n(v, x + 2 * p0);
#pragma unroll
      for (int i = 0; i < PV; ++i)
        turn(v[2 * i], v[2 * i + 1], sn[i], cs[i]);
      store_n(y + 2 * p0, v);
    } else {
      T v[VEC], w[VEC];
      load_n(v, x + p0);
      load_n(w, x + half + p0);
#pragma unroll
      for (int i = 0; i < PV; ++i)
        turn(v[i], w[i], sn[i], cs[i]);
      store_n(y + p0, v);
      store_n(y + half + p0, w);
    }
  }
}

// Heads of an odd number of channels, whose rows lie one behind the other: a
// workgroup's rows as one stretch, in and out 16 bytes at a time and turned in LDS
// (a lane's own loads and stores would straddle). 4,000 x (20 + 32) x 4 heads of 43,
// interleaved, in bf16 30 us for 41, in fp32 58 for 104, 8 heads of 127 in bf16 166
// for 279; 200 x (20 + 32) x 4 of 43 6.0 for 5.5: taken where there are two
// workgroups a CU.
constexpr int kStretchRows = 256;
template <typename T>
constexpr int kStretch = 16384 / int(sizeof(T));   // elements of a workgroup's rows
template <typename T, bool INTER>
__global__ __launch_bounds__(kBlock) void k_rotate_odd(RotArgs a, int tile_rows) {
  __shared__ __align__(16) T tile[kStretch<T>];
  extern __shared__ __align__(16) char lds[];   // (as much as the pairs take: eight workgroups a CU mostly)
  __shared__ int64_t pos[kStretchRows];
  const int sd = int64_t(blockIdx.x) >= a.side[1].first ? 1 : 0, tid = threadIdx.x;
  const Side &s = a.side[sd];
  const int64_t row0 = (int64_t(blockIdx.x) - s.first) * tile_rows;
  const int rows = int(min(int64_t(tile_rows), s.rows - row0)), width = s.H * a.dh, n = rows * width, half = a.rot / 2;
  const Steps steps(lds, half);
  const T *x = static_cast<const T *>(s.x) + row0 * width;
  T *y = static_cast<T *>(s.y) + row0 * width;
  constexpr int E = 16 / int(sizeof(T));
  auto copy = [&](T *to, const T *from) {
    for (int i = tid * E; i + E <= n; i += kBlock * E) {
      T v[E];
      load_n(v, from + i);
      store_n(to + i, v);
    }
    for (int i = n / E * E + tid; i < n; i += kBlock) to[i] = from[i];
  };
  const double f = tid < half ? a.freqs[tid] : 0.0;   // (on its way beside the rows)
  copy(tile, x);
  if (tid < half) steps.put(tid, turn_step(f));
  for (int i = tid + kBlock; i < half; i += kBlock) steps.put(i, turn_step(a.freqs[i]));
  for (int i = tid; i < rows; i += kBlock) {
    const int64_t seq = (row0 + i) / s.L, t = row0 + i - seq * s.L;
    pos[i] = s.pos[seq * s.pn + t * s.pt];
  }
  __syncthreads();
  for (int i = tid; i < rows * half; i += kBlock) {
    const int r = i / half, p = i - r * half;
    float sn, cs;
    sincos_at(pos[r], steps.at(p), a.gain, a.way, sn, cs);
    T *v = tile + r * width + (INTER ? 2 * p : p);
    constexpr int one = INTER ? 1 : 0;
    const int other = one != 0 ? 1 : half;
    for (int h = 0; h < s.H; ++h, v += a.dh) turn(v[0], v[other], sn, cs);
  }
  __syncthreads();
  copy(y, tile);
}
// Rows of a workgroup (16 bytes each workgroup's start), or 0: not of that kind.
template <typename T>
int odd_rows(const RotArgs &a) {
  if (a.dh % 2 == 0 || a.rot == 0) return 0;
  int most = kStretchRows;
  int64_t all = 0;
  for (const Side &s : a.side) {
    if (s.rows == 0) continue;
    const int64_t width = int64_t(s.H) * a.dh;
    if (width > kStretch<T> / 8 || s.sh != a.dh || s.st != width || (s.sn != s.L * width && s.rows != s.L)) return 0;
    most = min(most, int(kStretch<T> / width) / 8 * 8);
    all += s.rows;
  }
  return all / most >= 512 ? most : 0;
}

template <typename T, int VEC, bool INTER>
void go(RotArgs a, dim3 grid, hipStream_t stream) {
  const size_t steps = size_t(a.rot / 2) * kStepBytes;
  if (a.rot / 2 <= kSteps) launch(&k_rotate<T, VEC, INTER, true>, grid, dim3(kBlock), steps, stream, a);
  else launch(&k_rotate<T, VEC, INTER, false>, grid, dim3(kBlock), 0, stream, a);
}
template <typename T, bool INTER>
int run(RotArgs a, hipStream_t stream) {
  constexpr int MOST = (INTER ? 16 : 8) / int(sizeof(T)), LEAST = INTER ? 2 : 1;
  const int half = a.rot / 2;
  if (const int rows = odd_rows<T>(a)) {
    int64_t grid = 0;
    for (int i = 0; i < 2; ++i) {
      a.side[i].first = grid;
      grid += (a.side[i].rows + rows - 1) / rows;
    }
    if (a.side[1].rows == 0) a.side[1].first = INT64_MAX;
    SGL_REQUIRE(grid < (1 << 24), "rotary: too many rows");
    launch(&k_rotate_odd<T, INTER>, dim3(unsigned(grid)), dim3(kBlock), size_t(half) * kStepBytes, stream, a, rows);
    SGL_CHECK_LAUNCH();
    return SGL_OK;
  }
  // A lane moves 16 bytes at a time (two loads of 8 in the half layout), or half
  // of that where rows are not whole words (4 heads of 43 in bf16, interleaved 54 us
  // with 16 bytes and 43 with 8, halves 53 with 8 and 45 with 4; 44 channels: 30
  // with 8, 31 with 4; 128: 87 and 94), and no more than the pairs there are.
  int vec = MOST;
  if (a.dh * int(sizeof(T)) % 4 != 0) vec /= 2;
  while (vec > LEAST && half > 0 && half < (INTER ? vec / 2 : vec)) vec /= 2;
  const int pairs = INTER ? vec / 2 : vec;
  const int64_t units = (half + pairs - 1) / pairs + (a.dh - a.rot + vec - 1) / vec;
  int64_t grid = 0;
  for (int i = 0; i < 2; ++i) {
    a.side[i].first = grid;
    grid += (a.side[i].rows * units + kBlock - 1) / kBlock;
  }
  if (a.side[1].rows == 0) a.side[1].first = INT64_MAX;
  SGL_REQUIRE(grid < (1 << 24), "rotary: too many rows");   // (a launch has 2^32 threads)
  if (grid == 0) return SGL_OK;
  const dim3 g{unsigned(grid)};
  if (vec == MOST) go<T, MOST, INTER>(a, g, stream);
  else if (MOST / 2 > LEAST && vec == MOST / 2) go<T, MOST / 2, INTER>(a, g, stream);
  else go<T, LEAST, INTER>(a, g, stream);
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
