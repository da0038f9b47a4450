// Shared pieces of the token operators: rotations by positions of several axes, places in a paged cache.
#pragma once

#include "feat_common.h"
#include "splat_tokens.h"

namespace splat {

constexpr int kMaxAxes = 4, kMaxHead = 128;

// cos and sin of w quarter turns: w is reduced to the nearest quarter in 64 bits (adding 1.5 * 2^52 leaves the whole number in
// the last bits), what is left by polynomials fitted for the least error on half a quarter either side (3e-9 and 5e-11, 9e-8
// evaluated in float32). A position of 2^31 still has 22 bits behind the quarter's point. Past 2^51 quarters none are left and
// the steps of the 64-bit sum leave more than half a quarter, which counts as half of one: any angle, but always a rotation.
__device__ __forceinline__ void turn(double p, double quarters, float& c, float& s) {
  constexpr double kRound = 6755399441055744.0;
  const double t = fma(p, quarters, kRound), q = t - kRound;
  float x = (float)fma(p, quarters, -q);
  x = fabsf(x) > 0.5f ? 0.5f : x;   // no number stays none
  const unsigned n = (unsigned)__double2loint(t);
  const float z = x * x;
  float a = fmaf(-0.00460165785625577f, z, 0.07968003302812576f);
  a = fmaf(a, z, -0.6459634900093079f);
  a = fmaf(a, z, 1.5707963705062866f) * x;
  float b = fmaf(0.0009040216682478786f, z, -0.02086028829216957f);
  b = fmaf(b, z, 0.25366923213005066f);
  b = fmaf(b, z, -1.2337005138397217f);
  b = fmaf(b, z, 1.f);
  const float u = n & 1 ? a : b, v = n & 1 ? b : a;
  c = (n + 1) & 2 ? -u : u;
  s = n & 2 ? -v : v;
}

__device__ __forceinline__ double position(const splat_positions& p, long long at) {
  return p.type == 0 ? (double)((const float*)p.p)[at] : p.type == 1 ? (double)((const int*)p.p)[at]
                                                                     : (double)((const long long*)p.p)[at];
}

// A unit of a head: two runs of W values at e0 and e1 that turn as pairs (halves: run 0's value i with run 1's; neighbours:
// the 2 W values from e0 on, two by two), or that pass (axis < 0). `pair` is its first pair, `second` whether there is a second run.
struct PairUnit {
  int axis, pair, e0, e1;
  bool second;
};
template <int W>
__device__ __forceinline__ PairUnit pair_unit(const splat_rotation& r, int D, int u) {
  int e = 0, pair = 0;
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    if (a >= r.axes) break;
    const int half = r.dims[a] / 2, n = half / W;
    if (u < n) return {a, pair + u * W, r.interleaved ? e + 2 * u * W : e + u * W,
                       r.interleaved ? e + (2 * u + 1) * W : e + half + u * W, true};
    u -= n;
    pair += half;
    e += r.dims[a];
  }
  e += 2 * u * W;
  return {-1, 0, e, e + W, e + W < D};
}

// Units of W pairs need every half axis and what passes to be whole runs.
struct Units {
  int W, n;
};
inline Units pair_units(const splat_rotation& r, int D, int widest) {
  int W = widest, sum = 0, pairs = 0;
  for (int a = 0; a < r.axes; ++a) sum += r.dims[a];
  pairs = sum / 2;
  auto fits = [&](int w) {
    for (int a = 0; a < r.axes; ++a)
      if (r.dims[a] / 2 % w) return false;
    return (D - sum) % w == 0;
  };
  while (!fits(W)) W /= 2;
  return {W, pairs / W + (D - sum + 2 * W - 1) / (2 * W)};
}

inline int check_rotation(const char* who, const splat_rotation* r, const splat_positions* p, int D) {
  if (!r || r->axes == 0) return kOk;
  if (r->axes < 0 || r->axes > kMaxAxes) return set_error(kInvalid, "%s: %d axes", who, r->axes);
  int sum = 0;
  for (int a = 0; a < r->axes; ++a) {
    if (r->dims[a] < 2 || r->dims[a] % 2 || r->dims[a] > kMaxHead)
      return set_error(kInvalid, "%s: an axis of %d values", who, r->dims[a]);
    sum += r->dims[a];
  }
  if (sum > D) return set_error(kInvalid, "%s: axes of %d values in a head of %d", who, sum, D);
  if (!p || !p->p || p->type < 0 || p->type > 2) return set_error(kInvalid, "%s: positions are missing", who);
  return kOk;
}

// Turns the pairs of a unit's two runs by the angles whose cosines and sines are c and s (Back: by their negatives).
template <int W, bool Back>
__device__ __forceinline__ void turn_runs(float (&a)[W], float (&b)[W], const float (&c)[W], const float (&s)[W], bool neighbours) {
  auto one = [](float& x, float& y, float c, float s) {
    if (Back) s = -s;
    const float t = fmaf(x, c, -y * s);
    y = fmaf(x, s, y * c);
    x = t;
  };
  if constexpr (W > 1) {
    if (neighbours) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        one(a[2 * j], a[2 * j + 1], c[j], s[j]);
        one(b[2 * j], b[2 * j + 1], c[W / 2 + j], s[W / 2 + j]);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) one(a[j], b[j], c[j], s[j]);
}

template <typename T, int W>
__device__ __forceinline__ void store_run(T* p, const float (&f)[W]) {
  T v[W];
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = (T)f[j];
  __builtin_memcpy(p, v, sizeof(v));
}

// Tokens of sequence b: all of them, and the new ones among them.
__device__ __forceinline__ int cached_tokens(const splat_cache& c, int b) {
  const long long room = (long long)c.page * c.width;
  const int n = c.lengths[b];
  return n < 0 ? 0 : n > room ? (int)room : n;
}
__device__ __forceinline__ int new_tokens(const splat_cache& c, int b, int T) {
  const int n = c.counts ? c.counts[b] : T;
  return n < 0 ? 0 : n > T ? T : n;
}

inline int check_cache(const char* who, const splat_cache* c) {
  if (!c) return set_error(kInvalid, "%s: no cache", who);
  if (c->dtype != kF32 && c->dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", who, c->dtype);
  if (c->B < 0 || c->Hk < 1 || c->D < 1 || c->page < 1 || c->width < 0 || c->pages < 0)
    return set_error(kInvalid, "%s: B %d, Hk %d, D %d, page %d, width %d", who, c->B, c->Hk, c->D, c->page, c->width);
  if (c->D > kMaxHead) return set_error(kUnsupported, "%s: heads of %d values, %d at most", who, c->D, kMaxHead);
  if (c->pages > 0x7fffffffLL || (long long)c->page * c->width > 0x7fff0000LL)
    return set_error(kUnsupported, "%s: a table of %d pages of %d tokens", who, c->width, c->page);
  if (c->B > 0 && (!c->lengths || (c->width > 0 && !c->tables) || (c->pages > 0 && (!c->k || !c->v))))
    return set_error(kInvalid, "%s: null pointer", who);
  return kOk;
}

}  // namespace splat
