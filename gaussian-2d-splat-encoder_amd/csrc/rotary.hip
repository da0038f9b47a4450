// Rotary positions of several axes, x[B, L, H, D] -> y, and new tokens' keys (turned on the way) and values into a paged cache.
//
// Pair i of axis a turns by w = p_a * quarters[pair] quarter turns: (y0, y1) = (x0 cos w - x1 sin w, x0 sin w + x1 cos w). The
// input's gradient is the same turn back; dw = g1 y0 - g0 y1 = dx1 x0 - dx0 x1 (both turned back together), summed over heads
// and an axis' pairs for the positions' gradient.
//
// All of it is bound by memory. A thread has a unit of W pairs (16 bytes a run where the axes allow it) of a token, computes
// their angles once in 64 bits and turns the unit in several heads; a token's threads lie side by side, so that a wave's loads
// cover whole heads. Workgroups walk over tokens with the unit's rates in registers.
#include <algorithm>

#include "token_common.h"

namespace splat {
namespace {

constexpr int kThreads = 256;
constexpr int kGrid = 2048;   // workgroups at most

struct Turn {
  splat_rotation r;
  splat_positions pos;
  long long xb, xl, xh, gb, gl, gh;   // strides of x and of the gradient
  int B, L, H, D, M;                  // M = B L tokens
  int units, hs, rows;                // units of a head; threads of a unit (heads in turn); tokens of a workgroup
  FastDiv by_L, by_units, by_row, by_axes;   // by_row: by the threads of a token
};

// A thread's place in its workgroup's tokens.
struct Seat {
  int row, u, h;
  bool in;
};
__device__ __forceinline__ Seat seat(int units, int hs, int rows, FastDiv by_units, FastDiv by_row) {
  const int t = threadIdx.x, row = t / by_row, k = t - row * (units * hs), h = k / by_units;
  return {row, k - h * units, h, row < rows};
}

template <int W>
__device__ __forceinline__ void rates(const splat_rotation& r, const PairUnit& u, double (&f)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) f[j] = u.axis >= 0 ? r.quarters[u.pair + j] : 0.0;
}

template <int W>
__device__ __forceinline__ void angles(double p, const double (&f)[W], float (&c)[W], float (&s)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) turn(p, f[j], c[j], s[j]);
}

// y = x turned (Back: turned back).
template <typename T, int W, bool Back>
__global__ __launch_bounds__(kThreads) void k_rotary(Turn n, const T* __restrict__ x, T* __restrict__ y) {
  const Seat at = seat(n.units, n.hs, n.rows, n.by_units, n.by_row);
  if (!at.in) return;
  const PairUnit u = pair_unit<W>(n.r, n.D, at.u);
  double f[W];
  rates<W>(n.r, u, f);
  for (long long m = (long long)blockIdx.x * n.rows + at.row; m < n.M; m += (long long)gridDim.x * n.rows) {
    const int b = (int)m / n.by_L, l = (int)m - b * n.L;
    float c[W], s[W];
    if (u.axis >= 0) angles<W>(position(n.pos, b * n.pos.pb + l * n.pos.pl + u.axis * n.pos.pa), f, c, s);
    const T* xp = x + b * n.xb + l * n.xl;
    T* yp = y + m * n.H * n.D;
    for (int h = at.h; h < n.H; h += n.hs) {
      float p[W], q[W] = {};
      load_run<T, W>(xp + h * n.xh + u.e0, p);
      if (u.second) load_run<T, W>(xp + h * n.xh + u.e1, q);
      if (u.axis >= 0) turn_runs<W, Back>(p, q, c, s, n.r.interleaved);
      store_run<T, W>(yp + (long long)h * n.D + u.e0, p);
      if (u.second) store_run<T, W>(yp + (long long)h * n.D + u.e1, q);
    }
  }
}

// sum of a unit's pairs of dx1 x0 - dx0 x1, pair by pair.
template <int W>
__device__ __forceinline__ void add_pairs(float (&sum)[W], const float (&p)[W], const float (&q)[W], const float (&a)[W],
                                          const float (&e)[W], bool neighbours) {
  if constexpr (W > 1) {
    if (neighbours) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        sum[j] = fmaf(p[2 * j + 1], a[2 * j], fmaf(-p[2 * j], a[2 * j + 1], sum[j]));
        sum[W / 2 + j] = fmaf(q[2 * j + 1], e[2 * j], fmaf(-q[2 * j], e[2 * j + 1], sum[W / 2 + j]));
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) sum[j] = fmaf(q[j], a[j], fmaf(-p[j], e[j], sum[j]));
}

// The gradients of x and of the positions ([B, L, axes], every image's own): a token's threads are its units, each over all
// heads; an axis' units are added in order by one thread.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void k_rotary_bwd(Turn n, const T* __restrict__ x, const T* __restrict__ g,
                                                         T* __restrict__ dx, float* __restrict__ dpos) {
  __shared__ float part[2][kThreads];
  const Seat at = seat(n.units, 1, n.rows, n.by_units, n.by_row);
  const PairUnit u = pair_unit<W>(n.r, n.D, at.u);
  double f[W];
  rates<W>(n.r, u, f);
  int flip = 0;
  for (long long m0 = (long long)blockIdx.x * n.rows; m0 < n.M; m0 += (long long)gridDim.x * n.rows, flip ^= 1) {
    const long long m = m0 + at.row;
    if (at.in && m < n.M) {
      const int b = (int)m / n.by_L, l = (int)m - b * n.L;
      float c[W], s[W], sum[W] = {};
      if (u.axis >= 0) angles<W>(position(n.pos, b * n.pos.pb + l * n.pos.pl + u.axis * n.pos.pa), f, c, s);
      const T *xp = x + b * n.xb + l * n.xl, *gp = g + b * n.gb + l * n.gl;
      T* yp = dx + m * n.H * n.D;
      for (int h = 0; h < n.H; ++h) {
        float p[W], q[W] = {};
        load_run<T, W>(gp + h * n.gh + u.e0, p);
        if (u.second) load_run<T, W>(gp + h * n.gh + u.e1, q);
        if (u.axis >= 0) {
          float a[W], e[W];
          load_run<T, W>(xp + h * n.xh + u.e0, a);
          load_run<T, W>(xp + h * n.xh + u.e1, e);
          turn_runs<W, true>(p, q, c, s, n.r.interleaved);
          add_pairs<W>(sum, p, q, a, e, n.r.interleaved);
        }
        store_run<T, W>(yp + (long long)h * n.D + u.e0, p);
        if (u.second) store_run<T, W>(yp + (long long)h * n.D + u.e1, q);
      }
      constexpr float kHalfPi = 1.57079632679489662f;   // a quarter turn
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) t = fmaf(sum[j], (float)f[j], t);
      part[flip][threadIdx.x] = t * kHalfPi;
    }
    __syncthreads();   // the other half is read before the next one, so one barrier a round does
    const int row = threadIdx.x / n.by_axes, a = threadIdx.x - row * n.r.axes;
    if (row < n.rows && m0 + row < n.M) {
      int u0 = 0;
      for (int i = 0; i < a; ++i) u0 += n.r.dims[i] / 2 / W;
      const int nu = n.r.dims[a] / 2 / W;
      float t = 0.f;
      for (int i = 0; i < nu; ++i) t += part[flip][row * n.units + u0 + i];
      dpos[(m0 + row) * n.r.axes + a] = t;
    }
  }
}

// dpos[l, a] = sum over the images of part[b, l, a], in their order.
__global__ __launch_bounds__(kThreads) void k_rotary_join(const float* __restrict__ part, float* __restrict__ dpos, int B,
                                                          long long n) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  float t = 0.f;
  for (int b = 0; b < B; ++b) t += part[b * n + i];
  dpos[i] = t;
}

struct Append {
  splat_cache c;
  splat_rotation r;
  splat_positions pos;
  long long kb, kl, kh, vb, vl, vh, mb, ml;   // strides of the new keys, values and key mask
  const unsigned char* mask;                  // [B, T], 0: the token is left out; or null
  int T, M;                                   // M = B T tokens
  int units, hs, rows;
  FastDiv by_T, by_units, by_row, by_page;
};

// New token t of sequence b goes to place lengths[b] - counts[b] + t of its pages; tokens past the count, before the
// sequence's first place, behind its table or on a page that is none are left out.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void k_append(Append n, const T* __restrict__ k, const T* __restrict__ v) {
  const Seat at = seat(n.units, n.hs, n.rows, n.by_units, n.by_row);
  if (!at.in) return;
  const PairUnit u = pair_unit<W>(n.r, n.c.D, at.u);
  double f[W];
  rates<W>(n.r, u, f);
  const long long room = (long long)n.c.page * n.c.width;
  for (long long m = (long long)blockIdx.x * n.rows + at.row; m < n.M; m += (long long)gridDim.x * n.rows) {
    const int b = (int)m / n.by_T, t = (int)m - b * n.T, fresh = new_tokens(n.c, b, n.T);
    const long long slot = (long long)n.c.lengths[b] - fresh + t;
    if (t >= fresh || slot < 0 || slot >= room) continue;
    const int index = (int)slot / n.by_page, page = n.c.tables[b * n.c.tb + index], off = (int)slot - index * n.c.page;
    if (page < 0 || page >= n.c.pages) continue;
    float c[W], s[W];
    if (u.axis >= 0) angles<W>(position(n.pos, b * n.pos.pb + t * n.pos.pl + u.axis * n.pos.pa), f, c, s);
    const T *kp = k + b * n.kb + t * n.kl, *vp = v + b * n.vb + t * n.vl;
    T* ko = (T*)n.c.k + page * n.c.kp + off * n.c.kt;
    T* vo = (T*)n.c.v + page * n.c.vp + off * n.c.vt;
    for (int h = at.h; h < n.c.Hk; h += n.hs) {
      float p[W], q[W] = {};
      T v0[W], v1[W];
      load_run<T, W>(kp + h * n.kh + u.e0, p);
      __builtin_memcpy(v0, vp + h * n.vh + u.e0, sizeof(v0));
      if (u.second) {
        load_run<T, W>(kp + h * n.kh + u.e1, q);
        __builtin_memcpy(v1, vp + h * n.vh + u.e1, sizeof(v1));
      }
      if (u.axis >= 0) turn_runs<W, false>(p, q, c, s, n.r.interleaved);
      store_run<T, W>(ko + h * n.c.kh + u.e0, p);
      __builtin_memcpy(vo + h * n.c.vh + u.e0, v0, sizeof(v0));
      if (u.second) {
        store_run<T, W>(ko + h * n.c.kh + u.e1, q);
        __builtin_memcpy(vo + h * n.c.vh + u.e1, v1, sizeof(v1));
      }
    }
    if (n.c.live && at.u == 0 && at.h == 0)
      n.c.live[page * n.c.lp + off * n.c.lt] = !n.mask || n.mask[b * n.mb + t * n.ml] != 0;
  }
}

// Threads of a token and tokens of a workgroup: as many heads side by side as fit.
template <typename N>
void seats(N& n, const Units& u, int H, bool one) {
  n.units = u.n;
  n.hs = one ? 1 : std::min(H, std::max(1, kThreads / u.n));
  n.rows = kThreads / (n.units * n.hs);
  n.by_units = fast_div(n.units);
  n.by_row = fast_div(n.units * n.hs);
}

template <typename F>
int with_run(int dtype, int W, F&& f) {
  auto width = [&](auto t) {
    switch (W) {
      case 8: return sizeof(t) == 2 ? f(t, std::integral_constant<int, sizeof(t) == 2 ? 8 : 4>{}) : -1;
      case 4: return f(t, std::integral_constant<int, 4>{});
      case 2: return f(t, std::integral_constant<int, 2>{});
    }
    return f(t, std::integral_constant<int, 1>{});
  };
  return dtype == kF32 ? width(float{}) : width(bf16{});
}

int plan_turn(const char* who, const splat_rotation* r, const splat_positions* p, int dtype, int B, long long L, int H, int D,
              bool one, Turn* n, Units* u) {
  if (dtype != kF32 && dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", who, dtype);
  if (B < 0 || L < 0 || H < 1 || D < 1) return set_error(kInvalid, "%s: B %d, L %lld, H %d, D %d", who, B, L, H, D);
  if (D > kMaxHead) return set_error(kUnsupported, "%s: heads of %d values, %d at most", who, D, kMaxHead);
  if (L > 0x7fffffffLL || B * L > 0x7fffffffLL) return set_error(kUnsupported, "%s: %d x %lld tokens", who, B, L);
  if (!r) return set_error(kInvalid, "%s: no rotation", who);
  if (const int rc = check_rotation(who, r, p, D)) return rc;
  n->r = *r;
  n->pos = p ? *p : splat_positions{};
  n->B = B;
  n->L = (int)L;
  n->H = H;
  n->D = D;
  n->M = (int)(B * L);
  *u = pair_units(*r, D, dtype == kF32 ? 4 : 8);
  seats(*n, *u, H, one);
  n->by_L = fast_div(std::max(1, n->L));
  n->by_axes = fast_div(std::max(1, r->axes));
  return kOk;
}

template <typename N>
unsigned grid_of(const N& n) { return (unsigned)std::min<long long>(kGrid, div_up(n.M, n.rows)); }

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

int splat_rotary(const splat_rotation* r, const splat_positions* p, const void* x, long long xb, long long xl, long long xh,
                 int dtype, int B, long long L, int H, int D, int back, void* y, void* stream) {
  Turn n{};
  Units u;
  if (const int rc = plan_turn("splat_rotary", r, p, dtype, B, L, H, D, false, &n, &u)) return rc;
  if (n.M == 0) return kOk;
  if (!x || !y) return set_error(kInvalid, "splat_rotary: null pointer");
  n.xb = xb, n.xl = xl, n.xh = xh;
  return with_run(dtype, u.W, [&](auto t, auto w) {
    using T = decltype(t);
    constexpr int W = decltype(w)::value;
    (back ? k_rotary<T, W, true> : k_rotary<T, W, false>)<<<grid_of(n), kThreads, 0, (hipStream_t)stream>>>(n, (const T*)x,
                                                                                                           (T*)y);
    return check_launch("splat_rotary");
  });
}

size_t splat_rotary_bwd_workspace_bytes(int B, long long L, int axes, int shared) {
  return shared && B > 1 && L > 0 && axes > 0 ? sizeof(float) * B * L * axes : 0;
}

int splat_rotary_bwd(const splat_rotation* r, const splat_positions* p, const void* x, long long xb, long long xl, long long xh,
                     const void* g, long long gb, long long gl, long long gh, int dtype, int B, long long L, int H, int D,
                     void* dx, float* dpos, int shared, void* ws, size_t ws_bytes, void* stream) {
  Turn n{};
  Units u;
  if (const int rc = plan_turn("splat_rotary_bwd", r, p, dtype, B, L, H, D, true, &n, &u)) return rc;
  if (!r->axes) return set_error(kInvalid, "splat_rotary_bwd: no axes");
  if (n.M == 0) return kOk;
  if (!x || !g || !dx || !dpos) return set_error(kInvalid, "splat_rotary_bwd: null pointer");
  const size_t need = splat_rotary_bwd_workspace_bytes(B, L, r->axes, shared);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_rotary_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  n.xb = xb, n.xl = xl, n.xh = xh, n.gb = gb, n.gl = gl, n.gh = gh;
  float* each = need ? (float*)ws : dpos;
  return with_run(dtype, u.W, [&](auto t, auto w) {
    using T = decltype(t);
    constexpr int W = decltype(w)::value;
    k_rotary_bwd<T, W><<<grid_of(n), kThreads, 0, (hipStream_t)stream>>>(n, (const T*)x, (const T*)g, (T*)dx, each);
    if (need) {
      const long long m = L * r->axes;
      k_rotary_join<<<(unsigned)div_up(m, kThreads), kThreads, 0, (hipStream_t)stream>>>(each, dpos, B, m);
    }
    return check_launch("splat_rotary_bwd");
  });
}

int splat_cache_append(const splat_cache* c, const splat_rotation* r, const splat_positions* p, const void* k, long long kb,
                       long long kl, long long kh, const void* v, long long vb, long long vl, long long vh,
                       const unsigned char* mask, long long mb, long long ml, long long T, void* stream) {
  if (const int rc = check_cache("splat_cache_append", c)) return rc;
  if (T < 0) return set_error(kInvalid, "splat_cache_append: %lld tokens", T);
  if (T > 0x7fffffffLL || c->B * T > 0x7fffffffLL) return set_error(kUnsupported, "splat_cache_append: %d x %lld tokens", c->B, T);
  if (const int rc = check_rotation("splat_cache_append", r, p, c->D)) return rc;
  if (mask && !c->live) return set_error(kInvalid, "splat_cache_append: a key mask for a cache without one");
  if (c->B == 0 || T == 0 || c->pages == 0 || c->width == 0) return kOk;
  if (!k || !v) return set_error(kInvalid, "splat_cache_append: null pointer");
  Append n{};
  n.c = *c;
  if (r) n.r = *r;
  if (p) n.pos = *p;
  n.kb = kb, n.kl = kl, n.kh = kh, n.vb = vb, n.vl = vl, n.vh = vh, n.mask = mask, n.mb = mb, n.ml = ml;
  n.T = (int)T;
  n.M = (int)(c->B * T);
  const Units u = pair_units(n.r, c->D, c->dtype == kF32 ? 4 : 8);
  seats(n, u, c->Hk, false);
  n.by_T = fast_div(n.T);
  n.by_page = fast_div(c->page);
  return with_run(c->dtype, u.W, [&](auto t, auto w) {
    using E = decltype(t);
    k_append<E, decltype(w)::value><<<grid_of(n), kThreads, 0, (hipStream_t)stream>>>(n, (const E*)k, (const E*)v);
    return check_launch("splat_cache_append");
  });
}

}  // extern "C"
