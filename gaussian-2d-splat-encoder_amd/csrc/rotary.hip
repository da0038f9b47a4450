// Rotary positions of several axes, x[B, L, H, D] -> y, and new tokens' keys (turned on the way) and values into a paged cache.
//
// Pair i of axis a turns by w = p_a * quarters[pair] quarter turns: (y0, y1) = (x0 cos w - x1 sin w, x0 sin w + x1 cos w). The
// input's gradient is the same turn back; dw = g1 y0 - g0 y1 = dx1 x0 - dx0 x1 (both turned back together), summed over heads
// and an axis' pairs for the positions' gradient.
//
// All of it is bound by memory. A thread has a unit of W pairs (16 bytes a run where the axes allow it) of a token, computes
// their angles once in 64 bits and turns the unit in several heads; a token's threads lie side by side, so that a wave's loads
// cover whole heads. Measured (a large copy moves 4.9 TB/s here): 147,456 tokens of 4 heads of 64 bf16 35 us each way (4.3
// TB/s); 92,160 tokens of 4 heads of 64 bf16 appended 48 us (3.9 TB/s), whose writes go to a page and head of their own each.
#include <algorithm>

#include "token_common.h"

namespace splat {
namespace {

constexpr int kThreads = 256;
constexpr int kGrid = 1 << 16;   // workgroups at most

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

// Cosines and sines of a unit's pairs at the position of token l of image b.
template <int W>
__device__ __forceinline__ void angles(const splat_rotation& r, const splat_positions& pos, const PairUnit& u, int b, int l,
                                       float (&c)[W], float (&s)[W]) {
  const double p = position(pos, b * pos.pb + l * pos.pl + u.axis * pos.pa);
#pragma unroll
  for (int j = 0; j < W; ++j) turn(p, r.quarters[u.pair + j], c[j], s[j]);
}

// A unit of HB heads of a tensor, `step` heads apart from h on, as it lies in memory. Loads have no conditions, so that all are
// under way at once: heads past the last are the last one, a run that is none the first.
template <typename T, int W, int HB>
struct Runs {
  T a[HB][W], b[HB][W];
  __device__ __forceinline__ void load(const T* p, long long sh, const PairUnit& u, int h, int step, int H) {
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const T* at = p + min(h + i * step, H - 1) * sh;
      __builtin_memcpy(a[i], at + u.e0, sizeof(a[i]));
      __builtin_memcpy(b[i], at + (u.second ? u.e1 : u.e0), sizeof(b[i]));
    }
  }
  __device__ __forceinline__ void get(int i, float (&p)[W], float (&q)[W]) const {
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = (float)a[i][j], q[j] = (float)b[i][j];
  }
  __device__ __forceinline__ void put(int i, T* p, T* q, bool second) const {
    T x[W], y[W];
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = a[i][j], y[j] = b[i][j];
    __builtin_memcpy(p, x, sizeof(x));
    if (second) __builtin_memcpy(q, y, sizeof(y));
  }
};

// y = x turned (Back: turned back), HB heads at a time.
template <typename T, int W, int HB, bool Back>
__global__ __launch_bounds__(kThreads) void k_rotary(Turn n, const T* __restrict__ x, T* __restrict__ y) {
  const Seat at = seat(n.units, n.hs, n.rows, n.by_units, n.by_row);
  if (!at.in) return;
  const PairUnit u = pair_unit<W>(n.r, n.D, at.u);
  for (long long m = (long long)blockIdx.x * n.rows + at.row; m < n.M; m += (long long)gridDim.x * n.rows) {
    const int b = (int)m / n.by_L, l = (int)m - b * n.L;
    const T* xp = x + b * n.xb + l * n.xl;
    T* yp = y + m * n.H * n.D;
    float c[W], s[W];
    for (int h0 = at.h; h0 < n.H; h0 += HB * n.hs) {
      Runs<T, W, HB> r;
      r.load(xp, n.xh, u, h0, n.hs, n.H);
      if (u.axis >= 0 && h0 == at.h) angles<W>(n.r, n.pos, u, b, l, c, s);
#pragma unroll
      for (int i = 0; i < HB; ++i) {
        const int h = h0 + i * n.hs;
        if (HB > 1 && h >= n.H) continue;
        float p[W], q[W];
        r.get(i, p, q);
        if (u.axis >= 0) turn_runs<W, Back>(p, q, c, s, n.r.interleaved);
        store_run<T, W>(yp + (long long)h * n.D + u.e0, p);
        if (u.second) store_run<T, W>(yp + (long long)h * n.D + u.e1, q);
      }
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
template <typename T, int W, int HB>
__global__ __launch_bounds__(kThreads) void k_rotary_bwd(Turn n, const T* __restrict__ x, const T* __restrict__ g,
                                                         T* __restrict__ dx, float* __restrict__ dpos) {
  __shared__ float part[2][kThreads];
  const Seat at = seat(n.units, 1, n.rows, n.by_units, n.by_row);
  const PairUnit u = pair_unit<W>(n.r, n.D, at.u);
  int flip = 0;
  for (long long m0 = (long long)blockIdx.x * n.rows; m0 < n.M; m0 += (long long)gridDim.x * n.rows, flip ^= 1) {
    const long long m = m0 + at.row;
    if (at.in && m < n.M) {
      const int b = (int)m / n.by_L, l = (int)m - b * n.L;
      float c[W], s[W], sum[W] = {};
      if (u.axis >= 0) angles<W>(n.r, n.pos, u, b, l, c, s);
      const T *xp = x + b * n.xb + l * n.xl, *gp = g + b * n.gb + l * n.gl;
      T* yp = dx + m * n.H * n.D;
      for (int h0 = 0; h0 < n.H; h0 += HB) {
        Runs<T, W, HB> gr, xr;
        gr.load(gp, n.gh, u, h0, 1, n.H);
        if (u.axis >= 0) xr.load(xp, n.xh, u, h0, 1, n.H);
#pragma unroll
        for (int i = 0; i < HB; ++i) {
          const int h = h0 + i;
          if (HB > 1 && h >= n.H) continue;
          float p[W], q[W], a[W], e[W];
          gr.get(i, p, q);
          if (u.axis >= 0) {
            xr.get(i, a, e);
            turn_runs<W, true>(p, q, c, s, n.r.interleaved);
            add_pairs<W>(sum, p, q, a, e, n.r.interleaved);
          }
          store_run<T, W>(yp + (long long)h * n.D + u.e0, p);
          if (u.second) store_run<T, W>(yp + (long long)h * n.D + u.e1, q);
        }
      }
      constexpr float kHalfPi = 1.57079632679489662f;   // a quarter turn
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) t = fmaf(sum[j], u.axis >= 0 ? (float)n.r.quarters[u.pair + j] : 0.f, t);
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
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kThreads) {
    float t = 0.f;
    for (int b = 0; b < B; ++b) t += part[b * n + i];
    dpos[i] = t;
  }
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
template <typename T, int W, int HB>
__global__ __launch_bounds__(kThreads) void k_append(Append n, const T* __restrict__ k, const T* __restrict__ v) {
  const Seat at = seat(n.units, n.hs, n.rows, n.by_units, n.by_row);
  if (!at.in) return;
  const PairUnit u = pair_unit<W>(n.r, n.c.D, at.u);
  const long long room = (long long)n.c.page * n.c.width;
  for (long long m = (long long)blockIdx.x * n.rows + at.row; m < n.M; m += (long long)gridDim.x * n.rows) {
    const int b = (int)m / n.by_T, t = (int)m - b * n.T;
    const T *kp = k + b * n.kb + t * n.kl, *vp = v + b * n.vb + t * n.vl;
    Runs<T, W, HB> kr, vr;
    kr.load(kp, n.kh, u, at.h, n.hs, n.c.Hk);
    vr.load(vp, n.vh, u, at.h, n.hs, n.c.Hk);
    const int fresh = new_tokens(n.c, b, n.T);
    const long long slot = (long long)n.c.lengths[b] - fresh + t;
    if (t >= fresh || slot < 0 || slot >= room) continue;
    const int index = (int)slot / n.by_page, page = n.c.tables[b * n.c.tb + index], off = (int)slot - index * n.c.page;
    float c[W], s[W];
    if (u.axis >= 0) angles<W>(n.r, n.pos, u, b, t, c, s);
    if (page < 0 || page >= n.c.pages) continue;
    T* ko = (T*)n.c.k + page * n.c.kp + off * n.c.kt;
    T* vo = (T*)n.c.v + page * n.c.vp + off * n.c.vt;
    for (int h0 = at.h;;) {
#pragma unroll
      for (int i = 0; i < HB; ++i) {
        const int h = h0 + i * n.hs;
        if (HB > 1 && h >= n.c.Hk) continue;
        float p[W], q[W];
        kr.get(i, p, q);
        if (u.axis >= 0) turn_runs<W, false>(p, q, c, s, n.r.interleaved);
        store_run<T, W>(ko + h * n.c.kh + u.e0, p);
        vr.put(i, vo + h * n.c.vh + u.e0, vo + h * n.c.vh + u.e1, u.second);
        if (u.second) store_run<T, W>(ko + h * n.c.kh + u.e1, q);
      }
      h0 += HB * n.hs;
      if (h0 >= n.c.Hk) break;
      kr.load(kp, n.kh, u, h0, n.hs, n.c.Hk);
      vr.load(vp, n.vh, u, h0, n.hs, n.c.Hk);
    }
    if (n.c.live && at.u == 0 && at.h == 0)
      n.c.live[page * n.c.lp + off * n.c.lt] = !n.mask || n.mask[b * n.mb + t * n.ml] != 0;
  }
}

// Threads of a token and tokens of a workgroup. A thread turns several heads by the angles it computes once, two at a time, as
// long as `lanes` threads are left. Rotations, 2^18, 2^19 and 2^20, us: 36,864 tokens of 8 heads of 64 floats 34.1, 32.5, 34.2;
// 8,192 of 32 of 128 bf16 32.6, 29.3, 32.1; 4,096 of 16 of 64 floats 10.4, 11.1, 11.0. Appends: 8,192 of 8 of 128 bf16 15.2,
// 18.4, 18.4; 92,160 of 4 of 64 bf16 46.1, 45.1, 45.7; 36,864 of 8 of 64 floats 64.1, 61.1, 61.8. (Four heads at a time, or the
// next token's loads under way while one is turned, cost more waves than they gain.)
constexpr long long kTurnLanes = 1 << 19, kAppendLanes = 1 << 18;
template <typename N>
int seats(N& n, const Units& u, int H, long long lanes) {
  n.units = u.n;
  n.hs = 1;
  while (n.hs < H && (n.hs + 1) * u.n <= kThreads && (long long)n.M * u.n * n.hs < lanes) ++n.hs;
  n.rows = kThreads / (n.units * n.hs);
  n.by_units = fast_div(n.units);
  n.by_row = fast_div(n.units * n.hs);
  return H > n.hs ? 2 : 1;
}

template <typename F>
int with_run(int dtype, int W, int HB, F&& f) {
  using std::integral_constant;
  auto heads = [&](auto t, auto w) {
    return HB == 2 ? f(t, w, integral_constant<int, 2>{}) : f(t, w, integral_constant<int, 1>{});
  };
  auto width = [&](auto t) {
    switch (W) {
      case 8: return heads(t, integral_constant<int, sizeof(t) == 2 ? 8 : 4>{});   // floats: 4 at most
      case 4: return heads(t, integral_constant<int, 4>{});
      case 2: return heads(t, integral_constant<int, 2>{});
    }
    return heads(t, integral_constant<int, 1>{});
  };
  return dtype == kF32 ? width(float{}) : width(bf16{});
}

int plan_turn(const char* who, const splat_rotation* r, const splat_positions* p, int dtype, int B, long long L, int H, int D,
              bool one, Turn* n, Units* u, int* heads) {
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
  *heads = seats(*n, *u, H, one ? 0 : kTurnLanes);
  n->by_L = fast_div(std::max(1, n->L));
  n->by_axes = fast_div(std::max(1, r->axes));
  return kOk;
}

template <typename N>
unsigned grid_of(const N& n) { return (unsigned)std::min(kGrid, div_up(n.M, n.rows)); }

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

int splat_rotary(const splat_rotation* r, const splat_positions* p, const void* x, long long xb, long long xl, long long xh,
                 int dtype, int B, long long L, int H, int D, int back, void* y, void* stream) {
  Turn n{};
  Units u;
  int heads;
  if (const int rc = plan_turn("splat_rotary", r, p, dtype, B, L, H, D, false, &n, &u, &heads)) return rc;
  if (n.M == 0) return kOk;
  if (!x || !y) return set_error(kInvalid, "splat_rotary: null pointer");
  n.xb = xb, n.xl = xl, n.xh = xh;
  return with_run(dtype, u.W, heads, [&](auto t, auto w, auto hb) {
    using T = decltype(t);
    constexpr int W = decltype(w)::value, HB = decltype(hb)::value;
    (back ? k_rotary<T, W, HB, true> : k_rotary<T, W, HB, false>)<<<grid_of(n), kThreads, 0, (hipStream_t)stream>>>(
        n, (const T*)x, (T*)y);
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
  int heads;
  if (const int rc = plan_turn("splat_rotary_bwd", r, p, dtype, B, L, H, D, true, &n, &u, &heads)) return rc;
  if (!r->axes) return set_error(kInvalid, "splat_rotary_bwd: no axes");
  if (n.M == 0) return kOk;
  if (!x || !g || !dx || !dpos) return set_error(kInvalid, "splat_rotary_bwd: null pointer");
  const size_t need = splat_rotary_bwd_workspace_bytes(B, L, r->axes, shared);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_rotary_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  n.xb = xb, n.xl = xl, n.xh = xh, n.gb = gb, n.gl = gl, n.gh = gh;
  float* each = need ? (float*)ws : dpos;
  return with_run(dtype, u.W, heads, [&](auto t, auto w, auto hb) {
    using T = decltype(t);
    constexpr int W = decltype(w)::value, HB = decltype(hb)::value;
    k_rotary_bwd<T, W, HB><<<grid_of(n), kThreads, 0, (hipStream_t)stream>>>(n, (const T*)x, (const T*)g, (T*)dx, each);
    if (need) {
      const long long m = L * r->axes;
      k_rotary_join<<<(unsigned)std::min(kGrid, div_up(m, kThreads)), kThreads, 0, (hipStream_t)stream>>>(each, dpos, B, m);
    }
    return check_launch("splat_rotary_bwd");
  });
}

int splat_cache_append(const splat_cache* c, const splat_rotation* r, const splat_positions* p, const void* k, long long kb,
                       long long kl, long long kh, const void* v, long long vb, long long vl, long long vh,
                       const unsigned char* mask, long long mb, long long ml, long long T, void* stream) {
  if (const int rc = check_cache("splat_cache_append", c)) return rc;
  if (T < 0) return set_error(kInvalid, "splat_cache_append: %lld tokens", T);
  if (T > 0x7fffffffLL || c->B * T > 0x7fffffffLL)
    return set_error(kUnsupported, "splat_cache_append: %d x %lld tokens", c->B, T);
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
  const int heads = seats(n, u, c->Hk, kAppendLanes);
  n.by_T = fast_div(n.T);
  n.by_page = fast_div(c->page);
  return with_run(c->dtype, u.W, heads, [&](auto t, auto w, auto hb) {
    using E = decltype(t);
    k_append<E, decltype(w)::value, decltype(hb)::value><<<grid_of(n), kThreads, 0, (hipStream_t)stream>>>(n, (const E*)k,
                                                                                                           (const E*)v);
    return check_launch("splat_cache_append");
  });
}

}  // extern "C"
