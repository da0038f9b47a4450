// Group norm with an activation on channels-last maps x[B, L, C] (L positions), forward and backward.
//
//   act_first: u = act(x), y = w (u - mean) rstd + b;     otherwise: u = x, y = act(w (u - mean) rstd + b)
//
// with mean and rstd = 1 / sqrt(var + eps) over the C / G channels of a group and all positions of an image.
//
// A workgroup covers a channel tile (whole groups, or a part of one group wider than a tile) and a range of positions:
// thread (rt, cc) holds the 16-byte chunk cc of the tile's channels at the positions rt, rt + RT, ... Both directions are
// bound by memory. Where one workgroup's registers hold a group, everything is one launch that reads x once; otherwise
// one launch reduces each range to partial sums and a second one joins them and writes the result, x coming from
// the caches the second time where it fits them.
#include "feat_common.h"

namespace splat {
namespace {

constexpr int kThreads = 512;
constexpr int kKeep = 16;   // chunks of x that a thread keeps in registers in the one-launch forward

struct Norm {
  long long L, xsb, xsl, gsb, gsl;   // positions; strides of x and of dy per image and position (channels are dense)
  int B, C, G, Cg;
  int Ct, tiles, tpg;                // channels of a tile; tiles; tiles of one group (1 unless a group passes a tile)
  int nch, RT;                       // chunks of a tile; positions a workgroup takes at a time
  int splits;                        // ranges of positions
  long long per;                     // positions of a range
  float eps;
};

// A thread's place: its channels [c, c + nv) of the map and its first position rt.
struct Place {
  int rt, cc, c, nv, c0, ct;   // c0, ct: the tile's first channel and its channels
  bool on;
};

template <typename T>
__device__ __forceinline__ Place place(const Norm& n, int tile) {
  Place p;
  if (n.tpg == 1) {
    p.c0 = tile * n.Ct;
    p.ct = min(n.Ct, n.C - p.c0);
  } else {
    const int g = tile / n.tpg, k = tile % n.tpg;
    p.c0 = g * n.Cg + k * n.Ct;
    p.ct = min(n.Ct, n.Cg - k * n.Ct);
  }
  p.rt = threadIdx.x / n.nch;
  p.cc = threadIdx.x % n.nch;
  p.c = p.c0 + p.cc * kV<T>;
  p.nv = min(kV<T>, p.ct - p.cc * kV<T>);
  p.on = p.rt < n.RT && p.nv > 0;
  return p;
}

// The tile's groups: the first one and how many (1 where the tile is a part of one group).
__device__ __forceinline__ int tile_groups(const Norm& n, const Place& p, int* g0) {
  *g0 = p.c0 / n.Cg;
  return n.tpg == 1 ? p.ct / n.Cg : 1;
}

// Group of the thread's channel j within the tile.
__device__ __forceinline__ int group_of(const Norm& n, const Place& p, int j) {
  return n.tpg == 1 ? (p.c - p.c0 + j) / n.Cg : 0;
}

// out[g] = sum over the workgroup's threads and the channels of group g of v. One value per thread goes through LDS
// where no chunk meets two groups, one per channel otherwise; either way a group's values lie next to each other
// (channel-major), and one wave adds them in a fixed order. `red` holds kThreads * kV floats.
template <typename T>
__device__ __forceinline__ void group_sums(const Norm& n, const Place& p, int ng, const float* v, float* red, float* out) {
  const bool whole = n.Cg % kV<T> == 0 || n.tpg > 1;
  __syncthreads();
  if (threadIdx.x < (unsigned)(n.RT * n.nch)) {
    if (whole) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) s += v[j];
      red[p.cc * n.RT + p.rt] = s;
    } else {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) red[(p.cc * kV<T> + j) * n.RT + p.rt] = v[j];
    }
  }
  __syncthreads();
  const int seg = n.tpg > 1 ? n.nch * n.RT : (whole ? n.Cg / kV<T> : n.Cg) * n.RT;
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < ng; g += kThreads / 64) {
    float s = 0.f;
    for (int e = lane; e < seg; e += 64) s += red[g * seg + e];
    s = wave_sum(s);
    if (lane == 0) out[g] = s;
  }
  __syncthreads();
}

__device__ __forceinline__ long long rows_of(long long lo, long long hi, int rt, int RT) {
  const long long r = hi - lo - rt;
  return r <= 0 ? 0 : (r + RT - 1) / RT;
}

template <typename T, int A, bool First>
__device__ __forceinline__ float pre(T x) {
  return First ? act_fwd<A, T>((float)x) : (float)x;
}

template <typename T, int A, bool First>
__device__ __forceinline__ T post(float u, float mean, float a, float b) {
  const float z = fmaf(u - mean, a, b);
  return (T)(First ? z : act_fwd<A, T>(z));
}

// Per-channel scale (rstd w) and shift of a thread's chunk, and its groups' means.
template <typename T>
__device__ __forceinline__ void affine(const Norm& n, const Place& p, const float* gmean, const float* grstd,
                                       const float* w, const float* b, float* m, float* a, float* s) {
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const bool in = p.on && j < p.nv;
    const int g = in ? group_of(n, p, j) : 0;
    m[j] = gmean[g];
    a[j] = in ? (w ? w[p.c + j] : 1.f) * grstd[g] : 0.f;
    s[j] = in && b ? b[p.c + j] : 0.f;
  }
}

// Statistics and result in one launch, one workgroup per image and tile of whole groups: x stays in registers between
// the two sums (the mean, then the squared deviations from it) and the result.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_whole(Norm n, const T* __restrict__ x, const float* __restrict__ w,
                                                         const float* __restrict__ b, T* __restrict__ y,
                                                         float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[kThreads * kV<T>], gm[kThreads * kV<T>], gr[kThreads * kV<T>];
  const int img = blockIdx.y;
  const Place p = place<T>(n, blockIdx.x);
  int g0;
  const int ng = tile_groups(n, p, &g0);
  const int rows = p.on ? (int)rows_of(0, n.L, p.rt, n.RT) : 0;
  const T* xp = x + (long long)img * n.xsb + (long long)p.rt * n.xsl + p.c;
  Chunk<T> keep[kKeep];
  float v[kV<T>] = {};
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    if (i < rows) keep[i] = load_chunk(xp + (long long)i * n.RT * n.xsl, p.nv);
  }
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    if (i < rows) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j)
        if (j < p.nv) v[j] += pre<T, A, First>(keep[i].v[j]);
    }
  }
  const float inv = 1.f / ((float)n.L * (float)n.Cg);
  group_sums<T>(n, p, ng, v, red, gm);
  for (int g = threadIdx.x; g < ng; g += kThreads) gm[g] *= inv;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) v[j] = 0.f;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    if (i < rows) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) {
        if (j < p.nv) {
          const float d = pre<T, A, First>(keep[i].v[j]) - gm[group_of(n, p, j)];
          v[j] = fmaf(d, d, v[j]);
        }
      }
    }
  }
  group_sums<T>(n, p, ng, v, red, gr);
  for (int g = threadIdx.x; g < ng; g += kThreads) {
    const float r = 1.f / sqrtf(gr[g] * inv + n.eps);
    gr[g] = r;
    if (mean) {
      mean[(long long)img * n.G + g0 + g] = gm[g];
      rstd[(long long)img * n.G + g0 + g] = r;
    }
  }
  __syncthreads();
  float m[kV<T>], a[kV<T>], s[kV<T>];
  affine<T>(n, p, gm, gr, w, b, m, a, s);
  T* yp = y + ((long long)img * n.L + p.rt) * n.C + p.c;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    if (i < rows) {
      Chunk<T> o;
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) o.v[j] = post<T, A, First>(pre<T, A, First>(keep[i].v[j]), m[j], a[j], s[j]);
      store_chunk(yp + (long long)i * n.RT * n.C, o, p.nv);
    }
  }
}

// Partial statistics of one range: (count, mean, squared deviations from it) per group. Each thread's sums are taken
// about its own first value of the channel, so that a mean far from zero costs no digits.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_stats(Norm n, const T* __restrict__ x, float* __restrict__ part) {
  __shared__ float red[kThreads * kV<T>], gm[kThreads * kV<T>], gq[kThreads * kV<T>];
  const int img = blockIdx.z, split = blockIdx.x;
  const Place p = place<T>(n, blockIdx.y);
  int g0;
  const int ng = tile_groups(n, p, &g0);
  const long long lo = (long long)split * n.per, hi = min(n.L, lo + n.per);
  const int rows = p.on ? (int)rows_of(lo, hi, p.rt, n.RT) : 0;
  const T* xp = x + (long long)img * n.xsb + (lo + p.rt) * n.xsl + p.c;
  const long long step = (long long)n.RT * n.xsl;
  float k0[kV<T>], s[kV<T>] = {}, q[kV<T>] = {};
  if (rows > 0) {
    const Chunk<T> c = load_chunk(xp, p.nv);
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) k0[j] = pre<T, A, First>(c.v[j]);
#pragma unroll 4
    for (int i = 1; i < rows; ++i) {
      const Chunk<T> d = load_chunk(xp + i * step, p.nv);
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) {
        const float u = pre<T, A, First>(d.v[j]) - k0[j];
        s[j] += u;
        q[j] = fmaf(u, u, q[j]);
      }
    }
  }
  const float cnt = (float)rows, icnt = rows > 0 ? 1.f / cnt : 0.f;
  float v[kV<T>];
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const bool in = rows > 0 && j < p.nv;
    k0[j] = in ? fmaf(s[j], icnt, k0[j]) : 0.f;                // the thread's mean
    q[j] = in ? fmaxf(q[j] - s[j] * s[j] * icnt, 0.f) : 0.f;   // its squared deviations (NaN: below)
    if (in && s[j] != s[j]) q[j] = s[j];
    v[j] = in ? cnt * k0[j] : 0.f;
  }
  group_sums<T>(n, p, ng, v, red, gm);
  const float total = (float)(hi - lo) * (float)(n.tpg == 1 ? n.Cg : p.ct);
  for (int g = threadIdx.x; g < ng; g += kThreads) gm[g] /= total;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const bool in = rows > 0 && j < p.nv;
    const float d = in ? k0[j] - gm[group_of(n, p, j)] : 0.f;
    v[j] = in ? fmaf(cnt * d, d, q[j]) : 0.f;
  }
  group_sums<T>(n, p, ng, v, red, gq);
  const int slots = n.splits * n.tpg, slot = split * n.tpg + (n.tpg > 1 ? blockIdx.y % n.tpg : 0);
  for (int g = threadIdx.x; g < ng; g += kThreads) {
    float* o = part + 3 * (((long long)img * n.G + g0 + g) * slots + slot);
    o[0] = total;
    o[1] = gm[g];
    o[2] = gq[g];
  }
}

// Joins the partial statistics of the tile's groups (one wave a group), then writes the result of one range.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_apply(Norm n, const T* __restrict__ x, const float* __restrict__ w,
                                                         const float* __restrict__ b, const float* __restrict__ part,
                                                         T* __restrict__ y, float* __restrict__ mean,
                                                         float* __restrict__ rstd) {
  __shared__ float gm[kThreads * kV<T>], gr[kThreads * kV<T>];
  const int img = blockIdx.z, split = blockIdx.x;
  const Place p = place<T>(n, blockIdx.y);
  int g0;
  const int ng = tile_groups(n, p, &g0);
  const int slots = n.splits * n.tpg;
  const int lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)n.L * (float)n.Cg);
  for (int g = threadIdx.x >> 6; g < ng; g += kThreads / 64) {
    const float* o = part + 3 * ((long long)img * n.G + g0 + g) * slots;
    float s = 0.f;
    for (int e = lane; e < slots; e += 64) s = fmaf(o[3 * e], o[3 * e + 1], s);
    const float m = wave_sum(s) * inv;
    float q = 0.f;
    for (int e = lane; e < slots; e += 64) {
      const float d = o[3 * e + 1] - m;
      q += fmaf(o[3 * e] * d, d, o[3 * e + 2]);
    }
    const float r = 1.f / sqrtf(wave_sum(q) * inv + n.eps);
    if (lane == 0) {
      gm[g] = m;
      gr[g] = r;
      if (mean && split == 0 && (n.tpg == 1 || blockIdx.y % n.tpg == 0)) {
        mean[(long long)img * n.G + g0 + g] = m;
        rstd[(long long)img * n.G + g0 + g] = r;
      }
    }
  }
  __syncthreads();
  const long long lo = (long long)split * n.per, hi = min(n.L, lo + n.per);
  const int rows = p.on ? (int)rows_of(lo, hi, p.rt, n.RT) : 0;
  float m[kV<T>], a[kV<T>], s[kV<T>];
  affine<T>(n, p, gm, gr, w, b, m, a, s);
  const T* xp = x + (long long)img * n.xsb + (lo + p.rt) * n.xsl + p.c;
  T* yp = y + ((long long)img * n.L + lo + p.rt) * n.C + p.c;
  const long long step = (long long)n.RT * n.xsl, ystep = (long long)n.RT * n.C;
#pragma unroll 4
  for (int i = 0; i < rows; ++i) {
    const Chunk<T> c = load_chunk(xp + i * step, p.nv);
    Chunk<T> o;
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) o.v[j] = post<T, A, First>(pre<T, A, First>(c.v[j]), m[j], a[j], s[j]);
    store_chunk(yp + i * ystep, o, p.nv);
  }
}

// g = dL/dz at the norm's output z (before the activation where that comes after), and the normalised input.
template <typename T, int A, bool First>
__device__ __forceinline__ float grad_at(float dy, float uhat, float wj, float bj) {
  return First ? dy : dy * act_grad<A, T>(fmaf(uhat, wj, bj));
}

// a b - c with the product rounded by itself: a group of one value has c = round(a b), and a zero difference.
__device__ __forceinline__ float rounded_product_less(float a, float b, float c) {
#pragma clang fp contract(off)
  const float p = a * b;
  return p - c;
}

// Backward sums of one range: per channel sum g and sum g uhat (`cpart`, for the parameters), per group the same weighted
// by w (`gpart`, for dx).
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_sums(Norm n, const T* __restrict__ x, const T* __restrict__ dy,
                                                            const float* __restrict__ w, const float* __restrict__ b,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, float* __restrict__ cpart,
                                                            float* __restrict__ gpart) {
  __shared__ float red[kThreads * kV<T>], ga[kThreads * kV<T>], gb[kThreads * kV<T>];
  const int img = blockIdx.z, split = blockIdx.x;
  const Place p = place<T>(n, blockIdx.y);
  int g0;
  const int ng = tile_groups(n, p, &g0);
  const long long lo = (long long)split * n.per, hi = min(n.L, lo + n.per);
  const int rows = p.on ? (int)rows_of(lo, hi, p.rt, n.RT) : 0;
  float m[kV<T>], r[kV<T>], wj[kV<T>], bj[kV<T>], sa[kV<T>] = {}, sb[kV<T>] = {};
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const bool in = p.on && j < p.nv;
    const long long g = (long long)img * n.G + g0 + (in ? group_of(n, p, j) : 0);
    m[j] = mean[g];
    r[j] = rstd[g];
    wj[j] = in && w ? w[p.c + j] : 1.f;
    bj[j] = in && b ? b[p.c + j] : 0.f;
  }
  const T* xp = x + (long long)img * n.xsb + (lo + p.rt) * n.xsl + p.c;
  const T* gp = dy + (long long)img * n.gsb + (lo + p.rt) * n.gsl + p.c;
  const long long step = (long long)n.RT * n.xsl, gstep = (long long)n.RT * n.gsl;
#pragma unroll 2
  for (int i = 0; i < rows; ++i) {
    const Chunk<T> c = load_chunk(xp + i * step, p.nv), d = load_chunk(gp + i * gstep, p.nv);
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) {
      if (j < p.nv) {
        const float uh = (pre<T, A, First>(c.v[j]) - m[j]) * r[j];
        const float g = grad_at<T, A, First>((float)d.v[j], uh, wj[j], bj[j]);
        sa[j] += g;
        sb[j] = fmaf(g, uh, sb[j]);
      }
    }
  }
  // per channel, over the workgroup's positions: channel-major in LDS, a few lanes a channel
  const int lanes = p.ct * 8 <= kThreads ? 8 : 1;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    __syncthreads();
    if (threadIdx.x < (unsigned)(n.RT * n.nch)) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) red[(p.cc * kV<T> + j) * n.RT + p.rt] = pass ? sb[j] : sa[j];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < (p.ct * lanes + 63) / 64 * 64; e += kThreads) {
      const int c = e / lanes;
      float s = 0.f;
      if (c < p.ct)
        for (int k = e % lanes; k < n.RT; k += lanes) s += red[c * n.RT + k];
      if (lanes == 8) {
        s += __shfl_xor(s, 1, 64);
        s += __shfl_xor(s, 2, 64);
        s += __shfl_xor(s, 4, 64);
      }
      if (c < p.ct && e % lanes == 0)
        cpart[(((long long)img * n.splits + split) * 2 + pass) * n.C + p.c0 + c] = s;
    }
  }
  float v[kV<T>];
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) v[j] = wj[j] * sa[j];
  group_sums<T>(n, p, ng, v, red, ga);
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) v[j] = wj[j] * sb[j];
  group_sums<T>(n, p, ng, v, red, gb);
  const int slots = n.splits * n.tpg, slot = split * n.tpg + (n.tpg > 1 ? blockIdx.y % n.tpg : 0);
  for (int g = threadIdx.x; g < ng; g += kThreads) {
    float* o = gpart + 2 * (((long long)img * n.G + g0 + g) * slots + slot);
    o[0] = ga[g];
    o[1] = gb[g];
  }
}

// dx of one range; in the workgroups past the maps' (blockIdx.z == B) the parameters' gradients, 32 channels each.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_apply(Norm n, const T* __restrict__ x, const T* __restrict__ dy,
                                                             const float* __restrict__ w, const float* __restrict__ b,
                                                             const float* __restrict__ mean,
                                                             const float* __restrict__ rstd,
                                                             const float* __restrict__ cpart,
                                                             const float* __restrict__ gpart, T* __restrict__ dx,
                                                             float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float ga[kThreads * kV<T>], gb[kThreads * kV<T>];
  const int img = blockIdx.z;
  if (img == n.B) {
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, nrow = kThreads / 32;
    for (int c0 = (blockIdx.y * gridDim.x + blockIdx.x) * 32; c0 < n.C; c0 += 32 * gridDim.x * gridDim.y) {
      const int c = c0 + lane;
      float a = 0.f, q = 0.f;
      if (c < n.C) {
        const long long R = (long long)n.B * n.splits;
        for (long long i = row; i < R; i += nrow) {
          a += cpart[2 * i * n.C + c];
          q += cpart[(2 * i + 1) * n.C + c];
        }
      }
      __syncthreads();
      ga[row * 32 + lane] = a;
      gb[row * 32 + lane] = q;
      __syncthreads();
      if (row == 0 && c < n.C) {
        for (int i = 1; i < nrow; ++i) {
          a += ga[i * 32 + lane];
          q += gb[i * 32 + lane];
        }
        if (db) db[c] = a;
        if (dw) dw[c] = q;
      }
    }
    return;
  }
  const int split = blockIdx.x;
  const Place p = place<T>(n, blockIdx.y);
  int g0;
  const int ng = tile_groups(n, p, &g0);
  const int slots = n.splits * n.tpg;
  const int lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)n.L * (float)n.Cg);
  for (int g = threadIdx.x >> 6; g < ng; g += kThreads / 64) {
    const float* o = gpart + 2 * ((long long)img * n.G + g0 + g) * slots;
    float s = 0.f, q = 0.f;
    for (int e = lane; e < slots; e += 64) {
      s += o[2 * e];
      q += o[2 * e + 1];
    }
    s = wave_sum(s);
    q = wave_sum(q);
    if (lane == 0) {
      ga[g] = s * inv;
      gb[g] = q * inv;
    }
  }
  __syncthreads();
  const long long lo = (long long)split * n.per, hi = min(n.L, lo + n.per);
  const int rows = p.on ? (int)rows_of(lo, hi, p.rt, n.RT) : 0;
  float m[kV<T>], r[kV<T>], wj[kV<T>], bj[kV<T>], s1[kV<T>], s2[kV<T>];
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const bool in = p.on && j < p.nv;
    const int gl = in ? group_of(n, p, j) : 0;
    const long long g = (long long)img * n.G + g0 + gl;
    m[j] = mean[g];
    r[j] = rstd[g];
    wj[j] = in && w ? w[p.c + j] : 1.f;
    bj[j] = in && b ? b[p.c + j] : 0.f;
    s1[j] = ga[gl];
    s2[j] = gb[gl];
  }
  const T* xp = x + (long long)img * n.xsb + (lo + p.rt) * n.xsl + p.c;
  const T* gp = dy + (long long)img * n.gsb + (lo + p.rt) * n.gsl + p.c;
  T* op = dx + ((long long)img * n.L + lo + p.rt) * n.C + p.c;
  const long long step = (long long)n.RT * n.xsl, gstep = (long long)n.RT * n.gsl, ostep = (long long)n.RT * n.C;
#pragma unroll 2
  for (int i = 0; i < rows; ++i) {
    const Chunk<T> c = load_chunk(xp + i * step, p.nv), d = load_chunk(gp + i * gstep, p.nv);
    Chunk<T> o;
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) {
      const float xv = (float)c.v[j];
      const float uh = (pre<T, A, First>(c.v[j]) - m[j]) * r[j];
      const float du = r[j] * (rounded_product_less(grad_at<T, A, First>((float)d.v[j], uh, wj[j], bj[j]), wj[j], s1[j]) -
                               uh * s2[j]);
      o.v[j] = (T)(First ? du * act_grad<A, T>(xv) : du);
    }
    store_chunk(op + i * ostep, o, p.nv);
  }
}

// The launch geometry of a call. whole: one workgroup holds its groups' values in registers.
template <typename T>
Norm plan(int B, long long L, int C, int G, bool want_whole, bool* whole) {
  Norm n{};
  constexpr int V = kV<T>;
  n.B = B; n.L = L; n.C = C; n.G = G; n.Cg = C / G;
  const int most = kThreads * V;   // channels that the threads of a workgroup hold at one position
  *whole = false;
  if (want_whole && n.Cg <= most) {
    // as few groups a workgroup as make 64-byte runs of a position's channels, for the most workgroups
    const int run = 64 / (int)sizeof(T);
    const int gpt = n.Cg >= run ? 1 : (run + n.Cg - 1) / n.Cg < G ? (run + n.Cg - 1) / n.Cg : G;
    const int nch = (gpt * n.Cg + V - 1) / V;
    const int RT = nch <= kThreads ? kThreads / nch : 0;
    if (RT > 0 && L <= (long long)RT * kKeep) {
      n.Ct = gpt * n.Cg; n.tpg = 1; n.tiles = (G + gpt - 1) / gpt; n.nch = nch; n.RT = RT;
      n.splits = 1; n.per = L;
      *whole = true;
      return n;
    }
  }
  if (n.Cg <= most) {
    int gpt = most / n.Cg < G ? most / n.Cg : G;
    while (gpt > 1 && (gpt * n.Cg + V - 1) / V > kThreads) --gpt;
    n.Ct = gpt * n.Cg; n.tpg = 1; n.tiles = (G + gpt - 1) / gpt;
  } else {
    n.Ct = most; n.tpg = (n.Cg + most - 1) / most; n.tiles = G * n.tpg;
  }
  n.nch = (n.Ct + V - 1) / V;
  n.RT = kThreads / n.nch;
  // about 512 workgroups, two per CU, of at least four passes over their threads' positions each
  const long long want = 512 / ((long long)B * n.tiles) > 0 ? 512 / ((long long)B * n.tiles) : 1;
  const long long room = (L + 4LL * n.RT - 1) / (4LL * n.RT);
  n.splits = (int)(want < room ? want : room);
  if (n.splits < 1) n.splits = 1;
  n.per = (L + n.splits - 1) / n.splits;
  n.splits = (int)((L + n.per - 1) / n.per);
  return n;
}

int check_norm(const char* what, int dtype, int B, long long L, int C, int G, int act) {
  if (dtype != kF32 && dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", what, dtype);
  if (B < 0 || L < 0 || C < 1 || G < 1 || C % G) return set_error(kInvalid, "%s: B %d, L %lld, C %d, G %d", what, B, L, C, G);
  if (act < 0 || act >= kActCount) return set_error(kInvalid, "%s: unknown activation %d", what, act);
  if (B > 65534 || L > 0x7fffffffLL * 4) return set_error(kUnsupported, "%s: %d images of %lld positions", what, B, L);
  return kOk;
}

template <typename F>
int with_type(int dtype, F&& f) {
  return dtype == kF32 ? f(float{}) : f(bf16{});
}

Norm plan_of(int dtype, int B, long long L, int C, int G, bool want_whole, bool* whole) {
  return dtype == kF32 ? plan<float>(B, L, C, G, want_whole, whole) : plan<bf16>(B, L, C, G, want_whole, whole);
}

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

size_t splat_group_norm_workspace_bytes(int dtype, int B, long long L, int C, int G) {
  if (check_norm("splat_group_norm_workspace_bytes", dtype, B, L, C, G, 0) || B == 0 || L == 0) return 0;
  bool whole;
  const Norm n = plan_of(dtype, B, L, C, G, true, &whole);
  return whole ? 0 : 3 * sizeof(float) * (size_t)B * G * n.splits * n.tpg;
}

int splat_group_norm_fwd(const void* x, long long xsb, long long xsl, const float* weight, const float* bias, int dtype,
                         int B, long long L, int C, int G, float eps, int act, int act_first, void* y, float* mean,
                         float* rstd, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_norm("splat_group_norm_fwd", dtype, B, L, C, G, act)) return rc;
  if (B == 0 || L == 0) return kOk;
  if (!x || !y || !mean != !rstd) return set_error(kInvalid, "splat_group_norm_fwd: null pointer");
  bool whole;
  Norm n = plan_of(dtype, B, L, C, G, true, &whole);
  n.xsb = xsb; n.xsl = xsl; n.eps = eps;
  const size_t need = whole ? 0 : 3 * sizeof(float) * (size_t)B * G * n.splits * n.tpg;
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_group_norm_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  if (n.tiles > 65535) return set_error(kUnsupported, "splat_group_norm_fwd: %d channel tiles", n.tiles);
  const hipStream_t st = (hipStream_t)stream;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      constexpr int A = decltype(a)::value;
      auto go = [&](auto f) {
        constexpr bool First = decltype(f)::value;
        if (whole) {
          k_norm_whole<T, A, First><<<dim3(n.tiles, B), kThreads, 0, st>>>(n, (const T*)x, weight, bias, (T*)y, mean, rstd);
        } else {
          const dim3 grid(n.splits, n.tiles, B);
          k_norm_stats<T, A, First><<<grid, kThreads, 0, st>>>(n, (const T*)x, (float*)ws);
          k_norm_apply<T, A, First><<<grid, kThreads, 0, st>>>(n, (const T*)x, weight, bias, (const float*)ws, (T*)y, mean,
                                                               rstd);
        }
        return check_launch("splat_group_norm_fwd");
      };
      return act_first && A != kActNone ? go(std::true_type{}) : go(std::false_type{});
    });
  });
}

size_t splat_group_norm_bwd_workspace_bytes(int dtype, int B, long long L, int C, int G) {
  if (check_norm("splat_group_norm_bwd_workspace_bytes", dtype, B, L, C, G, 0) || B == 0 || L == 0) return 0;
  bool whole;
  const Norm n = plan_of(dtype, B, L, C, G, false, &whole);
  return 2 * sizeof(float) * ((size_t)B * n.splits * C + (size_t)B * G * n.splits * n.tpg);
}

int splat_group_norm_bwd(const void* x, long long xsb, long long xsl, const void* dy, long long gsb, long long gsl,
                         const float* weight, const float* bias, const float* mean, const float* rstd, int dtype, int B,
                         long long L, int C, int G, int act, int act_first, void* dx, float* dweight, float* dbias,
                         void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_norm("splat_group_norm_bwd", dtype, B, L, C, G, act)) return rc;
  if (B == 0 || L == 0) return kOk;
  if (!x || !dy || !mean || !rstd || !dx) return set_error(kInvalid, "splat_group_norm_bwd: null pointer");
  bool whole;
  Norm n = plan_of(dtype, B, L, C, G, false, &whole);
  n.xsb = xsb; n.xsl = xsl; n.gsb = gsb; n.gsl = gsl;
  const size_t need = splat_group_norm_bwd_workspace_bytes(dtype, B, L, C, G);
  if (!ws || ws_bytes < need)
    return set_error(kWorkspace, "splat_group_norm_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  if (n.tiles > 65535) return set_error(kUnsupported, "splat_group_norm_bwd: %d channel tiles", n.tiles);
  float* cpart = (float*)ws;
  float* gpart = cpart + 2 * (size_t)B * n.splits * C;
  const hipStream_t st = (hipStream_t)stream;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      constexpr int A = decltype(a)::value;
      auto go = [&](auto f) {
        constexpr bool First = decltype(f)::value;
        k_norm_bwd_sums<T, A, First><<<dim3(n.splits, n.tiles, B), kThreads, 0, st>>>(
            n, (const T*)x, (const T*)dy, weight, bias, mean, rstd, cpart, gpart);
        k_norm_bwd_apply<T, A, First><<<dim3(n.splits, n.tiles, B + (dweight || dbias ? 1 : 0)), kThreads, 0, st>>>(
            n, (const T*)x, (const T*)dy, weight, bias, mean, rstd, cpart, gpart, (T*)dx, dweight, dbias);
        return check_launch("splat_group_norm_bwd");
      };
      return act_first && A != kActNone ? go(std::true_type{}) : go(std::false_type{});
    });
  });
}

}  // extern "C"
