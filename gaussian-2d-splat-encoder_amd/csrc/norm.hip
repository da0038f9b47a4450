// Group norm with an activation on channels-last maps x[B, L, C] (L positions), forward and backward.
//
//   act_first: u = act(x), y = w (u - mean) rstd + b;     otherwise: u = x, y = act(w (u - mean) rstd + b)
//
// with mean and rstd = 1 / sqrt(var + eps) over the C / G channels of a group and all positions of an image.
//
// A workgroup covers a channel tile (whole groups, or a part of one group wider than a tile) and a range of positions:
// thread (rt, cc) holds the 16-byte chunk cc of the tile's channels at the positions rt, rt + RT, ... Where one workgroup's
// registers hold a group, everything is one launch that reads x once; otherwise one launch reduces each range to partial
// sums and a second one joins them and writes the result, x coming from the caches the second time where it fits them.
// Both directions are bound by memory, and maps of a few megabytes by the chain of loads, reductions and barriers of a
// workgroup: x's first rows are requested before anything else, and a reduction is one exchange through LDS.
//
// Measured at 8 x 192 x 192 x 128 bf16, gelu first (37.7M values, 75 MB a tensor; a large copy moves 4.9 TB/s here):
// statistics 32 us, result 30 us (5.0 TB/s), backward sums 32 us (4.7), dx 41 us (5.5). The vector unit is busy 60 to 80%
// of that time, half of it with gelu (15 instructions a value, once per pass).
#include "feat_common.h"

namespace splat {
namespace {

constexpr int kThreads = 512;
constexpr int kTile = 2048;   // channels of a tile at most
constexpr int kKeep = 16;     // chunks of x that a thread keeps in registers in the one-launch forward, at most

struct Norm {
  long long L, xsb, xsl, gsb, gsl;   // positions; strides of x and of dy per image and position (channels are dense)
  int B, C, G, Cg;
  int Ct, tiles, tpg;                // channels of a tile; tiles; tiles of one group (1 unless a group passes a tile)
  int nch, RT;                       // chunks of a tile; positions a workgroup takes at a time
  int splits;                        // ranges of positions
  long long per;                     // positions of a range
  FastDiv by_nch, by_RT, by_Cg, by_splits, by_tiles;
  float eps;
};

// A workgroup's work: ranges of a tile follow each other, tiles of an image, images. (One grid dimension: the others hold
// 65,535, fewer than the images of a norm per token.)
struct Unit {
  int img, tile, split;
};
__device__ __forceinline__ Unit unit(const Norm& n) {
  const int id = blockIdx.x, u = __builtin_amdgcn_readfirstlane(id / n.by_splits);
  const int img = __builtin_amdgcn_readfirstlane(u / n.by_tiles);
  return {img, u - img * n.tiles, id - u * n.splits};
}

// A thread's place: its channels [c, c + nv) of the map, its first position rt and its positions of the range [lo, hi).
struct Place {
  int rt, cc, c, nv, c0, ct;   // c0, ct: the tile's first channel and its channels
  int g0, ng;                  // the tile's groups: the first one and how many (1 where the tile is a part of a group)
  long long lo, hi;
  int rows;
};

__device__ __forceinline__ int rows_of(const Norm& n, int range, int rt) {
  return range <= rt ? 0 : (range - rt + n.RT - 1) / n.by_RT;
}

template <typename T>
__device__ __forceinline__ Place place(const Norm& n, int tile, int split) {
  Place p;
  if (n.tpg == 1) {
    p.c0 = tile * n.Ct;
    p.ct = min(n.Ct, n.C - p.c0);
  } else {
    const int g = tile / n.tpg, k = tile % n.tpg;
    p.c0 = g * n.Cg + k * n.Ct;
    p.ct = min(n.Ct, n.Cg - k * n.Ct);
  }
  p.g0 = p.c0 / n.by_Cg;
  p.ng = n.tpg == 1 ? p.ct / n.by_Cg : 1;
  p.rt = (int)threadIdx.x / n.by_nch;
  p.cc = threadIdx.x - p.rt * n.nch;
  p.c = p.c0 + p.cc * kV<T>;
  p.nv = p.rt < n.RT ? max(0, min(kV<T>, p.ct - p.cc * kV<T>)) : 0;
  p.lo = (long long)split * n.per;
  p.hi = min(n.L, p.lo + n.per);
  p.rows = p.nv > 0 ? rows_of(n, (int)(p.hi - p.lo), p.rt) : 0;
  return p;
}

// Group of the thread's channel j within the tile.
__device__ __forceinline__ int group_of(const Norm& n, const Place& p, int j) {
  return n.tpg == 1 ? (p.c - p.c0 + j) / n.by_Cg : 0;
}

// Entries of a group in LDS, one after another: (chunk, rt) where no chunk meets two groups, else (channel, rt).
struct Entries {
  bool whole;
  int per, n;   // entries of a chunk (1 or V); of a group
};
template <typename T>
__device__ __forceinline__ Entries entries(const Norm& n) {
  const bool whole = n.Cg % kV<T> == 0 || n.tpg > 1;
  return {whole, whole ? 1 : kV<T>, n.tpg > 1 ? n.nch * n.RT : (whole ? n.Cg / kV<T> : n.Cg) * n.RT};
}

// f(g, mean, m2) in one lane for each group of the tile, from every thread's mean m and squared deviations q of each of its
// channels over its `rows` positions. m2 = sum q + sum count (m - mean)^2, both sums over positive terms.
template <typename T, typename F>
__device__ __forceinline__ void group_stats(const Norm& n, const Place& p, float (&m)[kV<T>], float (&q)[kV<T>],
                                            float2* red, F&& f) {
  const Entries e = entries<T>(n);
  if (threadIdx.x < (unsigned)(n.RT * n.nch)) {
    if (e.whole) {
      float s = 0.f, v = 0.f;
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) s += j < p.nv ? m[j] : 0.f;
      s = p.nv > 0 ? s / p.nv : 0.f;
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) {
        const float d = m[j] - s;
        v += j < p.nv ? fmaf((float)p.rows * d, d, q[j]) : 0.f;
      }
      red[p.cc * n.RT + p.rt] = make_float2(s, v);
    } else {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) red[(p.cc * kV<T> + j) * n.RT + p.rt] = make_float2(m[j], q[j]);
    }
  }
  __syncthreads();
  const float inv = 1.f / ((float)(p.hi - p.lo) * (float)(n.tpg == 1 ? n.Cg : p.ct));
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < p.ng; g += kThreads / 64) {
    // an entry's values: its row count times its channels
    auto count = [&](int k) {
      const int at = k / n.by_RT, rows = rows_of(n, (int)(p.hi - p.lo), k - at * n.RT);
      return (float)rows * (float)(e.whole ? max(0, min(kV<T>, p.ct - at * kV<T>)) : 1);
    };
    float s = 0.f;
    for (int k = g * e.n + lane; k < (g + 1) * e.n; k += 64) s = fmaf(count(k), red[k].x, s);
    const float mean = wave_add(s) * inv;
    float v = 0.f;
    for (int k = g * e.n + lane; k < (g + 1) * e.n; k += 64) {
      const float d = red[k].x - mean;
      v += fmaf(count(k) * d, d, red[k].y);
    }
    v = wave_add(v);
    if (lane == 0) f(g, mean, v);
  }
}

template <typename T, int A, bool First>
__device__ __forceinline__ float pre(T x) {
  return First ? act_fwd<A>((float)x) : (float)x;
}

template <typename T, int A, bool First>
__device__ __forceinline__ T post(float u, float mean, float a, float b) {
  const float z = fmaf(u - mean, a, b);
  return (T)(First ? z : act_fwd<A>(z));
}

// Parameters of the thread's channels, `none` where there are none.
template <typename T>
__device__ __forceinline__ void params(const float* w, const Place& p, float none, float (&o)[kV<T>]) {
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) o[j] = none;
  if (w && p.nv == kV<T>) {
    __builtin_memcpy(o, w + p.c, sizeof(o));
  } else if (w) {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j)
      if (j < p.nv) o[j] = w[p.c + j];
  }
}

// Statistics and result in one launch, one workgroup per image and tile of whole groups: x stays in registers between the
// statistics (each thread's own mean and deviations, joined per group) and the result. 24 x 24 x 64 float: 8 us, the chain
// of a load, the reduction and a store.
template <typename T, int A, bool First, int Keep>
__global__ __launch_bounds__(kThreads) void k_norm_whole(Norm n, const T* __restrict__ x, const float* __restrict__ w,
                                                         const float* __restrict__ b, T* __restrict__ y,
                                                         float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float2 red[kThreads * kV<T>];
  __shared__ float gm[kTile], gr[kTile];
  const Unit u = unit(n);
  const int img = u.img, tile = u.tile, split = u.split;
  const Place p = place<T>(n, tile, split);
  const T* xp = x + (long long)img * n.xsb + (long long)p.rt * n.xsl + p.c;
  Chunk<T> keep[Keep];
#pragma unroll
  for (int i = 0; i < Keep; ++i)
    if (i < p.rows) keep[i] = load_chunk(xp + (long long)i * n.RT * n.xsl, p.nv);
  float wj[kV<T>], bj[kV<T>], m[kV<T>] = {}, q[kV<T>] = {};
  params<T>(w, p, 1.f, wj);
  params<T>(b, p, 0.f, bj);
#pragma unroll
  for (int i = 0; i < Keep; ++i) {
    if (i < p.rows) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) m[j] += pre<T, A, First>(keep[i].v[j]);
    }
  }
  const float inv = p.rows > 0 ? 1.f / (float)p.rows : 0.f;
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) m[j] *= inv;
#pragma unroll
  for (int i = 0; i < Keep; ++i) {
    if (i < p.rows) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) {
        const float d = pre<T, A, First>(keep[i].v[j]) - m[j];
        q[j] = fmaf(d, d, q[j]);
      }
    }
  }
  const float ivar = 1.f / ((float)n.L * (float)n.Cg);
  group_stats<T>(n, p, m, q, red, [&](int g, float mu, float m2) {
    const float r = 1.f / sqrtf(fmaf(m2, ivar, n.eps));
    gm[g] = mu;
    gr[g] = r;
    if (mean) {
      mean[(long long)img * n.G + p.g0 + g] = mu;
      rstd[(long long)img * n.G + p.g0 + g] = r;
    }
  });
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const int g = j < p.nv ? group_of(n, p, j) : 0;
    m[j] = gm[g];
    wj[j] *= gr[g];
  }
  T* yp = y + ((long long)img * n.L + p.rt) * n.C + p.c;
#pragma unroll
  for (int i = 0; i < Keep; ++i) {
    if (i < p.rows) {
      Chunk<T> o;
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) o.v[j] = post<T, A, First>(pre<T, A, First>(keep[i].v[j]), m[j], wj[j], bj[j]);
      store_chunk(yp + (long long)i * n.RT * n.C, o, p.nv);
    }
  }
}

// Partial statistics of one range: (count, mean, squared deviations from it) per group. Each thread's sums are taken about
// its own first value of the channel, so that a mean far from zero costs no digits.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_stats(Norm n, const T* __restrict__ x, float4* __restrict__ part) {
  __shared__ float2 red[kThreads * kV<T>];
  const Unit u = unit(n);
  const int img = u.img, tile = u.tile, split = u.split;
  const Place p = place<T>(n, tile, split);
  RowStream<T, 4, false> xs;
  xs.begin(x + (long long)img * n.xsb + (p.lo + p.rt) * n.xsl + p.c, n.RT * n.xsl, nullptr, 0, p.rows, p.nv);
  float k0[kV<T>] = {}, s[kV<T>] = {}, q[kV<T>] = {};
  xs.run([&](const Chunk<T>& d, const Chunk<T>&, int i) {
    if (i == 0) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) k0[j] = pre<T, A, First>(d.v[j]);
    }
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) {
      const float u = pre<T, A, First>(d.v[j]) - k0[j];
      s[j] += u;
      q[j] = fmaf(u, u, q[j]);
    }
  });
  const float inv = p.rows > 0 ? 1.f / (float)p.rows : 0.f;
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const float d = fmaf(-s[j] * inv, s[j], q[j]);
    q[j] = d > 0.f || d != d ? d : 0.f;   // rounding may leave less than zero; NaN stays
    k0[j] = fmaf(s[j], inv, k0[j]);
  }
  const int slots = n.splits * n.tpg, slot = split * n.tpg + (n.tpg > 1 ? tile % n.tpg : 0);
  group_stats<T>(n, p, k0, q, red, [&](int g, float mu, float m2) {
    part[((long long)img * n.G + p.g0 + g) * slots + slot] =
        make_float4((float)(p.hi - p.lo) * (float)(n.tpg == 1 ? n.Cg : p.ct), mu, m2, 0.f);
  });
}

// Joins the partial statistics of the tile's groups (one wave a group), then writes the result of one range.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_apply(Norm n, const T* __restrict__ x, const float* __restrict__ w,
                                                         const float* __restrict__ b, const float4* __restrict__ part,
                                                         T* __restrict__ y, float* __restrict__ mean,
                                                         float* __restrict__ rstd) {
  __shared__ float gm[kTile], gr[kTile];
  const Unit u = unit(n);
  const int img = u.img, tile = u.tile, split = u.split;
  const Place p = place<T>(n, tile, split);
  RowStream<T, 4, false> xs;
  xs.begin(x + (long long)img * n.xsb + (p.lo + p.rt) * n.xsl + p.c, n.RT * n.xsl, nullptr, 0, p.rows, p.nv);
  float wj[kV<T>], bj[kV<T>], m[kV<T>];
  params<T>(w, p, 1.f, wj);
  params<T>(b, p, 0.f, bj);
  const int slots = n.splits * n.tpg;
  const int lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)n.L * (float)n.Cg);
  for (int g = threadIdx.x >> 6; g < p.ng; g += kThreads / 64) {
    const float4* o = part + ((long long)img * n.G + p.g0 + g) * slots;
    float cnt = 0.f, mu = 0.f, q = 0.f;   // the lane's ranges so far
#pragma unroll 4
    for (int e = lane; e < slots; e += 64) {
      const float4 v = o[e];
      const float d = v.y - mu, r = v.x * hw_rcp(cnt + v.x);
      mu = fmaf(d, r, mu);
      q += fmaf(d * d, cnt * r, v.z);
      cnt += v.x;
    }
    const float lm = mu;
    mu = wave_add(cnt * lm) * inv;
    const float d = lm - mu;
    const float r = 1.f / sqrtf(fmaf(wave_add(fmaf(cnt * d, d, q)), inv, n.eps));
    if (lane == 0) {
      gm[g] = mu;
      gr[g] = r;
      if (mean && split == 0 && (n.tpg == 1 || tile % n.tpg == 0)) {
        mean[(long long)img * n.G + p.g0 + g] = mu;
        rstd[(long long)img * n.G + p.g0 + g] = r;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const int g = j < p.nv ? group_of(n, p, j) : 0;
    m[j] = gm[g];
    wj[j] *= gr[g];
  }
  T* yp = y + ((long long)img * n.L + p.lo + p.rt) * n.C + p.c;
  const long long ystep = (long long)n.RT * n.C;
  xs.run([&](const Chunk<T>& c, const Chunk<T>&, int i) {
    Chunk<T> o;
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) o.v[j] = post<T, A, First>(pre<T, A, First>(c.v[j]), m[j], wj[j], bj[j]);
    store_chunk(yp + i * ystep, o, p.nv);
  });
}

// g = dL/dz at the norm's output z (before the activation where that comes after), and the normalised input.
template <typename T, int A, bool First>
__device__ __forceinline__ float grad_at(float dy, float uhat, float wj, float bj) {
  return First ? dy : dy * act_grad<A>(fmaf(uhat, wj, bj));
}

// a b - c with the product rounded by itself: a group of one value has c = round(a b), and a zero difference.
__device__ __forceinline__ float rounded_product_less(float a, float b, float c) {
#pragma clang fp contract(off)
  const float p = a * b;
  return p - c;
}

// Means and inverse deviations of the groups of the thread's channels.
template <typename T>
__device__ __forceinline__ void group_params(const Norm& n, const Place& p, int img, const float* mean, const float* rstd,
                                             float (&m)[kV<T>], float (&r)[kV<T>]) {
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const long long g = (long long)img * n.G + p.g0 + (j < p.nv ? group_of(n, p, j) : 0);
    m[j] = mean[g];
    r[j] = rstd[g];
  }
}

// Backward sums of one range: per channel sum g and sum g uhat (`cpart`, for the parameters), per group the same weighted
// by w (`gpart`, for dx).
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_sums(Norm n, const T* __restrict__ x, const T* __restrict__ dy,
                                                            const float* __restrict__ w, const float* __restrict__ b,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, float* __restrict__ cpart,
                                                            float* __restrict__ gpart) {
  __shared__ float2 red[kThreads * kV<T>], chan[kTile];
  const Unit u = unit(n);
  const int img = u.img, tile = u.tile, split = u.split;
  const Place p = place<T>(n, tile, split);
  RowStream<T, 2, true> xs;
  xs.begin(x + (long long)img * n.xsb + (p.lo + p.rt) * n.xsl + p.c, n.RT * n.xsl,
           dy + (long long)img * n.gsb + (p.lo + p.rt) * n.gsl + p.c, n.RT * n.gsl, p.rows, p.nv);
  float m[kV<T>], r[kV<T>], wj[kV<T>], bj[kV<T>], sa[kV<T>] = {}, sb[kV<T>] = {};
  group_params<T>(n, p, img, mean, rstd, m, r);
  params<T>(w, p, 1.f, wj);
  params<T>(b, p, 0.f, bj);
  xs.run([&](const Chunk<T>& c, const Chunk<T>& d, int) {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) {
      const float uh = (pre<T, A, First>(c.v[j]) - m[j]) * r[j];
      const float g = grad_at<T, A, First>((float)d.v[j], uh, wj[j], bj[j]);
      sa[j] += g;
      sb[j] = fmaf(g, uh, sb[j]);
    }
  });
  // per channel over the workgroup's positions (channel-major in LDS, 8 lanes a channel where they suffice), then per group
  if (threadIdx.x < (unsigned)(n.RT * n.nch)) {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) red[(p.cc * kV<T> + j) * n.RT + p.rt] = make_float2(sa[j], sb[j]);
  }
  __syncthreads();
  const int lanes = n.RT >= 8 ? 8 : 1;
  for (int e = threadIdx.x; e < (p.ct * lanes + 63) / 64 * 64; e += kThreads) {
    const int c = e / lanes;
    float2 s = make_float2(0.f, 0.f);
    if (c < p.ct) {
      for (int k = e % lanes; k < n.RT; k += lanes) {
        const float2 v = red[c * n.RT + k];
        s.x += v.x;
        s.y += v.y;
      }
    }
    if (lanes == 8) {
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) {
        s.x += __shfl_xor(s.x, d, 64);
        s.y += __shfl_xor(s.y, d, 64);
      }
    }
    if (c < p.ct && e % lanes == 0) {
      float* o = cpart + ((long long)img * n.splits + split) * 2 * n.C + p.c0 + c;
      o[0] = s.x;
      o[n.C] = s.y;
      const float wc = w ? w[p.c0 + c] : 1.f;
      chan[c] = make_float2(wc * s.x, wc * s.y);
    }
  }
  __syncthreads();
  const int slots = n.splits * n.tpg, slot = split * n.tpg + (n.tpg > 1 ? tile % n.tpg : 0);
  const int wide = n.tpg > 1 ? p.ct : n.Cg, lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < p.ng; g += kThreads / 64) {
    float a = 0.f, q = 0.f;
    for (int c = lane; c < wide; c += 64) {
      a += chan[g * wide + c].x;
      q += chan[g * wide + c].y;
    }
    a = wave_add(a);
    q = wave_add(q);
    if (lane == 0) {
      float* o = gpart + 2 * (((long long)img * n.G + p.g0 + g) * slots + slot);
      o[0] = a;
      o[1] = q;
    }
  }
}

// dx of one range; in the workgroups past the maps' (image B) the parameters' gradients, 32 channels each.
template <typename T, int A, bool First>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_apply(Norm n, const T* __restrict__ x, const T* __restrict__ dy,
                                                             const float* __restrict__ w, const float* __restrict__ b,
                                                             const float* __restrict__ mean,
                                                             const float* __restrict__ rstd,
                                                             const float* __restrict__ cpart,
                                                             const float* __restrict__ gpart, T* __restrict__ dx,
                                                             float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float ga[kTile], gb[kTile];
  const int maps = n.B * n.tiles * n.splits;   // workgroups of the maps
  if ((int)blockIdx.x >= maps) {
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, nrow = kThreads / 32;
    for (int c0 = (blockIdx.x - maps) * 32; c0 < n.C; c0 += (gridDim.x - maps) * 32) {
      const int c = c0 + lane;
      float a = 0.f, q = 0.f;
      if (c < n.C) {
        const long long R = (long long)n.B * n.splits;
#pragma unroll 4
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
  const Unit u = unit(n);
  const int img = u.img, tile = u.tile, split = u.split;
  const Place p = place<T>(n, tile, split);
  RowStream<T, 2, true> xs;
  xs.begin(x + (long long)img * n.xsb + (p.lo + p.rt) * n.xsl + p.c, n.RT * n.xsl,
           dy + (long long)img * n.gsb + (p.lo + p.rt) * n.gsl + p.c, n.RT * n.gsl, p.rows, p.nv);
  float m[kV<T>], r[kV<T>], wj[kV<T>], bj[kV<T>], s1[kV<T>], s2[kV<T>];
  group_params<T>(n, p, img, mean, rstd, m, r);
  params<T>(w, p, 1.f, wj);
  params<T>(b, p, 0.f, bj);
  const int slots = n.splits * n.tpg;
  const int lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)n.L * (float)n.Cg);
  for (int g = threadIdx.x >> 6; g < p.ng; g += kThreads / 64) {
    const float* o = gpart + 2 * ((long long)img * n.G + p.g0 + g) * slots;
    float s = 0.f, q = 0.f;
#pragma unroll 4
    for (int e = lane; e < slots; e += 64) {
      s += o[2 * e];
      q += o[2 * e + 1];
    }
    s = wave_add(s);
    q = wave_add(q);
    if (lane == 0) {
      ga[g] = s * inv;
      gb[g] = q * inv;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) {
    const int g = j < p.nv ? group_of(n, p, j) : 0;
    s1[j] = ga[g];
    s2[j] = gb[g];
  }
  T* op = dx + ((long long)img * n.L + p.lo + p.rt) * n.C + p.c;
  const long long ostep = (long long)n.RT * n.C;
  xs.run([&](const Chunk<T>& c, const Chunk<T>& d, int i) {
    Chunk<T> o;
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) {
      const float uh = (pre<T, A, First>(c.v[j]) - m[j]) * r[j];
      const float du = r[j] * (rounded_product_less(grad_at<T, A, First>((float)d.v[j], uh, wj[j], bj[j]), wj[j], s1[j]) -
                               uh * s2[j]);
      o.v[j] = (T)(First ? du * act_grad<A>((float)c.v[j]) : du);
    }
    store_chunk(op + i * ostep, o, p.nv);
  });
}

// The launch geometry of a call. whole: one workgroup holds its groups' values in registers.
template <typename T>
Norm plan(int B, long long L, int C, int G, bool want_whole, bool* whole) {
  Norm n{};
  constexpr int V = kV<T>;
  n.B = B; n.L = L; n.C = C; n.G = G; n.Cg = C / G;
  n.by_Cg = fast_div(n.Cg);
  const int most = kThreads * V < kTile ? kThreads * V : kTile;   // channels of a tile
  auto tile = [&](int gpt) {   // whole groups
    n.Ct = gpt * n.Cg; n.tpg = 1; n.tiles = (G + gpt - 1) / gpt;
    n.nch = (n.Ct + V - 1) / V;
    n.RT = kThreads / n.nch;
  };
  *whole = false;
  if (n.Cg <= most) {
    // one launch: as few groups a workgroup as make 64-byte runs of a position's channels, for the most workgroups
    const int run = 64 / (int)sizeof(T), gpt = (run + n.Cg - 1) / n.Cg;
    tile(gpt < G ? gpt : G);
    if (want_whole && L <= (long long)n.RT * kKeep) {
      n.splits = 1; n.per = L;
      *whole = true;
    } else {
      tile(most / n.Cg < G ? most / n.Cg : G);
    }
  } else {
    n.Ct = most; n.tpg = (n.Cg + most - 1) / most; n.tiles = G * n.tpg;
    n.nch = n.Ct / V;
    n.RT = kThreads / n.nch;
  }
  n.by_nch = fast_div(n.nch);
  n.by_RT = fast_div(n.RT);
  n.by_tiles = fast_div(n.tiles);
  n.by_splits = fast_div(1);
  if (*whole) return n;
  // 512 workgroups, the two per CU that registers allow at a time, of at least a batch of rows of their threads
  const long long want = 512 / ((long long)B * n.tiles) > 0 ? 512 / ((long long)B * n.tiles) : 1;
  const long long batch = 4LL * n.RT;
  n.per = (L + want - 1) / want;
  if (n.per < batch) n.per = batch;
  if (n.per > (1LL << 30)) n.per = 1LL << 30;   // a range's rows are counted in 32 bits
  n.splits = (int)((L + n.per - 1) / n.per);
  n.by_splits = fast_div(n.splits);
  return n;
}

// Workgroups of `images` images, 0 where a launch (2^32 threads) does not hold them.
unsigned grid_of(const Norm& n, long long images) {
  const long long per = (long long)n.tiles * n.splits;
  return per < (1 << 23) && images * per < (1 << 23) ? (unsigned)(images * per) : 0;
}

int check_norm(const char* what, int dtype, int B, long long L, int C, int G, int act) {
  if (dtype != kF32 && dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", what, dtype);
  if (B < 0 || L < 0 || C < 1 || G < 1 || C % G) return set_error(kInvalid, "%s: B %d, L %lld, C %d, G %d", what, B, L, C, G);
  if (act < 0 || act >= kActCount) return set_error(kInvalid, "%s: unknown activation %d", what, act);
  if (L > 0x7fffffffLL * 4) return set_error(kUnsupported, "%s: %d images of %lld positions", what, B, L);
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
  return whole ? 0 : sizeof(float4) * (size_t)B * G * n.splits * n.tpg;
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
  const size_t need = whole ? 0 : sizeof(float4) * (size_t)B * G * n.splits * n.tpg;
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_group_norm_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  const unsigned grid = grid_of(n, B);
  if (!grid) return set_error(kUnsupported, "splat_group_norm_fwd: %d images of %d channel tiles", B, n.tiles);
  const hipStream_t st = (hipStream_t)stream;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      constexpr int A = decltype(a)::value;
      auto go = [&](auto f) {
        constexpr bool First = decltype(f)::value;
        if (whole) {
          auto whole_of = [&](auto keep) {
            k_norm_whole<T, A, First, decltype(keep)::value><<<grid, kThreads, 0, st>>>(
                n, (const T*)x, weight, bias, (T*)y, mean, rstd);
          };
          if (L <= 4LL * n.RT) whole_of(std::integral_constant<int, 4>{});
          else if (L <= 8LL * n.RT) whole_of(std::integral_constant<int, 8>{});
          else whole_of(std::integral_constant<int, kKeep>{});
        } else {
          k_norm_stats<T, A, First><<<grid, kThreads, 0, st>>>(n, (const T*)x, (float4*)ws);
          k_norm_apply<T, A, First><<<grid, kThreads, 0, st>>>(n, (const T*)x, weight, bias, (const float4*)ws, (T*)y, mean,
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
  const unsigned maps = grid_of(n, B), all = grid_of(n, B + (dweight || dbias ? 1LL : 0));   // parameters come last
  if (!all) return set_error(kUnsupported, "splat_group_norm_bwd: %d images of %d channel tiles", B, n.tiles);
  float* cpart = (float*)ws;
  float* gpart = cpart + 2 * (size_t)B * n.splits * C;
  const hipStream_t st = (hipStream_t)stream;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      constexpr int A = decltype(a)::value;
      auto go = [&](auto f) {
        constexpr bool First = decltype(f)::value;
        k_norm_bwd_sums<T, A, First><<<maps, kThreads, 0, st>>>(
            n, (const T*)x, (const T*)dy, weight, bias, mean, rstd, cpart, gpart);
        k_norm_bwd_apply<T, A, First><<<all, kThreads, 0, st>>>(
            n, (const T*)x, (const T*)dy, weight, bias, mean, rstd, cpart, gpart, (T*)dx, dweight, dbias);
        return check_launch("splat_group_norm_bwd");
      };
      return act_first && A != kActNone ? go(std::true_type{}) : go(std::false_type{});
    });
  });
}

}  // extern "C"
