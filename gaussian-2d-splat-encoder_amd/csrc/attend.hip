// Cross attention: o = softmax(scale q k^T) v over the valid keys, for queries q[B, Lq, H, D] and another sequence's
// keys and values k, v[B, Lk, Hk, D] (H a multiple of Hk: H / Hk query heads share a key head), and its gradients.
//
// The H / Hk heads that share keys are rows of one problem: row r = query * rep + head within the group, R = Lq * rep
// rows per (image, key head). Scores are held transposed, a lane per query (forward, dq) or per key (dk, dv), so that a
// softmax row is one lane pair and the probabilities are the next product's operand as they leave the first. One pass
// over the keys with a running maximum and sum; sums, statistics and accumulators are 32-bit floats, probabilities and
// score gradients are rounded to the inputs' type for the matrix instructions only.
//
// Keys that a length or a mask leaves out are replaced by zeros as they are loaded, so that nothing they hold (NaN
// included) reaches a product; a row without valid keys gives zeros, and zero gradients.
#include "feat_common.h"
#include "splat_attention.h"

namespace splat {
namespace {

constexpr int kThreads = 256, kWaves = 4;

struct Attn {
  splat_attention a;
  int rep, R;            // query heads per key head; rows per (image, key head)
  int tiles, splits;     // workgroups per (image, key head) along the rows (or keys), and along the other axis
  int per;               // tiles of the other axis that a split takes
};

template <typename T, int DP>
struct Shape {
  static constexpr int V = kV<T>;
  static constexpr int nc = DP / (2 * V);   // chunks that a lane holds of a row
  static constexpr int nd = DP / 32;        // 32-wide blocks of a row
  static constexpr int ld = DP + V;         // LDS row: 16 bytes of padding
};

template <typename T, int DP> using RowFrag = Chunk<T>[Shape<T, DP>::nc];
template <typename T, int DP> using RowAcc = f32x16[Shape<T, DP>::nd];

// Rows of an operand in registers: lane l holds the chunks of row l % 32 (zeros where !in).
template <typename T, int DP>
__device__ __forceinline__ void load_rows(RowFrag<T, DP>& f, const T* row, bool in, int D, int h) {
#pragma unroll
  for (int c = 0; c < Shape<T, DP>::nc; ++c) {
    const int d = (2 * c + h) * kV<T>;
    f[c] = load_chunk(row + d, in ? D - d : 0);
  }
}

__device__ __forceinline__ int key_count(const splat_attention& a, int b) {
  const int n = a.kv_lengths ? a.kv_lengths[b] : (int)a.Lk;
  return n < 0 ? 0 : n > (int)a.Lk ? (int)a.Lk : n;
}

// Bit i: key k0 + i is valid (i < 64), the same in every lane.
__device__ __forceinline__ unsigned long long valid_keys(const splat_attention& a, int b, int k0, int len) {
  const int k = k0 + (threadIdx.x & 63);
  bool in = k < len;
  if (a.key_mask && in) in = a.key_mask[(long long)b * a.mb + (long long)k * a.ml] != 0;
  return __ballot(in);
}

// Adds 32 x 32 scores: acc = rows of `t` (LDS) times the lanes' register rows.
template <typename T, int DP>
__device__ __forceinline__ void scores(f32x16& acc, const T* t, const RowFrag<T, DP>& f, int lane) {
#pragma unroll
  for (int c = 0; c < Shape<T, DP>::nc; ++c)
    mma(acc, row_frag(t + 2 * c * kV<T>, Shape<T, DP>::ld, lane), f[c]);
}

// acc[d][lane] += sum over the 32 LDS rows from t of row[d] * p[row][lane], p as the results of scores().
template <typename T, int DP>
__device__ __forceinline__ void gather(RowAcc<T, DP>& acc, const T* t, const f32x16& p, int lane) {
  constexpr int V = kV<T>;
#pragma unroll
  for (int c = 0; c < 16 / V; ++c) {
    Chunk<T> b;
#pragma unroll
    for (int j = 0; j < V; ++j) b.v[j] = (T)p[c * V + j];
#pragma unroll
    for (int d = 0; d < Shape<T, DP>::nd; ++d)
      mma(acc[d], col_frag<true>(t + 2 * V * c * Shape<T, DP>::ld + 32 * d, Shape<T, DP>::ld, lane), b);
  }
}

// N rows of an LDS tile: global -> registers -> LDS, zeros for rows whose bit is off and columns past D.
template <typename T, int DP, int N>
struct Rows {
  static constexpr int V = kV<T>, chunks = N * (DP / V), per = (chunks + kThreads - 1) / kThreads;
  template <typename F>
  __device__ static void load(Chunk<T> (&c)[per], int D, F&& row) {   // row(i): pointer of row i, or null
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int e = threadIdx.x + i * kThreads, col = e % (DP / V) * V;
      const T* p = chunks % kThreads == 0 || e < chunks ? row(e / (DP / V)) : nullptr;
      c[i] = load_chunk(p + col, p ? D - col : 0);
    }
  }
  __device__ static void put(const Chunk<T> (&c)[per], T* t) {
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int e = threadIdx.x + i * kThreads;
      if (chunks % kThreads == 0 || e < chunks)
        *(f32x4*)(t + e / (DP / V) * Shape<T, DP>::ld + e % (DP / V) * V) = *(const f32x4*)c[i].v;
    }
  }
};

// Writes the lane's row of DP values, scaled, from the accumulators.
template <typename T, typename O, int DP>
__device__ __forceinline__ void store_row(O* row, const RowAcc<T, DP>& acc, float s, int D, bool in, int h) {
#pragma unroll
  for (int d = 0; d < Shape<T, DP>::nd; ++d) {
    float run[16 / kV<O>][kV<O>];
    acc_runs<O>(acc[d], run);
#pragma unroll
    for (int t = 0; t < 16 / kV<O>; ++t) {
      const int c = 32 * d + run_row<O>(t, h);
      Chunk<O> o;
#pragma unroll
      for (int e = 0; e < kV<O>; ++e) o.v[e] = (O)(run[t][e] * s);
      if (in) store_chunk(row + c, o, D - c);
    }
  }
}

struct Work {
  int tile, split, b, hk, bh;
};

// Workgroup -> (image, key head), tile and split: a head's tiles follow each other on one XCD, whose L2 then holds the
// other side of them.
__device__ __forceinline__ Work work_of(const Attn& n) {
  const int id = xcd_swizzle(blockIdx.x, gridDim.x);
  Work w;
  w.tile = id % n.tiles;
  w.split = id / n.tiles % n.splits;
  w.bh = id / (n.tiles * n.splits);
  w.b = w.bh / n.a.Hk;
  w.hk = w.bh % n.a.Hk;
  return w;
}

// Address of row r's head vector in a tensor of strides (sb, sl, sh).
template <typename T>
__device__ __forceinline__ const T* head_row(const void* p, const Attn& n, const Work& w, int r, long long sb, long long sl,
                                             long long sh) {
  const int q = r / n.rep, j = r - q * n.rep;
  return (const T*)p + w.b * sb + q * sl + (long long)(w.hk * n.rep + j) * sh;
}

// ------------------------------------------------------------------------------------------------ forward
// QW = 4: the workgroup's waves take 32 rows each and share every key tile. QW = 1: they share 32 rows and take a quarter
// of every key tile each, ending in four partial results. Partial results (maximum, sum, unscaled output) of splits and
// waves are joined by k_attn_join; without any the output is final.
template <typename T, int DP, int QW>
__global__ __launch_bounds__(kThreads) void k_attn_fwd(Attn n, const T* __restrict__ q, const T* __restrict__ k,
                                                       const T* __restrict__ v, T* __restrict__ o, float* __restrict__ lse,
                                                       float* __restrict__ part, float* __restrict__ stat) {
  using S = Shape<T, DP>;
  constexpr int KB = QW == 4 ? 64 / (int)sizeof(T) / 16 : 1;   // 32-key blocks a wave takes of a tile: 2 bf16, 1 float
  constexpr int KT = QW == 4 ? 32 * KB : 128;
  __shared__ __align__(16) T tk[KT * S::ld];
  __shared__ __align__(16) T tv[KT * S::ld];
  const splat_attention& a = n.a;
  const Work w = work_of(n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int r = w.tile * 32 * QW + (QW == 4 ? wave * 32 : 0) + (lane & 31);
  const bool in = r < n.R;
  const int kw = QW == 4 ? 0 : wave * 32;   // the wave's first key of a tile
  Chunk<T> fq[S::nc];
  load_rows<T, DP>(fq, head_row<T>(q, n, w, in ? r : 0, a.qb, a.ql, a.qh), in, a.D, h);
  const int len = key_count(a, w.b);
  const int t0 = w.split * n.per, t1 = min((len + KT - 1) / KT, t0 + n.per);
  const float c = a.scale * kLog2e;
  f32x16 acc[S::nd] = {};
  float m = -INFINITY, l = 0.f;
  using R = Rows<T, DP, KT>;
  Chunk<T> ck[R::per], cv[R::per];
  unsigned long long ok[2] = {};   // valid keys of the tile (128 at most)
  const T* kb = k + w.b * a.kb + w.hk * a.kh;
  const T* vb = v + w.b * a.vb + w.hk * a.vh;
  auto fetch = [&](int t) {
    const int k0 = t * KT;
    ok[0] = valid_keys(a, w.b, k0, len);
    if (KT > 64) ok[1] = valid_keys(a, w.b, k0 + 64, len);
    auto bit = [&](int i) { return (ok[KT > 64 ? i >> 6 : 0] >> (i & 63)) & 1; };
    R::load(ck, a.D, [&](int i) { return bit(i) ? kb + (long long)(k0 + i) * a.kl : nullptr; });
    R::load(cv, a.D, [&](int i) { return bit(i) ? vb + (long long)(k0 + i) * a.vl : nullptr; });
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const unsigned long long good = KT > 64 && kw >= 64 ? ok[1] : ok[0];
    __syncthreads();
    R::put(ck, tk);
    R::put(cv, tv);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    f32x16 s[KB] = {};
    float mx = -INFINITY;
#pragma unroll
    for (int kb2 = 0; kb2 < KB; ++kb2) {
      scores<T, DP>(s[kb2], tk + (kw + 32 * kb2) * S::ld, fq, lane);
      const unsigned bits = (unsigned)(good >> ((kw & 63) + 32 * kb2)) >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb2][i] = (bits >> acc_row(i, 0)) & 1 ? s[kb2][i] * c : -INFINITY;
        mx = fmaxf(mx, s[kb2][i]);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn;
    const float al = hw_exp2(m - mu);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int kb2 = 0; kb2 < KB; ++kb2) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb2][i] = hw_exp2(s[kb2][i] - mu);
        sum += s[kb2][i];
      }
    }
    l = fmaf(l, al, sum);
#pragma unroll
    for (int d = 0; d < S::nd; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] *= al;
#pragma unroll
    for (int kb2 = 0; kb2 < KB; ++kb2) gather<T, DP>(acc, tv + (kw + 32 * kb2) * S::ld, s[kb2], lane);
  }
  l += __shfl_xor(l, 32, 64);
  if (part) {
    const int slot = QW == 4 ? w.split : w.split * kWaves + wave;
    const long long at = ((long long)slot * n.a.B * n.a.Hk + w.bh) * n.R + r;
    if (in && h == 0) {
      stat[2 * at] = m;
      stat[2 * at + 1] = l;
    }
    store_row<T, float, DP>(part + at * a.D, acc, 1.f, a.D, in, h);
  } else {
    const float inv = l > 0.f ? 1.f / l : l;   // 0 for a row without keys, NaN stays
    if (lse && in && h == 0) lse[(long long)w.bh * n.R + r] = l == 0.f ? INFINITY : m + hw_log2(l);
    const int qi = r / n.rep, j = r - qi * n.rep;
    store_row<T, T, DP>(o + ((w.b * a.Lq + qi) * a.H + w.hk * n.rep + j) * a.D, acc, inv, a.D, in, h);
  }
}

// Joins the partial results of a row: one wave a row, lanes over the head's values.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_attn_join(Attn n, const float* __restrict__ part, const float* __restrict__ stat,
                                                        int slots, T* __restrict__ o, float* __restrict__ lse) {
  const splat_attention& a = n.a;
  const long long rows = (long long)a.B * a.Hk * n.R;
  const long long row = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int s = lane; s < slots; s += 64) m = fmaxf(m, stat[2 * (s * rows + row)]);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = lane; s < slots; s += 64) l = fmaf(stat[2 * (s * rows + row) + 1], hw_exp2(stat[2 * (s * rows + row)] - mu), l);
  l = wave_sum(l);
  const float inv = l > 0.f ? 1.f / l : l;
  const int bh = (int)(row / n.R), r = (int)(row - (long long)bh * n.R);
  const int qi = r / n.rep, j = r - qi * n.rep, b = bh / a.Hk, hk = bh % a.Hk;
  T* op = o + (((long long)b * a.Lq + qi) * a.H + hk * n.rep + j) * a.D;
  for (int d = lane; d < a.D; d += 64) {
    float s = 0.f;
    for (int i = 0; i < slots; ++i) {
      const long long at = i * rows + row;
      s = fmaf(part[at * a.D + d], hw_exp2(stat[2 * at] - mu), s);
    }
    op[d] = (T)(s * inv);
  }
  if (lse && lane == 0) lse[row] = l == 0.f ? INFINITY : m + hw_log2(l);
}

// ----------------------------------------------------------------------------------------------- backward
// delta[row] = sum over d of do * o.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_attn_delta(Attn n, const T* __restrict__ o, const T* __restrict__ g,
                                                         float* __restrict__ delta) {
  const splat_attention& a = n.a;
  // eight lanes a row
  const long long row = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;
  if (row >= (long long)a.B * a.Hk * n.R) return;
  const int bh = (int)(row / n.R), r = (int)(row - (long long)bh * n.R);
  const int qi = r / n.rep, j = r - qi * n.rep, b = bh / a.Hk, hq = bh % a.Hk * n.rep + j;
  const T* op = o + (((long long)b * a.Lq + qi) * a.H + hq) * a.D;
  const T* gp = g + b * a.gb + qi * a.gl + hq * a.gh;
  float s = 0.f;
  for (int d = (threadIdx.x & 7) * kV<T>; d < a.D; d += 8 * kV<T>) {
    const Chunk<T> x = load_chunk(op + d, a.D - d), y = load_chunk(gp + d, a.D - d);
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) s = fmaf((float)x.v[e], (float)y.v[e], s);
  }
  s += __shfl_xor(s, 1, 64);
  s += __shfl_xor(s, 2, 64);
  s += __shfl_xor(s, 4, 64);
  if ((threadIdx.x & 7) == 0) delta[row] = s;
}

// dk and dv: a wave holds 32 keys and values, the workgroup's four share tiles of query rows. With s = q k^T a lane is a
// key: p and ds are the operands of dv = p^T do and dk = ds^T q as they are.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void k_attn_bwd_kv(Attn n, const T* __restrict__ q, const T* __restrict__ k,
                                                          const T* __restrict__ v, const T* __restrict__ g,
                                                          const float* __restrict__ lse, const float* __restrict__ delta,
                                                          T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
  using S = Shape<T, DP>;
  constexpr int QT = 32;
  __shared__ __align__(16) T tq[QT * S::ld];
  __shared__ __align__(16) T tg[QT * S::ld];
  __shared__ __align__(16) float tl[QT], td[QT];
  const splat_attention& a = n.a;
  const Work w = work_of(n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int len = key_count(a, w.b);
  const int k0 = w.tile * 128 + (wave & 2) * 32;
  const unsigned long long ok = valid_keys(a, w.b, k0, len);
  const int ki = w.tile * 128 + wave * 32 + (lane & 31);
  const bool good = (ok >> ((wave & 1) * 32 + (lane & 31))) & 1;
  Chunk<T> fk[S::nc], fv[S::nc];
  load_rows<T, DP>(fk, k + w.b * a.kb + w.hk * a.kh + (good ? ki : 0) * a.kl, good, a.D, h);
  load_rows<T, DP>(fv, v + w.b * a.vb + w.hk * a.vh + (good ? ki : 0) * a.vl, good, a.D, h);
  const bool any = w.tile * 128 < len;
  const int t0 = w.split * n.per, t1 = any ? min((n.R + QT - 1) / QT, t0 + n.per) : t0;
  const float c = a.scale * kLog2e;
  f32x16 ak[S::nd] = {}, av[S::nd] = {};
  using R = Rows<T, DP, QT>;
  Chunk<T> cq[R::per], cg[R::per];
  float sl = 0.f, sd = 0.f;
  auto fetch = [&](int t) {
    const int r0 = t * QT;
    R::load(cq, a.D, [&](int i) { return r0 + i < n.R ? head_row<T>(q, n, w, r0 + i, a.qb, a.ql, a.qh) : nullptr; });
    R::load(cg, a.D, [&](int i) { return r0 + i < n.R ? head_row<T>(g, n, w, r0 + i, a.gb, a.gl, a.gh) : nullptr; });
    if (threadIdx.x < QT) {
      const int r = r0 + threadIdx.x;
      sl = r < n.R ? lse[(long long)w.bh * n.R + r] : INFINITY;
      sd = r < n.R ? delta[(long long)w.bh * n.R + r] : 0.f;
    }
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    R::put(cq, tq);
    R::put(cg, tg);
    if (threadIdx.x < QT) {
      tl[threadIdx.x] = sl;
      td[threadIdx.x] = sd;
    }
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    f32x16 s = {}, dp = {};
    scores<T, DP>(s, tq, fk, lane);
    scores<T, DP>(dp, tg, fv, lane);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const f32x4 L = *(const f32x4*)(tl + acc_row(i, h)), D = *(const f32x4*)(td + acc_row(i, h));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = good ? hw_exp2(fmaf(s[i + e], c, -L[e])) : 0.f;
        s[i + e] = p;
        dp[i + e] = p * (dp[i + e] - D[e]);
      }
    }
    gather<T, DP>(av, tg, s, lane);
    gather<T, DP>(ak, tq, dp, lane);
  }
  const bool in = ki < a.Lk;
  if (part) {
    const long long rows = (long long)a.B * a.Lk * a.Hk;
    const long long at = ((long long)w.b * a.Lk + ki) * a.Hk + w.hk;
    store_row<T, float, DP>(part + ((long long)w.split * 2 * rows + at) * a.D, ak, a.scale, a.D, in, h);
    store_row<T, float, DP>(part + ((long long)(w.split * 2 + 1) * rows + at) * a.D, av, 1.f, a.D, in, h);
  } else {
    const long long at = ((long long)w.b * a.Lk + ki) * a.Hk + w.hk;
    store_row<T, T, DP>(dk + at * a.D, ak, a.scale, a.D, in, h);
    store_row<T, T, DP>(dv + at * a.D, av, 1.f, a.D, in, h);
  }
}

// dq: as the forward, a lane per query row; ds^T is the operand of dq^T = k^T ds^T as it is.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void k_attn_bwd_q(Attn n, const T* __restrict__ q, const T* __restrict__ k,
                                                         const T* __restrict__ v, const T* __restrict__ g,
                                                         const float* __restrict__ lse, const float* __restrict__ delta,
                                                         T* __restrict__ dq, float* __restrict__ part) {
  using S = Shape<T, DP>;
  constexpr int KT = 32;
  __shared__ __align__(16) T tk[KT * S::ld];
  __shared__ __align__(16) T tv[KT * S::ld];
  const splat_attention& a = n.a;
  const Work w = work_of(n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int r = w.tile * 128 + wave * 32 + (lane & 31);
  const bool in = r < n.R;
  Chunk<T> fq[S::nc], fg[S::nc];
  load_rows<T, DP>(fq, head_row<T>(q, n, w, in ? r : 0, a.qb, a.ql, a.qh), in, a.D, h);
  load_rows<T, DP>(fg, head_row<T>(g, n, w, in ? r : 0, a.gb, a.gl, a.gh), in, a.D, h);
  const float L = in ? lse[(long long)w.bh * n.R + r] : INFINITY;
  const float dl = in ? delta[(long long)w.bh * n.R + r] : 0.f;
  const int len = key_count(a, w.b);
  const int t0 = w.split * n.per, t1 = min((len + KT - 1) / KT, t0 + n.per);
  const float c = a.scale * kLog2e;
  f32x16 acc[S::nd] = {};
  using R = Rows<T, DP, KT>;
  Chunk<T> ck[R::per], cv[R::per];
  unsigned ok = 0;
  const T* kb = k + w.b * a.kb + w.hk * a.kh;
  const T* vb = v + w.b * a.vb + w.hk * a.vh;
  auto fetch = [&](int t) {
    const int k0 = t * KT;
    ok = (unsigned)valid_keys(a, w.b, k0, len);
    R::load(ck, a.D, [&](int i) { return (ok >> i) & 1 ? kb + (long long)(k0 + i) * a.kl : nullptr; });
    R::load(cv, a.D, [&](int i) { return (ok >> i) & 1 ? vb + (long long)(k0 + i) * a.vl : nullptr; });
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const unsigned bits = ok >> (4 * h);
    __syncthreads();
    R::put(ck, tk);
    R::put(cv, tv);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    f32x16 s = {}, dp = {};
    scores<T, DP>(s, tk, fq, lane);
    scores<T, DP>(dp, tv, fg, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = (bits >> acc_row(i, 0)) & 1 ? hw_exp2(fmaf(s[i], c, -L)) : 0.f;
      dp[i] = p * (dp[i] - dl);
    }
    gather<T, DP>(acc, tk, dp, lane);
  }
  if (part) {
    const long long rows = (long long)a.B * a.Hk * n.R;
    store_row<T, float, DP>(part + (w.split * rows + (long long)w.bh * n.R + r) * a.D, acc, a.scale, a.D, in, h);
  } else {
    const int qi = r / n.rep, j = r - qi * n.rep;
    store_row<T, T, DP>(dq + ((w.b * a.Lq + qi) * a.H + w.hk * n.rep + j) * a.D, acc, a.scale, a.D, in, h);
  }
}

// Adds the splits' partial gradients in their order. Rows of `part` are the output's own order, or (heads) the rows of
// (image, key head) problems.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_attn_add(Attn n, const float* __restrict__ part, int splits, long long stride,
                                                       long long count, bool heads, T* __restrict__ out) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= count) return;
  float s = 0.f;
  for (int k = 0; k < splits; ++k) s += part[k * stride + i];
  long long at = i;
  if (heads) {
    const splat_attention& a = n.a;
    const long long row = i / a.D;
    const int d = (int)(i - row * a.D), bh = (int)(row / n.R), r = (int)(row - (long long)bh * n.R);
    const int qi = r / n.rep, j = r - qi * n.rep, b = bh / a.Hk, hk = bh % a.Hk;
    at = (((long long)b * a.Lq + qi) * a.H + hk * n.rep + j) * a.D + d;
  }
  out[at] = (T)s;
}

// ---------------------------------------------------------------------------------------------- launches
int check_attn(const char* what, const splat_attention* a) {
  if (!a) return set_error(kInvalid, "%s: null description", what);
  if (a->dtype != kF32 && a->dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", what, a->dtype);
  if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk || a->D < 1)
    return set_error(kInvalid, "%s: B %d, Lq %lld, Lk %lld, H %d, Hk %d, D %d", what, a->B, a->Lq, a->Lk, a->H, a->Hk, a->D);
  if (a->D > 128) return set_error(kUnsupported, "%s: heads of %d values (128 at most)", what, a->D);
  // rows and keys are 32-bit within a head, workgroups 32-bit in all
  const long long heads = (long long)a->B * a->Hk, rows = a->Lq * (a->H / a->Hk);
  if (rows > 0x7fffff00LL || a->Lk > 0x7fffff00LL || heads * ((rows + 31) / 32 + 1) > 0xffffffLL ||
      heads * ((a->Lk + 31) / 32 + 1) > 0xffffffLL)
    return set_error(kUnsupported, "%s: B %d, Lq %lld, Lk %lld", what, a->B, a->Lq, a->Lk);
  return kOk;
}

template <typename F>
int with_shape(const splat_attention& a, F&& f) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if (a.D <= 32) return f(T{}, std::integral_constant<int, 32>{});
    if (a.D <= 64) return f(T{}, std::integral_constant<int, 64>{});
    if (a.D <= 96) return f(T{}, std::integral_constant<int, 96>{});
    return f(T{}, std::integral_constant<int, 128>{});
  };
  return a.dtype == kF32 ? go(float{}) : go(bf16{});
}

// Splits of an axis of `tiles` tiles where `groups` workgroups would run: as many as make about 512, of at least `least`
// tiles each.
void split(Attn& n, long long groups, int tiles, int least) {
  long long s = groups >= 256 || groups == 0 ? 1 : 512 / groups;
  if (s > (tiles + least - 1) / least) s = (tiles + least - 1) / least;
  if (s < 1) s = 1;
  n.per = (int)((tiles + s - 1) / s);
  if (n.per < 1) n.per = 1;
  n.splits = tiles > 0 ? (tiles + n.per - 1) / n.per : 1;
}

Attn base(const splat_attention& a) {
  Attn n{};
  n.a = a;
  n.rep = a.H / a.Hk;
  n.R = (int)(a.Lq * n.rep);
  return n;
}

Attn plan_fwd(const splat_attention& a, bool* shared) {
  Attn n = base(a);
  *shared = n.R <= 32;   // few rows: the waves split the keys
  n.tiles = *shared ? 1 : div_up(n.R, 128);
  const int kt = *shared ? 128 : a.dtype == kF32 ? 32 : 64;
  split(n, (long long)n.tiles * a.B * a.Hk, div_up(a.Lk, kt), 4);
  return n;
}

Attn plan_kv(const splat_attention& a) {
  Attn n = base(a);
  n.tiles = div_up(a.Lk, 128);
  split(n, (long long)n.tiles * a.B * a.Hk, div_up(n.R, 32), 8);
  return n;
}

Attn plan_q(const splat_attention& a) {
  Attn n = base(a);
  n.tiles = div_up(n.R, 128);
  split(n, (long long)n.tiles * a.B * a.Hk, div_up(a.Lk, 32), 8);
  return n;
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

size_t splat_attention_workspace_bytes(const splat_attention* a) {
  if (check_attn("splat_attention_workspace_bytes", a) || a->B == 0 || a->Lq == 0) return 0;
  bool shared;
  const Attn n = plan_fwd(*a, &shared);
  if (!shared && n.splits == 1) return 0;
  return sizeof(float) * (size_t)n.splits * (shared ? kWaves : 1) * a->B * a->Hk * n.R * (a->D + 2);
}

int splat_attention_fwd(const splat_attention* a, const void* q, const void* k, const void* v, void* o, float* lse,
                        void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_attn("splat_attention_fwd", a)) return rc;
  if (a->B == 0 || a->Lq == 0) return kOk;
  if (!q || !o || (a->Lk > 0 && (!k || !v))) return set_error(kInvalid, "splat_attention_fwd: null pointer");
  bool shared;
  const Attn n = plan_fwd(*a, &shared);
  const size_t need = splat_attention_workspace_bytes(a);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_attention_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  const int slots = n.splits * (shared ? kWaves : 1);
  const long long rows = (long long)a->B * a->Hk * n.R;
  float* part = need ? (float*)ws : nullptr;
  float* stat = need ? part + (size_t)slots * rows * a->D : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  return with_shape(*a, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    const int grid = n.tiles * n.splits * a->B * a->Hk;
    if (shared)
      k_attn_fwd<T, DP, 1><<<grid, kThreads, 0, st>>>(n, (const T*)q, (const T*)k, (const T*)v, (T*)o, lse, part, stat);
    else
      k_attn_fwd<T, DP, 4><<<grid, kThreads, 0, st>>>(n, (const T*)q, (const T*)k, (const T*)v, (T*)o, lse, part, stat);
    if (need) k_attn_join<T><<<div_up(rows, kWaves), kThreads, 0, st>>>(n, part, stat, slots, (T*)o, lse);
    return check_launch("splat_attention_fwd");
  });
}

size_t splat_attention_bwd_workspace_bytes(const splat_attention* a) {
  if (check_attn("splat_attention_bwd_workspace_bytes", a) || a->B == 0) return 0;
  const Attn nk = plan_kv(*a), nq = plan_q(*a);
  const size_t rows = (size_t)a->B * a->Hk * nk.R;
  size_t n = up(sizeof(float) * rows);
  const size_t kv = nk.splits > 1 ? sizeof(float) * 2 * nk.splits * a->B * a->Lk * a->Hk * a->D : 0;
  const size_t dq = nq.splits > 1 ? sizeof(float) * nq.splits * rows * a->D : 0;
  return n + (kv > dq ? kv : dq);   // the two launches' partial sums follow each other in the same memory
}

int splat_attention_bwd(const splat_attention* a, const void* q, const void* k, const void* v, const void* o,
                        const float* lse, const void* g, void* dq, void* dk, void* dv, void* ws, size_t ws_bytes,
                        void* stream) {
  if (const int rc = check_attn("splat_attention_bwd", a)) return rc;
  if (a->B == 0 || (a->Lq == 0 && a->Lk == 0)) return kOk;
  if ((a->Lq > 0 && (!q || !o || !lse || !g || !dq)) || (a->Lk > 0 && (!k || !v || !dk || !dv)))
    return set_error(kInvalid, "splat_attention_bwd: null pointer");
  const Attn nk = plan_kv(*a), nq = plan_q(*a);
  const size_t need = splat_attention_bwd_workspace_bytes(a);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_attention_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  const long long rows = (long long)a->B * a->Hk * nk.R;
  float* delta = (float*)ws;
  float* part = (float*)((char*)ws + up(sizeof(float) * rows));
  const hipStream_t st = (hipStream_t)stream;
  return with_shape(*a, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    const T *tq = (const T*)q, *tk = (const T*)k, *tv = (const T*)v, *tg = (const T*)g;
    if (rows) k_attn_delta<T><<<div_up(rows, kThreads / 8), kThreads, 0, st>>>(nk, (const T*)o, tg, delta);
    if (a->Lk > 0) {
      const long long cnt = (long long)a->B * a->Lk * a->Hk * a->D;
      float* pk = nk.splits > 1 ? part : nullptr;
      k_attn_bwd_kv<T, DP><<<nk.tiles * nk.splits * a->B * a->Hk, kThreads, 0, st>>>(nk, tq, tk, tv, tg, lse, delta, (T*)dk,
                                                                                     (T*)dv, pk);
      if (pk) {
        k_attn_add<T><<<div_up(cnt, kThreads), kThreads, 0, st>>>(nk, pk, nk.splits, 2 * cnt, cnt, false, (T*)dk);
        k_attn_add<T><<<div_up(cnt, kThreads), kThreads, 0, st>>>(nk, pk + cnt, nk.splits, 2 * cnt, cnt, false, (T*)dv);
      }
    }
    if (a->Lq > 0) {
      const long long cnt = rows * a->D;
      float* pq = nq.splits > 1 ? part : nullptr;
      k_attn_bwd_q<T, DP><<<nq.tiles * nq.splits * a->B * a->Hk, kThreads, 0, st>>>(nq, tq, tk, tv, tg, lse, delta, (T*)dq,
                                                                                    pq);
      if (pq) k_attn_add<T><<<div_up(cnt, kThreads), kThreads, 0, st>>>(nq, pq, nq.splits, cnt, cnt, true, (T*)dq);
    }
    return check_launch("splat_attention_bwd");
  });
}

}  // extern "C"
