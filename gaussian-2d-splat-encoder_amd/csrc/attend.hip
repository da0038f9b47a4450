// Cross attention: o = softmax(scale q k^T) v over the valid keys, for queries q[B, Lq, H, D] and another sequence's
// keys and values k, v[B, Lk, Hk, D] (H a multiple of Hk: H / Hk query heads share a key head), and its gradients.
//
// The H / Hk heads that share keys are rows of one problem: row r = query * rep + head within the group, R = Lq * rep
// rows per (image, key head). Scores are held transposed, a lane per query (forward, dq) or per key (dk, dv), so that a
// softmax row is one lane pair and the probabilities are the next product's operand as they leave the first. One pass
// over the keys with a running maximum and sum; sums, statistics and accumulators are 32-bit floats, probabilities and
// score gradients are rounded to the inputs' type for the matrix instructions only (or taken as two values of it).
//
// Keys that a length or a mask leaves out are replaced by zeros as they are loaded, so that nothing they hold (NaN
// included) reaches a product; a row without valid keys gives zeros, and zero gradients.
//
// Measured on 36,864 rows and 9,216 keys of four heads of 64, bf16 (174 GFLOP a product; a large library
// product reaches 1,394 TFLOP/s here): forward 446 us (780 TFLOP/s), dk and dv 753 us (924), dq 543 us (962). Matrix and
// vector instructions take about the same time and overlap only in part: matrix units 37 to 47% busy, vector units 41 to
// 65%, LDS 54 to 60%. One pass for all three gradients would do with five products instead of seven, but dq would need
// atomics (whose order changes results) or 2.7 GB of partial sums.
#include "feat_common.h"
#include "splat_attention.h"

namespace splat {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kMaxSplits = 512;

// Probabilities and score gradients are operands of the second products and rounded to bf16 for them, once: results of many
// terms then are 2.35e-3 off where their own rounding is 1.66e-3. Few terms or few results do not average that (up to twice
// a result's own rounding), and score gradients of short heads lose more against the keys' weighted mean, which their sum
// of zero leaves out (dq of heads of 16 2.7e-3, of 40 2.5e-3, of 64 2.4e-3). Both are taken as sums of two bf16 values there
// (1.66e-3): in the forward of at most 64 rows, where memory is waited for (a token of 92,160 keys 24.8 -> 25.9 us), in the
// backward of at most kFineRows rows or keys (162 -> 163 us for 4 x 64 rows of 18,432 keys), and for dq of heads of at most
// kFineHead (8,192 x 8,192, four heads, forward and backward: of 32 261 -> 288 us, of 48 354 -> 387).
constexpr int kFineRows = 128, kFineHead = 48;

struct Attn {
  splat_attention a;
  int rep, R;            // query heads per key head; rows per (image, key head)
  FastDiv by_rep;
  int tiles, splits;     // workgroups per (image, key head) along the rows (or keys), and along the other axis
  int per;               // tiles of the other axis that a split takes
  bool chunked;          // heads are whole chunks, and offsets within a tile are 31-bit
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

// Bit i: key k0 + i counts (i < 64), the same in every lane. mask: the image's row, or null.
__device__ __forceinline__ unsigned long long valid_keys(const unsigned char* mask, long long ml, int k0, int len) {
  const int k = k0 + (threadIdx.x & 63);
  bool in = k < len;
  if (mask && in) in = mask[(long long)k * ml] != 0;
  return __ballot(in);
}

__device__ __forceinline__ const unsigned char* mask_row(const splat_attention& a, int b) {
  return a.key_mask ? a.key_mask + b * a.mb : nullptr;
}

// Adds 32 x 32 scores: acc = rows of `t` (LDS) times the lanes' register rows. Part: D leaves the last of a row's chunks
// empty, and the empty ones are skipped (4,096 x 4,096, four heads, forward and backward, float: heads of 40 617 us instead
// of 714, of 112 1,246 instead of 1,301; bf16: of 80 204 instead of 211, of 112 249 instead of 285). Kernels of their own:
// the branches cost heads of 64 2%. The loop has to unroll, as the rows' registers have no addresses: with more than eight
// chunks a row a way out of it keeps it rolled and the rows in memory (heads of 112, float: 2,432 us), so those are skipped
// one by one; the way out is 1% faster where it does unroll.
template <typename T, int DP, bool Part>
__device__ __forceinline__ void scores(f32x16& acc, const T* t, const RowFrag<T, DP>& f, int D, int lane) {
  constexpr int nc = Shape<T, DP>::nc, last = nc - 16 / kV<T>;   // the first chunk of the last 32 values holds some
#pragma unroll
  for (int c = 0; c < nc; ++c) {
    if (Part && c > last && (c == nc - 1 || 2 * c * kV<T> >= D)) {
      if constexpr (nc <= 8) break;
      else continue;
    }
    mma(acc, row_frag(t + 2 * c * kV<T>, Shape<T, DP>::ld, lane), f[c]);
  }
}

// What rounding x to o leaves.
template <typename O>
__device__ __forceinline__ O left_of(float x, O o) { return (O)(x - (float)o); }

// acc[d][lane] += sum over the 32 LDS rows from t of row[d] * p[row][lane], p as the results of scores(). Fine: p as the sum
// of two bf16 values, its rounding and what that leaves.
template <typename T, int DP, bool Fine>
__device__ __forceinline__ void gather(RowAcc<T, DP>& acc, const T* t, const f32x16& p, int lane) {
  constexpr int V = kV<T>;
#pragma unroll
  for (int c = 0; c < 16 / V; ++c) {
    Chunk<T> b, r;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      b.v[j] = (T)p[c * V + j];
      if (Fine) r.v[j] = left_of(p[c * V + j], b.v[j]);
    }
#pragma unroll
    for (int d = 0; d < Shape<T, DP>::nd; ++d) {
      const Chunk<T> f = col_frag<true>(t + 2 * V * c * Shape<T, DP>::ld + 32 * d, Shape<T, DP>::ld, lane);
      mma(acc[d], f, b);
      if (Fine) mma(acc[d], f, r);
    }
  }
}

struct Work {
  int tile, split, b, hk, bh;
};

// Workgroup -> (image, key head), tile and split. The card works on one head's workgroups after the other, each XCD on a
// band of them: its L2 holds the other side's head, and images without keys leave no XCD idle (with a band of heads each,
// a third of the XCDs had nothing to do where one image of three was empty: 55 us instead of 40).
__device__ __forceinline__ Work work_of(const Attn& n) {
  const int per = n.tiles * n.splits, bh = blockIdx.x / per, id = xcd_swizzle(blockIdx.x - bh * per, per);
  Work w;
  w.tile = id % n.tiles;
  w.split = id / n.tiles;
  w.bh = bh;
  w.b = w.bh / n.a.Hk;
  w.hk = w.bh % n.a.Hk;
  return w;
}

// Place `at` of what the outputs' rounding left, null where that is not kept (floats, inference).
template <typename T>
__device__ __forceinline__ T* rest_of(const splat_attention& a, long long at) {
  return sizeof(T) == 2 && a.rest ? (T*)a.rest + at : nullptr;
}
// The same of floats' inverse sums.
template <typename T>
__device__ __forceinline__ float* inverse_of(const splat_attention& a, long long at) {
  return sizeof(T) == 4 && a.rest ? (float*)a.rest + at : nullptr;
}

// What the backward takes of a row: its maximum m in exponents of two and its sum l of 2^(score - m), as p = 2^(score - lse)
// with lse = m + log2 l, or p = 2^(score - m) / l for floats: lse is a number of about 20, whose own last bit would move all
// of a row's probabilities by 7e-7 (one token of 33,793 keys: dv 1.2e-6 off instead of 7.6e-7).
template <typename T>
__device__ __forceinline__ void keep_row(const splat_attention& a, float* lse, long long at, float m, float l) {
  float* inv = inverse_of<T>(a, at);
  lse[at] = l == 0.f ? INFINITY : inv ? m : m + hw_log2(l);
  if (inv) *inv = l > 0.f ? 1.f / l : l;
}

// Address of row r's head vector in a tensor of strides (sb, sl, sh).
template <typename T>
__device__ __forceinline__ const T* head_row(const void* p, const Attn& n, const Work& w, int r, long long sb, long long sl,
                                             long long sh) {
  const int q = r / n.by_rep, j = r - q * n.rep;
  return (const T*)p + w.b * sb + q * sl + (long long)(w.hk * n.rep + j) * sh;
}

// N rows of an LDS tile: global -> registers -> LDS. A thread has one column of chunks and every RS-th row, so that whole
// tiles load from scalar bases and one offset that stays, without address arithmetic per tile. Heads that are not whole
// chunks (D no multiple of V) are copied value by value when the tile is written.
template <typename T, int DP, int N>
struct Rows {
  static constexpr int V = kV<T>, CP = DP == 96 ? 128 / V : DP / V;   // chunks of a row, a power of two
  static constexpr int RS = kThreads / CP, per = N > RS ? N / RS : 1;
  Chunk<T> c[per];
  unsigned off;   // the thread's elements from the tile's base
  bool on;        // its column holds values

  __device__ static int row0() { return threadIdx.x / CP; }
  __device__ static int col() { return threadIdx.x % CP * V; }
  __device__ static T* place(T* t, int i) { return t + (row0() + i * RS) * Shape<T, DP>::ld + col(); }
  __device__ static bool holds() { return (N >= RS || row0() < N) && (DP != 96 || col() < DP); }
  // offset: elements from a tile's base to the thread's row row0().
  __device__ void init(int D, int offset) {
    off = offset + col();
    on = col() < D && (N >= RS || row0() < N);
  }
  __device__ void load(const T* base, long long step) {   // step: elements from row to row + RS
#pragma unroll
    for (int i = 0; i < per; ++i) {
      c[i] = Chunk<T>{};
      if (on) __builtin_memcpy(c[i].v, base + i * step + off, 16);
    }
  }
  template <typename F>
  __device__ void load(F&& row) {   // row(i): pointer of row i, or null for zeros
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const T* p = on ? row(row0() + i * RS) : nullptr;
      c[i] = Chunk<T>{};
      if (p) __builtin_memcpy(c[i].v, p + col(), 16);
    }
  }
  __device__ void put(T* t) const {
#pragma unroll
    for (int i = 0; i < per; ++i)
      if (holds()) *(f32x4*)place(t, i) = *(const f32x4*)c[i].v;
  }
  __device__ static void scale(Chunk<T>& x, float by) {
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = (T)((float)x.v[j] * by);
  }
  __device__ void scale(const float (&by)[per]) {   // row i by by[i]
#pragma unroll
    for (int i = 0; i < per; ++i) scale(c[i], by[i]);
  }
  template <typename F>
  __device__ static void copy(T* t, int D, F&& row) {
    copy(t, D, row, [](int, Chunk<T>&) {});
  }
  template <typename F, typename G>
  __device__ static void copy(T* t, int D, F&& row, G&& change) {   // change(i, chunk of row i)
#pragma unroll 1
    for (int i = 0; i < per; ++i) {
      if (!holds()) continue;
      const T* p = row(row0() + i * RS);
      Chunk<T> x = load_chunk(p + col(), p ? D - col() : 0);
      change(row0() + i * RS, x);
      *(f32x4*)place(t, i) = *(const f32x4*)x.v;
    }
  }
};

// Tiles of N keys and values in turn: fetch(t) loads tile t to registers and says which of its keys count, put() writes it.
template <typename T, int DP, int N>
struct KeyTiles {
  const T *k, *v;               // the head's first key and value
  long long kl, vl, ml;
  const unsigned char* mask;
  int D, len;
  bool chunked;                 // rows are whole chunks
  Rows<T, DP, N> rk, rv;
  unsigned long long ok0, ok1;  // the fetched tile's keys that count: the first 64, the others
  unsigned char m0, m1;         // the lane's mask bytes of the tile to be fetched next
  int k0;

  __device__ KeyTiles(const Attn& n, const Work& w, const T* kp, const T* vp)
      : k(kp + w.b * n.a.kb + w.hk * n.a.kh), v(vp + w.b * n.a.vb + w.hk * n.a.vh), kl(n.a.kl), vl(n.a.vl), ml(n.a.ml),
        mask(mask_row(n.a, w.b)), D(n.a.D), len(key_count(n.a, w.b)), chunked(n.chunked), ok0(0), ok1(0), m0(0), m1(0), k0(0) {
    rk.init(D, rk.row0() * (int)kl);
    rv.init(D, rv.row0() * (int)vl);
  }
  // Requests the mask of tile t: before its keys are, which wait for it.
  __device__ __forceinline__ void peek(int t) {
    const int i = t * N + (threadIdx.x & 63);
    m0 = i < len && (!mask || mask[(long long)i * ml] != 0);
    m1 = N > 64 && i + 64 < len && (!mask || mask[(long long)(i + 64) * ml] != 0);
  }
  __device__ __forceinline__ void begin(int t) {
    peek(t);
    fetch(t);
  }
  __device__ __forceinline__ const T* row(const T* p, long long l, int i) const {
    return ((N > 64 && i >= 64 ? ok1 : ok0) >> (i & 63)) & 1 ? p + (k0 + i) * l : nullptr;
  }
  __device__ __forceinline__ void fetch(int t) {
    k0 = t * N;
    if (chunked && !mask && k0 + N <= len) {
      ok0 = ok1 = ~0ull;
      rk.load(k + k0 * kl, rk.RS * kl);
      rv.load(v + k0 * vl, rv.RS * vl);
      return;
    }
    if (!mask) peek(t);
    ok0 = __ballot(m0);
    ok1 = N > 64 ? __ballot(m1) : 0;
    if (chunked) {
      rk.load([&](int i) { return row(k, kl, i); });
      rv.load([&](int i) { return row(v, vl, i); });
    }
    if (mask) peek(t + 1);
  }
  __device__ __forceinline__ void put(T* tk, T* tv) const {
    if (chunked) {
      rk.put(tk);
      rv.put(tv);
    } else {
      Rows<T, DP, N>::copy(tk, D, [&](int i) { return row(k, kl, i); });
      Rows<T, DP, N>::copy(tv, D, [&](int i) { return row(v, vl, i); });
    }
  }
};

// Writes the lane's row of DP values, scaled, from the accumulators; to `rest`, unless null, what rounding them leaves.
template <typename T, typename O, int DP>
__device__ __forceinline__ void store_row(O* row, const RowAcc<T, DP>& acc, float s, int D, bool in, int h,
                                          O* rest = nullptr) {
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
      if (in && rest) {
        Chunk<O> r;
#pragma unroll
        for (int e = 0; e < kV<O>; ++e) r.v[e] = left_of(run[t][e] * s, o.v[e]);
        store_chunk(rest + c, r, D - c);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ forward
// Of the workgroup's four waves QW take 32 rows each and 4 / QW share the keys of a tile between them: few rows would
// leave waves idle otherwise. A wave's 32-key blocks of a tile (two for bf16, one for float) are one softmax step. Key and
// value tiles go through registers into two LDS buffers in turn: the next tile's loads are in flight during a step, and
// one barrier a tile suffices (where only one buffer fits, two). Waves that shared keys join their results in LDS, splits
// of the key axis in k_attn_join. Few rows are bound by reading keys and values: one token, 92,160 keys of four heads of 64
// in bf16 (94 MB) 22 us, 4.3 TB/s, and 4 us to join.
template <typename T, int DP, int QW>
struct FwdShape {
  static constexpr int KW = kWaves / QW;
  static constexpr bool fine = sizeof(T) == 2 && QW < 4;
  static constexpr int KB = sizeof(T) == 2 && QW > 1 ? 2 : 1;   // 32-key blocks of a wave
  static constexpr int KT = 32 * KB * KW;
  static constexpr int tile = KT * Shape<T, DP>::ld;
  static constexpr int buffers = 4 * tile * (int)sizeof(T) <= 140 * 1024 ? 2 : 1;
  static constexpr int lds = 2 * buffers * tile;                // elements: keys and values
  static_assert(lds * sizeof(T) >= sizeof(float) * (kWaves - QW) * 64 * (DP / 2 + 2), "the join's values fit");
};

// Adds to the running softmax of the lane's row the scores s of a step, `live` the keys that count (0 .. 32 KB - 1): m the
// maximum that l and acc are scaled by, in units of the raw scores; c > 0 turns those into exponents of two. The maximum
// is only raised when it grew by more than 2^8 in the result: l and acc are scaled by 2^-m either way.
template <typename T, int DP, int KB>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[KB], unsigned long long live, float c, float& m, float& l,
                                             RowAcc<T, DP>& acc, int h) {
  if (live != (KB == 2 ? ~0ull : 0xffffffffull)) {
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const unsigned bits = (unsigned)(live >> (32 * b)) >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = (bits >> acc_row(i, 0)) & 1 ? s[b][i] : -INFINITY;
    }
  }
  float mx = s[0][0];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
  const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
  mx = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1]));
  if (__any(mx > m + fminf(8.f / c, 1e30f))) {
    const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn;
    const float al = hw_exp2((m - mu) * c);
    m = mn;
    l *= al;
#pragma unroll
    for (int d = 0; d < Shape<T, DP>::nd; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] *= al;
  }
  const float mc = m == -INFINITY ? 0.f : m * c;
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < KB; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[b][i] = hw_exp2(fmaf(s[b][i], c, -mc));
      sum += s[b][i];
    }
  }
  l += sum;
}

template <typename T, int DP, bool Part, int QW>
__global__ __launch_bounds__(kThreads) void k_attn_fwd(Attn n, const T* __restrict__ q, const T* __restrict__ k,
                                                       const T* __restrict__ v, T* __restrict__ o, float* __restrict__ lse,
                                                       float* __restrict__ part, float* __restrict__ stat) {
  using S = Shape<T, DP>;
  using F = FwdShape<T, DP, QW>;
  __shared__ __align__(16) T tiles[F::lds];
  const splat_attention& a = n.a;
  const Work w = work_of(n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int wq = wave % QW, wk = wave / QW;
  const int r = (w.tile * QW + wq) * 32 + (lane & 31);
  const bool in = r < n.R;
  const int kw = wk * 32 * F::KB;   // the wave's first key of a tile
  Chunk<T> fq[S::nc];
  load_rows<T, DP>(fq, head_row<T>(q, n, w, in ? r : 0, a.qb, a.ql, a.qh), in, a.D, h);
  if (a.scale < 0.f) {   // the running maximum is of raw scores: their sign goes to the queries
#pragma unroll
    for (int i = 0; i < S::nc; ++i)
#pragma unroll
      for (int j = 0; j < S::V; ++j) fq[i].v[j] = -fq[i].v[j];
  }
  const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.17549435e-38f);
  KeyTiles<T, DP, F::KT> kt(n, w, k, v);
  const int t0 = w.split * n.per, t1 = min((kt.len + F::KT - 1) / F::KT, t0 + n.per);
  f32x16 acc[S::nd] = {};
  float m = -INFINITY, l = 0.f;
  if (t0 < t1) kt.begin(t0);
  for (int t = t0; t < t1; ++t) {
    unsigned long long live = F::KT > 64 && kw >= 64 ? kt.ok1 : kt.ok0;
    live >>= kw & 63;
    if (F::KB == 1) live &= 0xffffffffull;
    T* tk = tiles + (F::buffers == 2 ? (t & 1) * 2 * F::tile : 0);
    T* tv = tk + F::tile;
    if (F::buffers == 1) __syncthreads();
    kt.put(tk, tv);
    __syncthreads();
    if (t + 1 < t1) kt.fetch(t + 1);
    if (!live) continue;
    f32x16 s[F::KB] = {};
#pragma unroll
    for (int b = 0; b < F::KB; ++b) scores<T, DP, Part>(s[b], tk + (kw + 32 * b) * S::ld, fq, a.D, lane);
    softmax_step<T, DP, F::KB>(s, live, c, m, l, acc, h);
#pragma unroll
    for (int b = 0; b < F::KB; ++b) gather<T, DP, F::fine>(acc, tv + (kw + 32 * b) * S::ld, s[b], lane);
  }
  l += __shfl_xor(l, 32, 64);
  if (QW < kWaves) {   // the waves of the same rows: the first one adds the others' results in their order
    __syncthreads();
    float* join = (float*)tiles;
    constexpr int per = 64 * (DP / 2 + 2);   // a wave's values
    if (wk > 0) {
      float* p = join + ((wk - 1) * QW + wq) * per + lane;
      p[0] = m;
      p[64] = l;
#pragma unroll
      for (int d = 0; d < S::nd; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) p[64 * (2 + 16 * d + i)] = acc[d][i];
    }
    __syncthreads();
    if (wk > 0) return;
    for (int j = 1; j < F::KW; ++j) {
      const float* p = join + ((j - 1) * QW + wq) * per + lane;
      const float mo = p[0], mn = fmaxf(m, mo), mu = mn == -INFINITY ? 0.f : mn;
      const float x = hw_exp2((m - mu) * c), y = hw_exp2((mo - mu) * c);
      m = mn;
      l = fmaf(l, x, p[64] * y);
#pragma unroll
      for (int d = 0; d < S::nd; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = fmaf(acc[d][i], x, p[64 * (2 + 16 * d + i)] * y);
    }
  }
  m *= c;   // from here in exponents of two
  if (part) {
    const long long at = ((long long)w.split * n.a.B * n.a.Hk + w.bh) * n.R + r;
    if (in && h == 0) {
      stat[2 * at] = m;
      stat[2 * at + 1] = l;
    }
    store_row<T, float, DP>(part + at * a.D, acc, 1.f, a.D, in, h);
  } else {
    const float inv = l > 0.f ? 1.f / l : l;   // 0 for a row without keys, NaN stays
    if (lse && in && h == 0) keep_row<T>(a, lse, (long long)w.bh * n.R + r, m, l);
    const int qi = r / n.by_rep, j = r - qi * n.rep;
    const long long at = ((w.b * a.Lq + qi) * a.H + w.hk * n.rep + j) * a.D;
    store_row<T, T, DP>(o + at, acc, inv, a.D, in, h, rest_of<T>(a, at));
  }
}

// Joins the splits' partial results of a row, one workgroup a row: lanes over the head's values, groups of lanes over the
// splits, whose sums are added in LDS in their order. The first values are on their way while the statistics are joined:
// 4 us for 120 splits of four rows, 6 with them asked for afterwards.
constexpr int kJoinThreads = 1024;
template <typename T, int DP>
__global__ __launch_bounds__(kJoinThreads) void k_attn_join(Attn n, const float* __restrict__ part,
                                                            const float* __restrict__ stat, T* __restrict__ o,
                                                            float* __restrict__ lse) {
  constexpr int W = DP == 96 ? 128 : DP, GS = kJoinThreads / W, U = 8;   // groups; splits that a lane asks for at a time
  __shared__ float weight[kMaxSplits], sums[GS * W], total;
  const splat_attention& a = n.a;
  const long long rows = (long long)a.B * a.Hk * n.R, row = blockIdx.x;
  const int d = threadIdx.x % W, g = threadIdx.x / W, lane = threadIdx.x & 63;
  const float* p = part + row * a.D + d;
  float v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = d < a.D && g + u * GS < n.splits ? p[(g + u * GS) * rows * a.D] : 0.f;
  if (threadIdx.x < 64) {
    float m = -INFINITY;
    for (int s = lane; s < n.splits; s += 64) m = fmaxf(m, stat[2 * (s * rows + row)]);
#pragma unroll
    for (int e = 32; e >= 1; e >>= 1) m = fmaxf(m, __shfl_xor(m, e, 64));
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < n.splits; s += 64) {
      const float e = hw_exp2(stat[2 * (s * rows + row)] - mu);
      weight[s] = e;
      l = fmaf(stat[2 * (s * rows + row) + 1], e, l);
    }
    l = wave_add(l);
    if (lane == 0) {
      total = l > 0.f ? 1.f / l : l;
      if (lse) keep_row<T>(a, lse, row, m, l);
    }
  }
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (g + u * GS < n.splits) s = fmaf(v[u], weight[g + u * GS], s);
  if (d < a.D) {
    for (int i = g + U * GS; i < n.splits; i += GS) s = fmaf(p[i * rows * a.D], weight[i], s);
  }
  sums[g * W + d] = s;
  __syncthreads();
  if (threadIdx.x < a.D) {
    s = sums[threadIdx.x];
#pragma unroll
    for (int i = 1; i < GS; ++i) s += sums[i * W + threadIdx.x];
    const int bh = (int)(row / n.R), r = (int)(row - (long long)bh * n.R);
    const int qi = r / n.by_rep, j = r - qi * n.rep, b = bh / a.Hk, hk = bh % a.Hk;
    const long long at = (((long long)b * a.Lq + qi) * a.H + hk * n.rep + j) * a.D + threadIdx.x;
    o[at] = (T)(s * total);
    if (T* r = rest_of<T>(a, at)) *r = left_of(s * total, o[at]);
  }
}

// Four values of a row to its place, of which `left` are the row's.
template <typename T>
__device__ __forceinline__ void store_head(T* p, const float (&s)[4], int left) {
  T x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (T)s[e];
  if (left >= 4) {
    __builtin_memcpy(p, x, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = x[e];
  }
}

// The same for few splits (rows are many then): a thread per four values of a row. Two splits of 147,456 rows of 64: 17 us
// (5.5 TB/s), 20 with what the outputs' rounding leaves.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_attn_join_few(Attn n, FastDiv by_quads, int quads, const float* __restrict__ part,
                                                            const float* __restrict__ stat, T* __restrict__ o,
                                                            float* __restrict__ lse) {
  const splat_attention& a = n.a;
  const int rows = a.B * a.Hk * n.R, i = blockIdx.x * kThreads + threadIdx.x;
  const int row = i / by_quads, d = (i - row * quads) * 4;
  if (row >= rows) return;
  Chunk<float> s = load_chunk(part + (long long)row * a.D + d, a.D - d);
  float2 ml = *(const float2*)(stat + 2LL * row);
  for (int k = 1; k < n.splits; ++k) {
    const long long at = (long long)k * rows + row;
    const Chunk<float> x = load_chunk(part + at * a.D + d, a.D - d);
    const float2 mo = *(const float2*)(stat + 2 * at);
    const float mn = fmaxf(ml.x, mo.x), mu = mn == -INFINITY ? 0.f : mn;
    const float e = hw_exp2(ml.x - mu), f = hw_exp2(mo.x - mu);
    ml = make_float2(mn, fmaf(ml.y, e, mo.y * f));
#pragma unroll
    for (int j = 0; j < 4; ++j) s.v[j] = fmaf(s.v[j], e, x.v[j] * f);
  }
  const float inv = ml.y > 0.f ? 1.f / ml.y : ml.y;
  const int bh = row / n.R, r = row - bh * n.R;
  const int qi = r / n.by_rep, j = r - qi * n.rep, b = bh / a.Hk, hk = bh % a.Hk;
  const long long at = (((long long)b * a.Lq + qi) * a.H + hk * n.rep + j) * a.D + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) s.v[e] *= inv;
  store_head(o + at, s.v, a.D - d);
  if (T* r = rest_of<T>(a, at)) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = s.v[e] - (float)(T)s.v[e];
    store_head(r, x, a.D - d);
  }
  if (lse && d == 0) keep_row<T>(a, lse, row, ml.x, ml.y);
}

// ----------------------------------------------------------------------------------------------- backward
// delta[row] = sum over d of do * o, which the score gradients p (dp - delta) take, o with what its rounding left: where a few
// keys hold most of a row's weight, dp - delta is far smaller than either, and a bf16 output's rounding four times the
// gradients' own (8 keys, heads of 32: dq 5.9e-3 off instead of 2.3e-3). Bound by memory: 147,456 rows of 64 bf16 16.5 us
// (3.4 TB/s).
template <typename T>
__global__ __launch_bounds__(kThreads) void k_attn_delta(Attn n, const T* __restrict__ o, const T* __restrict__ g,
                                                         float* __restrict__ delta) {
  const splat_attention& a = n.a;
  // eight lanes a row
  const long long row = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;
  if (row >= (long long)a.B * a.Hk * n.R) return;
  const int bh = (int)(row / n.R), r = (int)(row - (long long)bh * n.R);
  const int qi = r / n.by_rep, j = r - qi * n.rep, b = bh / a.Hk, hq = bh % a.Hk * n.rep + j;
  const long long at = (((long long)b * a.Lq + qi) * a.H + hq) * a.D;
  const T *op = o + at, *rp = rest_of<T>(a, at);
  const T* gp = g + b * a.gb + qi * a.gl + hq * a.gh;
  float s = 0.f;
  for (int d = (threadIdx.x & 7) * kV<T>; d < a.D; d += 8 * kV<T>) {
    const Chunk<T> x = load_chunk(op + d, a.D - d), y = load_chunk(gp + d, a.D - d);
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) s = fmaf((float)x.v[e], (float)y.v[e], s);
    if (rp) {
      const Chunk<T> r = load_chunk(rp + d, a.D - d);
#pragma unroll
      for (int e = 0; e < kV<T>; ++e) s = fmaf((float)r.v[e], (float)y.v[e], s);
    }
  }
  s += __shfl_xor(s, 1, 64);
  s += __shfl_xor(s, 2, 64);
  s += __shfl_xor(s, 4, 64);
  if ((threadIdx.x & 7) == 0) delta[row] = s;
}

// Rows (dk, dv) or keys (dq) of an LDS tile of the backward; two of them in turn, as in the forward.
template <typename T> constexpr int kBwdTile = sizeof(T) == 2 ? 64 : 32;

// dk and dv: a wave holds 32 keys and values, the workgroup's four share tiles of query rows. With s = q k^T a lane is a
// key: p and ds are the operands of dv = p^T do and dk = ds^T q as they are. 64 keys a wave would halve the LDS reads but
// leave one wave a SIMD (1,014 us instead of 793).
template <typename T, int DP, bool Part, bool Fine>
__global__ __launch_bounds__(kThreads) void k_attn_bwd_kv(Attn n, const T* __restrict__ q, const T* __restrict__ k,
                                                          const T* __restrict__ v, const T* __restrict__ g,
                                                          const float* __restrict__ lse, const float* __restrict__ delta,
                                                          T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
  using S = Shape<T, DP>;
  constexpr int QT = kBwdTile<T>, tile = QT * S::ld;
  __shared__ __align__(16) T tiles[4 * tile];
  __shared__ __align__(16) float stats[4 * QT];
  const splat_attention& a = n.a;
  const Work w = work_of(n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int len = key_count(a, w.b);
  const int k0 = w.tile * 128 + (wave & 2) * 32;
  const unsigned long long ok = valid_keys(mask_row(a, w.b), a.ml, k0, len);
  const int ki = w.tile * 128 + wave * 32 + (lane & 31);
  const bool good = (ok >> ((wave & 1) * 32 + (lane & 31))) & 1;
  Chunk<T> fk[S::nc], fv[S::nc];
  load_rows<T, DP>(fk, k + w.b * a.kb + w.hk * a.kh + (good ? ki : 0) * a.kl, good, a.D, h);
  load_rows<T, DP>(fv, v + w.b * a.vb + w.hk * a.vh + (good ? ki : 0) * a.vl, good, a.D, h);
  const bool any = w.tile * 128 < len;
  const int t0 = w.split * n.per, t1 = any ? min((n.R + QT - 1) / QT, t0 + n.per) : t0;
  const float c = a.scale * kLog2e;
  f32x16 ak[S::nd] = {}, av[S::nd] = {};
  Rows<T, DP, QT> rq, rg;
  // tiles, and a thread's rows of one, are whole queries apart where their row counts are multiples of rep
  const bool whole = n.chunked && QT % n.rep == 0 && (rq.per == 1 || rq.RS % n.rep == 0);
  const int qi0 = rq.row0() / n.by_rep, j0 = rq.row0() - qi0 * n.rep, qs = rq.RS / n.by_rep;
  rq.init(a.D, qi0 * (int)a.ql + j0 * (int)a.qh);
  rg.init(a.D, qi0 * (int)a.gl + j0 * (int)a.gh);
  const T* qp = head_row<T>(q, n, w, 0, a.qb, a.ql, a.qh);
  const T* gp = head_row<T>(g, n, w, 0, a.gb, a.gl, a.gh);
  const float* lp = lse + (long long)w.bh * n.R;
  const float* dp0 = delta + (long long)w.bh * n.R;
  // Floats' probabilities lack the factor 1 / l, which the gradient's rows and delta carry instead: ds and dv take both.
  const float* ip = inverse_of<T>(a, (long long)w.bh * n.R);
  float sl = 0.f, sd = 0.f, inv[rg.per];
  int r0 = 0;
  auto qrow = [&](int i) { return r0 + i < n.R ? head_row<T>(q, n, w, r0 + i, a.qb, a.ql, a.qh) : nullptr; };
  auto grow = [&](int i) { return r0 + i < n.R ? head_row<T>(g, n, w, r0 + i, a.gb, a.gl, a.gh) : nullptr; };
  auto inverse = [&](int i) { return ip[min(r0 + i, n.R - 1)]; };
  auto fetch = [&](int t) {
    r0 = t * QT;
    if (whole && r0 + QT <= n.R) {
      const int q0 = r0 / n.by_rep;
      rq.load(qp + q0 * a.ql, qs * a.ql);
      rg.load(gp + q0 * a.gl, qs * a.gl);
    } else if (n.chunked) {
      rq.load(qrow);
      rg.load(grow);
    }
    if (ip) {
#pragma unroll
      for (int i = 0; i < rg.per; ++i) inv[i] = inverse(rg.row0() + i * rg.RS);
    }
    if (threadIdx.x < QT) {
      const int r = r0 + threadIdx.x;
      sl = r < n.R ? -lp[r] : -INFINITY;
      sd = r < n.R ? -dp0[r] : 0.f;
      if (ip && r < n.R) sd *= ip[r];
    }
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    T* tq = tiles + (t & 1) * 2 * tile;
    T* tg = tq + tile;
    float* tl = stats + (t & 1) * 2 * QT;
    float* td = tl + QT;
    if (n.chunked) {
      rq.put(tq);
      if (ip) rg.scale(inv);
      rg.put(tg);
    } else {
      Rows<T, DP, QT>::copy(tq, a.D, qrow);
      Rows<T, DP, QT>::copy(tg, a.D, grow, [&](int i, Chunk<T>& x) {
        if (ip) rg.scale(x, inverse(i));
      });
    }
    if (threadIdx.x < QT) {
      tl[threadIdx.x] = sl;
      td[threadIdx.x] = sd;
    }
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
#pragma unroll 1
    for (int rb = 0; rb < QT; rb += 32) {
      f32x16 s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; i += 4) {   // dp starts at -delta
        const f32x4 D = *(const f32x4*)(td + rb + acc_row(i, h));
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[i + e] = D[e];
      }
      scores<T, DP, Part>(s, tq + rb * S::ld, fk, a.D, lane);
      scores<T, DP, Part>(dp, tg + rb * S::ld, fv, a.D, lane);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 L = *(const f32x4*)(tl + rb + acc_row(i, h));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i + e] = hw_exp2(fmaf(s[i + e], c, L[e]));
          dp[i + e] *= s[i + e];
        }
      }
      gather<T, DP, Fine>(av, tg + rb * S::ld, s, lane);
      gather<T, DP, Fine>(ak, tq + rb * S::ld, dp, lane);
    }
  }
  if (!good) {   // the lane gathered what a key of zeros would get (infinite where the rows' scores are far below zero)
#pragma unroll
    for (int d = 0; d < S::nd; ++d) ak[d] = av[d] = f32x16{};
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
// Three waves a SIMD for bf16 heads of 64, at the cost of 20 bytes of scratch a lane (with a few registers more there are two
// waves: 646 us instead of 578 at 36,864 rows and 9,216 keys of 4 heads).
template <typename T, int DP, bool Part, bool Fine>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && DP <= 64 && !Fine ? 3 : 1)
void k_attn_bwd_q(Attn n, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ g,
                  const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dq,
                  float* __restrict__ part) {
  using S = Shape<T, DP>;
  constexpr int KT = kBwdTile<T>, tile = KT * S::ld;
  __shared__ __align__(16) T tiles[4 * tile];
  const splat_attention& a = n.a;
  const Work w = work_of(n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int r = w.tile * 128 + wave * 32 + (lane & 31);
  const bool in = r < n.R;
  Chunk<T> fq[S::nc], fg[S::nc];
  load_rows<T, DP>(fq, head_row<T>(q, n, w, in ? r : 0, a.qb, a.ql, a.qh), in, a.D, h);
  load_rows<T, DP>(fg, head_row<T>(g, n, w, in ? r : 0, a.gb, a.gl, a.gh), in, a.D, h);
  const float L = in ? -lse[(long long)w.bh * n.R + r] : -INFINITY;
  const float dl = in ? -delta[(long long)w.bh * n.R + r] : 0.f;
  KeyTiles<T, DP, KT> kt(n, w, k, v);
  const int t0 = w.split * n.per, t1 = min((kt.len + KT - 1) / KT, t0 + n.per);
  const float c = a.scale * kLog2e;
  f32x16 acc[S::nd] = {};
  if (t0 < t1) kt.begin(t0);
  for (int t = t0; t < t1; ++t) {
    const unsigned long long live = KT == 64 ? kt.ok0 : kt.ok0 & 0xffffffffull;
    T* tk = tiles + (t & 1) * 2 * tile;
    T* tv = tk + tile;
    kt.put(tk, tv);
    __syncthreads();
    if (t + 1 < t1) kt.fetch(t + 1);
    if (!live) continue;
#pragma unroll 1
    for (int k0 = 0; k0 < KT; k0 += 32) {
      f32x16 s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = dl;   // dp starts at -delta
      scores<T, DP, Part>(s, tk + k0 * S::ld, fq, a.D, lane);
      scores<T, DP, Part>(dp, tv + k0 * S::ld, fg, a.D, lane);
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] *= hw_exp2(fmaf(s[i], c, L));
      if (live != (KT == 64 ? ~0ull : 0xffffffffull)) {
        const unsigned bits = (unsigned)(live >> k0) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = (bits >> acc_row(i, 0)) & 1 ? dp[i] : 0.f;
      }
      gather<T, DP, Fine>(acc, tk + k0 * S::ld, dp, lane);
    }
  }
  const float* ip = inverse_of<T>(a, (long long)w.bh * n.R);
  const float sc = ip && in ? a.scale * ip[r] : a.scale;
  if (part) {
    const long long rows = (long long)a.B * a.Hk * n.R;
    store_row<T, float, DP>(part + (w.split * rows + (long long)w.bh * n.R + r) * a.D, acc, sc, a.D, in, h);
  } else {
    const int qi = r / n.by_rep, j = r - qi * n.rep;
    store_row<T, T, DP>(dq + ((w.b * a.Lq + qi) * a.H + w.hk * n.rep + j) * a.D, acc, sc, a.D, in, h);
  }
}

// Adds the splits' partial gradients in their order, a thread per four values of a row, four splits asked for at a time.
// Rows of `part` are the output's own order, or (heads) the rows of (image, key head) problems; the grid's second half in y
// adds the rows behind them to out1. Bound by memory: two splits of 147,456 rows of 64 to bf16 15.5 us (6.1 TB/s, part of
// it still cached; 34 with a thread a value), seven splits of twice 36,864 rows 22 us (two launches: 33).
template <typename T>
__global__ __launch_bounds__(kThreads) void k_attn_add(Attn n, FastDiv by_quads, int quads, const float* __restrict__ part,
                                                       int splits, long long stride, int rows, bool heads,
                                                       T* __restrict__ out0, T* __restrict__ out1) {
  const splat_attention& a = n.a;
  const int i = blockIdx.x * kThreads + threadIdx.x, row = i / by_quads, d = (i - row * quads) * 4;
  if (row >= rows) return;
  const float* p = part + ((long long)blockIdx.y * rows + row) * a.D + d;
  float s[4] = {};
  auto add = [&](auto m, int k) {
    constexpr int M = decltype(m)::value;
    Chunk<float> v[M];
#pragma unroll
    for (int j = 0; j < M; ++j) v[j] = load_chunk(p + (k + j) * stride, a.D - d);
#pragma unroll
    for (int j = 0; j < M; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[j].v[e];
  };
  int k = 0;
  for (; k + 4 <= splits; k += 4) add(std::integral_constant<int, 4>{}, k);
  if (k + 2 <= splits) {
    add(std::integral_constant<int, 2>{}, k);
    k += 2;
  }
  if (k < splits) add(std::integral_constant<int, 1>{}, k);
  long long at = row;
  if (heads) {
    const int bh = row / n.R, r = row - bh * n.R, qi = r / n.by_rep, j = r - qi * n.rep, b = bh / a.Hk, hk = bh % a.Hk;
    at = ((long long)b * a.Lq + qi) * a.H + hk * n.rep + j;
  }
  store_head((blockIdx.y ? out1 : out0) + at * a.D + d, s, a.D - d);
}

// ---------------------------------------------------------------------------------------------- launches
int check_attn(const char* what, const splat_attention* a) {
  if (!a) return set_error(kInvalid, "%s: null description", what);
  if (a->dtype != kF32 && a->dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", what, a->dtype);
  if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk || a->D < 1)
    return set_error(kInvalid, "%s: B %d, Lq %lld, Lk %lld, H %d, Hk %d, D %d", what, a->B, a->Lq, a->Lk, a->H, a->Hk, a->D);
  if (!(fabsf(a->scale) <= 3.40282347e+38f)) return set_error(kInvalid, "%s: scale %g", what, (double)a->scale);
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
    auto width = [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      return a.D <= DP - 2 * kV<T> ? f(t, dp, std::true_type{}) : f(t, dp, std::false_type{});
    };
    if (a.D <= 32) return width(std::integral_constant<int, 32>{});
    if (a.D <= 64) return width(std::integral_constant<int, 64>{});
    if (a.D <= 96) return width(std::integral_constant<int, 96>{});
    return width(std::integral_constant<int, 128>{});
  };
  return a.dtype == kF32 ? go(float{}) : go(bf16{});
}

// Splits of an axis of `tiles` tiles for `groups` workgroups of which `slots` run at a time: the number with the least
// estimated time, in tiles, of the rounds that the card takes (a last round that is not full runs faster, by about half of
// what it lacks) where writing and joining partial results costs a split about as much as six tiles. At least three tiles a
// split (64 rows and 18,432 masked bf16 keys: 16 us; 18 with four, 23 with eight).
// A float tile takes sixteen times the matrix instructions' time: one workgroup a CU is a round there, and a split costs
// about one tile. Where lengths or a mask, which only the device knows, may leave workgroups idle, more of them even out
// what is left: two rounds are added to the estimate. Training calls' kernels with them and without, the last image empty,
// lengths / mask: float, 3 x 1,201 x 777 (2 key heads of 40) 177 (205) / 206 (205) us, 2 x 4,000 x 3,000 (4 of 64) 612 (871)
// / 826 (1,076), 4 x 300 x 5,000 (4 of 64) 335 (321) / 370 (389), 2 x 9,000 x 2,000 (2 of 32) 486 (654) / 641 (683). bf16
// tiles are too short for it: the first two 75 (71) / 91 (83) and 175 (157) / 228 (202), the last 145 (159) / 196 (201).
void split(Attn& n, long long groups, int tiles, int slots) {
  n.splits = 1;
  n.per = tiles < 1 ? 1 : tiles;
  if (groups == 0) return;
  const bool f32 = n.a.dtype == kF32, masked = f32 && (n.a.kv_lengths || n.a.key_mask);
  if (f32) slots = 256;
  double best = 0;
  for (int s = 1; s <= kMaxSplits && (s == 1 || tiles / s >= 3); ++s) {
    const int per = (tiles + s - 1) / s;
    const double r = (double)groups * s / slots, whole = (double)((groups * s + slots - 1) / slots);
    const double cost = (masked ? r + 2 : r < 1 ? 1 : 0.5 * (r + whole)) * (per + (s == 1 ? 0 : f32 ? 1 : 6));
    if (s == 1 || cost < 0.97 * best) {
      best = cost;
      n.per = per < 1 ? 1 : per;
      n.splits = tiles > 0 ? (tiles + n.per - 1) / n.per : 1;
    }
    if (r > 8) break;
  }
}

// Workgroups that the card's 256 CUs hold at a time (bf16), from the kernels' registers and (few rows) their LDS.
int slots_rows(const splat_attention& a, int qw) {
  return 256 * (qw < 4 ? (a.D <= 64 ? 2 : 1) : a.D <= 64 ? 3 : 2);
}
int slots_keys(const splat_attention& a) { return 256 * (a.D <= 64 ? 2 : 1); }

Attn base(const splat_attention& a) {
  Attn n{};
  n.a = a;
  n.rep = a.H / a.Hk;
  n.by_rep = fast_div(n.rep);
  n.R = (int)(a.Lq * n.rep);
  n.chunked = a.D % (a.dtype == kF32 ? 4 : 8) == 0;
  for (const long long s : {a.ql, a.qh, a.kl, a.vl, a.gl, a.gh}) n.chunked = n.chunked && s >= 0 && s < (1 << 22);
  return n;
}

// qw: waves along the rows, as few as the rows need (the others share the keys).
Attn plan_fwd(const splat_attention& a, int* qw) {
  Attn n = base(a);
  *qw = n.R <= 32 ? 1 : n.R <= 64 ? 2 : 4;
  n.tiles = div_up(n.R, 32 * *qw);
  const int kt = 32 * (kWaves / *qw) * (a.dtype == kBf16 && *qw > 1 ? 2 : 1);
  split(n, (long long)n.tiles * a.B * a.Hk, div_up(a.Lk, kt), slots_rows(a, *qw));
  return n;
}

Attn plan_kv(const splat_attention& a) {
  Attn n = base(a);
  n.tiles = div_up(a.Lk, 128);
  split(n, (long long)n.tiles * a.B * a.Hk, div_up(n.R, a.dtype == kBf16 ? 64 : 32), slots_keys(a));
  return n;
}

Attn plan_q(const splat_attention& a) {
  Attn n = base(a);
  n.tiles = div_up(n.R, 128);
  split(n, (long long)n.tiles * a.B * a.Hk, div_up(a.Lk, a.dtype == kBf16 ? 64 : 32), slots_rows(a, 4));
  return n;
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// A split forward's workspace: two statistics of every split and row, then the partial rows.
size_t stat_bytes(const Attn& n) { return up(2 * sizeof(float) * (size_t)n.splits * n.a.B * n.a.Hk * n.R); }

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

size_t splat_attention_workspace_bytes(const splat_attention* a) {
  if (check_attn("splat_attention_workspace_bytes", a) || a->B == 0 || a->Lq == 0) return 0;
  int qw;
  const Attn n = plan_fwd(*a, &qw);
  return n.splits == 1 ? 0 : stat_bytes(n) + sizeof(float) * (size_t)n.splits * a->B * a->Hk * n.R * a->D;
}

int splat_attention_fwd(const splat_attention* a, const void* q, const void* k, const void* v, void* o, float* lse,
                        void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_attn("splat_attention_fwd", a)) return rc;
  if (a->B == 0 || a->Lq == 0) return kOk;
  if (!q || !o || (a->Lk > 0 && (!k || !v))) return set_error(kInvalid, "splat_attention_fwd: null pointer");
  int qw;
  const Attn n = plan_fwd(*a, &qw);
  const size_t need = splat_attention_workspace_bytes(a);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_attention_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  const long long rows = (long long)a->B * a->Hk * n.R;
  float* stat = need ? (float*)ws : nullptr;
  float* part = need ? (float*)((char*)ws + stat_bytes(n)) : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  return with_shape(*a, [&](auto t, auto dp, auto some) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool Part = decltype(some)::value;
    const int grid = n.tiles * n.splits * a->B * a->Hk;
    auto go = [&](auto w) {
      k_attn_fwd<T, DP, Part, decltype(w)::value><<<grid, kThreads, 0, st>>>(n, (const T*)q, (const T*)k, (const T*)v, (T*)o, lse,
                                                                       part, stat);
    };
    if (qw == 1) go(std::integral_constant<int, 1>{});
    else if (qw == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
    const int quads = (a->D + 3) / 4;
    if (need && n.splits <= 8 && rows * quads < 0x7fffff00LL)
      k_attn_join_few<T><<<div_up(rows * quads, kThreads), kThreads, 0, st>>>(n, fast_div(quads), quads, part, stat, (T*)o,
                                                                             lse);
    else if (need)
      k_attn_join<T, DP><<<(unsigned)rows, kJoinThreads, 0, st>>>(n, part, stat, (T*)o, lse);
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
  return with_shape(*a, [&](auto t, auto dp, auto some) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool Part = decltype(some)::value;
    const T *tq = (const T*)q, *tk = (const T*)k, *tv = (const T*)v, *tg = (const T*)g;
    if (rows) k_attn_delta<T><<<div_up(rows, kThreads / 8), kThreads, 0, st>>>(nk, (const T*)o, tg, delta);
    // rows that are split fill the card a few times at most: their values' quads are 32-bit
    const int quads = (a->D + 3) / 4;
    auto wgs = [&](long long r) { return (unsigned)div_up(r * quads, kThreads); };
    if (a->Lk > 0) {
      const long long keys = (long long)a->B * a->Lk * a->Hk;
      float* pk = nk.splits > 1 ? part : nullptr;
      const bool fine = sizeof(T) == 2 && (nk.R <= kFineRows || a->Lk <= kFineRows);
      (fine ? k_attn_bwd_kv<T, DP, Part && sizeof(T) == 4, sizeof(T) == 2> : k_attn_bwd_kv<T, DP, Part, false>)
          <<<nk.tiles * nk.splits * a->B * a->Hk, kThreads, 0, st>>>(nk, tq, tk, tv, tg, lse, delta, (T*)dk, (T*)dv, pk);
      if (pk)
        k_attn_add<T><<<dim3(wgs(keys), 2), kThreads, 0, st>>>(nk, fast_div(quads), quads, pk, nk.splits, 2 * keys * a->D,
                                                               (int)keys, false, (T*)dk, (T*)dv);
    }
    if (a->Lq > 0) {
      float* pq = nq.splits > 1 ? part : nullptr;
      const bool fine = sizeof(T) == 2 && (a->D <= kFineHead || nq.R <= kFineRows || a->Lk <= kFineRows);
      (fine ? k_attn_bwd_q<T, DP, Part && (sizeof(T) == 4 || DP <= 64), sizeof(T) == 2>
            : k_attn_bwd_q<T, DP, Part, false>)
          <<<nq.tiles * nq.splits * a->B * a->Hk, kThreads, 0, st>>>(nq, tq, tk, tv, tg, lse, delta, (T*)dq, pq);
      if (pq)
        k_attn_add<T><<<wgs(rows), kThreads, 0, st>>>(nq, fast_div(quads), quads, pq, nq.splits, rows * a->D, (int)rows, true,
                                                      (T*)dq, (T*)nullptr);
    }
    return check_launch("splat_attention_bwd");
  });
}

}  // extern "C"
