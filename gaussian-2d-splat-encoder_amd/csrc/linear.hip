// Products with an epilogue: y = act(x W^T + b) + r for rows x[M, K] and a weight W[N, K], and the gradients
// g = dy act'(z), dx = g W, dW = g^T x, db = sum over rows of g.
//
// All three products are one kernel: out[q][p] = sum_k A(p, k) B(q, k) on 32 x 32 matrix-instruction tiles, p along the
// output's rows (so that a lane's results are runs of them), either operand stored along k or across it. Sums are 32-bit
// floats. A long contraction with few outputs (dW) is cut into slices whose partial sums a second launch adds in order.
//
// Measured at 36,864 rows, bf16 (a large library product reaches 1,394 TFLOP/s here, a large copy 4.9 TB/s): 256 -> 1,024
// 42 us (460 TFLOP/s, 2.2 TB/s), 57 us with gelu and its input kept; its dx 36 us (535), dW 40 us (480) and 10.5 us to join
// 32 slices. 1,024 -> 1,024: 105 us (735). float, 1,024 -> 1,024: 594 us (130 of 153). Operands reach the matrix units
// through one LDS buffer and registers: three workgroups a CU hide the barriers better than two buffers with two workgroups
// (117 us instead of 105) or smaller tiles (124 us).
#include "feat_common.h"

namespace splat {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr long long kMaxThreads = 1LL << 32;   // a launch holds fewer
constexpr int kBytesK = 128;   // bytes of contraction indices staged at a time

// The activation's input, kept for its backward: float, or for bf16 a half of the same size. Its rounding (to the nearest,
// 2^-11 of the value at most, one instruction for two values) moves act' by an eighth of what bf16's would, which cost
// tanh's gradients half as much again as their own roundings. Cutting bits off, which takes as long, moved every slope one
// way: 3e-4 in the mean of tanh's over inputs from 0.5 to 1.
template <int A>
__device__ __forceinline__ float keep(float z) {   // a positive value stays positive, which relu's slope needs
  return A == kActRelu && z > 0.f ? fmaxf(z, 5.9604645e-8f) : z;
}
template <int A>
__device__ __forceinline__ void keep(const float (&z)[4], Chunk<float>& c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c.v[e] = z[e];
}
template <int A>
__device__ __forceinline__ void keep(const float (&z)[8], Chunk<bf16>& c) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x2 two = {keep<A>(z[e]), keep<A>(z[e + 1])};
    const auto h = __builtin_convertvector(two, f16x2);
    __builtin_memcpy(c.v + e, &h, 4);
  }
}
__device__ __forceinline__ float kept(float z) { return z; }
__device__ __forceinline__ float kept(bf16 z) { return (float)__builtin_bit_cast(_Float16, z); }
// act' at a kept input, infinite where a half could not hold it: the factor that gelu' and silu' multiply with stays finite
// (both are constant long before; a NaN passes through their other terms).
template <int A>
__device__ __forceinline__ float slope(float z) {
  return act_grad<A>(z, __builtin_amdgcn_fmed3f(z, -65504.f, 65504.f));
}

struct Gemm {
  const void *A, *B;       // A(p, k), B(q, k)
  long long lda, ldb;      // elements from row to row of the stored matrices
  int P, Q;
  long long K, kper;       // contraction; a slice's share of it
  long long rest;          // where B is the sum of two matrices (Two): elements from the first to the second, otherwise 0
  int tp, tq;              // tiles along p and q
  // epilogues
  const void *bias, *res;
  long long ldr;
  void *out, *z;
  float *part, *bpart;     // partial sums of the slices [slice][Q][P], and sum over k of B [slice][Q]
};

enum Epilogue { kOut, kForward, kPartial };

// One operand's tile: R operand rows by KE contraction indices, global -> registers -> LDS. Stored along k it is R rows of
// KE in LDS, across it KE rows of R. Padding keeps the reads on different banks (of 64 words): 16 bytes where 16 rows are read
// at the same column; across k, where a read takes 4 rows of 16 words (bf16), rows lie 16 words apart or as much before
// the next multiple of 64, and where it takes rows k and k + 4 of 32 words (float), four rows lie 32 apart.
// A thread's chunks keep their places from tile to tile. Operand rows past the matrix are read from its last row (their
// results are not stored); contraction indices past the end have to be zeros.
template <typename T, int R, bool Col>
struct Stage {
  static constexpr int V = kV<T>, KE = kBytesK / (int)sizeof(T);
  static constexpr int rows = Col ? KE : R, cols = Col ? R : KE;
  static constexpr int ld = !Col ? cols + V : sizeof(T) == 4 ? cols + 8 : cols % 64 == 0 ? cols + 32 : cols;
  static constexpr int cc = cols / V;                                // chunks of an LDS row
  static constexpr int RS = kThreads / cc, per = rows / RS;          // rows from chunk to chunk of a thread
  static_assert(kThreads % cc == 0 && rows % RS == 0, "every thread stages the same number of chunks");
  Chunk<T> c[per];
  const T* p[per];   // the chunks of the next tile
  long long step;    // elements from tile to tile
  int in;            // Col: operand rows that the thread's chunk holds

  __device__ static int row0() { return threadIdx.x / cc; }
  __device__ static int col() { return threadIdx.x % cc * V; }
  __device__ void init(const T* m, long long ldm, int r0, int R_all, long long k0) {
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int row = row0() + i * RS;
      p[i] = Col ? m + (k0 + row) * ldm + r0 + col() : m + (long long)min(r0 + row, R_all - 1) * ldm + k0 + col();
    }
    step = Col ? KE * ldm : KE;
    in = R_all - r0 - col();
  }
  // left: contraction indices from the tile's first one to the end.
  __device__ __forceinline__ void load(long long left) {
    if (left >= KE && (!Col || in >= V)) {
#pragma unroll
      for (int i = 0; i < per; ++i) __builtin_memcpy(c[i].v, p[i], 16);
    } else {
#pragma unroll
      for (int i = 0; i < per; ++i) {
        if constexpr (Col) c[i] = load_chunk(p[i], row0() + i * RS < left ? in : 0);
        else c[i] = load_chunk(p[i], left - col());
      }
    }
#pragma unroll
    for (int i = 0; i < per; ++i) p[i] += step;
  }
  __device__ void put(T* t) const {
#pragma unroll
    for (int i = 0; i < per; ++i) *(f32x4*)(t + (row0() + i * RS) * ld + col()) = *(const f32x4*)c[i].v;
  }
  // Operand chunk of the 32 rows from r at the contraction index k.
  __device__ static Chunk<T> frag(const T* t, int r, int k, int lane) {
    if constexpr (Col) return col_frag<false>(t + k * ld + r, ld, lane);
    else return row_frag(t + r * ld + k, ld, lane);
  }
};

// A workgroup's WP x WQ waves take PB x QB blocks of 32 x 32 each. The epilogue passes the results through LDS, 32 WQ rows
// of the output at a time, so that every load and store of it is a run of whole rows (stored straight from the matrix
// instructions' layout, 32 bytes a row at a time, the writes were 1.5 times the output).
template <typename T, int PB, int QB, int WP, int WQ, bool ACol, bool BCol, int Epi, int A, bool Two>
__global__ __launch_bounds__(kThreads) void k_gemm(Gemm g) {
  static_assert(WP * WQ * 64 == kThreads, "four waves");
  constexpr int V = kV<T>;
  constexpr int TP = PB * WP * 32, TQ = QB * WQ * 32;
  using SA = Stage<T, TP, ACol>;
  using SB = Stage<T, TQ, BCol>;
  constexpr int na = SA::rows * SA::ld, nb = SB::rows * SB::ld, ldo = TP + 4;
  constexpr int bytes = (na + nb) * (int)sizeof(T) > WQ * 32 * ldo * 4 ? (na + nb) * (int)sizeof(T) : WQ * 32 * ldo * 4;
  __shared__ __align__(16) char lds[bytes];
  T* ta = (T*)lds;
  T* tb = ta + na;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  // neighbouring workgroups of an XCD share rows of B
  const int tile = xcd_swizzle(blockIdx.x, gridDim.x);
  const int p0 = tile % g.tp * TP, q0 = tile / g.tp * TQ;
  const int wp = wave % WP * PB * 32, wq = wave / WP * 32;   // block j of a wave: rows q0 + 32 WQ j + wq ..
  const long long k0 = (long long)blockIdx.y * g.kper, k1 = min(g.K, k0 + g.kper);
  f32x16 acc[PB][QB] = {};
  f32x16 bsum[QB] = {};
  Chunk<T> one;
#pragma unroll
  for (int j = 0; j < V; ++j) one.v[j] = (T)1.f;
  const bool sums = Epi == kPartial && g.bpart && p0 == 0 && wp == 0;
  const T* B = (const T*)g.B;
  for (int left = Two ? 2 : 1; left > 0; --left, B += g.rest) {
    SA sa;
    SB sb;
    sa.init((const T*)g.A, g.lda, p0, g.P, k0);
    sb.init(B, g.ldb, q0, g.Q, k0);
    sa.load(k1 - k0);
    sb.load(k1 - k0);
    for (long long k = k0; k < k1; k += SA::KE) {
      __syncthreads();
      sa.put(ta);
      sb.put(tb);
      __syncthreads();
      if (k + SA::KE < k1) {
        sa.load(k1 - k - SA::KE);
        sb.load(k1 - k - SA::KE);
      }
#pragma unroll
      for (int s = 0; s < SA::KE; s += 2 * V) {
        Chunk<T> a[PB], b[QB];
#pragma unroll
        for (int i = 0; i < PB; ++i) a[i] = SA::frag(ta, wp + 32 * i, s, lane);
#pragma unroll
        for (int i = 0; i < QB; ++i) b[i] = SB::frag(tb, 32 * WQ * i + wq, s, lane);
#pragma unroll
        for (int i = 0; i < PB; ++i)
#pragma unroll
          for (int j = 0; j < QB; ++j) mma(acc[i][j], a[i], b[j]);
        if (sums) {
#pragma unroll
          for (int j = 0; j < QB; ++j) mma(bsum[j], one, b[j]);
        }
      }
    }
  }
  float* to = (float*)lds;
  constexpr int VO = Epi == kPartial ? 4 : V, cc = TP / VO;   // values a thread writes at a time
  const int p = p0 + threadIdx.x % cc * VO, n = g.P - p;
  Chunk<T> bias{};
  if (Epi == kForward && g.bias) bias = load_chunk((const T*)g.bias + p, n);
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    const int qj = q0 + 32 * WQ * j;
    if (sums && h == 0 && qj + wq + lane < g.Q) g.bpart[(long long)blockIdx.y * g.Q + qj + wq + lane] = bsum[j][0];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PB; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 run = {acc[i][j][4 * t], acc[i][j][4 * t + 1], acc[i][j][4 * t + 2], acc[i][j][4 * t + 3]};
        *(f32x4*)(to + (wq + (lane & 31)) * ldo + wp + 32 * i + acc_row(4 * t, h)) = run;
      }
    __syncthreads();
    if (n <= 0) continue;
#pragma unroll
    for (int r = threadIdx.x / cc; r < 32 * WQ; r += kThreads / cc) {
      const int q = qj + r;
      if (q >= g.Q) break;
      float x[VO];
#pragma unroll
      for (int e = 0; e < VO; e += 4) {
        const f32x4 run = *(const f32x4*)(to + r * ldo + (p - p0) + e);
#pragma unroll
        for (int f = 0; f < 4; ++f) x[e + f] = run[f];
      }
      if constexpr (Epi == kPartial) {
        Chunk<float> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = x[e];
        store_chunk(g.part + ((long long)blockIdx.y * g.Q + q) * g.P + p, o, n);
      } else {
        Chunk<T> o;
        if constexpr (Epi == kForward) {
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] += (float)bias.v[e];
          if (g.z) {
            keep<A>(x, o);
            store_chunk((T*)g.z + (long long)q * g.P + p, o, n);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] = act_fwd<A>(x[e]);
          if (g.res) {
            const Chunk<T> rs = load_chunk((const T*)g.res + q * g.ldr + p, n);
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] += (float)rs.v[e];
          }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = (T)x[e];
        store_chunk((T*)g.out + (long long)q * g.P + p, o, n);
      }
    }
  }
}

// The forward where outputs are few (tokens, small maps): bound by reading the weight, and for a small one by the chain of
// its loads. A workgroup makes 32 outputs of 32 rows; its eight waves share the contraction and load their operands straight
// from memory in the matrix instructions' layout, four steps in flight, and their sums meet in LDS once. Every 32 rows read
// the weight and every 32 outputs the rows again, so it pays up to `few_tiles` workgroups, whatever the contraction. Kernel
// times with k_gemm's staged tiles in brackets, K = 64 / 256 / 1,024 / 4,096: bf16, 256 workgroups (512 x 512 outputs) 3.3
// (3.4) / 3.9 (4.5) / 6.7 (9.8) / 17 (38) us, 512 3.7 (3.5) / 5.0 (4.7) / 10.8 (12.2) / 31 (39), 1,024 5.1 (3.7) / 8.1 (4.9)
// / 17 (12.5) / 59 (39); float, 512 4.8 (4.9) / 7.7 (9.2) / 20 (27) / 65 (98), 1,024 7.5 (5.3) / 14.8 (9.9) / 37 (28) / 123
// (98). One row of 256 -> 1,024, bf16: 3.4 (7.8).
constexpr int kFewThreads = 512;
template <typename T> constexpr long long few_tiles = sizeof(T) == 4 ? 512 : 256;
template <typename T, int A>
__global__ __launch_bounds__(kFewThreads) void k_few_rows(Gemm g) {
  constexpr int V = kV<T>, S = 2 * V, U = 4, W = kFewThreads / 64;
  __shared__ __align__(16) float sums[W][32][36];   // [wave][row][output]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int p0 = blockIdx.x * 32, q0 = blockIdx.y * 32, nq = min(32, g.Q - q0);
  // lanes past the last output or row read the last one's values; what they make is not stored
  const T* a = (const T*)g.A + (long long)min(p0 + (lane & 31), g.P - 1) * g.lda;
  const T* b = (const T*)g.B + (long long)min(q0 + (lane & 31), g.Q - 1) * g.ldb;
  const int steps = (int)((g.K + S - 1) / S), whole = (int)(g.K / S);
  f32x16 acc = {};
  for (int s0 = wave * U; s0 < steps; s0 += W * U) {
    Chunk<T> ca[U], cb[U];
    if (s0 + U <= whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        __builtin_memcpy(ca[u].v, a + (s0 + u) * S + h * V, 16);
        __builtin_memcpy(cb[u].v, b + (s0 + u) * S + h * V, 16);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long k = (long long)(s0 + u) * S + h * V;
        ca[u] = load_chunk(a + k, g.K - k);
        cb[u] = load_chunk(b + k, g.K - k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) mma(acc, ca[u], cb[u]);
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const f32x4 run = {acc[4 * t], acc[4 * t + 1], acc[4 * t + 2], acc[4 * t + 3]};
    *(f32x4*)&sums[wave][lane & 31][acc_row(4 * t, h)] = run;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nq * 32; e += kFewThreads) {
    const int c = e & 31, p = p0 + c, q = q0 + (e >> 5);
    if (p >= g.P) continue;
    float x = sums[0][e >> 5][c];
#pragma unroll
    for (int w = 1; w < W; ++w) x += sums[w][e >> 5][c];
    if (g.bias) x += (float)((const T*)g.bias)[p];
    if (g.z) {
      float z[V] = {x};
      Chunk<T> c;
      keep<A>(z, c);
      ((T*)g.z)[(long long)q * g.P + p] = c.v[0];
    }
    x = act_fwd<A>(x);
    if (g.res) x += (float)((const T*)g.res)[q * g.ldr + p];
    ((T*)g.out)[(long long)q * g.P + p] = (T)x;
  }
}

// out[i] = sum over the slices, in their order, of part[slice][i]; in the workgroups from `wgs` on the same for the bias,
// 32 columns each, 8 groups of threads over its slices.
template <typename T>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, int slices, long long n, T* __restrict__ out,
                                              unsigned wgs, const float* __restrict__ bpart, int bslices, int nb,
                                              T* __restrict__ bout) {
  __shared__ float red[8][32];
  if (blockIdx.x < wgs) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 s = {};
#pragma unroll 8
    for (int k = 0; k < slices; ++k) {
      const Chunk<float> c = load_chunk(part + k * n + i, n - i);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += c.v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) out[i + j] = (T)s[j];
    return;
  }
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, c = (blockIdx.x - wgs) * 32 + lane;
  float s = 0.f;
  if (c < nb) {
#pragma unroll 8
    for (int k = grp; k < bslices; k += 8) s += bpart[(long long)k * nb + c];
  }
  red[grp][lane] = s;
  __syncthreads();
  if (grp == 0 && c < nb) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][lane];
    bout[c] = (T)s;
  }
}

// g = dy act'(z) (z as it was kept) over `per` rows a workgroup, 64 chunks of columns wide, the rows' sums of g before its
// rounding, and (Two) `rest` elements behind g what the rounding leaves. Bound by memory: 36,864 x 1,024 bf16 with gelu 44 us
// (5.1 TB/s).
template <typename T, int A, bool Two>
__global__ __launch_bounds__(256) void k_act_grad(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ g,
                                                  long long rest, long long M, int N, int per,
                                                  float* __restrict__ bpart) {
  constexpr int V = kV<T>;
  __shared__ float red[4][64 * V];
  const int col = (blockIdx.x * 64 + (threadIdx.x & 63)) * V;
  const long long r0 = (long long)blockIdx.y * per, r1 = min(M, r0 + per);
  const long long r = r0 + (threadIdx.x >> 6);
  const int rows = col < N && r < r1 ? (int)((r1 - r + 3) / 4) : 0;
  float s[V] = {};
  RowStream<T, 4, true> in;
  in.begin(dy + r * N + col, 4LL * N, z + r * N + col, 4LL * N, rows, min(V, N - col));
  in.run([&](const Chunk<T>& d, const Chunk<T>& c, int i) {
    Chunk<T> o, left;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float x = (float)d.v[j] * slope<A>(kept(c.v[j]));
      s[j] += x;
      o.v[j] = (T)x;
      if (Two) left.v[j] = (T)(x - (float)o.v[j]);
    }
    T* p = g + (r + 4LL * i) * N + col;
    store_chunk(p, o, N - col);
    if (Two) store_chunk(p + rest, left, N - col);
  });
  if (!bpart) return;
#pragma unroll
  for (int j = 0; j < V; ++j) red[threadIdx.x >> 6][(threadIdx.x & 63) * V + j] = s[j];
  __syncthreads();
  for (int c = threadIdx.x; c < 64 * V; c += 256) {
    const int n = blockIdx.x * 64 * V + c;
    if (n < N) bpart[(long long)blockIdx.y * N + n] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
  }
}

template <typename T, int PB, int QB, int WP, int WQ, bool ACol, bool BCol, int Epi, int A, bool Two>
int launch(Gemm g, int slices, hipStream_t st) {
  g.tp = div_up(g.P, PB * WP * 32);
  g.tq = div_up(g.Q, QB * WQ * 32);
  if ((long long)g.tp * g.tq >= kMaxThreads / kThreads)
    return set_error(kUnsupported, "product of %d x %d outputs", g.Q, g.P);
  k_gemm<T, PB, QB, WP, WQ, ACol, BCol, Epi, A, Two><<<dim3(g.tp * g.tq, slices), kThreads, 0, st>>>(g);
  return kOk;
}

// Tiles of 128 x 128 where they fill the card, otherwise the smaller ones whose workgroups are more; 32 along an
// output dimension that is no longer.
template <typename T, bool ACol, bool BCol, int Epi, int A, bool Two = false>
int gemm(const Gemm& g, int slices, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && Epi != kForward && !Two) {
    if (g.rest) return gemm<T, ACol, BCol, Epi, A, true>(g, slices, st);
  }
  const long long big = (long long)div_up(g.P, 128) * div_up(g.Q, 128) * slices;
  if (g.P <= 32) return launch<T, 1, 1, 1, 4, ACol, BCol, Epi, A, Two>(g, slices, st);
  if (Epi != kForward && g.Q <= 32) return launch<T, 1, 1, 4, 1, ACol, BCol, Epi, A, Two>(g, slices, st);
  if (big >= 256) return launch<T, 2, 2, 2, 2, ACol, BCol, Epi, A, Two>(g, slices, st);
  return launch<T, 1, 1, 2, 2, ACol, BCol, Epi, A, Two>(g, slices, st);
}

// Slices of the contraction over M rows for a weight gradient [N, K]: about 512 workgroups, of at least 256 rows each.
int weight_slices(long long M, int N, int K) {
  const int t = N >= 128 && K >= 128 ? 128 : 64;
  const long long tiles = (long long)div_up(N, t) * div_up(K, t);
  const long long want = (512 + tiles - 1) / tiles;
  const long long room = (M + 255) / 256;
  const long long s = want < room ? want : room;
  return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

// Rows of a workgroup of k_act_grad: about 1024 workgroups, of at least 16 rows each.
int grad_rows(int dtype, long long M, int N) {
  const long long wide = div_up(N, 64 * (dtype == kF32 ? 4 : 8)), want = (1024 + wide - 1) / wide;
  const long long per = (M + want - 1) / want;
  return (int)(per < 16 ? 16 : per);
}

// Whether g goes into its products as the sum of two bf16 matrices. Rounded to one, results of many terms are 2.35e-3 off
// where their own rounding is 1.66e-3; few terms or few results do not average that (76 x 17 -> 9 with a sigmoid: 2.7e-3).
// Where g is small the second matrix does not show behind the call's launches, nor where the weight is (forward and backward
// of 36,864 x 64 -> 64 131 and 132 us, of 128 x 1,024 -> 1,024 131 and 132).
bool two_grads(int dtype, long long M, int N, int K, int act) {
  return dtype == kBf16 && act != kActNone && (M * N <= 1 << 17 || (long long)N * K <= 1 << 12);
}

size_t grad_bytes(int dtype, long long M, int N) { return ((size_t)M * N * (dtype == kF32 ? 4 : 2) + 255) & ~(size_t)255; }

int check_linear(const char* what, int dtype, long long M, int N, int K, int act) {
  if (dtype != kF32 && dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", what, dtype);
  if (M < 0 || N < 1 || K < 1) return set_error(kInvalid, "%s: M %lld, N %d, K %d", what, M, N, K);
  if (act < 0 || act >= kActCount) return set_error(kInvalid, "%s: unknown activation %d", what, act);
  if (M > 0x7fffff00LL || N > 0x7fffff00 || K > 0x7fffff00)
    return set_error(kUnsupported, "%s: M %lld, N %d, K %d", what, M, N, K);
  return kOk;
}

template <typename F>
int with_type(int dtype, F&& f) {
  return dtype == kF32 ? f(float{}) : f(bf16{});
}

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

int splat_linear_fwd(const void* x, long long ldx, const void* weight, const void* bias, const void* residual,
                     long long ldr, int dtype, long long M, int N, int K, int act, void* y, void* z, void* stream) {
  if (const int rc = check_linear("splat_linear_fwd", dtype, M, N, K, act)) return rc;
  if (M == 0) return kOk;
  if (!x || !weight || !y) return set_error(kInvalid, "splat_linear_fwd: null pointer");
  Gemm g{};
  g.A = weight; g.lda = K; g.P = N;
  g.B = x; g.ldb = ldx; g.Q = (int)M;
  g.K = g.kper = K;
  g.bias = bias; g.res = residual; g.ldr = ldr; g.out = y; g.z = z;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(act, [&](auto a) {
      constexpr int A = decltype(a)::value;
      if (M <= 32 || (long long)div_up(N, 32) * div_up(M, 32) <= few_tiles<T>) {
        if (div_up(N, 32) >= kMaxThreads / kFewThreads)
          return set_error(kUnsupported, "splat_linear_fwd: %d outputs of %lld rows", N, M);
        k_few_rows<T, A><<<dim3(div_up(N, 32), div_up(M, 32)), kFewThreads, 0, (hipStream_t)stream>>>(g);
        return check_launch("splat_linear_fwd");
      }
      const int rc = gemm<T, false, false, kForward, A>(g, 1, (hipStream_t)stream);
      return rc ? rc : check_launch("splat_linear_fwd");
    });
  });
}

size_t splat_linear_bwd_workspace_bytes(int dtype, long long M, int N, int K, int act) {
  if (check_linear("splat_linear_bwd_workspace_bytes", dtype, M, N, K, act) || M == 0) return 0;
  const size_t slices = weight_slices(M, N, K);
  if (act == kActNone) return sizeof(float) * slices * ((size_t)N * K + N);
  return grad_bytes(dtype, M, N) * (two_grads(dtype, M, N, K, act) ? 2 : 1) + sizeof(float) * (slices * N * K + (size_t)div_up(M, grad_rows(dtype, M, N)) * N);
}

int splat_linear_bwd(const void* x, long long ldx, const void* weight, const void* dy, const void* z, int dtype,
                     long long M, int N, int K, int act, void* dx, void* dweight, void* dbias, void* ws, size_t ws_bytes,
                     void* stream) {
  if (const int rc = check_linear("splat_linear_bwd", dtype, M, N, K, act)) return rc;
  if (M == 0) return kOk;
  if (!dy || (act != kActNone && !z) || (dx && !weight) || (dweight && !x))
    return set_error(kInvalid, "splat_linear_bwd: null pointer");
  const size_t need = splat_linear_bwd_workspace_bytes(dtype, M, N, K, act);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_linear_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  // the join of a weight gradient: four values a thread
  const long long n = dweight ? (long long)N * K : 0, wgs = (n + 1023) / 1024, bwgs = dbias ? div_up(N, 32) : 0;
  if (wgs + bwgs >= kMaxThreads / 256) return set_error(kUnsupported, "splat_linear_bwd: a weight of %d x %d", N, K);
  const hipStream_t st = (hipStream_t)stream;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int s = weight_slices(M, N, K);
    const T* gr = (const T*)dy;
    const size_t gbytes = grad_bytes(dtype, M, N);
    const long long rest = two_grads(dtype, M, N, K, act) ? gbytes / sizeof(T) : 0;
    float* part = (float*)((char*)ws + (act == kActNone ? 0 : rest ? 2 * gbytes : gbytes));
    float* bpart = dbias ? part + (size_t)s * N * K : nullptr;
    int bslices = s;
    if (act != kActNone) {
      const int per = grad_rows(dtype, M, N);
      bslices = div_up(M, per);
      with_act(act, [&](auto a) {
        if constexpr (decltype(a)::value != kActNone) {
          constexpr int A = decltype(a)::value;
          const dim3 grid(div_up(N, 64 * kV<T>), bslices);
          (rest ? k_act_grad<T, A, sizeof(T) == 2> : k_act_grad<T, A, false>)<<<grid, 256, 0, st>>>(
              (const T*)dy, (const T*)z, (T*)ws, rest, M, N, per, bpart);
        }
        return kOk;
      });
      gr = (const T*)ws;
    }
    if (dx) {
      Gemm g{};
      g.A = weight; g.lda = K; g.P = K;
      g.B = gr; g.ldb = N; g.Q = (int)M; g.rest = rest;
      g.K = g.kper = N;
      g.out = dx;
      if (const int rc = gemm<T, true, false, kOut, 0>(g, 1, st)) return rc;
    }
    if (dweight || dbias) {
      if (dweight || act == kActNone) {
        Gemm g{};
        // dbias alone: one column of products, with the gradient itself for want of x
        g.A = dweight ? x : gr; g.lda = dweight ? ldx : N; g.P = dweight ? K : 1;
        g.B = gr; g.ldb = N; g.Q = N; g.rest = rest;
        g.K = M; g.kper = (M + s - 1) / s;
        g.part = part;
        g.bpart = act == kActNone ? bpart : nullptr;
        if (const int rc = gemm<T, true, true, kPartial, 0>(g, s, st)) return rc;
      }
      k_join<T><<<(unsigned)(wgs + bwgs), 256, 0, st>>>(part, s, n, (T*)dweight, (unsigned)wgs, bpart, bslices, N, (T*)dbias);
    }
    return check_launch("splat_linear_bwd");
  });
}

}  // extern "C"
