// Products with an epilogue: y = act(x W^T + b) + r for rows x[M, K] and a weight W[N, K], and the gradients
// g = dy act'(z), dx = g W, dW = g^T x, db = sum over rows of g.
//
// All three products are one kernel: out[q][p] = sum_k A(p, k) B(q, k) on 32 x 32 matrix-instruction tiles, p along the
// output's rows (so that a lane's results are runs of them), either operand stored along k or across it. Sums are 32-bit
// floats. A long contraction with few outputs (dW) is cut into slices whose partial sums a second launch adds in order.
#include "feat_common.h"

namespace splat {
namespace {

constexpr int kThreads = 256;
constexpr int kBytesK = 128;   // bytes of contraction indices staged at a time

struct Gemm {
  const void *A, *B;       // A(p, k), B(q, k)
  long long lda, ldb;      // elements from row to row of the stored matrices
  int P, Q;
  long long K, kper;       // contraction; a slice's share of it
  int tp, tq;              // tiles along p and q
  // epilogues
  const void *bias, *res;
  long long ldr;
  void *out, *z;
  float *part, *bpart;     // partial sums of the slices [slice][Q][P], and sum over k of B [slice][Q]
};

enum Epilogue { kOut, kForward, kPartial };

// One operand's tile in LDS: R operand rows by KE contraction indices. Stored along k as R rows of KE, across it as KE
// rows of R; 16 bytes of padding a row keep the reads of neighbouring rows on different banks.
template <typename T, int R, bool Col>
struct Stage {
  static constexpr int V = kV<T>, KE = kBytesK / (int)sizeof(T);
  static constexpr int rows = Col ? KE : R, cols = Col ? R : KE;
  static constexpr int ld = cols + V;
  static constexpr int chunks = rows * cols / V, per = chunks / kThreads;
  static_assert(chunks % kThreads == 0, "every thread stages the same number of chunks");

  // The thread's chunks of the tile at operand row r0 (of R_all) and contraction index k0 (up to k1).
  __device__ static void load(Chunk<T> (&c)[per], const T* m, long long ldm, int r0, int R_all, long long k0, long long k1) {
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int e = threadIdx.x + i * kThreads, row = e / (cols / V), col = e % (cols / V) * V;
      if constexpr (Col) {
        const long long k = k0 + row;
        c[i] = load_chunk(m + k * ldm + r0 + col, k < k1 ? (long long)R_all - r0 - col : 0);
      } else {
        c[i] = load_chunk(m + (long long)(r0 + row) * ldm + k0 + col, r0 + row < R_all ? k1 - k0 - col : 0);
      }
    }
  }
  __device__ static void put(const Chunk<T> (&c)[per], T* t) {
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int e = threadIdx.x + i * kThreads, row = e / (cols / V), col = e % (cols / V) * V;
      *(f32x4*)(t + row * ld + col) = *(const f32x4*)c[i].v;
    }
  }
  // Operand chunk of the 32 rows from r at the contraction index k.
  __device__ static Chunk<T> frag(const T* t, int r, int k, int lane) {
    if constexpr (Col) return col_frag<false>(t + k * ld + r, ld, lane);
    else return row_frag(t + r * ld + k, ld, lane);
  }
};

// A workgroup's WP x WQ waves take PB x QB blocks of 32 x 32 each.
template <typename T, int PB, int QB, int WP, int WQ, bool ACol, bool BCol, int Epi, int A>
__global__ __launch_bounds__(kThreads) void k_gemm(Gemm g) {
  static_assert(WP * WQ * 64 == kThreads, "four waves");
  constexpr int V = kV<T>;
  using SA = Stage<T, PB * WP * 32, ACol>;
  using SB = Stage<T, QB * WQ * 32, BCol>;
  __shared__ __align__(16) T ta[SA::rows * SA::ld];
  __shared__ __align__(16) T tb[SB::rows * SB::ld];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  // neighbouring workgroups of an XCD share rows of B
  const int tile = xcd_swizzle(blockIdx.x, gridDim.x);
  const int p0 = tile % g.tp * (PB * WP * 32), q0 = tile / g.tp * (QB * WQ * 32);
  const int wp = wave % WP * PB * 32, wq = wave / WP * QB * 32;
  const long long k0 = (long long)blockIdx.y * g.kper, k1 = min(g.K, k0 + g.kper);
  f32x16 acc[PB][QB] = {};
  f32x16 bsum[QB] = {};
  Chunk<T> one;
#pragma unroll
  for (int j = 0; j < V; ++j) one.v[j] = (T)1.f;
  const bool sums = Epi == kPartial && g.bpart && p0 == 0 && wp == 0;
  Chunk<T> ca[SA::per], cb[SB::per];
  SA::load(ca, (const T*)g.A, g.lda, p0, g.P, k0, k1);
  SB::load(cb, (const T*)g.B, g.ldb, q0, g.Q, k0, k1);
  for (long long k = k0; k < k1; k += SA::KE) {
    __syncthreads();
    SA::put(ca, ta);
    SB::put(cb, tb);
    __syncthreads();
    if (k + SA::KE < k1) {
      SA::load(ca, (const T*)g.A, g.lda, p0, g.P, k + SA::KE, k1);
      SB::load(cb, (const T*)g.B, g.ldb, q0, g.Q, k + SA::KE, k1);
    }
#pragma unroll
    for (int s = 0; s < SA::KE; s += 2 * V) {
      Chunk<T> a[PB], b[QB];
#pragma unroll
      for (int i = 0; i < PB; ++i) a[i] = SA::frag(ta, wp + 32 * i, s, lane);
#pragma unroll
      for (int i = 0; i < QB; ++i) b[i] = SB::frag(tb, wq + 32 * i, s, lane);
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
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    const int q = q0 + wq + 32 * j + (lane & 31);
    if (q >= g.Q) continue;
    if (sums && h == 0) g.bpart[(long long)blockIdx.y * g.Q + q] = bsum[j][0];
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      if constexpr (Epi == kPartial) {
        float run[4][4];
        acc_runs<float>(acc[i][j], run);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int p = p0 + wp + 32 * i + run_row<float>(t, h);
          Chunk<float> o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o.v[e] = run[t][e];
          store_chunk(g.part + ((long long)blockIdx.y * g.Q + q) * g.P + p, o, g.P - p);
        }
      } else {
        float run[16 / V][V];
        acc_runs<T>(acc[i][j], run);
#pragma unroll
        for (int t = 0; t < 16 / V; ++t) {
          const int p = p0 + wp + 32 * i + run_row<T>(t, h);
          const int n = g.P - p;
          if (n <= 0) continue;
          Chunk<T> o;
          if constexpr (Epi == kForward) {
            if (g.bias) {
              const Chunk<T> b = load_chunk((const T*)g.bias + p, n);
#pragma unroll
              for (int e = 0; e < V; ++e) run[t][e] += (float)b.v[e];
            }
            if (g.z) {
#pragma unroll
              for (int e = 0; e < V; ++e) o.v[e] = (T)run[t][e];
              store_chunk((T*)g.z + (long long)q * g.P + p, o, n);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) run[t][e] = act_fwd<A, T>(run[t][e]);
            if (g.res) {
              const Chunk<T> r = load_chunk((const T*)g.res + q * g.ldr + p, n);
#pragma unroll
              for (int e = 0; e < V; ++e) run[t][e] += (float)r.v[e];
            }
          }
#pragma unroll
          for (int e = 0; e < V; ++e) o.v[e] = (T)run[t][e];
          store_chunk((T*)g.out + (long long)q * g.P + p, o, n);
        }
      }
    }
  }
}

// out[i] = sum over the slices, in their order, of part[slice][i].
template <typename T>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, int slices, long long n, T* __restrict__ out,
                                              const float* __restrict__ bpart, long long nb, T* __restrict__ bout) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i < n) {
    f32x4 s = {};
    for (int k = 0; k < slices; ++k) {
      const Chunk<float> c = load_chunk(part + k * n + i, n - i);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += c.v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) out[i + j] = (T)s[j];
  } else {
    for (long long e = i - (n + 3) / 4 * 4; e < i - (n + 3) / 4 * 4 + 4; ++e) {
      if (e >= nb) return;
      float s = 0.f;
      for (int k = 0; k < slices; ++k) s += bpart[k * nb + e];
      bout[e] = (T)s;
    }
  }
}

// g = dy act'(z)
template <typename T, int A>
__global__ __launch_bounds__(256) void k_act_grad(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ g,
                                                  long long n) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * kV<T>;
  if (i >= n) return;
  const Chunk<T> d = load_chunk(dy + i, n - i), c = load_chunk(z + i, n - i);
  Chunk<T> o;
#pragma unroll
  for (int j = 0; j < kV<T>; ++j) o.v[j] = (T)((float)d.v[j] * act_grad<A, T>((float)c.v[j]));
  store_chunk(g + i, o, n - i);
}

template <typename T, int PB, int QB, int WP, int WQ, bool ACol, bool BCol, int Epi, int A>
void launch(Gemm g, int slices, hipStream_t st) {
  g.tp = div_up(g.P, PB * WP * 32);
  g.tq = div_up(g.Q, QB * WQ * 32);
  k_gemm<T, PB, QB, WP, WQ, ACol, BCol, Epi, A><<<dim3(g.tp * g.tq, slices), kThreads, 0, st>>>(g);
}

// Tiles of 128 x 128 where they fill the card, otherwise the smaller ones whose workgroups are more; 32 along an
// output dimension that is no longer.
template <typename T, bool ACol, bool BCol, int Epi, int A>
void gemm(const Gemm& g, int slices, hipStream_t st) {
  const long long big = (long long)div_up(g.P, 128) * div_up(g.Q, 128) * slices;
  if (g.P <= 32) launch<T, 1, 1, 1, 4, ACol, BCol, Epi, A>(g, slices, st);
  else if (g.Q <= 32) launch<T, 1, 1, 4, 1, ACol, BCol, Epi, A>(g, slices, st);
  else if (big >= 256) launch<T, 2, 2, 2, 2, ACol, BCol, Epi, A>(g, slices, st);
  else launch<T, 1, 1, 2, 2, ACol, BCol, Epi, A>(g, slices, st);
}

// Slices of the contraction over M rows for a weight gradient [N, K].
int weight_slices(long long M, int N, int K) {
  const long long tiles = (long long)div_up(N, 64) * div_up(K, 64);
  const long long want = 512 / tiles > 0 ? 512 / tiles : 1;
  const long long room = (M + 255) / 256;
  const long long s = want < room ? want : room;
  return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

int check_linear(const char* what, int dtype, long long M, int N, int K, int act) {
  if (dtype != kF32 && dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", what, dtype);
  if (M < 0 || N < 1 || K < 1) return set_error(kInvalid, "%s: M %lld, N %d, K %d", what, M, N, K);
  if (act < 0 || act >= kActCount) return set_error(kInvalid, "%s: unknown activation %d", what, act);
  const long long tiles = ((M + 31) / 32) * (((long long)N + 31) / 32);
  if (M > 0x7fffff00LL || N > 0x7fffff00 || K > 0x7fffff00 || tiles > 0x7fffff00LL || ((M + 31) / 32) * (((long long)K + 31) / 32) > 0x7fffff00LL)
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
      gemm<T, false, false, kForward, decltype(a)::value>(g, 1, (hipStream_t)stream);
      return check_launch("splat_linear_fwd");
    });
  });
}

size_t splat_linear_bwd_workspace_bytes(int dtype, long long M, int N, int K, int act) {
  if (check_linear("splat_linear_bwd_workspace_bytes", dtype, M, N, K, act) || M == 0) return 0;
  const int s = weight_slices(M, N, K);
  const size_t grad = act == kActNone ? 0 : ((size_t)M * N * (dtype == kF32 ? 4 : 2) + 255) & ~(size_t)255;
  return grad + sizeof(float) * (size_t)s * ((size_t)N * K + N);
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
  const hipStream_t st = (hipStream_t)stream;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const size_t grad = act == kActNone ? 0 : ((size_t)M * N * sizeof(T) + 255) & ~(size_t)255;
    const T* gr = (const T*)dy;
    if (act != kActNone) {
      with_act(act, [&](auto a) {
        const long long n = M * N;
        k_act_grad<T, decltype(a)::value><<<div_up(n, 256 * kV<T>), 256, 0, st>>>((const T*)dy, (const T*)z, (T*)ws, n);
        return kOk;
      });
      gr = (const T*)ws;
    }
    if (dx) {
      Gemm g{};
      g.A = weight; g.lda = K; g.P = K;
      g.B = gr; g.ldb = N; g.Q = (int)M;
      g.K = g.kper = N;
      g.out = dx;
      gemm<T, true, false, kOut, 0>(g, 1, st);
    }
    if (dweight || dbias) {
      const int s = weight_slices(M, N, K);
      Gemm g{};
      // dbias alone: one column of products, with the gradient itself for want of x
      g.A = dweight ? x : gr; g.lda = dweight ? ldx : N; g.P = dweight ? K : 1;
      g.B = gr; g.ldb = N; g.Q = N;
      g.K = M; g.kper = (M + s - 1) / s;
      g.part = (float*)((char*)ws + grad);
      g.bpart = dbias ? g.part + (size_t)s * N * K : nullptr;
      gemm<T, true, true, kPartial, 0>(g, s, st);
      const long long n = dweight ? (long long)N * K : 0;
      k_join<T><<<div_up((n + 3) / 4 + (dbias ? (N + 3) / 4 : 0), 256), 256, 0, st>>>(g.part, s, n, (T*)dweight, g.bpart,
                                                                                     dbias ? N : 0, (T*)dbias);
    }
    return check_launch("splat_linear_bwd");
  });
}

}  // extern "C"
