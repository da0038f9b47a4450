// Norms per token with a block's gate and residual, forward and backward, on rows of C channels:
//
//   u = (h - m1) r1, z = w1 u + b1, y = x + scale act(gate) z, v = (y - m2) r2, n = w2 v + b2
//
// layer norms: m the row's mean, r = 1 / sqrt(mean((h - m)^2) + eps); root-mean-square norms: m = 0. Either norm may be left
// out, and with h the whole block: then y = x, and n is a plain norm per token. The gate has a row for all tokens, for each
// image's, or for every token. Backward, with dv = dn w2:
//
//   dy' = dy + r2 (dv - mean(dv) - v mean(dv v)), dx = dy', dz = scale act(gate) dy', dgate = scale act'(gate) dy' z,
//   du = dz w1, dh = r1 (du - mean(du) - u mean(du u)); the means of dv and du of layer norms only
//   dw2 = sum dn v, db2 = sum dn, dw1 = sum dz u, db1 = sum dz over the tokens
//
// A row is held by TPR threads, K 16-byte chunks each, in registers; it is read once, and its sums are exchanged within a wave
// (TPR <= 64) or through LDS. A workgroup takes rows a step apart with the parameters' columns in registers. The backward reads x
// and h again (y's rounding would show in the parameters' float32 gradients) with the rows' statistics kept by the forward, and
// sums columns in registers over its rows, whose partial sums a second kernel adds in order.
//
// Bound by memory: 73,728 x 256 bf16 with a gate of each image's (a large copy moves 4.9 TB/s here) forward 38 us (151 MB, 4.0
// TB/s), backward 52 (227 MB, 4.4 TB/s), the join of 512 partial sums 5, the launch and two rounds of loads. (Stores that pass the
// caches by take a tenth off the forward alone, and cost the product that reads its result as much again.)
#include <algorithm>

#include "feat_common.h"
#include "splat_tokens.h"

namespace splat {
namespace {

constexpr int kMaxChannels = 8192;   // a row's values and column sums in the registers of 1,024 threads
enum Gate : int { kNoGate = 0, kRowGate = 1, kTokenGate = 2 };   // none; a row for each segment of tokens; a row for each token

struct TokenNorm {
  splat_token_norm a;
  const void *x, *h, *gate, *dy, *dn;
  const float *w1, *b1, *w2, *b2;
  void *y, *n, *dx, *dh, *dgate;  // dgate: of a gate for every token
  float4* stat;                   // m1, r1, m2, r2 of each row
  float *cols, *gates;            // partial sums [workgroups][4][C] of dw1, db1, dw2, db2; [segments][splits][C] of the gate
  long long seg;                  // rows of a segment
  int segs, splits, whole;        // segments; workgroups of one, or whole segments of a workgroup (the other is 1)
  long long step;                 // rows that a segment's workgroups take at a time
};

// Sum over groups of TPR lanes, the same in each lane.
template <int TPR>
__device__ __forceinline__ float lanes_add(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if constexpr (TPR >= 2) v += dpp(v, std::integral_constant<int, 0xb1>{});
  if constexpr (TPR >= 4) v += dpp(v, std::integral_constant<int, 0x4e>{});
  if constexpr (TPR >= 8) v += dpp(v, std::integral_constant<int, 0x141>{});
  if constexpr (TPR >= 16) v += dpp(v, std::integral_constant<int, 0x140>{});
  if constexpr (TPR >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (TPR >= 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return v;
}

// Sums of N values over a row's threads. Rows of more than a wave exchange through LDS (all threads of the workgroup take part):
// two buffers in turn, so that one barrier a sum does.
template <int TPR, int N>
struct RowSum {
  float (*red)[2][N][16];
  int flip = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_add<TPR < 64 ? TPR : 64>(v[i]);
    if constexpr (TPR > 64) {
      const int w = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) (*red)[flip][i][w] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) s += (*red)[flip][i][w / (TPR / 64) * (TPR / 64) + k];
        v[i] = s;
      }
      flip ^= 1;
    }
  }
};

template <typename T, int TPR, int K>
struct Cols {
  static constexpr int V = kV<T>;
  int C, c[K], nv[K];   // channels; the thread's first one of each chunk, and its channels there
  __device__ __forceinline__ Cols(int n) : C(n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      c[k] = (k * TPR + (threadIdx.x & (TPR - 1))) * V;
      nv[k] = max(0, min(V, C - c[k]));
    }
  }
};

template <typename T, int K>
using Vals = float[K][kV<T>];

// A row's chunks as they lie in memory. Lanes past C load the first chunk, and where C is not whole chunks (!Whole) the lane of
// the last ones loads the row's last 16 bytes, so that no load has a condition of its own and the next row's are under way
// while this one is worked on (60,033 x 333 bf16 in training: 338 us with conditions, 250 without).
template <typename T, int K>
using Raw = Chunk<T>[K];

template <bool Whole, typename T, int TPR, int K>
__device__ __forceinline__ void load_raw(const T* p, const Cols<T, TPR, K>& at, Raw<T, K>& f) {
  constexpr int V = kV<T>;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!Whole && TPR == 4 && at.C < V) f[k] = load_chunk(p, at.nv[k]);
    else __builtin_memcpy(f[k].v, p + (at.nv[k] == V ? at.c[k] : Whole || at.nv[k] == 0 ? 0 : at.C - V), 16);
  }
}
// Their values, zeros past C (and everywhere unless `in`).
template <bool Whole, typename T, int TPR, int K>
__device__ __forceinline__ void values(const Raw<T, K>& c, const Cols<T, TPR, K>& at, Vals<T, K>& f, bool in = true) {
  constexpr int V = kV<T>;
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[k][j] = (float)c[k].v[j];
    if (!Whole) {   // the lane of the last values: they end its chunk
      float t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = f[k][j];
      const int up = TPR == 4 && at.C < V ? 0 : (V - at.C % V) % V;
#pragma unroll
      for (int s = 1; s < V; s *= 2) {
        if (up & s) {
#pragma unroll
          for (int j = 0; j + s < V; ++j) t[j] = t[j + s];
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) f[k][j] = at.nv[k] == V ? f[k][j] : j < at.nv[k] ? t[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) f[k][j] = in && (!Whole || at.nv[k]) ? f[k][j] : 0.f;
  }
}
template <typename T, int TPR, int K>
__device__ __forceinline__ void store_row(T* p, const Cols<T, TPR, K>& at, const Vals<T, K>& f) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Chunk<T> c;
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) c.v[j] = (T)f[k][j];
    store_chunk(p + at.c[k], c, at.nv[k]);
  }
}
// A row of float parameters, `none` where there are none.
template <typename T, int TPR, int K>
__device__ __forceinline__ void load_params(const float* p, const Cols<T, TPR, K>& at, float none, Vals<T, K>& f) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) f[k][j] = none;
    if (p && at.nv[k] == kV<T>) {
      __builtin_memcpy(f[k], p + at.c[k], sizeof(f[k]));
    } else if (p) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j)
        if (j < at.nv[k]) f[k][j] = p[at.c[k] + j];
    }
  }
}

__device__ __forceinline__ float gate_of(int act, float g) {
  return act == kActNone ? g : act == kActSigmoid ? sigmoidf(g) : act == kActSilu ? act_fwd<kActSilu>(g) : tanh_of(g);
}
__device__ __forceinline__ float gate_grad(int act, float g) {
  return act == kActNone      ? 1.f
         : act == kActSigmoid ? act_grad<kActSigmoid>(g)
         : act == kActSilu    ? act_grad<kActSilu>(g)
                              : act_grad<kActTanh>(g);
}

// Mean and inverse deviation of a row whose channels past C are zeros.
template <bool Lean, int TPR, int K, typename T, typename Sum>
__device__ __forceinline__ float2 row_stats(const TokenNorm& a, const Cols<T, TPR, K>& at, const Vals<T, K>& f, Sum& sum) {
  const float inv = 1.f / (float)a.a.C;
  float m = 0.f, q[1] = {0.f};
  if (!Lean && a.a.layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) s[0] += f[k][j];
    sum(s);
    m = s[0] * inv;
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) {
      const float d = j < at.nv[k] ? f[k][j] - m : 0.f;
      q[0] = fmaf(d, d, q[0]);
    }
  sum(q);
  return make_float2(m, 1.f / sqrtf(fmaf(q[0], inv, a.a.eps)));
}

template <int TPR>
constexpr int kBlock = TPR > 256 ? TPR : 256;

// f(segment's first row, segment, split) for the workgroup's segments. Its rows of each are split * RB + r, a.step apart: those
// that workgroups work on at a time lie together.
template <typename F>
__device__ __forceinline__ void segments(const TokenNorm& a, F&& f) {
  const int s0 = blockIdx.x / a.splits * a.whole, split = blockIdx.x % a.splits;
  for (int s = s0; s < min(a.segs, s0 + a.whole); ++s) f(s * a.seg, s, split);
}

// Lean: root-mean-square norms without biases, whose registers and sums it saves.
template <typename T, int TPR, int K, bool Whole, bool Lean>
__global__ __launch_bounds__(kBlock<TPR>) void k_token_norm(TokenNorm a) {
  constexpr int RB = kBlock<TPR> / TPR;
  __shared__ float red[2][1][16];
  const Cols<T, TPR, K> at(a.a.C);
  RowSum<TPR, 1> sum{&red};
  const bool block = a.h, token = a.a.gate == kTokenGate;
  Vals<T, K> w1, b1, w2, b2, gs;
  load_params(a.a.post ? a.w1 : nullptr, at, 1.f, w1);
  load_params(a.a.next ? a.w2 : nullptr, at, 1.f, w2);
  if (!Lean) {
    load_params(a.a.post ? a.b1 : nullptr, at, 0.f, b1);
    load_params(a.a.next ? a.b2 : nullptr, at, 0.f, b2);
  }
  segments(a, [&](long long row0, int seg, int split) {
    const long long rows = a.seg, r0 = split * RB;
    const int r = threadIdx.x / TPR;
    if (r0 >= rows) return;
    Raw<T, K> rx, rh, rg;
    auto fetch = [&](long long i) {
      const long long row = row0 + min(i, rows - 1);
      load_raw<Whole>((const T*)a.x + row * a.a.xl, at, rx);
      if (block) load_raw<Whole>((const T*)a.h + row * a.a.hl, at, rh);
      if (token) load_raw<Whole>((const T*)a.gate + row * a.a.gl, at, rg);
    };
    fetch(r0 + r);
    if (!token && block) {
      load_params(a.a.gate ? (const float*)a.gate + (long long)seg * a.a.C : nullptr, at, 1.f, gs);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < kV<T>; ++j) gs[k][j] = a.a.scale * (a.a.gate ? gate_of(a.a.act, gs[k][j]) : 1.f);
    }
    for (long long i = r0; i < rows; i += a.step) {
      const bool in = RB == 1 || i + r < rows;
      const long long row = row0 + i + r;
      Vals<T, K> x, h;
      values<Whole>(rx, at, x);
      if (block) values<Whole>(rh, at, h);
      if (token) {
        values<Whole>(rg, at, gs);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) gs[k][j] = a.a.scale * gate_of(a.a.act, gs[k][j]);
      }
      fetch(i + r + a.step);
      float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
      if (block) {
        if (a.a.post) {
          const float2 s = row_stats<Lean>(a, at, h, sum);
          st.x = s.x, st.y = s.y;
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < kV<T>; ++j) {
              const float u = (Lean ? h[k][j] : h[k][j] - s.x) * s.y;
              h[k][j] = Lean ? u * w1[k][j] : fmaf(u, w1[k][j], b1[k][j]);
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) x[k][j] = j < at.nv[k] ? fmaf(gs[k][j], h[k][j], x[k][j]) : 0.f;
        if (in) store_row((T*)a.y + row * a.a.C, at, x);
      }
      if (a.a.next) {
        const float2 s = row_stats<Lean>(a, at, x, sum);
        st.z = s.x, st.w = s.y;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) {
            const float v = (Lean ? x[k][j] : x[k][j] - s.x) * s.y;
            x[k][j] = Lean ? v * w2[k][j] : fmaf(v, w2[k][j], b2[k][j]);
          }
        if (in) store_row((T*)a.n + row * a.a.C, at, x);
      }
      if (a.stat && in && (threadIdx.x & (TPR - 1)) == 0) a.stat[row] = st;
    }
  });
}

// Column sums over the workgroup's row groups, in their order: out[c] for the chunks of the first group.
template <typename T, int TPR, int K>
__device__ __forceinline__ void fold_rows(Vals<T, K>& f, const Cols<T, TPR, K>& at, float* lds, float* out) {
  constexpr int RB = kBlock<TPR> / TPR, V = kV<T>;
  const int r = threadIdx.x / TPR, l = threadIdx.x & (TPR - 1);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if constexpr (RB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) lds[(r * TPR + l) * V + j] = f[k][j];
      __syncthreads();
      // columns of the chunk round k, spread over all threads
      for (int c = threadIdx.x; c < TPR * V; c += kBlock<TPR>) {
        float s = 0.f;
#pragma unroll 4
        for (int i = 0; i < RB; ++i) s += lds[i * TPR * V + c];
        const int col = k * TPR * V + c;
        if (col < at.C) out[col] = s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < at.nv[k]) out[at.c[k] + j] = f[k][j];
    }
  }
}

template <typename T, int TPR, int K, bool Whole, bool Lean>
__global__ __launch_bounds__(kBlock<TPR>) void k_token_norm_bwd(TokenNorm a) {
  constexpr int RB = kBlock<TPR> / TPR;
  __shared__ float red[2][2][16];
  __shared__ float lds[RB > 1 ? kBlock<TPR> * kV<T> : 1];
  const Cols<T, TPR, K> at(a.a.C);
  RowSum<TPR, 2> sum{&red};
  RowSum<TPR, 1> sum1{(float(*)[2][1][16])&red};
  const bool block = a.h, token = a.a.gate == kTokenGate;
  const float inv = 1.f / (float)a.a.C, mean = !Lean && a.a.layer ? inv : 0.f;
  Vals<T, K> w1, b1, w2, gs, aw1 = {}, ab1 = {}, aw2 = {}, ab2 = {}, ag = {};
  load_params(a.a.post ? a.w1 : nullptr, at, 1.f, w1);
  load_params(a.a.next ? a.w2 : nullptr, at, 1.f, w2);
  if (!Lean) load_params(a.a.post ? a.b1 : nullptr, at, 0.f, b1);
  // the row's sums of f and of f v
  auto both = [&](const Vals<T, K>& f, const Vals<T, K>& v, float& m, float& q) {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) {
        if (!Lean) s[0] += f[k][j];
        s[1] = fmaf(f[k][j], v[k][j], s[1]);
      }
    if (Lean) {
      float t[1] = {s[1]};
      sum1(t);
      m = 0.f, q = t[0] * inv;
    } else {
      sum(s);
      m = s[0] * mean, q = s[1] * inv;
    }
  };
  segments(a, [&](long long row0, int seg, int split) {
    const long long rows = a.seg, r0 = split * RB;
    const int r = threadIdx.x / TPR;
    Raw<T, K> rx, rh, rg, ry, rn;
    float4 rs;
    auto fetch = [&](long long i) {
      const long long row = row0 + min(i, rows - 1);
      load_raw<Whole>((const T*)a.x + row * a.a.xl, at, rx);
      if (block) load_raw<Whole>((const T*)a.h + row * a.a.hl, at, rh);
      if (token) load_raw<Whole>((const T*)a.gate + row * a.a.gl, at, rg);
      if (a.dy) load_raw<Whole>((const T*)a.dy + row * a.a.dyl, at, ry);
      if (a.dn) load_raw<Whole>((const T*)a.dn + row * a.a.dnl, at, rn);
      rs = a.stat[row];
    };
    if (r0 < rows) fetch(r0 + r);
    if (!token && block) {
      load_params(a.a.gate ? (const float*)a.gate + (long long)seg * a.a.C : nullptr, at, 1.f, gs);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < kV<T>; ++j) gs[k][j] = a.a.scale * (a.a.gate ? gate_of(a.a.act, gs[k][j]) : 1.f);
    }
    for (long long i = r0; i < rows; i += a.step) {
      const bool in = RB == 1 || i + r < rows;   // rows past the last one count as the last one without gradients
      const long long row = row0 + i + r;
      Vals<T, K> x, h, g, d, up;   // y, then v; u; the gate's slope; dn, then dy', then dh
      values<Whole>(rx, at, x);
      if (block) values<Whole>(rh, at, h);
      if (a.dy) values<Whole>(ry, at, up, in);
      if (a.dn) values<Whole>(rn, at, d, in);
      const float4 st = rs;
      if (token) {
        values<Whole>(rg, at, g);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) {
            gs[k][j] = a.a.scale * gate_of(a.a.act, g[k][j]);
            g[k][j] = a.a.scale * gate_grad(a.a.act, g[k][j]);
          }
      }
      fetch(i + r + a.step);
      if (block) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) {
            if (a.a.post) h[k][j] = (Lean ? h[k][j] : h[k][j] - st.x) * st.y;
            const float z = Lean ? h[k][j] * w1[k][j] : fmaf(h[k][j], w1[k][j], b1[k][j]);
            x[k][j] = fmaf(gs[k][j], z, x[k][j]);
          }
      }
      if (a.dn) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) {
            x[k][j] = (Lean ? x[k][j] : x[k][j] - st.z) * st.w;
            if (!Lean) ab2[k][j] += d[k][j];
            aw2[k][j] = fmaf(d[k][j], x[k][j], aw2[k][j]);
            d[k][j] *= w2[k][j];
          }
        float m, q;
        both(d, x, m, q);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) {
            const float t = st.w * fmaf(-x[k][j], q, Lean ? d[k][j] : d[k][j] - m);
            d[k][j] = j < at.nv[k] ? (a.dy ? up[k][j] + t : t) : 0.f;
          }
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) d[k][j] = up[k][j];
      }
      if (a.dx && in) store_row((T*)a.dx + row * a.a.C, at, d);
      if (!block) continue;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < kV<T>; ++j) {
          const float dz = gs[k][j] * d[k][j], z = Lean ? h[k][j] * w1[k][j] : fmaf(h[k][j], w1[k][j], b1[k][j]);
          if (token) g[k][j] *= d[k][j] * z;
          else ag[k][j] = fmaf(d[k][j], z, ag[k][j]);
          if (!Lean) ab1[k][j] += dz;
          aw1[k][j] = fmaf(dz, h[k][j], aw1[k][j]);
          d[k][j] = dz * w1[k][j];
        }
      if (token && a.dgate && in) store_row((T*)a.dgate + row * a.a.C, at, g);
      if (a.a.post) {
        float m, q;
        both(d, h, m, q);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < kV<T>; ++j) d[k][j] = st.y * fmaf(-h[k][j], q, Lean ? d[k][j] : d[k][j] - m);
      }
      if (a.dh && in) store_row((T*)a.dh + row * a.a.C, at, d);
    }
    if (a.gates) {
      fold_rows(ag, at, lds, a.gates + ((long long)seg * a.splits + split) * a.a.C);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < kV<T>; ++j) ag[k][j] = 0.f;
    }
  });
  if (a.cols) {
    float* out = a.cols + (long long)blockIdx.x * 4 * a.a.C;
    if (a.a.post) fold_rows(aw1, at, lds, out);
    if (a.dn) fold_rows(aw2, at, lds, out + 2 * a.a.C);
    if (!Lean) {
      if (a.a.post) fold_rows(ab1, at, lds, out + a.a.C);
      if (a.dn) fold_rows(ab2, at, lds, out + 3 * a.a.C);
    }
  }
}

// Adds the workgroups' column sums in a fixed order: 64 columns a workgroup, its waves each a part of the sums. Entries 0 to 3
// are the parameters' gradients, the others the gate's rows.
constexpr int kJoin = 1024;
__global__ __launch_bounds__(kJoin) void k_token_norm_join(TokenNorm a, int wgs, int tiles, long long units, float* dw1,
                                                           float* db1, float* dw2, float* db2, float* dgate) {
  __shared__ float part[kJoin / 64][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long e = unit / tiles, seg = e - 4;
    const int c = (int)(unit - e * tiles) * 64 + lane;
    float* out = e == 0 ? dw1 : e == 1 ? db1 : e == 2 ? dw2 : e == 3 ? db2 : dgate + seg * a.a.C;
    if (e < 4 && !out) continue;
    const long long step = e < 4 ? 4LL * a.a.C : a.a.C;
    const float* p = e < 4 ? a.cols + e * a.a.C : a.gates + seg * a.splits * a.a.C;
    const int n = e < 4 ? wgs : a.splits;
    float s = 0.f;
    if (c < a.a.C) {
#pragma unroll 4
      for (int i = w; i < n; i += kJoin / 64) s += p[i * step + c];
    }
    part[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < a.a.C) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < kJoin / 64; ++i) t += part[i][lane];
      if (e >= 4) t *= a.a.scale * gate_grad(a.a.act, ((const float*)a.gate)[seg * a.a.C + c]);
      out[c] = t;
    }
    __syncthreads();
  }
}

// At most 8 values a lane. Training passes, us, this rule's side first. Rows of 65 to 128 chunks: of floats two chunks in each
// lane of a wave, or one in each of two waves (36,864 rows of 400 channels 131 and 135, of 512 156 and 159); of bf16 one in each
// of two waves, or two a lane (24,576 x 640 109 and 135, 18,432 x 1,024 97 and 119). Up to 512 chunks of bf16 one in each of
// eight waves, or two in each of four (6,144 x 3,000 119 and 151, 4,608 x 4,096 103 and 129). Up to 192 chunks of floats one in
// each of four waves, or three a lane (5,001 x 517 48 and 62, 16,384 x 600 106 and 113, 12,288 x 768 87 and 95).
struct Shape {
  int tpr, k, rows;   // threads of a row; chunks of a thread; rows of a workgroup at a time
  bool whole, lean;
};
Shape shape_of(const splat_token_norm& a, bool biases) {
  const bool f32 = a.dtype == kF32, whole = a.C % (f32 ? 4 : 8) == 0;
  const int chunks = div_up(a.C, f32 ? 4 : 8);
  int tpr = 4;
  while (tpr < (f32 ? 64 : 512) && tpr < chunks) tpr *= 2;
  if (f32 && chunks > 128) tpr = 256;
  if (chunks > 512) tpr = 1024;
  return {tpr, div_up(chunks, tpr), std::max(1, 256 / tpr), whole, whole && !a.layer && !biases};
}

template <typename F>
int with_shape(int dtype, const Shape& s, F&& f) {
  using std::integral_constant;
  auto kind = [&](auto t, auto tpr, auto k) {
    if (s.lean) return f(t, tpr, k, std::true_type{}, std::true_type{});
    if (s.whole) return f(t, tpr, k, std::true_type{}, std::false_type{});
    return f(t, tpr, k, std::false_type{}, std::false_type{});
  };
  auto type = [&](auto t) {
    constexpr bool f32 = sizeof(t) == 4;
    auto one = [&](auto tpr) { return kind(t, tpr, integral_constant<int, 1>{}); };
    auto two = [&](auto tpr) {   // chunks of floats
      if constexpr (f32)
        if (s.k == 2) return kind(t, tpr, integral_constant<int, 2>{});
      return one(tpr);
    };
    switch (s.tpr) {
      case 4: return one(integral_constant<int, 4>{});
      case 8: return one(integral_constant<int, 8>{});
      case 16: return one(integral_constant<int, 16>{});
      case 32: return one(integral_constant<int, 32>{});
      case 64: return two(integral_constant<int, 64>{});
      case 256: return two(integral_constant<int, 256>{});
    }
    if constexpr (!f32) {
      if (s.tpr == 128) return one(integral_constant<int, 128>{});
      if (s.tpr == 512) return one(integral_constant<int, 512>{});
    }
    return two(integral_constant<int, 1024>{});
  };
  return dtype == kF32 ? type(float{}) : type(bf16{});
}

int check_norm(const char* who, const splat_token_norm* a) {
  if (!a) return set_error(kInvalid, "%s: no description", who);
  if (a->dtype != kF32 && a->dtype != kBf16) return set_error(kInvalid, "%s: unknown element type %d", who, a->dtype);
  if (a->C < 1 || a->M < 0 || a->gate < 0 || a->gate > 2 || !(a->eps >= 0.f))
    return set_error(kInvalid, "%s: C %d, M %lld, gate %d, eps %g", who, a->C, a->M, a->gate, a->eps);
  if (a->act != kActNone && a->act != kActSigmoid && a->act != kActSilu && a->act != kActTanh)
    return set_error(kInvalid, "%s: activation %d of a gate", who, a->act);
  if (a->C > kMaxChannels) return set_error(kUnsupported, "%s: %d channels, %d at most", who, a->C, kMaxChannels);
  if (a->gate == kRowGate && (a->segs < 1 || a->M % a->segs))
    return set_error(kInvalid, "%s: %lld tokens do not divide over %lld gates", who, a->M, a->segs);
  if (a->M > 0x7fffffffLL || (a->gate == kRowGate && a->segs > 0x1000000LL))
    return set_error(kUnsupported, "%s: %lld tokens, %lld gates", who, a->M, a->segs);
  return kOk;
}

// Segments and splits for about `target` workgroups. Returns their number.
unsigned plan(TokenNorm& n, const Shape& s, long long target) {
  n.segs = n.a.gate == kRowGate ? (int)n.a.segs : 1;
  n.seg = n.a.M / n.segs;
  n.whole = (int)((n.segs + target - 1) / target);
  const long long most = std::max<long long>(1, (n.seg + s.rows - 1) / s.rows);
  n.splits = (int)std::min(most, n.segs >= target ? 1 : (target + n.segs - 1) / n.segs);
  n.step = (long long)n.splits * s.rows;
  return (unsigned)((n.segs + n.whole - 1) / n.whole * n.splits);
}

// Workgroups aimed at: what the card holds at once, by the registers of a lane (four waves a SIMD; in the backward three or two
// for 4 or 8 values a lane, four of 1,024 threads, whose registers spill). Training passes for 2, 3 and 4 waves, us: bf16
// 73,728 x 256 97, 110, 101 (64 to 1,024 channels the same to 3%), 4,608 x 4,096 103, 123, 114, 2,304 x 8,192 274, 226, 209;
// floats of four values a lane 36,864 x 256 85, 82, 86, 9,216 x 1,024 87, 84, 86, 5,001 x 517 49, 47, 56; of eight 73,728 x 300
// 204, 231, 209, 4,608 x 2,048 87, 97, 96. (More waves than fit are a second round, shorter than the first.)
long long resident(const Shape& s, int dtype, bool back) {
  const int values = s.k * (dtype == kF32 ? 4 : 8), waves = !back || s.tpr == 1024 ? 4 : values == 4 ? 3 : 2;
  return 256LL * waves * 4 * 64 / std::max(256, s.tpr);
}

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

int splat_token_norm_fwd(const splat_token_norm* a, const void* x, const void* h, const void* gate, const float* w1,
                         const float* b1, const float* w2, const float* b2, void* y, void* n, float* stat, void* stream) {
  if (const int rc = check_norm("splat_token_norm_fwd", a)) return rc;
  if (a->M == 0) return kOk;
  if (!x || (h && !y) || (a->next && !n) || (!h && (a->post || a->gate || !a->next)) || (a->gate && !gate))
    return set_error(kInvalid, "splat_token_norm_fwd: null pointer");
  TokenNorm p{};
  p.a = *a;
  p.x = x, p.h = h, p.gate = gate, p.w1 = w1, p.b1 = b1, p.w2 = w2, p.b2 = b2, p.y = y, p.n = n, p.stat = (float4*)stat;
  const Shape s = shape_of(*a, b1 || b2);
  const unsigned grid = plan(p, s, resident(s, a->dtype, false));
  return with_shape(a->dtype, s, [&](auto t, auto tpr, auto k, auto whole, auto lean) {
    constexpr int TPR = decltype(tpr)::value;
    k_token_norm<decltype(t), TPR, decltype(k)::value, decltype(whole)::value, decltype(lean)::value>
        <<<grid, kBlock<TPR>, 0, (hipStream_t)stream>>>(p);
    return check_launch("splat_token_norm_fwd");
  });
}

size_t splat_token_norm_bwd_workspace_bytes(const splat_token_norm* a) {
  if (check_norm("splat_token_norm_bwd_workspace_bytes", a) || a->M == 0) return 0;
  TokenNorm p{};
  p.a = *a;
  const Shape s = shape_of(*a, false);
  const size_t grid = plan(p, s, resident(s, a->dtype, true));
  return sizeof(float) * a->C * (4 * grid + (a->gate == kRowGate ? (size_t)p.segs * p.splits : 0));
}

int splat_token_norm_bwd(const splat_token_norm* a, const void* x, const void* h, const void* gate, const float* w1,
                         const float* b1, const float* w2, const void* dy, const void* dn, const float* stat, void* dx, void* dh,
                         void* dgate, float* dw1, float* db1, float* dw2, float* db2, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_norm("splat_token_norm_bwd", a)) return rc;
  if (a->M == 0) return kOk;
  if (!x || !stat || (!dy && !dn) || (dn && !a->next) || (!h && (a->post || a->gate || !dn)) || (a->gate && !gate) ||
      ((dw1 || db1) && !a->post) || ((dw2 || db2) && !dn) || (dh && !h) || (dgate && !a->gate))
    return set_error(kInvalid, "splat_token_norm_bwd: null pointer");
  TokenNorm p{};
  p.a = *a;
  p.x = x, p.h = h, p.gate = gate, p.w1 = w1, p.b1 = b1, p.w2 = w2, p.dy = dy, p.dn = dn, p.stat = (float4*)stat;
  p.dx = dx, p.dh = dh, p.dgate = a->gate == kTokenGate ? dgate : nullptr;
  const Shape s = shape_of(*a, b1 || db1 || db2);
  const unsigned grid = plan(p, s, resident(s, a->dtype, true));
  const bool cols = dw1 || db1 || dw2 || db2, gates = dgate && a->gate == kRowGate;
  const size_t need = cols || gates ? splat_token_norm_bwd_workspace_bytes(a) : 0;
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_token_norm_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  if (cols) p.cols = (float*)ws;
  if (gates) p.gates = (float*)ws + (size_t)4 * grid * a->C;
  const hipStream_t st = (hipStream_t)stream;
  return with_shape(a->dtype, s, [&](auto t, auto tpr, auto k, auto whole, auto lean) {
    constexpr int TPR = decltype(tpr)::value;
    k_token_norm_bwd<decltype(t), TPR, decltype(k)::value, decltype(whole)::value, decltype(lean)::value>
        <<<grid, kBlock<TPR>, 0, st>>>(p);
    if (need) {
      const int tiles = div_up(a->C, 64);
      const long long units = (long long)tiles * (4 + (gates ? p.segs : 0));
      k_token_norm_join<<<(unsigned)std::min(units, 1LL << 20), kJoin, 0, st>>>(p, (int)grid, tiles, units, dw1, db1, dw2, db2,
                                                                                gates ? (float*)dgate : nullptr);
    }
    return check_launch("splat_token_norm_bwd");
  });
}

}  // extern "C"
