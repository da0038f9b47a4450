// Shared pieces of the feature operators (group norm, products with an epilogue, cross attention): element types,
// activations, 16-byte chunks at any alignment, and 32 x 32 matrix-instruction tiles.
#pragma once

#include <type_traits>

#include "splat_common.h"

namespace splat {

using bf16 = __bf16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Element types and activations of the C-ABI.
enum DType : int { kF32 = 0, kBf16 = 1 };
enum Act : int { kActNone = 0, kActGelu = 1, kActSilu = 2, kActRelu = 3, kActTanh = 4, kActSigmoid = 5, kActCount = 6 };

// ------------------------------------------------------------------------------------------ activations

// Phi(x), the normal distribution's integral (gelu(x) = x Phi(x)): the logistic function of an odd polynomial of degree 13,
// fitted for the least error of x Phi(x) over |x| <= 5.6 and held there beyond; 7e-8, and 6e-7 at most evaluated in float32
// (at x = 4.99, where a unit of the result is 4.8e-7).
// About 15 instructions where erfc takes about 60: the group norm's passes were bound by them (statistics of a bf16 map of
// 37.7M values 63 us). A shorter fit (degree 5, 2.5e-5) saves four more, but parameter gradients are float32.
__device__ __forceinline__ float normal_cdf(float x) {
  const float s = fminf(x * x, 31.36f);
  float p = fmaf(-5.23388132833702e-09f, s, 3.860164383695519e-07f);
  p = fmaf(p, s, -1.146674003393855e-05f);
  p = fmaf(p, s, 0.000159485251060687f);
  p = fmaf(p, s, 9.529501403449103e-05f);
  p = fmaf(p, s, -0.10483819246292114f);
  p = fmaf(p, s, -2.3022074699401855f);
  return hw_rcp(1.f + hw_exp2(p * x));
}
// The normal distribution's density.
__device__ __forceinline__ float normal_pdf(float x) { return 0.39894228040143268f * hw_exp2(-0.5f * kLog2e * x * x); }
__device__ __forceinline__ float sigmoidf(float x) { return hw_rcp(1.f + hw_exp2(-kLog2e * x)); }

// Odd series to x^9 (fitted, 8e-8 relative) up to 0.6, beyond it 1 - 2 / (e^2|x| + 1), which loses no digits there.
__device__ __forceinline__ float tanh_of(float x) {
  const float a = fabsf(x), s = x * x;
  float p = fmaf(0.015612435527145863f, s, -0.052211690694093704f);
  p = fmaf(p, s, 0.13313114643096924f);
  p = fmaf(p, s, -0.33332598209381104f);
  p = fmaf(p * s, x, x);
  const float big = fmaf(-2.f, hw_rcp(1.f + hw_exp2(2.f * kLog2e * a)), 1.f);
  return a < 0.6f ? p : copysignf(big, x);
}

template <int A>
__device__ __forceinline__ float act_fwd(float x) {
  if constexpr (A == kActGelu) {
    return x * normal_cdf(x);
  } else if constexpr (A == kActSilu) {
    return x * sigmoidf(x);
  } else if constexpr (A == kActRelu) {
    return x > 0.f ? x : x != x ? x : 0.f;
  } else if constexpr (A == kActTanh) {
    return tanh_of(x);
  } else if constexpr (A == kActSigmoid) {
    return sigmoidf(x);
  } else {
    return x;
  }
}

// d act / dx at x; `factor` is x, or a finite value in the place of an infinite one.
template <int A>
__device__ __forceinline__ float act_grad(float x, float factor) {
  if constexpr (A == kActGelu) {
    return fmaf(factor, normal_pdf(x), normal_cdf(x));
  } else if constexpr (A == kActSilu) {
    const float s = sigmoidf(x);
    return fmaf(factor * s, 1.f - s, s);
  } else if constexpr (A == kActRelu) {
    return x > 0.f ? 1.f : 0.f;
  } else if constexpr (A == kActTanh) {
    const float t = tanh_of(x);
    return fmaf(-t, t, 1.f);
  } else if constexpr (A == kActSigmoid) {
    const float s = sigmoidf(x);
    return s * (1.f - s);
  } else {
    return 1.f;
  }
}
template <int A>
__device__ __forceinline__ float act_grad(float x) { return act_grad<A>(x, x); }

// Calls f with the activation as a compile-time constant.
template <typename F>
inline int with_act(int act, F&& f) {
  switch (act) {
    case kActNone: return f(std::integral_constant<int, kActNone>{});
    case kActGelu: return f(std::integral_constant<int, kActGelu>{});
    case kActSilu: return f(std::integral_constant<int, kActSilu>{});
    case kActRelu: return f(std::integral_constant<int, kActRelu>{});
    case kActTanh: return f(std::integral_constant<int, kActTanh>{});
    case kActSigmoid: return f(std::integral_constant<int, kActSigmoid>{});
  }
  return set_error(kInvalid, "unknown activation %d", act);
}

// Sum over a wave's 64 lanes, the same in every lane, without LDS: two exchanges within four lanes, mirrors within 8 and
// 16, swaps of rows of 16 and 32.
__device__ __forceinline__ float wave_add(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += dpp(v, std::integral_constant<int, 0xb1>{});    // lanes 1 0 3 2
  v += dpp(v, std::integral_constant<int, 0x4e>{});    // lanes 2 3 0 1
  v += dpp(v, std::integral_constant<int, 0x141>{});   // mirror within 8
  v += dpp(v, std::integral_constant<int, 0x140>{});   // mirror within 16
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// n / d for 0 <= n < 2^31 by a multiplication, d >= 1 fixed on the host.
struct FastDiv {
  unsigned mul, shift;
};
inline FastDiv fast_div(unsigned d) {
  FastDiv f{0, 0};
  while ((1ull << f.shift) < d) ++f.shift;
  f.mul = (unsigned)((((1ull << f.shift) - d) << 32) / d + 1);
  return f;
}
__device__ __forceinline__ int operator/(int n, FastDiv f) { return (int)((__umulhi(n, f.mul) + (unsigned)n) >> f.shift); }

// ---------------------------------------------------------------------------------------------- chunks
// A chunk is 16 bytes of consecutive elements, the unit of every load and store. Rows may start at any element: the
// copies carry the element's alignment, and the target's unaligned global accesses keep them one instruction.
template <typename T> constexpr int kV = 16 / (int)sizeof(T);

template <typename T>
struct Chunk {
  T v[kV<T>];
};

// The first n (clamped to 0..kV) elements at p, the others zero; nothing past them is read.
template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p, long long n) {
  Chunk<T> c;
  if (n >= kV<T>) {
    __builtin_memcpy(c.v, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) c.v[j] = j < n ? p[j] : (T)0.f;
  }
  return c;
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T>& c, long long n) {
  if (n >= kV<T>) {
    __builtin_memcpy(p, c.v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j)
      if (j < n) p[j] = c.v[j];
  }
}

// The thread's rows of one or two tensors, U at a time: begin() requests the first U, run() hands every row's chunks to
// f(chunk of a, chunk of b, row) with the next U in flight. Whole chunks load without conditions (the last U repeat the
// last row where there are fewer), so that all are issued before the first is needed; a last chunk with fewer channels goes
// row by row.
template <typename T, int U, bool Two>
struct RowStream {
  const T *a, *b;
  long long sa, sb;
  int rows, nv;   // rows; channels of the chunk
  Chunk<T> ca[U], cb[U];

  __device__ __forceinline__ void get(int i, Chunk<T> (&x)[U], Chunk<T> (&y)[U]) const {   // rows i .. i + U - 1
    if (i + U <= rows) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        __builtin_memcpy(x[u].v, a + (i + u) * sa, 16);
        if (Two) __builtin_memcpy(y[u].v, b + (i + u) * sb, 16);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        __builtin_memcpy(x[u].v, a + min(i + u, rows - 1) * sa, 16);
        if (Two) __builtin_memcpy(y[u].v, b + min(i + u, rows - 1) * sb, 16);
      }
    }
  }
  __device__ __forceinline__ void begin(const T* a_, long long sa_, const T* b_, long long sb_, int rows_, int nv_) {
    a = a_; sa = sa_; b = b_; sb = sb_; rows = rows_; nv = nv_;
    if (rows > 0 && nv == kV<T>) get(0, ca, cb);
  }
  template <typename F>
  __device__ __forceinline__ void run(F&& f) {
    if (nv == kV<T>) {
      int i = 0;
      for (; i + U < rows; i += U) {
        Chunk<T> na[U], nb[U];
        get(i + U, na, nb);
#pragma unroll
        for (int u = 0; u < U; ++u) f(ca[u], cb[u], i + u);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          ca[u] = na[u];
          if (Two) cb[u] = nb[u];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < rows) f(ca[u], cb[u], i + u);
    } else {
#pragma unroll 1
      for (int i = 0; i < rows; ++i, a += sa, b += Two ? sb : 0)
        f(load_chunk(a, nv), Two ? load_chunk(b, nv) : Chunk<T>{}, i);
    }
  }
};

// --------------------------------------------------------------------------- 32 x 32 matrix-instruction tiles
// acc(32 x 32) += A(32 x 2V) B(2V x 32), V = kV<T>: one 32x32x16 bf16 instruction, or four 32x32x2 float ones. Lane l
// gives row (A) or column (B) l % 32; with h = l / 32 its chunk holds the contraction indices h V .. h V + V - 1 of the
// 2 V, or any others, as long as A and B hold the same ones. The lane's 16 results are column l % 32 at the rows
// acc_row(r, h).
__device__ __forceinline__ void mma(f32x16& acc, const Chunk<bf16>& a, const Chunk<bf16>& b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)a.v, *(const bf16x8*)b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const Chunk<float>& a, const Chunk<float>& b) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], acc, 0, 0, 0);
}

__device__ __forceinline__ constexpr int acc_row(int r, int h) { return (r / 4) * 8 + h * 4 + r % 4; }

// Operand chunk from an LDS tile whose rows are the operand's rows (the contraction runs along a row): `t` points at
// the operand's first row and contraction index.
template <typename T>
__device__ __forceinline__ Chunk<T> row_frag(const T* t, int ld, int lane) {
  Chunk<T> c;
  *(f32x4*)c.v = *(const f32x4*)(t + (lane & 31) * ld + (lane >> 5) * kV<T>);
  return c;
}

// Operand chunk from an LDS tile whose rows are contraction indices: `t` points at the first index and the operand's
// first row (a tile column). AccOrder: the indices come in the order in which a lane holds results (acc_row), so that
// results are the other operand as they are; otherwise in row_frag's order. For float the two are the same. For bf16 a
// transposing read hands each group of 16 lanes 4 tile rows by 16 columns.
template <bool AccOrder>
__device__ __forceinline__ Chunk<bf16> col_frag(const bf16* t, int ld, int lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int h = lane >> 5, i = lane & 15;
  const bf16* p = t + (h * (AccOrder ? 4 : 8) + (i >> 2)) * ld + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
  Chunk<bf16> c;
  *(s16x4*)c.v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  *(s16x4*)(c.v + 4) = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (AccOrder ? 8 : 4) * ld));
  return c;
}
template <bool AccOrder>
__device__ __forceinline__ Chunk<float> col_frag(const float* t, int ld, int lane) {
  const float* p = t + (lane >> 5) * 4 * ld + (lane & 31);
  Chunk<float> c;
#pragma unroll
  for (int j = 0; j < 4; ++j) c.v[j] = p[j * ld];
  return c;
}

// The lane's 16 results as 16 / V runs of V consecutive rows: out[t] holds the rows run_row<T>(t, h) .. + V - 1. For
// bf16 the two half-waves exchange four values each way per run.
template <typename T>
__device__ __forceinline__ constexpr int run_row(int t, int h) { return 2 * kV<T> * t + kV<T> * h; }

template <typename T>
__device__ __forceinline__ void acc_runs(const f32x16& acc, float (&out)[16 / kV<T>][kV<T>]) {
  if constexpr (kV<T> == 4) {
#pragma unroll
    for (int r = 0; r < 16; ++r) out[r / 4][r % 4] = acc[r];
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[8 * t + j]), __float_as_uint(acc[8 * t + 4 + j]),
                                                        false, false);
        out[t][j] = __uint_as_float(s[0]);
        out[t][4 + j] = __uint_as_float(s[1]);
      }
    }
  }
}

}  // namespace splat
