// Attention of a few new tokens over a paged cache: o = softmax(scale q k^T) v for queries q[B, T, H, D] (turned by their
// positions on the way in) over the tokens of each sequence's pages, all of them or (causal) those up to the query's own.
//
// The H / Hk heads that share keys are rows of one problem, r = token * rep + head within the group. Tokens are read once:
// time is memory's, so the work is cut along the cache, each workgroup a piece of one sequence's tokens for one key head and up
// to 32 rows. Pieces are as long for all sequences (each workgroup finds its own from the lengths on the device, so that ragged
// batches fill the card and a captured graph follows its lengths); a second kernel joins them.
//
// A wave takes tiles of its own: 32 tokens (16 of floats), keys straight from memory into matrix-instruction operands, values
// through LDS for a transposing read, the next tile in flight, places in the pages looked up three tiles ahead. Scores are held
// transposed, a lane per row, so that probabilities are the second product's operand as they leave the first. Running maxima
// and sums, accumulators and partial results are 32-bit floats. Probabilities, and queries that were turned, are taken as sums
// of two bf16 values: matrix instructions wait for memory here, and a single rounding would show next to the result's own.
//
// Tokens past the length or marked dead are not read and count as zeros; their places hold a neighbour's values, zeros for
// floats, so that an infinite value that counts stays infinite (368,640 tokens of 4 heads of 64 floats, 60% live, 102 us, 100
// without; bf16 would still multiply it by a probability's second part, of either sign or zero, and give NaN). Tokens after a
// causal query have probability zero; a tile whose values there are not finite is multiplied query by query with those values
// as zeros.
//
// Measured: one token in each of sixteen sequences of 0 to 32,768 tokens, 32 heads over 8 of 128 bf16 (1.06 GB) 188 us, 5.6
// TB/s, floats (2.1 GB) 372 with the join, 5.7; one token over 368,640, of which 60% count, 4 heads of 64 bf16 (226 MB) 48 us, 4.7
// TB/s, with a join of 190 pieces 5, of floats, all live (755 MB), 141 with the join, 5.4 TB/s; one over 900 tokens 8.1 us, six
// loads behind each other, and a join of 4. Many rows are not what this is for: 1,024 tokens of 32 heads over 8,192 take 626 us
// (205 TFLOP/s), rows of 32 a workgroup and two products for one.
#include <algorithm>

#include "token_common.h"

namespace splat {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kLeast = 128;      // tokens of a piece at least: one bf16 tile for each wave
constexpr int kRounds = 4;       // of workgroups, where sequences are many
// Workgroups that a CU holds, by the registers of their kernels (16 NR rows, heads of DP).
constexpr int held(int DP, int NR) { return NR == 1 ? DP == 32 ? 4 : DP == 64 ? 3 : 2 : DP == 32 ? 3 : DP == 64 ? 2 : 1; }

// Sequences are whole, cut by a scan in each workgroup (up to 64 of them), or as a list has it.
enum Cut : int { kWhole = 0, kScanned = 1, kMapped = 2 };

struct Cached {
  splat_cache c;
  splat_rotation r;
  splat_positions pos;
  const void* q;
  void* o;
  long long qb, ql, qh;
  float scale;                 // of the scores, times log2 e
  int T, H, rep, R;            // new tokens; query heads; of a key head; rows = T rep
  int tiles, pieces, causal;   // row tiles; pieces aimed at, over all sequences
  int units;                   // of a head, single pairs
  bool alike, fit;             // keys and values have the same strides; all pieces shall be on the card at once
  int cut;                     // how a workgroup finds its piece
  int4* map;                   // the pieces, where many sequences are cut
  FastDiv by_rep, by_page, by_units;
  float* part;                 // rows of the pieces of split sequences
  float2* stat;                // their maxima and sums
  int2* split;                 // pieces of each sequence and the first one's slot
};

template <typename T> constexpr int kTile = sizeof(T) == 2 ? 32 : 16;   // tokens of a wave's tile

// Inclusive sums over a wave's lanes, without LDS: within rows of 16, then rows' last ones added to the rows behind them.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // one lane up within 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);    // lane 15 of rows 0 and 2 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);    // lane 31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ int last_of(int v) { return __builtin_amdgcn_readlane(v, 63); }

// Pieces of a sequence of len tokens (!in: of none).
__device__ __forceinline__ int pieces_of(int len, int per, bool in) {
  return in ? len > 0 ? (len - 1) / kLeast / per + 1 : 1 : 0;
}

// The piece of a workgroup: `i` of the n of sequence b (n < 1: none), which has len tokens; `slot` is the sequence's first one
// among those of split sequences. Pieces are as long for all sequences, in units of kLeast tokens: what the aimed at number of
// them would have, and where all shall be on the card at once (`fit`) longer until their number is no more than that; a
// sequence without tokens has one.
struct Piece {
  int b, i, n, len, slot;
};
__device__ __forceinline__ Piece find(const Cached& a, int s) {
  if (a.cut == kWhole) return s < a.c.B ? Piece{s, 0, 1, cached_tokens(a.c, s), 0} : Piece{};
  if (a.cut == kMapped) {
    const int4 m = a.map[s];
    return m.z ? Piece{m.x, m.y, m.z, cached_tokens(a.c, m.x), m.w} : Piece{};
  }
  const int lane = threadIdx.x & 63;
  int len = 0;   // of the lane's sequence
  if (lane < a.c.B) len = cached_tokens(a.c, lane);
  const int units = last_of(wave_scan((len + kLeast - 1) / kLeast));   // 2^24 a sequence at most
  int per = max(1, (units + a.pieces - 1) / a.pieces);                 // units of a piece
  for (int i = 0; a.fit && i < 3; ++i) {
    const int n = last_of(wave_scan(len > 0 ? (len - 1) / kLeast / per + 1 : 0));
    if (n <= a.pieces) break;
    per = (int)(((long long)per * n + a.pieces - 1) / a.pieces);
  }
  const int n = pieces_of(len, per, lane < a.c.B), m = n > 1 ? n : 0, upto = wave_scan(n), slots = wave_scan(m);
  const unsigned long long hit = __ballot(upto > s);
  if (!hit) return Piece{};
  const int f = __builtin_ctzll(hit), nf = __builtin_amdgcn_readlane(n, f);
  return {f, s - (__builtin_amdgcn_readlane(upto, f) - nf), nf, __builtin_amdgcn_readlane(len, f),
          __builtin_amdgcn_readlane(slots, f) - __builtin_amdgcn_readlane(m, f)};
}

// The same for more than 64 sequences, whose scan each workgroup would repeat: one workgroup writes all pieces into a.map
// (sequence, piece, pieces of the sequence, its first slot), and zeros behind them.
constexpr int kPlan = 1024;
__global__ __launch_bounds__(kPlan) void k_cached_plan(Cached a) {
  __shared__ long long part[kPlan / 64];
  __shared__ int sums[2][kPlan / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  long long units = 0;
  for (int b0 = 0; b0 < a.c.B; b0 += kPlan) {
    const int b = b0 + threadIdx.x, len = b < a.c.B ? cached_tokens(a.c, b) : 0;
    units += last_of(wave_scan((len + kLeast - 1) / kLeast));   // of the wave's 64
  }
  if (lane == 0) part[w] = units;
  __syncthreads();
  units = 0;
#pragma unroll
  for (int i = 0; i < kPlan / 64; ++i) units += part[i];
  const int per = max(1, (int)min((units + a.pieces - 1) / a.pieces, 0xffffffLL));
  int first = 0, slot = 0;
  for (int b0 = 0; b0 < a.c.B; b0 += kPlan) {
    const int b = b0 + threadIdx.x, len = b < a.c.B ? cached_tokens(a.c, b) : 0;
    const int n = pieces_of(len, per, b < a.c.B), m = n > 1 ? n : 0, upto = wave_scan(n), slots = wave_scan(m);
    if (lane == 63) sums[0][w] = upto, sums[1][w] = slots;
    __syncthreads();
    int at = first + upto - n, sl = slot + slots - m;
#pragma unroll
    for (int i = 0; i < kPlan / 64; ++i) {
      at += i < w ? sums[0][i] : 0;
      sl += i < w ? sums[1][i] : 0;
      first += sums[0][i];
      slot += sums[1][i];
    }
    for (int i = 0; i < n; ++i) a.map[at + i] = make_int4(b, i, n, sl);
    __syncthreads();
  }
  for (int i = first + threadIdx.x; i < a.pieces + a.c.B; i += kPlan) a.map[i] = make_int4(0, 0, 0, 0);
}

template <typename T, int DP>
struct Form {
  static constexpr int V = kV<T>, KT = kTile<T>, NT = KT / 16;
  static constexpr int nc = DP / (4 * V);                  // chunks that a lane holds of a key
  static constexpr int nd = DP / 16;                       // 16-wide blocks of a head
  static constexpr int cp = DP == 96 ? 128 / V : DP / V;   // lanes along a row of values, a power of two
  static constexpr int rs = 64 / cp, nv = KT / rs;         // rows of values a load; loads
  static constexpr int ld = DP + V;                        // LDS row
};

// acc(16 x 16) += A(16 x 4V) B(4V x 16): lane l gives row (A) or column (B) l % 16 and the indices of its chunk, the same for
// both; its four results are column l % 16 at the rows 4 (l / 16) + r.
__device__ __forceinline__ void mma16(f32x4& acc, const Chunk<bf16>& a, const Chunk<bf16>& b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)a.v, *(const bf16x8*)b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4& acc, const Chunk<float>& a, const Chunk<float>& b) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], acc, 0, 0, 0);
}

// Largest and sum over the four lanes of a row (16 apart).
__device__ __forceinline__ float row_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_add(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Values of the 16-wide block at t as an operand: the lane's column l % 16 of the tile's rows in the order of its probabilities.
__device__ __forceinline__ Chunk<bf16> values16(const bf16* t, int ld, int lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int g = lane >> 4, i = lane & 15;
  const bf16* p = t + (g * 4 + (i >> 2)) * ld + (i & 3) * 4;
  Chunk<bf16> c;
  *(s16x4*)c.v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  *(s16x4*)(c.v + 4) = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * ld));
  return c;
}
__device__ __forceinline__ Chunk<float> values16(const float* t, int ld, int lane) {
  const float* p = t + (lane >> 4) * 4 * ld + (lane & 15);
  Chunk<float> c;
#pragma unroll
  for (int j = 0; j < 4; ++j) c.v[j] = p[j * ld];
  return c;
}

// Keeps the wave's LDS writes and reads in the order of the source (the LDS itself takes a wave's accesses in order).
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A lane's token of a tile: its page and place there, and whether the piece holds it.
struct Place {
  int page, off;
  bool in;
};

template <typename T, int DP, int NR>
struct Lds {
  using F = Form<T, DP>;
  union alignas(16) {
    T values[kWaves][F::KT * F::ld];
    struct {
      float o[kWaves][16 * NR][DP + 4];
      float m[kWaves][16 * NR], l[kWaves][16 * NR];
    } join;
    T q[2][16 * NR * F::ld];   // the rows' queries, and what rounding them left
  };
};

// What a head's width asks of its loads: nothing (D = DP), zeros behind its chunks, or its last chunk value by value.
enum Fill : int { kFull = 0, kChunks = 1, kValues = 2 };

template <typename T, int DP, int NR, int Fit>
__global__ __launch_bounds__(kThreads, held(DP, NR)) void k_cached(Cached a) {
  using F = Form<T, DP>;
  constexpr int V = F::V, KT = F::KT;
  __shared__ Lds<T, DP, NR> lds;
  const int rt = blockIdx.x % a.tiles, sh = blockIdx.x / a.tiles, hk = sh % a.c.Hk;
  const Piece pc = find(a, sh / a.c.Hk);
  if (pc.n < 1) return;
  if (a.split && pc.i == 0 && hk == 0 && rt == 0 && threadIdx.x == 0) a.split[pc.b] = make_int2(pc.n, pc.slot);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, b = pc.b, len = pc.len;
  const int per = ((len - 1) / pc.n + 32) / 32 * 32, k0 = pc.i * per;
  const int k1 = len - k0 < per ? len : k0 + per;   // the last piece's k0 + per may be past 2^31
  const int tend = (k1 + KT - 1) / KT;
  const int fresh = new_tokens(a.c, b, a.T), r0 = rt * 16 * NR;
  const int* table = a.c.tables + b * a.c.tb;
  const T *kb = (const T*)a.c.k + hk * a.c.kh, *vb = (const T*)a.c.v + hk * a.c.vh;

  // Loads below have no conditions of their own, so that they are all under way before the first is waited for: places past
  // the piece are those of its last token, rows that do not count those of the tile's first one that does.
  auto lookup = [&](int t) {
    const int key = t * KT + (lane & (KT - 1)), at = min(key, k1 - 1), i = at / a.by_page;
    return Place{table[i], at - i * a.c.page, key < k1};
  };
  auto alive = [&](const Place& p) {
    const bool known = p.page >= 0 && p.page < a.c.pages;
    return (unsigned char)(a.c.live ? a.c.live[(known ? p.page : 0) * a.c.lp + p.off * a.c.lt] : 1);
  };
  Chunk<T> kf[F::NT][F::nc], vr[F::nv];
  unsigned ok;   // the tile's tokens that count
  auto fetch = [&](const Place& p, unsigned char m) {
    ok = (unsigned)(__ballot(p.in && p.page >= 0 && p.page < a.c.pages && m != 0) & ((1ull << KT) - 1));
    if (!ok) return;
    const int first = __builtin_ctz(ok);
    const long long ko = p.page * a.c.kp + p.off * a.c.kt, vo = a.alike ? ko : p.page * a.c.vp + p.off * a.c.vt;
    auto chunk = [&](const T* at, int d) {
      Chunk<T> c;
      if (Fit == kValues) return load_chunk(at + d, a.c.D - d);
      __builtin_memcpy(c.v, at + ((Fit == kFull && DP != 96) || d < a.c.D ? d : 0), 16);
      return c;
    };
#pragma unroll
    for (int t = 0; t < F::NT; ++t) {
      const int row = 16 * t + (lane & 15);
      const T* at = kb + __shfl(ko, (ok >> row) & 1 ? row : first);
#pragma unroll
      for (int c = 0; c < F::nc; ++c) kf[t][c] = chunk(at, (c * 4 + g) * V);
    }
#pragma unroll
    for (int i = 0; i < F::nv; ++i) {
      const int row = lane / F::cp + i * F::rs;
      vr[i] = chunk(vb + __shfl(vo, (ok >> row) & 1 ? row : first), lane % F::cp * V);
    }
  };

  int t = k0 / KT + w;
  Place p1{}, p2{};
  unsigned char m1 = 0;
  ok = 0;
  if (k1 > k0) {
    const Place p0 = lookup(t);
    p1 = lookup(t + kWaves);
    p2 = lookup(t + 2 * kWaves);
    const unsigned char m0 = alive(p0);
    m1 = alive(p1);
    fetch(p0, m0);
  }

  // the rows' queries
  const int rows = min(16 * NR, a.R - r0);
  for (int i = threadIdx.x; i < 16 * NR * a.units; i += kThreads) {
    const int r = i / a.by_units;
    const PairUnit u = pair_unit<1>(a.r, a.c.D, i - r * a.units);
    float x[1] = {0.f}, y[1] = {0.f};
    if (r < rows) {
      const int qt = (r0 + r) / a.by_rep, h = hk * a.rep + (r0 + r - qt * a.rep);
      const T* q = (const T*)a.q + b * a.qb + qt * a.ql + h * a.qh;
      x[0] = (float)q[u.e0];
      if (u.second) y[0] = (float)q[u.e1];
      if (u.axis >= 0) {
        float c[1], s[1];
        turn(position(a.pos, b * a.pos.pb + qt * a.pos.pl + u.axis * a.pos.pa), a.r.quarters[u.pair], c[0], s[0]);
        turn_runs<1, false>(x, y, c, s, false);
      }
    }
    auto put = [&](int e, float f) {
      const T hi = (T)f;
      lds.q[0][r * F::ld + e] = hi;
      if (sizeof(T) == 2) lds.q[1][r * F::ld + e] = fabsf((float)hi) < INFINITY ? (T)(f - (float)hi) : (T)0.f;
    };
    put(u.e0, x[0]);
    if (u.second) put(u.e1, y[0]);
  }
  const int gap = DP - a.c.D;
  for (int i = threadIdx.x; i < 16 * NR * gap; i += kThreads) {
    const int r = i / gap, e = a.c.D + i - r * gap;
    lds.q[0][r * F::ld + e] = (T)0.f;
    if (sizeof(T) == 2) lds.q[1][r * F::ld + e] = (T)0.f;
  }
  __syncthreads();
  const bool fine = sizeof(T) == 2 && a.r.axes > 0;
  Chunk<T> qf[NR][F::nc], ql[NR][F::nc];
  int lim[NR], own[NR];   // tokens that the lane's row sees; its query
  const int all = max(0, a.c.lengths[b]);   // with those that the table has no room for: a query's place goes by them
  auto seen_by = [&](int q) { return q >= fresh ? 0 : a.causal ? min(len, max(0, all - (fresh - 1 - q))) : len; };
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int c = 0; c < F::nc; ++c) {
      const int at = (16 * n + (lane & 15)) * F::ld + (c * 4 + g) * V;
      *(f32x4*)qf[n][c].v = *(const f32x4*)&lds.q[0][at];
      if (sizeof(T) == 2) *(f32x4*)ql[n][c].v = *(const f32x4*)&lds.q[1][at];
    }
    const int r = r0 + 16 * n + (lane & 15);
    own[n] = r / a.by_rep;
    lim[n] = r >= a.R ? len : seen_by(own[n]);
  }
  // the fewest tokens that a row sees: its first query's, or none where the last one is past the new tokens
  const int q0 = r0 / a.by_rep, q1 = (r0 + rows - 1) / a.by_rep, least = q1 >= fresh ? 0 : seen_by(q0);
  __syncthreads();

  T* tv = lds.values[w];
  float m[NR], l[NR];
  f32x4 acc[NR][F::nd];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < F::nd; ++d) acc[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 1
  for (; t < tend; t += kWaves) {
    const unsigned char m2 = alive(p2);
    const Place p3 = lookup(t + 3 * kWaves);
    const unsigned here = ok;
    const bool edge = (t + 1) * KT > least;
    bool odd = false;   // values that some row does not see are not finite
    f32x4 s[NR][F::NT];
    if (here) {
#pragma unroll
      for (int i = 0; i < F::NT; ++i) {
#pragma unroll
        for (int c = 0; c < F::nc; ++c)
          if (Fit == kChunks && (c * 4 + g) * V >= a.c.D) kf[i][c] = Chunk<T>{};
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < F::nc; ++c) mma16(s[n][i], kf[i][c], qf[n][c]);
          if (fine) {
#pragma unroll
            for (int c = 0; c < F::nc; ++c) mma16(s[n][i], kf[i][c], ql[n][c]);
          }
        }
      }
      wave_order();
#pragma unroll
      for (int i = 0; i < F::nv; ++i) {
        const int row = lane / F::cp + i * F::rs, d = lane % F::cp * V;
        f32x4 v = *(const f32x4*)vr[i].v;
        if (sizeof(T) == 4 && !((here >> row) & 1)) v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (DP != 96 || d < DP) *(f32x4*)(tv + row * F::ld + d) = v;
        if (edge) {
#pragma unroll
          for (int j = 0; j < V; ++j) odd |= !(fabsf((float)vr[i].v[j]) < INFINITY);
        }
      }
      wave_order();
      odd = __any(odd);
    }
    fetch(p1, m1);
    p1 = p2, m1 = m2, p2 = p3;
    if (!here) continue;

    const bool all = !edge && here == (unsigned)((1ull << KT) - 1);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < F::NT; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = 16 * i + 4 * g + r;
          s[n][i][r] *= a.scale;
          if (!all) s[n][i][r] = ((here >> key) & 1) && t * KT + key < lim[n] ? s[n][i][r] : -INFINITY;
          top = fmaxf(top, s[n][i][r]);
        }
      }
      top = fmaxf(m[n], row_max(top));
      if (__any(top > m[n])) {
        const float by = m[n] == -INFINITY ? 0.f : hw_exp2(m[n] - top);
        m[n] = top;
        l[n] *= by;
#pragma unroll
        for (int d = 0; d < F::nd; ++d) acc[n][d] *= by;
      }
      const float base = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int i = 0; i < F::NT; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[n][i][r] = hw_exp2(s[n][i][r] - base);
          l[n] += s[n][i][r];
        }
      }
    }
    // acc += values p. Part: for the rows of one query, whose values from `seen` on count as zeros.
    auto add = [&](bool part, int query, int seen) {
      Chunk<T> hi[NR], lo[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float p = s[n][j / 4][j % 4];
          hi[n].v[j] = (T)p;
          if (sizeof(T) == 2) lo[n].v[j] = (T)(p - (float)hi[n].v[j]);
        }
      }
#pragma unroll
      for (int d = 0; d < F::nd; ++d) {
        Chunk<T> f = values16(tv + 16 * d, F::ld, lane);
        if (part) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            {
              const int key = 16 * (j / 4) + 4 * g + j % 4;
              if (t * KT + key >= seen || !((here >> key) & 1)) f.v[j] = (T)0.f;
            }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          f32x4 o = acc[n][d];
          mma16(o, f, hi[n]);
          if (sizeof(T) == 2) mma16(o, f, lo[n]);
          if (!part || own[n] == query) acc[n][d] = o;   // a lane's results are its own row's
        }
      }
    };
    if (!odd) {
      add(false, 0, 0);
    } else {
      for (int q = q0; q <= q1; ++q) add(true, q, seen_by(q));
    }
  }

  // the waves' rows
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = 16 * n + (lane & 15);
    const float sum = row_add(l[n]);
    if (g == 0) {
      lds.join.m[w][r] = m[n];
      lds.join.l[w][r] = sum;
    }
#pragma unroll
    for (int d = 0; d < F::nd; ++d) *(f32x4*)&lds.join.o[w][r][16 * d + 4 * g] = acc[n][d];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * NR * (DP / 4); i += kThreads) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    if (r >= rows || d >= a.c.D) continue;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) top = fmaxf(top, lds.join.m[k][r]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float by = hw_exp2(lds.join.m[k][r] - base);
      sum = fmaf(lds.join.l[k][r], by, sum);
      o += *(const f32x4*)&lds.join.o[k][r][d] * by;
    }
    if (pc.n == 1) {
      const int qt = (r0 + r) / a.by_rep, h = hk * a.rep + (r0 + r - qt * a.rep);
      T* to = (T*)a.o + (((long long)b * a.T + qt) * a.H + h) * a.c.D + d;
      const float by = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < a.c.D) to[j] = (T)(sum == 0.f ? 0.f : o[j] * by);
    } else {
      const long long at = ((long long)(pc.slot + pc.i) * a.c.Hk + hk) * a.R + r0 + r;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < a.c.D) a.part[at * a.c.D + d + j] = o[j];
      if (d == 0) a.stat[at] = make_float2(top, sum);
    }
  }
}

// Joins the pieces of a split sequence's rows, `share` workgroups a sequence: a thread has four values of the head in every
// 256 / (D / 4)-th piece, with a running maximum and sum of its own; those are joined in order. 4 us for 8 pieces, 5 for 190: the
// launch and two loads behind each other.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_cached_join(Cached a, int share) {
  __shared__ f32x4 part[kThreads];
  __shared__ float tops[kThreads], sums[kThreads];
  const int b = blockIdx.x / share, first = blockIdx.x - b * share;
  const int2 sp = a.split[b];
  if (sp.x <= 1) return;
  const int D = a.c.D, quads = (D + 3) / 4, groups = kThreads / quads, q = threadIdx.x % quads, gr = threadIdx.x / quads;
  for (int row = first; row < a.c.Hk * a.R; row += share) {
    const int hk = row / a.R, r = row - hk * a.R;
    float top = -INFINITY, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (gr < groups) {
#pragma unroll 4
      for (int i = gr; i < sp.x; i += groups) {
        const long long at = ((long long)(sp.y + i) * a.c.Hk + hk) * a.R + r;
        const float2 st = a.stat[at];
        const float* p = a.part + at * D + 4 * q;
        f32x4 v;
        if (D % 4 == 0) {
          __builtin_memcpy(&v, p, 16);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = p[min(j, D - 1 - 4 * q)];
        }
        const float now = fmaxf(top, st.x), base = now == -INFINITY ? 0.f : now;
        const float by = hw_exp2(top - base), w = hw_exp2(st.x - base);
        top = now;
        sum = fmaf(sum, by, st.y * w);
        o = o * by + v * w;
      }
    }
    part[threadIdx.x] = o;
    tops[threadIdx.x] = top;
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (gr == 0) {
      for (int i = 1; i < groups; ++i) top = fmaxf(top, tops[i * quads + q]);
      const float base = top == -INFINITY ? 0.f : top;
      o = f32x4{0.f, 0.f, 0.f, 0.f}, sum = 0.f;
      for (int i = 0; i < groups; ++i) {
        const float w = hw_exp2(tops[i * quads + q] - base);
        sum = fmaf(sums[i * quads + q], w, sum);
        o += part[i * quads + q] * w;
      }
      const int qt = r / a.by_rep, h = hk * a.rep + (r - qt * a.rep);
      T* to = (T*)a.o + (((long long)b * a.T + qt) * a.H + h) * D + 4 * q;
      const float by = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * q + j < D) to[j] = (T)(sum == 0.f ? 0.f : o[j] * by);
    }
    __syncthreads();
  }
}

int check_call(const char* who, const splat_cache* c, const splat_rotation* r, const splat_positions* p, int H, long long T,
               float scale) {
  if (const int rc = check_cache(who, c)) return rc;
  if (H < 1 || H % c->Hk || T < 0) return set_error(kInvalid, "%s: %d heads over %d, %lld tokens", who, H, c->Hk, T);
  if (!(fabsf(scale) <= 3.402823466e38f)) return set_error(kInvalid, "%s: scale %g", who, scale);
  if (T > 0x7fffffffLL || T * H > 0x7fffffffLL || c->B * T * H > 0x7fffffffLL)
    return set_error(kUnsupported, "%s: %d x %lld tokens of %d heads", who, c->B, T, H);
  return check_rotation(who, r, p, c->D);
}

Cached plan(const splat_cache& c, int H, int T) {
  Cached n{};
  n.c = c;
  n.H = H;
  n.T = T;
  n.rep = H / c.Hk;
  n.R = T * n.rep;
  n.tiles = div_up(n.R, n.R > 16 ? 32 : 16);
  // One round of workgroups, as many as the card holds, while there are sequences to cut; rounds of smaller pieces, which make
  // up for different lengths, where there are many.
  const int all = 256 * held(c.D <= 32 ? 32 : c.D <= 64 ? 64 : c.D <= 96 ? 96 : 128, n.R > 16 ? 2 : 1);
  const long long each = (long long)c.Hk * n.tiles, once = std::max(1LL, all / each);
  n.fit = c.B <= 64 && 2 * c.B <= once;
  n.pieces = (int)(n.fit ? once : (kRounds * all + each - 1) / each);
  n.cut = (long long)c.page * c.width <= kLeast || n.pieces <= 1 ? kWhole : c.B <= 64 ? kScanned : kMapped;
  n.by_rep = fast_div(n.rep);
  n.by_page = fast_div(c.page);
  return n;
}

// Parts of the workspace: the list of pieces, the sequences' pieces, statistics and rows of the pieces of split sequences, of
// which there are at most twice as many as aimed at (each sequence has fewer than one more than its tokens would fill).
struct Bytes {
  size_t map, split, rows, all;
};
Bytes bytes_of(const Cached& n) {
  if (n.cut == kWhole) return {0, 0, 0, 0};
  const size_t map = n.cut == kMapped ? sizeof(int4) * ((size_t)n.pieces + n.c.B) : 0, split = sizeof(int2) * n.c.B;
  const size_t rows = (size_t)2 * n.pieces * n.c.Hk * n.R;
  return {map, split, rows, map + split + sizeof(float) * rows * (n.c.D + 2)};
}

template <typename F>
int with_form(int dtype, int D, int R, F&& f) {
  auto fit = [&](auto t, auto dp, auto nr) {
    if (D == decltype(dp)::value) return f(t, dp, nr, std::integral_constant<int, kFull>{});
    if (D % kV<decltype(t)> == 0) return f(t, dp, nr, std::integral_constant<int, kChunks>{});
    return f(t, dp, nr, std::integral_constant<int, kValues>{});
  };
  auto rows = [&](auto t, auto dp) {
    return R > 16 ? fit(t, dp, std::integral_constant<int, 2>{}) : fit(t, dp, std::integral_constant<int, 1>{});
  };
  auto head = [&](auto t) {
    if (D <= 32) return rows(t, std::integral_constant<int, 32>{});
    if (D <= 64) return rows(t, std::integral_constant<int, 64>{});
    if (D <= 96) return rows(t, std::integral_constant<int, 96>{});
    return rows(t, std::integral_constant<int, 128>{});
  };
  return dtype == kF32 ? head(float{}) : head(bf16{});
}

}  // namespace
}  // namespace splat

using namespace splat;

extern "C" {

size_t splat_cached_attention_workspace_bytes(const splat_cache* c, int H, long long T) {
  if (check_call("splat_cached_attention_workspace_bytes", c, nullptr, nullptr, H, T, 0.f) || c->B == 0 || T == 0) return 0;
  const Cached n = plan(*c, H, (int)T);
  return bytes_of(n).all;
}

int splat_cached_attention(const splat_cache* c, const splat_rotation* r, const splat_positions* p, const void* q, long long qb,
                           long long ql, long long qh, int H, long long T, float scale, int causal, void* o, void* ws,
                           size_t ws_bytes, void* stream) {
  if (const int rc = check_call("splat_cached_attention", c, r, p, H, T, scale)) return rc;
  if (c->B == 0 || T == 0) return kOk;
  if (!q || !o) return set_error(kInvalid, "splat_cached_attention: null pointer");
  Cached n = plan(*c, H, (int)T);
  if (c->pages == 0) n.c.width = 0;   // nothing can be read: no sequence has tokens
  const size_t need = splat_cached_attention_workspace_bytes(c, H, T);
  if (need && (!ws || ws_bytes < need))
    return set_error(kWorkspace, "splat_cached_attention: workspace of %zu bytes, %zu needed", ws_bytes, need);
  const long long grid = ((long long)(n.cut == kWhole ? 0 : n.pieces) + c->B) * c->Hk * n.tiles;
  if (grid > 0xffffffLL) return set_error(kUnsupported, "splat_cached_attention: %d sequences of %d heads", c->B, H);
  if (r) n.r = *r;
  if (p) n.pos = *p;
  n.q = q, n.o = o, n.qb = qb, n.ql = ql, n.qh = qh, n.causal = causal;
  n.scale = scale * kLog2e;
  n.units = pair_units(n.r, c->D, 1).n;
  n.by_units = fast_div(n.units);
  n.alike = c->kp == c->vp && c->kt == c->vt;
  if (need) {
    const Bytes at = bytes_of(n);
    n.map = (int4*)ws;
    n.split = (int2*)((char*)ws + at.map);
    n.stat = (float2*)((char*)n.split + at.split);
    n.part = (float*)(n.stat + at.rows);
  }
  const hipStream_t st = (hipStream_t)stream;
  return with_form(c->dtype, c->D, n.R, [&](auto t, auto dp, auto nr, auto fit) {
    using E = decltype(t);
    if (n.cut == kMapped) k_cached_plan<<<1, kPlan, 0, st>>>(n);
    k_cached<E, decltype(dp)::value, decltype(nr)::value, decltype(fit)::value><<<(unsigned)grid, kThreads, 0, st>>>(n);
    if (need) {   // a workgroup a row for few sequences; of many, the most are not split
      const int share = std::max(1, std::min(c->Hk * n.R, 16384 / c->B));
      k_cached_join<E><<<(unsigned)(c->B * share), kThreads, 0, st>>>(n, share);
    }
    return check_launch("splat_cached_attention");
  });
}

}  // extern "C"
