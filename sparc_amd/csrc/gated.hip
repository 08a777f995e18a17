// The gated half of a feed-forward block (include/sparc_hip.h):
//   y = act(x Wg^T) * (x Wu^T)
// and with g = x Wg^T, u = x Wu^T, dg = dy u act'(g), du = dy act(g):
//   dx = dg Wg + du Wu,   dWg = dg^T x,   dWu = du^T x.
//
// All of them are matrix products: out[q][p] = sum over k of Q[q][k] P[p][k].  A launch
// makes g and u of a tile together and leaves y, or (the backward computes them again
// instead of keeping them: nothing of the width of the block is saved, and dg and du
// come from unrounded g and u) dg and du.  dx is one launch over both contractions, the
// weights' gradients are one launch of two products.
//
// Bound by what feeds the matrix instructions from LDS (a step of 64 values of a tile of
// 256 x 256 takes 192 KB of reads there, about as long as its products), and where the
// contraction is short by a tile's first loads and its results, which nothing overlaps
// with one tile to a CU.  bf16, forward, in long runs: 8192 x 4096 on 4096 484 us (1.14
// PFLOP/s), 32768 x 768 on 2048 247 us (0.83 PFLOP/s; the whole backward 789); 256 rows of
// 2048 on 8192 28 us, 1 row 14 us (67 MB of weights, 4.8 TB/s).  fp32: 1237 x 1001 on 2731
// 91 us (148 TFLOP/s as one product's, 890 as the six bf16 ones).
#include "matrix.h"

namespace sparc {
namespace {

enum Act : int { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2, ACT_SIGMOID = 3 };

// act(g), and its derivative.  For results in bf16 the sigmoid is that of the hardware's
// base-2 exponential and reciprocal: off by some 2^-22 of its value, and for negative g
// by |g| 2^-24 more, what rounding the exponent |g| / ln 2 leaves (2^-17 at g = -80,
// where a result's rounding is 2^-8).  The library's functions take 30 instructions more
// for each value, and a tile of 256 x 256 results is computed in little more time than
// its activations were.
template <typename IO> __device__ __forceinline__ float act_of(int act, float g, float& slope) {
  if (act == ACT_RELU) {
    slope = g > 0.0f ? 1.0f : 0.0f;
    return g < 0.0f ? 0.0f : g;  // NaN stays
  }
  if (act == ACT_GELU) {
    const float phi = 0.5f * erfcf(g * -0.70710678118654752f);
    slope = phi + g * expf(-0.5f * g * g) * 0.39894228040143268f;
    return g * phi;
  }
  const float sig = sizeof(IO) == 2 ? __builtin_amdgcn_rcpf(1.0f + fast_exp(-g)) : 1.0f / (1.0f + expf(-g));
  if (act == ACT_SIGMOID) {
    slope = sig * (1.0f - sig);
    return sig;
  }
  slope = sig * (1.0f + g * (1.0f - sig));
  return g * sig;
}

// An operand: rows r (the result's p or q) and the contraction k; element (r, k) at
// r ld + k, or (ACROSS) at k ld + r.  Each part has a tensor of its own.
struct Operand {
  const void* p[4];
  int64_t ld, rows;
};
struct ProductArgs {
  Operand P, Q;
  int64_t nk;             // contraction of a part
  int parts;              // PARTS: of the contraction; PAIR: of each product's
  int p_tiles, q_tiles;   // workgroups; in PAIR and of a gated product each side's own tiles
  void* out[4];           // [rows q, rows p], row stride out_ld; GATED_BACK: [2], [3] what rounding took (or NULL)
  int64_t out_ld;
  const void* dy;         // GATED_BACK: [Q.rows, P.rows]
  int act;
  int split_steps;        // steps of the contraction (over all parts) of one workgroup
  float* partial;         // [splits, sides, Q.rows, P.rows]; NULL: one workgroup does all
};

// GATED: both parts of P at once, out[0] = act(.) * (.).  GATED_BACK: out[0] and out[1]
// the gradients of both projections.  PARTS: the sum over all parts.  PAIR: a product
// for each of two tensors of Q, and over every second part.
enum Kind : int { GATED = 0, GATED_BACK = 1, PARTS = 2, PAIR = 3 };

// What rounding to bf16 takes from values (nothing where that is not finite)
__device__ __forceinline__ f32x4 rest_of(const f32x4& x) {
  f32x4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float rest = x[r] - bf16_bits_to_float(pack_bf16(x[r]));
    y[r] = fabsf(rest) < __builtin_inff() ? rest : 0.0f;
  }
  return y;
}

// An offset that no buffer reaches: loads there give zero.
constexpr uint32_t kNowhere = 0x80000000u;

// LINES x COLS values of an operand on their way from memory to LDS, through a buffer
// that ends with the last line, so that no load is under a condition: what lies behind
// the last line or column is zero.  A vector that the columns' end would cut is read so
// that it ends with them, and shifted.  fp32 values become the sum of three bf16 values
// (truncated, then the rest truncated, then the rest, which is exact: 8 bits each).
// WHOLE: no vector is cut.
template <typename IO, int LINES, int COLS, int THREADS, bool ACROSS, bool WHOLE> struct Feed {
  static constexpr int VEC = kVec<IO>, PER = COLS / VEC, SIZE = sizeof(IO), STEP = THREADS / PER, N = LINES / STEP;
  static constexpr int PARTS = SIZE == 2 ? 1 : 3;
  using L = Panel<bf16, COLS, ACROSS>;
  static constexpr int kSize = LINES * L::kStride;  // of one part
  static_assert(THREADS % PER == 0 && LINES % STEP == 0, "whole vectors per thread");
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  u4 r[N];
  int lack;

  static __device__ __forceinline__ int line() { return static_cast<int>(threadIdx.x) / PER; }
  static __device__ __forceinline__ int column() { return static_cast<int>(threadIdx.x) % PER * VEC; }
  // Columns up to ``end`` of lines of ``size`` values; at(i) is the byte of line(i)'s
  // first column in the buffer, or kNowhere.
  template <typename F>
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t buffer, int64_t end, int64_t size, F&& at) {
    fetch_by(end, size, [&](int) __attribute__((always_inline)) { return buffer; }, at);
  }
  template <typename B, typename F>
  __device__ __forceinline__ void fetch_by(int64_t end, int64_t size, B&& buffer, F&& at) {
    const int64_t c = column();
    const int64_t left = WHOLE || c + VEC <= end || size < VEC ? c : end - VEC;
    lack = static_cast<int>(c - left);
    const bool there = lack < VEC && c < end;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = one(buffer(i), at(i), there, left, end, size);
  }
  static __device__ __forceinline__ u4 one(__amdgpu_buffer_rsrc_t buffer, uint32_t line_at, bool there, int64_t left,
                                           int64_t end, int64_t size) {
    const uint32_t first = there && line_at < kNowhere ? line_at + static_cast<uint32_t>(left * SIZE) : kNowhere;
    if (WHOLE || size >= VEC) return __builtin_amdgcn_raw_buffer_load_b128(buffer, first, 0, 0);
    // lines shorter than a vector, value by value: a vector would end behind the last one
    u4 u = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const uint32_t from = left + k < end ? first + k * SIZE : kNowhere;
      if constexpr (SIZE == 4) u[k] = __builtin_amdgcn_raw_buffer_load_b32(buffer, from, 0, 0);
      else u[k / 2] |= static_cast<uint32_t>(__builtin_amdgcn_raw_buffer_load_b16(buffer, from, 0, 0)) << (16 * (k % 2));
    }
    return u;
  }
  __device__ __forceinline__ void put(bf16* lds, bool ragged) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      u4 u = r[i];
      if (!WHOLE && ragged) {
        const int words = lack * SIZE / 4, odd = lack * SIZE % 4;
        uint32_t w[5];
#pragma unroll
        for (int k = 0; k < 5; ++k) {
          w[k] = 0;
#pragma unroll
          for (int m = k; m < 4; ++m) w[k] = words == m - k ? u[m] : w[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = odd ? w[k] >> 16 | w[k + 1] << 16 : w[k];
      }
      bf16* const to = lds + L::at(line() + i * STEP, column());
      if constexpr (SIZE == 2) {
        *reinterpret_cast<u4*>(to) = u;
      } else {
        float x[4];
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          typedef uint32_t u2 __attribute__((ext_vector_type(2)));
          *reinterpret_cast<u2*>(to + part * kSize) = u2{upper_halves(u[0], u[1]), upper_halves(u[2], u[3])};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[k] = __uint_as_float(u[k]) - __uint_as_float(u[k] & 0xffff0000u);
            u[k] = __float_as_uint(x[k]);
          }
        }
      }
    }
  }
};

// TP x TQ results by WP x WQ waves; BK values of the contraction at a time, in BUFFERS
// places in LDS.  KS: groups of so many waves that share the BK values and are added up
// at the end, where tiles are small and more waves would each have fewer results for what
// they read (1 row of 2048 on 8192 in fp32: 53 us with eight waves beside one another, 41
// with two groups of four).  Tiles of 128 have eight waves rather than four, which leave
// a SIMD one each (1500 rows of 768 on 2048 29.5 -> 24.8 us, 256 of 3549 on 4105 78 -> 63).
template <typename IO, int KIND, bool PA, bool QA, int TP, int TQ, int WP, int WQ, int KS, int BK, int BUFFERS, bool WHOLE>
__global__ __launch_bounds__(64 * WP * WQ * KS, 2) void product_kernel(const ProductArgs a) {
  constexpr bool DUAL = KIND == GATED || KIND == GATED_BACK;
  constexpr int THREADS = 64 * WP * WQ * KS, VEC = kVec<IO>, SIZE = sizeof(IO);
  constexpr int LP = TP / WP, LQ = TQ / WQ, MP = LP / 16, MQ = LQ / 16;  // a wave's results, and in tiles
  constexpr int PT = DUAL ? TP / 2 : TP;
  using FP = Feed<IO, PA ? BK : TP, PA ? TP : BK, THREADS, PA, WHOLE>;
  using FQ = Feed<IO, QA ? BK : TQ, QA ? TQ : BK, THREADS, QA, WHOLE>;
  constexpr int SP = FP::kSize * FP::PARTS, SQ = FQ::kSize * FQ::PARTS, SUM = FP::PARTS;
  __shared__ __attribute__((aligned(16))) bf16 lds[BUFFERS * (SP + SQ)];

  const int lane = threadIdx.x & 63, col = lane & 15, quad = 4 * (lane >> 4);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % (WP * WQ);
  const int share = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / (WP * WQ);  // of the BK values
  const int wp = wave % WP * LP, wq = wave / WP * LQ;
  // neighbouring workgroups of an XCD: eight tiles of q beside all of p
  const int sides = KIND == PAIR ? 2 : 1;
  const int per_split = a.p_tiles * a.q_tiles * sides, id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int split = id / per_split, rest = id % per_split;
  const int all_q = a.q_tiles * sides, group = rest / (8 * a.p_tiles), first_q = 8 * group;
  const int here = all_q - first_q < 8 ? all_q - first_q : 8, within = rest - 8 * group * a.p_tiles;
  const int q_tile = first_q + within % here, p_tile = within / here;
  const int side = KIND == PAIR ? q_tile / a.q_tiles : 0;
  const int64_t p0 = static_cast<int64_t>(p_tile) * PT, q0 = static_cast<int64_t>(q_tile - side * a.q_tiles) * TQ;
  const int64_t k1 = a.nk;

  FP fp;
  FQ fq;
  // a tile's lines of the contraction from k on, or its rows
  const auto fetch = [&](auto& feed, const Operand& o, auto across, auto dual, int64_t r0, int64_t k, int part)
                         __attribute__((always_inline)) {
    using F = std::remove_reference_t<decltype(feed)>;
    if constexpr (decltype(across)::value) {
      const int lines = static_cast<int>(k1 - k < BK ? k1 - k : BK);
      // a vector's start may have to move left of the tile: offsets count from the lines' start
      const auto buffer = make_rsrc(static_cast<const IO*>(o.p[part]) + k * o.ld,
                                    static_cast<uint32_t>(((lines - 1) * o.ld + o.rows) * SIZE));
      feed.fetch(buffer, o.rows - r0, o.rows, [&](int i) __attribute__((always_inline)) {
        return static_cast<uint32_t>((F::line() + i * F::STEP) * o.ld + r0) * SIZE;
      });
    } else {
      const int64_t rows = o.rows - r0 < TP + TQ ? o.rows - r0 : TP + TQ;
      const auto buffer_of = [&](int which) __attribute__((always_inline)) {
        return make_rsrc(static_cast<const IO*>(o.p[which]) + r0 * o.ld,
                         static_cast<uint32_t>(((rows - 1) * o.ld + a.nk) * SIZE));
      };
      const auto at = [&](int row) __attribute__((always_inline)) {
        return row < rows ? static_cast<uint32_t>(row * o.ld + k) * SIZE : kNowhere;
      };
      if constexpr (decltype(dual)::value) {
        // of a wave's lines one half is of the first part, the other of the second; the
        // lines of one load are of one of them
        const auto gate = buffer_of(0), up = buffer_of(1);
        feed.fetch_by(k1 - k, a.nk, [&](int i) __attribute__((always_inline)) {
          return __builtin_amdgcn_readfirstlane(F::line() + i * F::STEP) / (LP / 2) % 2 ? up : gate;
        }, [&](int i) __attribute__((always_inline)) {
          const int line = F::line() + i * F::STEP;
          return at(line / LP * (LP / 2) + line % (LP / 2));
        });
      } else {
        feed.fetch(buffer_of(part), k1 - k, a.nk, [&](int i) __attribute__((always_inline)) {
          return at(F::line() + i * F::STEP);
        });
      }
    }
  };
  using PAcross = std::integral_constant<bool, PA>;
  using QAcross = std::integral_constant<bool, QA>;
  using Dual = std::integral_constant<bool, DUAL>;
  const auto fetch_p = [&](int64_t k, int part) __attribute__((always_inline)) {
    fetch(fp, a.P, PAcross(), Dual(), p0, k, part);
  };
  const auto fetch_q = [&](int64_t k, int part) __attribute__((always_inline)) {
    fetch(fq, a.Q, QAcross(), std::false_type(), q0, k, KIND == PAIR ? side + 2 * part : part);
  };
  const auto tail = [&](int64_t k) { return k1 - k < BK && (k1 - k) % VEC != 0 && a.nk >= VEC; };
  const auto put_p = [&](int place, int64_t k) __attribute__((always_inline)) {
    fp.put(lds + place * (SP + SQ), PA ? p0 + TP > a.P.rows && a.P.rows % VEC != 0 && a.P.rows >= VEC : tail(k));
  };
  const auto put_q = [&](int place, int64_t k) __attribute__((always_inline)) {
    fq.put(lds + place * (SP + SQ) + SP, QA ? q0 + TQ > a.Q.rows && a.Q.rows % VEC != 0 && a.Q.rows >= VEC : tail(k));
  };
  f32x4 acc[MP][MQ];
#pragma unroll
  for (int i = 0; i < MP; ++i)
#pragma unroll
    for (int j = 0; j < MQ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Frag<bf16> p[SUM][MP], q[SUM][MQ];
  // fragments of 32 values of the contraction, c of a place's BK on
  const auto read = [&](int place, int c) __attribute__((always_inline)) {
    const bf16* const lp = lds + place * (SP + SQ);
    const bf16* const lq = lp + SP;
#pragma unroll
    for (int n = 0; n < SUM; ++n) {
#pragma unroll
      for (int i = 0; i < MP; ++i) {
        if constexpr (PA) p[n][i] = read_columns<typename FP::L>(lp + n * FP::kSize, c, wp + 16 * i);
        else p[n][i] = read_rows<typename FP::L>(lp + n * FP::kSize, wp + 16 * i, c);
      }
#pragma unroll
      for (int j = 0; j < MQ; ++j) {
        if constexpr (QA) q[n][j] = read_columns<typename FQ::L>(lq + n * FQ::kSize, c, wq + 16 * j);
        else q[n][j] = read_rows<typename FQ::L>(lq + n * FQ::kSize, wq + 16 * j, c);
      }
    }
  };
  // of three parts each the six products that reach the 24 bits, the small ones first
  const auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int order = SUM - 1; order >= 0; --order)
#pragma unroll
      for (int n = 0; n <= order; ++n)
#pragma unroll
        for (int i = 0; i < MP; ++i)
#pragma unroll
          for (int j = 0; j < MQ; ++j) acc[i][j] = mma(p[n][i], q[order - n][j], acc[i][j]);
  };
  // steps: all of one part, then all of the next
  const int per_part = static_cast<int>((a.nk + BK - 1) / BK), all = per_part * (DUAL ? 1 : a.parts);
  const int begin = split * a.split_steps, end = begin + a.split_steps < all ? begin + a.split_steps : all;
  const int count = end - begin;
  // Goes from step to step and stays at the last one: what is fetched and put behind it
  // is not read, and without conditions a wait for some rows waits for no later ones.
  struct Walk {
    int64_t k;
    int part, left;
    __device__ __forceinline__ void next(int64_t nk) {
      if (left <= 1) return;
      --left;
      k += BK;
      if ((KIND == PARTS || KIND == PAIR) && k >= nk) k = 0, ++part;
    }
  };
  Walk at = {static_cast<int64_t>(begin % per_part) * BK, begin / per_part, count}, put_at = at;
  if constexpr (BUFFERS == 2) {
    // Places take turns: while a step is multiplied, the rows of the next go from
    // registers to the other place, and those of the one after it are fetched.
    fetch_p(at.k, at.part);
    fetch_q(at.k, at.part);
    put_p(0, put_at.k);
    put_q(0, put_at.k);
    at.next(a.nk);
    fetch_p(at.k, at.part);
    fetch_q(at.k, at.part);
    for (int step = 0; step < count; ++step) {
      const int place = step & 1;
      const auto next = [&]() __attribute__((always_inline)) {
        put_at.next(a.nk);
        at.next(a.nk);
        put_p(1 - place, put_at.k);
        put_q(1 - place, put_at.k);
        fetch_p(at.k, at.part);
        fetch_q(at.k, at.part);
      };
      __syncthreads();  // this step's place is filled, and the other one no longer read
#pragma unroll
      for (int c = 0; c < BK; c += 32 * KS) {
        // the other place is filled in the middle of a step: before it the rows would be
        // waited for at once, and no matrix instruction would run meanwhile
        if (KS == 1 && c == BK / 64 * 32) next();
        read(place, c + 32 * share);
        if (KS > 1 && c == 0) next();
        multiply();
      }
    }
  } else {
    fetch_p(at.k, at.part);
    fetch_q(at.k, at.part);
    for (int step = 0; step < count; ++step) {
      __syncthreads();
      put_p(0, put_at.k);
      put_q(0, put_at.k);
      __syncthreads();
      put_at.next(a.nk);
      at.next(a.nk);
      fetch_p(at.k, at.part);
      fetch_q(at.k, at.part);
#pragma unroll
      for (int c = 0; c < BK; c += 32 * KS) {
        read(0, c + 32 * share);
        multiply();
      }
    }
  }
  if constexpr (KS > 1) {
    static_assert(KS == 2 && sizeof(lds) >= sizeof(float) * TP * TQ, "the second group's results pass through LDS");
    f32x4* const sums = reinterpret_cast<f32x4*>(lds) + wave * MP * MQ * 64 + lane;
    __syncthreads();
    if (share == 1) {
#pragma unroll
      for (int i = 0; i < MP; ++i)
#pragma unroll
        for (int j = 0; j < MQ; ++j) sums[(i * MQ + j) * 64] = acc[i][j];
    }
    __syncthreads();
    if (share == 1) return;
#pragma unroll
    for (int i = 0; i < MP; ++i)
#pragma unroll
      for (int j = 0; j < MQ; ++j) acc[i][j] += sums[(i * MQ + j) * 64];
  }
  // all of dy first: a wait for a load behind a store waits for the store too
  f32x4 dys[KIND == GATED_BACK ? MP / 2 : 1][KIND == GATED_BACK ? MQ : 1];
  if constexpr (KIND == GATED_BACK) {
#pragma unroll
    for (int j = 0; j < MQ; ++j)
#pragma unroll
      for (int i = 0; i < MP / 2; ++i) {
        const int64_t q = q0 + wq + 16 * j + col, p = p0 + wp / 2 + 16 * i + quad;
        const int n = q < a.Q.rows ? static_cast<int>(a.P.rows - p < 4 ? a.P.rows - p : 4) : 0;
        dys[i][j] = load_quad(static_cast<const IO*>(a.dy) + q * a.P.rows + p, n);
      }
  }
#pragma unroll
  for (int j = 0; j < MQ; ++j) {
    const int64_t q = q0 + wq + 16 * j + col;
    if (q >= a.Q.rows) continue;
    if constexpr (DUAL) {
#pragma unroll
      for (int i = 0; i < MP / 2; ++i) {
        const int64_t p = p0 + wp / 2 + 16 * i + quad;
        const int n = static_cast<int>(a.P.rows - p < 4 ? a.P.rows - p : 4);
        if (n <= 0) continue;
        f32x4 slope, h;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float d;
          h[r] = act_of<IO>(a.act, acc[i][j][r], d);
          slope[r] = d;
        }
        const int64_t at = q * a.out_ld + p;
        if constexpr (KIND == GATED) {
          store_quad(static_cast<IO*>(a.out[0]) + at, n, h * acc[i + MP / 2][j]);
        } else {
          const f32x4 dy = dys[i][j];
          const f32x4 dg = dy * acc[i + MP / 2][j] * slope, du = dy * h;
          store_quad(static_cast<IO*>(a.out[0]) + at, n, dg);
          store_quad(static_cast<IO*>(a.out[1]) + at, n, du);
          if (sizeof(IO) == 2 && a.out[2]) {
            store_quad(static_cast<IO*>(a.out[2]) + at, n, rest_of(dg));
            store_quad(static_cast<IO*>(a.out[3]) + at, n, rest_of(du));
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < MP; ++i) {
        const int64_t p = p0 + wp + 16 * i + quad;
        const int n = static_cast<int>(a.P.rows - p < 4 ? a.P.rows - p : 4);
        if (n <= 0) continue;
        if (a.partial) store_quad(a.partial + ((split * sides + side) * a.Q.rows + q) * a.P.rows + p, n, acc[i][j]);
        else store_quad(static_cast<IO*>(a.out[side]) + q * a.out_ld + p, n, acc[i][j]);
      }
    }
  }
}

// The sum of the partial products, in order
template <typename IO>
__global__ __launch_bounds__(256) void product_sum_kernel(const float* partial, int splits, int64_t total, int64_t half,
                                                          IO* out0, IO* out1) {
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < total;
       e += static_cast<int64_t>(gridDim.x) * 256) {
    float s = 0.0f;
    for (int i = 0; i < splits; ++i) s += partial[i * total + e];
    IO* const o = e < half ? out0 + e : out1 + (e - half);
    if constexpr (sizeof(IO) == 4) *o = s;
    else o->bits = pack_bf16(s);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
const char* fault_of(int64_t rows, int64_t dim, int64_t hidden, int32_t io, int32_t act) {
  if (rows < 0 || dim < 1 || hidden < 1) return "gated linear unit: rows must not be negative, dim and hidden positive";
  // a tile's lines lie within 2^31 bytes
  if (rows >= (1LL << 31) || dim >= (1LL << 20) || hidden >= (1LL << 20)) return "gated linear unit: too large";
  if (io != SPARC_F32 && io != SPARC_BF16) return "gated linear unit: io_dtype must be F32 or BF16";
  if (act < ACT_SILU || act > ACT_SIGMOID) return "gated linear unit: unknown activation";
  return nullptr;
}
size_t size_of(int32_t io) { return io == SPARC_BF16 ? 2 : 4; }

int64_t tiles(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }
// values of the contraction that splits are counted in
template <typename IO> constexpr int kStep = sizeof(IO) == 2 ? 64 : 32;
int step_of(int32_t io) { return io == SPARC_BF16 ? kStep<bf16> : kStep<float>; }

// How a product is cut: into large tiles where they are enough for most CUs, into small
// ones, two to a CU, else; and its contraction into as many splits as fill the GPU, each
// of eight steps at least.
struct Cut {
  bool large;
  int splits, split_steps;
};
Cut cut_of(int32_t io, bool whole, int64_t np, int64_t nq, int64_t nk, int parts, bool may_split) {
  Cut c;
  const int64_t steps = tiles(nk, step_of(io)) * parts, most = may_split && steps >= 16 ? steps / 8 : 1;
  const int64_t big = tiles(np, 256) * tiles(nq, 256), small = tiles(np, 128) * tiles(nq, 128);
  c.large = io == SPARC_BF16 && whole && big * most >= 192;
  const int64_t count = c.large ? big : small, slots = c.large ? 256 : 512;
  int64_t n = count > 0 ? slots / count : 1;
  if (n > most) n = most;
  if (n > 64) n = 64;
  if (n < 1) n = 1;
  c.split_steps = static_cast<int>(tiles(steps, n));
  if (c.split_steps < 1) c.split_steps = 1;
  c.splits = static_cast<int>(tiles(steps, c.split_steps));
  if (c.splits < 1) c.splits = 1;
  return c;
}
// Whether no line's end cuts a vector, for lines of these lengths
bool is_whole(int32_t io, int64_t m, int64_t n = 0) { return io == SPARC_BF16 ? (m | n) % 8 == 0 : (m | n) % 4 == 0; }

// dg and du are rounded to bf16 for the products with them, which makes their results'
// errors 1.4 times as large as one rounding's: 0.00235 of the gradients instead of
// 0.00166 (two library products that keep the projections in bf16: 0.0034 to 0.0039).
// Where launches take the time rather than the products, what the rounding took is
// multiplied too, and the errors are one rounding's: the backward's kernels of 32 rows of
// 64 on 96 17.6 -> 21.6 us, of 1000 of 256 on 1024, at the border, 42 -> 50, behind some
// 50 of autograd.  Above it the products would be as many again as dx and the weights
// take: 512 rows of 1024 on 1024 38 -> 52 us, 512 of 1024 on 4096 64 -> 110, 2048 of
// 2048 on 8192 436 -> 660, 32768 of 768 on 2048 789 -> 1312.
constexpr int64_t kRestUpTo = 1LL << 28;  // rows x dim x hidden

struct GatedPlan {
  Cut dx, dw;
  int64_t g_ld;
  int parts;             // of dg and du: 2 with what rounding took
  size_t g, partial;     // bytes of a part of dg or du; of the partial sums, which dx and the weights' share
  size_t all() const { return 2 * parts * g + partial; }
};
GatedPlan gated_plan(int64_t rows, int64_t dim, int64_t hidden, int32_t io) {
  GatedPlan p;
  p.parts = io == SPARC_BF16 && rows <= kRestUpTo / (dim * hidden) ? 2 : 1;
  p.dx = cut_of(io, is_whole(io, dim, hidden), dim, rows, hidden, 2 * p.parts, true);
  p.dw = cut_of(io, is_whole(io, dim, hidden), dim, 2 * hidden, rows, p.parts, true);
  p.g_ld = tiles(hidden, 8) * 8;  // whole vectors, whatever the width
  p.g = up256(rows * p.g_ld * size_of(io));
  const size_t x = p.dx.splits > 1 ? sizeof(float) * p.dx.splits * rows * dim : 0;
  const size_t w = p.dw.splits > 1 ? sizeof(float) * p.dw.splits * 2 * hidden * dim : 0;
  p.partial = up256(x > w ? x : w);
  return p;
}

template <typename IO, int KIND, bool PA, bool QA, int TP, int TQ, int WP, int WQ, int KS, int BK, int BUFFERS, bool WHOLE>
void product_tiled(ProductArgs& a, int splits, hipStream_t stream) {
  constexpr bool DUAL = KIND == GATED || KIND == GATED_BACK;
  static_assert(DUAL || BK == kStep<IO>, "a split begins at a step of its own");  // (and a dual product has none)
  a.p_tiles = static_cast<int>(tiles(a.P.rows, DUAL ? TP / 2 : TP));
  a.q_tiles = static_cast<int>(tiles(a.Q.rows, TQ));
  const int64_t count = static_cast<int64_t>(a.p_tiles) * a.q_tiles * (KIND == PAIR ? 2 : 1) * splits;
  product_kernel<IO, KIND, PA, QA, TP, TQ, WP, WQ, KS, BK, BUFFERS, WHOLE><<<static_cast<unsigned>(count), 64 * WP * WQ * KS, 0, stream>>>(a);
}
template <typename IO, int KIND, bool PA, bool QA>
void product(ProductArgs& a, const Cut& cut, bool whole, hipStream_t stream) {
  a.split_steps = cut.split_steps;
  constexpr bool DUAL = KIND == GATED || KIND == GATED_BACK;
  if constexpr (DUAL) {
    // A few rows, for which the weights' way is all the time: tiles so small that most
    // CUs have one, all of them under way at once, each step of a whole 256 bytes of a
    // row (weights of 8192 x 2048 for 1 row 28.0 -> 16.6 us, for 64 30.7 -> 17.7, for
    // 128 31.5 -> 25.8; for 256, where they no longer are, 33.9 instead of 44.5; in fp32
    // for 1 row 121 -> 41; 14 rows of 3549 on 4105 bf16 73 -> 30).
    if (tiles(a.P.rows, 32) * tiles(a.Q.rows, 64) <= 512) {
      if constexpr (sizeof(IO) == 2) {
        if (whole) product_tiled<IO, KIND, PA, QA, 64, 64, 2, 2, 2, 128, 2, true>(a, 1, stream);
        else product_tiled<IO, KIND, PA, QA, 64, 64, 2, 2, 2, 128, 2, false>(a, 1, stream);
      } else {
        if (whole) product_tiled<IO, KIND, PA, QA, 64, 64, 2, 2, 2, 64, 2, true>(a, 1, stream);
        else product_tiled<IO, KIND, PA, QA, 64, 64, 2, 2, 2, 64, 2, false>(a, 1, stream);
      }
      return;
    }
  }
  if constexpr (sizeof(IO) == 2) {
    if (!whole) product_tiled<IO, KIND, PA, QA, 128, 128, 4, 2, 1, 64, 2, false>(a, cut.splits, stream);
    else if (cut.large) product_tiled<IO, KIND, PA, QA, 256, 256, 4, 2, 1, 64, 2, true>(a, cut.splits, stream);
    else product_tiled<IO, KIND, PA, QA, 128, 128, 4, 2, 1, 64, 2, true>(a, cut.splits, stream);
  } else {
    if (whole) product_tiled<IO, KIND, PA, QA, 128, 128, 4, 2, 1, 32, 1, true>(a, cut.splits, stream);
    else product_tiled<IO, KIND, PA, QA, 128, 128, 4, 2, 1, 32, 1, false>(a, cut.splits, stream);
  }
}

template <typename IO>
void gated_run(int32_t io, int64_t rows, int64_t dim, int64_t hidden, int act, const void* x, const void* wg,
               const void* wu, const void* dy, void* const (&out)[4], int64_t out_ld, hipStream_t stream) {
  ProductArgs a = {};
  a.P = {{wg, wu}, dim, hidden};
  a.Q = {{x, x}, dim, rows};
  a.nk = dim;
  for (int i = 0; i < 4; ++i) a.out[i] = out[i];
  a.out_ld = out_ld;
  a.dy = dy;
  a.act = act;
  const bool whole = is_whole(io, dim);
  const Cut cut = cut_of(io, whole, 2 * hidden, rows, dim, 1, false);
  if (dy) product<IO, GATED_BACK, false, false>(a, cut, whole, stream);
  else product<IO, GATED, false, false>(a, cut, whole, stream);
}
template <typename IO>
void sum_partial(const float* partial, int splits, int64_t total, int64_t half, void* out0, void* out1, hipStream_t stream) {
  product_sum_kernel<IO><<<op_grid((total + 255) / 256), 256, 0, stream>>>(partial, splits, total, half,
                                                                           static_cast<IO*>(out0), static_cast<IO*>(out1));
}
template <typename IO>
void gated_grads(int32_t io, int64_t rows, int64_t dim, int64_t hidden, const void* x, const void* wg, const void* wu,
                 void* const (&g)[4], void* dx, void* dwg, void* dwu, float* partial, const GatedPlan& plan,
                 hipStream_t stream) {
  const bool whole = is_whole(io, dim, hidden);
  if (dx) {
    ProductArgs a = {};
    a.P = {{wg, wu, wg, wu}, dim, dim};
    a.Q = {{g[0], g[1], g[2], g[3]}, plan.g_ld, rows};
    a.nk = hidden;
    a.parts = 2 * plan.parts;
    a.out[0] = a.out[1] = dx;
    a.out_ld = dim;
    a.partial = plan.dx.splits > 1 ? partial : nullptr;
    product<IO, PARTS, true, false>(a, plan.dx, whole, stream);
    if (a.partial) sum_partial<IO>(partial, plan.dx.splits, rows * dim, rows * dim, dx, dx, stream);
  }
  if (dwg) {
    ProductArgs a = {};
    a.P = {{x, x}, dim, dim};
    a.Q = {{g[0], g[1], g[2], g[3]}, plan.g_ld, hidden};
    a.nk = rows;
    a.parts = plan.parts;
    a.out[0] = dwg, a.out[1] = dwu;
    a.out_ld = dim;
    a.partial = plan.dw.splits > 1 ? partial : nullptr;
    if (rows > 0) product<IO, PAIR, true, true>(a, plan.dw, whole, stream);
    if (rows == 0 || a.partial)
      sum_partial<IO>(partial, rows > 0 ? plan.dw.splits : 0, 2 * hidden * dim, hidden * dim, dwg, dwu, stream);
  }
}

}  // namespace
}  // namespace sparc

using namespace sparc;

extern "C" {

sparc_status sparc_gated_forward(int64_t rows, int64_t dim, int64_t hidden, int32_t io_dtype, int32_t activation,
                                 const void* x, const void* gate_weight, const void* up_weight, void* y,
                                 sparc_stream_t stream_) {
  if (const char* fault = fault_of(rows, dim, hidden, io_dtype, activation)) return op_fail(SPARC_EINVAL, fault);
  if (rows == 0) return SPARC_OK;
  if (!x || !gate_weight || !up_weight || !y) return op_fail(SPARC_EINVAL, "gated linear unit: a tensor is NULL");
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (io_dtype == SPARC_BF16)
    gated_run<bf16>(io_dtype, rows, dim, hidden, activation, x, gate_weight, up_weight, nullptr, {y}, hidden, stream);
  else
    gated_run<float>(io_dtype, rows, dim, hidden, activation, x, gate_weight, up_weight, nullptr, {y}, hidden, stream);
  return op_launched("sparc_gated_forward");
}

size_t sparc_gated_workspace_bytes(int64_t rows, int64_t dim, int64_t hidden, int32_t io_dtype) {
  if (fault_of(rows, dim, hidden, io_dtype, 0)) return 0;
  const GatedPlan p = gated_plan(rows, dim, hidden, io_dtype);
  return p.all();
}

sparc_status sparc_gated_backward(int64_t rows, int64_t dim, int64_t hidden, int32_t io_dtype, int32_t activation,
                                  const void* x, const void* gate_weight, const void* up_weight, const void* dy,
                                  void* dx, void* dgate_weight, void* dup_weight, void* workspace,
                                  size_t workspace_bytes, sparc_stream_t stream_) {
  if (const char* fault = fault_of(rows, dim, hidden, io_dtype, activation)) return op_fail(SPARC_EINVAL, fault);
  if ((rows > 0 && (!x || !dy)) || !gate_weight || !up_weight || !dgate_weight != !dup_weight)
    return op_fail(SPARC_EINVAL, "gated linear unit: a tensor is NULL");
  const GatedPlan plan = gated_plan(rows, dim, hidden, io_dtype);
  if (rows > 0 && (!workspace || workspace_bytes < plan.all()))
    return op_fail(SPARC_EWORKSPACE, "gated linear unit: workspace missing or too small");
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  char* const ws = static_cast<char*>(workspace);
  void* const g[4] = {ws, ws + plan.g, plan.parts == 2 ? ws + 2 * plan.g : nullptr, plan.parts == 2 ? ws + 3 * plan.g : nullptr};
  float* const partial = reinterpret_cast<float*>(ws + 2 * plan.parts * plan.g);
  const auto go = [&](auto type) {
    using IO = decltype(type);
    if (rows > 0) gated_run<IO>(io_dtype, rows, dim, hidden, activation, x, gate_weight, up_weight, dy, g, plan.g_ld, stream);
    gated_grads<IO>(io_dtype, rows, dim, hidden, x, gate_weight, up_weight, g, rows > 0 ? dx : nullptr, dgate_weight,
                    dup_weight, partial, plan, stream);
  };
  if (io_dtype == SPARC_BF16) go(bf16());
  else go(float());
  return op_launched("sparc_gated_backward");
}

}  // extern "C"
