// Operands of the matrix instructions (16x16 results in fp32), for fp32 and bf16
// values in one form.
//
// A fragment holds, for lane l of a wave, eight of 32 consecutive indices of the
// contraction of row (or column) l % 16: bf16 those from 8 (l / 16) on, fp32 16 h + 4
// (l / 16) + i (h < 2, i < 4).  Both operands of a product are held in this order, so
// the order in which the instruction itself numbers the contraction does not matter.
// A result has rows 4 (l / 16) + i of column l % 16 in lane l.  Two results are a
// fragment of the operand whose contraction runs over their rows, without any exchange
// between lanes, if their rows stand for the indices that tile_row gives.
#ifndef SPARC_MATRIX_H
#define SPARC_MATRIX_H

#include "rows.h"

namespace sparc {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename IO> struct QuadOf;  // four values
template <> struct QuadOf<bf16> { typedef s16x4 T; };
template <> struct QuadOf<float> { typedef f32x4 T; };
template <typename IO> using Quad = typename QuadOf<IO>::T;
template <typename IO> struct alignas(16) Frag { Quad<IO> q[2]; };

// c + a b over the 32 indices of the contraction
__device__ __forceinline__ f32x4 mma(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.q[h][i], b.q[h][i], c, 0, 0, 0);
  return c;
}

// Index of the contraction (of 32) that element e of a fragment is, quad = 4 (l / 16)
template <typename IO> __device__ __forceinline__ constexpr int step_of(int quad, int e) {
  return sizeof(IO) == 2 ? 2 * quad + e : 16 * (e / 4) + quad + e % 4;
}
// Index that row quad + r of the i-th result stands for
template <typename IO> __device__ __forceinline__ constexpr int tile_row(int i, int quad, int r) {
  return sizeof(IO) == 2 ? 32 * (i / 2) + 2 * quad + 4 * (i % 2) + r : 16 * i + quad + r;
}

// Rows of COLS values in LDS, longer by some bytes so that a wave's accesses spread over
// the banks: 16 bytes where rows are read along them, 32 where bf16 columns are read
// across them (4 rows of 16 columns then lie in different banks).
template <typename IO, int COLS, bool ACROSS> struct Panel {
  static constexpr int kStride = COLS + (sizeof(IO) == 2 && ACROSS ? 32 : 16) / sizeof(IO);
  static __device__ __forceinline__ int at(int row, int col) { return row * kStride + col; }
};

// Rows row0 + l % 16, the contraction from column col0 on (multiples of 16 and 32)
template <typename L, typename IO> __device__ __forceinline__ Frag<IO> read_rows(const IO* lds, int row0, int col0) {
  const int lane = threadIdx.x & 63, row = row0 + (lane & 15);
  Frag<IO> f;
  if constexpr (sizeof(IO) == 2) {
    f = *reinterpret_cast<const Frag<IO>*>(lds + L::at(row, col0 + 8 * (lane >> 4)));
  } else {
    const IO* p = lds + L::at(row, col0 + 4 * (lane >> 4));
    f.q[0] = *reinterpret_cast<const Quad<IO>*>(p);
    f.q[1] = *reinterpret_cast<const Quad<IO>*>(p + 16);
  }
  return f;
}
// 16 columns, of which lane l gets column_of(l % 16), four at a time in a row; the
// contraction over the rows from row0 on (a multiple of 32)
template <typename L, typename IO, typename F>
__device__ __forceinline__ Frag<IO> gather_columns(const IO* lds, int row0, F&& column_of) {
  const int lane = threadIdx.x & 63;
  Frag<IO> f;
  if constexpr (sizeof(IO) == 2) {
    // 16 lanes exchange a block of 4 rows x 16 columns that they read in quads of a row
    const int row = row0 + 8 * (lane >> 4) + ((lane & 15) >> 2), col = column_of(4 * (lane & 3));
    f.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + L::at(row, col)));
    f.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + L::at(row + 4, col)));
  } else {
    const IO* p = lds + L::at(row0 + 4 * (lane >> 4), column_of(lane & 15));
#pragma unroll
    for (int e = 0; e < 8; ++e) f.q[e / 4][e % 4] = p[(16 * (e / 4) + e % 4) * L::kStride];
  }
  return f;
}
// Columns col0 + l % 16
template <typename L, typename IO> __device__ __forceinline__ Frag<IO> read_columns(const IO* lds, int row0, int col0) {
  return gather_columns<L>(lds, row0, [&](int m) { return col0 + m; });
}
// The columns that the rows of the i-th result stand for
template <typename L, typename IO> __device__ __forceinline__ Frag<IO> read_tile_columns(const IO* lds, int row0, int i) {
  return gather_columns<L>(lds, row0, [&](int m) { return tile_row<IO>(i, m & ~3, m & 3); });
}

// Bytes 2 and 3 of a and b, a's below: both truncated to bf16
__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// fp32 values as a sum of N fragments.  Two parts are rounded to nearest: of a value
// from 1 to 2 the first leaves 2^-8 at most, of which the second leaves 2^-17 (truncated
// they would leave 2^-15, and always on the same side).  Three are truncated, 8 bits
// each, and hold all 24.  (A value that is infinite, or that two parts round to it,
// which takes 3.39e38, becomes NaN for N > 1.)
template <int N> __device__ __forceinline__ void split(const float (&x)[8], Frag<bf16> (&f)[N]) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(x[i]);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t &a = r[2 * i], &b = r[2 * i + 1];
      u[i] = N == 2 ? pack_bf16x2(__uint_as_float(a), __uint_as_float(b)) : upper_halves(a, b);
      if (n + 1 < N) {
        const uint32_t low = N == 2 ? u[i] << 16 : a & 0xffff0000u, high = N == 2 ? u[i] & 0xffff0000u : b & 0xffff0000u;
        a = __float_as_uint(__uint_as_float(a) - __uint_as_float(low));
        b = __float_as_uint(__uint_as_float(b) - __uint_as_float(high));
      }
    }
    __builtin_memcpy(&f[n], u, sizeof(u));
  }
}
template <int N> __device__ __forceinline__ void split(const float (&x)[8], Frag<float> (&f)[N]) {
  static_assert(N == 1, "fp32 holds all bits");
#pragma unroll
  for (int i = 0; i < 8; ++i) f[0].q[i / 4][i % 4] = x[i];
}
__device__ __forceinline__ float widen(bf16 x) { return bf16_bits_to_float(x.bits); }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ void widen(const Frag<bf16>& f, float (&x)[8]) {
  uint32_t u[4];
  __builtin_memcpy(u, &f, sizeof(u));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen(const Frag<float>& f, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = f.q[i / 4][i % 4];
}

// Whether a value of the fragments that top has seen is infinite or no number: the
// largest exponent is kept, of bf16 two at a time
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t see(uint32_t top, const Frag<bf16>& f) {
  uint32_t u[4];
  __builtin_memcpy(u, &f, sizeof(u));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                 __builtin_bit_cast(u16x2, u[i] & 0x7fff7fffu)));
  return top;
}
__device__ __forceinline__ uint32_t see(uint32_t top, const Frag<float>& f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(f.q[i / 4][i % 4]) & 0x7fffffffu;
    top = top > u ? top : u;
  }
  return top;
}
template <typename IO> __device__ __forceinline__ bool is_odd(uint32_t top) {
  return sizeof(IO) == 4 ? top >= 0x7f800000u : (top & 0xffffu) >= 0x7f80u || top >= 0x7f800000u;
}

// n (at most 4) values to p, rounded to OUT
template <typename OUT> __device__ __forceinline__ void store_quad(OUT* p, int n, f32x4 v) {
  if constexpr (sizeof(OUT) == 4) {
    typedef f32x4 loose __attribute__((aligned(4)));
    if (n >= 4) {
      *reinterpret_cast<loose*>(p) = v;
      return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) p[i] = v[i];
  } else {
    typedef uint32_t loose __attribute__((ext_vector_type(2), aligned(2)));
    const uint32_t lo = pack_bf16x2(v[0], v[1]), hi = pack_bf16x2(v[2], v[3]);
    if (n >= 4) {
      *reinterpret_cast<loose*>(p) = loose{lo, hi};
      return;
    }
    if (n > 0) p[0].bits = static_cast<uint16_t>(lo);
    if (n > 1) p[1].bits = static_cast<uint16_t>(lo >> 16);
    if (n > 2) p[2].bits = static_cast<uint16_t>(hi);
  }
}

// n (at most 4) values from p, the others zero
template <typename IN> __device__ __forceinline__ f32x4 load_quad(const IN* p, int n) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n >= 4) {
    if constexpr (sizeof(IN) == 4) {
      typedef f32x4 loose __attribute__((aligned(4)));
      v = *reinterpret_cast<const loose*>(p);
    } else {
      typedef uint32_t loose __attribute__((ext_vector_type(2), aligned(2)));
      const loose u = *reinterpret_cast<const loose*>(p);
      v = f32x4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
                __uint_as_float(u[1] & 0xffff0000u)};
    }
    return v;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) v[i] = widen(p[i]);
  return v;
}

}  // namespace
}  // namespace sparc

#endif  // SPARC_MATRIX_H
