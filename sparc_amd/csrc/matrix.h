// Operands of the matrix instructions (16x16 results in fp32), for fp32 and bf16
// values in one form.
//
// A fragment holds, for lane l of a wave, the eight values at 32 consecutive indices
// of the contraction that lie at 16 h + 4 (l / 16) + i (h < 2, i < 4) of row (or
// column) l % 16.  Both operands of a product are held in this order, so the order in
// which the instruction itself numbers the contraction does not matter.  A result has
// rows 4 (l / 16) + i of column l % 16 in lane l: two results, one above the other,
// are a fragment of the operand whose contraction runs over their rows, without any
// exchange between lanes.
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
template <typename IO> struct Frag { Quad<IO> q[2]; };

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

// Rows row0 + l % 16 of an LDS array whose rows lie ``stride`` values apart (a multiple
// of a quad), the contraction from column col0 on
template <typename IO> __device__ __forceinline__ Frag<IO> read_rows(const IO* lds, int stride, int row0, int col0) {
  const int lane = threadIdx.x & 63;
  const IO* p = lds + (row0 + (lane & 15)) * stride + col0 + 4 * (lane >> 4);
  Frag<IO> f;
  f.q[0] = *reinterpret_cast<const Quad<IO>*>(p);
  f.q[1] = *reinterpret_cast<const Quad<IO>*>(p + 16);
  return f;
}
// Columns col0 + l % 16, the contraction over the rows from row0 on
__device__ __forceinline__ Frag<bf16> read_columns(const bf16* lds, int stride, int row0, int col0) {
  const int lane = threadIdx.x & 63;
  // 16 lanes exchange a block of 4 rows x 16 columns that they read in quads of a row
  const bf16* p = lds + (row0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * stride + col0 + 4 * (lane & 3);
  Frag<bf16> f;
  f.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
  f.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * stride));
  return f;
}
__device__ __forceinline__ Frag<float> read_columns(const float* lds, int stride, int row0, int col0) {
  const int lane = threadIdx.x & 63;
  const float* p = lds + (row0 + 4 * (lane >> 4)) * stride + col0 + (lane & 15);
  Frag<float> f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[h][i] = p[(16 * h + i) * stride];
  return f;
}

// fp32 values as a sum of N fragments: N bf16 values hold 8 N bits of each (a value
// that is not finite becomes NaN for N > 1)
template <int N> __device__ __forceinline__ void split(const float (&x)[8], Frag<bf16> (&f)[N]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      if (n + 1 < N) {
        r[2 * i] -= __uint_as_float(u[i] << 16);
        r[2 * i + 1] -= __uint_as_float(u[i] & 0xffff0000u);
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

// Bits that are set where a value is infinite or no number
__device__ __forceinline__ uint32_t odd_bits(const Frag<bf16>& f) {
  uint32_t u[4], odd = 0;
  __builtin_memcpy(u, &f, sizeof(u));
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= ((u[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  return odd;
}
__device__ __forceinline__ uint32_t odd_bits(const Frag<float>& f) {
  uint32_t odd = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) odd |= ((__float_as_uint(f.q[i / 4][i % 4]) & 0x7f800000u) + 0x00800000u) & 0x80000000u;
  return odd;
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

}  // namespace
}  // namespace sparc

#endif  // SPARC_MATRIX_H
