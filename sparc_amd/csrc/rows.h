// Helpers of the row operators (layer norm, embedding, gradient norm, beam
// search): 16-byte accesses at any alignment, sums over the waves of a row,
// and the host side's error texts.
#ifndef SPARC_ROWS_H
#define SPARC_ROWS_H

#include <type_traits>

#include "common.h"
#include "sparc_hip.h"

namespace sparc {
namespace {

// Values of type IO in 16 bytes
template <typename IO> constexpr int kVec = 16 / sizeof(IO);
template <typename IO> using Vec = typename Raw<IO, kVec<IO>>::T;

// The kVec values from base[index] on, at any alignment of the values (global
// memory is in unaligned access mode: one 16-byte instruction).  Where fewer
// than kVec are left (n), the others are zero and are not read.
template <typename IO> struct Loose;  // 16 bytes at the alignment of a value
template <> struct Loose<float> { typedef uint32_t T __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Loose<bf16> { typedef uint32_t T __attribute__((ext_vector_type(4), aligned(2))); };

// STREAM: non-temporal, for values that a launch reads once and nothing else
// will soon.
template <typename IO, bool STREAM = false>
__device__ __forceinline__ Vec<IO> load_vec(const void* base, int64_t index, int n) {
  Vec<IO> r;
  const IO* p = static_cast<const IO*>(base) + index;
  if (n >= kVec<IO>) {
    const auto* v = reinterpret_cast<const typename Loose<IO>::T*>(p);
    typename Loose<IO>::T u;
    if constexpr (STREAM) u = __builtin_nontemporal_load(v);
    else u = *v;
    __builtin_memcpy(&r, &u, sizeof(r));
  } else {
    IO e[kVec<IO>] = {};
#pragma unroll
    for (int i = 0; i < kVec<IO> - 1; ++i)
      if (i < n) e[i] = p[i];
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <typename IO, bool STREAM = false>
__device__ __forceinline__ void store_vec(void* base, int64_t index, int n, const Vec<IO>& r) {
  IO* p = static_cast<IO*>(base) + index;
  if (n >= kVec<IO>) {
    typename Loose<IO>::T u;
    __builtin_memcpy(&u, &r, sizeof(r));
    auto* v = reinterpret_cast<typename Loose<IO>::T*>(p);
    if constexpr (STREAM) __builtin_nontemporal_store(u, v);
    else *v = u;
  } else {
    IO e[kVec<IO>];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < kVec<IO> - 1; ++i)
      if (i < n) p[i] = e[i];
  }
}
// N values of any type T into fp32, those past n zero
template <typename T, int N>
__device__ __forceinline__ void load_f32(const void* base, int64_t index, int n, float (&o)[N]) {
  constexpr int V = kVec<T> < N ? kVec<T> : N;
  static_assert(V == kVec<T>, "whole vectors");
#pragma unroll
  for (int k = 0; k < N; k += V) {
    float f[V];
    unpack<T, V>(load_vec<T>(base, index + k, n - k), f);
#pragma unroll
    for (int i = 0; i < V; ++i) o[k + i] = f[i];
  }
}

template <int N> using Int = std::integral_constant<int, N>;

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
inline sparc_status op_fail(sparc_status s, const char* msg) {
  snprintf(error_buffer(), 512, "%s", msg);
  return s;
}
inline sparc_status op_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return SPARC_OK;
  snprintf(error_buffer(), 512, "%s: %s", what, hipGetErrorString(e));
  return SPARC_EHIP;
}
inline size_t up256(size_t b) { return (b + 255) / 256 * 256; }
// Workgroups of a launch whose workgroups loop: at most 2^20 (a launch holds
// less than 2^32 threads per dimension)
inline unsigned op_grid(int64_t groups) {
  return static_cast<unsigned>(groups < 1 ? 1 : (groups < (1 << 20) ? groups : (1 << 20)));
}

}  // namespace
}  // namespace sparc

#endif  // SPARC_ROWS_H
