// Layer norm over the rows of a [rows, cols] matrix, with its gradients:
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xhat = (x - mu) rstd,
//   y = xhat w + b
//   g = dy w,  dx = rstd (g - mean(g) - xhat mean(g xhat)),
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
// in fp32 arithmetic: x, y, dy, dx in the I/O type, w, b, dw, db in the
// parameter type (the I/O type, or fp32 beside bf16 I/O), each output rounded
// once.  The mean is taken about the row's first value, and the mean difference from
// it is corrected by what is left of the differences, beside the sum of their squares:
// a sum of the values themselves would be off by some units of a large mean, which a
// nearly constant row's variance does not outweigh.  What remains of a mean that is
// large beside the deviations is its own rounding to fp32.
//
// A row is held in registers by the L lanes that own it, 8 to 64 of a wave or a
// workgroup of 256 to 1024, each NCH vectors of 16 bytes, at any alignment.  Rows
// too wide for that are read again for each pass over them (the *_wide kernels).
// The backward keeps the columns' sums of dy xhat and dy in registers over the
// rows that its waves walk, beside the weight (in LDS for the widest rows, whose
// registers are full), reads the next row while it works on one, and writes one
// partial row per workgroup; a second kernel adds the partial rows in a fixed
// order, so the parameters' gradients do not depend on timing.

#include "rows.h"

namespace sparc {
namespace {

constexpr int kRowWaves = 4;       // forward, up to a wave per row: waves per workgroup (1 with few rows)
constexpr int kBwdRowWaves = 8;    // backward, up to a wave per row: waves per workgroup
template <int L> constexpr int kBwdRows = L <= 64 ? kBwdRowWaves * 64 / L : 1;
constexpr int64_t kFewRows = 1024; // below this a forward workgroup is one wave or one row: one per CU before two

// columns from c on, as load_vec counts them
__device__ __forceinline__ int left(int64_t D, int64_t c) {
  return static_cast<int>(D - c < 64 ? D - c : 64);
}

// How a row of D columns ends in vectors of V:
//   kWhole  D is a multiple of V
//   kLap    the last vector ends with the row and repeats some columns of the one
//           before it, which count once in a sum over the row; both lanes come to
//           the same values for them and store them both (D >= V)
//   kShort  the last vector is short.  The branches of a short access make every
//           load wait for the one before it, so all rows but the array's last ones
//           read it whole, with values of the next row behind the end.
enum Ends { kWhole, kLap, kShort };

// The columns of vector k of a lane's NCH; those before kLast are whole, as the
// forms are chosen.
template <int NCH> constexpr int kLast = NCH <= 4 ? NCH - 1 : NCH - 2;
template <int V, int NCH, int L, int E>
struct Columns {
  bool any;      // whether the row reaches the vector
  int at, n;     // its first column and how many it has
  int twice;     // of them repeated

  __device__ __forceinline__ Columns(int k, int t, int D) {
    const int c = (k * L + t) * V;
    const bool last = k >= kLast<NCH>;
    any = c < D;  // a branch for every vector, which keeps the registers of one from the next's
    at = E == kLap && last && c > D - V ? D - V : c;
    n = E == kShort && last && D - c < V ? D - c : V;
    twice = c - at;
  }
  // value i of the vector in a sum over the row
  __device__ __forceinline__ float once(int i, float v) const {
    if constexpr (E == kLap) return i < twice ? 0.0f : v;
    if constexpr (E == kShort) return i < n ? v : 0.0f;
    return v;
  }
};
__device__ __forceinline__ bool reads_whole(int64_t row, int64_t R, int D, int v) {
  return (row + 1) * D + v - 1 <= R * D;
}
// zeros behind the first n values
template <typename IO>
__device__ __forceinline__ void keep_first(Vec<IO>& raw, int n) {
  float v[kVec<IO>];
  unpack<IO, kVec<IO>>(raw, v);
#pragma unroll
  for (int i = 0; i < kVec<IO>; ++i) v[i] = i < n ? v[i] : 0.0f;
  raw = pack<IO, kVec<IO>>(v);
}

// Sums of N values over the L lanes that share a row, in each of them.  With
// W waves, red: two buffers used in turn (``turn``), so that one barrier per
// call is enough.
template <int L> constexpr int kWaves = L > 64 ? L / 64 : 1;
template <int N, int L, int W = kWaves<L>>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[N][W], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = group_sum(v[i], L < 64 ? L : 64);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[turn][i][wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k) s += red[turn][i][k];
      v[i] = s;
    }
    turn ^= 1;
  }
}

// The mean and 1 / sqrt(variance + eps) of a row from the means of x - about and of its
// square.  (An infinite variance stays so.)
__device__ __forceinline__ void finish_stats(float about, float diff, float square, float eps, float& mean,
                                             float& rstd) {
  mean = about + diff;
  const float shift = diff * diff;
  rstd = 1.0f / sqrtf((shift < square ? square - shift : square) + eps);
}

// The forward, a row per L lanes: one read and one write of each value, and bound
// by them: 32768 x 768 bf16 20 us (50 MB read, 50 written: 5.0 TB/s), 300000 x 64
// 16 us.  Where one workgroup fills a CU its arithmetic is not hidden: 8192 x 24576
// 192 us at best (4.2 TB/s; 180 with a mean that is not taken about the first value,
// smaller rows 1 to 4 % less).  256 rows of 2048 take 3.6 us: the launch, two reads
// one after the other and two sums over the row's lanes.  Rows that begin at odd
// multiples of two bytes cost up to a third more (20000 bf16 rows of 5000 columns 73
// us, of 5001 94), since each access is split.  (kWhole in the forward measured no
// faster than kLap.)
template <typename IO, typename PT, int NCH, int L, int E>
__global__ void __launch_bounds__(L <= 64 ? 64 * kRowWaves : L)
layer_norm_fwd_kernel(int64_t R, int D, const void* x, const void* w, const void* b, float eps, void* y, float* mean,
                      float* rstd) {
  constexpr int V = kVec<IO>;
  __shared__ float red[2][1][kWaves<L>], red2[2][2][kWaves<L>];
  int turn = 0;
  const int t = threadIdx.x & (L - 1), per = L <= 64 ? blockDim.x / L : 1;
  int64_t first = static_cast<int64_t>(blockIdx.x) * per;
  if constexpr (L == 64) first += __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  else if constexpr (L < 64) first += threadIdx.x / L;
  const float inv_d = 1.0f / static_cast<float>(D);
  for (int64_t row = first; row < R; row += static_cast<int64_t>(gridDim.x) * per) {  // uniform over a row's lanes
    const int64_t base = row * D;
    const float first_value = load1<IO>(x, base);
    Vec<IO> raw[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
      if (c.any) raw[k] = load_vec<IO>(x, base + c.at, c.n);
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
      if (c.any) {
        float v[V];
        unpack<IO, V>(raw[k], v);
#pragma unroll
        for (int i = 0; i < V; ++i) s[0] = fmaf(c.once(i, v[i] - first_value), inv_d, s[0]);
      }
    }
    row_sums<1, L>(s, red, turn);
    const float about = first_value + s[0];
    float m[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
      if (c.any) {
        float v[V];
        unpack<IO, V>(raw[k], v);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = c.once(i, v[i] - about);
          m[0] += d;
          m[1] = fmaf(d, d, m[1]);
        }
      }
    }
    row_sums<2, L>(m, red2, turn);
    float mu, r;
    finish_stats(about, m[0] * inv_d, m[1] * inv_d, eps, mu, r);
    if (t == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
      if (c.any) {
        float v[V], o[V];
        unpack<IO, V>(raw[k], v);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (v[i] - mu) * r;
        if (w) {
          float p[V];
          load_f32<PT, V>(w, c.at, c.n, p);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] *= p[i];
        }
        if (b) {
          float p[V];
          load_f32<PT, V>(b, c.at, c.n, p);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] += p[i];
        }
        store_vec<IO>(y, base + c.at, c.n, pack<IO, V>(o));
      }
    }
  }
}

// The backward: x and dy in, dx out, once each, and the partial rows beside them.
// Memory again: 32768 x 768 bf16 31 us (102 MB read, 53 written: 5.0 TB/s), 8192 x
// 24576 228 us (807 and 453: 5.5 TB/s); 3711 x 1001 fp32 13 us, a few rows per
// wave, whose start and end count.
template <typename IO, typename PT, int NCH, int L, int E>
__global__ void __launch_bounds__(L <= 64 ? 64 * kBwdRowWaves : L)
layer_norm_bwd_kernel(int64_t R, int D, const void* x, const void* w, const float* mean, const float* rstd,
                      const void* dy, void* dx, float* dw_part, float* db_part) {
  constexpr int V = kVec<IO>;
  constexpr int W = kWaves<L>;
  constexpr int kRows = kBwdRows<L>;                // rows a workgroup works on at once
  constexpr int NP = V / kVec<PT>;                  // parameter vectors per vector of a row
  constexpr bool kWeightInLds = W == 16;
  // the next row into registers of its own while this one is worked on; with
  // more than 16 columns per lane there are none left for it, and each vector
  // of the next row is read once this row's is done with
  constexpr bool kAhead = NCH * V <= 16;
  __shared__ float red[2][2][W];
  __shared__ Vec<PT> w_lds[kWeightInLds ? NCH * L * NP : 1];
  int turn = 0;
  const int t = threadIdx.x & (L - 1), lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  Vec<IO> xr[NCH], dr[NCH];
  Vec<PT> wr[kWeightInLds ? 1 : NCH][NP];
  float aw[NCH][V], ab[NCH][V];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const Columns<V, NCH, L, E> c(k, t, D);
#pragma unroll
    for (int i = 0; i < V; ++i) { aw[k][i] = 0.0f; ab[k][i] = 0.0f; }
#pragma unroll
    for (int q = 0; q < NP; ++q) {  // without a weight: ones
      float ones[kVec<PT>];
#pragma unroll
      for (int i = 0; i < kVec<PT>; ++i) ones[i] = 1.0f;
      Vec<PT> p = pack<PT, kVec<PT>>(ones);
      if (w && c.any) p = load_vec<PT>(w, c.at + q * kVec<PT>, c.n - q * kVec<PT>);
      if constexpr (kWeightInLds) w_lds[(k * L + t) * NP + q] = p;  // read back by this thread only
      else wr[k][q] = p;
    }
  }
  const auto weight = [&](int k, float (&p)[V]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      float f[kVec<PT>];
      if constexpr (kWeightInLds) unpack<PT, kVec<PT>>(w_lds[(k * L + t) * NP + q], f);
      else unpack<PT, kVec<PT>>(wr[k][q], f);
#pragma unroll
      for (int i = 0; i < kVec<PT>; ++i) p[q * kVec<PT> + i] = f[i];
    }
  };
  const float inv_d = 1.0f / static_cast<float>(D);
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows;
  if constexpr (L == 64) row += wave;
  else if constexpr (L < 64) row += threadIdx.x / L;
  const auto load_row = [&](int64_t at, Vec<IO> (&xo)[NCH], Vec<IO> (&dyo)[NCH]) __attribute__((always_inline)) {
    if (E != kShort || reads_whole(at, R, D, V)) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const Columns<V, NCH, L, E> c(k, t, D);
        if (c.any) {
          xo[k] = load_vec<IO>(x, at * D + c.at, V);
          dyo[k] = load_vec<IO>(dy, at * D + c.at, V);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const Columns<V, NCH, L, E> c(k, t, D);
        if (c.any) {
          xo[k] = load_vec<IO>(x, at * D + c.at, c.n);
          dyo[k] = load_vec<IO>(dy, at * D + c.at, c.n);
        }
      }
    }
  };
  if (row < R) load_row(row, xr, dr);
  for (; row < R; row += step) {  // uniform over a row's lanes
    Vec<IO> xn[kAhead ? NCH : 1], dn[kAhead ? NCH : 1];
    if constexpr (kAhead) {
      if (row + step < R) load_row(row + step, xn, dn);
    }
    const float mu = mean[row], r = rstd[row];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
      if (c.any) {
        if (E == kShort && c.n < V) {
          keep_first<IO>(xr[k], c.n);
          keep_first<IO>(dr[k], c.n);
        }
        float xv[V], dv[V], p[V];
        unpack<IO, V>(xr[k], xv);
        unpack<IO, V>(dr[k], dv);
        weight(k, p);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // xhat too is 0 behind a short row's end: 0 - mu may overflow times r
          const float xh = E == kShort && i >= c.n ? 0.0f : (xv[i] - mu) * r, g = c.once(i, dv[i] * p[i]);
          s[0] += g;
          s[1] = fmaf(g, xh, s[1]);
          aw[k][i] = fmaf(dv[i], xh, aw[k][i]);
          ab[k][i] += dv[i];
        }
      }
    }
    row_sums<2, L>(s, red, turn);
    const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
      if (c.any) {
        if (dx) {
          float xv[V], dv[V], p[V], o[V];
          unpack<IO, V>(xr[k], xv);
          unpack<IO, V>(dr[k], dv);
          weight(k, p);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float xh = (xv[i] - mu) * r;
            o[i] = r * (fmaf(-xh, m1, dv[i] * p[i]) - m0);
          }
          store_vec<IO>(dx, row * D + c.at, c.n, pack<IO, V>(o));
        }
        if constexpr (kAhead) {
          xr[k] = xn[k];
          dr[k] = dn[k];
        } else if (E != kShort ? row + step < R : reads_whole(row + step, R, D, V)) {
          xr[k] = load_vec<IO>(x, (row + step) * D + c.at, V);
          dr[k] = load_vec<IO>(dy, (row + step) * D + c.at, V);
        } else if (E == kShort && row + step < R) {
          xr[k] = load_vec<IO>(x, (row + step) * D + c.at, c.n);
          dr[k] = load_vec<IO>(dy, (row + step) * D + c.at, c.n);
        }
      }
    }
  }
  // one partial row per workgroup; where it has several rows in hand, their sums
  // are added first, those of a wave and then wave 0, 1, 2, ...
  __shared__ float4 lds[W == 1 ? kBwdRowWaves - 1 : 1][V / 4][64];
  const auto write = [&](float (&a)[NCH][V], float* part) __attribute__((always_inline)) {
    const int64_t out = static_cast<int64_t>(blockIdx.x) * D;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const Columns<V, NCH, L, E> c(k, t, D);
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
#pragma unroll
        for (int o = L; o < 64; o <<= 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) a[k][4 * q + i] += __shfl_xor(a[k][4 * q + i], o);
        }
        float4 u = make_float4(a[k][4 * q], a[k][4 * q + 1], a[k][4 * q + 2], a[k][4 * q + 3]);
        if constexpr (W == 1) {
          if (wave > 0) lds[wave - 1][q][lane] = u;
          __syncthreads();
          if (wave == 0) {
            for (int v = 0; v < kBwdRowWaves - 1; ++v) {
              const float4 o = lds[v][q][lane];
              u.x += o.x; u.y += o.y; u.z += o.z; u.w += o.w;
            }
          }
          __syncthreads();
        }
        if ((W > 1 || (wave == 0 && lane < L)) && c.any)
          store_vec<float>(part, out + c.at + 4 * q, c.n - 4 * q, u);
      }
    }
  };
  if (dw_part) write(aw, dw_part);
  if (db_part) write(ab, db_part);
}

// Rows of any width, read again for each pass over them, mostly out of a cache:
// 3172 x 40000 fp32 forward 302 us (1 GB: 3.4 TB/s); backward of 6009 x 16641 fp32
// 291 us for dx and 157 for the sums over rows, which read x and dy once more.
constexpr int kWideThreads = 1024;
template <typename IO, typename PT>
__global__ void __launch_bounds__(kWideThreads)
layer_norm_fwd_wide_kernel(int64_t R, int64_t D, const void* x, const void* w, const void* b, float eps, void* y,
                           float* mean, float* rstd) {
  constexpr int V = kVec<IO>;
  __shared__ float red[2][1][kWaves<kWideThreads>], red2[2][2][kWaves<kWideThreads>];
  int turn = 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  const int64_t c0 = static_cast<int64_t>(threadIdx.x) * V;
  for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
    const int64_t base = row * D;
    const float first_value = load1<IO>(x, base);
    float s[1] = {0.0f}, v[V];
    for (int64_t c = c0; c < D; c += kWideThreads * V) {
      const int n = left(D, c);
      unpack<IO, V>(load_vec<IO>(x, base + c, n), v);
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] = fmaf(i < n ? v[i] - first_value : 0.0f, inv_d, s[0]);
    }
    row_sums<1, kWideThreads>(s, red, turn);
    const float about = first_value + s[0];
    float m[2] = {0.0f, 0.0f};
    for (int64_t c = c0; c < D; c += kWideThreads * V) {
      const int n = left(D, c);
      unpack<IO, V>(load_vec<IO>(x, base + c, n), v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = i < n ? v[i] - about : 0.0f;
        m[0] += d;
        m[1] = fmaf(d, d, m[1]);
      }
    }
    row_sums<2, kWideThreads>(m, red2, turn);
    float mu, r;
    finish_stats(about, m[0] * inv_d, m[1] * inv_d, eps, mu, r);
    if (threadIdx.x == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
    for (int64_t c = c0; c < D; c += kWideThreads * V) {
      const int n = left(D, c);
      float p[V], q[V];
      unpack<IO, V>(load_vec<IO>(x, base + c, n), v);
      if (w) load_f32<PT, V>(w, c, n, p);
      if (b) load_f32<PT, V>(b, c, n, q);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = (v[i] - mu) * r;
        if (w) v[i] *= p[i];
        if (b) v[i] += q[i];
      }
      store_vec<IO>(y, base + c, n, pack<IO, V>(v));
    }
  }
}
template <typename IO, typename PT>
__global__ void __launch_bounds__(kWideThreads)
layer_norm_dx_wide_kernel(int64_t R, int64_t D, const void* x, const void* w, const float* mean, const float* rstd,
                          const void* dy, void* dx) {
  constexpr int V = kVec<IO>;
  __shared__ float red[2][2][kWaves<kWideThreads>];
  int turn = 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  const int64_t c0 = static_cast<int64_t>(threadIdx.x) * V;
  for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
    const int64_t base = row * D;
    const float mu = mean[row], r = rstd[row];
    float s[2] = {0.0f, 0.0f}, g[V], xh[V];
    // g and xhat of the columns from c on, 0 behind the row
    const auto load = [&](int64_t c, int n) __attribute__((always_inline)) {
      unpack<IO, V>(load_vec<IO>(dy, base + c, n), g);
      unpack<IO, V>(load_vec<IO>(x, base + c, n), xh);
      float p[V];
      if (w) load_f32<PT, V>(w, c, n, p);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (w) g[i] *= p[i];
        xh[i] = i < n ? (xh[i] - mu) * r : 0.0f;
      }
    };
    for (int64_t c = c0; c < D; c += kWideThreads * V) {
      load(c, left(D, c));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[0] += g[i];
        s[1] = fmaf(g[i], xh[i], s[1]);
      }
    }
    row_sums<2, kWideThreads>(s, red, turn);
    const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
    for (int64_t c = c0; c < D; c += kWideThreads * V) {
      const int n = left(D, c);
      load(c, n);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = r * (fmaf(-xh[i], m1, g[i]) - m0);
      store_vec<IO>(dx, base + c, n, pack<IO, V>(g));
    }
  }
}
// partial column sums of dy xhat and dy over the rows blockIdx.y, + gridDim.y, ...
template <typename IO>
__global__ void __launch_bounds__(256)
layer_norm_params_wide_kernel(int64_t R, int64_t D, const void* x, const float* mean, const float* rstd,
                              const void* dy, float* dw_part, float* db_part) {
  constexpr int V = kVec<IO>;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * V;
  if (c >= D) return;
  const int n = left(D, c);
  float aw[V], ab[V];
#pragma unroll
  for (int i = 0; i < V; ++i) { aw[i] = 0.0f; ab[i] = 0.0f; }
  for (int64_t row = blockIdx.y; row < R; row += gridDim.y) {
    float d[V], v[V];
    unpack<IO, V>(load_vec<IO>(dy, row * D + c, n), d);
    unpack<IO, V>(load_vec<IO>(x, row * D + c, n), v);
    const float mu = mean[row], r = rstd[row];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      aw[i] = fmaf(d[i], (v[i] - mu) * r, aw[i]);
      ab[i] += d[i];
    }
  }
#pragma unroll
  for (int q = 0; q < V; q += 4) {
    const int64_t at = blockIdx.y * D + c + q;
    if (dw_part) store_vec<float>(dw_part, at, n - q, make_float4(aw[q], aw[q + 1], aw[q + 2], aw[q + 3]));
    if (db_part) store_vec<float>(db_part, at, n - q, make_float4(ab[q], ab[q + 1], ab[q + 2], ab[q + 3]));
  }
}

// out[c] = sum over the n partial rows: CW columns by 1024 / CW slices of rows
// per workgroup, the slices added in order.  blockIdx.y: dw, db.  4 us for 512
// partial rows of 768 (a launch), 10 us for 256 of 24576 (50 MB).
template <typename PT, int CW>
__global__ void __launch_bounds__(1024)
layer_norm_reduce_kernel(int n, int64_t D, const float* dw_part, const float* db_part, void* dw, void* db) {
  constexpr int S = 1024 / CW;
  __shared__ float red[S][CW];
  const float* part = blockIdx.y ? db_part : dw_part;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;  // uniform over the workgroup
  const int cl = threadIdx.x & (CW - 1), slice = threadIdx.x / CW;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * CW + cl;
  float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < D) {
    int r = slice;
    for (; r + 3 * S < n; r += 4 * S) {
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] += part[(r + k * S) * D + c];
    }
    for (; r < n; r += S) a[0] += part[r * D + c];
  }
  red[slice][cl] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
#pragma unroll
  for (int h = S / 2; h > 0; h >>= 1) {
    if (slice < h) red[slice][cl] += red[slice + h][cl];
    __syncthreads();
  }
  if (slice == 0 && c < D) store1<PT>(out, c, red[0][cl]);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// f(NCH, L) for the narrowest form that holds a row of D columns in registers, L
// lanes with NCH vectors each, so that few lanes idle and as few waves as can
// hold a row wait for one another (a wave per row: 88 us instead of 30 for
// 300000 x 120 bf16; 1024 lanes with one vector each: 129 instead of 75 for
// 20000 x 5000).  With few rows a lane's chain of vectors is what takes time: one
// vector each up to 1024 lanes (4 x 2048 bf16: 2.7 us, 4 vectors in one wave 3.5).
// False: wider than that.
template <typename IO, typename F>
bool fwd_form(int64_t R, int64_t D, F&& f) {
  const int64_t vecs = (D + kVec<IO> - 1) / kVec<IO>;
  if (R < kFewRows && vecs > 64 && vecs <= 256) return f(Int<1>{}, Int<256>{}), true;
  if (R < kFewRows && vecs > 512 && vecs <= 1024) return f(Int<1>{}, Int<1024>{}), true;
  if (vecs <= 8) return f(Int<1>{}, Int<8>{}), true;
  if (vecs <= 16) return f(Int<1>{}, Int<16>{}), true;
  if (vecs <= 32) return f(Int<1>{}, Int<32>{}), true;
  if (vecs <= 64) return f(Int<1>{}, Int<64>{}), true;
  if (vecs <= 96) return f(Int<3>{}, Int<32>{}), true;
  if (vecs <= 128) return f(Int<2>{}, Int<64>{}), true;
  if (vecs <= 192) return f(Int<3>{}, Int<64>{}), true;
  if (vecs <= 256) return f(Int<4>{}, Int<64>{}), true;
  if (vecs <= 512) return f(Int<2>{}, Int<256>{}), true;
  if (vecs <= 768) return f(Int<3>{}, Int<256>{}), true;
  if (vecs <= 1024) return f(Int<4>{}, Int<256>{}), true;
  if (vecs <= 1536) return f(Int<3>{}, Int<512>{}), true;
  if (vecs <= 2048) return f(Int<2>{}, Int<1024>{}), true;
  if (vecs <= 3 * 1024) return f(Int<3>{}, Int<1024>{}), true;
  if (vecs <= 4096) return f(Int<4>{}, Int<1024>{}), true;
  if (vecs <= 6 * 1024) return f(Int<6>{}, Int<1024>{}), true;
  if constexpr (sizeof(IO) == 4) {  // bf16: too many registers
    if (vecs <= 8 * 1024) return f(Int<8>{}, Int<1024>{}), true;
  }
  return false;
}
// The backward holds two fp32 sums per column beside two rows of x and dy: up to
// 16 columns per lane, 32 (16 in fp32) with 1024 lanes.
template <typename IO, typename F>
bool bwd_form(int64_t D, F&& f) {
  const int64_t vecs = (D + kVec<IO> - 1) / kVec<IO>;
  if (vecs <= 8) return f(Int<1>{}, Int<8>{}), true;
  if (vecs <= 16) return f(Int<1>{}, Int<16>{}), true;
  if (vecs <= 32) return f(Int<1>{}, Int<32>{}), true;
  if (vecs <= 64) return f(Int<1>{}, Int<64>{}), true;
  if constexpr (sizeof(IO) == 4) {
    if (vecs <= 96) return f(Int<3>{}, Int<32>{}), true;
  }
  if (vecs <= 128) return f(Int<2>{}, Int<64>{}), true;
  if constexpr (sizeof(IO) == 4) {
    if (vecs <= 192) return f(Int<3>{}, Int<64>{}), true;
    if (vecs <= 256) return f(Int<4>{}, Int<64>{}), true;
  }
  if constexpr (sizeof(IO) == 2) {
    if (vecs <= 256) return f(Int<1>{}, Int<256>{}), true;
  }
  if (vecs <= 512) return f(Int<2>{}, Int<256>{}), true;
  if constexpr (sizeof(IO) == 4) {
    if (vecs <= 768) return f(Int<3>{}, Int<256>{}), true;
    if (vecs <= 1024) return f(Int<4>{}, Int<256>{}), true;
  } else {
    if (vecs <= 1024) return f(Int<1>{}, Int<1024>{}), true;
  }
  if (vecs <= 2048) return f(Int<2>{}, Int<1024>{}), true;
  if (vecs <= 3 * 1024) return f(Int<3>{}, Int<1024>{}), true;
  if (vecs <= 4096) return f(Int<4>{}, Int<1024>{}), true;
  return false;
}

// Workgroups of the backward = partial rows: never more than rows need, and
// enough to fill the GPU: 256 CUs of 16 waves at its registers, of 8 with 4
// vectors per lane, which keep as much in flight (8192 x 1000 fp32: 21 against
// 25 us; 32768 x 768 bf16, 2 vectors: 41 against 31).  With a workgroup per row,
// a partial row costs as much as a row: 2 of these at least for each, and 8
// behind the first 512 (944 x 2827 bf16 with the sum of the partial rows: 19
// against 24 us, 4096 x 2880: 24 against 26).
template <int NCH, int L>
int64_t bwd_groups(int64_t R) {
  const int64_t need = L <= 64 ? (R + kBwdRows<L> - 1) / kBwdRows<L> : (R + 1) / 2;
  const int64_t fill = 256 * (NCH >= 4 && L < 1024 ? 8 : 16) / (L <= 64 ? kBwdRowWaves : kWaves<L>);
  int64_t n = need < fill ? need : fill;
  if (L > 64 && n > 512) n = R / 8 > 512 ? (R / 8 < n ? R / 8 : n) : 512;
  return n;
}
// How rows of other widths than whole vectors end: with vectors that lap (20000 x
// 5004 bf16, fp32 parameters 141 us, short ones 201; 300000 x 68 33 and 40; 60000 x
// 701 57 and 73), but for 4 vectors in each of 1024 lanes, which have no registers
// left for it (3944 x 25353: 224 and 178).
template <int NCH, int L>
constexpr int bwd_ends() {
  return NCH >= 4 && L == 1024 ? kShort : kLap;
}
constexpr int64_t kWideSlices = 64;
// The most partial rows that a backward of rows of D columns leaves
template <typename IO>
int64_t most_partials(int64_t D) {
  int64_t n = kWideSlices;
  bwd_form<IO>(D, [&](auto NCH, auto L) { n = bwd_groups<NCH(), L()>(INT32_MAX); });
  return n;
}

template <typename PT>
void launch_reduce(hipStream_t st, int64_t n, int64_t D, const float* dw_part, const float* db_part, void* dw,
                   void* db) {
  // few columns: 16 of them per workgroup, so that more workgroups share the rows;
  // many: 64, whole lines
  if (D < 8192)
    hipLaunchKernelGGL((layer_norm_reduce_kernel<PT, 16>), dim3(static_cast<unsigned>((D + 15) / 16), 2), dim3(1024), 0,
                       st, static_cast<int>(n), D, dw_part, db_part, dw, db);
  else
    hipLaunchKernelGGL((layer_norm_reduce_kernel<PT, 64>), dim3(static_cast<unsigned>((D + 63) / 64), 2), dim3(1024), 0,
                       st, static_cast<int>(n), D, dw_part, db_part, dw, db);
}

sparc_status ln_check(int64_t rows, int64_t cols, int32_t io, int32_t pt) {
  if (rows < 0 || cols <= 0) return op_fail(SPARC_EINVAL, "layer norm: rows >= 0 and cols > 0 required");
  if (io != SPARC_F32 && io != SPARC_BF16) return op_fail(SPARC_EINVAL, "layer norm: unknown io_dtype");
  if (pt != SPARC_F32 && pt != io)
    return op_fail(SPARC_EINVAL, "layer norm: parameters are in the I/O type, or fp32 beside bf16 I/O");
  if (rows > INT32_MAX || cols > (int64_t(1) << 28) || rows > (int64_t(1) << 46) / cols)
    return op_fail(SPARC_EINVAL, "layer norm: too large");
  return SPARC_OK;
}

template <typename IO, typename PT>
sparc_status ln_forward(hipStream_t st, int64_t R, int64_t D, const void* x, const void* w, const void* b, float eps,
                        void* y, float* mean, float* rstd) {
  const bool held = fwd_form<IO>(R, D, [&](auto NCH, auto L) {
    const int threads = L() > 64 ? L() : (R < kFewRows ? 64 : 64 * kRowWaves), per = threads / L();
    const dim3 grid(op_grid((R + per - 1) / per)), block(threads);
    const auto launch = [&](auto E) {
      hipLaunchKernelGGL((layer_norm_fwd_kernel<IO, PT, NCH(), L(), E()>), grid, block, 0, st, R, static_cast<int>(D),
                         x, w, b, eps, y, mean, rstd);
    };
    if constexpr (L() == 8) {
      if (D < kVec<IO>) return launch(Int<kShort>{});
    }
    launch(Int<kLap>{});
  });
  if (!held)
    hipLaunchKernelGGL((layer_norm_fwd_wide_kernel<IO, PT>), dim3(op_grid(R)), dim3(kWideThreads), 0, st, R, D, x, w, b,
                       eps, y, mean, rstd);
  return op_launched("layer norm forward");
}

template <typename IO, typename PT>
sparc_status ln_backward(hipStream_t st, int64_t R, int64_t D, const void* x, const void* w, const float* mean,
                         const float* rstd, const void* dy, void* dx, void* dw, void* db, float* ws) {
  float* dw_part = dw ? ws : nullptr;
  float* db_part = db ? ws : nullptr;  // behind dw's partial rows where there are any
  int64_t n = 0;
  const bool held = bwd_form<IO>(D, [&](auto NCH, auto L) {
    n = bwd_groups<NCH(), L()>(R);
    if (dw && db) db_part = ws + n * D;
    const dim3 grid(static_cast<unsigned>(n)), block(L() > 64 ? L() : 64 * kBwdRowWaves);
    const auto launch = [&](auto E) {
      hipLaunchKernelGGL((layer_norm_bwd_kernel<IO, PT, NCH(), L(), E()>), grid, block, 0, st, R, static_cast<int>(D),
                         x, w, mean, rstd, dy, dx, dw_part, db_part);
    };
    if constexpr (L() == 8) {
      if (D < kVec<IO>) return launch(Int<kShort>{});
    }
    if (D % kVec<IO> == 0) return launch(Int<kWhole>{});
    launch(Int<bwd_ends<NCH(), L()>()>{});
  });
  if (!held) {
    if (dx)
      hipLaunchKernelGGL((layer_norm_dx_wide_kernel<IO, PT>), dim3(op_grid(R)), dim3(kWideThreads), 0, st, R, D, x, w,
                         mean, rstd, dy, dx);
    if (dw || db) {
      n = R < kWideSlices ? R : kWideSlices;
      if (dw && db) db_part = ws + n * D;
      hipLaunchKernelGGL((layer_norm_params_wide_kernel<IO>),
                         dim3(static_cast<unsigned>((D - 1) / (256 * kVec<IO>) + 1), static_cast<unsigned>(n)),
                         dim3(256), 0, st, R, D, x, mean, rstd, dy, dw_part, db_part);
    }
  }
  if (sparc_status s = op_launched("layer norm backward")) return s;
  if (!dw && !db) return SPARC_OK;
  launch_reduce<PT>(st, n, D, dw_part, db_part, dw, db);
  return op_launched("layer norm backward");
}

}  // namespace
}  // namespace sparc

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

sparc_status sparc_layer_norm_forward(int64_t rows, int64_t cols, int32_t io_dtype, int32_t param_dtype, const void* x,
                                      const void* weight, const void* bias, float eps, void* y, float* mean,
                                      float* rstd, sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = ln_check(rows, cols, io_dtype, param_dtype)) return s;
  if (!(eps >= 0.0f)) return op_fail(SPARC_EINVAL, "layer norm forward: eps must be >= 0");
  if (rows == 0) return SPARC_OK;
  if (!x || !y || !mean != !rstd)
    return op_fail(SPARC_EINVAL, "layer norm forward: NULL pointer (mean and rstd come together)");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (io_dtype == SPARC_F32) return ln_forward<float, float>(st, rows, cols, x, weight, bias, eps, y, mean, rstd);
  if (param_dtype == SPARC_F32)
    return ln_forward<sparc::bf16, float>(st, rows, cols, x, weight, bias, eps, y, mean, rstd);
  return ln_forward<sparc::bf16, sparc::bf16>(st, rows, cols, x, weight, bias, eps, y, mean, rstd);
}

size_t sparc_layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
  using namespace sparc;
  if (ln_check(rows, cols, SPARC_F32, SPARC_F32)) return 0;
  int64_t n = most_partials<float>(cols);
  if (most_partials<bf16>(cols) > n) n = most_partials<bf16>(cols);
  if (rows < n) n = rows;
  return static_cast<size_t>(2 * n) * static_cast<size_t>(cols) * sizeof(float) + 256;
}

sparc_status sparc_layer_norm_backward(int64_t rows, int64_t cols, int32_t io_dtype, int32_t param_dtype,
                                       const void* x, const void* weight, const float* mean, const float* rstd,
                                       const void* dy, void* dx, void* dweight, void* dbias, void* workspace,
                                       size_t workspace_bytes, sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = ln_check(rows, cols, io_dtype, param_dtype)) return s;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!dx && !dweight && !dbias) return SPARC_OK;
  if (rows == 0) {  // the parameters' gradients are sums over no rows
    if (!dweight && !dbias) return SPARC_OK;
    if (param_dtype == SPARC_F32) launch_reduce<float>(st, 0, cols, nullptr, nullptr, dweight, dbias);
    else launch_reduce<sparc::bf16>(st, 0, cols, nullptr, nullptr, dweight, dbias);
    return op_launched("layer norm backward");
  }
  if (!x || !mean || !rstd || !dy) return op_fail(SPARC_EINVAL, "layer norm backward: NULL pointer");
  if ((dweight || dbias) && (!workspace || workspace_bytes < sparc_layer_norm_workspace_bytes(rows, cols)))
    return op_fail(SPARC_EWORKSPACE, "layer norm backward: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % sizeof(float))
    return op_fail(SPARC_EINVAL, "layer norm backward: the workspace must be 4-byte aligned");
  float* ws = static_cast<float*>(workspace);
  if (io_dtype == SPARC_F32)
    return ln_backward<float, float>(st, rows, cols, x, weight, mean, rstd, dy, dx, dweight, dbias, ws);
  if (param_dtype == SPARC_F32)
    return ln_backward<sparc::bf16, float>(st, rows, cols, x, weight, mean, rstd, dy, dx, dweight, dbias, ws);
  return ln_backward<sparc::bf16, sparc::bf16>(st, rows, cols, x, weight, mean, rstd, dy, dx, dweight, dbias, ws);
}

}  // extern "C"
