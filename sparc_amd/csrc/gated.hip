// The gated half of a feed-forward block (include/sparc_hip.h):
//   y = act(x Wg^T) * (x Wu^T)
// and with g = x Wg^T, u = x Wu^T, dg = dy u act'(g), du = dy act(g):
//   dx = dg Wg + du Wu,   dWg = dg^T x,   dWu = du^T x.
//
// All of them are matrix products: out[q][p] = sum over k of Q[q][k] P[p][k].  A launch
// makes g and u of a tile together and leaves y, or (the backward computes them again
// instead of keeping them: nothing of the width of the block is saved, and dg and du
// come from unrounded g and u) dg and du, side by side in one matrix G of 2 F columns.
// Then dx = G [Wg; Wu] and [dWg; dWu] = G^T x are one product each.
#include "matrix.h"

namespace sparc {
namespace {

enum Act : int { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2, ACT_SIGMOID = 3 };

// act(g), and its derivative
__device__ __forceinline__ float act_of(int act, float g, float& slope) {
  if (act == ACT_RELU) {
    slope = g > 0.0f ? 1.0f : 0.0f;
    return g > 0.0f ? g : g * 0.0f;  // NaN stays
  }
  if (act == ACT_GELU) {
    const float phi = 0.5f * erfcf(g * -0.70710678118654752f);
    slope = phi + g * expf(-0.5f * g * g) * 0.39894228040143268f;
    return g * phi;
  }
  const float sig = 1.0f / (1.0f + expf(-g));
  if (act == ACT_SIGMOID) {
    slope = sig * (1.0f - sig);
    return sig;
  }
  slope = sig * (1.0f + g * (1.0f - sig));
  return g * sig;
}

// An operand: rows r (the result's p or q) and the contraction k; element (r, k) at
// r ld + k, or (ACROSS) at k ld + r.  Two parts: rows (or, ACROSS, values of the
// contraction) from ``cut`` on are those of p1.
struct Operand {
  const void *p0, *p1;
  int64_t ld;
  int64_t cut;
};
struct ProductArgs {
  Operand P, Q;
  int64_t np, nq, nk;  // sizes of the result and of the contraction
  void *out0, *out1;   // rows q from out_cut on are those of out1
  int64_t out_ld, out_cut;
  const void* dy;      // GATED_BACK: [nq, F]
  int act;
  int64_t k_split;     // contraction of one workgroup; partial sums in fp32 where it is shorter than nk
  float* partial;      // [splits, nq, np]
};

enum Kind : int { GATED = 0, GATED_BACK = 1, PRODUCT = 2 };

constexpr int kTile = 128;

template <typename IO, int KIND, bool PA, bool QA>
__global__ __launch_bounds__(256, 2) void product_kernel(const ProductArgs a) {
  constexpr int BK = 32, VEC = kVec<IO>;
  constexpr bool DUAL = KIND != PRODUCT;
  // [tile rows][BK], or ACROSS [BK][tile rows]
  using LP = Panel<IO, PA ? kTile : BK, PA>;
  using LQ = Panel<IO, QA ? kTile : BK, QA>;
  __shared__ __attribute__((aligned(16))) IO lp[(PA ? BK : kTile) * LP::kStride];
  __shared__ __attribute__((aligned(16))) IO lq[(QA ? BK : kTile) * LQ::kStride];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, quad = 4 * (lane >> 4);
  constexpr int PT = DUAL ? kTile / 2 : kTile;
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * PT, q0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int64_t k0 = blockIdx.z * a.k_split, k1 = k0 + a.k_split < a.nk ? k0 + a.k_split : a.nk;

  constexpr int N = kTile * BK / VEC / 256;
  Vec<IO> rp[N], rq[N];
  const auto fetch = [&](const Operand& o, auto across, auto dual, int64_t r0, int64_t rows, int64_t k, Vec<IO>(&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + 256 * i;
      if constexpr (decltype(across)::value) {
        const int line = e / (kTile / VEC), c = e % (kTile / VEC) * VEC;
        const int64_t kk = k + line;
        const void* p = kk < o.cut ? o.p0 : o.p1;
        r[i] = load_vec<IO>(p, (kk < o.cut ? kk : kk - o.cut) * o.ld + r0 + c,
                            kk < k1 ? static_cast<int>(rows - r0 - c < VEC ? rows - r0 - c : VEC) : 0);
      } else {
        const int line = e / (BK / VEC), c = e % (BK / VEC) * VEC;
        // DUAL: of 64 lines, 32 of the gate's rows, then the same 32 of the other's
        const bool other = decltype(dual)::value && (line & 32);
        const int64_t row = r0 + (decltype(dual)::value ? (line >> 6) * 32 + (line & 31) : line);
        r[i] = load_vec<IO>(other ? o.p1 : o.p0, row * o.ld + k + c,
                            row < rows ? static_cast<int>(k1 - k - c < VEC ? k1 - k - c : VEC) : 0);
      }
    }
  };
  const auto put = [&](IO* lds, auto across, const Vec<IO>(&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + 256 * i;
      constexpr int cols = decltype(across)::value ? kTile : BK, per = cols / VEC;
      *reinterpret_cast<Vec<IO>*>(lds + Panel<IO, cols, decltype(across)::value>::at(e / per, e % per * VEC)) = r[i];
    }
  };
  using PAcross = std::integral_constant<bool, PA>;
  using QAcross = std::integral_constant<bool, QA>;
  using Dual = std::integral_constant<bool, DUAL>;
  const int wp = (wave & 1) * 64, wq = (wave >> 1) * 64;
  f32x4 acc[4][4];  // [p][q] tiles
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const auto fetch_both = [&](int64_t k) {
    fetch(a.P, PAcross(), Dual(), p0, a.np, k, rp);
    fetch(a.Q, QAcross(), std::false_type(), q0, a.nq, k, rq);
  };
  fetch_both(k0);
  for (int64_t k = k0; k < k1; k += BK) {
    __syncthreads();
    put(lp, PAcross(), rp);
    put(lq, QAcross(), rq);
    __syncthreads();
    if (k + BK < k1) fetch_both(k + BK);
    Frag<IO> fp[4], fq[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (PA) fp[i] = read_columns<LP>(lp, 0, wp + 16 * i);
      else fp[i] = read_rows<LP>(lp, wp + 16 * i, 0);
      if constexpr (QA) fq[i] = read_columns<LQ>(lq, 0, wq + 16 * i);
      else fq[i] = read_rows<LQ>(lq, wq + 16 * i, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mma(fp[i], fq[j], acc[i][j]);
  }
  if constexpr (DUAL) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t q = q0 + wq + 16 * j + col;
      if (q >= a.nq) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t p = p0 + wp / 2 + 16 * i + quad;
        const int n = static_cast<int>(a.np - p < 4 ? a.np - p : 4);
        if (n <= 0) continue;
        f32x4 slope, h;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float d;
          h[r] = act_of(a.act, acc[i][j][r], d);
          slope[r] = d;
        }
        if constexpr (KIND == GATED) {
          store_quad(static_cast<IO*>(a.out0) + q * a.out_ld + p, n, h * acc[i + 2][j]);
        } else {
          f32x4 dy = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r < n) {
              float y[1];
              unpack<IO, 1>(load_raw<IO, 1>(a.dy, q * a.np + p + r), y);
              dy[r] = y[0];
            }
          store_quad(static_cast<IO*>(a.out0) + q * a.out_ld + p, n, dy * acc[i + 2][j] * slope);
          store_quad(static_cast<IO*>(a.out0) + q * a.out_ld + a.np + p, n, dy * h);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t q = q0 + wq + 16 * j + col;
      if (q >= a.nq) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t p = p0 + wp + 16 * i + quad;
        const int n = static_cast<int>(a.np - p < 4 ? a.np - p : 4);
        if (n <= 0) continue;
        if (a.partial) {
          store_quad(a.partial + (blockIdx.z * a.nq + q) * a.np + p, n, acc[i][j]);
        } else {
          IO* out = static_cast<IO*>(q < a.out_cut ? a.out0 : a.out1);
          store_quad(out + (q < a.out_cut ? q : q - a.out_cut) * a.out_ld + p, n, acc[i][j]);
        }
      }
    }
  }
}

// The sum of the partial products, in order
template <typename IO>
__global__ __launch_bounds__(256) void product_sum_kernel(const float* partial, int splits, int64_t half, IO* out0,
                                                          IO* out1) {
  const int64_t total = 2 * half;
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
  if (rows >= (1LL << 31) || dim >= (1LL << 31) || hidden >= (1LL << 30)) return "gated linear unit: too large";
  if (io != SPARC_F32 && io != SPARC_BF16) return "gated linear unit: io_dtype must be F32 or BF16";
  if (act < ACT_SILU || act > ACT_SIGMOID) return "gated linear unit: unknown activation";
  return nullptr;
}
size_t size_of(int32_t io) { return io == SPARC_BF16 ? 2 : 4; }

// Parts of the contraction over the rows in the weights' gradient: as many as fill the GPU
int splits_of(int64_t rows, int64_t dim, int64_t hidden) {
  const int64_t tiles = ((dim + kTile - 1) / kTile) * ((2 * hidden + kTile - 1) / kTile);
  int64_t n = (512 + tiles - 1) / tiles, most = rows / 512;
  if (n > most) n = most;
  return static_cast<int>(n < 1 ? 1 : n > 64 ? 64 : n);
}
struct GatedPlan {
  int splits;
  int64_t k_split;
  size_t g, partial;
};
GatedPlan gated_plan(int64_t rows, int64_t dim, int64_t hidden, int32_t io) {
  GatedPlan p;
  p.splits = splits_of(rows, dim, hidden);
  p.k_split = ((rows + p.splits - 1) / p.splits + 31) / 32 * 32;
  if (p.k_split < 32) p.k_split = 32;
  p.splits = static_cast<int>((rows + p.k_split - 1) / p.k_split);
  if (p.splits < 1) p.splits = 1;
  p.g = up256(2 * rows * hidden * size_of(io));
  p.partial = p.splits > 1 ? up256(sizeof(float) * p.splits * 2 * hidden * dim) : 0;
  return p;
}
dim3 grid_of(int64_t np, int64_t nq, int tile_p, int splits) {
  return dim3(static_cast<unsigned>((np + tile_p - 1) / tile_p), static_cast<unsigned>((nq + kTile - 1) / kTile),
              static_cast<unsigned>(splits));
}

template <typename IO>
void gated_run(int64_t rows, int64_t dim, int64_t hidden, int act, const void* x, const void* wg, const void* wu,
               const void* dy, void* y, hipStream_t stream) {
  ProductArgs a = {};
  a.P = {wg, wu, dim, hidden};
  a.Q = {x, x, dim, rows};
  a.np = hidden, a.nq = rows, a.nk = a.k_split = dim;
  a.out0 = y;
  a.dy = dy;
  a.act = act;
  a.out_ld = dy ? 2 * hidden : hidden;
  const dim3 grid = grid_of(hidden, rows, kTile / 2, 1);
  if (dy) product_kernel<IO, GATED_BACK, false, false><<<grid, 256, 0, stream>>>(a);
  else product_kernel<IO, GATED, false, false><<<grid, 256, 0, stream>>>(a);
}
template <typename IO>
void gated_grads(int64_t rows, int64_t dim, int64_t hidden, const void* x, const void* wg, const void* wu, const void* g,
                 void* dx, void* dwg, void* dwu, float* partial, const GatedPlan& plan, hipStream_t stream) {
  if (dx) {
    ProductArgs a = {};
    a.P = {wg, wu, dim, hidden};
    a.Q = {g, g, 2 * hidden, 2 * hidden};
    a.np = dim, a.nq = rows, a.nk = a.k_split = 2 * hidden;
    a.out0 = a.out1 = dx;
    a.out_ld = dim, a.out_cut = rows;
    product_kernel<IO, PRODUCT, true, false><<<grid_of(dim, rows, kTile, 1), 256, 0, stream>>>(a);
  }
  if (dwg) {
    ProductArgs a = {};
    a.P = {x, x, dim, rows};
    a.Q = {g, g, 2 * hidden, rows};
    a.np = dim, a.nq = 2 * hidden, a.nk = rows, a.k_split = plan.k_split;
    a.out0 = dwg, a.out1 = dwu;
    a.out_ld = dim, a.out_cut = hidden;
    a.partial = plan.splits > 1 ? partial : nullptr;
    product_kernel<IO, PRODUCT, true, true><<<grid_of(dim, 2 * hidden, kTile, plan.splits), 256, 0, stream>>>(a);
    if (plan.splits > 1)
      product_sum_kernel<IO><<<op_grid((2 * hidden * dim + 255) / 256), 256, 0, stream>>>(
          partial, plan.splits, hidden * dim, static_cast<IO*>(dwg), static_cast<IO*>(dwu));
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
  if (io_dtype == SPARC_BF16) gated_run<bf16>(rows, dim, hidden, activation, x, gate_weight, up_weight, nullptr, y, stream);
  else gated_run<float>(rows, dim, hidden, activation, x, gate_weight, up_weight, nullptr, y, stream);
  return op_launched("sparc_gated_forward");
}

size_t sparc_gated_workspace_bytes(int64_t rows, int64_t dim, int64_t hidden, int32_t io_dtype) {
  if (fault_of(rows, dim, hidden, io_dtype, 0)) return 0;
  const GatedPlan p = gated_plan(rows, dim, hidden, io_dtype);
  return p.g + p.partial;
}

sparc_status sparc_gated_backward(int64_t rows, int64_t dim, int64_t hidden, int32_t io_dtype, int32_t activation,
                                  const void* x, const void* gate_weight, const void* up_weight, const void* dy,
                                  void* dx, void* dgate_weight, void* dup_weight, void* workspace,
                                  size_t workspace_bytes, sparc_stream_t stream_) {
  if (const char* fault = fault_of(rows, dim, hidden, io_dtype, activation)) return op_fail(SPARC_EINVAL, fault);
  if ((rows > 0 && (!x || !dy)) || !gate_weight || !up_weight || !dgate_weight != !dup_weight)
    return op_fail(SPARC_EINVAL, "gated linear unit: a tensor is NULL");
  const GatedPlan plan = gated_plan(rows, dim, hidden, io_dtype);
  if (rows > 0 && (!workspace || workspace_bytes < plan.g + plan.partial))
    return op_fail(SPARC_EWORKSPACE, "gated linear unit: workspace missing or too small");
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  char* const ws = static_cast<char*>(workspace);
  float* const partial = reinterpret_cast<float*>(ws + plan.g);
  const auto go = [&](auto type) {
    using IO = decltype(type);
    if (rows > 0) gated_run<IO>(rows, dim, hidden, activation, x, gate_weight, up_weight, dy, ws, stream);
    gated_grads<IO>(rows, dim, hidden, x, gate_weight, up_weight, ws, rows > 0 ? dx : nullptr, dgate_weight, dup_weight,
                    partial, plan, stream);
  };
  if (io_dtype == SPARC_BF16) go(bf16());
  else go(float());
  return op_launched("sparc_gated_backward");
}

}  // extern "C"
