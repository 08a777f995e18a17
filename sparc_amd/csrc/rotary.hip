// RMS norms of queries and keys for each head, and the rotation by their positions in
// the same pass (include/sparc_hip.h):
//   y = R(position) (x rstd w),   rstd = 1 / sqrt(mean(x^2) + eps)
// and with g = R^T dy:  dx = rstd (g w - xhat mean(g w xhat)),  dw = sum of g xhat.
//
// Bound by memory: a head (a row) lives in registers of a few lanes, so forward and
// backward read it once.  A lane holds both values of each pair that is rotated.
// 32768 tokens of 24 heads of 64 bf16: forward 40 us (201 MB, 5.0 TB/s), backward 74 us
// (302 MB, 4.1 TB/s) and 5 us for the weights' sums over its 1024 workgroups.
#include "rows.h"

namespace sparc {
namespace {

// Heads whose rows a lane of the forward holds at once where there are enough of them:
// the angles of a token are read once for all of them (they are twice a bf16 head's
// bytes), and more loads are in flight (32768 tokens of 24 heads of 64 bf16: 56 us with
// one head at once, 40 with 4).  The backward holds x and dy anyway, and two heads were
// no faster there (76 us, with one 74).
constexpr int kHeads = 4;

struct Side {  // queries or keys
  const void* x;
  int64_t sb, st, sh;  // strides in values
  const void* w;       // NULL: ones
  const void* dy;      // contiguous, like y and dx
  void* out;           // y or dx
  float* partial;      // [blocks, D]: sums of g xhat (NULL: not wanted)
  int heads, blocks, chunks;  // chunks: groups of heads of a token
  int64_t units;              // chunks of all tokens
};
struct RotaryArgs {
  Side side[2];
  const float* table;        // [table_rows, R]: cosines, sines
  const int64_t* positions;  // [B, T] or NULL: t
  int64_t table_rows;
  int T, D, R, lanes, params_f32, several;
  float eps;
};

// W values at the alignment of one
template <typename T, int W> __device__ __forceinline__ void load_few(const void* base, int64_t index, float (&o)[W]) {
  struct __attribute__((packed, aligned(sizeof(T)))) Bits { T v[W]; };
  const Bits bits = *reinterpret_cast<const Bits*>(static_cast<const T*>(base) + index);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 4) o[i] = bits.v[i];
    else o[i] = bf16_bits_to_float(bits.v[i].bits);
  }
}
template <typename T, int W> __device__ __forceinline__ void store_few(void* base, int64_t index, const float (&x)[W]) {
  struct __attribute__((packed, aligned(sizeof(T)))) Bits { T v[W]; } bits;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 4) bits.v[i] = x[i];
    else bits.v[i].bits = pack_bf16(x[i]);
  }
  *reinterpret_cast<Bits*>(static_cast<T*>(base) + index) = bits;
}

// A unit: W values and the W that they are paired with (for interleaved pairs the 2 W
// values in a row).  A lane has U units; heads of up to 512 values have at most 64 lanes
// of so many:
template <int W> constexpr int kUnits = W >= 4 ? 1 : W == 2 ? 2 : 4;

// W values at the alignment of one, as they lie in memory
template <typename T, int W> struct __attribute__((packed, aligned(sizeof(T)))) Few { T v[W]; };
template <int W> __device__ __forceinline__ void widen(const Few<float, W>& f, float* o) {
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] = f.v[i];
}
template <int W> __device__ __forceinline__ void widen(const Few<bf16, W>& f, float* o) {
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] = bf16_bits_to_float(f.v[i].bits);
}

// HB: heads at once
template <typename IO, int W, int U, bool INTER, bool BACK, int HB>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  const bool keys = static_cast<int>(blockIdx.x) >= a.side[0].blocks;
  const Side& s = a.side[keys];
  const int block = blockIdx.x - (keys ? a.side[0].blocks : 0);
  const int tid = threadIdx.x, lane = tid & (a.lanes - 1), group = tid / a.lanes, groups = 256 / a.lanes;
  const int half = a.R / 2;
  const float nan = __uint_as_float(0x7fc00000u), inverse = 1.0f / static_cast<float>(a.D);

  // where a lane's units lie, and the weights there
  int at[U][2];
  bool turns[U], there[U], second[U];
  float w[U][2 * W], sums[U][2 * W];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int first = (lane + u * a.lanes) * W;  // of the unit's pairs
    there[u] = 2 * first < a.D;
    turns[u] = first < half;
    at[u][0] = !INTER && turns[u] ? first : 2 * first;
    at[u][1] = !INTER && turns[u] ? half + first : 2 * first + W;
    second[u] = there[u] && at[u][1] < a.D;  // a head of odd width ends with one value
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) sums[u][i] = 0.0f, w[u][i] = 1.0f;
    if (s.w) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (m ? second[u] : there[u]) {
            const int e = at[u][m] + i;
            float y[1];
            if (a.params_f32) load_few<float, 1>(s.w, e, y);
            else load_few<IO, 1>(s.w, e, y);
            w[u][m * W + i] = y[0];
          }
    }
  }
  // a unit's two halves, in pairs: o[i] belongs to o[W + i], or (INTER: the 2 W values in
  // a row) o[2 i] to o[2 i + 1]
  // Nothing is read under a condition (a branch around a load makes the loads wait for
  // one another): a lane without a unit reads the head's first values and drops them, and
  // behind the last head the last one is read again.
  using Bits = Few<IO, W>;
  bool whole = true;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    whole = whole && second[u];
    if (!there[u]) at[u][0] = 0;
    if (!second[u]) at[u][1] = 0;
  }
  whole = __all(whole);
  const auto load = [&](const void* p, int64_t base, int u, Bits (&o)[2]) {
    const IO* const q = static_cast<const IO*>(p) + base;
    o[0] = *reinterpret_cast<const Bits*>(q + at[u][0]);
    o[1] = *reinterpret_cast<const Bits*>(q + at[u][1]);
  };
  const auto values = [&](const Bits (&o)[2], int u, float* x) {
    widen(o[0], x);
    widen(o[1], x + W);
    if (!whole) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        x[i] = there[u] ? x[i] : 0.0f;
        x[W + i] = second[u] ? x[W + i] : 0.0f;
      }
    }
  };
  const auto first_of = [](int i) { return INTER ? 2 * i : i; };
  const auto second_of = [](int i) { return INTER ? 2 * i + 1 : W + i; };

  for (int64_t unit = static_cast<int64_t>(block) * groups + group; unit < s.units;
       unit += static_cast<int64_t>(s.blocks) * groups) {
    const uint32_t token = static_cast<uint32_t>(unit) / static_cast<uint32_t>(s.chunks);
    const int head0 = static_cast<int>(static_cast<uint32_t>(unit) - token * s.chunks) * HB;
    const uint32_t b = token / static_cast<uint32_t>(a.T), t = token - b * a.T;
    const int64_t from = b * s.sb + t * s.st + head0 * s.sh;
    const int64_t to = (static_cast<int64_t>(token) * s.heads + head0) * a.D;
    const int64_t position = a.positions ? a.positions[token] : t;
    const bool known = position >= 0 && position < a.table_rows;
    Bits xs[HB][U][2], gs[BACK ? HB : 1][U][2];
    float cs[U][W], sn[U][W];
#pragma unroll
    for (int k = 0; k < HB; ++k)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = head0 + k < s.heads ? k : s.heads - 1 - head0;
        load(s.x, from + h * s.sh, u, xs[k][u]);
        if constexpr (BACK) load(s.dy, to + h * a.D, u, gs[k][u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < W; ++i) cs[u][i] = 1.0f, sn[u][i] = 0.0f;
      if (turns[u] && known) {
        const int64_t angle = position * a.R + (lane + u * a.lanes) * W;
        load_few<float, W>(a.table, angle, cs[u]);
        load_few<float, W>(a.table, angle + half, sn[u]);
      }
    }
#pragma unroll
    for (int k = 0; k < HB; ++k) {
      float x[U][2 * W], g[U][2 * W];
      float square = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        values(xs[k][u], u, x[u]);
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) square = fmaf(x[u][i], x[u][i], square);
      }
      square = group_sum(square, a.lanes);
      const float rstd = known ? rsqrtf(fmaf(square, inverse, a.eps)) : nan;
      float along = 0.0f;
      if constexpr (BACK) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          values(gs[k][u], u, g[u]);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            float &p = g[u][first_of(i)], &q = g[u][second_of(i)];
            const float c = p * cs[u][i] + q * sn[u][i], d = q * cs[u][i] - p * sn[u][i];
            p = c, q = d;
          }
          const bool real = head0 + k < s.heads;  // (else 0 NaN could reach the sums)
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) {
            x[u][i] *= rstd;
            sums[u][i] = real ? fmaf(g[u][i], x[u][i], sums[u][i]) : sums[u][i];
            g[u][i] *= w[u][i];
            along = fmaf(g[u][i], x[u][i], along);
          }
        }
        along = group_sum(along, a.lanes) * inverse;
      }
      if (head0 + k >= s.heads || !s.out) continue;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float y[2 * W];
        if constexpr (BACK) {
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) y[i] = rstd * (g[u][i] - x[u][i] * along);
        } else {
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) y[i] = x[u][i] * rstd * w[u][i];
#pragma unroll
          for (int i = 0; i < W; ++i) {
            float &p = y[first_of(i)], &q = y[second_of(i)];
            const float c = p * cs[u][i] - q * sn[u][i], d = q * cs[u][i] + p * sn[u][i];
            p = c, q = d;
          }
        }
        float lo[W], hi[W];
#pragma unroll
        for (int i = 0; i < W; ++i) lo[i] = y[i], hi[i] = y[W + i];
        if (there[u]) store_few<IO, W>(s.out, to + k * a.D + at[u][0], lo);
        if (second[u]) store_few<IO, W>(s.out, to + k * a.D + at[u][1], hi);
      }
    }
  }
  if constexpr (BACK) {
    if (!s.partial) return;
    __shared__ float part[256][2 * W * U + 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) part[tid][u * 2 * W + i] = sums[u][i];
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          float sum = 0.0f;
          for (int m = 0; m < groups; ++m) sum += part[m * a.lanes + lane][u * 2 * W + i];
          if (i < W ? there[u] : second[u])
            s.partial[static_cast<int64_t>(block) * a.D + (i < W ? at[u][0] + i : at[u][1] + i - W)] = sum;
        }
    }
  }
}

// dw[c] = the sum of the workgroups' partial rows, in order
struct RotarySums {
  const float* in[2];
  void* out[2];
  int rows[2], D, f32;
};
__global__ __launch_bounds__(1024) void rotary_sum_kernel(const RotarySums a) {
  __shared__ float part[32][33];
  const int which = blockIdx.y, col = threadIdx.x & 31, c = blockIdx.x * 32 + col, group = threadIdx.x >> 5;
  if (!a.out[which]) return;
  float sum = 0.0f;
  if (c < a.D) {
#pragma unroll 8
    for (int r = group; r < a.rows[which]; r += 32) sum += a.in[which][static_cast<int64_t>(r) * a.D + c];
  }
  part[group][col] = sum;
  __syncthreads();
  if (group || c >= a.D) return;
  for (int m = 1; m < 32; ++m) sum += part[m][col];
  if (a.f32) static_cast<float*>(a.out[which])[c] = sum;
  else static_cast<bf16*>(a.out[which])[c].bits = pack_bf16(sum);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int kBackBlocks = 1024;

const char* fault_of(const sparc_rotary_desc* d) {
  if (!d) return "qk_norm_rotary: desc is NULL";
  if (d->batch < 0 || d->length < 0 || d->q_heads < 1 || d->k_heads < 0)
    return "qk_norm_rotary: batch and length must not be negative, q_heads must be positive";
  if (d->head_dim < 1 || d->head_dim > 512) return "qk_norm_rotary: head_dim must be from 1 to 512";
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 2)
    return "qk_norm_rotary: rotary_dim must be even and at most head_dim";
  if (d->table_rows < 0) return "qk_norm_rotary: table_rows must not be negative";
  if (d->io_dtype != SPARC_F32 && d->io_dtype != SPARC_BF16) return "qk_norm_rotary: io_dtype must be F32 or BF16";
  if (d->param_dtype != d->io_dtype && d->param_dtype != SPARC_F32)
    return "qk_norm_rotary: parameters must be in io_dtype or F32";
  if (!(d->eps >= 0.0f)) return "qk_norm_rotary: eps must be >= 0";
  const int64_t most = 1LL << 31;
  if (d->batch >= most || d->length >= most || d->q_heads >= most || d->k_heads >= most ||
      (d->batch > 0 && d->length > 0 &&
       (d->length >= most / d->batch || d->q_heads >= most / (d->batch * d->length) ||
        d->k_heads >= most / (d->batch * d->length))))
    return "qk_norm_rotary: too large";
  return nullptr;
}
int width_of(const sparc_rotary_desc* d) {
  for (int w = d->io_dtype == SPARC_BF16 ? 8 : 4; w > 1; w /= 2)
    if (d->head_dim % (2 * w) == 0 && d->rotary_dim % (2 * w) == 0) return w;
  return 1;
}
template <typename IO, int W, int U, bool BACK, int HB> void rotary_pairs(const RotaryArgs& a, bool inter, hipStream_t stream) {
  const int grid = a.side[0].blocks + a.side[1].blocks;
  if (inter) rotary_kernel<IO, W, U, true, BACK, HB><<<grid, 256, 0, stream>>>(a);
  else rotary_kernel<IO, W, U, false, BACK, HB><<<grid, 256, 0, stream>>>(a);
}
template <typename IO, int W, bool BACK> void rotary_launch(const RotaryArgs& a, bool inter, hipStream_t stream) {
  if (!BACK && a.several) rotary_pairs<IO, W, 1, BACK, BACK ? 1 : kHeads>(a, inter, stream);
  else if (a.D <= 128 * W) rotary_pairs<IO, W, 1, BACK, 1>(a, inter, stream);
  else rotary_pairs<IO, W, kUnits<W>, BACK, 1>(a, inter, stream);
}
template <bool BACK> void rotary_dispatch(const sparc_rotary_desc* d, RotaryArgs& a, hipStream_t stream) {
  const int w = width_of(d);
  const bool inter = d->interleaved != 0;
  if (d->io_dtype == SPARC_BF16) {
    if (w == 8) rotary_launch<bf16, 8, BACK>(a, inter, stream);
    else if (w == 4) rotary_launch<bf16, 4, BACK>(a, inter, stream);
    else if (w == 2) rotary_launch<bf16, 2, BACK>(a, inter, stream);
    else rotary_launch<bf16, 1, BACK>(a, inter, stream);
  } else {
    if (w == 4) rotary_launch<float, 4, BACK>(a, inter, stream);
    else if (w == 2) rotary_launch<float, 2, BACK>(a, inter, stream);
    else rotary_launch<float, 1, BACK>(a, inter, stream);
  }
}
// Everything but the sides' tensors; ``most``: workgroups at most
RotaryArgs rotary_args(const sparc_rotary_desc* d, const float* table, const int64_t* positions, int64_t most, bool back) {
  RotaryArgs a = {};
  const int w = width_of(d);
  const int64_t units = (d->head_dim + 2 * w - 1) / (2 * w);
  a.lanes = 1;
  while (a.lanes < 64 && a.lanes < units) a.lanes *= 2;
  const int64_t tokens = d->batch * d->length, groups = 256 / a.lanes;
  const int64_t heads[2] = {d->q_heads, d->k_heads};
  // several heads at once where a lane group for each head would be many more than the GPU holds
  a.several = !back && tokens * (d->q_heads + d->k_heads) * a.lanes >= (1 << 20) && units <= 64;
  const int64_t hb = a.several ? kHeads : 1, chunks[2] = {(heads[0] + hb - 1) / hb, (heads[1] + hb - 1) / hb};
  const int64_t all = tokens * (chunks[0] + chunks[1]);
  for (int i = 0; i < 2; ++i) {
    Side& s = a.side[i];
    const int64_t* stride = i ? d->k_stride : d->q_stride;
    s.sb = stride[0], s.st = stride[1], s.sh = stride[2];
    s.heads = static_cast<int>(heads[i]);
    s.chunks = static_cast<int>(chunks[i]);
    s.units = tokens * chunks[i];
    int64_t blocks = (s.units + groups - 1) / groups;
    const int64_t share = all ? (most * s.units + all - 1) / all : 0;
    if (blocks > share) blocks = share;
    s.blocks = static_cast<int>(blocks);
  }
  a.table = table;
  a.positions = positions;
  a.table_rows = d->table_rows;
  a.T = static_cast<int>(d->length);
  a.D = static_cast<int>(d->head_dim);
  a.R = static_cast<int>(d->rotary_dim);
  a.params_f32 = d->param_dtype == SPARC_F32;
  a.eps = d->eps;
  return a;
}

}  // namespace
}  // namespace sparc

using namespace sparc;

extern "C" {

sparc_status sparc_qk_norm_rotary_forward(const sparc_rotary_desc* d, const void* q, const void* k,
                                          const void* q_weight, const void* k_weight, const float* table,
                                          const int64_t* positions, void* yq, void* yk, sparc_stream_t stream) {
  if (const char* fault = fault_of(d)) return op_fail(SPARC_EINVAL, fault);
  if (d->batch == 0 || d->length == 0) return SPARC_OK;
  if (!q || !yq || (d->k_heads > 0 && (!k || !yk)) || (d->rotary_dim > 0 && d->table_rows > 0 && !table))
    return op_fail(SPARC_EINVAL, "qk_norm_rotary: a tensor is NULL");
  RotaryArgs a = rotary_args(d, table, positions, 1 << 16, false);
  a.side[0].x = q, a.side[0].w = q_weight, a.side[0].out = yq;
  a.side[1].x = k, a.side[1].w = k_weight, a.side[1].out = yk;
  rotary_dispatch<false>(d, a, reinterpret_cast<hipStream_t>(stream));
  return op_launched("sparc_qk_norm_rotary_forward");
}

size_t sparc_qk_norm_rotary_workspace_bytes(const sparc_rotary_desc* d) {
  if (fault_of(d)) return 0;
  return up256(sizeof(float) * (kBackBlocks + 2) * d->head_dim);
}

sparc_status sparc_qk_norm_rotary_backward(const sparc_rotary_desc* d, const void* q, const void* k,
                                           const void* q_weight, const void* k_weight, const float* table,
                                           const int64_t* positions, const void* dyq, const void* dyk, void* dq,
                                           void* dk, void* dq_weight, void* dk_weight, void* workspace,
                                           size_t workspace_bytes, sparc_stream_t stream_) {
  if (const char* fault = fault_of(d)) return op_fail(SPARC_EINVAL, fault);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int64_t tokens = d->batch * d->length;
  if (tokens > 0 && (!q || !dyq || (d->k_heads > 0 && (!k || !dyk)) || (d->rotary_dim > 0 && d->table_rows > 0 && !table)))
    return op_fail(SPARC_EINVAL, "qk_norm_rotary: a tensor is NULL");
  const bool sums = dq_weight || dk_weight;
  if (sums && (!workspace || workspace_bytes < sparc_qk_norm_rotary_workspace_bytes(d)))
    return op_fail(SPARC_EWORKSPACE, "qk_norm_rotary: workspace missing or too small");
  RotaryArgs a = rotary_args(d, table, positions, kBackBlocks, true);
  float* const partial = static_cast<float*>(workspace);
  a.side[0].x = q, a.side[0].w = q_weight, a.side[0].dy = dyq, a.side[0].out = dq;
  a.side[1].x = k, a.side[1].w = k_weight, a.side[1].dy = dyk, a.side[1].out = dk;
  if (dq_weight) a.side[0].partial = partial;
  if (dk_weight) a.side[1].partial = partial + static_cast<int64_t>(a.side[0].blocks) * d->head_dim;
  if (tokens > 0) rotary_dispatch<true>(d, a, stream);
  if (sums) {
    const RotarySums r = {{partial, partial + static_cast<int64_t>(a.side[0].blocks) * d->head_dim},
                          {dq_weight, dk_weight},
                          {a.side[0].blocks, a.side[1].blocks},
                          a.D,
                          a.params_f32};
    rotary_sum_kernel<<<dim3((a.D + 31) / 32, 2), 1024, 0, stream>>>(r);
  }
  return op_launched("sparc_qk_norm_rotary_backward");
}

}  // extern "C"
