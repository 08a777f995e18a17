// Linear attention with a decay for each head (include/sparc_hip.h): the chunked form
// over a sequence, its gradients, and the recurrent form for one step.
//
// With a chunk of C steps that enters with the state S (key_dim x value_dim):
//   o_i  = a^(i+1) q_i S + sum over j <= i of a^(i-j) (q_i . k_j) v_j
//   S'   = a^C S + sum over j of a^(C-1-j) k_j v_j^T
// and the gradients are the same sums with other operands:
//   dq   = the forward of (do, v, k) with the states transposed;
//   dk   = the reversed sequence's of (v, do, q), dv that of (k, q, do), where the
//          state R is the gradient of the state before a step: it enters a step
//          undecayed (dS_t = R_(t+1) + q_t do_t^T) and leaves it decayed (R_t = a
//          dS_t), so the powers are a^i and a^(C-j) in place of a^(i+1) and a^(C-1-j).
// One kernel therefore does all four, and the backward is three problems of a launch.
//
// The state stays in the matrix instructions' accumulators of a wave for its whole chain,
// and every row is read once (with time segments keys and values twice).  What bounds a
// chain is neither memory nor the matrix instructions but one chunk after the other: load,
// scores, the split of scores and state into bf16 parts, products, update (65536 steps of
// 16 heads of 128 x 128 bf16: 134 us for the states of 32 segments, 17 to join them, 321
// for the outputs, at 3.6 TB/s, the matrix instructions busy 25 % and the VALU 33 % of the
// time, 423 in long runs; the gradients of 8 x 4096 steps of 8 heads 300 us, 192
// workgroups on 256 CUs).
#include "matrix.h"

namespace sparc {
namespace {

// ---------------------------------------------------------------------------
// the chunked form
// ---------------------------------------------------------------------------
// Rows of one operand: strides in values, query heads that share one of its heads
struct Rows {
  const void* p;
  int64_t sb, st, sh;
  int group;
};
struct Problem {
  Rows q, k, v;
  void* o;              // [B, T, H, V] contiguous, in the I/O type or (o_f32) in fp32
  const float* s_in;    // element (k, n) of chain c at c K V + k in_k + n in_n; NULL: zero
  float* s_out;         // the same with out_k, out_n; NULL: not wanted
  float* seg;           // [chains, segments, K, V]: what a segment adds, then what it enters with
  int in_k, in_n, out_k, out_n;
  int K, V, v_tiles;
  int extra;            // 1: the state is decayed before a step, 0: after it
  int reverse, o_f32;
  float intra, inter, update;  // factors of the scores, of q S, of what is added to S
};
struct Problems {
  Problem p[3];
  const float* decay;      // log a, per head
  const int64_t* lengths;  // NULL: T
  int64_t T, seg_len;
  int H, segments;
  int blocks[3];           // workgroups of each problem
};

// a^n for l2 = log2 a, n >= 0
__device__ __forceinline__ float power(float l2, float n) { return __builtin_amdgcn_exp2f(l2 * n); }
// log2 a.  Where a is zero a number so low that its powers are, but that of 0.
__device__ __forceinline__ float log2_decay(const float* decay, int h) {
  const float d = decay[h] * 1.4426950408889634f;
  return d < -1e30f ? -1e30f : d;
}
__device__ __forceinline__ int64_t steps_of(const Problems& a, int64_t b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n < a.T ? n : a.T;
}

// The value, which the compiler takes for another one each time: what is computed from
// it in a loop is computed there, and is not kept in registers that the loop needs.
__device__ __forceinline__ float anew(float x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ uint32_t anew(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Values of each operand that a bf16 product takes: the state and the scores as two
// bf16 values (each but 2^-17 of it); what is added to the state as three (all 24 bits)
// where the state is a result (EXACT), and as two where it only passes through to
// results in bf16.  Three everywhere would take registers and LDS that the chunks in
// flight need, for results whose own rounding is 2^-8: 16 x 2048 steps of 12 heads of 64
// with gradients 341 us for 222, 65536 steps of 16 heads of 128 537 for 431, 8 x 4096 of
// 8 heads 510 for 412.
template <typename IO> constexpr int kStateParts = sizeof(IO) == 2 ? 2 : 1;
template <typename IO> constexpr int kScoreParts = sizeof(IO) == 2 ? 2 : 1;

// An offset that no buffer reaches: loads there give zero, stores are dropped.
constexpr uint32_t kNowhere = 0x80000000u;

// Steps of a chunk, by the type and the padded key width
template <typename IO, int KP> constexpr int kChunk = sizeof(IO) == 2 && KP < 256 ? 64 : 32;

// NW: waves, each with NV tiles of 16 value columns
template <typename IO, int KP, int NW, int NV> struct Tiles {
  static constexpr int C = kChunk<IO, KP>;
  static constexpr int VT = 16 * NW * NV;              // value columns of a workgroup
  using Q = Panel<IO, KP, false>;
  using K = Panel<IO, KP, true>;
  using V = Panel<IO, VT, true>;
  using P = Panel<IO, C, false>;
};

// One operand's rows of a chunk on their way to LDS: TILE columns from ``from`` on of
// rows of ``width`` values.  A thread reads 16-byte vectors of one column position
// through a buffer that ends with the chunk's last row, so that nothing needs a
// condition (a branch around a load makes the loads wait for one another): what lies
// behind the last row (rows lie a row's width apart or more) or the last column is
// zero.  The vector that a row's end would cut is read so that it ends with the row,
// and shifted.
template <typename IO, int C, int TILE, int THREADS, bool WHOLE> struct Stage {
  static constexpr int VEC = kVec<IO>, PER = TILE / VEC, SIZE = sizeof(IO);
  static constexpr int STEP = THREADS / PER < C ? THREADS / PER : C, N = C / STEP;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  u4 r[N];
  const IO* p;      // uniform: the chain's step 0
  int64_t gap;      // values from a step's row to the next one's
  uint32_t at;      // the thread's bytes in a row
  int width, lack;  // columns that its vector lies further left than it should
  bool down;        // steps go down in memory

  static __device__ __forceinline__ int row() { return static_cast<int>(threadIdx.x) / PER; }
  __device__ __forceinline__ void begin(const Rows& o, int64_t b, int h, int width_, int from, bool reverse,
                                        int64_t steps) {
    const int c = from + static_cast<int>(threadIdx.x) % PER * VEC;
    width = width_;
    const int left = c + VEC <= width ? c : width > VEC ? width - VEC : 0;
    lack = c - left;
    at = lack < VEC && row() < C ? static_cast<uint32_t>(left * SIZE) : kNowhere;
    p = static_cast<const IO*>(o.p) + b * o.sb + (h / o.group) * o.sh + (reverse ? (steps - 1) * o.st : 0);
    gap = o.st;
    down = reverse;
  }
  // the rows of steps t0 .. t0 + have - 1
  __device__ __forceinline__ void fetch(int64_t t0, int have) {
    if (!WHOLE && width < VEC) return;
    const IO* const low = down ? p - (t0 + have - 1) * gap : p + t0 * gap;
    const auto buffer = make_rsrc(low, static_cast<uint32_t>(((have - 1) * gap + width) * SIZE));
    const uint32_t bytes = static_cast<uint32_t>(gap) * SIZE;
    const uint32_t first = at + bytes * static_cast<uint32_t>(down ? have - 1 - row() : row());
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t on = bytes * static_cast<uint32_t>(i * STEP);
      r[i] = __builtin_amdgcn_raw_buffer_load_b128(buffer, down ? first - on : first + on, 0, 0);
    }
  }
  template <typename L> __device__ __forceinline__ void put(IO* lds, int64_t t0, int have) {
    if (!WHOLE && width < VEC) {  // rows shorter than a vector, value by value
#pragma unroll 1
      for (int e = threadIdx.x; e < C * TILE; e += THREADS) {
        const int k = e / TILE, c = e % TILE;
        IO x = {};
        if (c < width && k < have) x = p[(t0 + k) * (down ? -gap : gap) + c];
        lds[L::at(k, c)] = x;
      }
      return;
    }
    if (THREADS / PER > C && row() >= C) return;  // fewer vectors than threads
    if (!WHOLE && width % VEC) {
      const int far = anew(lack * SIZE), words = far / 4, odd = far % 4;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u4 u = r[i];
        uint32_t w[5];
#pragma unroll
        for (int k = 0; k < 5; ++k) {
          w[k] = 0;
#pragma unroll
          for (int m = k; m < 4; ++m) w[k] = words == m - k ? u[m] : w[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) r[i][k] = odd ? w[k] >> 16 | w[k + 1] << 16 : w[k];
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      *reinterpret_cast<u4*>(lds + L::at(row() + i * STEP, static_cast<int>(threadIdx.x) % PER * VEC)) = r[i];
  }
};

// A workgroup of NW waves: one chain (batch row and head), 16 NW NV value columns, one
// segment of steps.  Each wave keeps the state of its 16 NV columns in registers.
// OUT: with outputs; else only what the segment adds to the state.  WHOLE: keys as wide
// as the tile, values that tiles divide and outputs in the I/O type; the other paths
// cost registers that the kernel for 128 x 128 needs (they spilled:
// 65536 steps of 16 heads 609 us with them, 527 without).
template <typename IO, int KP, int NW, int NV, bool OUT, bool EXACT, bool WHOLE>
__global__ __launch_bounds__(64 * NW, KP * NV >= 128 ? 2 : 3) void linear_kernel(const Problems a) {
  using W = Tiles<IO, KP, NW, NV>;
  constexpr int C = W::C, KT = KP / 16, NT = C / 16, THREADS = 64 * NW;
  constexpr int SP = kStateParts<IO>, PP = kScoreParts<IO>, AP = sizeof(IO) == 4 ? 1 : EXACT ? 3 : 2;
  __shared__ __attribute__((aligned(16))) IO lq[OUT ? C * W::Q::kStride : 1];
  __shared__ __attribute__((aligned(16))) IO lk[C * W::K::kStride];
  __shared__ __attribute__((aligned(16))) IO lv[C * W::V::kStride];
  __shared__ __attribute__((aligned(16))) IO lp[OUT ? PP : 1][OUT ? C * W::P::kStride : 1];

  int block = blockIdx.x, which = 0;
  while (which < 2 && block >= a.blocks[which]) block -= a.blocks[which++];
  const Problem& p = a.p[which];
  block = xcd_swizzle(block, a.blocks[which]);
  const int seg = block % a.segments, v_tile = block / a.segments % p.v_tiles;
  const int chain = block / a.segments / p.v_tiles, h = chain % a.H;
  const int64_t b = chain / a.H;
  const int lane = threadIdx.x & 63, col = lane & 15, quad = 4 * (lane >> 4);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t steps = steps_of(a, b), first = seg * a.seg_len;
  const int64_t last = first + a.seg_len < a.T ? first + a.seg_len : a.T, end = last < steps ? last : steps;
  const float l2_once = log2_decay(a.decay, h);
  const int v0 = v_tile * W::VT, w0 = wave * 16 * NV;  // first column of the workgroup, of the wave within it

  // the state: s[i][n] holds rows tile_row(i, quad, r) of column v0 + w0 + 16 n + col
  f32x4 s[KT][NV];
  const int64_t state = static_cast<int64_t>(chain) * p.K * p.V;
  // f(the value, its offset in bytes for these strides, or one that no buffer reaches)
  const auto each_state = [&](int of_k, int of_n, auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = v0 + w0 + 16 * n + col;
#pragma unroll
      for (int i = 0; i < KT; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = tile_row<IO>(i, quad, r);
          s[i][n][r] = f(s[i][n][r], row < p.K && c < p.V ? static_cast<uint32_t>(4 * (row * of_k + c * of_n)) : kNowhere);
        }
        __builtin_amdgcn_sched_barrier(0);  // offsets of few values at a time
      }
    }
  };
  const auto read_state = [&](const float* from, int of_k, int of_n) __attribute__((always_inline)) {
    const auto buffer = make_rsrc(from, static_cast<uint32_t>(4 * p.K * p.V));
    each_state(of_k, of_n, [&](float, uint32_t at) __attribute__((always_inline)) {
      return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buffer, at, 0, 0));
    });
  };
  const auto write_state = [&](float* to, int of_k, int of_n) __attribute__((always_inline)) {
    const auto buffer = make_rsrc(to, static_cast<uint32_t>(4 * p.K * p.V));
    each_state(of_k, of_n, [&](float x, uint32_t at) __attribute__((always_inline)) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), buffer, at, 0, 0);
      return x;
    });
  };
#pragma unroll
  for (int i = 0; i < KT; ++i)
#pragma unroll
    for (int n = 0; n < NV; ++n) s[i][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (OUT) {
    if (a.segments > 1) read_state(p.seg + (static_cast<int64_t>(chain) * a.segments + seg) * p.K * p.V, p.V, 1);
    else if (p.s_in) read_state(p.s_in + state, p.in_k, p.in_n);
  }

  Stage<IO, C, KP, THREADS, WHOLE> sq, sk;
  Stage<IO, C, W::VT, THREADS, WHOLE> sv;
  const int64_t rows = steps < 1 ? 1 : steps;
  if constexpr (OUT) sq.begin(p.q, b, h, p.K, 0, p.reverse, rows);
  sk.begin(p.k, b, h, p.K, 0, p.reverse, rows);
  sv.begin(p.v, b, h, p.V, v0, p.reverse, rows);
  const auto have_at = [&](int64_t t0) __attribute__((always_inline)) { return static_cast<int>(end - t0 < C ? end - t0 : C); };
  const auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
    const int have = have_at(t0);
    if constexpr (OUT) sq.fetch(t0, have);
    sk.fetch(t0, have);
    sv.fetch(t0, have);
  };
  // outputs of columns c4 .. c4 + 3 of steps t0 + 16 i + col, ``count`` steps from t0 on
  const int64_t o_gap = static_cast<int64_t>(a.H) * p.V;
  const auto emit = [&](int64_t t0, int count, bool down, int c4, const auto& x, auto tiles) __attribute__((always_inline)) {
    const int size = !WHOLE && p.o_f32 ? 4 : sizeof(IO);
    const int64_t low = down ? steps - t0 - count : t0;
    const auto buffer = make_rsrc(static_cast<char*>(p.o) + ((b * a.T + low) * o_gap + h * p.V) * size,
                                  static_cast<uint32_t>(((count - 1) * o_gap + p.V) * size));
    const uint32_t step = static_cast<uint32_t>(o_gap) * size;
    const uint32_t at = anew(static_cast<uint32_t>(down ? count - 1 - col : col) * step + c4 * size);
    const auto each = [&](auto&& store) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < tiles; ++i)
        store(x[i], 16 * i + col < count && c4 < p.V ? (down ? at - 16 * i * step : at + 16 * i * step) : kNowhere);
    };
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    if (!WHOLE && p.V % 4) {
      each([&](const f32x4& y, uint32_t to) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t one = c4 + r < p.V ? to + r * size : kNowhere;
          if (size == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[r]), buffer, one, 0, 0);
          else __builtin_amdgcn_raw_buffer_store_b16(pack_bf16(y[r]), buffer, one, 0, 0);
        }
      });
    } else if (size == 4) {
      each([&](const f32x4& y, uint32_t to) __attribute__((always_inline)) {
        const float f[4] = {y[0], y[1], y[2], y[3]};
        buffer_store_f32<4, 0>(buffer, to, f);
      });
    } else {
      each([&](const f32x4& y, uint32_t to) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_buffer_store_b64(u2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])}, buffer, to, 0, 0);
      });
    }
  };
  // powers of the decay: steps of a lane within a tile as fp32 numbers
  const float ahead = static_cast<float>(col - quad), lane_col = static_cast<float>(col);
  constexpr int kHalf = sizeof(IO) == 2 ? 4 : 16;  // from a fragment's first four steps to the others
  float leave[4];  // a^(31 - step) of those
#pragma unroll
  for (int r = 0; r < 4; ++r) leave[r] = power(l2_once, static_cast<float>(31 - step_of<IO>(quad, 4 + r)));
  const float leave_half = power(l2_once, static_cast<float>(kHalf));
  constexpr int TILES = NT * (NT + 1) / 2;  // of scores: a tile of queries with its own and earlier keys
  static_assert(NT <= 4, "the tiles' numbers");
  if constexpr (OUT) {  // the tile of keys behind an even tile of queries is read and stays zero
    if (wave < NT / 2)
#pragma unroll
      for (int n = 0; n < PP; ++n)
        *reinterpret_cast<Quad<IO>*>(&lp[n][W::P::at(32 * wave + col, 32 * wave + 16 + quad)]) = Quad<IO>{};
  }

  const auto put = [&](int64_t t0) __attribute__((always_inline)) {
    const int have = have_at(t0);
    if constexpr (OUT) sq.template put<typename W::Q>(lq, t0, have);
    sk.template put<typename W::K>(lk, t0, have);
    sv.template put<typename W::V>(lv, t0, have);
  };
  if (first < end) {
    fetch(first);
    put(first);
  }
  for (int64_t t0 = first; t0 < end; t0 += C) {
    const int have = have_at(t0);
    const float l2 = anew(l2_once);
    __syncthreads();  // the chunk is there

    f32x4 acc[OUT ? NV : 1][OUT ? NT : 1];
    if constexpr (OUT) {
      // scores of 16 queries with 16 keys, decayed, zero for later keys
#pragma unroll
      for (int m = 0; m < (TILES + NW - 1) / NW; ++m) {
        const int tile = wave + m * NW;
        if (tile >= TILES) break;
        const int qt = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, kt = tile - qt * (qt + 1) / 2;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < KP; c += 32)
          x = mma(read_rows<typename W::K>(lk, 16 * kt, c), read_rows<typename W::Q>(lq, 16 * qt, c), x);
        float y[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float n = ahead + static_cast<float>(16 * (qt - kt) - r);
          const float f = p.intra * power(l2, n < 0.0f ? 0.0f : n);
          y[r] = n < 0.0f ? 0.0f : x[r] * f;
          y[4 + r] = 0.0f;
        }
        Frag<IO> parts[PP];
        split(y, parts);
#pragma unroll
        for (int n = 0; n < PP; ++n)
          *reinterpret_cast<Quad<IO>*>(&lp[n][W::P::at(16 * qt + col, 16 * kt + quad)]) = parts[n].q[0];
      }
      // q S
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < KT; c += 2) {
        Frag<IO> sf[NV][SP];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const float x[8] = {s[c][n][0],     s[c][n][1],     s[c][n][2],     s[c][n][3],
                              s[c + 1][n][0], s[c + 1][n][1], s[c + 1][n][2], s[c + 1][n][3]};
          split(x, sf[n]);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const Frag<IO> q = read_rows<typename W::Q>(lq, 16 * i, 16 * c);
#pragma unroll
          for (int m = SP - 1; m >= 0; --m)
#pragma unroll
            for (int n = 0; n < NV; ++n) acc[n][i] = mma(sf[n][m], q, acc[n][i]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float f = p.inter * power(l2, lane_col + static_cast<float>(16 * i + p.extra));
#pragma unroll
        for (int n = 0; n < NV; ++n) acc[n][i] *= f;
      }
    }
    const float whole = power(l2, static_cast<float>(have));
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int n = 0; n < NV; ++n) s[i][n] *= whole;
    if constexpr (OUT) __syncthreads();  // the scores are there
    // early enough for the rows to arrive, and late enough that q S needs no registers
    if (t0 + C < end) fetch(t0 + C);
#pragma unroll
    for (int j = 0; j < C; j += 32) {
      Frag<IO> vf[NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) vf[n] = read_columns<typename W::V>(lv, j, w0 + 16 * n);
      if constexpr (OUT) {
        // a value that is not finite must not reach earlier steps of its block as 0 v
        uint32_t odd = 0;
#pragma unroll
        for (int n = 0; n < NV; ++n) odd = see(odd, vf[n]);
        const bool apart = __any(is_odd<IO>(odd));
        if (apart) {
#pragma unroll
          for (int i = j / 16; i < j / 16 + 2; ++i)
#pragma unroll 1
            for (int e = 0; e < 32; ++e) {
              if (j + e > 16 * i + col) continue;
              float x = 0.0f;
#pragma unroll
              for (int m = 0; m < PP; ++m) x += widen(lp[m][W::P::at(16 * i + col, j + e)]);
#pragma unroll
              for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  acc[n][i][r] = fmaf(x, widen(lv[W::V::at(j + e, w0 + 16 * n + quad + r)]), acc[n][i][r]);
            }
        }
#pragma unroll
        for (int i = j / 16; i < NT; ++i) {
          if (apart && i < j / 16 + 2) continue;
#pragma unroll
          for (int m = PP - 1; m >= 0; --m) {
            const Frag<IO> pf = read_rows<typename W::P>(lp[m], 16 * i, j);
#pragma unroll
            for (int n = 0; n < NV; ++n) acc[n][i] = mma(vf[n], pf, acc[n][i]);
          }
        }
      }
      // the state's share of these steps
      float f[8];
      if (have == C) {
        const float block = p.update * power(l2, static_cast<float>(C - 32 - j + 1 - p.extra));
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < 4 ? leave[e % 4] * (block * leave_half) : leave[e % 4] * block;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int n = have - p.extra - (j + step_of<IO>(quad, e));
          f[e] = p.update * power(l2, static_cast<float>(n < 0 ? 0 : n));
        }
      }
      Frag<IO> added[NV][AP];
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        float x[8];
        widen(vf[n], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f[e];
        split(x, added[n]);
      }
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const Frag<IO> kf = read_tile_columns<typename W::K>(lk, j, i);
#pragma unroll
        for (int m = AP - 1; m >= 0; --m)
#pragma unroll
          for (int n = 0; n < NV; ++n) s[i][n] = mma(kf, added[n][m], s[i][n]);
        if (i % 2) __builtin_amdgcn_sched_barrier(0);  // fragments of two tiles at a time: no more registers
      }
    }
    // Outputs are stored after the next chunk's rows have arrived: memory operations
    // end in order, and a wait for the rows must not wait for the stores.
    __syncthreads();  // the chunk is no longer read
    if (t0 + C < end) put(t0 + C);
    if constexpr (OUT) {
#pragma unroll
      for (int n = 0; n < NV; ++n) emit(t0, have, p.reverse, v0 + w0 + 16 * n + quad, acc[n], Int<NT>());
    }
  }
  if constexpr (OUT) {  // steps that a row does not have
    const f32x4 zero[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int64_t t = end > first ? end : first; t < last; t += 16)
#pragma unroll
      for (int n = 0; n < NV; ++n)
        emit(t, static_cast<int>(last - t < 16 ? last - t : 16), false, v0 + w0 + 16 * n + quad, zero, Int<1>());
    if (a.segments == 1 && p.s_out) write_state(p.s_out + state, p.out_k, p.out_n);
  } else {
    write_state(p.seg + (static_cast<int64_t>(chain) * a.segments + seg) * p.K * p.V, p.V, 1);
  }
}

// What each segment enters with, from what each adds; and the last state.  One thread
// per value of a chain's state of a problem (blockIdx.y); their states are equally large.
__global__ __launch_bounds__(256) void linear_join_kernel(const Problems a) {
  const Problem& p = a.p[blockIdx.y];
  const int size = p.K * p.V;
  const int blocks = (size + 255) / 256;  // of a chain
  const int64_t chain = blockIdx.x / blocks;
  const int e = blockIdx.x % blocks * 256 + threadIdx.x;
  if (e >= size) return;
  const int row = e / p.V, c = e % p.V;
  const int64_t steps = steps_of(a, chain / a.H);
  const float l2 = log2_decay(a.decay, static_cast<int>(chain % a.H));
  float s = p.s_in ? p.s_in[chain * size + row * p.in_k + c * p.in_n] : 0.0f;
  float* seg = p.seg + chain * a.segments * size + e;
  constexpr int N = 8;  // loads at a time: a store between them would keep them apart
  for (int n0 = 0; n0 < a.segments; n0 += N) {
    float add[N];
#pragma unroll
    for (int i = 0; i < N; ++i) add[i] = n0 + i < a.segments ? seg[static_cast<int64_t>(n0 + i) * size] : 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t left = steps - (n0 + i) * a.seg_len;
      const float f = power(l2, static_cast<float>(left < 0 ? 0 : left < a.seg_len ? left : a.seg_len));
      if (n0 + i < a.segments) seg[static_cast<int64_t>(n0 + i) * size] = s;
      s = n0 + i < a.segments ? f * s + add[i] : s;
    }
  }
  if (p.s_out) p.s_out[chain * size + row * p.out_k + c * p.out_n] = s;
}

// Sums over the query heads of a shared head: [rows, G, m, D] fp32 to [rows, G, D]
template <typename IO>
__global__ __launch_bounds__(256) void linear_shared_kernel(const float* in, IO* out, int64_t total, int m, int D) {
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < total;
       e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t head = e / D;
    const float* p = in + head * m * D + (e - head * D);
    float s = 0.0f;
    for (int i = 0; i < m; ++i) s += p[static_cast<int64_t>(i) * D];
    if constexpr (sizeof(IO) == 4) out[e] = s;
    else out[e].bits = pack_bf16(s);
  }
}

// ---------------------------------------------------------------------------
// one step
// ---------------------------------------------------------------------------
// A workgroup: one chain, 64 value columns; 16 lanes of four columns, 16 groups of rows.
// Bound by the state, read and written once (256 rows of 16 heads of 128 x 128: 86 us for
// 537 MB, 6.2 TB/s; 1 row: 5 us, two trips to memory).
template <typename IO>
__global__ __launch_bounds__(256) void linear_step_kernel(const Rows q, const Rows k, const Rows v, const float* decay,
                                                          const float* s_in, float* s_out, void* o, int H, int K,
                                                          int V, int v_tiles, float scale) {
  __shared__ float lq[256], lk[256];
  __shared__ f32x4 sums[16][17];
  const int chain = blockIdx.x / v_tiles, h = chain % H;
  const int64_t b = chain / H;
  const int tid = threadIdx.x, lane = tid & 15, group = tid >> 4, c = blockIdx.x % v_tiles * 64 + 4 * lane;
  if (tid < K) {
    float x[1];
    unpack<IO, 1>(load_raw<IO, 1>(q.p, b * q.sb + (h / q.group) * q.sh + tid), x);
    lq[tid] = x[0] * scale;
    unpack<IO, 1>(load_raw<IO, 1>(k.p, b * k.sb + (h / k.group) * k.sh + tid), x);
    lk[tid] = x[0];
  }
  const float a = expf(decay[h]);
  float x[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < V) {
      float y[1];
      unpack<IO, 1>(load_raw<IO, 1>(v.p, b * v.sb + (h / v.group) * v.sh + c + i), y);
      x[i] = y[0];
    }
  __syncthreads();
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int row = group; row < K; row += 16) {
    const int64_t at = (static_cast<int64_t>(chain) * K + row) * V + c;
    float s[4];
    unpack<float, 4>(load_vec<float>(s_in, at, V - c), s);
    f32x4 n;
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = fmaf(a, s[i], lk[row] * x[i]);
    store_quad(s_out + at, V - c, n);
    sum += lq[row] * n;
  }
  sums[group][lane] = sum;
  __syncthreads();
  if (group == 0) {
    for (int i = 1; i < 16; ++i) sum += sums[i][lane];
    store_quad(static_cast<IO*>(o) + static_cast<int64_t>(chain) * V + c, V - c, sum);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
const char* fault_of(const sparc_linear_desc* d) {
  if (!d) return "linear attention: desc is NULL";
  if (d->batch < 0 || d->length < 0) return "linear attention: batch and length must not be negative";
  if (d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads) return "linear attention: heads must be a positive multiple of kv_heads";
  if (d->key_dim < 1 || d->key_dim > 256 || d->value_dim < 1 || d->value_dim > 256)
    return "linear attention: key_dim and value_dim must be from 1 to 256";
  if (d->io_dtype != SPARC_F32 && d->io_dtype != SPARC_BF16) return "linear attention: io_dtype must be F32 or BF16";
  // a chunk's rows, and those of threads beside it, lie within 2^30 bytes: kNowhere and
  // as much more or less stays outside
  const int64_t* const strides[3] = {d->q_stride, d->k_stride, d->v_stride};
  for (int i = 0; i < 3; ++i)
    if (d->length > 1 && (strides[i][1] < (i < 2 ? d->key_dim : d->value_dim) || strides[i][1] >= (1LL << 22)))
      return "linear attention: time strides must be at least a row's values, and less than 2^22";
  if (d->heads * (d->key_dim > d->value_dim ? d->key_dim : d->value_dim) >= (1LL << 22)) return "linear attention: too large";
  // grids and chain numbers are 32-bit
  if (d->batch > (1 << 22) || d->batch * d->heads > (1 << 22) || d->length > (1LL << 31))
    return "linear attention: too large";
  return nullptr;
}

int padded(int64_t k) { return k <= 32 ? 32 : k <= 64 ? 64 : k <= 128 ? 128 : 256; }
// value columns of a workgroup
int columns_of(int64_t v) { return v > 64 ? 128 : 64; }

struct Plan {
  int keys, columns;  // padded keys and value columns of a workgroup
  int segments;
  int64_t seg_len;
};
// Time is cut into segments where the chains alone leave most of the GPU idle: into as
// many as the workgroups that it holds at once.  A second pass over keys and values,
// and the states between the passes, cost about as much as two thirds of idle CUs (16 x
// 2048 steps of 12 heads of 64, 192 workgroups of 768: 94 us in one pass, 80 with 4
// segments; the gradients of 8 x 4096 steps of 8 heads of 128, 192 of 512: 300 in one
// pass, 427 with 2 segments, 397 with 4).  Where chains are few or short, the length of
// a segment's chain is what counts: against segments of four chunks at least, 2 x 1000
// steps of 4 heads of 64 take 22.5 us instead of 34, 4096 of 8 heads of 128 45 (of one
// chunk 52: 512 workgroups, and 64 states to join) instead of 50.
int64_t groups_of(const sparc_linear_desc* d, int columns, int64_t v) {
  return d->batch * d->heads * ((v + columns - 1) / columns);
}
int64_t slots_of(int keys, int columns) { return keys * (columns / 64) >= 128 ? 512 : 768; }
Plan plan_of(const sparc_linear_desc* d, int keys, int columns, int64_t groups) {
  const int64_t chunk = d->io_dtype == SPARC_BF16 && keys < 256 ? 64 : 32;
  const int64_t slots = slots_of(keys, columns), chunks = d->length / chunk;
  int64_t n = groups < 1 || 3 * groups >= slots ? 1 : slots / groups;
  // segments of a chunk while every workgroup has a CU, of two at least else
  const int64_t most = groups < 1 || chunks / 2 > 256 / groups ? chunks / 2 : chunks < 256 / groups ? chunks : 256 / groups;
  if (n > most) n = most;
  if (n < 1) n = 1;
  int64_t len = (d->length + n - 1) / n;
  len = (len + chunk - 1) / chunk * chunk;
  if (len < chunk) len = chunk;
  n = d->length > 0 ? (d->length + len - 1) / len : 1;
  return {keys, columns, static_cast<int>(n), len};
}
Plan plan_of(const sparc_linear_desc* d, int64_t k, int64_t v, int problems) {
  const int columns = columns_of(v);
  return plan_of(d, padded(k), columns, groups_of(d, columns, v) * problems);
}
size_t segment_bytes(const sparc_linear_desc* d, const Plan& plan) {
  return plan.segments > 1 ? up256(sizeof(float) * d->batch * d->heads * plan.segments * d->key_dim * d->value_dim) : 0;
}

template <typename IO, int KP, int NW, int NV> void launch(Problems& a, int n, int64_t chains, hipStream_t stream) {
  constexpr int VT = Tiles<IO, KP, NW, NV>::VT;
  int total = 0;
  for (int i = 0; i < 3; ++i) a.blocks[i] = 0;
  for (int i = 0; i < n; ++i) {
    a.p[i].v_tiles = (a.p[i].V + VT - 1) / VT;
    a.blocks[i] = static_cast<int>(chains * a.p[i].v_tiles * a.segments);
    total += a.blocks[i];
  }
  if (total == 0) return;
  bool exact = false, whole = true;
  for (int i = 0; i < n; ++i) {
    exact = exact || (a.segments == 1 && a.p[i].s_out);  // with segments the joined states are the results
    whole = whole && a.p[i].K == KP && a.p[i].V % VT == 0 && !a.p[i].o_f32;
  }
  if (a.segments > 1) {
    if (whole) linear_kernel<IO, KP, NW, NV, false, true, true><<<total, 64 * NW, 0, stream>>>(a);
    else linear_kernel<IO, KP, NW, NV, false, true, false><<<total, 64 * NW, 0, stream>>>(a);
    linear_join_kernel<<<dim3(static_cast<unsigned>((a.p[0].K * a.p[0].V + 255) / 256 * chains), n), 256, 0, stream>>>(a);
  }
  constexpr bool kOne = sizeof(IO) == 4;  // fp32 products are exact either way
  if (whole) {
    if (exact) linear_kernel<IO, KP, NW, NV, true, true, true><<<total, 64 * NW, 0, stream>>>(a);
    else linear_kernel<IO, KP, NW, NV, true, kOne, true><<<total, 64 * NW, 0, stream>>>(a);
  } else {
    if (exact) linear_kernel<IO, KP, NW, NV, true, true, false><<<total, 64 * NW, 0, stream>>>(a);
    else linear_kernel<IO, KP, NW, NV, true, kOne, false><<<total, 64 * NW, 0, stream>>>(a);
  }
}
template <typename IO> void launch_io(const Plan& plan, Problems& a, int n, int64_t chains, hipStream_t stream) {
  const int k = plan.keys;
  if (plan.columns == 64) {
    if (k == 256) launch<IO, 256, 4, 1>(a, n, chains, stream);
    else if (k == 128) launch<IO, 128, 4, 1>(a, n, chains, stream);
    else if (k == 64) launch<IO, 64, 4, 1>(a, n, chains, stream);
    else launch<IO, 32, 4, 1>(a, n, chains, stream);
  } else {
    // Where no CU has a second workgroup the columns go to eight waves rather than four,
    // two to a SIMD (the gradients of 8 x 4096 steps of 8 heads of 128 x 128 bf16, 192
    // workgroups: 338 -> 304 us; 65536 steps of 16 heads, 512: 513 and 541).
    int64_t groups = 0;
    for (int i = 0; i < n; ++i) groups += chains * ((a.p[i].V + 127) / 128) * a.segments;
    const bool few = groups <= 256;
    if (k == 256) launch<IO, 256, 8, 1>(a, n, chains, stream);
    else if (k == 128 && few) launch<IO, 128, 8, 1>(a, n, chains, stream);
    else if (k == 128) launch<IO, 128, 4, 2>(a, n, chains, stream);
    else if (k == 64 && few) launch<IO, 64, 8, 1>(a, n, chains, stream);
    else if (k == 64) launch<IO, 64, 4, 2>(a, n, chains, stream);
    else if (few) launch<IO, 32, 8, 1>(a, n, chains, stream);
    else launch<IO, 32, 4, 2>(a, n, chains, stream);
  }
}
void launch_all(int32_t io, const Plan& plan, Problems& a, int n, int64_t chains, hipStream_t stream) {
  a.seg_len = plan.seg_len;
  a.segments = plan.segments;
  if (io == SPARC_BF16) launch_io<bf16>(plan, a, n, chains, stream);
  else launch_io<float>(plan, a, n, chains, stream);
}

// A row of ``width`` values for each step.  A chunk's absent steps are read as zero because
// they lie behind its last row, which takes a time stride of a row's width or more: one
// step, whose stride may be anything, gets that width.
Rows rows_of(const sparc_linear_desc* d, const void* p, const int64_t* stride, int64_t width, int64_t group) {
  return {p, stride[0], d->length == 1 ? width : stride[1], stride[2], static_cast<int>(group)};
}
// The backward's problems (dq with the two widths exchanged, dk too) are one launch
// where they are padded alike, and where all of them, padded to the larger keys, are on
// the GPU at once: what idle CUs do costs nothing (3 x 1237 steps of 6 heads, keys of 40
// and values of 72 in fp32: 111 -> 80 us; but keys of 32 beside values of 200, padded
// from 32 to 256, 126 -> 139, so at most to twice their width).
struct BackwardPlan {
  bool one;
  Plan qk, v;  // of dq and dk (or of all), of dv
  size_t seg_qk, seg_v, shared_k, shared_v, total;
};
BackwardPlan backward_plan(const sparc_linear_desc* d) {
  BackwardPlan r;
  const int64_t K = d->key_dim, V = d->value_dim;
  const int keys = padded(K > V ? K : V), columns = columns_of(K < V ? K : V);
  const int64_t groups = 2 * groups_of(d, columns, K) + groups_of(d, columns, V);
  r.one = (padded(K) == padded(V) && columns_of(K) == columns_of(V)) ||
          (keys <= 2 * padded(K < V ? K : V) && groups <= slots_of(keys, columns));
  r.qk = r.one ? plan_of(d, keys, columns, groups) : plan_of(d, V, K, 2);
  r.v = r.one ? r.qk : plan_of(d, K, V, 1);
  r.seg_qk = segment_bytes(d, r.qk);
  r.seg_v = segment_bytes(d, r.v);
  const bool shared = d->heads > d->kv_heads;
  const int64_t rows = d->batch * d->length * d->heads;
  r.shared_k = shared ? up256(sizeof(float) * rows * d->key_dim) : 0;
  r.shared_v = shared ? up256(sizeof(float) * rows * d->value_dim) : 0;
  r.total = 2 * r.seg_qk + r.seg_v + r.shared_k + r.shared_v;
  return r;
}

sparc_status check_desc(const sparc_linear_desc* d) {
  const char* fault = fault_of(d);
  return fault ? op_fail(SPARC_EINVAL, fault) : SPARC_OK;
}

}  // namespace
}  // namespace sparc

using namespace sparc;

extern "C" {

size_t sparc_linear_attention_workspace_bytes(const sparc_linear_desc* d, int backward) {
  if (fault_of(d) || d->batch == 0) return 0;
  if (backward) return backward_plan(d).total;
  return segment_bytes(d, plan_of(d, d->key_dim, d->value_dim, 1));
}

sparc_status sparc_linear_attention_forward(const sparc_linear_desc* d, const void* q, const void* k, const void* v,
                                            const float* log_decay, const int64_t* lengths, const float* state_in,
                                            void* o, float* state_out, void* workspace, size_t workspace_bytes,
                                            sparc_stream_t stream) {
  if (const sparc_status s = check_desc(d)) return s;
  if (d->batch == 0) return SPARC_OK;
  if ((d->length > 0 && (!q || !k || !v || !o)) || !log_decay)
    return op_fail(SPARC_EINVAL, "linear attention: a tensor is NULL");
  const Plan plan = plan_of(d, d->key_dim, d->value_dim, 1);
  if (workspace_bytes < segment_bytes(d, plan) || (plan.segments > 1 && !workspace))
    return op_fail(SPARC_EWORKSPACE, "linear attention: workspace missing or too small");
  const int K = static_cast<int>(d->key_dim), V = static_cast<int>(d->value_dim);
  const int64_t group = d->heads / d->kv_heads;
  Problems a = {};
  a.p[0] = {rows_of(d, q, d->q_stride, K, 1), rows_of(d, k, d->k_stride, K, group),
            rows_of(d, v, d->v_stride, V, group), o, state_in, state_out, static_cast<float*>(workspace),
            V, 1, V, 1, K, V, 0, 1, 0, 0, d->scale, d->scale, 1.0f};
  a.decay = log_decay;
  a.lengths = lengths;
  a.T = d->length;
  a.H = static_cast<int>(d->heads);
  launch_all(d->io_dtype, plan, a, 1, d->batch * d->heads, reinterpret_cast<hipStream_t>(stream));
  return op_launched("sparc_linear_attention_forward");
}

sparc_status sparc_linear_attention_backward(const sparc_linear_desc* d, const void* q, const void* k, const void* v,
                                             const float* log_decay, const int64_t* lengths, const float* state_in,
                                             const void* d_o, const float* dstate_out, void* dq, void* dk, void* dv,
                                             float* dstate_in, void* workspace, size_t workspace_bytes,
                                             sparc_stream_t stream_) {
  if (const sparc_status s = check_desc(d)) return s;
  if (d->batch == 0) return SPARC_OK;
  if ((d->length > 0 && (!q || !k || !v || !d_o || !dq || !dk || !dv)) || !log_decay)
    return op_fail(SPARC_EINVAL, "linear attention: a tensor is NULL");
  const BackwardPlan plan = backward_plan(d);
  if (workspace_bytes < plan.total || (plan.total > 0 && !workspace))
    return op_fail(SPARC_EWORKSPACE, "linear attention: workspace missing or too small");
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  char* ws = static_cast<char*>(workspace);
  float* const seg_q = reinterpret_cast<float*>(ws);
  float* const seg_k = reinterpret_cast<float*>(ws + plan.seg_qk);
  float* const seg_v = reinterpret_cast<float*>(ws + 2 * plan.seg_qk);
  float* const all_k = reinterpret_cast<float*>(ws + 2 * plan.seg_qk + plan.seg_v);
  float* const all_v = reinterpret_cast<float*>(ws + 2 * plan.seg_qk + plan.seg_v + plan.shared_k);
  const int K = static_cast<int>(d->key_dim), V = static_cast<int>(d->value_dim);
  const int64_t group = d->heads / d->kv_heads, H = d->heads, T = d->length, chains = d->batch * H;
  const int64_t o_stride[3] = {T * H * V, H * V, V};
  const Rows rq = rows_of(d, q, d->q_stride, K, 1), rk = rows_of(d, k, d->k_stride, K, group);
  const Rows rv = rows_of(d, v, d->v_stride, V, group), ro = rows_of(d, d_o, o_stride, V, 1);
  const int shared = group > 1;
  Problems a = {};
  // states of dq and dk are transposed: element (n, k) of the problem is (k, n) of the tensor
  a.p[0] = {ro, rv, rk, dq, state_in, nullptr, seg_q, 1, V, 1, V, V, K, 0, 1, 0, 0, d->scale, d->scale, 1.0f};
  a.p[1] = {rv, ro, rq, shared ? all_k : dk, dstate_out, nullptr, seg_k, 1, V, 1, V, V, K, 0, 0, 1, shared, d->scale, 1.0f, d->scale};
  a.p[2] = {rk, rq, ro, shared ? all_v : dv, dstate_out, dstate_in, seg_v, V, 1, V, 1, K, V, 0, 0, 1, shared, d->scale, 1.0f, d->scale};
  a.decay = log_decay;
  a.lengths = lengths;
  a.T = T;
  a.H = static_cast<int>(H);
  launch_all(d->io_dtype, plan.qk, a, plan.one ? 3 : 2, chains, stream);
  if (!plan.one) {
    a.p[0] = a.p[2];
    launch_all(d->io_dtype, plan.v, a, 1, chains, stream);
  }
  if (shared && T > 0) {
    const auto sum = [&](const float* in, void* out, int64_t D) {
      const int64_t total = d->batch * T * d->kv_heads * D;
      const unsigned grid = op_grid((total + 255) / 256);
      const int m = static_cast<int>(group), n = static_cast<int>(D);
      if (d->io_dtype == SPARC_BF16) linear_shared_kernel<<<grid, 256, 0, stream>>>(in, static_cast<bf16*>(out), total, m, n);
      else linear_shared_kernel<<<grid, 256, 0, stream>>>(in, static_cast<float*>(out), total, m, n);
    };
    sum(all_k, dk, K);
    sum(all_v, dv, V);
  }
  return op_launched("sparc_linear_attention_backward");
}

sparc_status sparc_linear_attention_step(const sparc_linear_desc* d, const void* q, const void* k, const void* v,
                                         const float* log_decay, const float* state_in, void* o, float* state_out,
                                         sparc_stream_t stream_) {
  if (const sparc_status s = check_desc(d)) return s;
  if (d->length != 1) return op_fail(SPARC_EINVAL, "linear attention: a step has length 1");
  if (d->batch == 0) return SPARC_OK;
  if (!q || !k || !v || !log_decay || !state_in || !o || !state_out)
    return op_fail(SPARC_EINVAL, "linear attention: a tensor is NULL");
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int64_t group = d->heads / d->kv_heads;
  const int H = static_cast<int>(d->heads), K = static_cast<int>(d->key_dim), V = static_cast<int>(d->value_dim);
  const Rows rq = rows_of(d, q, d->q_stride, K, 1), rk = rows_of(d, k, d->k_stride, K, group);
  const Rows rv = rows_of(d, v, d->v_stride, V, group);
  const int v_tiles = (V + 63) / 64;
  const unsigned grid = static_cast<unsigned>(d->batch * d->heads * v_tiles);
  if (d->io_dtype == SPARC_BF16)
    linear_step_kernel<bf16><<<grid, 256, 0, stream>>>(rq, rk, rv, log_decay, state_in, state_out, o, H, K, V, v_tiles, d->scale);
  else
    linear_step_kernel<float><<<grid, 256, 0, stream>>>(rq, rk, rv, log_decay, state_in, state_out, o, H, K, V, v_tiles, d->scale);
  return op_launched("sparc_linear_attention_step");
}

}  // extern "C"
