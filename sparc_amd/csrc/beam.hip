// One step of beam search, and the recurrent states in the new beams' order.
//
//   lse[k]        = log sum over v of exp(x[k, v])
//   score[k, v]   = score[k] + (x[k, v] - lse[k])
//   a finished beam has one candidate, (eos, score[k])
//   the best K of a batch row's K V candidates, ties to the lowest k V + v
//
// beam_scan_kernel reads the logits once: each wave takes a span of one row and
// keeps the span's maximum, its sum of exponentials and its K + 1 largest
// values.  beam_join_kernel (one workgroup per batch row) joins the spans and
// ranks the candidates by their rounded fp32 scores.  Different logits can
// round to one score, and then the lower index wins, not the larger logit:
// the first value left out tells whether that can matter, and such a row is
// read once more, ranked by score.  Where every candidate of a beam has the
// same score (an empty beam, or NaN in its logits) no reading is needed.
//
// The list of largest values: 64 keys per wave, one per lane, in descending
// order.  A key is the value's order-preserving bits above the complement of
// its index, so keys are distinct and compare as (value, lower index).
// Candidates above the list's bound are gathered in LDS; 64 at a time they are
// sorted and merged into the list by bitonic exchanges.  The bound starts at
// the (K + 1)-th largest of the lanes' first values, so few candidates follow.

#include "common.h"
#include "sparc_hip.h"

namespace sparc {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kScanWaves = 4;      // waves (spans) per scan workgroup
constexpr int kJoinWaves = 8;
constexpr int kMaxSpans = 64;      // per row: a lane each when they are joined
constexpr int kMinSpan = 2048;     // logits per span at least
constexpr int kMaxPlanes = 96;     // state planes per launch: 2.5 KB of kernel arguments

// ---------------------------------------------------------------------------
// keys
// ---------------------------------------------------------------------------
// Bits that compare as the values do; -0 as +0, NaN above everything
__device__ __forceinline__ uint32_t ordered(float x) {
  x += 0.0f;
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
  if (o == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) {
  return (static_cast<uint64_t>(ordered(x)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }
__device__ __forceinline__ float key_value(uint64_t key) { return unordered(static_cast<uint32_t>(key >> 32)); }

__device__ __forceinline__ uint64_t lane_key(uint64_t key, int lane) {
  return (static_cast<uint64_t>(__shfl(static_cast<uint32_t>(key >> 32), lane)) << 32) |
         __shfl(static_cast<uint32_t>(key), lane);
}
__device__ __forceinline__ uint64_t xor_key(uint64_t key, int mask) {
  return (static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(key >> 32), mask)) << 32) |
         __shfl_xor(static_cast<uint32_t>(key), mask);
}
__device__ __forceinline__ uint64_t exchange(uint64_t key, int mask, bool larger) {
  const uint64_t other = xor_key(key, mask);
  return (other > key) == larger ? other : key;
}
// the wave's 64 keys in descending (or ascending) order of the lanes
template <bool DESCENDING>
__device__ __forceinline__ uint64_t sort_keys(uint64_t key, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1) {
#pragma unroll
    for (int m = size / 2; m > 0; m >>= 1) {
      const bool up = (lane & size) == 0 || size == 64;  // this block of ``size`` lanes in the asked order
      key = exchange(key, m, ((lane & m) == 0) == (up == DESCENDING));
    }
  }
  return key;
}

// ---------------------------------------------------------------------------
// the list of the largest
// ---------------------------------------------------------------------------
struct TopList {
  uint64_t list;   // lane i: the i-th largest key so far, 0: none
  uint64_t bound;  // keys at or below it cannot be among the ``want`` largest
  uint32_t held;   // candidates in the buffer (wave-uniform)
  int want;
  uint64_t* buf;   // 128 keys of LDS of this wave

  __device__ __forceinline__ void init(uint64_t* b, int w) {
    list = 0;
    bound = 0;
    held = 0;
    want = w;
    buf = b;
  }
  // the first keys of all lanes: ``want`` of them are at least as large as the
  // want-th largest of the lanes' largest
  __device__ __forceinline__ void start(uint64_t lane_largest, int lane) {
    const uint64_t k = lane_key(sort_keys<true>(lane_largest, lane), want - 1);
    bound = k ? k - 1 : 0;
  }
  __device__ __forceinline__ void merge(uint64_t cand, int lane) {
    cand = sort_keys<false>(cand, lane);
    uint64_t k = list > cand ? list : cand;  // the 64 largest of both, bitonic
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) k = exchange(k, m, (lane & m) == 0);
    list = k;
    const uint64_t b = lane_key(list, want - 1);
    if (b > bound) bound = b;
  }
  // a key per lane, 0: none; every lane of the wave calls it
  __device__ __forceinline__ void push(uint64_t key, int lane) {
    const bool take = key > bound;
    const uint64_t who = __ballot(take);
    if (!who) return;
    if (take) buf[held + __popcll(who & ((uint64_t(1) << lane) - 1))] = key;
    held += __popcll(who);
    if (held >= 64) {
      wave_lds_fence();
      const uint64_t cand = buf[lane];
      const uint64_t rest = buf[64 + lane];
      wave_lds_fence();
      buf[lane] = rest;
      held -= 64;
      merge(cand, lane);
    }
    wave_lds_fence();
  }
  __device__ __forceinline__ void finish(int lane) {
    if (held) {
      wave_lds_fence();
      merge(static_cast<uint32_t>(lane) < held ? buf[lane] : 0, lane);
      held = 0;
    }
  }
};

// ---------------------------------------------------------------------------
// the scan of the logits
// ---------------------------------------------------------------------------
// A row in 16-byte vectors from the last aligned address at or before its
// start: vector j holds the elements j VEC - shift + i.
template <typename IO>
struct Row {
  static constexpr int VEC = 16 / sizeof(IO);
  const void* base;
  int64_t V;
  int shift;
  int64_t vectors;

  __device__ __forceinline__ Row(const void* logits, int64_t offset, int64_t v) {
    base = static_cast<const IO*>(logits) + offset;
    V = v;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(base) % 16 / sizeof(IO));
    vectors = (v + shift + VEC - 1) / VEC;
  }
  // the elements of vector j, -inf where it reaches past the row; the first
  // element's index is returned
  __device__ __forceinline__ int64_t load(int64_t j, int64_t end, float (&x)[VEC]) const {
    const int64_t at = j * VEC - shift;
    if (j < end && at >= 0 && at + VEC <= V) {
      unpack<IO, VEC>(load_raw<IO, VEC>(base, at), x);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = j < end && at + i >= 0 && at + i < V ? load1<IO>(base, at + i) : -INFINITY;
    }
    return at;
  }
};

// The span's largest values by make(x): every value whose key passes the bound
template <typename IO, typename F>
__device__ __forceinline__ void push_vector(TopList& top, const Row<IO>& row, int64_t at, int64_t j, int64_t end,
                                            const float (&x)[Row<IO>::VEC], int lane, F&& make) {
#pragma unroll
  for (int i = 0; i < Row<IO>::VEC; ++i) {
    const bool in = j < end && at + i >= 0 && at + i < row.V;
    top.push(in ? make_key(make(x[i]), static_cast<uint32_t>(at + i)) : 0, lane);
  }
}
template <typename IO, typename F>
__device__ __forceinline__ void start_list(TopList& top, const Row<IO>& row, int64_t at, int64_t j, int64_t end,
                                           const float (&x)[Row<IO>::VEC], int lane, F&& make) {
  uint64_t k = 0;
#pragma unroll
  for (int i = 0; i < Row<IO>::VEC; ++i) {
    const uint64_t key = j < end && at + i >= 0 && at + i < row.V ? make_key(make(x[i]), static_cast<uint32_t>(at + i)) : 0;
    k = key > k ? key : k;
  }
  top.start(k, lane);
}

// parts: [rows][spans] (maximum, sum of exp(x - maximum)); tops: [rows][spans][want] keys
template <typename IO>
__global__ void __launch_bounds__(64 * kScanWaves)
beam_scan_kernel(int64_t rows, int64_t V, int64_t ld, int spans, int want, const void* logits, float2* parts,
                 uint64_t* tops) {
  __shared__ uint64_t buf[kScanWaves][128];
  constexpr int VEC = Row<IO>::VEC;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * kScanWaves + wave;
  if (job >= rows * spans) return;  // no workgroup barrier below
  const int64_t r = job / spans;
  const int span = static_cast<int>(job - r * spans);
  const Row<IO> row(logits, r * ld, V);
  const int64_t per = (row.vectors + spans - 1) / spans;
  const int64_t begin = span * per, end = begin + per < row.vectors ? begin + per : row.vectors;
  TopList top;
  top.init(buf[wave], want);
  const auto same = [](float v) { return v; };
  float m = -INFINITY, s = 0.0f;
  for (int64_t j0 = begin; j0 < end; j0 += 64) {
    const int64_t j = j0 + lane;
    float x[VEC];
    const int64_t at = row.load(j, end, x);
    float big = x[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
    if (j0 == begin) start_list<IO>(top, row, at, j, end, x, lane, same);
    // no value of any lane passes the bound: the usual case
    if (__any(!(big < key_value(top.bound)))) push_vector<IO>(top, row, at, j, end, x, lane, same);
    const float mn = fmaxf(m, big);
    const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing but -inf so far: exp gives 0
    float add = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) add += fast_exp(x[i] - ref);
    s = fmaf(s, fast_exp(m - ref), add);
    m = mn;
  }
  top.finish(lane);
  float all = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
  s = group_sum(s * fast_exp(m - (all == -INFINITY ? 0.0f : all)), 64);
  if (lane == 0) parts[job] = make_float2(all, s);
  if (lane < want) tops[job * want + lane] = top.list;
}

// ---------------------------------------------------------------------------
// joining the spans, ranking the candidates
// ---------------------------------------------------------------------------
// The next smaller value of the I/O type
template <typename IO>
__device__ __forceinline__ float next_below(float x) {
  x += 0.0f;
  const uint32_t u = __float_as_uint(x), one = sizeof(IO) == 2 ? 0x10000u : 1u;
  if (u == 0) return __uint_as_float(0x80000000u | one);
  return __uint_as_float(u & 0x80000000u ? u + one : u - one);
}

struct BeamStep {
  int64_t batch, V, ld;
  int beams, spans, want;
  int64_t eos;               // -1: beams do not finish
  const void* logits;
  const float* scores;
  const uint8_t* finished;   // NULL: none is
  const float2* parts;
  const uint64_t* tops;
  int64_t* tokens;
  int64_t* parents;
  float* new_scores;
  uint8_t* new_finished;     // NULL: not wanted
};

template <typename IO>
__global__ void __launch_bounds__(64 * kJoinWaves)
beam_join_kernel(BeamStep p) {
  __shared__ uint64_t buf[kJoinWaves][128];
  __shared__ uint64_t cand[kMaxBeams * (kMaxBeams + 1)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int K = p.beams;
  const int keep = p.V < K ? static_cast<int>(p.V) : K;  // candidates of a beam that can count
  const int64_t b = blockIdx.x;
  for (int k = wave; k < K; k += kJoinWaves) {
    const int64_t r = b * K + k;
    const float cum = p.scores[r];
    const uint32_t flat = static_cast<uint32_t>(k * p.V);
    uint64_t mine = 0;  // lane i: the beam's i-th candidate
    if (p.finished && p.finished[r]) {
      // (eos, cum), and -inf for every other token
      if (lane < keep && lane != p.eos) mine = make_key(-INFINITY, flat + lane);
      if (lane == K && p.eos >= 0) mine = make_key(cum, flat + static_cast<uint32_t>(p.eos));
    } else {
      const float2 part = lane < p.spans ? p.parts[r * p.spans + lane] : make_float2(-INFINITY, 0.0f);
      float m = part.x;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
      const float s = group_sum(part.y * fast_exp(part.x - (m == -INFINITY ? 0.0f : m)), 64);
      // without a finite logit the beam is empty: every candidate -inf
      const bool empty = m == -INFINITY && s == 0.0f;
      const float lse = m + logf(s);
      if (empty || lse != lse || cum != cum || cum == -INFINITY) {  // one score for all
        if (lane < keep) mine = make_key(empty ? cum - INFINITY : cum + (0.0f - lse), flat + lane);
      } else {
        const auto score = [&](float x) { return cum + (x - lse); };
        TopList top;
        top.init(buf[wave], p.want);
        const int n = p.spans * p.want;
        const uint64_t* tops = p.tops + r * n;
        for (int i0 = 0; i0 < n; i0 += 64) {
          const uint64_t key = i0 + lane < n ? tops[i0 + lane] : 0;
          if (i0 == 0) top.start(key, lane);
          top.push(key, lane);
        }
        top.finish(lane);
        bool again = cum == INFINITY;
        if (p.V > K) {
          const uint64_t in = lane_key(top.list, K - 1), out = lane_key(top.list, K);
          const float low = key_value(in), left = key_value(out);
          again = again || score(left == low ? next_below<IO>(low) : left) == score(low);
        }
        if (again) {
          const Row<IO> row(p.logits, (b * K + k) * p.ld, p.V);
          top.init(buf[wave], keep);
          for (int64_t j0 = 0; j0 < row.vectors; j0 += 64) {
            float x[Row<IO>::VEC];
            const int64_t at = row.load(j0 + lane, row.vectors, x);
            if (j0 == 0) start_list<IO>(top, row, at, lane, row.vectors, x, lane, score);
            push_vector<IO>(top, row, at, j0 + lane, row.vectors, x, lane, score);
          }
          top.finish(lane);
          if (lane < keep) mine = make_key(key_value(top.list), flat + key_index(top.list));
        } else if (lane < keep) {
          mine = make_key(score(key_value(top.list)), flat + key_index(top.list));
        }
      }
    }
    if (lane <= K) cand[k * (K + 1) + lane] = mine;
  }
  __syncthreads();
  if (wave > 0) return;
  TopList top;
  top.init(buf[0], K);
  const int n = K * (K + 1);
  for (int i0 = 0; i0 < n; i0 += 64) {
    const uint64_t key = i0 + lane < n ? cand[i0 + lane] : 0;
    if (i0 == 0) top.start(key, lane);
    top.push(key, lane);
  }
  top.finish(lane);
  if (lane < K) {
    const uint32_t flat = key_index(top.list);
    const int64_t parent = flat / static_cast<uint32_t>(p.V), token = flat - parent * p.V;
    const int64_t o = b * K + lane;
    p.tokens[o] = token;
    p.parents[o] = parent;
    p.new_scores[o] = key_value(top.list);
    if (p.new_finished)
      p.new_finished[o] = (p.finished && p.finished[b * K + parent]) || token == p.eos;
  }
}

// ---------------------------------------------------------------------------
// states in the new beams' order
// ---------------------------------------------------------------------------
struct Planes {
  const void* src[kMaxPlanes];
  void* dst[kMaxPlanes];
  int64_t row_bytes[kMaxPlanes];
  uint32_t first[kMaxPlanes + 1];  // first tile of each plane: 256 accesses of a row
  int count;
};
template <int B> struct Bytes;
template <> struct Bytes<16> { using T = uint4; };
template <> struct Bytes<4> { using T = uint32_t; };
template <> struct Bytes<2> { using T = uint16_t; };

// A thread moves one access of B bytes of all K rows of a batch row: it reads
// them all before it writes, so src and dst may be the same.  KM >= K.  A
// parent outside the beams fills its row with ones (NaN).
template <int B, int KM>
__global__ void __launch_bounds__(256)
reorder_kernel(Planes pl, int K, int64_t batch, const int64_t* parents) {
  using T = typename Bytes<B>::T;
  const uint32_t tiles = pl.first[pl.count];
  const int64_t jobs = batch * tiles;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int64_t b = job / tiles;
    const uint32_t tile = static_cast<uint32_t>(job - b * tiles);
    int lo = 0, hi = pl.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (pl.first[mid] <= tile) lo = mid; else hi = mid - 1;
    }
    const int64_t rb = pl.row_bytes[lo];
    const int64_t at = (static_cast<int64_t>(tile - pl.first[lo]) * 256 + threadIdx.x) * B;
    if (at >= rb) continue;
    const char* src = static_cast<const char*>(pl.src[lo]) + b * K * rb + at;
    char* dst = static_cast<char*>(pl.dst[lo]) + b * K * rb + at;
    const bool in_place = src == dst;
    T v[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (k < K) {
        const int64_t p = parents[b * K + k];
        if (p >= 0 && p < K) {
          if (!(in_place && p == k)) v[k] = *reinterpret_cast<const T*>(src + p * rb);
        } else {
          __builtin_memset(&v[k], 0xff, B);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (k < K && !(in_place && parents[b * K + k] == k)) *reinterpret_cast<T*>(dst + k * rb) = v[k];
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
sparc_status bm_fail(sparc_status s, const char* msg) {
  snprintf(error_buffer(), 512, "%s", msg);
  return s;
}
sparc_status bm_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return SPARC_OK;
  snprintf(error_buffer(), 512, "%s: %s", what, hipGetErrorString(e));
  return SPARC_EHIP;
}

sparc_status bm_check(int64_t batch, int64_t beams, int64_t vocab) {
  if (batch < 0 || beams < 1 || beams > kMaxBeams || vocab < 1)
    return bm_fail(SPARC_EINVAL, "beam step: batch >= 0, 1 to 32 beams and vocab > 0 required");
  if (batch > (int64_t(1) << 22) / beams || vocab > INT32_MAX / beams)
    return bm_fail(SPARC_EINVAL, "beam step: too large");
  return SPARC_OK;
}
// Spans per row: about 8192 waves in all (32 per CU), none shorter than kMinSpan
int spans_of(int64_t rows, int64_t vocab) {
  int64_t s = 8192 / (rows > 0 ? rows : 1);
  const int64_t most = (vocab + kMinSpan - 1) / kMinSpan;
  s = s < most ? s : most;
  return static_cast<int>(s < 1 ? 1 : (s < kMaxSpans ? s : kMaxSpans));
}
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

template <int B>
void launch_reorder(hipStream_t st, const Planes& pl, int K, int64_t batch, const int64_t* parents) {
  const int64_t jobs = batch * pl.first[pl.count];
  const dim3 grid(static_cast<unsigned>(jobs < (1 << 20) ? jobs : (1 << 20))), block(256);
  if (K <= 4) hipLaunchKernelGGL((reorder_kernel<B, 4>), grid, block, 0, st, pl, K, batch, parents);
  else if (K <= 8) hipLaunchKernelGGL((reorder_kernel<B, 8>), grid, block, 0, st, pl, K, batch, parents);
  else if (K <= 16) hipLaunchKernelGGL((reorder_kernel<B, 16>), grid, block, 0, st, pl, K, batch, parents);
  else hipLaunchKernelGGL((reorder_kernel<B, 32>), grid, block, 0, st, pl, K, batch, parents);
}

int plane_access(const void* src, const void* dst, int64_t row_bytes) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | row_bytes;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

}  // namespace
}  // namespace sparc

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

size_t sparc_beam_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab) {
  using namespace sparc;
  if (bm_check(batch, beams, vocab)) return 0;
  const int64_t rows = batch * beams, spans = spans_of(rows, vocab);
  return up256(rows * spans * sizeof(float2)) + up256(rows * spans * (beams + 1) * sizeof(uint64_t)) + 256;
}

sparc_status sparc_beam_step(int64_t batch, int64_t beams, int64_t vocab, int64_t row_stride, int32_t io_dtype,
                             const void* logits, const float* scores, const uint8_t* finished, int64_t eos_id,
                             int64_t* tokens, int64_t* parents, float* new_scores, uint8_t* new_finished,
                             void* workspace, size_t workspace_bytes, sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = bm_check(batch, beams, vocab)) return s;
  if (io_dtype != SPARC_F32 && io_dtype != SPARC_BF16) return bm_fail(SPARC_EINVAL, "beam step: unknown io_dtype");
  if (row_stride < vocab) return bm_fail(SPARC_EINVAL, "beam step: row_stride below vocab");
  if (eos_id < -1 || eos_id >= vocab) return bm_fail(SPARC_EINVAL, "beam step: eos_id outside the vocabulary");
  if (finished && eos_id < 0) return bm_fail(SPARC_EINVAL, "beam step: finished beams need an eos_id");
  if (batch == 0) return SPARC_OK;
  if (!logits || !scores || !tokens || !parents || !new_scores) return bm_fail(SPARC_EINVAL, "beam step: NULL pointer");
  if (!workspace || workspace_bytes < sparc_beam_workspace_bytes(batch, beams, vocab))
    return bm_fail(SPARC_EWORKSPACE, "beam step: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8)
    return bm_fail(SPARC_EINVAL, "beam step: the workspace must be 8-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t rows = batch * beams;
  const int spans = spans_of(rows, vocab), want = static_cast<int>(beams) + 1;
  float2* parts = static_cast<float2*>(workspace);
  uint64_t* tops = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + up256(rows * spans * sizeof(float2)));
  const dim3 grid(static_cast<unsigned>((rows * spans + kScanWaves - 1) / kScanWaves)), block(64 * kScanWaves);
  BeamStep p{};
  p.batch = batch;
  p.V = vocab;
  p.ld = row_stride;
  p.beams = static_cast<int>(beams);
  p.spans = spans;
  p.want = want;
  p.eos = eos_id;
  p.logits = logits;
  p.scores = scores;
  p.finished = finished;
  p.parts = parts;
  p.tops = tops;
  p.tokens = tokens;
  p.parents = parents;
  p.new_scores = new_scores;
  p.new_finished = new_finished;
  const dim3 join(static_cast<unsigned>(batch)), jblock(64 * kJoinWaves);
  if (io_dtype == SPARC_F32) {
    hipLaunchKernelGGL((beam_scan_kernel<float>), grid, block, 0, st, rows, vocab, row_stride, spans, want, logits, parts, tops);
    hipLaunchKernelGGL((beam_join_kernel<float>), join, jblock, 0, st, p);
  } else {
    hipLaunchKernelGGL((beam_scan_kernel<sparc::bf16>), grid, block, 0, st, rows, vocab, row_stride, spans, want, logits, parts, tops);
    hipLaunchKernelGGL((beam_join_kernel<sparc::bf16>), join, jblock, 0, st, p);
  }
  return bm_launched("beam step");
}

sparc_status sparc_reorder_states(int64_t batch, int64_t beams, int64_t count, const void* const* src,
                                  void* const* dst, const int64_t* row_bytes, const int64_t* parents,
                                  sparc_stream_t stream) {
  using namespace sparc;
  if (batch < 0 || beams < 1 || beams > kMaxBeams || count < 0 || batch > (int64_t(1) << 22) / beams)
    return bm_fail(SPARC_EINVAL, "reorder states: batch >= 0, 1 to 32 beams and count >= 0 required");
  if (batch == 0 || count == 0) return SPARC_OK;
  if (!src || !dst || !row_bytes || !parents) return bm_fail(SPARC_EINVAL, "reorder states: NULL pointer");
  for (int64_t i = 0; i < count; ++i) {
    if (row_bytes[i] < 0 || row_bytes[i] % 2 || row_bytes[i] > (int64_t(1) << 31))
      return bm_fail(SPARC_EINVAL, "reorder states: rows of an even number of bytes up to 2^31 required");
    if (row_bytes[i] > 0 && (!src[i] || !dst[i])) return bm_fail(SPARC_EINVAL, "reorder states: NULL plane");
    if ((reinterpret_cast<uintptr_t>(src[i]) | reinterpret_cast<uintptr_t>(dst[i])) % 2)
      return bm_fail(SPARC_EINVAL, "reorder states: planes must be 2-byte aligned");
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  Planes pl;
  for (const int access : {16, 4, 2}) {  // planes of one access width share launches
    for (int64_t at = 0; at < count;) {
      pl.count = 0;
      uint32_t tiles = 0;
      for (; at < count && pl.count < kMaxPlanes && tiles < (1u << 30); ++at) {
        if (row_bytes[at] == 0 || plane_access(src[at], dst[at], row_bytes[at]) != access) continue;
        pl.src[pl.count] = src[at];
        pl.dst[pl.count] = dst[at];
        pl.row_bytes[pl.count] = row_bytes[at];
        pl.first[pl.count++] = tiles;
        tiles += static_cast<uint32_t>((row_bytes[at] + 256 * access - 1) / (256 * access));
      }
      pl.first[pl.count] = tiles;
      if (pl.count == 0) break;
      if (access == 16) launch_reorder<16>(st, pl, static_cast<int>(beams), batch, parents);
      else if (access == 4) launch_reorder<4>(st, pl, static_cast<int>(beams), batch, parents);
      else launch_reorder<2>(st, pl, static_cast<int>(beams), batch, parents);
    }
  }
  return bm_launched("reorder states");
}

}  // extern "C"
