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
// the (K + 1)-th largest of the maxima of the lanes' first values, those of all
// waves of a workgroup together where they share a row, so few candidates
// follow: most vectors cost a maximum and a comparison beside their
// exponentials.

#include "rows.h"

namespace sparc {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kScanWaves = 4;      // waves (spans) per scan workgroup
constexpr int kMostJoinWaves = 16;
constexpr int kMaxSpans = 64;      // per row: a lane each when they are joined
constexpr int kMinSpan = 2048;     // logits per span at least, and per key that it keeps
constexpr int kSpanPerKey = 128;
constexpr int kAhead = 4;          // vectors a lane reads at once
constexpr int kMaxPlanes = 96;     // state planes per launch: 2.3 KB of kernel arguments

// Vectors per span: whole rounds of 64
template <typename IO>
__device__ __forceinline__ int64_t span_vectors(int64_t V, int spans) {
  const int64_t rounds = (V / kVec<IO> + 63) / 64;
  return (rounds + spans - 1) / spans * 64;
}

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

// the key of one lane (the same for all) in every lane
__device__ __forceinline__ uint64_t lane_key(uint64_t key, int lane) {
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(key >> 32), lane);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(key), lane);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// Two lanes' words that are M apart: in both of them a and b are the two words,
// in some order.  DPP and the row swaps only: no trip through LDS.
template <int M>
__device__ __forceinline__ void pair_words(uint32_t x, uint32_t& a, uint32_t& b) {
  if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    a = r[0];
    b = r[1];
  } else if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    a = r[0];
    b = r[1];
  } else {
    a = x;
    if constexpr (M == 8) {
      b = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), kDppRowRor + 8, 0xF, 0xF, true);
    } else if constexpr (M == 4) {  // banks 1 and 3 read lane - 4, banks 0 and 2 lane + 4
      const int t = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), kDppRowShr + 4, 0xF, 0xA, false);
      b = __builtin_amdgcn_update_dpp(t, static_cast<int>(x), kDppRowShl + 4, 0xF, 0x5, false);
    } else {
      static_assert(M == 1 || M == 2, "a power of two up to 32");
      b = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), M == 1 ? kDppXor1 : kDppXor2, 0xF, 0xF, true);
    }
  }
}
// the larger or the smaller of the keys of this lane and the one M apart
template <int M>
__device__ __forceinline__ uint64_t exchange(uint64_t key, bool larger) {
  uint32_t ah, al, bh, bl;
  pair_words<M>(static_cast<uint32_t>(key >> 32), ah, bh);
  pair_words<M>(static_cast<uint32_t>(key), al, bl);
  const uint64_t a = (static_cast<uint64_t>(ah) << 32) | al, b = (static_cast<uint64_t>(bh) << 32) | bl;
  return (b > a) == larger ? b : a;
}
template <int M>
__device__ __forceinline__ uint32_t exchange(uint32_t x, bool larger) {
  uint32_t a, b;
  pair_words<M>(x, a, b);
  const uint32_t most = a > b ? a : b, least = a > b ? b : a;
  return larger ? most : least;
}
// a bitonic sequence of 2 M lanes into order: the larger keys to the lanes
// whose bit M is 0 where ``down``
template <int M, typename T>
__device__ __forceinline__ T merge_keys(T key, int lane, bool down) {
  key = exchange<M>(key, ((lane & M) == 0) == down);
  if constexpr (M > 1) key = merge_keys<M / 2>(key, lane, down);
  return key;
}
// the wave's 64 keys in descending (or ascending) order of the lanes
template <bool DESCENDING, int SIZE = 64, typename T>
__device__ __forceinline__ T sort_keys(T key, int lane) {
  if constexpr (SIZE > 2) key = sort_keys<DESCENDING, SIZE / 2>(key, lane);
  const bool asked = SIZE == 64 || (lane & SIZE) == 0;  // else this block of lanes the other way round
  return merge_keys<SIZE / 2>(key, lane, asked == DESCENDING);
}

// ---------------------------------------------------------------------------
// the list of the largest
// ---------------------------------------------------------------------------
struct TopList {
  uint64_t list;   // lane i: the i-th largest key so far, 0: none
  uint64_t bound;  // keys at or below it cannot be among the ``want`` largest
  float low;       // nor can later values at or below it (NaN: any can)
  uint32_t held;   // candidates in the buffer (wave-uniform)
  int want;
  uint64_t* buf;   // 128 keys of LDS of this wave

  __device__ __forceinline__ void init(uint64_t* b, int w) {
    list = 0;
    held = 0;
    want = w;
    buf = b;
    set_bound(0);
  }
  __device__ __forceinline__ void set_bound(uint64_t b) {
    bound = b;
    const uint32_t o = static_cast<uint32_t>(b >> 32);
    low = unordered(o == 0x7fffffffu ? o - 1 : o);  // not -0, which is not below 0
  }
  // largest: the ordered bits of the largest of each lane's first values (0:
  // none).  ``want`` values at least are not below the want-th largest of them,
  // here of the lanes of this wave and, with ``shared`` (LDS of a whole
  // workgroup, every wave of which calls this), of the other waves.
  __device__ __forceinline__ void start(uint32_t largest, int lane, uint32_t (*shared)[64] = nullptr, int wave = 0,
                                        int waves = 1) {
    uint32_t v = sort_keys<true>(largest, lane);
    if (shared) {
      shared[wave][lane] = v;
      __syncthreads();
      for (int o = 0; o < waves; ++o) {
        if (o == wave) continue;
        const uint32_t other = shared[o][63 - lane];
        v = merge_keys<32>(other > v ? other : v, lane, true);  // the 64 largest of both
      }
    }
    const uint64_t t = __builtin_amdgcn_readlane(v, want - 1);
    set_bound(t ? (t << 32) - 1 : 0);
  }
  __device__ __forceinline__ void merge(uint64_t cand, int lane) {
    cand = sort_keys<false>(cand, lane);
    list = merge_keys<32>(list > cand ? list : cand, lane, true);  // the 64 largest of both, bitonic
    const uint64_t b = lane_key(list, want - 1);
    if (b > bound) set_bound(b);
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

// Lists of ``len`` keys each, one behind the other (up to 64 lists), larger keys
// first or nearly so, and the largest of them all.
struct KeyLists {
  static constexpr int kAtOnce = 8;
  const uint64_t* keys;
  int lists, len;
  uint64_t head, key[kAtOnce];  // the lists' first keys, and the keys in hand

  __device__ __forceinline__ void load(int i0, int lane) {
    const int n = lists * len;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * 64 + lane;
      key[u] = keys[i < n ? i : n - 1];
    }
  }
  __device__ __forceinline__ KeyLists(const uint64_t* k, int ls, int ln, int lane) : keys(k), lists(ls), len(ln) {
    const int j = lane / lists;  // lane: key j of a list
    head = keys[j < len ? (lane - j * lists) * len + j : 0];
    if (j >= len) head = 0;
    load(0, lane);
  }
  // into the list, whose bound starts at the want-th largest of the first keys
  __device__ __forceinline__ void into(TopList& top, int lane) {
    const int n = lists * len;
    top.start(static_cast<uint32_t>(head >> 32), lane);
    for (int i0 = 0; i0 < n; i0 += 64 * kAtOnce) {
      if (i0 > 0) load(i0, lane);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (i0 + u * 64 < n) top.push(i0 + u * 64 + lane < n ? key[u] : 0, lane);
      }
    }
    top.finish(lane);
  }
};

// ---------------------------------------------------------------------------
// the scan of the logits
// ---------------------------------------------------------------------------
// Value i of a vector, i differing between lanes (an array indexed by it would
// go through memory)
template <typename IO>
__device__ __forceinline__ float pick(const Vec<IO>& r, int i) {
  if constexpr (sizeof(IO) == 4) {
    const float a = i & 1 ? r.y : r.x, b = i & 1 ? r.w : r.z;
    return i & 2 ? b : a;
  } else {
    const uint32_t a = i & 2 ? r.y : r.x, b = i & 2 ? r.w : r.z, c = i & 4 ? b : a;
    return __uint_as_float(i & 1 ? c & 0xffff0000u : c << 16);
  }
}

// A row of V logits in whole vectors of 16 bytes, at any alignment, and the
// V % VEC values behind them.
template <typename IO>
struct Row {
  static constexpr int VEC = kVec<IO>;
  const void* logits;
  int64_t offset, V;

  __device__ __forceinline__ int64_t vectors() const { return V / VEC; }
  __device__ __forceinline__ Vec<IO> load(int64_t j) const { return load_vec<IO, true>(logits, offset + j * VEC, VEC); }
  // the values behind the vectors, one per lane, -inf in the other lanes
  __device__ __forceinline__ float rest(int lane, int64_t& at) const {
    at = vectors() * VEC + lane;
    return at < V ? load1<IO>(logits, offset + at) : -INFINITY;
  }
  // Those of a vector's values x for which may(x) holds into the list, as
  // make(x); ``in``: this lane has a vector.  Few lanes hold any such value, so
  // every turn takes one from each lane that does, not one place of all lanes.
  template <typename P, typename F>
  __device__ __forceinline__ void push(TopList& top, bool in, int64_t j, const Vec<IO>& raw, int lane, P&& may,
                                       F&& make) const {
    uint32_t pass = 0;
    {
      float x[VEC];
      unpack<IO, VEC>(raw, x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) pass |= in && may(x[i]) ? 1u << i : 0u;
    }
    while (__any(pass != 0)) {
      const int i = __ffs(static_cast<int>(pass)) - 1;
      top.push(pass ? make_key(make(pick<IO>(raw, i)), static_cast<uint32_t>(j * VEC + i)) : 0, lane);
      pass &= pass - 1;
    }
  }
};

constexpr float kLog2E = 1.4426950408889634f;       // rounded to fp32
constexpr float kLog2ELow = 1.9259629911e-8f;       // and what is left of it
constexpr float kHuge = 1e38f;                      // beyond it x log2(e) may overflow

// A lane's maximum m and sum s of 2^(x log2(e) - m log2(e)), the product of m
// rounded: one fused multiply-add and one exponential per value.
struct SumExp {
  float m, s;

  // ``in``: the values count
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float big, bool in) {
#pragma clang fp contract(off)  // m log2(e) rounds the same way each time it is formed
    const float mn = in ? fmaxf(m, big) : m;
    const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing but -inf so far: every power is 0
    float sum = 0.0f;
    if (__any(fabsf(ref) > kHuge)) {
#pragma unroll
      for (int i = 0; i < N; ++i) sum += fast_exp(x[i] - ref);
      s = fmaf(s, fast_exp(m - ref), in ? sum : 0.0f);
    } else {
      const float r = ref * kLog2E;
#pragma unroll
      for (int i = 0; i < N; ++i) sum += __builtin_amdgcn_exp2f(fmaf(x[i], kLog2E, -r));
      s = fmaf(s, __builtin_amdgcn_exp2f(m * kLog2E - r), in ? sum : 0.0f);
    }
    m = mn;
  }
  // The maximum over the wave, and the sum of e^(x - maximum) over it: the
  // maximum's product with log2(e) is taken to twice fp32's precision here, so
  // that what the lanes' products were rounded by does not stay in the sum.
  __device__ __forceinline__ void join(float& all, float& sum) const {
#pragma clang fp contract(off)
    all = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
    const float ref = all == -INFINITY ? 0.0f : all;
    float f;
    if (fabsf(ref) > kHuge) {
      f = fast_exp(m - ref);
    } else {
      const float r = ref * kLog2E;
      f = __builtin_amdgcn_exp2f((m * kLog2E - r) - fmaf(ref, kLog2ELow, fmaf(ref, kLog2E, -r)));
    }
    sum = group_sum(m == -INFINITY ? s : s * f, 64);  // s: 0, or NaN
  }
};

// 1024 rows of 131072 bf16 logits 62 us (269 MB, read once: 4.3 TB/s): some 10 us
// of lists' starts and ends, and 5.3 TB/s between them; the VALU is 70 % busy, but a
// maximum less per logit and a rescaling less per vector took no time out.  160
// rows of 50001 fp32 ones 14 us, of which reading is 5: the sorts and merges of the
// lists, a chain of some 60 exchanges per wave, are the rest; 4 rows of 32768 6.6.
// parts: [rows][spans] (maximum, sum of exp(x - maximum)); tops: [rows][spans][want] keys
template <typename IO>
__global__ void __launch_bounds__(64 * kScanWaves, 4)
beam_scan_kernel(int64_t rows, int64_t V, int64_t ld, int spans, int want, const void* logits, float2* parts,
                 uint64_t* tops) {
  __shared__ uint64_t buf[kScanWaves][128];
  __shared__ uint32_t first[kScanWaves][64];
  constexpr int VEC = kVec<IO>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * kScanWaves + wave;
  const bool together = spans % kScanWaves == 0;  // the workgroup's waves share a row: they meet once
  if (job >= rows * spans) return;                // not where they do
  const int64_t r = job / spans;
  const int span = static_cast<int>(job - r * spans);
  const Row<IO> row{logits, r * ld, V};
  const int64_t per = span_vectors<IO>(V, spans), begin = span * per;
  const int64_t end = begin + per < row.vectors() ? begin + per : row.vectors();
  TopList top;
  top.init(buf[wave], want);
  const auto may = [&](float v) { return !(v <= top.low); };
  const auto same = [](float v) { return v; };
  SumExp acc{-INFINITY, 0.0f};
  // Loads past the span's end repeat its last vector: without a branch around
  // them the wave waits for the one it needs, not for all that it has issued.
  const auto load = [&](int64_t j) { return row.load(j < end ? j : end - 1); };
  Vec<IO> raw[kAhead] = {};
  if (begin < end) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = load(begin + u * 64 + lane);
  }
  uint32_t largest = 0;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    float x[VEC], big;
    unpack<IO, VEC>(raw[u], x);
    big = x[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
    const uint32_t o = begin + u * 64 + lane < end ? ordered(big) : 0;
    largest = o > largest ? o : largest;
  }
  top.start(largest, lane, together ? first : nullptr, wave, kScanWaves);
  for (int64_t j0 = begin; j0 < end; j0 += kAhead * 64) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t j = j0 + u * 64 + lane;
      const bool in = j < end;
      const Vec<IO> now = raw[u];
      // the vector of the next round, while this one is worked on
      raw[u] = load(j + kAhead * 64);
      float x[VEC];
      unpack<IO, VEC>(now, x);
      float big = x[0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
      if (__any(in && may(big))) row.push(top, in, j, now, lane, may, same);
      acc.add(x, big, in);
    }
  }
  if (span == spans - 1 && V % VEC != 0) {
    int64_t at;
    const float x = row.rest(lane, at);
    top.push(at < V ? make_key(x, static_cast<uint32_t>(at)) : 0, lane);
    const float one[1] = {x};
    acc.add(one, x, true);
  }
  top.finish(lane);
  float all, sum;
  acc.join(all, sum);
  if (lane == 0) parts[job] = make_float2(all, sum);
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

// the bits of the first kMostJoinWaves lanes together
__device__ __forceinline__ uint32_t bits_of(uint32_t v) {
#pragma unroll
  for (int o = kMostJoinWaves / 2; o > 0; o >>= 1) v |= __shfl_xor(v, o);
  return __builtin_amdgcn_readfirstlane(v);
}

// A workgroup per batch row, a wave per beam in turn.  7 to 8 us for up to 8 beams,
// 20 for 32: chains of sorts in few waves, bound by latency.  (A row that is ranked
// by score took 280 us more for 70581 logits when its one wave read it.)
template <typename IO>
__global__ void __launch_bounds__(64 * kMostJoinWaves)
beam_join_kernel(BeamStep p) {
  __shared__ uint64_t buf[kMostJoinWaves][128];
  __shared__ uint64_t cand[kMaxBeams * (kMaxBeams + 1)];
  __shared__ float lse_of[kMaxBeams], least_of[kMaxBeams];
  __shared__ uint32_t again_of[kMostJoinWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int waves = static_cast<int>(blockDim.x >> 6), K = p.beams;
  const int keep = p.V < K ? static_cast<int>(p.V) : K;  // candidates of a beam that can count
  const int64_t b = blockIdx.x;
  uint32_t again = 0;  // bit k: beam k's row is ranked by score
  for (int k = wave; k < K; k += waves) {
    const int64_t r = b * K + k;
    // everything is read at once, whichever of it counts
    KeyLists found(p.tops + r * p.spans * p.want, p.spans, p.want, lane);
    const float2 part = p.parts[r * p.spans + (lane < p.spans ? lane : 0)];
    const float cum = p.scores[r];
    const bool finished = p.finished && p.finished[r];
    const uint32_t flat = static_cast<uint32_t>(k * p.V);
    uint64_t mine = 0;  // lane i: the beam's i-th candidate
    if (finished) {
      // (eos, cum), and -inf for every other token
      if (lane < keep && lane != p.eos) mine = make_key(-INFINITY, flat + lane);
      if (lane == K && p.eos >= 0) mine = make_key(cum, flat + static_cast<uint32_t>(p.eos));
    } else {
      const float own = lane < p.spans ? part.x : -INFINITY;
      float m = own;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
      const float s = group_sum(lane < p.spans ? part.y * fast_exp(own - (m == -INFINITY ? 0.0f : m)) : 0.0f, 64);
      // without a finite logit the beam is empty: every candidate -inf
      const bool empty = m == -INFINITY && s == 0.0f;
      const float lse = m + logf(s);
      if (empty || lse != lse || cum != cum || cum == -INFINITY) {  // one score for all
        if (lane < keep) mine = make_key(empty ? cum - INFINITY : cum + (0.0f - lse), flat + lane);
      } else {
        const auto score = [&](float x) { return cum + (x - lse); };
        TopList top;
        top.init(buf[wave], p.want);
        found.into(top, lane);
        const float low = key_value(lane_key(top.list, keep - 1));
        bool more = cum == INFINITY;
        if (p.V > K) {
          const float left = key_value(lane_key(top.list, K));
          more = more || score(left == low ? next_below<IO>(low) : left) == score(low);
        }
        again |= more ? 1u << k : 0u;
        if (lane < keep) mine = make_key(score(key_value(top.list)), flat + key_index(top.list));
        if (lane == 0) {
          lse_of[k] = lse;
          least_of[k] = cum == INFINITY ? -INFINITY : score(low);
        }
      }
    }
    if (lane <= K) cand[k * (K + 1) + lane] = mine;
  }
  if (lane == 0) again_of[wave] = again;
  __syncthreads();
  // the rows that are ranked by score, all waves together: only values whose
  // score reaches the one found count
  again = bits_of(lane < waves ? again_of[lane] : 0);
  for (; again; again &= again - 1) {  // uniform over the workgroup
    const int k = __ffs(static_cast<int>(again)) - 1;
    const Row<IO> row{p.logits, (b * K + k) * p.ld, p.V};
    const float cum = p.scores[b * K + k], lse = lse_of[k], least = least_of[k];
    const auto score = [&](float x) { return cum + (x - lse); };
    const auto may = [&](float x) { return !(score(x) < least); };
    const int64_t vectors = row.vectors(), step = static_cast<int64_t>(waves) * 64;
    TopList top;
    top.init(buf[wave], keep);
    for (int64_t j0 = wave * 64; j0 < vectors; j0 += step * kAhead) {
      Vec<IO> raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t j = j0 + u * step + lane;
        raw[u] = row.load(j < vectors ? j : vectors - 1);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t j = j0 + u * step + lane;
        row.push(top, j < vectors, j, raw[u], lane, may, score);
      }
    }
    if (wave == 0) {
      int64_t at;
      const float x = row.rest(lane, at);
      top.push(at < p.V ? make_key(score(x), static_cast<uint32_t>(at)) : 0, lane);
    }
    top.finish(lane);
    buf[wave][lane] = top.list;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < waves; ++w) {
        const uint64_t other = buf[w][63 - lane];
        top.list = merge_keys<32>(top.list > other ? top.list : other, lane, true);
      }
      const uint32_t flat = static_cast<uint32_t>(k * p.V);
      if (lane < keep) cand[k * (K + 1) + lane] = make_key(key_value(top.list), flat + key_index(top.list));
    }
    __syncthreads();
  }
  if (wave > 0) return;
  TopList top;
  top.init(buf[0], K);
  KeyLists(cand, K, K + 1, lane).into(top, lane);
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
};
template <int B> struct Bytes;
template <> struct Bytes<16> { typedef uint32_t T __attribute__((ext_vector_type(4))); };
template <> struct Bytes<4> { using T = uint32_t; };
template <> struct Bytes<2> { using T = uint16_t; };

// Bound by memory: 4 planes of 1024 rows of 131 KB copied in 134 us (537 MB written,
// 176 read: beams share parents), 6 planes of 160 rows of 12 KB in place in 6 us.
//
// In place: batch rows blockIdx.y, + gridDim.y, ..., of plane blockIdx.z; a
// thread moves one access of B bytes of all K rows of a batch row and reads them
// all before it writes.  Rows that stay are left alone.  KM >= K.  A parent
// outside the beams fills its row with ones (NaN).
template <int B, int KM>
__global__ void __launch_bounds__(256)
reorder_in_place_kernel(Planes pl, int K, int batch, const int64_t* parents) {
  using T = typename Bytes<B>::T;
  const int lane = threadIdx.x & 63;
  const int64_t rb = pl.row_bytes[blockIdx.z], tile = static_cast<int64_t>(blockIdx.x) * (256 * B);
  const uint32_t t = threadIdx.x * B;
  char* const plane = static_cast<char*>(pl.dst[blockIdx.z]) + tile;
  for (int b = blockIdx.y; b < batch; b += gridDim.y) {
    // one load for all parents, every lane of the wave with it
    const int64_t own = parents[b * K + (lane < K ? lane : 0)];
    const int from = own >= 0 && own < K ? static_cast<int>(own) : -1;
    int p[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k) p[k] = k < K ? __builtin_amdgcn_readlane(from, k) : k;
    if (tile + t >= rb) continue;
    char* const col = plane + static_cast<int64_t>(b) * K * rb;
    T v[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k)
      if (p[k] >= 0 && p[k] != k) v[k] = *reinterpret_cast<const T*>(col + p[k] * rb + t);
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (p[k] == k) continue;
      if (p[k] < 0) v[k] = ~T(0);
      *reinterpret_cast<T*>(col + k * rb + t) = v[k];
    }
  }
}

// The same where few workgroups would result: 64 accesses of all K rows per
// workgroup, each of its 4 waves PW rows (4 PW >= K), so that no thread's chain of
// accesses is long (2 x 30 beams, 2 planes of 640 bytes: 4.1 us, 8.2 with all rows
// in a thread; 14 planes of 540 rows of 27 KB: 86 and 73).
constexpr int kSplitWaves = 4;
template <int B, int PW>
__global__ void __launch_bounds__(64 * kSplitWaves)
reorder_split_kernel(Planes pl, int K, int batch, const int64_t* parents) {
  using T = typename Bytes<B>::T;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t rb = pl.row_bytes[blockIdx.z], tile = static_cast<int64_t>(blockIdx.x) * (64 * B);
  if (tile >= rb) return;
  const uint32_t t = lane * B;
  const bool in = tile + t < rb;
  char* const plane = static_cast<char*>(pl.dst[blockIdx.z]) + tile;
  for (int b = blockIdx.y; b < batch; b += gridDim.y) {
    const int64_t own = parents[b * K + (lane < K ? lane : 0)];
    const int from = own >= 0 && own < K ? static_cast<int>(own) : -1;
    char* const col = plane + static_cast<int64_t>(b) * K * rb;
    int p[PW];
    T v[PW];
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int k = i * kSplitWaves + wave;
      p[i] = k < K ? __builtin_amdgcn_readlane(from, k) : k;
      if (p[i] >= 0 && p[i] != k && in) v[i] = *reinterpret_cast<const T*>(col + p[i] * rb + t);
    }
    __syncthreads();  // all rows are read
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int k = i * kSplitWaves + wave;
      if (p[i] == k || !in) continue;
      if (p[i] < 0) v[i] = ~T(0);
      *reinterpret_cast<T*>(col + k * rb + t) = v[i];
    }
  }
}

// To other memory: rows blockIdx.y, + gridDim.y, ..., of plane blockIdx.z; a
// workgroup copies kCopy accesses per thread of one row.
constexpr int kCopy = 4;
template <int B, int THREADS>
__global__ void __launch_bounds__(THREADS)
reorder_copy_kernel(Planes pl, int K, int rows, const int64_t* parents) {
  using T = typename Bytes<B>::T;
  const int64_t rb = pl.row_bytes[blockIdx.z], step = THREADS * B, tile = blockIdx.x * (step * kCopy);
  if (tile >= rb) return;
  const uint32_t t = threadIdx.x * B;
  const char* const from = static_cast<const char*>(pl.src[blockIdx.z]) + tile;
  char* const to = static_cast<char*>(pl.dst[blockIdx.z]) + tile;
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    const int64_t p = parents[row];
    const char* const src = from + (row / K * K + p) * rb;
    T v[kCopy];
#pragma unroll
    for (int i = 0; i < kCopy; ++i) {
      v[i] = ~T(0);
      if (p >= 0 && p < K && tile + i * step + t < rb) v[i] = *reinterpret_cast<const T*>(src + i * step + t);
    }
#pragma unroll
    for (int i = 0; i < kCopy; ++i)
      if (tile + i * step + t < rb) *reinterpret_cast<T*>(to + row * rb + i * step + t) = v[i];
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
sparc_status bm_check(int64_t batch, int64_t beams, int64_t vocab) {
  if (batch < 0 || beams < 1 || beams > kMaxBeams || vocab < 1)
    return op_fail(SPARC_EINVAL, "beam step: batch >= 0, 1 to 32 beams and vocab > 0 required");
  if (batch > (int64_t(1) << 22) / beams || vocab > INT32_MAX / beams)
    return op_fail(SPARC_EINVAL, "beam step: too large");
  return SPARC_OK;
}
// Spans per row, none shorter than kMinSpan: the whole workgroups per row that
// come nearest to 4096 waves in all (16 per CU, what their registers allow), or 1
// or 2 waves with more rows than 2048.  (537 rows of 114015 bf16 logits: 41 us
// with 4 spans, 37 with 8; 64 rows of 107383, 33 keys each: both kernels 36 us
// with 52 spans, 29 with 24.)
int spans_of(int64_t rows, int64_t want, int64_t vocab) {
  constexpr int64_t kWaves = 4096;
  const int64_t r = rows > 0 ? rows : 1, groups = (kWaves + kScanWaves / 2 * r) / (kScanWaves * r);
  int64_t s = groups > 0 ? groups * kScanWaves : (kWaves + r / 2) / r;
  const int64_t least = want * kSpanPerKey > kMinSpan ? want * kSpanPerKey : kMinSpan;
  const int64_t most = (vocab + least - 1) / least;
  s = s < most ? s : most;
  s = s < 1 ? 1 : (s < kMaxSpans ? s : kMaxSpans);
  return static_cast<int>(s < kScanWaves ? s : s / kScanWaves * kScanWaves);
}

// Copies of short rows take workgroups of 64 threads (10 planes of 1080 rows of
// 1280 bytes: 6 us, with 256 threads, most of them idle, 14).
template <int B>
void launch_reorder(hipStream_t st, const Planes& pl, int count, int64_t widest, bool in_place, int K, int batch,
                    const int64_t* parents) {
  const int rows = in_place ? batch : batch * K, threads = !in_place && widest <= 64 * B * kCopy ? 64 : 256;
  const bool split = in_place && (widest + 256 * B - 1) / (256 * B) * rows * count < 1024;
  const int64_t tile = static_cast<int64_t>(split ? 64 : threads) * B * (in_place ? 1 : kCopy);
  const dim3 grid(static_cast<unsigned>((widest + tile - 1) / tile), rows < 65535 ? rows : 65535, count);
  const dim3 block(threads);
  if (threads == 64) hipLaunchKernelGGL((reorder_copy_kernel<B, 64>), grid, block, 0, st, pl, K, rows, parents);
  else if (!in_place) hipLaunchKernelGGL((reorder_copy_kernel<B, 256>), grid, block, 0, st, pl, K, rows, parents);
  else if (split && K <= 4)
    hipLaunchKernelGGL((reorder_split_kernel<B, 1>), grid, block, 0, st, pl, K, batch, parents);
  else if (split && K <= 8)
    hipLaunchKernelGGL((reorder_split_kernel<B, 2>), grid, block, 0, st, pl, K, batch, parents);
  else if (split && K <= 16)
    hipLaunchKernelGGL((reorder_split_kernel<B, 4>), grid, block, 0, st, pl, K, batch, parents);
  else if (split) hipLaunchKernelGGL((reorder_split_kernel<B, 8>), grid, block, 0, st, pl, K, batch, parents);
  else if (K <= 4) hipLaunchKernelGGL((reorder_in_place_kernel<B, 4>), grid, block, 0, st, pl, K, batch, parents);
  else if (K <= 8) hipLaunchKernelGGL((reorder_in_place_kernel<B, 8>), grid, block, 0, st, pl, K, batch, parents);
  else if (K <= 16) hipLaunchKernelGGL((reorder_in_place_kernel<B, 16>), grid, block, 0, st, pl, K, batch, parents);
  else hipLaunchKernelGGL((reorder_in_place_kernel<B, 32>), grid, block, 0, st, pl, K, batch, parents);
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
  const int64_t rows = batch * beams, spans = spans_of(rows, beams + 1, vocab);
  return up256(rows * spans * sizeof(float2)) + up256(rows * spans * (beams + 1) * sizeof(uint64_t)) + 256;
}

sparc_status sparc_beam_step(int64_t batch, int64_t beams, int64_t vocab, int64_t row_stride, int32_t io_dtype,
                             const void* logits, const float* scores, const uint8_t* finished, int64_t eos_id,
                             int64_t* tokens, int64_t* parents, float* new_scores, uint8_t* new_finished,
                             void* workspace, size_t workspace_bytes, sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = bm_check(batch, beams, vocab)) return s;
  if (io_dtype != SPARC_F32 && io_dtype != SPARC_BF16) return op_fail(SPARC_EINVAL, "beam step: unknown io_dtype");
  if (row_stride < vocab) return op_fail(SPARC_EINVAL, "beam step: row_stride below vocab");
  if (eos_id < -1 || eos_id >= vocab) return op_fail(SPARC_EINVAL, "beam step: eos_id outside the vocabulary");
  if (finished && eos_id < 0) return op_fail(SPARC_EINVAL, "beam step: finished beams need an eos_id");
  if (batch == 0) return SPARC_OK;
  if (!logits || !scores || !tokens || !parents || !new_scores) return op_fail(SPARC_EINVAL, "beam step: NULL pointer");
  if (!workspace || workspace_bytes < sparc_beam_workspace_bytes(batch, beams, vocab))
    return op_fail(SPARC_EWORKSPACE, "beam step: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8)
    return op_fail(SPARC_EINVAL, "beam step: the workspace must be 8-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t rows = batch * beams;
  const int spans = spans_of(rows, beams + 1, vocab), want = static_cast<int>(beams) + 1;
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
  const dim3 join(static_cast<unsigned>(batch)), jblock(64 * (beams <= 8 ? 8 : kMostJoinWaves));
  if (io_dtype == SPARC_F32) {
    hipLaunchKernelGGL((beam_scan_kernel<float>), grid, block, 0, st, rows, vocab, row_stride, spans, want, logits,
                       parts, tops);
    hipLaunchKernelGGL((beam_join_kernel<float>), join, jblock, 0, st, p);
  } else {
    hipLaunchKernelGGL((beam_scan_kernel<sparc::bf16>), grid, block, 0, st, rows, vocab, row_stride, spans, want,
                       logits, parts, tops);
    hipLaunchKernelGGL((beam_join_kernel<sparc::bf16>), join, jblock, 0, st, p);
  }
  return op_launched("beam step");
}

sparc_status sparc_reorder_states(int64_t batch, int64_t beams, int64_t count, const void* const* src,
                                  void* const* dst, const int64_t* row_bytes, const int64_t* parents,
                                  sparc_stream_t stream) {
  using namespace sparc;
  if (batch < 0 || beams < 1 || beams > kMaxBeams || count < 0 || batch > (int64_t(1) << 22) / beams)
    return op_fail(SPARC_EINVAL, "reorder states: batch >= 0, 1 to 32 beams and count >= 0 required");
  if (batch == 0 || count == 0) return SPARC_OK;
  if (!src || !dst || !row_bytes || !parents) return op_fail(SPARC_EINVAL, "reorder states: NULL pointer");
  for (int64_t i = 0; i < count; ++i) {
    if (row_bytes[i] < 0 || row_bytes[i] % 2 || row_bytes[i] > (int64_t(1) << 31))
      return op_fail(SPARC_EINVAL, "reorder states: rows of an even number of bytes up to 2^31 required");
    if (row_bytes[i] > 0 && (!src[i] || !dst[i])) return op_fail(SPARC_EINVAL, "reorder states: NULL plane");
    if ((reinterpret_cast<uintptr_t>(src[i]) | reinterpret_cast<uintptr_t>(dst[i])) % 2)
      return op_fail(SPARC_EINVAL, "reorder states: planes must be 2-byte aligned");
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  Planes pl;
  // planes of one access width, in place or not, share launches
  for (const bool in_place : {false, true}) {
    for (const int access : {16, 4, 2}) {
      for (int64_t at = 0; at < count;) {
        int n = 0;
        int64_t widest = 0;
        for (; at < count && n < kMaxPlanes; ++at) {
          if (row_bytes[at] == 0 || (src[at] == dst[at]) != in_place ||
              plane_access(src[at], dst[at], row_bytes[at]) != access)
            continue;
          pl.src[n] = src[at];
          pl.dst[n] = dst[at];
          pl.row_bytes[n++] = row_bytes[at];
          widest = row_bytes[at] > widest ? row_bytes[at] : widest;
        }
        if (n == 0) break;
        const int K = static_cast<int>(beams), rows = static_cast<int>(batch);
        if (access == 16) launch_reorder<16>(st, pl, n, widest, in_place, K, rows, parents);
        else if (access == 4) launch_reorder<4>(st, pl, n, widest, in_place, K, rows, parents);
        else launch_reorder<2>(st, pl, n, widest, in_place, K, rows, parents);
      }
    }
  }
  return op_launched("reorder states");
}

}  // extern "C"
