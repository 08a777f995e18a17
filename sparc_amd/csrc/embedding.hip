// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   forward   y[n] = scale W[t_n]
//   backward  dW[v] = scale sum over n with t_n = v of dy[n], for every row v
//
// Rows in the I/O type, sums in fp32 rounded once.  An id outside [0, vocab)
// gives a row of NaN and takes no part in the gradient; the padding row gets a
// gradient of zero.
//
// The backward sorts the token positions by id (a stable radix sort, digits of
// up to 9 bits: two passes up to 2^18 ids), so that the positions of one id
// stand together in their order in the batch.  Up to kFew positions one launch
// does it all; up to 4096 one workgroup sorts them in LDS, ids and positions packed
// into 32 bits; more of them, or ids that do not fit beside the positions, take a
// counting and a scattering launch per pass (and one between them with many tiles).
// Pieces of sorted positions are then summed side by side, whatever the ids'
// frequencies: a run of equal ids inside a piece is written to its row at once; a
// run that crosses pieces leaves one fp32 partial row per piece, joined in order by
// a second kernel.  Every sum has a fixed order, so dW does not depend on timing.
// The sort keeps few CUs busy and is bound by latency, so further workgroups of its
// launches clear dW meanwhile, a share each; the rows that tokens name are then
// written once more.

#include "rows.h"

namespace sparc {
namespace {

constexpr int kBatch = 8;           // sorted positions that a lane reads at once
constexpr int kSortThreads = 256;   // 4 waves per sort tile
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kMaxDigits = 512;     // 9 bits
constexpr int kLocalThreads = 1024; // the sort in LDS
constexpr int kLocalWaves = kLocalThreads / 64;
constexpr int kLocalItems = 4;      // per thread
constexpr int kJoinWaves = 8;       // pieces per join workgroup
constexpr int kLongRun = 16;        // pieces of a run that a whole join workgroup adds up
// With more tiles than that a launch of its own sums their counts, else every
// scattering workgroup does (65 tiles: 28 against 31 us; 256: 48 against 33).
constexpr int kManyTiles = 96;
constexpr uint32_t kNone = 0xffffffffu;

// Jobs of a group of lpr lanes (a power of two up to 64): one block of NV lpr
// 16-byte vectors of one row, NV per lane and lpr apart.
struct Jobs {
  int D, lpr, blocks;  // blocks per row

  // the row and first column of this lane's part of a job
  template <int V, int NV = 1>
  __device__ __forceinline__ int64_t row_of(int64_t job, int& c) const {
    const int64_t row = blocks == 1 ? job : job / blocks;
    c = (static_cast<int>(job - row * blocks) * NV * lpr + static_cast<int>(threadIdx.x & (lpr - 1))) * V;
    return row;
  }
};

// Scaled copies of table rows, a group per job.  Bound by memory: 32768 x 768 bf16
// 17 us (50 MB written, the rows named in 26 MB of a table that is read out of
// caches), 65536 x 1024 35 us; 256 rows 3.7 us.
template <typename IO, int NV>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(int64_t N, int64_t vocab, Jobs jb, const void* tokens, int wide_ids, const void* w, float scale,
                 void* y) {
  constexpr int V = kVec<IO>;
  const int64_t per = 256 / jb.lpr, jobs = N * jb.blocks;
  for (int64_t job = blockIdx.x * per + threadIdx.x / jb.lpr; job < jobs; job += gridDim.x * per) {
    int c0;
    const int64_t n = jb.row_of<V, NV>(job, c0);
    const int64_t id = wide_ids ? static_cast<const int64_t*>(tokens)[n] : static_cast<const int32_t*>(tokens)[n];
    const bool known = id >= 0 && id < vocab;
    Vec<IO> raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * jb.lpr * V;
      if (known && c < jb.D) raw[k] = load_vec<IO>(w, id * jb.D + c, jb.D - c);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * jb.lpr * V;
      if (c >= jb.D) break;
      float v[V];
      unpack<IO, V>(raw[k], v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = known ? v[i] * scale : __uint_as_float(0x7fc00000u);
      store_vec<IO>(y, n * jb.D + c, jb.D - c, pack<IO, V>(v));
    }
  }
}

// ---------------------------------------------------------------------------
// the sort
// ---------------------------------------------------------------------------
struct SortPass {
  const void* tokens;     // the first pass reads ids, later ones keys
  int wide_ids;
  int64_t vocab, pad;
  const uint32_t* keys_in;
  const uint32_t* pos_in;
  uint32_t* keys_out;
  uint32_t* pos_out;
  uint32_t* counts;       // [tiles][digits] of this pass
  uint32_t* totals;       // [digits]; NULL: the counts are not yet summed over the tiles
  int64_t n;
  int shift, bits;
  int first;
  int tiles;              // sorting workgroups; those behind them clear
  char* dw;               // this launch's share of dW, in bytes
  int64_t dw_bytes;

  // by the workgroups behind the sorting ones, a stretch each (1 GB: 207 us; every
  // workgroup's stores spread over all of it 267)
  __device__ __forceinline__ void clear() const { clear(blockIdx.x - tiles, gridDim.x - tiles); }
  // by workgroup g of ``groups``
  __device__ __forceinline__ void clear(int64_t g, int64_t groups) const {
    const uintptr_t at = reinterpret_cast<uintptr_t>(dw);
    const int64_t head = static_cast<int64_t>((16 - at % 16) % 16) < dw_bytes ? (16 - at % 16) % 16 : dw_bytes;
    const int64_t vecs = (dw_bytes - head) / 16, tail = head + vecs * 16, each = (vecs + groups - 1) / groups;
    const int64_t end = (g + 1) * each < vecs ? (g + 1) * each : vecs;
    const int t = threadIdx.x;
    uint4* const body = reinterpret_cast<uint4*>(dw + head);
    for (int64_t v = g * each + t; v < end; v += blockDim.x) body[v] = make_uint4(0, 0, 0, 0);
    if (g == 0 && t < head) dw[t] = 0;
    if (g == 0 && tail + t < dw_bytes) dw[tail + t] = 0;
  }
  // The keys of ITEMS positions from ``at`` on, ``step`` apart, all read at
  // once.  A key is the position's id, or vocab (behind every row) where it
  // takes no part in the gradient; past the end it repeats the last one's.
  template <int ITEMS>
  __device__ __forceinline__ void load_keys(int64_t at, int64_t step, uint32_t (&key)[ITEMS]) const {
    int64_t i[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) i[k] = at + k * step < n ? at + k * step : n - 1;
    if (!first) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) key[k] = keys_in[i[k]];
      return;
    }
    int64_t id[ITEMS];
    if (wide_ids) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) id[k] = static_cast<const int64_t*>(tokens)[i[k]];
    } else {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) id[k] = static_cast<const int32_t*>(tokens)[i[k]];
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      key[k] = static_cast<uint32_t>(id[k] >= 0 && id[k] < vocab && id[k] != pad ? id[k] : vocab);
  }
};

// Digit counts of each tile of kSortThreads * ITEMS positions: 3 us for 32768, a
// launch and two trips to memory.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(SortPass p) {
  __shared__ uint32_t hist[kMaxDigits];
  if (static_cast<int>(blockIdx.x) >= p.tiles) return p.clear();
  const int digits = 1 << p.bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kSortThreads * ITEMS) + threadIdx.x;
  uint32_t key[ITEMS];
  p.load_keys<ITEMS>(base, kSortThreads, key);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (base + i * kSortThreads < p.n) atomicAdd(&hist[(key[i] >> p.shift) & (digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads)
    p.counts[static_cast<int64_t>(blockIdx.x) * digits + d] = hist[d];
}

// With many tiles: turns each tile's counts into those of the tiles before it, and
// leaves the digits' totals.  kScanDigits digits per workgroup, each by
// kScanSlices slices of the tiles.
constexpr int kScanDigits = 16;
constexpr int kScanSlices = 64;
__global__ void __launch_bounds__(kScanDigits * kScanSlices)
sort_scan_kernel(SortPass p) {
  __shared__ uint32_t sums[kScanSlices][kScanDigits];
  const int digits = 1 << p.bits, d = threadIdx.x % kScanDigits, slice = threadIdx.x / kScanDigits;
  const int digit = blockIdx.x * kScanDigits + d, each = (p.tiles + kScanSlices - 1) / kScanSlices;
  const int t0 = slice * each, t1 = t0 + each < p.tiles ? t0 + each : p.tiles;
  uint32_t* const at = p.counts + (digit < digits ? digit : 0);
  uint32_t sum = 0;
  for (int t = t0; t < t1; ++t) sum += at[static_cast<int64_t>(t) * digits];
  sums[slice][d] = sum;
  __syncthreads();
  if (digit >= digits) return;
  uint32_t before = 0;
  for (int k = 0; k < slice; ++k) before += sums[k][d];
  for (int t = t0; t < t1; ++t) {
    const uint32_t own = at[static_cast<int64_t>(t) * digits];
    at[static_cast<int64_t>(t) * digits] = before;
    before += own;
  }
  if (slice == kScanSlices - 1) p.totals[digit] = before;
}

// Moves each tile's positions behind all positions of smaller digits and those
// of its own digit in earlier tiles.  A wave ranks its 64 * ITEMS consecutive
// positions 64 at a time: the lanes of equal digit are found by one ballot per
// digit bit, and a counter per wave and digit in LDS carries the rank on.  32768
// positions 7 us (a chain of some 40 ballots, LDS and memory accesses, bound by
// their latency), 10 us while the other workgroups clear 25 MB.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(SortPass p) {
  __shared__ uint32_t cnt[kSortWaves][kMaxDigits];  // counts, then the waves' first places
  __shared__ uint32_t start[kMaxDigits];            // this tile's first place of each digit
  __shared__ uint32_t wsum[kSortWaves];
  if (static_cast<int>(blockIdx.x) >= p.tiles) return p.clear();
  const int digits = 1 << p.bits;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kSortThreads * ITEMS) + wave * (64 * ITEMS) + lane;
  uint32_t key[ITEMS], pos[ITEMS];
  p.load_keys<ITEMS>(first, 64, key);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t n = first + i * 64 < p.n ? first + i * 64 : p.n - 1;
    pos[i] = static_cast<uint32_t>(n);
    if (!p.first) pos[i] = p.pos_in[n];
  }
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) cnt[w][d] = 0;
  }
  // a thread's digits: 2 t and 2 t + 1, so that a scan over threads is one over digits
  uint32_t before[2] = {0, 0}, total[2] = {0, 0};
  if (2 * static_cast<int>(threadIdx.x) < digits) {
    const uint2* counts = reinterpret_cast<const uint2*>(p.counts) + threadIdx.x;
    const int tiles = p.totals ? 0 : p.tiles, mine = blockIdx.x;
    if (p.totals) {
      const uint2 b = counts[static_cast<int64_t>(mine) * (digits / 2)];
      const uint2 all = reinterpret_cast<const uint2*>(p.totals)[threadIdx.x];
      before[0] = b.x;
      before[1] = b.y;
      total[0] = all.x;
      total[1] = all.y;
    }
    for (int t0 = 0; t0 < tiles; t0 += 16) {
      uint2 c[16];
#pragma unroll
      for (int k = 0; k < 16; ++k)
        c[k] = t0 + k < tiles ? counts[static_cast<int64_t>(t0 + k) * (digits / 2)] : make_uint2(0, 0);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        total[0] += c[k].x;
        total[1] += c[k].y;
        if (t0 + k < mine) {
          before[0] += c[k].x;
          before[1] += c[k].y;
        }
      }
    }
  }
  uint32_t sum = total[0] + total[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 63) wsum[wave] = sum;
  __syncthreads();
  uint32_t base = sum - total[0] - total[1];
  for (int w = 0; w < wave; ++w) base += wsum[w];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = 2 * threadIdx.x + k;
    if (d < digits) start[d] = base + before[k];
    base += total[k];
  }
  uint32_t rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool valid = first + i * 64 < p.n;
    const uint32_t d = (key[i] >> p.shift) & (digits - 1);
    uint64_t same = __ballot(valid);
    for (int b = 0; b < p.bits; ++b) {
      const uint64_t one = __ballot((d >> b) & 1u);
      same &= (d >> b) & 1u ? one : ~one;
    }
    const uint32_t below = __popcll(same & ((uint64_t(1) << lane) - 1));
    const uint32_t old = cnt[wave][d];
    rank[i] = old + below;
    wave_lds_fence();
    if (valid && below == 0) cnt[wave][d] = old + __popcll(same);
    wave_lds_fence();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
    uint32_t at = start[d];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = cnt[w][d];
      cnt[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t n = first + i * 64;
    if (n < p.n) {
      const uint32_t to = cnt[wave][(key[i] >> p.shift) & (digits - 1)] + rank[i];
      p.keys_out[to] = key[i];
      p.pos_out[to] = pos[i];
    }
  }
}

// The whole sort in one workgroup: up to kLocalThreads * ITEMS positions, id
// << pos_bits | position in 32 bits, ranked as above and moved within LDS: 7 us
// for a few hundred positions, 9 for 4000, instead of 20 in four launches (32768
// in one workgroup took 80).  3711 positions of a table of 200 MB take 27 us, what
// clearing it takes (7.5 TB/s).
template <int ITEMS>
__global__ void __launch_bounds__(kLocalThreads)
sort_local_kernel(SortPass p, int pos_bits, int passes) {
  __shared__ uint32_t buf[kLocalThreads * ITEMS];
  __shared__ uint16_t cnt[kLocalWaves][kMaxDigits];
  __shared__ uint32_t wsum[kLocalWaves];
  if (static_cast<int>(blockIdx.x) >= p.tiles) return p.clear();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int digits = 1 << p.bits, at = wave * 64 * ITEMS + lane, N = static_cast<int>(p.n);
  uint32_t v[ITEMS];
  p.load_keys<ITEMS>(at, 64, v);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)  // what is behind the end stays behind all others
    v[i] = at + i * 64 < N ? v[i] << pos_bits | static_cast<uint32_t>(at + i * 64) : kNone;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pos_bits + pass * p.bits;
    for (int d = threadIdx.x; d < kLocalWaves * kMaxDigits / 2; d += kLocalThreads)
      reinterpret_cast<uint32_t*>(cnt)[d] = 0;
    __syncthreads();
    uint16_t rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t d = (v[i] >> shift) & (digits - 1);
      uint64_t same = ~uint64_t(0);
      for (int b = 0; b < p.bits; ++b) {
        const uint64_t one = __ballot((d >> b) & 1u);
        same &= (d >> b) & 1u ? one : ~one;
      }
      const uint32_t below = __popcll(same & ((uint64_t(1) << lane) - 1)), old = cnt[wave][d];
      rank[i] = static_cast<uint16_t>(old + below);
      wave_lds_fence();
      if (below == 0) cnt[wave][d] = static_cast<uint16_t>(old + __popcll(same));
      wave_lds_fence();
    }
    __syncthreads();
    // a thread per digit: the waves' counts before one another, behind the
    // smaller digits
    uint32_t c[kLocalWaves], total = 0;
    const int d = threadIdx.x;
    if (d < digits) {
#pragma unroll
      for (int w = 0; w < kLocalWaves; ++w) {
        c[w] = cnt[w][d];
        total += c[w];
      }
    }
    uint32_t sum = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t up = __shfl_up(sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 63) wsum[wave] = sum;
    __syncthreads();
    if (d < digits) {
      uint32_t to = sum - total;
      for (int w = 0; w < wave; ++w) to += wsum[w];
#pragma unroll
      for (int w = 0; w < kLocalWaves; ++w) {
        cnt[w][d] = static_cast<uint16_t>(to);  // below 2^15: positions before this one
        to += c[w];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) buf[cnt[wave][(v[i] >> shift) & (digits - 1)] + rank[i]] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) v[i] = buf[at + i * 64];
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (at + i * 64 < N) {
      p.keys_out[at + i * 64] = v[i] >> pos_bits;
      p.pos_out[at + i * 64] = v[i] & ((1u << pos_bits) - 1);
    }
  }
}

// ---------------------------------------------------------------------------
// the sums
// ---------------------------------------------------------------------------
template <typename IO>
__device__ __forceinline__ void write_row(void* dw, int64_t row, int D, int c, const float (&acc)[kVec<IO>],
                                          float scale) {
  float o[kVec<IO>];
#pragma unroll
  for (int i = 0; i < kVec<IO>; ++i) o[i] = acc[i] * scale;
  store_vec<IO>(dw, row * D + c, D - c, pack<IO, kVec<IO>>(o));
}

// Columns of a partial row: whole vectors of 4, so that no load of one needs a
// branch (45 us instead of 12 for the joining of 60360 rows of 143 columns)
__device__ __host__ __forceinline__ int64_t part_columns(int64_t D) { return (D + 3) / 4 * 4; }

// A group of lanes per piece and block of columns; every gradient row is read
// once, at random: 32768 x 768 bf16 18 us (51 MB read, 19 written: 3.9 TB/s).  part: [pieces][2][columns]
// fp32, the partial sums of a run that goes on from the piece before (0) and of
// one that begins here and goes on into the next (1).
template <typename IO>
__global__ void __launch_bounds__(256)
embed_sum_kernel(int64_t N, int piece_len, int64_t vocab, Jobs jb, const uint32_t* keys, const uint32_t* pos,
                 const void* dy, float scale, float* part, void* dw) {
  constexpr int V = kVec<IO>;
  const int D = jb.D;
  const int64_t last = N * D - V;  // where the gradient's last whole vector begins
  const int64_t per = 256 / jb.lpr, pieces = (N + piece_len - 1) / piece_len, jobs = pieces * jb.blocks;
  for (int64_t job = blockIdx.x * per + threadIdx.x / jb.lpr; job < jobs; job += gridDim.x * per) {
    int c;
    const int64_t piece = jb.row_of<V>(job, c);
    if (c >= D) continue;
    const int64_t p0 = piece * piece_len, p1 = p0 + piece_len < N ? p0 + piece_len : N;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    bool head = false;  // the run in hand goes on from the piece before
    for (int64_t p = p0; p < p1; p += kBatch) {
      uint32_t key[kBatch + 1], at[kBatch];
#pragma unroll
      for (int i = 0; i <= kBatch; ++i) {
        const int64_t q = p + i < N ? p + i : N - 1;
        key[i] = keys[q];
        if (i < kBatch) at[i] = pos[q];
      }
      if (p == p0) head = p0 > 0 && keys[p0 - 1] == key[0];
      if (key[0] >= static_cast<uint32_t>(vocab)) break;  // those that take no part stand behind all others
#pragma unroll
      for (int i = 1; i <= kBatch; ++i) key[i] = p + i < N ? key[i] : kNone;
      // All rows at once, also those that take no part, and whole vectors, whose
      // last values may be those of the next row: without a branch around them no
      // load waits for another.
      int64_t from[kBatch];
      Vec<IO> raw[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) from[i] = static_cast<int64_t>(at[i]) * D + c;
      if (last >= 0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) raw[i] = load_vec<IO>(dy, from[i] < last ? from[i] : last, V);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (p + i < p1 && key[i] < static_cast<uint32_t>(vocab)) {
          if (from[i] > last) raw[i] = load_vec<IO>(dy, from[i], D - c);
          float v[V];
          unpack<IO, V>(raw[i], v);
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += v[k];
          const bool more = key[i + 1] == key[i];
          if (!more || p + i + 1 == p1) {
            if (head || more) {
              float* to = part + (piece * 2 + (head ? 0 : 1)) * part_columns(D) + c;
#pragma unroll
              for (int q = 0; q < V; q += 4)
                if (c + q < D)
                  *reinterpret_cast<float4*>(to + q) = make_float4(acc[q], acc[q + 1], acc[q + 2], acc[q + 3]);
            } else {
              write_row<IO>(dw, key[i], D, c, acc, scale);
            }
            head = false;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = 0.0f;
          }
        }
      }
    }
  }
}

__device__ __forceinline__ float4 part_of(const float* part, int64_t row, int D, int c) {
  return *reinterpret_cast<const float4*>(part + row * part_columns(D) + c);
}
// s += the rows a, a + 1, ... below b of the running partial sums, 4 columns.
// (16 rows in flight: fewer workgroups at once, 17.6 us against 12.7 for 32768
// positions.)
__device__ __forceinline__ void add_parts(float (&s)[4], const float* part, int64_t a, int64_t b, int D, int c) {
  int64_t q = a;
  for (; q + 8 <= b; q += 8) {
    float4 u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = part_of(part, (q + k) * 2, D, c);
#pragma unroll
    for (int k = 0; k < 8; ++k) { s[0] += u[k].x; s[1] += u[k].y; s[2] += u[k].z; s[3] += u[k].w; }
  }
  for (; q < b; ++q) {
    const float4 u = part_of(part, q * 2, D, c);
    s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w;
  }
}

// Joins the runs that cross pieces, a wave per piece: where a run begins in its
// piece and goes on behind it, the piece's own partial sum, then the later
// pieces' in order.  (32768 x 768 in pieces of 16, whose commonest id fills 200
// of them: 10 us, rounds of 8 loads one after the other.)  Runs over more than
// kLongRun pieces are left to the whole workgroup, which adds kJoinWaves slices of
// them side by side.  blockIdx.y: a block of 256 columns.
template <typename IO>
__global__ void __launch_bounds__(64 * kJoinWaves)
embed_join_kernel(int64_t N, int piece_len, int64_t vocab, int D, const uint32_t* keys, float scale, const float* part,
                  void* dw) {
  __shared__ float4 red[kJoinWaves][64];
  __shared__ int64_t long_first[kJoinWaves], long_last[kJoinWaves];
  __shared__ uint32_t long_key[kJoinWaves];
  const int64_t pieces = (N + piece_len - 1) / piece_len;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  for (int64_t piece0 = static_cast<int64_t>(blockIdx.x) * kJoinWaves; piece0 + 1 < pieces;
       piece0 += static_cast<int64_t>(gridDim.x) * kJoinWaves) {
    const int64_t piece = piece0 + wave, p0 = piece * piece_len, p1 = p0 + piece_len;
    bool begins = piece + 1 < pieces;
    uint32_t key = kNone;
    if (begins) {
      key = keys[p1 - 1];
      const uint32_t next = keys[p1], own = keys[p0], before = keys[p0 > 0 ? p0 - 1 : 0];  // read together
      // it crosses, and does not come from an earlier piece
      begins = key < static_cast<uint32_t>(vocab) && next == key && !(p0 > 0 && own == key && before == key);
    }
    int64_t last = piece;
    if (begins) {
      // the last piece that begins with the key: those that do are consecutive.
      // The next 64 first, then a search with 64 probes a time
      const int64_t q = piece + 1 + lane;
      last = piece + __popcll(__ballot(q < pieces && keys[q * piece_len] == key));
      if (last == piece + 64) {
        for (int64_t end = pieces; end - last > 1;) {  // ``last`` does, ``end`` does not
          const int64_t step = (end - last + 63) / 64, probe = last + (lane + 1) * step;
          const int more = __popcll(__ballot(probe < end && keys[probe * piece_len] == key));
          const int64_t beyond = last + (more + 1) * step;
          last += more * step;
          end = beyond < end ? beyond : end;
        }
      }
    }
    const bool is_long = begins && last - piece > kLongRun;
    if (lane == 0) {
      long_first[wave] = is_long ? piece : -1;
      long_last[wave] = last;
      long_key[wave] = key;
    }
    if (begins && !is_long) {
      for (int c = (blockIdx.y * 64 + lane) * 4; c < D; c += gridDim.y * 256) {
        const float4 own = part_of(part, piece * 2 + 1, D, c);
        float s[4] = {own.x, own.y, own.z, own.w};
        add_parts(s, part, piece + 1, last + 1, D, c);
        for (int i = 0; i < 4 && c + i < D; ++i) store1<IO>(dw, static_cast<int64_t>(key) * D + c + i, s[i] * scale);
      }
    }
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
      const int64_t first = long_first[w];
      if (first < 0) continue;  // uniform over the workgroup
      const int64_t end = long_last[w] + 1, each = (end - first - 1 + kJoinWaves - 1) / kJoinWaves;
      const int64_t a = first + 1 + wave * each, b = a + each < end ? a + each : end;
      for (int c0 = blockIdx.y * 256; c0 < D; c0 += gridDim.y * 256) {
        const int c = c0 + lane * 4;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (c < D) {
          if (wave == 0) {
            const float4 own = part_of(part, first * 2 + 1, D, c);
            s[0] = own.x; s[1] = own.y; s[2] = own.z; s[3] = own.w;
          }
          add_parts(s, part, a, b, D, c);
        }
        red[wave][lane] = make_float4(s[0], s[1], s[2], s[3]);
        __syncthreads();
        if (wave == 0 && c < D) {
          float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int k = 0; k < kJoinWaves; ++k) {
            const float4 u = red[k][lane];
            t[0] += u.x; t[1] += u.y; t[2] += u.z; t[3] += u.w;
          }
          for (int i = 0; i < 4 && c + i < D; ++i)
            store1<IO>(dw, static_cast<int64_t>(long_key[w]) * D + c + i, t[i] * scale);
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// few positions
// ---------------------------------------------------------------------------
// Up to kFew positions in one launch: every workgroup sorts them all (a position's
// place is the number of those that come before it, N LDS reads), clears its share
// of dW's rows and sums the runs of the ids among them, a wave per run and 64
// vectors of columns.  64 positions of 64 columns: 6.4 us instead of 14.3 in three
// launches, 128 of 768 with 32768 rows 16.7 and 21.4, and what two launches cost the
// host; only 128 times the same id take longer, 23 and 14 (256: 45 and 14).
constexpr int kFew = 128;
constexpr int kFewThreads = 256;
template <typename IO>
__global__ void __launch_bounds__(kFewThreads)
embed_few_kernel(SortPass p, int D, int64_t rows_each, const void* dy, float scale, void* dw) {
  constexpr int V = kVec<IO>;
  __shared__ uint32_t key_in[kFew], key[kFew], pos[kFew];
  __shared__ int start[kFew], starts;
  const int N = static_cast<int>(p.n), i = threadIdx.x;
  if (i < N) {
    uint32_t one[1];
    p.load_keys<1>(i, 1, one);
    key_in[i] = one[0];
  }
  if (i == 0) starts = 0;
  const int64_t r0 = blockIdx.x * rows_each, r1 = r0 + rows_each < p.vocab ? r0 + rows_each : p.vocab;
  p.dw = static_cast<char*>(dw) + r0 * D * sizeof(IO);
  p.dw_bytes = (r1 - r0) * D * static_cast<int64_t>(sizeof(IO));
  p.clear(0, 1);
  __syncthreads();
  if (i < N) {
    const uint32_t own = key_in[i];
    int at = 0;
    for (int k = 0; k < N; ++k) at += key_in[k] < own || (key_in[k] == own && k < i);
    key[at] = own;
    pos[at] = i;
  }
  __syncthreads();
  if (i < N && key[i] >= r0 && key[i] < r1 && (i == 0 || key[i - 1] != key[i])) start[atomicAdd(&starts, 1)] = i;
  __syncthreads();  // behind the clearing too: the rows are written once more
  const int lane = i & 63, wave = __builtin_amdgcn_readfirstlane(i >> 6);
  const int blocks = (D + 64 * V - 1) / (64 * V), jobs = starts * blocks;
  const int64_t last = p.n * D - V;
  for (int job = wave; job < jobs; job += kFewThreads / 64) {
    const int run = job / blocks, c = ((job - run * blocks) * 64 + lane) * V;
    if (c >= D) continue;
    const int a = start[run];
    const uint32_t id = key[a];
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    for (int q = a; q < N && key[q] == id; q += kBatch) {
      int64_t from[kBatch];
      Vec<IO> raw[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) from[k] = static_cast<int64_t>(pos[q + k < N ? q + k : N - 1]) * D + c;
      if (last >= 0) {  // whole vectors, as above
#pragma unroll
        for (int k = 0; k < kBatch; ++k) raw[k] = load_vec<IO>(dy, from[k] < last ? from[k] : last, V);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (q + k < N && key[q + k] == id) {
          if (from[k] > last) raw[k] = load_vec<IO>(dy, from[k], D - c);
          float v[V];
          unpack<IO, V>(raw[k], v);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += v[e];
        }
      }
    }
    write_row<IO>(dw, id, D, c, acc, scale);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
sparc_status em_check(int64_t n, int64_t vocab, int64_t dim, int32_t io, int32_t id_bytes) {
  if (n < 0 || vocab <= 0 || dim <= 0)
    return op_fail(SPARC_EINVAL, "embedding: n >= 0, vocab > 0 and dim > 0 required");
  if (io != SPARC_F32 && io != SPARC_BF16) return op_fail(SPARC_EINVAL, "embedding: unknown io_dtype");
  if (id_bytes != 4 && id_bytes != 8) return op_fail(SPARC_EINVAL, "embedding: ids are 32- or 64-bit integers");
  if (n > (int64_t(1) << 30) || vocab > (int64_t(1) << 30) || dim > (int64_t(1) << 24) ||
      n > (int64_t(1) << 46) / dim || vocab > (int64_t(1) << 46) / dim)
    return op_fail(SPARC_EINVAL, "embedding: too large");
  return SPARC_OK;
}

struct Sort {
  int bits, passes, digit_bits, items;
  int64_t tiles;
  int pos_bits;  // of the sort in LDS, 0: not that
};
Sort sort_of(int64_t n, int64_t vocab) {
  Sort s;
  s.bits = 1;
  while ((vocab >> s.bits) > 0) ++s.bits;  // keys 0 .. vocab
  s.passes = (s.bits + 8) / 9;
  s.digit_bits = (s.bits + s.passes - 1) / s.passes;
  // positions per thread: the whole sort of 524288 positions 41 us with 4, 49 with
  // 16; of 2^22 169 and 130
  s.items = n <= (1 << 20) ? 4 : 16;
  s.tiles = (n + kSortThreads * s.items - 1) / (kSortThreads * s.items);
  s.pos_bits = 1;
  while ((n - 1) >> s.pos_bits > 0) ++s.pos_bits;
  if (n < 1 || n > kLocalItems * kLocalThreads || s.bits + s.pos_bits > 32) s.pos_bits = 0;
  return s;
}

// The widest group that leaves at most an eighth of its lanes idle (96
// vectors: 3 blocks of 32 lanes, not 2 of 64, a third of whose lanes would idle
// in a kernel that is bound by the rows in flight)
Jobs em_jobs(int64_t dim, int v) {
  const int64_t vecs = (dim + v - 1) / v;
  Jobs jb{static_cast<int>(dim), 64, 0};
  while (jb.lpr > 1 && (vecs + jb.lpr - 1) / jb.lpr * jb.lpr * 8 > vecs * 9) jb.lpr >>= 1;
  jb.blocks = static_cast<int>((vecs + jb.lpr - 1) / jb.lpr);
  return jb;
}
unsigned em_grid(const Jobs& jb, int64_t rows) {
  const int64_t per = 256 / jb.lpr;
  return op_grid((rows * jb.blocks + per - 1) / per);
}

// Four vectors per lane where rows have them for 8 lanes (39945 x 1680 fp32: 65 us
// instead of 91, 52164 x 600 bf16 15 instead of 17; 8 vectors: 20 instead of 16),
// and no more workgroups than fill the GPU twice (32768 x 768 bf16: 13 us instead
// of 15).
constexpr unsigned kForwardGroups = 4096;
template <typename IO>
void em_forward(hipStream_t st, int64_t n, int64_t vocab, int64_t dim, const void* tokens, int id_bytes, const void* w,
                float scale, void* y) {
  const auto launch = [&](auto NV, const Jobs& jb) {
    const unsigned all = em_grid(jb, n), grid = all < kForwardGroups ? all : kForwardGroups;
    hipLaunchKernelGGL((embed_fwd_kernel<IO, NV()>), dim3(grid), dim3(256), 0, st, n, vocab, jb, tokens, id_bytes == 8,
                       w, scale, y);
  };
  const int64_t vecs = (dim + kVec<IO> - 1) / kVec<IO>;
  int lpr = 8;
  while (lpr < 64 && lpr * 4 < vecs) lpr *= 2;
  if (vecs < 32) launch(Int<1>{}, em_jobs(dim, kVec<IO>));
  else launch(Int<4>{}, Jobs{static_cast<int>(dim), lpr, static_cast<int>((vecs + 4 * lpr - 1) / (4 * lpr))});
}

// The shares of dW that the launches of a sort clear, one behind the other, in
// whole multiples of 256 bytes, and their grids.
struct Clearing {
  char* dw;
  int64_t left;
  int launches;

  unsigned take(SortPass& p, int threads) {
    int64_t share = (left / launches + 255) / 256 * 256;
    if (launches == 1 || share > left) share = left;
    p.dw = dw;
    p.dw_bytes = share;
    dw += share;
    left -= share;
    --launches;
    const int64_t groups = (share / 16 + threads - 1) / threads, most = 4 * 256 * 1024 / threads;  // 4 per thread slot
    return p.tiles + static_cast<unsigned>(share == 0 ? 0 : groups < 1 ? 1 : groups < most ? groups : most);
  }
};

// A count and a scatter per pass; returns the buffer that holds the sorted
// positions.  (The next pass's counts as atomic additions of the scatter, for
// one launch less: 18 us instead of 6 + 3 at 32768 ids of natural frequencies,
// whose commonest meet in a few counters.)
template <int ITEMS>
int em_sort(hipStream_t st, const Sort& s, SortPass p, Clearing clear, uint32_t* const* keys, uint32_t* const* pos,
            uint32_t* counts) {
  int cur = 0;
  p.counts = counts;
  p.tiles = static_cast<int>(s.tiles);
  if (s.tiles > kManyTiles) p.totals = counts + (s.tiles << s.digit_bits);
  for (int k = 0; k < s.passes; ++k) {
    p.keys_in = keys[cur ^ 1];
    p.pos_in = pos[cur ^ 1];
    p.keys_out = keys[cur];
    p.pos_out = pos[cur];
    p.shift = k * s.digit_bits;
    p.first = k == 0;
    // the counts are over too soon to hide a share
    hipLaunchKernelGGL((sort_count_kernel<ITEMS>), dim3(p.tiles), dim3(kSortThreads), 0, st, p);
    if (p.totals)
      hipLaunchKernelGGL(sort_scan_kernel, dim3(((1 << p.bits) + kScanDigits - 1) / kScanDigits),
                         dim3(kScanDigits * kScanSlices), 0, st, p);
    const unsigned grid = clear.take(p, kSortThreads);
    hipLaunchKernelGGL((sort_scatter_kernel<ITEMS>), dim3(grid), dim3(kSortThreads), 0, st, p);
    cur ^= 1;
  }
  return cur ^ 1;
}

// Sorted positions per piece: as few as are read at once, unless the GPU (256 CUs
// of 16 waves) is full with longer pieces too, whose partial rows are fewer and
// long runs sooner joined (both kernels, 524288 rows of 64 bf16 values: 68 us in
// pieces of 8, 41 in pieces of 32).
int piece_of(int64_t n, int64_t dim) {
  int piece = kBatch;
  while (piece < 1024 && n * dim >= static_cast<int64_t>(2 * piece) << 20) piece *= 2;
  return piece;
}

template <typename IO>
void em_sums(hipStream_t st, int64_t n, int64_t vocab, int64_t dim, const uint32_t* keys, const uint32_t* pos,
             const void* dy, float scale, float* part, void* dw) {
  const int piece = piece_of(n, dim);
  const int64_t pieces = (n + piece - 1) / piece;
  const Jobs jb = em_jobs(dim, kVec<IO>);
  hipLaunchKernelGGL((embed_sum_kernel<IO>), dim3(em_grid(jb, pieces)), dim3(256), 0, st, n, piece, vocab, jb, keys,
                     pos, dy, scale, part, dw);
  if (pieces > 1) {
    const int64_t groups = (pieces + kJoinWaves - 1) / kJoinWaves, columns = (dim + 255) / 256;
    const dim3 grid(static_cast<unsigned>(groups < (1 << 18) ? groups : (1 << 18)),
                    static_cast<unsigned>(columns < 64 ? columns : 64));
    hipLaunchKernelGGL((embed_join_kernel<IO>), grid, dim3(64 * kJoinWaves), 0, st, n, piece, vocab,
                       static_cast<int>(dim), keys, scale, part, dw);
  }
}

// As many workgroups as clear 16 KB each, and one for 4 positions at least, so that
// a wave has one run
template <typename IO>
void em_few(hipStream_t st, const SortPass& p, int64_t dim, const void* dy, float scale, void* dw) {
  const int64_t bytes = p.vocab * dim * static_cast<int64_t>(sizeof(IO));
  int64_t groups = bytes / 16384 > p.n / 4 ? bytes / 16384 : p.n / 4;
  groups = groups < 1 ? 1 : groups < 4096 ? groups : 4096;
  const int64_t each = (p.vocab + groups - 1) / groups;
  hipLaunchKernelGGL((embed_few_kernel<IO>), dim3(static_cast<unsigned>((p.vocab + each - 1) / each)),
                     dim3(kFewThreads), 0, st, p, static_cast<int>(dim), each, dy, scale, dw);
}

}  // namespace
}  // namespace sparc

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

sparc_status sparc_embedding_forward(int64_t n, int64_t vocab, int64_t dim, int32_t io_dtype, int32_t id_bytes,
                                     const void* tokens, const void* weight, float scale, void* y,
                                     sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = em_check(n, vocab, dim, io_dtype, id_bytes)) return s;
  if (n == 0) return SPARC_OK;
  if (!tokens || !weight || !y) return op_fail(SPARC_EINVAL, "embedding forward: NULL pointer");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (io_dtype == SPARC_F32) em_forward<float>(st, n, vocab, dim, tokens, id_bytes, weight, scale, y);
  else em_forward<sparc::bf16>(st, n, vocab, dim, tokens, id_bytes, weight, scale, y);
  return op_launched("embedding forward");
}

size_t sparc_embedding_workspace_bytes(int64_t n, int64_t vocab, int64_t dim) {
  using namespace sparc;
  if (em_check(n, vocab, dim, SPARC_F32, 8)) return 0;
  const Sort s = sort_of(n, vocab);
  const int64_t piece = piece_of(n, dim), pieces = (n + piece - 1) / piece;
  return 4 * up256(n * sizeof(uint32_t)) + up256(((s.tiles + 1) << s.digit_bits) * sizeof(uint32_t)) +
         up256(static_cast<size_t>(pieces) * 2 * part_columns(dim) * sizeof(float)) + 256;
}

sparc_status sparc_embedding_backward(int64_t n, int64_t vocab, int64_t dim, int32_t io_dtype, int32_t id_bytes,
                                      const void* tokens, int64_t padding_id, const void* dy, float scale,
                                      void* dweight, void* workspace, size_t workspace_bytes, sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = em_check(n, vocab, dim, io_dtype, id_bytes)) return s;
  if (!dweight || (n > 0 && (!tokens || !dy))) return op_fail(SPARC_EINVAL, "embedding backward: NULL pointer");
  if (!workspace || workspace_bytes < sparc_embedding_workspace_bytes(n, vocab, dim))
    return op_fail(SPARC_EWORKSPACE, "embedding backward: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16)
    return op_fail(SPARC_EINVAL, "embedding backward: the workspace must be 16-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const Sort s = sort_of(n, vocab);
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t bytes) { char* p = at; at += up256(bytes); return p; };
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(take(n * 4)), reinterpret_cast<uint32_t*>(take(n * 4))};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(take(n * 4)), reinterpret_cast<uint32_t*>(take(n * 4))};
  uint32_t* counts = reinterpret_cast<uint32_t*>(take(((s.tiles + 1) << s.digit_bits) * 4));
  float* part = reinterpret_cast<float*>(at);
  SortPass p{};
  p.tokens = tokens;
  p.wide_ids = id_bytes == 8;
  p.vocab = vocab;
  p.pad = padding_id;
  p.n = n;
  p.bits = s.digit_bits;
  Clearing clear{static_cast<char*>(dweight), vocab * dim * (io_dtype == SPARC_F32 ? 4 : 2), 1};
  int cur = 0;
  if (n == 0) {
    hipLaunchKernelGGL((sort_count_kernel<4>), dim3(clear.take(p, kSortThreads)), dim3(kSortThreads), 0, st, p);
    return op_launched("embedding backward");
  }
  if (n <= kFew) {
    p.first = 1;
    if (io_dtype == SPARC_F32) em_few<float>(st, p, dim, dy, scale, dweight);
    else em_few<sparc::bf16>(st, p, dim, dy, scale, dweight);
    return op_launched("embedding backward");
  }
  if (s.pos_bits) {
    p.keys_out = keys[0];
    p.pos_out = pos[0];
    p.first = 1;
    p.tiles = 1;
    hipLaunchKernelGGL((sort_local_kernel<kLocalItems>), dim3(clear.take(p, kLocalThreads)), dim3(kLocalThreads), 0, st,
                       p, s.pos_bits, s.passes);
  } else {
    clear.launches = s.passes;
    cur = s.items == 4 ? em_sort<4>(st, s, p, clear, keys, pos, counts)
                       : em_sort<16>(st, s, p, clear, keys, pos, counts);
  }
  if (io_dtype == SPARC_F32) em_sums<float>(st, n, vocab, dim, keys[cur], pos[cur], dy, scale, part, dweight);
  else em_sums<sparc::bf16>(st, n, vocab, dim, keys[cur], pos[cur], dy, scale, part, dweight);
  return op_launched("embedding backward");
}

}  // extern "C"
