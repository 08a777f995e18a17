// The L2 norm over all values of many tensors, and the tensors scaled in place
// by min(1, max_norm / (norm + 1e-6)).
//
// The tensors' addresses and sizes travel as kernel arguments (kMaxTensors per
// launch), so a call copies nothing to the device and can be captured.  Each
// tensor is cut into pieces of 4096 to 16384 values; the workgroups of a launch
// walk the pieces of all its tensors, and each leaves one partial sum of
// squares.  The sums are kept in fp64: squares of fp32 values neither overflow
// nor vanish there, and at the memory's rate the fp64 units are nearly idle.
// The scaling kernel's workgroups each add up all the partial sums in one
// order, so the norm does not depend on timing and no launch stands between;
// where nothing is clipped they read nothing more.

#include <algorithm>
#include <new>

#include "rows.h"

namespace sparc {
namespace {

constexpr int kMaxTensors = 256;      // per launch: 3.6 KB of kernel arguments
constexpr int kMostPiece = 16384;     // values of a piece at most
constexpr int kLeastPiece = 4096;
constexpr int kMaxGroups = 1024;      // partial sums per launch
constexpr int kThreads = 256;

struct TensorList {
  void* data[kMaxTensors];
  uint32_t first[kMaxTensors + 1];    // first piece of each tensor
  uint16_t last[kMaxTensors];         // values of its last piece, and kNarrow for bf16 values
  int count;
  int piece;                          // values of a piece
};
constexpr uint16_t kNarrow = 0x8000;
static_assert(kMostPiece < kNarrow, "a piece's values beside the flag");

// A launch's list in LDS: one trip to the kernel arguments for all threads,
// where a search among them would make one for each of its steps.
struct ListInLds {
  void* data[kMaxTensors];
  uint32_t first[kMaxTensors + 1];
  uint16_t last[kMaxTensors];

  __device__ __forceinline__ void load(const TensorList& l) {
    for (int i = threadIdx.x; i <= l.count; i += kThreads) {
      first[i] = l.first[i];
      if (i < l.count) {
        data[i] = l.data[i];
        last[i] = l.last[i];
      }
    }
    __syncthreads();
  }
  // the piece's tensor: the last one whose first piece is not behind it
  __device__ __forceinline__ int tensor_of(uint32_t piece, int count) const {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first[mid] <= piece) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
  // f(first byte, end, whether bf16) for a piece
  template <typename F>
  __device__ __forceinline__ void piece(uint32_t p, int count, int piece_values, F&& f) const {
    const int t = __builtin_amdgcn_readfirstlane(tensor_of(p, count));
    const bool narrow = last[t] & kNarrow;
    const int64_t values = p + 1 < first[t + 1] ? piece_values : last[t] & (kNarrow - 1);
    const int size_of = narrow ? 2 : 4;
    const uintptr_t at = reinterpret_cast<uintptr_t>(data[t]) + int64_t(p - first[t]) * piece_values * size_of;
    f(at, at + values * size_of, narrow);
  }
};

// Values at an address out of the list: said to be global memory, which the
// compiler cannot know of an address that it reads from LDS
template <typename IO> struct GlobalTypes;
template <> struct GlobalTypes<float> {
  typedef __attribute__((address_space(1))) float One;
  typedef uint32_t V4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(1))) V4 Four;
};
template <> struct GlobalTypes<bf16> {
  typedef __attribute__((address_space(1))) uint16_t One;
  typedef uint32_t V4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(1))) V4 Four;
};
template <typename IO>
__device__ __forceinline__ float load_value(uintptr_t at) {
  const auto v = *reinterpret_cast<const typename GlobalTypes<IO>::One*>(at);
  if constexpr (sizeof(IO) == 4) return v;
  else return bf16_bits_to_float(v);
}
template <typename IO>
__device__ __forceinline__ void store_value(uintptr_t at, float v) {
  auto* p = reinterpret_cast<typename GlobalTypes<IO>::One*>(at);
  if constexpr (sizeof(IO) == 4) *p = v;
  else *p = pack_bf16(v);
}
// Both passes stream the values (non-temporal): 0.9 GB are read at 6.6 TB/s
// instead of 4.4, and the whole call takes 453 instead of 521 us; 512 MB 283
// instead of 334, 32 MB 45 instead of 49.  Only values that lie in the
// memory-side cache already are scaled faster without (128 MB: 86 against 101).
template <typename IO>
__device__ __forceinline__ void load_values(uintptr_t at, Vec<IO>& v) {
  const auto u = __builtin_nontemporal_load(reinterpret_cast<const typename GlobalTypes<IO>::Four*>(at));
  __builtin_memcpy(&v, &u, 16);
}
template <typename IO>
__device__ __forceinline__ void store_values(uintptr_t at, const Vec<IO>& v) {
  typename GlobalTypes<IO>::V4 u;
  __builtin_memcpy(&u, &v, 16);
  __builtin_nontemporal_store(u, reinterpret_cast<typename GlobalTypes<IO>::Four*>(at));
}

// Walks the bytes [at, end) of an array: four(a) for kInFlight whole 16-byte
// vectors a, a + 16 kThreads, ..., vec(a) for each of the others, one(a) for the
// values before the first aligned vector and behind the last
template <typename IO, int kInFlight, typename F1, typename FV, typename F4>
__device__ __forceinline__ void for_piece(uintptr_t at, uintptr_t end, F1&& one, FV&& vec, F4&& four) {
  constexpr uintptr_t kStep = 16 * kThreads;
  uintptr_t a = (at + 15) / 16 * 16;
  if (a > end) a = end;
  const uintptr_t b = a + (end - a) / 16 * 16, t = threadIdx.x;
  if (at + t * sizeof(IO) < a) one(at + t * sizeof(IO));
  uintptr_t v = a + 16 * t;
  for (; v + (kInFlight - 1) * kStep < b; v += kInFlight * kStep) four(v);
  for (; v < b; v += kStep) vec(v);
  if (b + t * sizeof(IO) < end) one(b + t * sizeof(IO));
}

template <typename IO>
__device__ __forceinline__ void add_vec(const Vec<IO>& raw, double& s0, double& s1) {
  float v[kVec<IO>];
  unpack<IO, kVec<IO>>(raw, v);
#pragma unroll
  for (int k = 0; k < kVec<IO>; k += 2) {
    s0 = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), s0);
    s1 = fma(static_cast<double>(v[k + 1]), static_cast<double>(v[k + 1]), s1);
  }
}
template <typename IO>
__device__ __forceinline__ void add_squares(uintptr_t at, uintptr_t end, double& s0, double& s1) {
  constexpr int kInFlight = 4;
  for_piece<IO, kInFlight>(
      at, end,
      [&](uintptr_t a) {
        const double v = load_value<IO>(a);
        s0 = fma(v, v, s0);
      },
      [&](uintptr_t a) {
        Vec<IO> r;
        load_values<IO>(a, r);
        add_vec<IO>(r, s0, s1);
      },
      [&](uintptr_t a) {
        Vec<IO> r[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) load_values<IO>(a + i * 16 * kThreads, r[i]);
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) add_vec<IO>(r[i], s0, s1);
      });
}

// The sum of a value per thread over the workgroup, in every thread
__device__ __forceinline__ double group_total(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) s += red[w];
  return s;
}

// 909 MB of bf16 gradients in 133 tensors: 135 us (6.7 TB/s); 1.1 MB in 12: 5.4 us,
// most of it the launch and three trips to memory, one after the other.
__global__ void __launch_bounds__(kThreads)
sum_squares_kernel(TensorList l, double* part) {
  __shared__ double red[kThreads / 64];
  __shared__ ListInLds list;
  list.load(l);
  double s0 = 0.0, s1 = 0.0;
  const uint32_t pieces = l.first[l.count];
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    list.piece(p, l.count, l.piece, [&](uintptr_t at, uintptr_t end, bool narrow) {
      if (narrow) add_squares<bf16>(at, end, s0, s1);
      else add_squares<float>(at, end, s0, s1);
    });
  }
  const double s = group_total(s0 + s1, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the norm from n partial sums, in every thread
__device__ __forceinline__ float norm_of(const double* part, int n, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += part[i];
  return static_cast<float>(sqrt(group_total(s, red)));
}

__global__ void __launch_bounds__(kThreads)
norm_kernel(const double* part, int n, float* norm) {
  __shared__ double red[kThreads / 64];
  const float v = norm_of(part, n, red);
  if (threadIdx.x == 0) *norm = v;
}

template <typename IO>
__device__ __forceinline__ Vec<IO> scaled(const Vec<IO>& raw, float f) {
  float v[kVec<IO>];
  unpack<IO, kVec<IO>>(raw, v);
#pragma unroll
  for (int k = 0; k < kVec<IO>; ++k) v[k] *= f;
  return pack<IO, kVec<IO>>(v);
}
template <typename IO>
__device__ __forceinline__ void scale_piece(uintptr_t at, uintptr_t end, float f) {
  constexpr int kInFlight = 2;  // 4: 329 against 318 us for 0.9 GB
  for_piece<IO, kInFlight>(
      at, end, [&](uintptr_t a) { store_value<IO>(a, load_value<IO>(a) * f); },
      [&](uintptr_t a) {
        Vec<IO> r;
        load_values<IO>(a, r);
        store_values<IO>(a, scaled<IO>(r, f));
      },
      [&](uintptr_t a) {
        Vec<IO> r[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) load_values<IO>(a + i * 16 * kThreads, r[i]);
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) store_values<IO>(a + i * 16 * kThreads, scaled<IO>(r[i], f));
      });
}

// Reads and writes everything: 909 MB 317 us (5.7 TB/s), 1.1 MB 3.7 us; nothing
// but the partial sums where nothing is clipped.
__global__ void __launch_bounds__(kThreads)
clip_kernel(TensorList l, const double* part, int n, float max_norm, float* norm) {
  __shared__ double red[kThreads / 64];
  const float v = norm_of(part, n, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float f = max_norm / (v + 1e-6f);
  if (f >= 1.0f) return;  // a NaN goes on, into every value
  __shared__ ListInLds list;
  list.load(l);
  const uint32_t pieces = l.first[l.count];
  for (uint32_t q = blockIdx.x; q < pieces; q += gridDim.x) {
    const uint32_t p = pieces - 1 - q;  // backwards: what is still in a cache is what was read last
    list.piece(p, l.count, l.piece, [&](uintptr_t at, uintptr_t end, bool narrow) {
      if (narrow) scale_piece<bf16>(at, end, f);
      else scale_piece<float>(at, end, f);
    });
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// The next list of up to kMaxTensors tensors with values, from ``at`` on; where
// they begin again is returned
int64_t next_list(int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes, int64_t at,
                  int piece, TensorList& l) {
  l.count = 0;
  l.piece = piece;
  uint32_t pieces = 0;
  for (; at < count && l.count < kMaxTensors; ++at) {
    if (sizes[at] == 0) continue;
    l.data[l.count] = data[at];
    l.last[l.count] = static_cast<uint16_t>((sizes[at] - 1) % piece + 1) |
                      (dtypes[at] == SPARC_BF16 ? kNarrow : uint16_t(0));
    l.first[l.count++] = pieces;
    pieces += static_cast<uint32_t>((sizes[at] + piece - 1) / piece);
  }
  l.first[l.count] = pieces;
  return at;
}
unsigned list_groups(const TensorList& l) {
  const uint32_t p = l.first[l.count];
  return p < kMaxGroups ? p : kMaxGroups;
}

// Values of a piece: few tensors' values are spread over more workgroups, down to
// 4 accesses per thread (1.1 MB of fp32 in 12 tensors: 9 us for both launches
// instead of 13)
int piece_of(int64_t count, const int64_t* sizes) {
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += sizes[i];
  int piece = kLeastPiece;
  while (piece < kMostPiece && total > static_cast<int64_t>(piece) * kMaxGroups) piece *= 2;
  return piece;
}

sparc_status gn_check(int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes) {
  if (count < 0 || count > (int64_t(1) << 24) || (count > 0 && (!data || !sizes || !dtypes)))
    return op_fail(SPARC_EINVAL, "gradient norm: bad tensor list");
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 40) - total)  // 2^26 pieces in all
      return op_fail(SPARC_EINVAL, "gradient norm: bad tensor size");
    total += sizes[i];
    if (dtypes[i] != SPARC_F32 && dtypes[i] != SPARC_BF16)
      return op_fail(SPARC_EINVAL, "gradient norm: unknown dtype");
    if (sizes[i] > 0 && !data[i]) return op_fail(SPARC_EINVAL, "gradient norm: NULL tensor");
    if (reinterpret_cast<uintptr_t>(data[i]) % (dtypes[i] == SPARC_BF16 ? 2 : 4))
      return op_fail(SPARC_EINVAL, "gradient norm: a tensor is not aligned to its values");
  }
  return SPARC_OK;
}

// Tensors that are scaled must not share values: two workgroups would scale them
// at once.
sparc_status check_apart(int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes) {
  struct Span { uintptr_t at, end; };
  Span* spans = new (std::nothrow) Span[static_cast<size_t>(count) + 1];
  if (!spans) return op_fail(SPARC_EINVAL, "gradient clipping: no host memory for the tensor list");
  int64_t n = 0;
  bool sorted = true;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(data[i]);
    spans[n] = Span{at, at + static_cast<uintptr_t>(sizes[i]) * (dtypes[i] == SPARC_BF16 ? 2 : 4)};
    sorted = sorted && (n == 0 || spans[n - 1].at <= at);
    ++n;
  }
  if (!sorted) std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.at < b.at; });
  bool apart = true;
  for (int64_t i = 1; i < n; ++i) apart = apart && spans[i - 1].end <= spans[i].at;
  delete[] spans;
  return apart ? SPARC_OK : op_fail(SPARC_EINVAL, "gradient clipping: two tensors overlap");
}

// the partial sums of all lists, one behind the other; their number
int launch_sums(hipStream_t st, int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes,
                double* part) {
  int n = 0;
  const int piece = piece_of(count, sizes);
  TensorList l;
  for (int64_t at = 0; at < count;) {
    at = next_list(count, data, sizes, dtypes, at, piece, l);
    if (l.count == 0) break;
    hipLaunchKernelGGL(sum_squares_kernel, dim3(list_groups(l)), dim3(kThreads), 0, st, l, part + n);
    n += static_cast<int>(list_groups(l));
  }
  return n;
}

}  // namespace
}  // namespace sparc

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

size_t sparc_grad_norm_workspace_bytes(int64_t count) {
  using namespace sparc;
  if (count < 0 || count > (int64_t(1) << 24)) return 0;
  return (static_cast<size_t>(count) / kMaxTensors + 1) * kMaxGroups * sizeof(double) + 256;
}

sparc_status sparc_grad_norm(int64_t count, void* const* tensors, const int64_t* sizes, const int32_t* dtypes,
                             float* norm, void* workspace, size_t workspace_bytes, sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = gn_check(count, tensors, sizes, dtypes)) return s;
  if (!norm) return op_fail(SPARC_EINVAL, "gradient norm: NULL pointer");
  if (!workspace || workspace_bytes < sparc_grad_norm_workspace_bytes(count))
    return op_fail(SPARC_EWORKSPACE, "gradient norm: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8)
    return op_fail(SPARC_EINVAL, "gradient norm: the workspace must be 8-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int n = launch_sums(st, count, tensors, sizes, dtypes, part);
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, part, n, norm);
  return op_launched("gradient norm");
}

sparc_status sparc_clip_grad_norm(int64_t count, void* const* tensors, const int64_t* sizes, const int32_t* dtypes,
                                  float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                                  sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = gn_check(count, tensors, sizes, dtypes)) return s;
  if (sparc_status s = check_apart(count, tensors, sizes, dtypes)) return s;
  if (!(max_norm >= 0.0f)) return op_fail(SPARC_EINVAL, "gradient clipping: max_norm must be >= 0");
  if (!norm) return op_fail(SPARC_EINVAL, "gradient clipping: NULL pointer");
  if (!workspace || workspace_bytes < sparc_grad_norm_workspace_bytes(count))
    return op_fail(SPARC_EWORKSPACE, "gradient clipping: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8)
    return op_fail(SPARC_EINVAL, "gradient clipping: the workspace must be 8-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int n = launch_sums(st, count, tensors, sizes, dtypes, part);
  const int piece = piece_of(count, sizes);
  TensorList l;
  bool any = false;
  for (int64_t at = 0; at < count;) {
    at = next_list(count, tensors, sizes, dtypes, at, piece, l);
    if (l.count == 0) break;
    hipLaunchKernelGGL(clip_kernel, dim3(list_groups(l)), dim3(kThreads), 0, st, l, part, n, max_norm,
                       any ? nullptr : norm);
    any = true;
  }
  if (!any) hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, part, 0, norm);
  return op_launched("gradient clipping");
}

}  // extern "C"
