// The L2 norm over all values of many tensors, and the tensors scaled in place
// by min(1, max_norm / (norm + 1e-6)).
//
// The tensors' addresses and sizes travel as kernel arguments (kMaxTensors per
// launch), so a call copies nothing to the device and can be captured.  Each
// tensor is cut into pieces of kPieceValues values; the workgroups of a launch
// walk the pieces of all its tensors, and each leaves one partial sum of
// squares.  The sums are kept in fp64: squares of fp32 values neither overflow
// nor vanish there, and at the memory's rate the fp64 units are nearly idle.
// The scaling kernel's workgroups each add up all the partial sums in one
// order, so the norm does not depend on timing and no launch stands between;
// where nothing is clipped they read nothing more.

#include "common.h"
#include "sparc_hip.h"

namespace sparc {
namespace {

constexpr int kMaxTensors = 128;      // per launch: 2.7 KB of kernel arguments
constexpr int kPieceValues = 16384;
constexpr int kMaxGroups = 1024;      // partial sums per launch
constexpr int kThreads = 256;

struct TensorList {
  void* data[kMaxTensors];
  int64_t size[kMaxTensors];
  uint32_t first[kMaxTensors + 1];    // first piece of each tensor
  uint8_t bf16_values[kMaxTensors];
  int count;
};

// The piece's tensor: the last one whose first piece is not behind it
__device__ __forceinline__ int tensor_of(const TensorList& l, uint32_t piece) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (l.first[mid] <= piece) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// f(values, first index, count) over [lo, hi) of an array: whole 16-byte
// accesses from the first aligned value on, single values before and behind
template <typename IO, typename F1, typename FV>
__device__ __forceinline__ void for_piece(const void* base, int64_t lo, int64_t hi, F1&& one, FV&& vec) {
  constexpr int V = 16 / sizeof(IO);
  const uintptr_t at = reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(lo) * sizeof(IO);
  int64_t a = lo + static_cast<int64_t>(((16 - at % 16) % 16) / sizeof(IO));
  if (a > hi) a = hi;
  const int64_t nv = (hi - a) / V;
  if (lo + threadIdx.x < a) one(lo + threadIdx.x);
  for (int64_t v = threadIdx.x; v < nv; v += kThreads) vec(a + v * V);
  const int64_t b = a + nv * V;
  if (b + threadIdx.x < hi) one(b + threadIdx.x);
}

template <typename IO>
__device__ __forceinline__ void add_squares(const void* base, int64_t lo, int64_t hi, double& s0, double& s1) {
  constexpr int V = 16 / sizeof(IO);
  for_piece<IO>(
      base, lo, hi,
      [&](int64_t i) {
        const double v = load1<IO>(base, i);
        s0 = fma(v, v, s0);
      },
      [&](int64_t i) {
        float v[V];
        unpack<IO, V>(load_raw<IO, V>(base, i), v);
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          s0 = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), s0);
          s1 = fma(static_cast<double>(v[k + 1]), static_cast<double>(v[k + 1]), s1);
        }
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

__global__ void __launch_bounds__(kThreads)
sum_squares_kernel(TensorList l, double* part) {
  __shared__ double red[kThreads / 64];
  double s0 = 0.0, s1 = 0.0;
  const uint32_t pieces = l.first[l.count];
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    const int t = tensor_of(l, p);
    const int64_t lo = static_cast<int64_t>(p - l.first[t]) * kPieceValues;
    const int64_t hi = lo + kPieceValues < l.size[t] ? lo + kPieceValues : l.size[t];
    if (l.bf16_values[t]) add_squares<bf16>(l.data[t], lo, hi, s0, s1);
    else add_squares<float>(l.data[t], lo, hi, s0, s1);
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
__device__ __forceinline__ void scale_piece(void* base, int64_t lo, int64_t hi, float f) {
  constexpr int V = 16 / sizeof(IO);
  for_piece<IO>(
      base, lo, hi, [&](int64_t i) { store1<IO>(base, i, load1<IO>(base, i) * f); },
      [&](int64_t i) {
        float v[V];
        unpack<IO, V>(load_raw<IO, V>(base, i), v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= f;
        store_raw<IO, V>(base, i, pack<IO, V>(v));
      });
}

__global__ void __launch_bounds__(kThreads)
clip_kernel(TensorList l, const double* part, int n, float max_norm, float* norm) {
  __shared__ double red[kThreads / 64];
  const float v = norm_of(part, n, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float f = max_norm / (v + 1e-6f);
  if (f >= 1.0f) return;  // a NaN goes on, into every value
  const uint32_t pieces = l.first[l.count];
  for (uint32_t q = blockIdx.x; q < pieces; q += gridDim.x) {
    const uint32_t p = pieces - 1 - q;  // the last read are the likeliest in the caches
    const int t = tensor_of(l, p);
    const int64_t lo = static_cast<int64_t>(p - l.first[t]) * kPieceValues;
    const int64_t hi = lo + kPieceValues < l.size[t] ? lo + kPieceValues : l.size[t];
    if (l.bf16_values[t]) scale_piece<bf16>(l.data[t], lo, hi, f);
    else scale_piece<float>(l.data[t], lo, hi, f);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
sparc_status gn_fail(sparc_status s, const char* msg) {
  snprintf(error_buffer(), 512, "%s", msg);
  return s;
}
sparc_status gn_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return SPARC_OK;
  snprintf(error_buffer(), 512, "%s: %s", what, hipGetErrorString(e));
  return SPARC_EHIP;
}

// The next list of up to kMaxTensors tensors with values, from ``at`` on; where
// they begin again is returned
int64_t next_list(int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes, int64_t at,
                  TensorList& l) {
  l.count = 0;
  uint32_t pieces = 0;
  for (; at < count && l.count < kMaxTensors; ++at) {
    if (sizes[at] == 0) continue;
    l.data[l.count] = data[at];
    l.size[l.count] = sizes[at];
    l.bf16_values[l.count] = dtypes[at] == SPARC_BF16;
    l.first[l.count++] = pieces;
    pieces += static_cast<uint32_t>((sizes[at] + kPieceValues - 1) / kPieceValues);
  }
  l.first[l.count] = pieces;
  return at;
}
unsigned list_groups(const TensorList& l) {
  const uint32_t p = l.first[l.count];
  return p < kMaxGroups ? p : kMaxGroups;
}

sparc_status gn_check(int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes) {
  if (count < 0 || count > (int64_t(1) << 24) || (count > 0 && (!data || !sizes || !dtypes)))
    return gn_fail(SPARC_EINVAL, "gradient norm: bad tensor list");
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 40) - total)  // 2^26 pieces in all
      return gn_fail(SPARC_EINVAL, "gradient norm: bad tensor size");
    total += sizes[i];
    if (dtypes[i] != SPARC_F32 && dtypes[i] != SPARC_BF16)
      return gn_fail(SPARC_EINVAL, "gradient norm: unknown dtype");
    if (sizes[i] > 0 && !data[i]) return gn_fail(SPARC_EINVAL, "gradient norm: NULL tensor");
    if (reinterpret_cast<uintptr_t>(data[i]) % (dtypes[i] == SPARC_BF16 ? 2 : 4))
      return gn_fail(SPARC_EINVAL, "gradient norm: a tensor is not aligned to its values");
  }
  return SPARC_OK;
}

// the partial sums of all lists, one behind the other; their number
int launch_sums(hipStream_t st, int64_t count, void* const* data, const int64_t* sizes, const int32_t* dtypes,
                double* part) {
  int n = 0;
  TensorList l;
  for (int64_t at = 0; at < count;) {
    at = next_list(count, data, sizes, dtypes, at, l);
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
  if (!norm) return gn_fail(SPARC_EINVAL, "gradient norm: NULL pointer");
  if (!workspace || workspace_bytes < sparc_grad_norm_workspace_bytes(count))
    return gn_fail(SPARC_EWORKSPACE, "gradient norm: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8)
    return gn_fail(SPARC_EINVAL, "gradient norm: the workspace must be 8-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int n = launch_sums(st, count, tensors, sizes, dtypes, part);
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, part, n, norm);
  return gn_launched("gradient norm");
}

sparc_status sparc_clip_grad_norm(int64_t count, void* const* tensors, const int64_t* sizes, const int32_t* dtypes,
                                  float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                                  sparc_stream_t stream) {
  using namespace sparc;
  if (sparc_status s = gn_check(count, tensors, sizes, dtypes)) return s;
  if (!(max_norm >= 0.0f)) return gn_fail(SPARC_EINVAL, "gradient clipping: max_norm must be >= 0");
  if (!norm) return gn_fail(SPARC_EINVAL, "gradient clipping: NULL pointer");
  if (!workspace || workspace_bytes < sparc_grad_norm_workspace_bytes(count))
    return gn_fail(SPARC_EWORKSPACE, "gradient clipping: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8)
    return gn_fail(SPARC_EINVAL, "gradient clipping: the workspace must be 8-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int n = launch_sums(st, count, tensors, sizes, dtypes, part);
  TensorList l;
  bool any = false;
  for (int64_t at = 0; at < count;) {
    at = next_list(count, tensors, sizes, dtypes, at, l);
    if (l.count == 0) break;
    hipLaunchKernelGGL(clip_kernel, dim3(list_groups(l)), dim3(kThreads), 0, st, l, part, n, max_norm,
                       any ? nullptr : norm);
    any = true;
  }
  if (!any) hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, part, 0, norm);
  return gn_launched("gradient clipping");
}

}  // extern "C"
