// Global gradient norm over many tensors, and clipping.
//
//   norm = sqrt(sum over every element g of every tensor of g^2), or max |g|
//   out  = g * min(1, max_norm / (norm + eps))
//
// Two kernels: the first reads everything once and leaves one partial norm per CTA, the second
// lets every CTA add those up (in one fixed order: the result does not depend on timing) and
// reads and writes everything once.  Both are bound by memory traffic: 85 M float32 values in 48
// tensors take 146 us, 1.02 GB at 7 TB/s with what L2 still holds of the first reading.
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "elem.cuh"

namespace fg {
namespace {

constexpr int kClipThreads = 256;
// Tensors a launch can name in its parameters.  The launch copies them all, so a few tensors
// take the short list (two tensors: 10.4 us a call with the long one).
constexpr int kFewTensors = 32, kManyTensors = 512;
constexpr int kClipMaxBlocks = 1184;  // CTAs (and partial norms) of one launch

// One launch's tensors, in the kernel's parameters: the pointers change from call to call, and
// parameters need no copy to the device and are recorded by a stream capture.
template <int MOST>
struct ClipTensors {
  static constexpr int kMost = MOST;
  const void* in[MOST];
  void* out[MOST];
  int64_t size[MOST];
  int32_t first_chunk[MOST + 1];  // chunks of kClipChunk elements, over all tensors
  uint8_t dtype[MOST];
  uint8_t vector[MOST];           // whether 16-byte accesses are aligned
  int n;
};
constexpr int kClipChunk = 8192;

template <typename Tensors>
__device__ __forceinline__ int find_tensor(const Tensors& t, int chunk) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first_chunk[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// Adds one group of values to a thread's part of the norm.  Squares are summed in groups of at most
// eight in fp32 and the groups in fp64; a group whose fp32 sum leaves the range in which fp32 squares are
// exact enough (overflow, or below 2^-100) is summed again in fp64.
template <bool MAX_NORM, int N>
__device__ __forceinline__ void add_group(const float (&x)[N], double& acc, float& top, bool& nan) {
  if (MAX_NORM) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      top = fmaxf(top, fabsf(x[k]));
      nan |= x[k] != x[k];
    }
    return;
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) s = fmaf(x[k], x[k], s);
  if (s > 1e-30f && s < 1e38f) {
    acc += (double)s;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) acc += (double)x[k] * (double)x[k];
  }
}

template <typename T, bool MAX_NORM>
__device__ __forceinline__ void chunk_norm(const T* __restrict__ p, int count, bool vector,
                                           double& acc, float& top, bool& nan) {
  constexpr int N = 16 / sizeof(T);
  int done = 0;
  if (vector) {
    const int vecs = count / N;
#pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += kClipThreads) {
      const Vec<T, N> v = load_vec<T, N>(p + (int64_t)i * N);
      float x[N];
      unpack<T, N>(v, x);
      add_group<MAX_NORM, N>(x, acc, top, nan);
    }
    done = vecs * N;
  }
  for (int i = done + threadIdx.x; i < count; i += kClipThreads) {
    const float x[1] = {to_float<T>(p[i])};
    add_group<MAX_NORM, 1>(x, acc, top, nan);
  }
}

template <bool MAX_NORM>
__device__ __forceinline__ double combine_norm(double a, double b) {
  if (!MAX_NORM) return a + b;
  if (a != a) return a;
  if (b != b) return b;
  return a > b ? a : b;
}

template <bool MAX_NORM>
__device__ double block_norm(double v, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    v = combine_norm<MAX_NORM>(v, __shfl_xor_sync(0xffffffffu, v, d));
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  double total = shared[0];
  for (int w = 1; w < kClipThreads / 32; ++w) total = combine_norm<MAX_NORM>(total, shared[w]);
  return total;
}

template <bool MAX_NORM, typename Tensors>
__global__ void __launch_bounds__(kClipThreads)
partial_norm_kernel(const __grid_constant__ Tensors t, double* __restrict__ partial) {
  begin_chained();
  __shared__ double shared[kClipThreads / 32];
  double acc = 0.0;
  float top = 0.f;
  bool nan = false;
  const int chunks = t.first_chunk[t.n];
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int k = find_tensor(t, chunk);
    const int64_t at = (int64_t)(chunk - t.first_chunk[k]) * kClipChunk;
    const int count = (int)(t.size[k] - at < kClipChunk ? t.size[k] - at : kClipChunk);
    const bool vector = t.vector[k];
#define FG_NORM(T) chunk_norm<T, MAX_NORM>(static_cast<const T*>(t.in[k]) + at, count, vector, acc, top, nan)
    FG_DISPATCH_DTYPE(t.dtype[k], FG_NORM)
#undef FG_NORM
  }
  if (MAX_NORM) acc = nan ? (double)__int_as_float(0x7fc00000) : (double)top;
  const double total = block_norm<MAX_NORM>(acc, shared);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* p, T* q, int count, bool vector, float share) {
  constexpr int N = 16 / sizeof(T);
  int done = 0;
  if (vector) {
    const int vecs = count / N;
#pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += kClipThreads) {
      float x[N];
      unpack<T, N>(load_vec_stream<T, N>(p + (int64_t)i * N), x);
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] *= share;
      store_vec_stream<T, N>(q + (int64_t)i * N, pack<T, N>(x));
    }
    done = vecs * N;
  }
  for (int i = done + threadIdx.x; i < count; i += kClipThreads)
    q[i] = from_float<T>(to_float<T>(p[i]) * share);
}

template <bool MAX_NORM, typename Tensors>
__global__ void __launch_bounds__(kClipThreads)
scale_kernel(const __grid_constant__ Tensors t, const double* __restrict__ partial,
             int n_partial, double max_norm, double eps, float* __restrict__ norm_out) {
  begin_chained();
  __shared__ double shared[kClipThreads / 32];
  double acc = 0.0;
  for (int i = threadIdx.x; i < n_partial; i += kClipThreads)
    acc = combine_norm<MAX_NORM>(acc, partial[i]);
  const double total = block_norm<MAX_NORM>(acc, shared);
  const double norm = MAX_NORM ? total : sqrt(total);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double ratio = max_norm / (norm + eps);
  // a NaN norm reaches every element, an infinite one scales by zero; without a bound nothing
  // is scaled
  float share = ratio < 1.0 ? (float)ratio : 1.f;
  if (norm != norm) share = __int_as_float(0x7fc00000);
  if (isinf(max_norm)) share = 1.f;
  const int chunks = t.first_chunk[t.n];
  for (int j = blockIdx.x; j < chunks; j += gridDim.x) {
    const int chunk = chunks - 1 - j;  // backwards: what the first kernel read last is in L2
    const int k = find_tensor(t, chunk);
    if (share == 1.f && t.in[k] == t.out[k]) continue;  // in place and nothing to scale
    const int64_t at = (int64_t)(chunk - t.first_chunk[k]) * kClipChunk;
    const int count = (int)(t.size[k] - at < kClipChunk ? t.size[k] - at : kClipChunk);
    const bool vector = t.vector[k];
#define FG_SCALE(T) \
  chunk_scale<T>(static_cast<const T*>(t.in[k]) + at, static_cast<T*>(t.out[k]) + at, count, vector, share)
    FG_DISPATCH_DTYPE(t.dtype[k], FG_SCALE)
#undef FG_SCALE
  }
}

// The two kernels over tensors of the C call, a launch per Tensors::kMost of them.
struct ClipCall {
  const void* const* grads;
  void* const* outs;
  const int64_t* sizes;
  const int32_t* dtypes;
  int32_t n_tensors;
  bool max_abs_norm;
  double max_norm, eps;
  float* norm;
  double* partial;
};
template <typename Tensors>
int run_clip(const ClipCall& call, cudaStream_t s) {
  Tensors t;
  int grid = 1, n_partial = 0;
  // the tensors from `first` on that one launch can name; returns the first one left
  auto fill = [&](int32_t first) -> int32_t {
    t.n = 0;
    int64_t chunks = 0;
    int32_t k = first;
    for (; k < call.n_tensors && t.n < Tensors::kMost; ++k) {
      t.in[t.n] = call.grads[k];
      t.out[t.n] = call.outs[k];
      t.size[t.n] = call.sizes[k];
      t.dtype[t.n] = (uint8_t)call.dtypes[k];
      t.vector[t.n] = (((uintptr_t)call.grads[k] | (uintptr_t)call.outs[k]) & 15) == 0;
      t.first_chunk[t.n++] = (int32_t)chunks;
      chunks += (call.sizes[k] + kClipChunk - 1) / kClipChunk;
    }
    t.first_chunk[t.n] = (int32_t)chunks;
    grid = (int)std::max<int64_t>(1, std::min<int64_t>(chunks, kClipMaxBlocks));
    return k;
  };
  int32_t next = 0;
  do {
    next = fill(next);
    FG_CUDA_TRY(launch(n_partial > 0,
                       call.max_abs_norm ? partial_norm_kernel<true, Tensors> : partial_norm_kernel<false, Tensors>,
                       grid, kClipThreads, 0, s, t, call.partial + n_partial));
    n_partial += grid;
  } while (next < call.n_tensors);
  const bool filled = next <= Tensors::kMost;   // one launch names them all: t is still right
  next = filled ? call.n_tensors : 0;
  do {
    if (!filled) next = fill(next);
    FG_CUDA_TRY(launch(true, call.max_abs_norm ? scale_kernel<true, Tensors> : scale_kernel<false, Tensors>,
                       grid, kClipThreads, 0, s, t, call.partial, n_partial, call.max_norm, call.eps, call.norm));
  } while (next < call.n_tensors);
  return FG_OK;
}

// Whether an output (the norm too) shares memory with another output or with an input other than its
// own (which it may be itself, but not in part).  `spans` has room for n_tensors.
struct Span {
  uint64_t begin, end;
  int32_t tensor;
};
bool outputs_overlap(const ClipCall& call, Span* spans) {
  int32_t n = 0;
  for (int32_t k = 0; k < call.n_tensors; ++k) {
    const uint64_t bytes = (uint64_t)call.sizes[k] * dtype_size(call.dtypes[k]);
    const uint64_t at = (uint64_t)(uintptr_t)call.outs[k];
    if (bytes > 0) spans[n++] = {at, at + bytes, k};
  }
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (int32_t i = 1; i < n; ++i)
    if (spans[i].begin < spans[i - 1].end) return true;
  const uint64_t norm = (uint64_t)(uintptr_t)call.norm;
  for (int32_t k = 0; k < call.n_tensors; ++k) {
    const uint64_t bytes = (uint64_t)call.sizes[k] * dtype_size(call.dtypes[k]);
    const uint64_t at = (uint64_t)(uintptr_t)call.grads[k], out = (uint64_t)(uintptr_t)call.outs[k];
    if (bytes > 0 && ((norm < at + bytes && at < norm + 4) || (norm < out + bytes && out < norm + 4))) return true;
    if (bytes == 0 || call.grads[k] == call.outs[k]) continue;
    // the first output that ends behind the input's begin
    const Span* hit = std::lower_bound(spans, spans + n, at, [](const Span& s, uint64_t v) { return s.end <= v; });
    if (hit != spans + n && hit->begin < at + bytes) return true;
  }
  return false;
}

}  // namespace
}  // namespace fg

extern "C" int64_t fg_gradient_clip_workspace_bytes(int32_t n_tensors) {
  if (n_tensors < 0) return 0;
  const int64_t launches = (n_tensors + fg::kManyTensors - 1) / fg::kManyTensors;
  return std::max<int64_t>(launches, 1) * fg::kClipMaxBlocks * (int64_t)sizeof(double);
}

extern "C" int fg_gradient_clip(const void* const* grads_host_array, void* const* outs_host_array,
                                const int64_t* sizes_host_array, const int32_t* dtypes_host_array,
                                int32_t n_tensors, int32_t max_abs_norm, double max_norm,
                                double eps, float* norm_dev, void* workspace_dev,
                                int64_t workspace_bytes, int32_t device, void* stream) {
  using namespace fg;
  if (n_tensors < 0 || (n_tensors > 0 && (!grads_host_array || !outs_host_array ||
                                          !sizes_host_array || !dtypes_host_array)))
    return fail(FG_ERR_INVALID_ARGUMENT, "bad n_tensors=%d or a null array", (int)n_tensors);
  if (!(max_norm >= 0.0) || !(eps >= 0.0))
    return fail(FG_ERR_INVALID_ARGUMENT, "max_norm=%g and eps=%g must not be negative or NaN",
                max_norm, eps);
  if (!norm_dev || ((uintptr_t)norm_dev & 3) != 0 || !workspace_dev || ((uintptr_t)workspace_dev & 7) != 0 ||
      workspace_bytes < fg_gradient_clip_workspace_bytes(n_tensors))
    return fail(FG_ERR_INVALID_ARGUMENT, "null norm_dev, or the workspace is smaller than %lld bytes",
                (long long)fg_gradient_clip_workspace_bytes(n_tensors));
  for (int32_t k = 0; k < n_tensors; ++k) {
    if (!dtype_known(dtypes_host_array[k]) || sizes_host_array[k] < 0)
      return fail(FG_ERR_INVALID_ARGUMENT, "tensor %d: dtype=%d size=%lld", (int)k,
                  (int)dtypes_host_array[k], (long long)sizes_host_array[k]);
    const uint64_t es = dtype_size(dtypes_host_array[k]);
    if (sizes_host_array[k] > 0 &&
        (!grads_host_array[k] || !outs_host_array[k] ||
         ((uintptr_t)grads_host_array[k] | (uintptr_t)outs_host_array[k]) % es != 0))
      return fail(FG_ERR_INVALID_ARGUMENT, "tensor %d: null or misaligned pointer", (int)k);
  }
  int64_t all_chunks = 0;
  for (int32_t k = 0; k < n_tensors; ++k)
    all_chunks += (sizes_host_array[k] + kClipChunk - 1) / kClipChunk;
  if (all_chunks > INT32_MAX)
    return fail(FG_ERR_UNSUPPORTED, "%lld chunks of %d elements are too many",
                (long long)all_chunks, kClipChunk);
  const ClipCall call = {grads_host_array, outs_host_array, sizes_host_array, dtypes_host_array, n_tensors,
                         max_abs_norm != 0, max_norm, eps, norm_dev, static_cast<double*>(workspace_dev)};
  Span some[kManyTensors];
  std::unique_ptr<Span[]> more;
  if (n_tensors > kManyTensors) {
    more.reset(new (std::nothrow) Span[n_tensors]);
    if (!more) return fail(FG_ERR_OUT_OF_MEMORY, "no host memory for %d tensors", (int)n_tensors);
  }
  if (outputs_overlap(call, more ? more.get() : some))
    return fail(FG_ERR_INVALID_ARGUMENT, "an output shares memory with another tensor than its own input");
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return n_tensors <= kFewTensors ? run_clip<ClipTensors<kFewTensors>>(call, s)
                                  : run_clip<ClipTensors<kManyTensors>>(call, s);
}
