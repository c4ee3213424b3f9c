// Element and index types of the training operators (lookup, cross entropy, clip): vector
// loads and stores of float32 / bfloat16 / float16 rows as fp32 values, index loads, and the
// dispatch over the types the C ABI names (fg_dtype, fg_index_type).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace fg {

inline size_t dtype_size(int32_t dtype) { return dtype == FG_FLOAT32 ? 4 : 2; }
inline bool dtype_known(int32_t dtype) { return dtype >= FG_FLOAT32 && dtype <= FG_FLOAT16; }
inline bool index_known(int32_t t) { return t == FG_INDEX_INT32 || t == FG_INDEX_INT64; }

// The widest of 16, 8, 4 and 2 bytes that divides every listed address, pitch and row length.
inline int common_vector_bytes(std::initializer_list<uint64_t> things) {
  uint64_t all = 16;
  for (uint64_t t : things) all |= t;
  return (int)(all & (~all + 1));
}

// An array of a call: rows of `width` elements, `ld` from one to the next.  `overlap`: whether two
// have a byte in common.  A kernel reads its inputs while it writes, in no order, so an output that
// is also an input is refused.
struct Array2d {
  const void* at;
  int64_t rows, width, ld;
  size_t element;
};
inline bool overlap(const Array2d& a, const Array2d& b) {
  if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  typedef __int128 Wide;   // a product of the sizes may pass 64 bits
  const Wide a0 = (Wide)(uintptr_t)a.at, b0 = (Wide)(uintptr_t)b.at;
  const Wide a1 = a0 + ((Wide)(a.rows - 1) * a.ld + a.width) * (Wide)a.element;
  const Wide b1 = b0 + ((Wide)(b.rows - 1) * b.ld + b.width) * (Wide)b.element;
  if (a1 <= b0 || b1 <= a0) return false;
  // columns of one array side by side
  const Wide pitch = (Wide)(a.rows > 1 ? a.ld * (Wide)a.element : b.ld * (Wide)b.element);
  if (a.rows > 1 && b.rows > 1 && (Wide)b.ld * (Wide)b.element != pitch) return true;
  if (a.rows == 1 && b.rows == 1) return true;
  const Wide apart = ((b0 - a0) % pitch + pitch) % pitch;   // where b's rows begin in a's pitch
  return !(apart >= (Wide)a.width * (Wide)a.element && apart + (Wide)b.width * (Wide)b.element <= pitch);
}
inline Array2d array1d(const void* at, int64_t n, size_t element) { return {at, n > 0 ? 1 : 0, n, n, element}; }

#ifdef __CUDACC__

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// Round to nearest even: the one rounding of a result to its type.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements as one memory access of N * sizeof(T) = 2, 4, 8 or 16 bytes.  They
// stay as loaded until they are unpacked: taken apart at the load, every load waited for the
// one before.
template <int BYTES>
struct RawVec;
template <>
struct RawVec<16> { using type = uint4; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<4> { using type = unsigned; };
template <>
struct RawVec<2> { using type = unsigned short; };

template <typename T, int N>
struct Vec {
  using Raw = typename RawVec<N * (int)sizeof(T)>::type;
  Raw raw;
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Vec<T, N>& v, float (&x)[N]) {
  if constexpr (sizeof(T) == 4) {
    memcpy(x, &v.raw, sizeof(v.raw));
  } else if constexpr (N == 1) {
    T one;
    memcpy(&one, &v.raw, 2);
    x[0] = to_float<T>(one);
  } else {
    uint32_t w[N / 2];
    memcpy(w, &v.raw, sizeof(v.raw));
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      } else {
        __half2 h;
        memcpy(&h, &w[k], 4);
        const float2 f = __half22float2(h);
        x[2 * k] = f.x;
        x[2 * k + 1] = f.y;
      }
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> pack(const float (&x)[N]) {
  T t[N];
#pragma unroll
  for (int k = 0; k < N; ++k) t[k] = from_float<T>(x[k]);
  Vec<T, N> v;
  memcpy(&v.raw, t, sizeof(v.raw));
  return v;
}

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  return {__ldg(reinterpret_cast<const typename Vec<T, N>::Raw*>(p))};
}
// Read-once data: evicted first.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec_stream(const T* p) {
  return {__ldcs(reinterpret_cast<const typename Vec<T, N>::Raw*>(p))};
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
  *reinterpret_cast<typename Vec<T, N>::Raw*>(p) = v.raw;
}
template <typename T, int N>
__device__ __forceinline__ void store_vec_stream(T* p, const Vec<T, N>& v) {
  __stcs(reinterpret_cast<typename Vec<T, N>::Raw*>(p), v.raw);
}

// Sets the status word; an expired wait, the larger code, is not hidden by an index out of range.
__device__ __forceinline__ void report(int32_t* status, int32_t code) { atomicMax(status, code); }

#endif  // __CUDACC__

// CALL(T) for the element type `dtype`, already checked with dtype_known.
#define FG_DISPATCH_DTYPE(dtype, CALL)          \
  switch (dtype) {                              \
    case FG_FLOAT32: CALL(float); break;        \
    case FG_BFLOAT16: CALL(__nv_bfloat16); break; \
    default: CALL(__half); break;               \
  }

// Launches a kernel; `chained`: programmatically behind the one before it in the stream, a
// kernel of the same call, so that its launch overlaps that one's run.  Every kernel that is
// launched this way begins with wait_for_prior_grids() before it touches memory, and lets the
// next one be launched (launch_dependents) only behind that, so nothing overtakes anything.
template <typename... P, typename... A>
cudaError_t launch(bool chained, void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                   cudaStream_t stream, A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = chained ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
  if (err != cudaSuccess) (void)cudaGetLastError();  // returned here, not to a later call
  return err;
}

// Lets a kernel use up to `most` bytes of dynamic shared memory on a device: the most that any
// call of it asks for, not this call's, since a later smaller limit would replace it.  Asking the
// runtime takes microseconds, so each host thread remembers the kernels that have theirs.
inline cudaError_t allow_shared(const void* kernel, int most, int device) {
  struct Known {
    const void* kernel;
    int device;
  };
  constexpr int kMost = 64;
  static thread_local Known known[kMost];
  static thread_local int n = 0;
  for (int k = 0; k < n; ++k)
    if (known[k].kernel == kernel && known[k].device == device) return cudaSuccess;
  const cudaError_t err =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (err == cudaSuccess && n < kMost) known[n++] = {kernel, device};
  if (err != cudaSuccess) (void)cudaGetLastError();
  return err;
}

#ifdef __CUDACC__
__device__ __forceinline__ void begin_chained() {
  wait_for_prior_grids();
  launch_dependents();
}
#endif

}  // namespace fg
