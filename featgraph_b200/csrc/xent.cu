// Softmax cross entropy over a large vocabulary (every vertex of a graph, every class),
// without keeping the logits, and its gradients.
//
//   z = scale * feat @ weight^T          (n x V, never stored whole)
//   lse_t  = log sum_v exp z_tv
//   loss_t = lse_t - z_{t, label_t}      (0 where the label is ignore_index)
//   dz     = scale * loss_grad_t * (exp(z - lse) - [v = label_t])    (0 on ignored rows)
//   feat_grad = dz @ weight,  weight_grad = dz^T @ feat
#include <algorithm>
#include <cmath>

#include "elem.cuh"

namespace fg {
namespace {

constexpr int kTile = 32;
constexpr int64_t kPiece = 8192;

__device__ __forceinline__ int64_t load_label(const void* labels, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long*>(labels) + i)
              : (int64_t)__ldg(static_cast<const int*>(labels) + i);
}

struct Batch {
  const void* labels;
  int wide;
  int64_t n, vocab, feat_len, ignore_index;
  float scale;
};

// One 32 x 32 tile of a product with fp32 accumulators, 256 threads, four results a thread:
// row ty + 8 i, column tx.
template <typename A, typename B>
__device__ __forceinline__ void product_tile(float (&acc)[4], int64_t m0, int64_t n0, int64_t m,
                                             int64_t n, int64_t k_len, const A* a, int64_t a_m,
                                             int64_t a_k, const B* b, int64_t b_n, int64_t b_k) {
  __shared__ float sa[kTile][kTile + 1], sb[kTile][kTile + 1];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = 0; i < 4; ++i) acc[i] = 0.f;
  for (int64_t k0 = 0; k0 < k_len; k0 += kTile) {
    for (int i = 0; i < 4; ++i) {
      const int r = ty + 8 * i;
      const int64_t k = k0 + tx;
      sa[r][tx] = m0 + r < m && k < k_len ? to_float<A>(a[(m0 + r) * a_m + k * a_k]) : 0.f;
      sb[r][tx] = n0 + r < n && k < k_len ? to_float<B>(b[(n0 + r) * b_n + k * b_k]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kTile; ++k)
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sa[ty + 8 * i][k], sb[tx][k], acc[i]);
    __syncthreads();
  }
}

// Running maximum and sum of exponentials of a tile row; one pair per (row, vocabulary tile).
template <typename T>
__global__ void __launch_bounds__(256)
logit_stats_kernel(Batch b, const T* feat, int64_t feat_ld, const T* weight, int64_t weight_ld,
                   float2* stats, float* picked) {
  const int64_t v0 = (int64_t)blockIdx.x * kTile, t0 = (int64_t)blockIdx.y * kTile;
  float acc[4];
  product_tile<T, T>(acc, t0, v0, b.n, b.vocab, b.feat_len, feat, feat_ld, 1, weight, weight_ld, 1);
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty + 8 * i, v = v0 + tx;
    const float z = v < b.vocab ? acc[i] * b.scale : -INFINITY;
    float top = z;
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    float s = top == -INFINITY ? (z != z ? z : 0.f) : expf(z - top);
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (t >= b.n) continue;
    if (tx == 0) stats[t * gridDim.x + blockIdx.x] = make_float2(top, s);
    if (v < b.vocab && load_label(b.labels, b.wide, t) == v) picked[t] = z;
  }
}

__global__ void __launch_bounds__(256)
join_stats_kernel(Batch b, const float2* stats, int64_t tiles, const float* picked, float* loss,
                  float* lse, int32_t* status) {
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= b.n) return;
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, s = 0.f;
  for (int64_t k = lane; k < tiles; k += 32) {
    const float2 p = stats[t * tiles + k];
    const float m = fmaxf(top, p.x);
    if (m == -INFINITY) { s += p.y; continue; }
    s = s * expf(top - m) + p.y * expf(p.x - m);
    top = m;
  }
  for (int d = 16; d > 0; d >>= 1) {
    const float top2 = __shfl_xor_sync(0xffffffffu, top, d), s2 = __shfl_xor_sync(0xffffffffu, s, d);
    const float m = fmaxf(top, top2);
    s = m == -INFINITY ? s + s2 : s * expf(top - m) + s2 * expf(top2 - m);
    top = m;
  }
  if (lane != 0) return;
  const float l = top + logf(s);
  lse[t] = l;
  const int64_t y = load_label(b.labels, b.wide, t);
  if (y == b.ignore_index) {
    loss[t] = 0.f;
  } else if ((uint64_t)y >= (uint64_t)b.vocab) {
    *status = FG_STATUS_BAD_INDEX;
    loss[t] = __int_as_float(0x7fc00000);
  } else {
    loss[t] = l - picked[t];
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
logit_grad_kernel(Batch b, const T* feat, int64_t feat_ld, const T* weight, int64_t weight_ld,
                  const float* lse, const float* loss_grad, int64_t v_begin, int64_t v_count,
                  float* dz) {
  const int64_t v0 = (int64_t)blockIdx.x * kTile, t0 = (int64_t)blockIdx.y * kTile;
  float acc[4];
  product_tile<T, T>(acc, t0, v0, b.n, v_count, b.feat_len, feat, feat_ld, 1,
                     weight + v_begin * weight_ld, weight_ld, 1);
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty + 8 * i, v = v0 + tx;
    if (t >= b.n || v >= v_count) continue;
    const int64_t y = load_label(b.labels, b.wide, t);
    const bool live = y != b.ignore_index && (uint64_t)y < (uint64_t)b.vocab;
    const float p = expf(acc[i] * b.scale - lse[t]) - (y == v_begin + v ? 1.f : 0.f);
    dz[t * v_count + v] = live ? p * loss_grad[t] * b.scale : 0.f;
  }
}

// feat_grad += dz @ weight over one piece; the sum over the pieces waits in fp32.
template <typename T>
__global__ void __launch_bounds__(256)
feat_grad_kernel(Batch b, const float* dz, const T* weight, int64_t weight_ld, int64_t v_begin,
                 int64_t v_count, float* acc_out, T* feat_grad, int first, int last) {
  const int64_t t0 = (int64_t)blockIdx.y * kTile, d0 = (int64_t)blockIdx.x * kTile;
  float acc[4];
  product_tile<float, T>(acc, t0, d0, b.n, b.feat_len, v_count, dz, v_count, 1,
                         weight + v_begin * weight_ld, 1, weight_ld);
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty + 8 * i, d = d0 + tx;
    if (t >= b.n || d >= b.feat_len) continue;
    const float v = acc[i] + (first ? 0.f : acc_out[t * b.feat_len + d]);
    if (last)
      feat_grad[t * b.feat_len + d] = from_float<T>(v);
    else
      acc_out[t * b.feat_len + d] = v;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
live_feat_kernel(Batch b, const T* feat, int64_t feat_ld, T* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= b.n * b.feat_len) return;
  const int64_t t = i / b.feat_len, d = i - t * b.feat_len;
  const int64_t y = load_label(b.labels, b.wide, t);
  const bool live = y != b.ignore_index && (uint64_t)y < (uint64_t)b.vocab;
  out[i] = live ? feat[t * feat_ld + d] : from_float<T>(0.f);
}

template <typename T>
__global__ void __launch_bounds__(256)
weight_grad_kernel(Batch b, const float* dz, const T* feat, int64_t feat_ld, int64_t v_begin,
                   int64_t v_count, T* weight_grad) {
  const int64_t v0 = (int64_t)blockIdx.y * kTile, d0 = (int64_t)blockIdx.x * kTile;
  float acc[4];
  product_tile<float, T>(acc, v0, d0, v_count, b.feat_len, b.n, dz, 1, v_count, feat, 1, feat_ld);
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = 0; i < 4; ++i) {
    const int64_t v = v0 + ty + 8 * i, d = d0 + tx;
    if (v < v_count && d < b.feat_len)
      weight_grad[(v_begin + v) * b.feat_len + d] = from_float<T>(acc[i]);
  }
}

struct XentLayout {
  size_t stats, picked, total_forward;
  size_t dz, live_feat, acc, total_grad;
};

XentLayout xent_layout(int32_t dtype, int64_t n, int64_t vocab, int64_t feat_len) {
  XentLayout l;
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const int64_t tiles = (vocab + kTile - 1) / kTile;
  l.stats = take((size_t)n * tiles * sizeof(float2));
  l.picked = take((size_t)n * 4);
  l.total_forward = at;
  at = 0;
  l.dz = take((size_t)n * std::min(vocab, kPiece) * 4);
  l.live_feat = take((size_t)n * feat_len * dtype_size(dtype));
  l.acc = take((size_t)n * feat_len * 4);
  l.total_grad = at;
  return l;
}

int check_xent(const void* feat, const void* weight, int32_t dtype, int64_t feat_ld,
               int64_t weight_ld, const void* labels, int32_t index_type, int64_t n, int64_t vocab,
               int64_t feat_len, const int32_t* status) {
  if (!dtype_known(dtype) || !index_known(index_type))
    return fail(FG_ERR_INVALID_ARGUMENT, "unknown dtype=%d or index_type=%d", (int)dtype,
                (int)index_type);
  if (n < 0 || vocab < 1 || feat_len < 1 || feat_ld < feat_len || weight_ld < feat_len)
    return fail(FG_ERR_INVALID_ARGUMENT,
                "bad shape: n=%lld vocab=%lld feat_len=%lld feat_ld=%lld weight_ld=%lld",
                (long long)n, (long long)vocab, (long long)feat_len, (long long)feat_ld,
                (long long)weight_ld);
  if (n >= INT32_MAX / 2 || vocab >= INT32_MAX / 2 || feat_len > (1 << 20))
    return fail(FG_ERR_UNSUPPORTED, "n and vocab must be below 2^30, feat_len at most 2^20");
  if (!weight || (n > 0 && (!feat || !labels || !status)))
    return fail(FG_ERR_INVALID_ARGUMENT, "null pointer");
  const size_t es = dtype_size(dtype);
  if (((uintptr_t)feat | (uintptr_t)weight) % es != 0)
    return fail(FG_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its type");
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" int64_t fg_softmax_xent_workspace_bytes(int32_t dtype, int64_t n, int64_t vocab,
                                                   int64_t feat_len, int32_t with_grad) {
  if (n <= 0 || vocab < 1 || feat_len < 1) return 0;
  const fg::XentLayout l = fg::xent_layout(dtype, n, vocab, feat_len);
  return (int64_t)(with_grad ? std::max(l.total_forward, l.total_grad) : l.total_forward);
}

extern "C" int fg_softmax_xent(const void* feat_dev, int64_t feat_ld, const void* weight_dev,
                               int64_t weight_ld, int32_t dtype, const void* labels_dev,
                               int32_t index_type, int64_t n, int64_t vocab, int64_t feat_len,
                               float scale, int64_t ignore_index, float* loss_dev, float* lse_dev,
                               void* workspace_dev, int64_t workspace_bytes, int32_t* status_dev,
                               int32_t device, void* stream) {
  using namespace fg;
  if (int rc = check_xent(feat_dev, weight_dev, dtype, feat_ld, weight_ld, labels_dev, index_type,
                          n, vocab, feat_len, status_dev))
    return rc;
  if (n == 0) return FG_OK;
  if (!loss_dev || !lse_dev) return fail(FG_ERR_INVALID_ARGUMENT, "null loss or lse");
  const XentLayout l = xent_layout(dtype, n, vocab, feat_len);
  if (!workspace_dev || ((uintptr_t)workspace_dev & 255) != 0 ||
      workspace_bytes < (int64_t)l.total_forward)
    return fail(FG_ERR_INVALID_ARGUMENT, "the workspace needs %lld bytes at a 256-byte boundary",
                (long long)l.total_forward);
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace_dev);
  const Batch b = {labels_dev, index_type == FG_INDEX_INT64, n, vocab, feat_len, ignore_index, scale};
  float2* stats = reinterpret_cast<float2*>(ws + l.stats);
  float* picked = reinterpret_cast<float*>(ws + l.picked);
  const int64_t tiles = (vocab + kTile - 1) / kTile;
  const dim3 grid((unsigned)tiles, (unsigned)((n + kTile - 1) / kTile));
#define FG_STATS(T)                                                                        \
  logit_stats_kernel<T><<<grid, 256, 0, s>>>(b, static_cast<const T*>(feat_dev), feat_ld,  \
                                             static_cast<const T*>(weight_dev), weight_ld, \
                                             stats, picked)
  FG_DISPATCH_DTYPE(dtype, FG_STATS)
#undef FG_STATS
  FG_CUDA_TRY(cudaGetLastError());
  join_stats_kernel<<<(unsigned)((n + 7) / 8), 256, 0, s>>>(b, stats, tiles, picked, loss_dev,
                                                            lse_dev, status_dev);
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}

extern "C" int fg_softmax_xent_grad(const float* loss_grad_dev, const void* feat_dev,
                                    int64_t feat_ld, const void* weight_dev, int64_t weight_ld,
                                    int32_t dtype, const void* labels_dev, int32_t index_type,
                                    int64_t n, int64_t vocab, int64_t feat_len, float scale,
                                    int64_t ignore_index, const float* lse_dev,
                                    void* feat_grad_dev, void* weight_grad_dev,
                                    void* workspace_dev, int64_t workspace_bytes,
                                    int32_t* status_dev, int32_t device, void* stream) {
  using namespace fg;
  if (int rc = check_xent(feat_dev, weight_dev, dtype, feat_ld, weight_ld, labels_dev, index_type,
                          n, vocab, feat_len, status_dev))
    return rc;
  if (!feat_grad_dev && !weight_grad_dev)
    return fail(FG_ERR_INVALID_ARGUMENT, "neither gradient is asked for");
  if (n > 0) {
    if (!loss_grad_dev || !lse_dev) return fail(FG_ERR_INVALID_ARGUMENT, "null loss_grad or lse");
    const int64_t need = fg_softmax_xent_workspace_bytes(dtype, n, vocab, feat_len, 1);
    if (!workspace_dev || ((uintptr_t)workspace_dev & 255) != 0 || workspace_bytes < need)
      return fail(FG_ERR_INVALID_ARGUMENT, "the workspace needs %lld bytes at a 256-byte boundary",
                  (long long)need);
  }
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    if (weight_grad_dev)
      FG_CUDA_TRY(cudaMemsetAsync(weight_grad_dev, 0, (size_t)vocab * feat_len * dtype_size(dtype), s));
    return FG_OK;
  }
  const XentLayout l = xent_layout(dtype, n, vocab, feat_len);
  char* ws = static_cast<char*>(workspace_dev);
  const Batch b = {labels_dev, index_type == FG_INDEX_INT64, n, vocab, feat_len, ignore_index, scale};
  float* dz = reinterpret_cast<float*>(ws + l.dz);
  float* acc = reinterpret_cast<float*>(ws + l.acc);
  const unsigned t_tiles = (unsigned)((n + kTile - 1) / kTile);
  const unsigned d_tiles = (unsigned)((feat_len + kTile - 1) / kTile);
#define FG_LIVE(T)                                                                         \
  live_feat_kernel<T><<<(unsigned)((n * feat_len + 255) / 256), 256, 0, s>>>(              \
      b, static_cast<const T*>(feat_dev), feat_ld, reinterpret_cast<T*>(ws + l.live_feat))
  FG_DISPATCH_DTYPE(dtype, FG_LIVE)
#undef FG_LIVE
  for (int64_t v0 = 0; v0 < vocab; v0 += kPiece) {
    const int64_t count = std::min(kPiece, vocab - v0);
    const unsigned v_tiles = (unsigned)((count + kTile - 1) / kTile);
#define FG_PIECE(T)                                                                              \
  {                                                                                              \
    const T* w = static_cast<const T*>(weight_dev);                                              \
    logit_grad_kernel<T><<<dim3(v_tiles, t_tiles), 256, 0, s>>>(                                 \
        b, static_cast<const T*>(feat_dev), feat_ld, w, weight_ld, lse_dev, loss_grad_dev, v0,   \
        count, dz);                                                                              \
    if (feat_grad_dev)                                                                           \
      feat_grad_kernel<T><<<dim3(d_tiles, t_tiles), 256, 0, s>>>(                                \
          b, dz, w, weight_ld, v0, count, acc, static_cast<T*>(feat_grad_dev), v0 == 0,          \
          v0 + count == vocab);                                                                  \
    if (weight_grad_dev)                                                                         \
      weight_grad_kernel<T><<<dim3(d_tiles, v_tiles), 256, 0, s>>>(                              \
          b, dz, reinterpret_cast<const T*>(ws + l.live_feat), feat_len, v0, count,              \
          static_cast<T*>(weight_grad_dev));                                                     \
  }
    FG_DISPATCH_DTYPE(dtype, FG_PIECE)
#undef FG_PIECE
  }
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}
