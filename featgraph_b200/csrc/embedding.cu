// Vertex embedding lookup with scaling, and its gradient by sorted ids.
//
//   out[i, :]  = scale * table[ids[i], :]
//   grad[v, :] = scale * sum of out_grad[i, :] over the i with ids[i] = v, i ascending
//
// Both only move bytes: the lookup reads the rows it names and writes them once, the gradient
// reads every row of out_grad once and writes every row of the table's gradient once.
#include <algorithm>
#include <cmath>

#include "elem.cuh"

namespace fg {
namespace {

__device__ __forceinline__ int64_t load_index(const void* ids, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long*>(ids) + i)
              : (int64_t)__ldg(static_cast<const int*>(ids) + i);
}

// ------------------------------------------------------------------ lookup --
// A group of `lanes` (a power of two, at most 32) lanes copies kRows rows side by side: their
// ids first, then the kRows gathers, so that a lane has kRows loads of up to 16 bytes in
// flight behind one round trip for the ids.
constexpr int kLookupThreads = 256;
constexpr int kLookupRows = 4;

template <typename T, int N>
__global__ void __launch_bounds__(kLookupThreads)
lookup_kernel(const T* __restrict__ table, int64_t table_ld, int64_t n_vertices,
              const void* __restrict__ ids, int wide, int64_t n_ids, int feat_len, float scale,
              T* __restrict__ out, int64_t out_ld, int log_lanes, int32_t* status) {
  const int lanes = 1 << log_lanes;
  const int64_t group = ((int64_t)blockIdx.x * kLookupThreads + threadIdx.x) >> log_lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t n_groups = ((int64_t)gridDim.x * kLookupThreads) >> log_lanes;
  for (int64_t first = group; first < n_ids; first += n_groups * kLookupRows) {
    int64_t id[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      const int64_t i = first + u * n_groups;
      id[u] = i < n_ids ? load_index(ids, wide, i) : 0;
    }
    bool bad[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      bad[u] = (uint64_t)id[u] >= (uint64_t)n_vertices;
      if (bad[u] && lane == 0) *status = FG_STATUS_BAD_INDEX;
    }
    for (int c = lane * N; c < feat_len; c += lanes * N) {
      Vec<T, N> row[kLookupRows];
#pragma unroll
      for (int u = 0; u < kLookupRows; ++u)
        if (!bad[u] && first + u * n_groups < n_ids)
          row[u] = load_vec<T, N>(table + id[u] * table_ld + c);
#pragma unroll
      for (int u = 0; u < kLookupRows; ++u) {
        const int64_t i = first + u * n_groups;
        if (i >= n_ids) break;
#pragma unroll
        for (int k = 0; k < N; ++k)
          row[u].v[k] = from_float<T>(bad[u] ? __int_as_float(0x7fc00000)
                                             : to_float<T>(row[u].v[k]) * scale);
        store_vec_stream<T, N>(out + i * out_ld + c, row[u]);
      }
    }
  }
}

// ------------------------------------------------------- gradient: the sort --
// Stable least-significant-digit radix sort of (id, position) pairs, at most 9 bits a pass:
// per block of kSortTile keys a histogram (sort_count_kernel), per digit an exclusive sum over
// the blocks (sort_scan_kernel), then every key to its place (sort_place_kernel).  Equal ids
// keep the order of their positions, so the sums below run in an order that only the ids fix.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 16;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;

// The key of position i: its id, or n_vertices for a row that gets no gradient (the padding
// id, or an id out of range), which sorts behind every vertex.
struct KeySource {
  const void* ids;           // first pass: the caller's ids
  const uint32_t* keys;      // later passes: the pairs of the pass before
  const uint32_t* positions;
  int wide;
  int64_t n_vertices;
  int64_t padding;           // -1: none
  int32_t* status;
};
__device__ __forceinline__ uint32_t source_key(const KeySource& s, int64_t i) {
  if (s.keys) return s.keys[i];
  const int64_t id = load_index(s.ids, s.wide, i);
  if ((uint64_t)id >= (uint64_t)s.n_vertices) {
    *s.status = FG_STATUS_BAD_INDEX;
    return (uint32_t)s.n_vertices;
  }
  return id == s.padding ? (uint32_t)s.n_vertices : (uint32_t)id;
}

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(KeySource src, int64_t n, int shift, int bits, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kMaxBins];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
#pragma unroll 4
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = base + k * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(source_key(src, i) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads)
    counts[(int64_t)b * gridDim.x + blockIdx.x] = hist[b];
}

// One warp per digit: counts[digit][block] becomes the digit's count in the blocks before.
__global__ void __launch_bounds__(kSortThreads)
sort_scan_kernel(uint32_t* __restrict__ counts, int n_blocks, int bins,
                 uint32_t* __restrict__ totals) {
  const int digit = blockIdx.x * kSortWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (digit >= bins) return;
  uint32_t* row = counts + (int64_t)digit * n_blocks;
  uint32_t running = 0;
  for (int b0 = 0; b0 < n_blocks; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t c = b < n_blocks ? row[b] : 0;
    uint32_t incl = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    if (b < n_blocks) row[b] = running + incl - c;
    running += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) totals[digit] = running;
}

__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(KeySource src, int64_t n, int shift, int bits,
                  const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                  uint32_t* __restrict__ keys_out, uint32_t* __restrict__ positions_out) {
  __shared__ uint32_t warp_hist[kSortWarps][kMaxBins];
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t warp_sum[kSortWarps];
  const int bins = 1 << bits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads)
    (&warp_hist[0][0])[b] = 0;
  // exclusive sum of the digits' totals: bins / kSortThreads = at most two digits a thread
  const int per = (bins + kSortThreads - 1) / kSortThreads;
  uint32_t mine = 0;
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    if (b < bins) mine += totals[b];
  }
  uint32_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  uint32_t before = incl - mine;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    if (b < bins) {
      base[b] = before + counts[(int64_t)b * gridDim.x + blockIdx.x];
      before += totals[b];
    }
  }
  // each warp takes kSortItems * 32 consecutive keys, 32 at a time and in order
  const int64_t first = (int64_t)blockIdx.x * kSortTile + warp * (kSortItems * 32);
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = first + k * 32 + lane;
    const bool live = i < n;
    key[k] = live ? source_key(src, i) : 0;
    const uint32_t digit = live ? (key[k] >> shift) & (bins - 1) : (uint32_t)bins;
    const uint32_t peers = __match_any_sync(0xffffffffu, digit);
    const uint32_t below = __popc(peers & ((1u << lane) - 1));
    uint32_t old = 0;
    if (live) old = warp_hist[warp][digit];
    __syncwarp();
    if (live && below == 0) warp_hist[warp][digit] = old + __popc(peers);
    __syncwarp();
    rank[k] = old + below;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) {
    uint32_t run = base[b];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = warp_hist[w][b];
      warp_hist[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = first + k * 32 + lane;
    if (i >= n) continue;
    const uint32_t at = warp_hist[warp][(key[k] >> shift) & (bins - 1)] + rank[k];
    keys_out[at] = key[k];
    positions_out[at] = src.keys ? src.positions[i] : (uint32_t)i;
  }
}

// ------------------------------------------------------- gradient: the sums --
template <typename T, int N>
__device__ __forceinline__ void store_grad_row(T* p, const float (&acc)[N], float scale,
                                               int accumulate) {
  Vec<T, N> v;
  if (accumulate) v = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int k = 0; k < N; ++k)
    v.v[k] = from_float<T>(accumulate ? to_float<T>(v.v[k]) + acc[k] * scale : acc[k] * scale);
  store_vec<T, N>(p, v);
}

// The sorted list is cut into pieces of `piece` positions; a group of lanes walks one piece
// and sums its rows.  A vertex whose rows all lie inside the piece is written at once; the sum
// of one that began in an earlier piece goes to partial[piece][0], of one that goes on into
// the next piece to partial[piece][1] (a piece that is one vertex throughout uses only [0]
// unless the vertex begins there), and join_kernel adds those up in order.
constexpr int kSumThreads = 256;
constexpr int kSumAhead = 8;

template <typename T, int N>
__global__ void __launch_bounds__(kSumThreads)
sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ positions, int64_t n,
           int64_t n_vertices, const T* __restrict__ out_grad, int64_t out_grad_ld, int feat_len,
           float scale, int accumulate, T* __restrict__ grad, float* __restrict__ partial,
           int piece, int log_lanes, int slabs) {
  const int lanes = 1 << log_lanes;
  const int64_t item = ((int64_t)blockIdx.x * kSumThreads + threadIdx.x) >> log_lanes;
  const int64_t p = item / slabs;
  const int c = ((int)(item - p * slabs) * lanes + (threadIdx.x & (lanes - 1))) * N;
  const int64_t begin = p * piece;
  if (begin >= n || c >= feat_len) return;
  const int64_t end = begin + piece < n ? begin + piece : n;
  const uint32_t none = (uint32_t)n_vertices;
  uint32_t current = keys[begin];
  bool open_before = begin > 0 && keys[begin - 1] == current;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  for (int64_t j = begin; j < end; j += kSumAhead) {
    uint32_t key[kSumAhead];
    Vec<T, N> row[kSumAhead];
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      key[u] = j + u < end ? keys[j + u] : none;
      if (key[u] != none)
        row[u] = load_vec_stream<T, N>(out_grad + (int64_t)positions[j + u] * out_grad_ld + c);
    }
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      if (j + u >= end) break;
      if (key[u] != current) {
        if (current != none) {
          if (open_before) {
            float* to = partial + (p * 2 + 0) * feat_len + c;
#pragma unroll
            for (int k = 0; k < N; ++k) to[k] = acc[k];
          } else {
            store_grad_row<T, N>(grad + (int64_t)current * feat_len + c, acc, scale, accumulate);
          }
        }
        open_before = false;
        current = key[u];
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = 0.f;
      }
      if (key[u] != none) {
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += to_float<T>(row[u].v[k]);
      }
    }
  }
  if (current == none) return;
  const bool open_after = end < n && keys[end] == current;
  if (!open_before && !open_after) {
    store_grad_row<T, N>(grad + (int64_t)current * feat_len + c, acc, scale, accumulate);
  } else {
    float* to = partial + (p * 2 + (open_before ? 0 : 1)) * feat_len + c;
#pragma unroll
    for (int k = 0; k < N; ++k) to[k] = acc[k];
  }
}

// One CTA per piece; works only where a vertex begins in the piece and goes on behind it.  Its
// partial sums are partial[piece][1], then partial[q][0] of the pieces q that it reaches:
// every column's are cut into kJoinParts runs, summed in order, and the runs added in order.
constexpr int kJoinParts = 8;
constexpr int kJoinColumns = 32;

template <typename T>
__global__ void __launch_bounds__(kJoinParts * kJoinColumns)
join_kernel(const uint32_t* __restrict__ keys, int64_t n, int64_t n_vertices, int feat_len,
            float scale, int accumulate, T* __restrict__ grad, const float* __restrict__ partial,
            int piece) {
  const int64_t p = blockIdx.x;
  const int64_t end = (p + 1) * piece;
  if (end >= n) return;
  const uint32_t key = keys[end - 1];
  if (key == (uint32_t)n_vertices || keys[end] != key) return;
  const int64_t begin = p * piece;
  if (begin > 0 && keys[begin] == key && keys[begin - 1] == key) return;  // it began earlier
  // the last piece that the vertex reaches: the first position behind it, by bisection
  int64_t lo = end, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] == key) lo = mid + 1; else hi = mid;
  }
  const int64_t last = (lo - 1) / piece;
  const int64_t terms = last - p + 1;
  const int part = threadIdx.x / kJoinColumns, lane = threadIdx.x % kJoinColumns;
  const int64_t per = (terms + kJoinParts - 1) / kJoinParts;
  __shared__ float sums[kJoinParts][kJoinColumns];
  for (int c0 = 0; c0 < feat_len; c0 += kJoinColumns) {
    const int c = c0 + lane;
    float s = 0.f;
    if (c < feat_len) {
      const int64_t t1 = (part + 1) * per < terms ? (part + 1) * per : terms;
#pragma unroll 8
      for (int64_t t = part * per; t < t1; ++t)
        s += partial[((p + t) * 2 + (t == 0 ? 1 : 0)) * feat_len + c];
    }
    sums[part][lane] = s;
    __syncthreads();
    if (part == 0 && c < feat_len) {
      float total = 0.f;
#pragma unroll
      for (int q = 0; q < kJoinParts; ++q) total += sums[q][lane];
      float one[1] = {total};
      store_grad_row<T, 1>(grad + (int64_t)key * feat_len + c, one, scale, accumulate);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------- host --
int ceil_log2(int64_t v) {
  int b = 0;
  while (((int64_t)1 << b) < v) ++b;
  return b;
}

struct GradLayout {
  int piece;
  int64_t pieces, blocks;
  int passes, digit_bits;
  size_t keys[2], positions[2], counts, totals, partial, total;
};

GradLayout grad_layout(int64_t n, int64_t n_vertices, int64_t feat_len) {
  GradLayout l;
  l.piece = 32;
  l.pieces = (n + l.piece - 1) / l.piece;
  l.blocks = (n + kSortTile - 1) / kSortTile;
  const int bits = std::max(1, ceil_log2(n_vertices + 1));  // n_vertices itself is a key
  l.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  l.digit_bits = (bits + l.passes - 1) / l.passes;
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int k = 0; k < 2; ++k) {
    l.keys[k] = take((size_t)n * 4);
    l.positions[k] = take((size_t)n * 4);
  }
  l.counts = take(((size_t)l.blocks << l.digit_bits) * 4);
  l.totals = take(kMaxBins * 4);
  l.partial = take((size_t)l.pieces * 2 * feat_len * 4);
  l.total = at;
  return l;
}

int check_common(const void* values, const void* ids, const int32_t* status, int32_t dtype,
                 int32_t index_type, int64_t n_vertices, int64_t n_ids, int64_t feat_len) {
  if (!dtype_known(dtype) || !index_known(index_type))
    return fail(FG_ERR_INVALID_ARGUMENT, "unknown dtype=%d or index_type=%d", (int)dtype,
                (int)index_type);
  if (n_vertices < 0 || n_ids < 0 || feat_len < 1)
    return fail(FG_ERR_INVALID_ARGUMENT, "bad shape: n_vertices=%lld n_ids=%lld feat_len=%lld",
                (long long)n_vertices, (long long)n_ids, (long long)feat_len);
  if (n_vertices >= INT32_MAX || n_ids >= INT32_MAX || feat_len > (1 << 24))
    return fail(FG_ERR_UNSUPPORTED, "n_vertices, n_ids must be below 2^31 - 1, feat_len at most 2^24");
  if (n_ids > 0 && (!values || !ids || !status))
    return fail(FG_ERR_INVALID_ARGUMENT, "null pointer");
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" int fg_embedding_lookup(const void* table_dev, int32_t dtype, int64_t table_ld,
                                   int64_t n_vertices, const void* ids_dev, int32_t index_type,
                                   int64_t n_ids, int64_t feat_len, float scale, void* out_dev,
                                   int64_t out_ld, int32_t* status_dev, int32_t device,
                                   void* stream) {
  using namespace fg;
  if (int rc = check_common(out_dev, ids_dev, status_dev, dtype, index_type, n_vertices, n_ids,
                            feat_len))
    return rc;
  if (table_ld < feat_len || out_ld < feat_len)
    return fail(FG_ERR_INVALID_ARGUMENT, "a row pitch is shorter than feat_len=%lld",
                (long long)feat_len);
  if (n_ids == 0) return FG_OK;
  if (n_vertices > 0 && !table_dev) return fail(FG_ERR_INVALID_ARGUMENT, "null table");
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  const size_t es = dtype_size(dtype);
  const int vb = common_vector_bytes({(uint64_t)(uintptr_t)table_dev, (uint64_t)(uintptr_t)out_dev,
                                      (uint64_t)(table_ld * es), (uint64_t)(out_ld * es),
                                      (uint64_t)(feat_len * es)});
  if (vb < (int)es) return fail(FG_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its type");
  const int per_row = (int)((feat_len * es + vb - 1) / vb);
  const int log_lanes = std::min(5, ceil_log2(per_row));
  const int64_t groups_per_block = kLookupThreads >> log_lanes;
  const int64_t want = (n_ids + groups_per_block * kLookupRows - 1) / (groups_per_block * kLookupRows);
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(want, 1), 1 << 20);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FG_LOOKUP(T, N)                                                                        \
  lookup_kernel<T, N><<<grid, kLookupThreads, 0, s>>>(                                         \
      static_cast<const T*>(table_dev), table_ld, n_vertices, ids_dev,                         \
      index_type == FG_INDEX_INT64, n_ids, (int)feat_len, scale, static_cast<T*>(out_dev),     \
      out_ld, log_lanes, status_dev)
#define FG_LOOKUP_T(T)                                                    \
  switch (vb / (int)sizeof(T)) {                                          \
    case 8: if constexpr (sizeof(T) == 2) FG_LOOKUP(T, 8 / (sizeof(T) / 2)); break; \
    case 4: FG_LOOKUP(T, 4); break;                                       \
    case 2: FG_LOOKUP(T, 2); break;                                       \
    default: FG_LOOKUP(T, 1); break;                                      \
  }
  FG_DISPATCH_DTYPE(dtype, FG_LOOKUP_T)
#undef FG_LOOKUP_T
#undef FG_LOOKUP
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}

extern "C" int64_t fg_embedding_grad_workspace_bytes(int64_t n_ids, int64_t n_vertices,
                                                     int64_t feat_len) {
  if (n_ids <= 0 || n_vertices < 0 || feat_len < 1) return 0;
  return (int64_t)fg::grad_layout(n_ids, n_vertices, feat_len).total;
}

extern "C" int fg_embedding_grad(const void* out_grad_dev, int32_t dtype, int64_t out_grad_ld,
                                 const void* ids_dev, int32_t index_type, int64_t n_ids,
                                 int64_t n_vertices, int64_t feat_len, float scale,
                                 int64_t padding_id, int32_t accumulate, void* grad_dev,
                                 void* workspace_dev, int64_t workspace_bytes,
                                 int32_t* status_dev, int32_t device, void* stream) {
  using namespace fg;
  if (int rc = check_common(out_grad_dev, ids_dev, status_dev, dtype, index_type, n_vertices,
                            n_ids, feat_len))
    return rc;
  if (out_grad_ld < feat_len)
    return fail(FG_ERR_INVALID_ARGUMENT, "a row pitch is shorter than feat_len=%lld",
                (long long)feat_len);
  if (padding_id >= n_vertices)
    return fail(FG_ERR_INVALID_ARGUMENT, "padding_id=%lld is not below n_vertices=%lld",
                (long long)padding_id, (long long)n_vertices);
  if (n_vertices == 0 && n_ids == 0) return FG_OK;
  if (n_vertices > 0 && !grad_dev) return fail(FG_ERR_INVALID_ARGUMENT, "null gradient");
  const GradLayout l = grad_layout(std::max<int64_t>(n_ids, 1), n_vertices, feat_len);
  if (n_ids > 0 && (!workspace_dev || workspace_bytes < (int64_t)l.total ||
                    ((uintptr_t)workspace_dev & 15) != 0))
    return fail(FG_ERR_INVALID_ARGUMENT, "the workspace needs %lld bytes at a 16-byte boundary",
                (long long)l.total);
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  const size_t es = dtype_size(dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int vb = common_vector_bytes({(uint64_t)(uintptr_t)out_grad_dev,
                                      (uint64_t)(uintptr_t)grad_dev, (uint64_t)(out_grad_ld * es),
                                      (uint64_t)(feat_len * es)});
  if (vb < (int)es) return fail(FG_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its type");
  if (!accumulate && n_vertices > 0)
    FG_CUDA_TRY(cudaMemsetAsync(grad_dev, 0, (size_t)n_vertices * feat_len * es, s));
  if (n_ids == 0) return FG_OK;

  char* ws = static_cast<char*>(workspace_dev);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws + l.keys[0]),
                       reinterpret_cast<uint32_t*>(ws + l.keys[1])};
  uint32_t* positions[2] = {reinterpret_cast<uint32_t*>(ws + l.positions[0]),
                            reinterpret_cast<uint32_t*>(ws + l.positions[1])};
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + l.counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + l.totals);
  float* partial = reinterpret_cast<float*>(ws + l.partial);
  KeySource src = {ids_dev, nullptr, nullptr, index_type == FG_INDEX_INT64, n_vertices,
                   padding_id < 0 ? -1 : padding_id, status_dev};
  const int bins = 1 << l.digit_bits;
  for (int pass = 0; pass < l.passes; ++pass) {
    const int shift = pass * l.digit_bits;
    sort_count_kernel<<<(int)l.blocks, kSortThreads, 0, s>>>(src, n_ids, shift, l.digit_bits, counts);
    sort_scan_kernel<<<(bins + kSortWarps - 1) / kSortWarps, kSortThreads, 0, s>>>(
        counts, (int)l.blocks, bins, totals);
    sort_place_kernel<<<(int)l.blocks, kSortThreads, 0, s>>>(
        src, n_ids, shift, l.digit_bits, counts, totals, keys[pass & 1], positions[pass & 1]);
    src.keys = keys[pass & 1];
    src.positions = positions[pass & 1];
  }
  const int per_row = (int)((feat_len * es + vb - 1) / vb);
  const int log_lanes = std::min(5, ceil_log2(per_row));
  const int slabs = (per_row + (1 << log_lanes) - 1) >> log_lanes;
  const int64_t threads = (l.pieces * slabs) << log_lanes;
  const int64_t grid = (threads + kSumThreads - 1) / kSumThreads;
  if (grid > INT32_MAX) return fail(FG_ERR_UNSUPPORTED, "n_ids x feat_len is too large");
#define FG_SUM(T, N)                                                                          \
  sum_kernel<T, N><<<(int)grid, kSumThreads, 0, s>>>(                                         \
      src.keys, src.positions, n_ids, n_vertices, static_cast<const T*>(out_grad_dev),        \
      out_grad_ld, (int)feat_len, scale, accumulate, static_cast<T*>(grad_dev), partial,      \
      l.piece, log_lanes, slabs)
#define FG_SUM_T(T)                                                       \
  switch (vb / (int)sizeof(T)) {                                          \
    case 8: if constexpr (sizeof(T) == 2) FG_SUM(T, 8 / (sizeof(T) / 2)); break; \
    case 4: FG_SUM(T, 4); break;                                          \
    case 2: FG_SUM(T, 2); break;                                          \
    default: FG_SUM(T, 1); break;                                         \
  }                                                                       \
  join_kernel<T><<<(int)l.pieces, kJoinParts * kJoinColumns, 0, s>>>(     \
      src.keys, n_ids, n_vertices, (int)feat_len, scale, accumulate,      \
      static_cast<T*>(grad_dev), partial, l.piece);
  FG_DISPATCH_DTYPE(dtype, FG_SUM_T)
#undef FG_SUM_T
#undef FG_SUM
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}
