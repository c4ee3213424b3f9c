// Vertex embedding lookup with scaling, and its gradient by sorted ids.
//
//   out[i, :]  = scale * table[ids[i], :]
//   grad[v, :] = scale * sum of out_grad[i, :] over the i with ids[i] = v, i ascending
//
// Both only move bytes: the lookup reads the rows it names and writes them once, the gradient
// reads every row of out_grad once and writes every row of the table's gradient once.  On one
// B200, 1 048 576 rows of 256 bytes, a table of 232 965, skewed ids: lookup 67 us (4.9 TB/s),
// gradient 144 us, of which 85 are the sums (3.4 TB/s of rows in random order) and 40 the sort.
#include <algorithm>
#include <cmath>

#include "elem.cuh"

namespace fg {
namespace {

// The ids' type is a template parameter wherever a thread loads several: a choice at every load
// makes each wait for the one before (5003 ids by 512 threads: 8000 cycles instead of 2000).
template <typename I>
__device__ __forceinline__ I load_id(const void* ids, int64_t i) {
  return __ldg(static_cast<const I*>(ids) + i);
}
// ------------------------------------------------------------------ lookup --
// A group of `lanes` (a power of two, at most 32) lanes copies kLookupRows consecutive rows side
// by side, so that a lane has that many loads of up to 16 bytes in flight, and has the ids of
// its next rows on the way meanwhile.
constexpr int kLookupThreads = 256;
constexpr int kLookupRows = 4;
constexpr int kLookupBlocks = 4;   // CTAs on an SM: 1M rows of 256 bytes 67 us; 8 rows and 2 CTAs took 14 % more

template <typename T, int N, typename I>
__global__ void __launch_bounds__(kLookupThreads, kLookupBlocks)
lookup_kernel(const T* __restrict__ table, int64_t table_ld, int64_t n_vertices,
              const void* __restrict__ ids, int64_t n_ids, int feat_len, float scale,
              T* __restrict__ out, int64_t out_ld, int log_lanes, int32_t* status) {
  const int lanes = 1 << log_lanes;
  const int64_t group = ((int64_t)blockIdx.x * kLookupThreads + threadIdx.x) >> log_lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t stride = (((int64_t)gridDim.x * kLookupThreads) >> log_lanes) * kLookupRows;
  int64_t first = group * kLookupRows;
  I id[kLookupRows];
#pragma unroll
  for (int u = 0; u < kLookupRows; ++u)
    id[u] = first + u < n_ids ? load_id<I>(ids, first + u) : 0;
  for (; first < n_ids; first += stride) {
    bool ok[kLookupRows];
    int64_t from[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      const bool in = first + u < n_ids;
      ok[u] = in && (uint64_t)(int64_t)id[u] < (uint64_t)n_vertices;
      if (in && !ok[u] && lane == 0) report(status, FG_STATUS_BAD_INDEX);
      from[u] = id[u] * table_ld;
      id[u] = first + stride + u < n_ids ? load_id<I>(ids, first + stride + u) : 0;
    }
    for (int c = lane * N; c < feat_len; c += lanes * N) {
      Vec<T, N> row[kLookupRows];
#pragma unroll
      for (int u = 0; u < kLookupRows; ++u)
        if (ok[u]) row[u] = load_vec<T, N>(table + from[u] + c);
#pragma unroll
      for (int u = 0; u < kLookupRows; ++u) {
        if (first + u >= n_ids) break;
        float x[N];
        unpack<T, N>(row[u], x);
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = ok[u] ? x[k] * scale : __int_as_float(0x7fc00000);
        store_vec_stream<T, N>(out + (first + u) * out_ld + c, pack<T, N>(x));
      }
    }
  }
}

// ------------------------------------------------------- gradient: the sort --
// The key of position i: its id, or n_vertices for a row that gets no gradient (the padding
// id, or an id out of range), which sorts behind every vertex.
struct KeySource {
  const void* from;          // the caller's ids, or the pairs of the pass before
  int64_t n_vertices;
  int64_t padding;           // -1: none
  int32_t* status;
};
// What keys are made of as it lies in memory (S: int, long long, or uint2 for pairs), and the
// pair it makes.  Apart, so that a thread has all its loads on the way before it looks at the
// first (and may have to report it).
template <typename S>
__device__ __forceinline__ S load_source(const KeySource& s, int64_t i) {
  if constexpr (std::is_same<S, uint2>::value)
    return static_cast<const uint2*>(s.from)[i];
  else
    return load_id<S>(s.from, i);
}
template <typename S>
__device__ __forceinline__ uint2 make_pair(const KeySource& s, S id, int64_t i) {
  if constexpr (std::is_same<S, uint2>::value) {
    return id;
  } else {
    const int64_t v = id;
    uint32_t key = (uint32_t)v;
    if ((uint64_t)v >= (uint64_t)s.n_vertices) {
      report(s.status, FG_STATUS_BAD_INDEX);
      key = (uint32_t)s.n_vertices;
    } else if (v == s.padding) {
      key = (uint32_t)s.n_vertices;
    }
    return make_uint2(key, (uint32_t)i);
  }
}

// The table's gradient starts as zeros: spare CTAs of the sort's kernels write a part of them
// each while the others wait for memory anyway.  `bytes` of it at `to`.
struct ZeroFill {
  uint8_t* to;
  int64_t bytes;
};
__device__ __forceinline__ void zero_fill(const ZeroFill& z, int block, int blocks, int threads) {
  const int64_t head = min(z.bytes, (int64_t)((16 - (uintptr_t)z.to % 16) % 16));
  const int64_t vecs = (z.bytes - head) / 16;
  uint4* at = reinterpret_cast<uint4*>(z.to + head);
  for (int64_t i = (int64_t)block * threads + threadIdx.x; i < vecs; i += (int64_t)blocks * threads)
    at[i] = make_uint4(0, 0, 0, 0);
  if (block == 0) {
    for (int64_t i = threadIdx.x; i < head; i += threads) z.to[i] = 0;
    for (int64_t i = head + vecs * 16 + threadIdx.x; i < z.bytes; i += threads) z.to[i] = 0;
  }
}

// Stable least-significant-digit radix sort of (id, position) pairs, at most 9 bits a pass:
// per block of kSortTile keys a histogram (sort_count_kernel), per digit an exclusive sum over
// the blocks (sort_scan_kernel), then every pair to its place (sort_place_kernel).  Equal ids
// keep the order of their positions, so the sums below run in an order that only the ids fix.
// All keys of a thread are loaded before the first is used: with the loads inside the ranking
// rounds a block took 22 us.
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;
static_assert(kMaxBins == kSortThreads, "one thread per digit");

template <typename S>
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(KeySource src, int64_t n, int shift, int bits, uint32_t* __restrict__ counts,
                  int sort_blocks, ZeroFill zero) {
  begin_chained();
  if ((int)blockIdx.x >= sort_blocks) {
    zero_fill(zero, blockIdx.x - sort_blocks, gridDim.x - sort_blocks, kSortThreads);
    return;
  }
  __shared__ uint32_t hist[kMaxBins];
  const int bins = 1 << bits;
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  S id[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = base + k * kSortThreads + threadIdx.x;
    id[k] = i < n ? load_source<S>(src, i) : S();
  }
  hist[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k)
    if (base + k * kSortThreads + threadIdx.x < n)
      atomicAdd(&hist[(make_pair<S>(src, id[k], 0).x >> shift) & (bins - 1)], 1u);
  __syncthreads();
  if ((int)threadIdx.x < bins) counts[(int64_t)threadIdx.x * sort_blocks + blockIdx.x] = hist[threadIdx.x];
}

// One warp per digit: counts[digit][block] becomes the digit's count in the blocks before.
__global__ void __launch_bounds__(kSortThreads)
sort_scan_kernel(uint32_t* __restrict__ counts, int n_blocks, int bins,
                 uint32_t* __restrict__ totals) {
  begin_chained();
  const int digit = blockIdx.x * kSortWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (digit >= bins) return;
  uint32_t* row = counts + (int64_t)digit * n_blocks;
  uint32_t running = 0;
  for (int b0 = 0; b0 < n_blocks; b0 += 256) {
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = b0 + k * 32 + lane < n_blocks ? row[b0 + k * 32 + lane] : 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t incl = c[k];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      if (b0 + k * 32 + lane < n_blocks) row[b0 + k * 32 + lane] = running + incl - c[k];
      running += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  if (lane == 0) totals[digit] = running;
}

// A block orders its pairs in shared memory first, so that those of one digit (eight on
// average with 512 digits) are written side by side.
struct PlaceShared {
  uint2 pairs[kSortTile];
  uint16_t warp_hist[kSortWarps][kMaxBins];  // counts, then places within the block
  uint32_t base[kMaxBins];                   // where the digit's pairs go, less their place here
  uint32_t warp_sum[2][kSortWarps];
};

template <typename S>
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(KeySource src, int64_t n, int shift, int bits,
                  const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                  uint2* __restrict__ pairs_out, int sort_blocks, ZeroFill zero) {
  begin_chained();
  if ((int)blockIdx.x >= sort_blocks) {
    zero_fill(zero, blockIdx.x - sort_blocks, gridDim.x - sort_blocks, kSortThreads);
    return;
  }
  extern __shared__ __align__(16) uint8_t raw[];
  PlaceShared& sh = *reinterpret_cast<PlaceShared*>(raw);
  const int bins = 1 << bits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t block_first = (int64_t)blockIdx.x * kSortTile;
  // each warp takes kSortItems * 32 consecutive keys, 32 at a time and in order
  const int64_t first = block_first + warp * (kSortItems * 32);
  S id[kSortItems];
  uint2 pair[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = first + k * 32 + lane;
    id[k] = i < n ? load_source<S>(src, i) : S();
  }
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = first + k * 32 + lane;
    pair[k] = i < n ? make_pair<S>(src, id[k], i) : make_uint2(0, 0);
  }
  // a thread per digit: what it takes in all, and in the blocks before
  const int digit_here = threadIdx.x;
  const uint32_t total = digit_here < bins ? totals[digit_here] : 0;
  const uint32_t ahead = digit_here < bins ? counts[(int64_t)digit_here * sort_blocks + blockIdx.x] : 0;
  for (int b = threadIdx.x; b < kSortWarps * kMaxBins / 2; b += kSortThreads)
    reinterpret_cast<uint32_t*>(&sh.warp_hist[0][0])[b] = 0;
  __syncthreads();
  uint32_t rank[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const bool live = first + k * 32 + lane < n;
    const uint32_t digit = live ? (pair[k].x >> shift) & (bins - 1) : (uint32_t)bins;
    // the lanes with the same digit, bit by bit (__match_any_sync waits on the shared-memory
    // pipe: 17 us a pass of 1M keys)
    uint32_t peers = __ballot_sync(0xffffffffu, live);
    if (!live) peers = ~peers;
    for (int b = 0; b < bits; ++b) {
      const bool set = digit >> b & 1;
      const uint32_t votes = __ballot_sync(0xffffffffu, set);
      peers &= set ? votes : ~votes;
    }
    const uint32_t below = __popc(peers & ((1u << lane) - 1));
    uint32_t old = 0;
    if (live) old = sh.warp_hist[warp][digit];
    __syncwarp();
    if (live && below == 0) sh.warp_hist[warp][digit] = (uint16_t)(old + __popc(peers));
    __syncwarp();
    rank[k] = old + below;
  }
  __syncthreads();
  // exclusive sums over the digits, of their totals and of this block's counts
  uint32_t here = 0;
  if (digit_here < bins)
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) here += sh.warp_hist[w][digit_here];
  uint32_t sum_total = total, sum_here = here;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, sum_total, d);
    const uint32_t b = __shfl_up_sync(0xffffffffu, sum_here, d);
    if (lane >= d) {
      sum_total += a;
      sum_here += b;
    }
  }
  if (lane == 31) {
    sh.warp_sum[0][warp] = sum_total;
    sh.warp_sum[1][warp] = sum_here;
  }
  __syncthreads();
  for (int w = 0; w < warp; ++w) {
    sum_total += sh.warp_sum[0][w];
    sum_here += sh.warp_sum[1][w];
  }
  if (digit_here < bins) {
    uint32_t run = sum_here - here;
    sh.base[digit_here] = sum_total - total + ahead - run;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = sh.warp_hist[w][digit_here];
      sh.warp_hist[w][digit_here] = (uint16_t)run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k)
    if (first + k * 32 + lane < n)
      sh.pairs[sh.warp_hist[warp][(pair[k].x >> shift) & (bins - 1)] + rank[k]] = pair[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int i = k * kSortThreads + threadIdx.x;
    if (block_first + i >= n) continue;
    const uint2 p = sh.pairs[i];
    pairs_out[sh.base[(p.x >> shift) & (bins - 1)] + i] = p;
  }
}

// ------------------------------------------------------- gradient: the sums --
template <typename T, int N>
__device__ __forceinline__ void store_grad_row(T* p, const float (&acc)[N], float scale,
                                               int accumulate) {
  float x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = acc[k] * scale;
  if (accumulate) {
    float before[N];
    unpack<T, N>(*reinterpret_cast<const Vec<T, N>*>(p), before);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] += before[k];
  }
  store_vec<T, N>(p, pack<T, N>(x));
}

// The sorted list, a run of equal keys per vertex.  A run of up to kWindow rows is summed by
// one group of lanes.  Of a longer one every window of the list (positions that are a multiple
// of kWindow and those behind) is summed by a warp of its own, and join_kernel adds the windows
// up in order.  64: a group walks 80 rows at most; with 256 the longest of them held its CTA
// for 40 us (1M skewed ids: 221 us for the sums), with 32 the joining took longer (43 us
// against 28).  A CTA whose windows lie whole in one run leaves one sum for all of them.
constexpr int kWindow = 64;
struct Runs {
  const uint2* pairs;        // (key, position)
  int64_t n;
  uint32_t none;             // the key of rows that go nowhere
};
constexpr int kSumThreads = 256;
constexpr int kSumWarps = kSumThreads / 32;
constexpr int kSumAhead = 4;   // rows in flight per lane; with 8, fewer CTAs fit (182 us against 159)
constexpr int kSumPiece = 16;  // positions whose runs (those that begin there) a group sums
constexpr int kSumLeastLanes = 4;  // of a group, also where a row has less to load

// What part of long runs a window holds: its first `head` rows belong to one that began in an
// earlier window or on its first row; the rows from `tail` on to one that begins later in it.
struct WindowParts {
  int head, tail, count;
  bool head_begins;
};
// All lanes of a warp, two positions each.
__device__ __forceinline__ WindowParts find_parts(const Runs& r, int64_t window_index) {
  static_assert(kWindow == 64, "two positions a lane");
  const int lane = threadIdx.x & 31;
  const int64_t begin = window_index * kWindow;
  WindowParts p;
  p.count = (int)(r.n - begin < kWindow ? r.n - begin : kWindow);
  uint32_t key[2], before[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 32 + lane;
    key[h] = i < p.count ? r.pairs[begin + i].x : r.none;
    before[h] = begin - 1 - i >= 0 ? r.pairs[begin - 1 - i].x : r.none;
  }
  const uint32_t first = __shfl_sync(0xffffffffu, key[0], 0);
  const uint32_t last0 = __shfl_sync(0xffffffffu, key[0], (p.count - 1) & 31);
  const uint32_t last1 = __shfl_sync(0xffffffffu, key[1], (p.count - 1) & 31);
  const uint32_t last = p.count > 32 ? last1 : last0;
  int back = 0, same_last = 0;
  p.head = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // equal keys stand together
    const int i = h * 32 + lane;
    p.head += __popc(__ballot_sync(0xffffffffu, i < p.count && key[h] == first));
    same_last += __popc(__ballot_sync(0xffffffffu, i < p.count && key[h] == last));
    back += __popc(__ballot_sync(0xffffffffu, begin - 1 - i >= 0 && before[h] == first));
  }
  p.tail = p.count - same_last;
  // a run is long if the row kWindow behind its first is of the same vertex
  auto is_long = [&](int64_t s, uint32_t key) {
    return key != r.none && s + kWindow < r.n && r.pairs[s + kWindow].x == key;
  };
  p.head_begins = back == 0;
  if (back == kWindow ? first == r.none : !is_long(begin - back, first)) p.head = 0;
  if (p.tail == 0 || !is_long(begin + p.tail, last)) p.tail = p.count;
  return p;
}

// Whether the kSumWarps windows from `w` on lie whole in one run (which is long then).
__device__ __forceinline__ bool whole_block(const Runs& r, int64_t w) {
  const int64_t begin = w * kWindow, end = begin + kSumWarps * kWindow;
  return end <= r.n && r.pairs[begin].x != r.none && r.pairs[begin].x == r.pairs[end - 1].x;
}
__device__ __forceinline__ int ceil_log2_device(int v) { return v <= 1 ? 0 : 32 - __clz(v - 1); }

// The sum of `count` rows from position `from` on, all lanes of a warp, into to[feat_len].
template <typename T, int N>
__device__ __forceinline__ void sum_part(const Runs& r, int64_t from, int count, const T* out_grad,
                                         int64_t out_grad_ld, int feat_len, int log_lanes, float* to) {
  const int lanes = 1 << log_lanes, groups = 32 >> log_lanes;
  const int lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) >> log_lanes;
  for (int c0 = 0; c0 < feat_len; c0 += lanes * N) {
    const int c = c0 + lane * N;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    for (int i0 = group; i0 < count; i0 += groups * kSumAhead) {
      Vec<T, N> row[kSumAhead];
#pragma unroll
      for (int u = 0; u < kSumAhead; ++u) {
        const int i = i0 + u * groups;
        if (i < count && c < feat_len)
          row[u] = load_vec_stream<T, N>(out_grad + (int64_t)r.pairs[from + i].y * out_grad_ld + c);
      }
#pragma unroll
      for (int u = 0; u < kSumAhead; ++u)
        if (i0 + u * groups < count && c < feat_len) {
          float x[N];
          unpack<T, N>(row[u], x);
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += x[k];
        }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < N; ++k)
      for (int d = lanes; d < 32; d <<= 1) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], d);
    if (group == 0 && c < feat_len) {
#pragma unroll
      for (int k = 0; k < N; ++k) to[c + k] = acc[k];
    }
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kSumThreads, 5)
sum_kernel(Runs r, int n_windows, int window_blocks, const T* __restrict__ out_grad,
           int64_t out_grad_ld, int feat_len, float scale, int accumulate, T* __restrict__ grad,
           float* __restrict__ partial, int pitch, int log_lanes) {
  begin_chained();
  if ((int)blockIdx.x < window_blocks) {
    if (blockIdx.y > 0) return;
    const int64_t w = (int64_t)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
    const int64_t begin = w * kWindow;
    const int64_t block_w = (int64_t)blockIdx.x * kSumWarps;
    if (whole_block(r, block_w)) {
      // one long run throughout: the warps' sums, added up in order, at the first window
      __shared__ float whole[kSumWarps][128];
      for (int c0 = 0; c0 < feat_len; c0 += 128) {
        const int span = min(128, feat_len - c0);
        const int span_lanes = min(log_lanes, ceil_log2_device((span + N - 1) / N));
        sum_part<T, N>(r, begin, kWindow, out_grad + c0, out_grad_ld, span, span_lanes,
                       whole[threadIdx.x >> 5]);
        __syncthreads();
        for (int c = threadIdx.x; c < span; c += kSumThreads) {
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < kSumWarps; ++k) s += whole[k][c];
          partial[(block_w * 2 + 0) * pitch + c0 + c] = s;
        }
        __syncthreads();
      }
      return;
    }
    if (w >= n_windows) return;
    const WindowParts p = find_parts(r, w);
    if (p.head > 0)
      sum_part<T, N>(r, begin, p.head, out_grad, out_grad_ld, feat_len, log_lanes,
                     partial + (w * 2 + 0) * pitch);
    if (p.tail < p.count)
      sum_part<T, N>(r, begin + p.tail, p.count - p.tail, out_grad, out_grad_ld, feat_len, log_lanes,
                     partial + (w * 2 + 1) * pitch);
    return;
  }
  // A group of lanes per piece of kSumPiece positions.  The CTA's stretch of the list, the row
  // in front of it and all that its groups may look at behind it come into shared memory in one
  // round trip, so that a group's only waits are for its rows.
  constexpr int kBehind = kSumPiece + 2 * kWindow;
  __shared__ uint2 list[1 + (kSumThreads / kSumLeastLanes) * kSumPiece + kBehind];
  const int lanes = 1 << log_lanes, groups = kSumThreads >> log_lanes;
  const int64_t block_first = (int64_t)(blockIdx.x - window_blocks) * groups * kSumPiece;
  for (int i = threadIdx.x; i < 1 + groups * kSumPiece + kBehind; i += kSumThreads) {
    const int64_t at = block_first - 1 + i;
    list[i] = at >= 0 && at < r.n ? r.pairs[at] : make_uint2(r.none, 0);
  }
  __syncthreads();
  const int c = ((int)blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * N;
  const int begin = 1 + (threadIdx.x >> log_lanes) * kSumPiece, end = begin + kSumPiece;
  if (c >= feat_len) return;
  uint32_t current = list[begin - 1].x;
  bool mine = false;                   // whether the current run is this group's to sum
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  // behind the piece's end only the run that is under way goes on, by kWindow rows at most
  for (int j = begin; j < end || (mine && list[j].x == current); j += kSumAhead) {
    // which of these rows count: those of runs that begin in the piece and are not long
    uint32_t take = 0, starts = 0;
    uint32_t at = current;
    bool is_mine = mine;
    Vec<T, N> row[kSumAhead];
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      const uint2 p = list[j + u];
      if (p.x != at) {
        at = p.x;
        starts |= 1u << u;
        is_mine = j + u < end && at != r.none && list[j + u + kWindow].x != at;
      }
      if (is_mine) {
        take |= 1u << u;
        row[u] = load_vec_stream<T, N>(out_grad + (int64_t)p.y * out_grad_ld + c);
      }
    }
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      if (starts >> u & 1) {
        if (mine) store_grad_row<T, N>(grad + (int64_t)current * feat_len + c, acc, scale, accumulate);
        current = list[j + u].x;
        mine = take >> u & 1;
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = 0.f;
      }
      if (take >> u & 1) {
        float x[N];
        unpack<T, N>(row[u], x);
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += x[k];
      }
    }
  }
  if (mine) store_grad_row<T, N>(grad + (int64_t)current * feat_len + c, acc, scale, accumulate);
}

// A warp per window; works only where a long run begins in it.  The run's parts are this
// window's and the heads of the windows behind.  A run of up to kJoinAlone parts is added up
// by that warp, a longer one by all warps of the CTA: cut into as many stretches, each summed
// in order, and these added in order.
constexpr int kJoinAlone = 32;

// The parts of a long run: `count` windows from `first` on, of which those in whole blocks
// have one sum between them.  Part t is that of window first + t up to the first block that is
// whole, then of a block each, then of the windows behind the last.
struct RunParts {
  int64_t first, whole0, whole1, last;  // windows; blocks [whole0, whole1) are whole
  int slot;
  __device__ __forceinline__ int64_t count() const {
    return whole1 > whole0 ? (whole0 - first) + (whole1 - whole0) / kSumWarps + (last + 1 - whole1)
                           : last + 1 - first;
  }
  __device__ __forceinline__ int64_t window(int64_t t) const {
    if (whole1 <= whole0 || t < whole0 - first) return first + t;
    t -= whole0 - first;
    const int64_t blocks = (whole1 - whole0) / kSumWarps;
    return t < blocks ? whole0 + t * kSumWarps : whole1 + (t - blocks);
  }
};
__device__ __forceinline__ RunParts run_parts(const Runs& r, int64_t first, int64_t windows, int slot) {
  RunParts p;
  p.first = first;
  p.slot = slot;
  p.last = first + windows - 1;
  // whole blocks begin on a multiple of kSumWarps windows; the run's own first window counts
  // only if the run begins on its first row, and the last block only if it is full of the run
  p.whole0 = (first + kSumWarps - 1) / kSumWarps * kSumWarps;
  if (p.whole0 == first && slot == 1) p.whole0 += kSumWarps;
  p.whole1 = (p.last + 1) / kSumWarps * kSumWarps;
  if (p.whole1 > p.whole0 && !whole_block(r, p.whole1 - kSumWarps)) p.whole1 -= kSumWarps;
  return p;
}

// The sum of parts t0 <= t < t1, for four columns from c on.
__device__ __forceinline__ float4 join_terms(const float* partial, const RunParts& p, int64_t t0,
                                             int64_t t1, int pitch, int c) {
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int64_t t = t0; t < t1; ++t) {
    const float4 v = *reinterpret_cast<const float4*>(
        partial + (p.window(t) * 2 + (t == 0 ? p.slot : 0)) * pitch + c);
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  return s;
}
template <typename T>
__device__ __forceinline__ void store_joined(T* row, int feat_len, int c, float4 s, float scale,
                                             int accumulate) {
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float one[1] = {v[k]};
    if (c + k < feat_len) store_grad_row<T, 1>(row + c + k, one, scale, accumulate);
  }
}

template <typename T>
__global__ void __launch_bounds__(kSumThreads)
join_kernel(Runs r, int n_windows, int feat_len, float scale, int accumulate, T* __restrict__ grad,
            const float* __restrict__ partial, int pitch) {
  begin_chained();
  __shared__ RunParts runs[kSumWarps];     // those that the whole CTA adds up; slot -1: none
  __shared__ float4 sums[kSumWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kSumWarps + warp;
  const int64_t behind = (w + 1) * kWindow;   // a long run goes on in the next window
  int slot = -1;
  uint32_t key = r.none;
  if (w < n_windows && behind < r.n) {
    key = r.pairs[behind - 1].x;
    if (key != r.none && r.pairs[behind].x == key) {
      const WindowParts p = find_parts(r, w);
      if (p.tail < p.count) slot = 1;
      else if (p.head > 0 && p.head_begins) slot = 0;
    }
  }
  RunParts parts;
  parts.slot = -1;
  if (slot >= 0) {  // how many windows behind this one begin with the same vertex
    int64_t windows = 1;
    for (bool more = true; more;) {
      uint32_t same[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t at = (w + windows + k * 32 + lane) * kWindow;
        same[k] = __ballot_sync(0xffffffffu, at < r.n && r.pairs[at < r.n ? at : 0].x == key);
      }
      const int count = __popc(same[0]) + __popc(same[1]) + __popc(same[2]) + __popc(same[3]);
      windows += count;
      more = count == 128;
    }
    parts = run_parts(r, w, windows, slot);
    const int64_t terms = parts.count();
    if (terms <= kJoinAlone) {
      for (int c = lane * 4; c < feat_len; c += 128)
        store_joined<T>(grad + (int64_t)key * feat_len, feat_len, c,
                        join_terms(partial, parts, 0, terms, pitch, c), scale, accumulate);
      parts.slot = -1;
    }
  }
  if (lane == 0) runs[warp] = parts;
  __syncthreads();
  for (int q = 0; q < kSumWarps; ++q) {
    const RunParts run = runs[q];
    if (run.slot < 0) continue;
    const int64_t n = run.count(), per = (n + kSumWarps - 1) / kSumWarps;
    const int64_t t0 = min(n, warp * per), t1 = min(n, (warp + 1) * per);
    const uint32_t vertex = r.pairs[(run.first + 1) * kWindow].x;
    for (int c0 = 0; c0 < feat_len; c0 += 128) {
      const int c = c0 + lane * 4;
      if (c < feat_len) sums[warp][lane] = join_terms(partial, run, t0, t1, pitch, c);
      __syncthreads();
      if (warp == 0 && c < feat_len) {
        float4 s = sums[0][lane];
#pragma unroll
        for (int k = 1; k < kSumWarps; ++k) {
          const float4 v = sums[k][lane];
          s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        store_joined<T>(grad + (int64_t)vertex * feat_len, feat_len, c, s, scale, accumulate);
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------ gradient: few ids --
// Up to kFewIds ids the whole gradient is one launch.  The vertices are dealt out to kSlices
// CTAs (times the slabs of columns): each looks through all ids for its own, keeps them in
// order, ranks the few it has by (vertex, position), and sums.  A slice has one vertex of
// every kSlices neighbours, at a place that changes from one such stretch to the next, so that neither
// neighbouring nor evenly spaced popular vertices meet in one.  5003 skewed ids of 400-byte rows:
// 17 us; the sort, sums and join in launches of their own took 29.
constexpr int64_t kFewIds = 8192;
constexpr int kSliceBits = 7;
constexpr int kSlices = 1 << kSliceBits;
constexpr int kSliceThreads = 512;
constexpr int kSliceAhead = 8;
constexpr int kSliceWarps = kSliceThreads / 32;
constexpr int kSliceChunks = (int)(kFewIds / kSliceThreads);
constexpr int kSliceParts = 8;
constexpr int kSliceAlone = 32;   // rows that one group of lanes sums alone
constexpr int kSliceRank = 64;   // rows that are ranked by comparing each with each

__device__ __forceinline__ uint32_t slice_shift(uint32_t high) {
  return (high ^ high >> kSliceBits ^ high >> 2 * kSliceBits) & (kSlices - 1);
}
__device__ __forceinline__ uint32_t slice_of(uint32_t v) {
  return (v & (kSlices - 1)) ^ slice_shift(v >> kSliceBits);
}

inline size_t slice_shared_bytes(int64_t n) { return (size_t)((n + 31) / 32 * 32) * 12; }

template <typename T, int N, typename I>
__global__ void __launch_bounds__(kSliceThreads)
slice_kernel(KeySource src, int n, const T* __restrict__ out_grad, int64_t out_grad_ld, int feat_len,
             float scale, int accumulate, T* __restrict__ grad, int log_lanes) {
  extern __shared__ __align__(16) uint8_t raw[];
  const int room = (n + 31) / 32 * 32;
  uint32_t* mine = reinterpret_cast<uint32_t*>(raw);            // this slice's keys, in order
  uint32_t* sorted_keys = mine + room;                          // the same, vertex by vertex
  uint16_t* found = reinterpret_cast<uint16_t*>(sorted_keys + room);  // their positions
  uint16_t* sorted = found + room;                              // the same, vertex by vertex
  __shared__ uint16_t before[kSliceChunks * kSliceWarps];
  __shared__ int warp_count[kSliceWarps];
  __shared__ int n_long, long_run[kFewIds / kSliceAlone];
  __shared__ float sums[kSliceThreads * N], part_sums[kSliceParts * 32 * N];
  const int warp = threadIdx.x >> 5, lane32 = threadIdx.x & 31;
  const int lanes = 1 << log_lanes, groups = kSliceThreads >> log_lanes;
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> log_lanes;
  const int c = ((int)blockIdx.y * lanes + lane) * N;
  const bool in = c < feat_len;

  // Looks through the ids, kSliceThreads at a time, and notes which are this slice's: key[k] is
  // the thread's id of stretch k, hits[k] which lanes of its warp have one of the slice's.  Every
  // CTA begins with another stretch, so that they do not all ask for the same lines.
  const int stretches = (n + kSliceThreads - 1) / kSliceThreads;   // kSliceChunks at most
  const int rotate = (blockIdx.x + blockIdx.y) % stretches;
  uint32_t key[kSliceChunks], hits[kSliceChunks];
  {
    I id[kSliceChunks];
#pragma unroll
    for (int k = 0; k < kSliceChunks; ++k) {
      const int stretch = k + rotate < stretches ? k + rotate : k + rotate - stretches;
      const int i = stretch * kSliceThreads + threadIdx.x;
      id[k] = k < stretches && i < n ? load_source<I>(src, i) : I();
    }
#pragma unroll
    for (int k = 0; k < kSliceChunks; ++k) {
      hits[k] = 0;
      if (k >= stretches) continue;
      const int stretch = k + rotate < stretches ? k + rotate : k + rotate - stretches;
      const int i = stretch * kSliceThreads + threadIdx.x;
      key[k] = i < n ? make_pair<I>(src, id[k], 0).x : (uint32_t)src.n_vertices;
      hits[k] = __ballot_sync(0xffffffffu, key[k] < (uint32_t)src.n_vertices && slice_of(key[k]) == blockIdx.x);
      if (lane32 == 0) before[stretch * kSliceWarps + warp] = (uint16_t)__popc(hits[k]);
    }
  }
  // zeros first; the sums overwrite them behind the barriers below
  if (!accumulate && in) {
    float zeros[N];
#pragma unroll
    for (int k = 0; k < N; ++k) zeros[k] = 0.f;
    const Vec<T, N> zero = pack<T, N>(zeros);
    for (int64_t high = group; high * kSlices < src.n_vertices; high += groups) {
      const int64_t v = high * kSlices + (blockIdx.x ^ slice_shift((uint32_t)high));
      if (v < src.n_vertices) store_vec<T, N>(grad + v * feat_len + c, zero);
    }
  }
  if (threadIdx.x == 0) n_long = 0;
  __syncthreads();
  // counts of the warps' stretches, in the order of positions, become those in front of them
  int m;
  {
    const int total = stretches * kSliceWarps;   // at most kSliceChunks * kSliceWarps
    static_assert(kSliceChunks * kSliceWarps <= kSliceThreads, "a thread each");
    const int count = (int)threadIdx.x < total ? before[threadIdx.x] : 0;
    int incl = count;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane32 >= d) incl += up;
    }
    if (lane32 == 31) warp_count[warp] = incl;
    __syncthreads();
    m = 0;
    int ahead = 0;
#pragma unroll
    for (int w = 0; w < kSliceWarps; ++w) {
      if (w < warp) ahead += warp_count[w];
      m += warp_count[w];
    }
    if ((int)threadIdx.x < total) before[threadIdx.x] = (uint16_t)(ahead + incl - count);
    __syncthreads();
  }
  if (m == 0) return;
#pragma unroll
  for (int k = 0; k < kSliceChunks; ++k) {
    if (!(hits[k] >> lane32 & 1)) continue;
    const int stretch = k + rotate < stretches ? k + rotate : k + rotate - stretches;
    const int e = before[stretch * kSliceWarps + warp] + __popc(hits[k] & ((1u << lane32) - 1));
    found[e] = (uint16_t)(stretch * kSliceThreads + threadIdx.x);
    mine[e] = key[k];
  }
  __syncthreads();
  // While there are many: the rows of one vertex of theirs after the other are taken out, in
  // order.  The vertex in the middle of the list is most likely the one that has most rows.
  int left = m, out = 0;
  __shared__ int warp_taken[kSliceThreads / 32];
  for (int round = 0; left > kSliceRank && round < 64; ++round) {
    const uint32_t pivot = mine[left / 2];
    __syncthreads();
    int kept = 0;
    for (int e0 = 0; e0 < left; e0 += kSliceThreads) {
      const int e = e0 + threadIdx.x;
      const uint32_t key = e < left ? mine[e] : 0;
      const uint16_t position = e < left ? found[e] : 0;
      const uint32_t take = __ballot_sync(0xffffffffu, e < left && key == pivot);
      const uint32_t keep = __ballot_sync(0xffffffffu, e < left && key != pivot);
      if (lane32 == 0) {
        warp_taken[warp] = __popc(take);
        warp_count[warp] = __popc(keep);
      }
      __syncthreads();
      int to_taken = out, to_kept = kept;
#pragma unroll
      for (int w = 0; w < kSliceThreads / 32; ++w) {
        if (w < warp) {
          to_taken += warp_taken[w];
          to_kept += warp_count[w];
        }
        out += warp_taken[w];
        kept += warp_count[w];
      }
      const uint32_t below = (1u << lane32) - 1;
      if (take >> lane32 & 1) {
        sorted[to_taken + __popc(take & below)] = position;
        sorted_keys[to_taken + __popc(take & below)] = key;
      }
      if (keep >> lane32 & 1) {
        mine[to_kept + __popc(keep & below)] = key;
        found[to_kept + __popc(keep & below)] = position;
      }
      __syncthreads();
    }
    left = kept;
  }
  // the others by counting what stands before them
  for (int e = threadIdx.x; e < left; e += kSliceThreads) {
    const uint32_t key = mine[e];
    int rank = 0;
    for (int f = 0; f < left; ++f) rank += mine[f] < key + (f < e);
    sorted[out + rank] = found[e];
    sorted_keys[out + rank] = key;
  }
  __syncthreads();
  // a run per vertex; where they start, in order
  uint16_t* starts = found;
  int n_runs = 0;
  for (int e0 = 0; e0 < m; e0 += kSliceThreads) {
    const int e = e0 + threadIdx.x;
    const bool start = e < m && (e == 0 || sorted_keys[e - 1] != sorted_keys[e]);
    const uint32_t all = __ballot_sync(0xffffffffu, start);
    if (lane32 == 0) warp_count[warp] = __popc(all);
    __syncthreads();
    int to_start = n_runs;
#pragma unroll
    for (int w = 0; w < kSliceThreads / 32; ++w) {
      if (w < warp) to_start += warp_count[w];
      n_runs += warp_count[w];
    }
    if (start) starts[to_start + __popc(all & ((1u << lane32) - 1))] = (uint16_t)e;
    __syncthreads();
  }
  // short runs to a group of lanes each
  auto row_of = [&](int e) { return out_grad + (int64_t)sorted[e] * out_grad_ld + c; };
  for (int q = group; q < n_runs; q += groups) {
    const int e = starts[q], end = q + 1 < n_runs ? starts[q + 1] : m;
    const uint32_t key = sorted_keys[e];
    if (end - e > kSliceAlone) {
      if (lane == 0) long_run[atomicAdd(&n_long, 1)] = q;
      continue;
    }
    if (!in) continue;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    for (int j = e; j < end; j += kSliceAhead) {
      Vec<T, N> row[kSliceAhead];
#pragma unroll
      for (int u = 0; u < kSliceAhead; ++u)
        if (j + u < end) row[u] = load_vec_stream<T, N>(row_of(j + u));
#pragma unroll
      for (int u = 0; u < kSliceAhead; ++u)
        if (j + u < end) {
          float x[N];
          unpack<T, N>(row[u], x);
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += x[k];
        }
    }
    store_grad_row<T, N>(grad + (int64_t)key * feat_len + c, acc, scale, accumulate);
  }
  __syncthreads();
  // long ones to all groups, a stretch each, and their sums added up in order
  for (int q = 0; q < n_long; ++q) {
    const int run = long_run[q], e = starts[run], lo = run + 1 < n_runs ? starts[run + 1] : m;
    const uint32_t key = sorted_keys[e];
    const int stretch = (lo - e + groups - 1) / groups;
    const int j0 = min(lo, e + group * stretch), j1 = min(lo, j0 + stretch);
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    if (in)
      for (int j = j0; j < j1; j += kSliceAhead) {
        Vec<T, N> row[kSliceAhead];
#pragma unroll
        for (int u = 0; u < kSliceAhead; ++u)
          if (j + u < j1) row[u] = load_vec_stream<T, N>(row_of(j + u));
#pragma unroll
        for (int u = 0; u < kSliceAhead; ++u)
          if (j + u < j1) {
            float x[N];
            unpack<T, N>(row[u], x);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += x[k];
          }
      }
#pragma unroll
    for (int k = 0; k < N; ++k) sums[threadIdx.x * N + k] = acc[k];
    __syncthreads();
    // kSliceParts threads a column, each kSliceParts-th group; then one of them
    const int width = lanes * N;
    for (int i = threadIdx.x; i < width * kSliceParts; i += kSliceThreads) {
      float total = 0.f;
      for (int g = i / width; g < groups; g += kSliceParts) total += sums[g * width + i % width];
      part_sums[i] = total;
    }
    __syncthreads();
    if (group == 0 && in) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        acc[k] = part_sums[lane * N + k];
#pragma unroll
        for (int g = 1; g < kSliceParts; ++g) acc[k] += part_sums[g * width + lane * N + k];
      }
      store_grad_row<T, N>(grad + (int64_t)key * feat_len + c, acc, scale, accumulate);
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
  bool few;                  // one launch of slice_kernel
  int64_t windows, blocks;
  int passes, digit_bits;
  int pitch;                 // of a partial sum, in floats
  size_t pairs[2], counts, totals, partial, total;
};

GradLayout grad_layout(int64_t n, int64_t n_vertices, int64_t feat_len) {
  GradLayout l = {};
  l.few = n <= kFewIds;
  if (l.few) {
    l.total = 256;           // the kernel needs none; a caller always brings some
    return l;
  }
  l.windows = (n + kWindow - 1) / kWindow;
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
  l.pairs[0] = take((size_t)n * 8);
  l.pairs[1] = take((size_t)n * 8);
  l.counts = take(((size_t)l.blocks << l.digit_bits) * 4);
  l.totals = take(kMaxBins * 4);
  l.pitch = (int)((feat_len + 3) / 4 * 4);
  l.partial = take((size_t)l.windows * 2 * l.pitch * 4);
  l.total = at;
  return l;
}

int check_common(const void* values, const void* ids, const int32_t* status, int32_t dtype,
                 int32_t index_type, int64_t n_vertices, int64_t n_ids, int64_t feat_len, float scale) {
  if (!std::isfinite(scale))
    return fail(FG_ERR_INVALID_ARGUMENT, "scale=%g is not finite", (double)scale);
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
  if (((uintptr_t)ids & (index_type == FG_INDEX_INT64 ? 7 : 3)) != 0 || ((uintptr_t)status & 3) != 0)
    return fail(FG_ERR_INVALID_ARGUMENT, "ids or status are not aligned to their type");
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
                            feat_len, scale))
    return rc;
  if (table_ld < feat_len || out_ld < feat_len)
    return fail(FG_ERR_INVALID_ARGUMENT, "a row pitch is shorter than feat_len=%lld",
                (long long)feat_len);
  if (n_ids == 0) return FG_OK;
  if (n_vertices > 0 && !table_dev) return fail(FG_ERR_INVALID_ARGUMENT, "null table");
  const Array2d out_array = {out_dev, n_ids, feat_len, out_ld, dtype_size(dtype)};
  if (overlap(out_array, {table_dev, n_vertices, feat_len, table_ld, dtype_size(dtype)}) ||
      overlap(out_array, array1d(ids_dev, n_ids, index_type == FG_INDEX_INT64 ? 8 : 4)))
    return fail(FG_ERR_INVALID_ARGUMENT, "out shares memory with an input");
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
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(want, 1), 148 * 2 * kLookupBlocks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FG_LOOKUP(T, N)                                                                         \
  {                                                                                             \
    const T* table = static_cast<const T*>(table_dev);                                          \
    T* out = static_cast<T*>(out_dev);                                                          \
    if (index_type == FG_INDEX_INT64)                                                           \
      lookup_kernel<T, N, long long><<<grid, kLookupThreads, 0, s>>>(                           \
          table, table_ld, n_vertices, ids_dev, n_ids, (int)feat_len, scale, out, out_ld,       \
          log_lanes, status_dev);                                                               \
    else                                                                                        \
      lookup_kernel<T, N, int><<<grid, kLookupThreads, 0, s>>>(                                 \
          table, table_ld, n_vertices, ids_dev, n_ids, (int)feat_len, scale, out, out_ld,       \
          log_lanes, status_dev);                                                               \
  }
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
                            n_ids, feat_len, scale))
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
  const size_t es = dtype_size(dtype);
  const Array2d grad_array = {grad_dev, n_vertices, feat_len, feat_len, es};
  if (overlap(grad_array, {out_grad_dev, n_ids, feat_len, out_grad_ld, es}) ||
      overlap(grad_array, array1d(ids_dev, n_ids, index_type == FG_INDEX_INT64 ? 8 : 4)))
    return fail(FG_ERR_INVALID_ARGUMENT, "the gradient shares memory with an input");
  const int vb = common_vector_bytes({(uint64_t)(uintptr_t)out_grad_dev,
                                      (uint64_t)(uintptr_t)grad_dev, (uint64_t)(out_grad_ld * es),
                                      (uint64_t)(feat_len * es)});
  if (vb < (int)es) return fail(FG_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its type");
  // the launch shape of the sums; refused before anything is launched.  Few ids: slabs of 256 bytes
  // where the rows allow 16-byte accesses, so that a popular vertex of long rows is the work of
  // several CTAs
  const int per_row = (int)((feat_len * es + vb - 1) / vb);
  const int log_lanes = l.few ? std::min(vb == 16 ? 4 : 5, ceil_log2(per_row))
                              : std::max(ceil_log2(kSumLeastLanes), std::min(5, ceil_log2(per_row)));
  const int64_t slabs = (per_row + (1 << log_lanes) - 1) >> log_lanes;
  const int64_t pieces = (n_ids + kSumPiece - 1) / kSumPiece;
  const int64_t window_blocks = (l.windows + kSumWarps - 1) / kSumWarps;
  const int64_t blocks_x = window_blocks + ((pieces << log_lanes) + kSumThreads - 1) / kSumThreads;
  if (n_ids > 0 && (blocks_x > INT32_MAX || slabs > 65535))
    return fail(FG_ERR_UNSUPPORTED, "n_ids=%lld x feat_len=%lld is too large", (long long)n_ids,
                (long long)feat_len);
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const ZeroFill zero = {static_cast<uint8_t*>(grad_dev),
                         accumulate ? 0 : (int64_t)((size_t)n_vertices * feat_len * es)};
  if (n_ids == 0) {
    if (zero.bytes > 0) FG_CUDA_TRY(cudaMemsetAsync(grad_dev, 0, zero.bytes, s));
    return FG_OK;
  }
  // the zeros in `parts` equal parts (multiples of 64 KB, the last may be shorter)
  auto zero_part = [&](int part, int parts) {
    const int64_t each = (zero.bytes / parts + 65535) / 65536 * 65536;
    const int64_t from = std::min(zero.bytes, part * each);
    return ZeroFill{zero.to + from, std::min(zero.bytes - from, part + 1 == parts ? zero.bytes : each)};
  };
  auto zero_blocks = [](const ZeroFill& z) { return (int)std::min<int64_t>(2 * 148, (z.bytes + 65535) / 65536); };

  char* ws = static_cast<char*>(workspace_dev);
  uint2* pairs[2] = {reinterpret_cast<uint2*>(ws + l.pairs[0]), reinterpret_cast<uint2*>(ws + l.pairs[1])};
  float* partial = reinterpret_cast<float*>(ws + l.partial);
  KeySource src = {ids_dev, n_vertices, padding_id < 0 ? -1 : padding_id, status_dev};
  const bool wide = index_type == FG_INDEX_INT64;
  if (l.few) {
    const size_t smem = slice_shared_bytes(n_ids);
    const dim3 grid(kSlices, (unsigned)slabs);
#define FG_SLICE(T, N)                                                                             \
  {                                                                                                \
    auto kernel = wide ? slice_kernel<T, N, long long> : slice_kernel<T, N, int>;                  \
    FG_CUDA_TRY(allow_shared((const void*)kernel, (int)slice_shared_bytes(kFewIds), device));      \
    kernel<<<grid, kSliceThreads, smem, s>>>(src, (int)n_ids, static_cast<const T*>(out_grad_dev), \
                                             out_grad_ld, (int)feat_len, scale, accumulate,        \
                                             static_cast<T*>(grad_dev), log_lanes);                \
  }
#define FG_SLICE_T(T)                                                       \
  switch (vb / (int)sizeof(T)) {                                            \
    case 8: if constexpr (sizeof(T) == 2) FG_SLICE(T, 8 / (sizeof(T) / 2)); break; \
    case 4: FG_SLICE(T, 4); break;                                          \
    case 2: FG_SLICE(T, 2); break;                                          \
    default: FG_SLICE(T, 1); break;                                         \
  }
    FG_DISPATCH_DTYPE(dtype, FG_SLICE_T)
#undef FG_SLICE_T
#undef FG_SLICE
    FG_CUDA_TRY(cudaGetLastError());
    return FG_OK;
  }
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + l.counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + l.totals);
  const int bins = 1 << l.digit_bits, blocks = (int)l.blocks;
  for (int pass = 0; pass < l.passes; ++pass) {
    const int shift = pass * l.digit_bits;
    const ZeroFill z0 = zero_part(2 * pass, 2 * l.passes), z1 = zero_part(2 * pass + 1, 2 * l.passes);
    auto count = pass > 0 ? sort_count_kernel<uint2> : wide ? sort_count_kernel<long long> : sort_count_kernel<int>;
    auto place = pass > 0 ? sort_place_kernel<uint2> : wide ? sort_place_kernel<long long> : sort_place_kernel<int>;
    FG_CUDA_TRY(allow_shared((const void*)place, (int)sizeof(PlaceShared), device));
    FG_CUDA_TRY(launch(pass > 0, count, blocks + zero_blocks(z0), kSortThreads, 0, s, src, n_ids,
                       shift, l.digit_bits, counts, blocks, z0));
    FG_CUDA_TRY(launch(true, sort_scan_kernel, (bins + kSortWarps - 1) / kSortWarps, kSortThreads, 0, s,
                       counts, blocks, bins, totals));
    FG_CUDA_TRY(launch(true, place, blocks + zero_blocks(z1), kSortThreads, sizeof(PlaceShared),
                       s, src, n_ids, shift, l.digit_bits, counts, totals, pairs[pass & 1], blocks, z1));
    src.from = pairs[pass & 1];
  }
  const Runs runs = {static_cast<const uint2*>(src.from), n_ids, (uint32_t)n_vertices};
  const dim3 grid((unsigned)blocks_x, (unsigned)slabs);
#define FG_SUM(T, N)                                                                             \
  FG_CUDA_TRY(launch(true, sum_kernel<T, N>, grid, kSumThreads, 0, s, runs, (int)l.windows,      \
                     (int)window_blocks, static_cast<const T*>(out_grad_dev), out_grad_ld,       \
                     (int)feat_len, scale, accumulate, static_cast<T*>(grad_dev), partial, l.pitch, \
                     log_lanes))
#define FG_SUM_T(T)                                                       \
  switch (vb / (int)sizeof(T)) {                                          \
    case 8: if constexpr (sizeof(T) == 2) FG_SUM(T, 8 / (sizeof(T) / 2)); break; \
    case 4: FG_SUM(T, 4); break;                                          \
    case 2: FG_SUM(T, 2); break;                                          \
    default: FG_SUM(T, 1); break;                                                                \
  }                                                                                              \
  FG_CUDA_TRY(launch(true, join_kernel<T>, (int)window_blocks, kSumThreads, 0, s, runs,          \
                     (int)l.windows, (int)feat_len, scale, accumulate, static_cast<T*>(grad_dev), \
                     partial, l.pitch));
  FG_DISPATCH_DTYPE(dtype, FG_SUM_T)
#undef FG_SUM_T
#undef FG_SUM
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}
