// Softmax cross entropy over a large vocabulary (every vertex of a graph, every class),
// without keeping the logits, and its gradients.
//
//   z = scale * feat @ weight^T          (n x V, never stored)
//   lse_t  = log sum_v exp z_tv
//   loss_t = lse_t - z_{t, label_t}      (0 where the label is ignore_index)
//   dz     = scale * loss_grad_t * (exp(z - lse) - [v = label_t])    (0 on ignored rows)
//   feat_grad = dz @ weight,  weight_grad = dz^T @ feat
//
// One tensor-core kernel in three modes.  A CTA keeps 128 rows of one operand in shared memory
// and streams the other past them; a tile S of logits goes from tcgen05.mma into TMEM, from
// there through the registers of the epilogue warps, and either ends there as a running
// maximum and sum (the loss) or goes back into TMEM in 16 bits as the left operand of the
// second product, whose accumulators stay in TMEM until the streamed operand has passed:
//   loss         rows = samples,  streamed = vocabulary:  m, s of every row
//   feat_grad    rows = samples,  streamed = vocabulary:  P W
//   weight_grad  rows = vocabulary, streamed = samples:   P^T H
// so the logits are computed three times and never leave the SM.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elem.cuh"
#include "tensor.cuh"

namespace fg {
namespace {

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
// The row's label, -1 if it takes no part.
__device__ __forceinline__ int32_t live_label(const Batch& b, int64_t t) {
  if (t >= b.n) return -1;
  const int64_t y = load_label(b.labels, b.wide, t);
  return y != b.ignore_index && (uint64_t)y < (uint64_t)b.vocab ? (int32_t)y : -1;
}

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) {  // results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------- the tensor-core kernel --
enum Mode { kLoss = 0, kFeatGrad = 1, kWeightGrad = 2 };

constexpr int kTileRows = 128;
constexpr int kTileBytes = kTileRows * 128;   // 128 rows of 64 16-bit elements
constexpr int kMmaThreads = 384;              // loads, mma, TMEM, one idle; then 8 epilogue warps
constexpr int kEpilogueWarp = 4;
constexpr int kMaxStages = 8;
constexpr int kMaxResidentTiles = 4;          // 64-element tiles of a row that stay in shared memory
constexpr int kSharedBudget = 12 * kTileBytes;

struct MmaArgs {
  int64_t n_rows, n_cols;
  int kb;                 // 64-element tiles of a row (of one piece of it, for float32)
  int row_tiles, splits, steps, steps_per_split, stages;
  int feat_len, out_cols; // out_cols: feat_len rounded up to 16
  int negate;             // a negative scale: |scale| with -A
  float logit_scale;      // |scale| * log2(e)
  const float* unscale;   // float32: what undoes the operands' scaling; else null
  float2* stats;          // loss: (maximum, sum) per row, split and epilogue group, base 2
  const float* row_bias;  // feat_grad: log2(hot) - lse * log2(e) of a row, -inf: takes no part
  const int32_t* row_label;
  const float* col_bias;  // weight_grad: the same of a column, plus log2 |weight|
  const float* col_weight;
  const int32_t* col_label;
  float hot;              // what a probability of 1 is held as
  const float* row_factor;  // feat_grad: factor of a row of the results
  const float* out_scale; // factor of all of them, on the device; null: 1
  void* out;              // one split: the results
  float* partial;         // several: a partial sum each, for join_partial_kernel
  int32_t* status;
};

template <int MODE, typename T>
struct MmaShape {
  static constexpr bool kSplit = sizeof(T) == 4;  // float32 as two fp16 pieces, three products
  static constexpr int kCols = MODE == kLoss ? 256 : 128;
  static constexpr int kOutAt = 256;              // TMEM columns: S, S, then the accumulators
  static constexpr int kLowAt = 384;              // and float32's low pieces of P
};

// Two probabilities in 16 bits each, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 unpack_half2(uint32_t r) {
  __half2 h;
  memcpy(&h, &r, 4);
  return __half22float2(h);
}

// P in 16 bits to TMEM: 32 columns of S become 16.  Rounding it to the operands' type (half a
// step, 2^-9 for bfloat16 and 2^-12 for float16) is what the second product's rate costs;
// float32 keeps a second piece, together 2^-22.
template <int MODE, typename T>
__device__ __forceinline__ void store_p(uint32_t s_at, uint32_t low_at, int chunk, const float (&p)[32]) {
  uint32_t r[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) r[k] = pack2<T>(p[2 * k], p[2 * k + 1]);
  tc::tmem_store16(s_at + chunk * 16, r);
  if (MmaShape<MODE, T>::kSplit) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 hi = unpack_half2(r[k]);
      r[k] = pack2<T>(p[2 * k] - hi.x, p[2 * k + 1] - hi.y);
    }
    tc::tmem_store16(low_at + chunk * 16, r);
  }
}

// One verdict for the whole warp: it either goes on together or gives up together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, tc::bar_wait(bar, parity));
}

template <int MODE, typename T>
__global__ void __launch_bounds__(kMmaThreads, 1)
xent_mma_kernel(const __grid_constant__ CUtensorMap row_map,
                const __grid_constant__ CUtensorMap col_map, const __grid_constant__ MmaArgs a) {
  using Shape = MmaShape<MODE, T>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t bars[2 * kMaxStages + 9];
  __shared__ uint32_t tmem_where;
  __shared__ __align__(16) float col_bias_s[MODE == kWeightGrad ? 8 : 1][128];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_u32(raw_smem) + 1023) & ~1023u;
  const int planes = Shape::kSplit ? 2 : 1;
  const int tiles = a.kb * planes;                       // tiles of a resident row
  const int stage_tiles = MODE == kLoss ? 1 : tiles;     // tiles of a stage
  const uint32_t stage_bytes = (uint32_t)stage_tiles * (Shape::kCols / 128) * kTileBytes;
  const uint32_t rows_at = smem, ring_at = smem + tiles * kTileBytes;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxStages;
  const uint32_t rows_full = empty + 8 * kMaxStages, rows_empty = rows_full + 8;
  const uint32_t s_full = rows_full + 16, s_done = rows_full + 32;   // two each
  const uint32_t out_full = rows_full + 48, out_empty = rows_full + 56, drained = rows_full + 64;

  if (threadIdx.x == 0) {
    for (int k = 0; k < a.stages; ++k) {
      tc::bar_init(full + 8 * k, 1);
      tc::bar_init(empty + 8 * k, 1);
    }
    tc::bar_init(rows_full, 1);
    tc::bar_init(rows_empty, 1);
    for (int k = 0; k < 2; ++k) {
      tc::bar_init(s_full + 8 * k, 1);
      tc::bar_init(s_done + 8 * k, 128);
    }
    tc::bar_init(out_full, 1);
    tc::bar_init(out_empty, 256);
    tc::bar_init(drained, 1);
    tc::bar_init_fence();
    tc::prefetch_map(&row_map);
    tc::prefetch_map(&col_map);
  }
  if (warp == 2) tc::tmem_alloc(smem_u32(&tmem_where), 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_where;
  const int items = a.row_tiles * a.splits;
  // item = (split, row tile), row tiles first: CTAs beside each other stream the same part
  auto steps_of = [&](int item, int& first) {
    first = item / a.row_tiles * a.steps_per_split;
    return min(a.steps_per_split, a.steps - first);
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, it = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < items; item += gridDim.x, ++it) {
        int first;
        const int n = steps_of(item, first);
        if (it > 0 && !(ok = tc::bar_wait(rows_empty, (it - 1) & 1))) break;
        tc::bar_expect(rows_full, tiles * kTileBytes);
        for (int q = 0; q < tiles; ++q)
          tc::load_tile(rows_at + q * kTileBytes, &row_map, q * 64, item % a.row_tiles * kTileRows,
                        rows_full);
        for (int j = 0; ok && j < n; ++j) {
          for (int q = 0; q < tiles; q += stage_tiles, ++stage) {
            const uint32_t slot = stage % a.stages, round = stage / a.stages;
            if (round > 0 && !(ok = tc::bar_wait(empty + 8 * slot, (round - 1) & 1))) break;
            tc::bar_expect(full + 8 * slot, stage_bytes);
            for (int k = 0; k < stage_tiles; ++k)
              tc::load_tile(ring_at + slot * stage_bytes + k * kTileBytes, &col_map, (q + k) * 64,
                            (first + j) * Shape::kCols, full + 8 * slot);
          }
        }
      }
      if (!ok) {  // give up only once nothing is in flight into this CTA's shared memory
        *a.status = FG_STATUS_WAIT_EXPIRED;
        tc::bar_wait(rows_full, it & 1);
        for (uint32_t k = stage > (uint32_t)a.stages ? stage - a.stages : 0; k < stage; ++k)
          tc::bar_wait(full + 8 * (k % a.stages), (k / a.stages) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t s_desc = tc::mma_desc(kBf16, Shape::kCols, a.negate != 0, false);
      const uint32_t o_desc = tc::mma_desc(kBf16, a.out_cols, false, true);
      uint32_t stage = 0, step = 0, it = 0;
      bool ok = true;
      // one product of 64 k: a tile of the rows with a tile of the stage
      auto product = [&](uint32_t d, int row_tile, uint32_t col_tile_at, bool add) {
        const uint64_t da = tc::tile_desc(rows_at + row_tile * kTileBytes, 16);
        const uint64_t db = tc::tile_desc(col_tile_at, 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::mma_ss(d, da + 2 * k, db + 2 * k, s_desc, add || k > 0);
      };
      // S of one step, tile q of the streamed operand at `at`
      auto logits = [&](uint32_t d, int q, uint32_t at) {
        if (!Shape::kSplit) {
          product(d, q, at, q > 0);
        } else if (q < a.kb) {              // high x high, low x high
          product(d, q, at, q > 0);
          product(d, a.kb + q, at, true);
        } else {                            // high x low
          product(d, q - a.kb, at, true);
        }
      };
      for (int item = blockIdx.x; ok && item < items; item += gridDim.x, ++it) {
        int first;
        const int n = steps_of(item, first);
        if (!(ok = tc::bar_wait(rows_full, it & 1))) break;
        if (MODE == kLoss) {
          for (int j = 0; ok && j < n; ++j, ++step) {
            const uint32_t buf = step & 1, use = step >> 1;
            if (use > 0 && !(ok = tc::bar_wait(s_done + 8 * buf, (use - 1) & 1))) break;
            for (int q = 0; q < tiles; ++q, ++stage) {
              const uint32_t slot = stage % a.stages;
              if (!(ok = tc::bar_wait(full + 8 * slot, (stage / a.stages) & 1))) break;
              tc::fence_after();
              logits(tmem + buf * Shape::kCols, q, ring_at + slot * stage_bytes);
              tc::mma_commit(empty + 8 * slot);
            }
            if (ok) tc::mma_commit(s_full + 8 * buf);
          }
          if (ok) tc::mma_commit(rows_empty);
        } else {
          // S of step j + 1 is issued before the second product of step j, so that the
          // tensor cores work on it while the epilogue warps turn S of step j into P.  The
          // products run in the order of their issue: S of step j + 2 may overwrite P of j.
          auto issue_s = [&](uint32_t g) {
            const uint32_t slot = g % a.stages, buf = g & 1;
            if (!tc::bar_wait(full + 8 * slot, (g / a.stages) & 1)) return false;
            tc::fence_after();
            for (int q = 0; q < tiles; ++q)
              logits(tmem + buf * Shape::kCols, q, ring_at + slot * stage_bytes + q * kTileBytes);
            tc::mma_commit(s_full + 8 * buf);
            return true;
          };
          auto issue_o = [&](uint32_t g, bool begin) {
            const uint32_t slot = g % a.stages, buf = g & 1;
            if (!tc::bar_wait(s_done + 8 * buf, (g >> 1) & 1)) return false;
            tc::fence_after();
            const uint32_t d = tmem + Shape::kOutAt, at = ring_at + slot * stage_bytes;
            const uint32_t hi = tmem + buf * Shape::kCols, lo = tmem + Shape::kLowAt + buf * 64;
            const uint64_t b_hi = tc::tile_desc(at, kTileBytes);
            const uint64_t b_lo = tc::tile_desc(at + a.kb * kTileBytes, kTileBytes);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              tc::mma_ts(d, hi + 8 * k, b_hi + 128 * k, o_desc, !begin || k > 0);
              if (Shape::kSplit) {
                tc::mma_ts(d, lo + 8 * k, b_hi + 128 * k, o_desc, true);
                tc::mma_ts(d, hi + 8 * k, b_lo + 128 * k, o_desc, true);
              }
            }
            tc::mma_commit(empty + 8 * slot);
            return true;
          };
          ok = issue_s(step);
          for (int j = 0; ok && j < n; ++j, ++step) {
            if (j + 1 < n) ok = issue_s(step + 1);
            if (j + 1 == n) tc::mma_commit(rows_empty);
            if (ok && j == 0 && it > 0) ok = tc::bar_wait(out_empty, (it - 1) & 1);
            ok = ok && issue_o(step, j == 0);
          }
          if (ok) tc::mma_commit(out_full);
        }
      }
      // the last barrier arrivals of the tensor cores land before this CTA's memory is freed
      tc::mma_commit(drained);
      if (!tc::bar_wait(drained, 0) || !ok) *a.status = FG_STATUS_WAIT_EXPIRED;
    }
  } else if (warp >= kEpilogueWarp) {
    const uint32_t group = (warp - kEpilogueWarp) >> 2;   // serves the S buffer of this number
    const int quarter = warp & 3;                         // TMEM lanes 32 * quarter ...
    const uint32_t lanes_at = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lanes_at + group * Shape::kCols;
    const float scale = fmaxf(a.logit_scale * (a.unscale ? *a.unscale : 1.f), 1.17549435e-38f);
    uint32_t step = 0, it = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x, ++it) {
      int first;
      const int n = steps_of(item, first);
      const int64_t row0 = (int64_t)(item % a.row_tiles) * kTileRows;
      const int64_t row = row0 + quarter * 32 + lane;
      const bool warp_live = row0 + quarter * 32 < a.n_rows;
      if (MODE == kLoss) {
        float top = -INFINITY, sum = 0.f;
        for (int j = 0; j < n; ++j, ++step) {
          if ((step & 1) != group) continue;
          if (!(ok = warp_wait(s_full + 8 * group, (step >> 1) & 1))) break;
          if (warp_live) {
            tc::fence_after();
            const int64_t left = a.n_cols - (int64_t)(first + j) * Shape::kCols;
            float x[2][32];
            tc::tmem_load32(s_at, x[0]);
#pragma unroll
            for (int c = 0; c < Shape::kCols / 32; ++c) {
              float(&v)[32] = x[c & 1];
              tc::wait_ld32(v);
              if (c + 1 < Shape::kCols / 32) tc::tmem_load32(s_at + (c + 1) * 32, x[(c + 1) & 1]);
              if (left < (c + 1) * 32) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (c * 32 + k >= left) v[k] = -INFINITY;
              }
              float m = top;
#pragma unroll
              for (int k = 0; k < 32; ++k) m = fmaxf(m, v[k]);
              const float base = m == -INFINITY ? 0.f : m;
              sum *= exp2_fast((top - base) * scale);
              top = m;
              const float off = -base * scale;
              float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int k = 0; k < 32; ++k) part[k & 3] += exp2_fast(fmaf(v[k], scale, off));
              sum += (part[0] + part[1]) + (part[2] + part[3]);
            }
            tc::fence_before();
          }
          tc::bar_arrive(s_done + 8 * group);
        }
        if (row < a.n_rows)
          a.stats[row * (a.splits * 2) + item / a.row_tiles * 2 + group] =
              make_float2(top == -INFINITY ? -INFINITY : top * scale, sum);
      } else {
        float bias = -INFINITY;
        int64_t label = -1;
        if (MODE == kFeatGrad && row < a.n_rows) {
          bias = a.row_bias[row];
          label = a.row_label[row];
        }
        for (int j = 0; j < n; ++j, ++step) {
          if ((step & 1) != group) continue;
          const int64_t col0 = (int64_t)(first + j) * Shape::kCols;
          // whether a column of this step can be the label of a row of the tile, or has a
          // negative weight: rare where the vocabulary is large, and then looked at one by one
          bool special;
          if (MODE == kFeatGrad) {
            special = label >= col0 && label < col0 + Shape::kCols;
          } else {
            special = false;
            __syncwarp();
#pragma unroll
            for (int c = lane; c < 128; c += 32) {
              const int32_t l = a.col_label[col0 + c];
              special |= (l >= row0 && l < row0 + kTileRows) || a.col_weight[col0 + c] < 0.f;
              col_bias_s[warp - kEpilogueWarp][c] = a.col_bias[col0 + c];
            }
            __syncwarp();
          }
          special = __any_sync(0xffffffffu, special);
          const int64_t left = a.n_cols - col0;
          if (!(ok = warp_wait(s_full + 8 * group, (step >> 1) & 1))) break;
          tc::fence_after();
          float x[2][32];
          tc::tmem_load32(s_at, x[0]);
#pragma unroll
          for (int c = 0; c < Shape::kCols / 32; ++c) {
            float(&v)[32] = x[c & 1];
            tc::wait_ld32(v);
            if (c + 1 < Shape::kCols / 32) tc::tmem_load32(s_at + (c + 1) * 32, x[(c + 1) & 1]);
            if (MODE == kFeatGrad) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = exp2_fast(fmaf(v[k], scale, bias));
              if (special) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (label == col0 + c * 32 + k) v[k] -= a.hot;
              }
              if (left < (c + 1) * 32) {  // behind the vocabulary: no probability, whatever lse
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (c * 32 + k >= left) v[k] = 0.f;
              }
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 e = *reinterpret_cast<const float4*>(&col_bias_s[warp - kEpilogueWarp][c * 32 + k]);
                v[k] = exp2_fast(fmaf(v[k], scale, e.x));
                v[k + 1] = exp2_fast(fmaf(v[k + 1], scale, e.y));
                v[k + 2] = exp2_fast(fmaf(v[k + 2], scale, e.z));
                v[k + 3] = exp2_fast(fmaf(v[k + 3], scale, e.w));
              }
              if (special) {
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float w = a.col_weight[col0 + c * 32 + k];
                  if (w < 0.f) v[k] = -v[k];
                  if (a.col_label[col0 + c * 32 + k] == row) v[k] -= w * a.hot;
                }
              }
            }
            store_p<MODE, T>(s_at, lanes_at + Shape::kLowAt + group * 64, c, v);
          }
          tc::wait_st();
          tc::fence_before();
          tc::bar_arrive(s_done + 8 * group);
        }
        if (!ok || !(ok = warp_wait(out_full, it & 1))) break;
        tc::fence_after();
        // the two groups take alternate 16-column pieces of the accumulators
        float factor = 0.f;
        if (a.splits == 1 && row < a.n_rows)
          factor = (a.out_scale ? *a.out_scale : 1.f) * (MODE == kFeatGrad ? a.row_factor[row] : 1.f);
        for (int c = group * 16; c < a.out_cols; c += 32) {
          float v[16];
          __syncwarp();
          tc::tmem_load16(lanes_at + Shape::kOutAt + c, v);
          tc::wait_ld16(v);
          if (row < a.n_rows) {
            if (a.splits > 1) {  // a partial sum, rows out_cols apart
              float* to = a.partial + ((int64_t)(item / a.row_tiles) * a.n_rows + row) * a.out_cols + c;
#pragma unroll
              for (int k = 0; k < 16; k += 4)
                *reinterpret_cast<float4*>(to + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
            } else {
              if (MODE == kFeatGrad && label < 0) {
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = 0.f;
              }
              T* to = static_cast<T*>(a.out) + row * a.feat_len + c;
              constexpr int N = 16 / sizeof(T);
              if (a.feat_len % N == 0 && ((uintptr_t)a.out & 15) == 0) {
#pragma unroll
                for (int k = 0; k < 16; k += N) {
                  if (c + k >= a.feat_len) break;
                  Vec<T, N> piece;
#pragma unroll
                  for (int i = 0; i < N; ++i) piece.v[i] = from_float<T>(v[k + i] * factor);
                  store_vec<T, N>(to + k, piece);
                }
              } else {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if (c + k < a.feat_len) to[k] = from_float<T>(v[k] * factor);
              }
            }
          }
        }
        __syncwarp();
        tc::fence_before();
        tc::bar_arrive(out_empty);
      }
    }
    if (!ok && lane == 0) *a.status = FG_STATUS_WAIT_EXPIRED;
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == 2) tc::tmem_free(tmem, 512);
}

// ------------------------------------------- without tensor cores: wide features --
constexpr int kTile = 32;
constexpr int64_t kPiece = 8192;

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


// ------------------------------------------------------------ around the kernel --
// Scalars of a call, on the device (setup_kernel).
struct Consts {
  float scale_feat, scale_weight;   // powers of two that float32 operands are held with
  float unscale;                    // 1 / (scale_feat * scale_weight), of the logits
  float out_feat, out_weight;       // factors of the two gradients
  float inv_weight_max;             // 1 / the largest |loss_grad|
};
constexpr int kMaxPartials = 256;

// Largest finite magnitude per CTA of the rows that take part, for both float32 operands.
__global__ void __launch_bounds__(256)
abs_max_kernel(Batch b, const float* __restrict__ feat, int64_t feat_ld,
               const float* __restrict__ weight, int64_t weight_ld, float* __restrict__ partial) {
  float top = 0.f;
  const bool second = blockIdx.y == 1;
  const float* p = second ? weight : feat;
  const int64_t rows = second ? b.vocab : b.n, ld = second ? weight_ld : feat_ld;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
    if (!second && live_label(b, r) < 0) continue;
#pragma unroll 4
    for (int64_t c = threadIdx.x & 31; c < b.feat_len; c += 32) {
      const float v = fabsf(p[r * ld + c]);
      if (v < INFINITY) top = fmaxf(top, v);
    }
  }
  __shared__ float warps[8];
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) top = fmaxf(top, warps[w]);
    partial[blockIdx.y * kMaxPartials + blockIdx.x] = top;
  }
}

__device__ __forceinline__ float block_max(float v, float* shared) {
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < (int)blockDim.x / 32; ++w) v = fmaxf(v, shared[w]);
  return v;
}
// The power of two that brings `top` to [2^12, 2^13): the two fp16 pieces of a value then end
// at 2^-37 of the largest, and values up to 16 times the largest still fit.
__device__ __forceinline__ int operand_exponent(float top) {
  if (!(top > 0.f)) return 0;
  int e;
  frexpf(top, &e);
  return min(60, max(-60, 13 - e));
}

__global__ void __launch_bounds__(1024)
setup_kernel(Batch b, const float* __restrict__ loss_grad, const float* __restrict__ abs_max,
             int n_abs_max, float hot, Consts* consts) {
  __shared__ float shared[32];
  float top = 0.f;
  if (loss_grad)
    for (int64_t t = threadIdx.x; t < b.n; t += 1024)
      if (live_label(b, t) >= 0) top = fmaxf(top, fabsf(loss_grad[t]));
  top = block_max(top, shared);
  int ef = 0, ew = 0;
  if (abs_max) {
    const bool in = threadIdx.x < n_abs_max;
    ef = operand_exponent(block_max(in ? abs_max[threadIdx.x] : 0.f, shared));
    ew = operand_exponent(block_max(in ? abs_max[kMaxPartials + threadIdx.x] : 0.f, shared));
  }
  if (threadIdx.x == 0) {
    Consts c;
    c.scale_feat = ldexpf(1.f, ef);
    c.scale_weight = ldexpf(1.f, ew);
    c.unscale = ldexpf(1.f, -ef - ew);
    c.out_feat = ldexpf(1.f, -ew);
    c.out_weight = top * b.scale / hot * ldexpf(1.f, -ef);
    c.inv_weight_max = top >= 1.17549435e-38f ? 1.f / top : 0.f;
    *consts = c;
  }
}

// An operand as the tensor maps want it: rows of `pitch` 16-bit elements, zero behind feat_len.
// float32 becomes two fp16 pieces, the second behind the first.  A row whose label is out of
// play (`masked`) becomes zero, whatever it held.
template <typename T>
__global__ void __launch_bounds__(256)
pack_kernel(Batch b, const T* __restrict__ from, int64_t ld, int64_t rows, int64_t pitch,
            int masked, const float* __restrict__ factor, uint16_t* __restrict__ to) {
  const int64_t piece = sizeof(T) == 4 ? pitch / 2 : pitch;
  const float f = sizeof(T) == 4 ? *factor : 1.f;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
    const bool live = !masked || live_label(b, r) >= 0;
    for (int64_t c = threadIdx.x & 31; c < piece; c += 32) {
      const bool in = live && c < b.feat_len;
      if (sizeof(T) == 4) {
        const float x = in ? to_float<T>(from[r * ld + c]) * f : 0.f;
        const __half hi = __float2half_rn(x);
        to[r * pitch + c] = __half_as_ushort(hi);
        to[r * pitch + piece + c] = __half_as_ushort(__float2half_rn(x - __half2float(hi)));
      } else {
        uint16_t raw = 0;
        if (in) memcpy(&raw, &from[r * ld + c], 2);
        to[r * pitch + c] = raw;
      }
    }
  }
}

struct SampleArrays {
  float *row_bias, *row_factor, *col_bias, *col_weight;
  int32_t* label;
};
// Per sample, and for the padding up to a whole tile: what the gradients' kernels need of it.
__global__ void __launch_bounds__(256)
sample_kernel(Batch b, const float* __restrict__ lse, const float* __restrict__ loss_grad, float hot,
              const Consts* __restrict__ consts, int64_t padded, SampleArrays s) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= padded) return;
  const int32_t y = live_label(b, t);
  float bias = -INFINITY, weight = 0.f, g = 0.f;
  if (y >= 0) {
    g = loss_grad[t];
    weight = g * consts->inv_weight_max;
    bias = log2f(hot) - lse[t] * kLog2e;
  }
  s.label[t] = y;
  s.row_bias[t] = bias;
  s.row_factor[t] = g * b.scale / hot;
  s.col_weight[t] = weight;
  s.col_bias[t] = weight == 0.f ? -INFINITY : bias + log2f(fabsf(weight));
}

// loss and lse of a sample from its partial maxima and sums (base 2); the label's logit is
// computed here once more, one warp a sample.
template <typename T>
__global__ void __launch_bounds__(256)
join_loss_kernel(Batch b, const T* __restrict__ feat, int64_t feat_ld, const T* __restrict__ weight,
                 int64_t weight_ld, const float2* __restrict__ stats, int parts,
                 float* __restrict__ loss, float* __restrict__ lse, int32_t* status) {
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= b.n) return;
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.f;
  auto add = [&](float top2, float sum2) {
    const float m = fmaxf(top, top2);
    if (m == -INFINITY) {
      sum += sum2;  // 0, or NaN
    } else {
      sum = sum * exp2f(top - m) + sum2 * exp2f(top2 - m);
      top = m;
    }
  };
  for (int k = lane; k < parts; k += 32) {
    const float2 p = stats[t * parts + k];
    add(p.x, p.y);
  }
  for (int d = 16; d > 0; d >>= 1) {
    const float top2 = __shfl_xor_sync(0xffffffffu, top, d), sum2 = __shfl_xor_sync(0xffffffffu, sum, d);
    add(top2, sum2);
  }
  const float l = (top + log2f(sum)) * 0.6931471805599453f;
  const int64_t y = load_label(b.labels, b.wide, t);
  float z = 0.f;
  if (y != b.ignore_index && (uint64_t)y < (uint64_t)b.vocab)
    for (int64_t c = lane; c < b.feat_len; c += 32)
      z = fmaf(to_float<T>(feat[t * feat_ld + c]), to_float<T>(weight[y * weight_ld + c]), z);
  for (int d = 16; d > 0; d >>= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
  if (lane != 0) return;
  lse[t] = l;
  if (y == b.ignore_index) {
    loss[t] = 0.f;
  } else if ((uint64_t)y >= (uint64_t)b.vocab) {
    *status = FG_STATUS_BAD_INDEX;
    loss[t] = __int_as_float(0x7fc00000);
  } else {
    loss[t] = l - z * b.scale;
  }
}

// A gradient from the partial sums of its splits, added in order.
template <typename T>
__global__ void __launch_bounds__(256)
join_partial_kernel(const float* __restrict__ partial, int splits, int64_t rows, int out_cols,
                    int feat_len, const float* __restrict__ row_factor,
                    const int32_t* __restrict__ row_label, const float* __restrict__ out_scale,
                    T* __restrict__ out) {
  const int quads = out_cols / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / quads;
  const int c = (int)(i - row * quads) * 4;
  if (row >= rows) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    const float4 p = *reinterpret_cast<const float4*>(partial + (k * rows + row) * out_cols + c);
    sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
  }
  const float factor = (out_scale ? *out_scale : 1.f) * (row_factor ? row_factor[row] : 1.f);
  const bool live = !row_label || row_label[row] >= 0;
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c + k < feat_len) out[row * feat_len + c + k] = from_float<T>(live ? v[k] * factor : 0.f);
}

// ------------------------------------------------------------------------- host --
constexpr int kSms = 148;  // the grids below are sized for B200's 148 SMs, one CTA each

// How often the streamed operand is cut so that row_tiles x splits CTAs fill the machine: the
// count that ends first when every item costs its steps plus kItemSteps of start and end.
struct Cut {
  int splits, steps_per_split;
};
Cut cut_steps(int64_t row_tiles, int64_t steps, int item_steps) {
  Cut best = {1, (int)steps};
  int64_t best_time = INT64_MAX;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(steps, 4 * kSms / std::max<int64_t>(row_tiles, 1)));
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t per = (steps + s - 1) / s, used = (steps + per - 1) / per;
    const int64_t waves = (row_tiles * used + kSms - 1) / kSms;
    const int64_t time = waves * (per + item_steps);
    if (time < best_time) {
      best_time = time;
      best = {(int)used, (int)per};
    }
  }
  return best;
}

struct XentLayout {
  bool mma;                     // the tensor-core path
  int kb, tiles;                // 64-element tiles of a row: of one piece, of all
  int64_t pitch;                // elements of a packed row
  int64_t padded;               // n up to a whole tile
  int64_t t_tiles, v_tiles;
  int out_cols;
  Cut loss, feat, weight;
  size_t consts, abs_max, packed_feat, packed_weight;
  size_t stats, row_bias, row_factor, col_bias, col_weight, label, partial;
  size_t s_stats, s_picked, s_dz, s_live, s_acc;  // the path without tensor cores
  size_t total;
};

XentLayout xent_layout(int32_t dtype, int64_t n, int64_t vocab, int64_t feat_len, bool with_grad) {
  XentLayout l = {};
  const int planes = dtype == FG_FLOAT32 ? 2 : 1;
  l.kb = (int)((feat_len + 63) / 64);
  l.tiles = l.kb * planes;
  l.mma = l.tiles <= kMaxResidentTiles;
  l.pitch = (int64_t)l.tiles * 64;
  l.t_tiles = (n + kTileRows - 1) / kTileRows;
  l.v_tiles = (vocab + kTileRows - 1) / kTileRows;
  l.padded = l.t_tiles * kTileRows;
  l.out_cols = (int)((feat_len + 15) / 16 * 16);
  l.loss = cut_steps(l.t_tiles, (vocab + 255) / 256, 2);
  l.feat = cut_steps(l.t_tiles, l.v_tiles, 4);
  l.weight = cut_steps(l.v_tiles, l.t_tiles, 4);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (l.mma) {
    l.consts = take(sizeof(Consts));
    l.abs_max = take(2 * kMaxPartials * 4);
    l.packed_feat = take((size_t)n * l.pitch * 2);
    l.packed_weight = take((size_t)vocab * l.pitch * 2);
    l.stats = take((size_t)n * l.loss.splits * 2 * sizeof(float2));
    if (with_grad) {
      l.row_bias = take((size_t)l.padded * 4);
      l.row_factor = take((size_t)l.padded * 4);
      l.col_bias = take((size_t)l.padded * 4);
      l.col_weight = take((size_t)l.padded * 4);
      l.label = take((size_t)l.padded * 4);
      size_t rows = 0;
      if (l.feat.splits > 1) rows = (size_t)l.feat.splits * n;
      if (l.weight.splits > 1) rows = std::max(rows, (size_t)l.weight.splits * vocab);
      l.partial = take(rows * l.out_cols * 4);
    }
  } else {
    const int64_t tiles = (vocab + kTile - 1) / kTile;
    l.s_stats = take((size_t)n * tiles * sizeof(float2));
    l.s_picked = take((size_t)n * 4);
    if (with_grad) {
      l.s_dz = take((size_t)n * std::min(vocab, kPiece) * 4);
      l.s_live = take((size_t)n * feat_len * dtype_size(dtype));
      l.s_acc = take((size_t)n * feat_len * 4);
    }
  }
  l.total = at;
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

// The operands of one call as the tensor maps need them.
struct Operands {
  const void *feat, *weight;
  int64_t feat_ld, weight_ld;
};

// A 16-bit operand whose rows start on 16-byte boundaries is read where it lies.
bool fits_map(int32_t dtype, const void* p, int64_t ld) {
  return dtype != FG_FLOAT32 && ((uintptr_t)p & 15) == 0 && ld % 8 == 0;
}

template <typename T>
int pack_operand(const Batch& b, const T* from, int64_t ld, int64_t rows, int64_t pitch, int masked,
                 const float* factor, void* to, cudaStream_t s) {
  const int grid = (int)std::min<int64_t>((rows + 7) / 8, 8 * kSms);
  pack_kernel<T><<<grid, 256, 0, s>>>(b, from, ld, rows, pitch, masked, factor,
                                      static_cast<uint16_t*>(to));
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}

// Scales of float32 operands, consts, packed copies where they are needed.
template <typename T>
int prepare_operands(const Batch& b, const XentLayout& l, char* ws, const T* feat, int64_t feat_ld,
                     const T* weight, int64_t weight_ld, int32_t dtype, const float* loss_grad,
                     float hot, bool masked, cudaStream_t s, Operands* o) {
  Consts* consts = reinterpret_cast<Consts*>(ws + l.consts);
  float* abs_max = reinterpret_cast<float*>(ws + l.abs_max);
  if constexpr (sizeof(T) == 4) {
    abs_max_kernel<<<dim3(kMaxPartials, 2), 256, 0, s>>>(b, feat, feat_ld, weight, weight_ld, abs_max);
    FG_CUDA_TRY(cudaGetLastError());
  }
  if (sizeof(T) == 4 || loss_grad) {
    setup_kernel<<<1, 1024, 0, s>>>(b, loss_grad, sizeof(T) == 4 ? abs_max : nullptr, kMaxPartials,
                                    hot, consts);
    FG_CUDA_TRY(cudaGetLastError());
  }
  *o = {feat, weight, feat_ld, weight_ld};
  if (masked || !fits_map(dtype, feat, feat_ld)) {
    if (int rc = pack_operand<T>(b, feat, feat_ld, b.n, l.pitch, masked, &consts->scale_feat,
                                 ws + l.packed_feat, s))
      return rc;
    o->feat = ws + l.packed_feat;
    o->feat_ld = l.pitch;
  }
  if (!fits_map(dtype, weight, weight_ld)) {
    if (int rc = pack_operand<T>(b, weight, weight_ld, b.vocab, l.pitch, 0, &consts->scale_weight,
                                 ws + l.packed_weight, s))
      return rc;
    o->weight = ws + l.packed_weight;
    o->weight_ld = l.pitch;
  }
  return FG_OK;
}

template <int MODE, typename T>
int launch_mma(const Batch& b, const XentLayout& l, const Operands& o, const Cut& cut, MmaArgs a,
               cudaStream_t s) {
  const bool rows_are_samples = MODE != kWeightGrad;
  const void* row_p = rows_are_samples ? o.feat : o.weight;
  const void* col_p = rows_are_samples ? o.weight : o.feat;
  const int64_t row_ld = rows_are_samples ? o.feat_ld : o.weight_ld;
  const int64_t col_ld = rows_are_samples ? o.weight_ld : o.feat_ld;
  // a packed row is as wide as its pitch, an operand read where it lies as feat_len
  const int64_t row_cols = row_ld == l.pitch && sizeof(T) == 4 ? l.pitch : b.feat_len;
  const int64_t col_cols = col_ld == l.pitch && sizeof(T) == 4 ? l.pitch : b.feat_len;
  a.n_rows = rows_are_samples ? b.n : b.vocab;
  a.n_cols = rows_are_samples ? b.vocab : b.n;
  constexpr int kCols = MmaShape<MODE, T>::kCols;
  CUtensorMap row_map, col_map;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  if (!make_tile_map(&row_map, row_p, kBf16, a.n_rows, row_cols, row_ld, kTileRows) ||
      !make_tile_map(&col_map, col_p, kBf16, a.n_cols, col_cols, col_ld, kCols))
    return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  a.kb = l.kb;
  a.row_tiles = (int)((a.n_rows + kTileRows - 1) / kTileRows);
  a.steps = (int)((a.n_cols + kCols - 1) / kCols);
  a.splits = cut.splits;
  a.steps_per_split = cut.steps_per_split;
  a.feat_len = (int)b.feat_len;
  a.out_cols = l.out_cols;
  a.negate = b.scale < 0.f;
  a.logit_scale = std::fabs(b.scale) * kLog2e;
  const int stage_tiles = (MODE == kLoss ? 1 : l.tiles) * (kCols / 128);
  a.stages = std::min(kMaxStages, (kSharedBudget / kTileBytes - l.tiles) / stage_tiles);
  const size_t smem = (size_t)(l.tiles + a.stages * stage_tiles) * kTileBytes + 1024;
  auto kernel = xent_mma_kernel<MODE, T>;
  FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t items = (int64_t)a.row_tiles * a.splits;
  kernel<<<(int)std::min<int64_t>(items, kSms), kMmaThreads, smem, s>>>(row_map, col_map, a);
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}

template <typename T>
int loss_mma(const Batch& b, const XentLayout& l, char* ws, const T* feat, int64_t feat_ld,
             const T* weight, int64_t weight_ld, int32_t dtype, float* loss, float* lse,
             int32_t* status, cudaStream_t s) {
  Operands o;
  if (int rc = prepare_operands<T>(b, l, ws, feat, feat_ld, weight, weight_ld, dtype, nullptr, 1.f,
                                   false, s, &o))
    return rc;
  MmaArgs a = {};
  a.unscale = sizeof(T) == 4 ? &reinterpret_cast<Consts*>(ws + l.consts)->unscale : nullptr;
  a.stats = reinterpret_cast<float2*>(ws + l.stats);
  a.status = status;
  if (int rc = launch_mma<kLoss, T>(b, l, o, l.loss, a, s)) return rc;
  join_loss_kernel<T><<<(unsigned)((b.n + 7) / 8), 256, 0, s>>>(
      b, feat, feat_ld, weight, weight_ld, a.stats, l.loss.splits * 2, loss, lse, status);
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}

template <typename T>
int grad_mma(const Batch& b, const XentLayout& l, char* ws, const float* loss_grad, const T* feat,
             int64_t feat_ld, const T* weight, int64_t weight_ld, int32_t dtype, const float* lse,
             T* feat_grad, T* weight_grad, int32_t* status, cudaStream_t s) {
  // fp16 holds down to 2^-24: a probability of 1 is held as 2^14, so that the smallest that
  // count are 2^-38
  const float hot = dtype == FG_BFLOAT16 ? 1.f : 16384.f;
  Operands o;
  if (int rc = prepare_operands<T>(b, l, ws, feat, feat_ld, weight, weight_ld, dtype, loss_grad, hot,
                                   true, s, &o))
    return rc;
  Consts* consts = reinterpret_cast<Consts*>(ws + l.consts);
  SampleArrays arrays = {reinterpret_cast<float*>(ws + l.row_bias),
                         reinterpret_cast<float*>(ws + l.row_factor),
                         reinterpret_cast<float*>(ws + l.col_bias),
                         reinterpret_cast<float*>(ws + l.col_weight),
                         reinterpret_cast<int32_t*>(ws + l.label)};
  sample_kernel<<<(unsigned)((l.padded + 255) / 256), 256, 0, s>>>(b, lse, loss_grad, hot, consts,
                                                                   l.padded, arrays);
  FG_CUDA_TRY(cudaGetLastError());
  MmaArgs a = {};
  a.unscale = sizeof(T) == 4 ? &consts->unscale : nullptr;
  a.row_bias = arrays.row_bias;
  a.row_factor = arrays.row_factor;
  a.row_label = a.col_label = arrays.label;
  a.col_bias = arrays.col_bias;
  a.col_weight = arrays.col_weight;
  a.hot = hot;
  a.partial = reinterpret_cast<float*>(ws + l.partial);
  a.status = status;
  auto join = [&](const Cut& cut, int64_t rows, const float* row_factor, const int32_t* row_label,
                  const float* out_scale, T* out) {
    if (cut.splits == 1) return;
    const int64_t threads = rows * (l.out_cols / 4);
    join_partial_kernel<T><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(
        a.partial, cut.splits, rows, l.out_cols, (int)b.feat_len, row_factor, row_label, out_scale, out);
  };
  if (feat_grad) {
    a.out = feat_grad;
    a.out_scale = &consts->out_feat;
    if (int rc = launch_mma<kFeatGrad, T>(b, l, o, l.feat, a, s)) return rc;
    join(l.feat, b.n, arrays.row_factor, arrays.label, a.out_scale, feat_grad);
    FG_CUDA_TRY(cudaGetLastError());
  }
  if (weight_grad) {
    a.out = weight_grad;
    a.out_scale = &consts->out_weight;
    if (int rc = launch_mma<kWeightGrad, T>(b, l, o, l.weight, a, s)) return rc;
    join(l.weight, b.vocab, nullptr, nullptr, a.out_scale, weight_grad);
    FG_CUDA_TRY(cudaGetLastError());
  }
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" int64_t fg_softmax_xent_workspace_bytes(int32_t dtype, int64_t n, int64_t vocab,
                                                   int64_t feat_len, int32_t with_grad) {
  if (n <= 0 || vocab < 1 || feat_len < 1) return 0;
  return (int64_t)fg::xent_layout(dtype, n, vocab, feat_len, with_grad != 0).total;
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
  const XentLayout l = xent_layout(dtype, n, vocab, feat_len, false);
  if (!workspace_dev || ((uintptr_t)workspace_dev & 255) != 0 || workspace_bytes < (int64_t)l.total)
    return fail(FG_ERR_INVALID_ARGUMENT, "the workspace needs %lld bytes at a 256-byte boundary",
                (long long)l.total);
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace_dev);
  const Batch b = {labels_dev, index_type == FG_INDEX_INT64, n, vocab, feat_len, ignore_index, scale};
  if (l.mma) {
    int rc = FG_OK;
#define FG_LOSS(T)                                                                               \
  rc = loss_mma<T>(b, l, ws, static_cast<const T*>(feat_dev), feat_ld,                           \
                   static_cast<const T*>(weight_dev), weight_ld, dtype, loss_dev, lse_dev, status_dev, s)
    FG_DISPATCH_DTYPE(dtype, FG_LOSS)
#undef FG_LOSS
    return rc;
  }
  float2* stats = reinterpret_cast<float2*>(ws + l.s_stats);
  float* picked = reinterpret_cast<float*>(ws + l.s_picked);
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
  const XentLayout l = xent_layout(dtype, n, vocab, feat_len, true);
  char* ws = static_cast<char*>(workspace_dev);
  const Batch b = {labels_dev, index_type == FG_INDEX_INT64, n, vocab, feat_len, ignore_index, scale};
  if (l.mma) {
    int rc = FG_OK;
#define FG_GRAD(T)                                                                              \
  rc = grad_mma<T>(b, l, ws, loss_grad_dev, static_cast<const T*>(feat_dev), feat_ld,           \
                   static_cast<const T*>(weight_dev), weight_ld, dtype, lse_dev,                \
                   static_cast<T*>(feat_grad_dev), static_cast<T*>(weight_grad_dev), status_dev, s)
    FG_DISPATCH_DTYPE(dtype, FG_GRAD)
#undef FG_GRAD
    return rc;
  }
  float* dz = reinterpret_cast<float*>(ws + l.s_dz);
  float* acc = reinterpret_cast<float*>(ws + l.s_acc);
  const unsigned t_tiles = (unsigned)((n + kTile - 1) / kTile);
  const unsigned d_tiles = (unsigned)((feat_len + kTile - 1) / kTile);
#define FG_LIVE(T)                                                                         \
  live_feat_kernel<T><<<(unsigned)((n * feat_len + 255) / 256), 256, 0, s>>>(              \
      b, static_cast<const T*>(feat_dev), feat_ld, reinterpret_cast<T*>(ws + l.s_live))
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
          b, dz, reinterpret_cast<const T*>(ws + l.s_live), feat_len, v0, count,              \
          static_cast<T*>(weight_grad_dev));                                                     \
  }
    FG_DISPATCH_DTYPE(dtype, FG_PIECE)
#undef FG_PIECE
  }
  FG_CUDA_TRY(cudaGetLastError());
  return FG_OK;
}
