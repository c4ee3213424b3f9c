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
//
// float32 runs as two fp16 pieces and three products.  Every row of either operand is scaled by a
// power of two of its own, so that a masked, an infinite or a large row costs the others no bits
// (2048 x 50 021 x 128: loss 81 us, gradients 325; with one scale per operand 74 and 278).
//
// 4096 samples x 232 965 vertices x 256, bfloat16, on one B200: loss 416 us (1170 TFLOP/s; 290 us
// at the GEMM peak), loss and both gradients 2000 us (1220 TFLOP/s over the five products).  The
// loss is bound by products and exponentials alike (both units 63 % busy), the gradients by the
// products; the operands are read from DRAM once.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "elem.cuh"
#include "ring.cuh"
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
// The row's label, -1 if it takes no part; `status`: reports one out of range.
__device__ __forceinline__ int32_t live_label(const Batch& b, int64_t t, int32_t* status = nullptr) {
  if (t >= b.n) return -1;
  const int64_t y = load_label(b.labels, b.wide, t);
  if (y == b.ignore_index) return -1;
  if ((uint64_t)y < (uint64_t)b.vocab) return (int32_t)y;
  if (status) report(status, FG_STATUS_BAD_INDEX);
  return -1;
}

constexpr float kLog2e = 1.4426950408889634f;
// Off by 2^-22 of the result (a term of a sum of probabilities, or one that is rounded to 16 bits);
// results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------- the tensor-core kernel --
enum Mode { kLoss = 0, kFeatGrad = 1, kWeightGrad = 2 };

constexpr int kTileRows = 128;
constexpr int kTileBytes = kTileRows * 128;   // 128 rows of 64 16-bit elements
constexpr int kEpilogueWarp = 4;              // before them: loads, mma, TMEM, one idle
constexpr int kMaxSlots = 14;
constexpr int kMaxBuffers = 3;
constexpr int kMaxResidentTiles = 4;          // 64-element tiles of a row that stay in shared memory

struct MmaArgs {
  int64_t n_rows, n_cols;
  int kb;                 // 64-element tiles of a row (of one piece of it, for float32)
  int row_tiles, splits, steps, steps_per_split;
  int chunks;             // pieces of at most kChunkTiles tiles that the results are cut into
  int slots;              // of the ring in shared memory
  int paired;             // the second product takes two slots at a time (128 columns)
  int buffers;            // S tiles in TMEM
  int feat_len, out_cols; // out_cols: feat_len rounded up to 16
  int out_vec;            // bytes of an aligned access to the results' rows
  int negate;             // a negative scale: |scale| with -A
  float logit_scale;      // |scale| * log2(e)
  // float32: what undoes the scaling of each row (a power of two; NaN: the row holds an infinity
  // or a NaN), and the operands themselves, for the logits of such rows
  const float *row_mul, *col_mul, *row_src, *col_src;
  int64_t row_src_ld, col_src_ld;
  float2* stats;          // loss: (maximum, sum) per row, split and group of warps, base 2
  const float* row_bias;  // feat_grad: log2(hot) - lse * log2(e) of a row, -inf: takes no part
  const int32_t* row_label;
  const float* col_bias;  // weight_grad: the same of a column, plus log2 |weight|
  const float* col_weight;
  const int32_t* col_label;
  float hot;              // what a probability of 1 is held as
  const float* row_factor;  // feat_grad: factor of a row of the results
  const float* out_scale; // weight_grad, 16 bits: factor of all of them, on the device
  float out_factor;       // weight_grad, float32: the same
  void* out;              // one split: the results
  float* partial;         // several: a partial sum each, for join_partial_kernel
  int32_t* status;
};

// kStream: the rows do not stay in shared memory but come along with every step (wide rows).
template <int MODE, typename T, bool STREAM>
struct MmaShape {
  static constexpr bool kSplit = sizeof(T) == 4;  // float32 as two fp16 pieces, three products
  static constexpr int kCols = MODE == kLoss ? 256 : 128;
  // Groups of four epilogue warps.  The loss only reads S, in 64 columns a group: with four
  // warps on every scheduler the exponentials' unit stays busy across the waits of each.  The
  // gradients' groups take turns with the steps: in 16 bits two that hold twice the registers, in
  // float32 two pairs of which each group has half a step's columns (one group a step: 402 us for
  // both gradients of 2048 x 50 021 x 128 instead of 339: a warp waits for one entry's chain of
  // loads, factors and exponentials after the other, and only more warps hide that).
  static constexpr int kGroups = MODE == kLoss || kSplit ? 4 : 2;
  static constexpr int kStepGroups = MODE == kLoss ? kGroups : kGroups / 2;  // those of one step
  static constexpr int kThreads = 32 * (kEpilogueWarp + 4 * kGroups);
  static constexpr int kChunkTiles = kSplit ? 2 : 4;
  // tiles of 16 KB that a slot of the ring holds: a tile of the streamed operand, with one of
  // the rows where these are streamed too (or, for the second product, two of the first)
  static constexpr int kSlotTiles = MODE == kLoss ? (STREAM ? 3 : 2) : (STREAM ? 2 : 1);
  // float32: steps after which the accumulators are added up in registers.  Every step has an
  // exponent of its own (see the gradients' epilogue).  It also keeps the cutting small with which
  // tcgen05.mma adds to fp32, about 2^-26 of the sum each time and always towards zero: several
  // thousand additions were 1.1e-5.
  static constexpr int kSegment = kSplit ? 1 : 1 << 30;
  static constexpr int kHalfOut = 128;            // float32: the second half's accumulators
  // What the epilogue warps keep of a step's columns in shared memory: arrays, and columns a warp.
  static constexpr int kColArrays = kSplit ? (MODE == kLoss ? 1 : 2) : (MODE == kWeightGrad ? 1 : 0);
  static constexpr int kMyCols = kCols / kStepGroups;
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

// 32 columns of S become 32 k of P in 16 of the same columns.  Rounding P to the operands' type
// (half a step: 2^-8 for bfloat16, 2^-11 for float16) is what the second product's rate costs.
template <typename T>
__device__ __forceinline__ void store_p(uint32_t at, const float (&p)[32]) {
  uint32_t r[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) r[k] = pack2<T>(p[2 * k], p[2 * k + 1]);
  tc::tmem_store16(at, r);
}
// float32: 16 columns of S become 16 k of P in two pieces, eight columns each: together 2^-22.
__device__ __forceinline__ void store_p_pieces(uint32_t at, const float (&p)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    r[k] = pack2<float>(p[2 * k], p[2 * k + 1]);
    const float2 rest = __ffma2_rn(unpack_half2(r[k]), make_float2(-1.f, -1.f),
                                   make_float2(p[2 * k], p[2 * k + 1]));
    r[8 + k] = pack2<float>(rest.x, rest.y);
  }
  tc::tmem_store16(at, r);
}

// float32: factors that turn products of two scaled rows into logits in base 2.  `row` holds
// |scale| log2(e) too.  Where the two powers of two together overflow, the products are 0 or their
// logits far beyond what exp tells apart: the largest power does for both.  (It also stands for a
// NaN, whose row gets its logits from plain_logit.)
__device__ __forceinline__ float2 logit_factors(float row, float col0, float col1) {
  const float2 m = __fmul2_rn(make_float2(row, row), make_float2(col0, col1));
  return make_float2(fminf(m.x, 0x1p127f), fminf(m.y, 0x1p127f));
}
// The exponent of a power of two, 0 for NaN.
__device__ __forceinline__ float exponent_of(float power) {
  return power == power ? (float)((int)(__float_as_uint(power) >> 23) - 127) : 0.f;
}
// A row that holds an infinity or a NaN has a NaN for its factor, whose low bits say where: the first
// column, and whether it is the only one.
constexpr uint32_t kOddNan = 0x7fc00000u, kOddAlone = 1u << 20, kOddColumn = kOddAlone - 1;
constexpr int64_t kMostFeatures = kOddAlone;   // of a row
// The product of two float32 rows of which one holds an infinity or a NaN, `mark` its factor: what
// is finite does not count.  In two pieces an infinity would meet the zeros and the second pieces of
// the other row and become NaN.  (Not unrolled and not a call: registers are short where it stands.)
__device__ __forceinline__ float plain_logit(const float* x, const float* y, float mark, int n) {
  int c = __float_as_uint(mark) & kOddColumn;
  if (__float_as_uint(mark) & kOddAlone) n = c + 1;
  float z = 0.f;
#pragma unroll 1
  do z = fmaf(__ldg(x + c), __ldg(y + c), z); while (++c < n && z == z);
  return z;
}

// One verdict for the whole warp: it either goes on together or gives up together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, tc::bar_wait(bar, parity));
}

// What one item of a CTA's work is: a tile of the rows, a range of steps over the streamed
// operand, and (for the gradients of wide rows) a piece of the results' columns.  Row tiles run
// fastest: CTAs beside each other stream the same part.
struct Item {
  int row_tile, split, chunk, first, steps;
};
__device__ __forceinline__ Item item_at(const MmaArgs& a, int i) {
  Item it;
  it.row_tile = i % a.row_tiles;
  const int rest = i / a.row_tiles;
  it.chunk = rest % a.chunks;
  it.split = rest / a.chunks;
  it.first = it.split * a.steps_per_split;
  it.steps = min(a.steps_per_split, a.steps - it.first);
  return it;
}

// x[0 ... min(16, left)), N (a divisor of what `left` can be) at a time.
template <typename T, int N>
__device__ __forceinline__ void store_pieces(T* to, int left, const float (&x)[16]) {
#pragma unroll
  for (int k = 0; k < 16; k += N) {
    if (k >= left) break;
    float piece[N];
#pragma unroll
    for (int i = 0; i < N; ++i) piece[i] = x[k + i];
    store_vec<T, N>(to + k, pack<T, N>(piece));
  }
}

// Stores 16 columns of one row of the results.
template <int MODE, typename T>
__device__ __forceinline__ void store_out(const MmaArgs& a, const Item& item, int64_t row, int c,
                                          const float (&v)[16], float factor, bool live) {
  if (c >= a.out_cols) return;
  if (a.splits > 1) {  // a partial sum, rows out_cols apart
    float* to = a.partial + ((int64_t)item.split * a.n_rows + row) * a.out_cols + c;
#pragma unroll
    for (int k = 0; k < 16; k += 4)
      *reinterpret_cast<float4*>(to + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    return;
  }
  T* to = static_cast<T*>(a.out) + row * a.feat_len + c;
  float x[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = live ? v[k] * factor : 0.f;
  // as wide as every row of the results is aligned
  if (a.out_vec == 16) store_pieces<T, 16 / sizeof(T)>(to, a.feat_len - c, x);
  else if (a.out_vec == 8) store_pieces<T, 8 / sizeof(T)>(to, a.feat_len - c, x);
  else if (a.out_vec == 4) store_pieces<T, 4 / sizeof(T)>(to, a.feat_len - c, x);
  else store_pieces<T, 1>(to, a.feat_len - c, x);
}

template <int MODE, typename T, bool STREAM>
__global__ void __launch_bounds__((MmaShape<MODE, T, STREAM>::kThreads), 1)
xent_mma_kernel(const __grid_constant__ CUtensorMap row_map,
                const __grid_constant__ CUtensorMap col_map, const __grid_constant__ MmaArgs a) {
  using Shape = MmaShape<MODE, T, STREAM>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kPlanes = Shape::kSplit ? 2 : 1;
  constexpr uint32_t kSlotBytes = Shape::kSlotTiles * kTileBytes;
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t bars[2 * kMaxSlots + 2 * kMaxBuffers + 5];
  __shared__ uint32_t tmem_where;
  constexpr int kColArrays = Shape::kColArrays > 0 ? Shape::kColArrays : 1;
  constexpr int kColWarps = Shape::kColArrays > 0 ? 4 * Shape::kGroups : 1;
  __shared__ __align__(16) float col_s[kColArrays][kColWarps][Shape::kMyCols];
  // float32 gradients: what undoes a step's exponent, for every row of the last four steps
  __shared__ float undo_s[Shape::kSplit && MODE != kLoss ? 4 : 1][2][kTileRows];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_u32(raw_smem) + 1023) & ~1023u;
  const int tiles = a.kb * kPlanes;                      // tiles of a whole row
  const uint32_t rows_at = smem, ring_at = smem + (STREAM ? 0 : tiles * kTileBytes);
  const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxSlots;
  const uint32_t s_full = empty + 8 * kMaxSlots, s_done = s_full + 8 * kMaxBuffers;
  const uint32_t rows_full = s_done + 8 * kMaxBuffers, rows_empty = rows_full + 8;
  const uint32_t out_full = rows_full + 16, out_empty = rows_full + 24, drained = rows_full + 32;

  if (threadIdx.x == 0) {
    for (int k = 0; k < a.slots; ++k) {
      tc::bar_init(full + 8 * k, 1);
      tc::bar_init(empty + 8 * k, 1);
    }
    for (int k = 0; k < a.buffers; ++k) {
      tc::bar_init(s_full + 8 * k, 1);
      tc::bar_init(s_done + 8 * k, 128 * Shape::kStepGroups);
    }
    tc::bar_init(rows_full, 1);
    tc::bar_init(rows_empty, 1);
    tc::bar_init(out_full, 1);
    tc::bar_init(out_empty, 128 * Shape::kGroups);
    tc::bar_init(drained, 1);
    tc::bar_init_fence();
    tc::prefetch_map(&row_map);
    tc::prefetch_map(&col_map);
  }
  if (warp == 2) tc::tmem_alloc(smem_u32(&tmem_where), 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  begin_chained();
  // all 512 columns are this CTA's: they start at address 0, and the S tiles there
  constexpr uint32_t tmem = 0;
  const uint32_t out_at = tmem + a.buffers * Shape::kCols;
  const int items = a.row_tiles * a.splits * a.chunks;

  if (warp == 0) {
    if (lane == 0) {
      Place slot;
      Loads rows;                       // of the rows that stay
      uint32_t loaded = 0, it = 0;
      bool ok = tmem_where == tmem;
      // the next slot, free, with `n` tiles announced; 0 if the wait expired
      auto next_slot = [&](int n) -> uint32_t {
        if (loaded >= (uint32_t)a.slots && !tc::bar_wait(empty + 8 * slot.at, slot.parity ^ 1)) {
          ok = false;
          return 0;
        }
        tc::bar_expect(full + 8 * slot.at, n * kTileBytes);
        return ring_at + slot.at * kSlotBytes;
      };
      auto load = [&](uint32_t to, const CUtensorMap* map, int tile, int row) {
        tc::load_tile(to, map, tile * 64, row, full + 8 * slot.at);
      };
      auto loaded_one = [&]() {
        slot.next(a.slots);
        ++loaded;
      };
      for (int i = blockIdx.x; ok && i < items; i += gridDim.x, ++it) {
        const Item item = item_at(a, i);
        const int row0 = item.row_tile * kTileRows;
        if (!STREAM) {
          if (it > 0 && !(ok = tc::bar_wait(rows_empty, (it - 1) & 1))) break;
          tc::bar_expect(rows_full, tiles * kTileBytes);
          for (int q = 0; q < tiles; ++q)
            tc::load_tile(rows_at + q * kTileBytes, &row_map, q * 64, row0, rows_full);
          ++rows.issued;
          for (int j = 0; ok && j < item.steps; ++j)
            for (int q = 0; q < tiles; ++q) {
              const uint32_t to = next_slot(Shape::kCols / 128);
              if (!ok) break;
              load(to, &col_map, q, (item.first + j) * Shape::kCols);
              loaded_one();
            }
        } else {
          // in the order in which the products below take them
          auto load_s = [&](int j) {
            for (int kb = 0; ok && kb < a.kb; ++kb)
              for (int u = 0; u < (Shape::kSplit ? 3 : 1); ++u) {
                const uint32_t to = next_slot(1 + Shape::kCols / 128);
                if (!ok) break;
                load(to, &row_map, u == 1 ? a.kb + kb : kb, row0);
                load(to + kTileBytes, &col_map, u == 2 ? a.kb + kb : kb,
                     (item.first + j) * Shape::kCols);
                loaded_one();
              }
          };
          auto load_o = [&](int j) {
            const int t0 = item.chunk * Shape::kChunkTiles, t1 = min(a.kb, t0 + Shape::kChunkTiles);
            for (int plane = 0; ok && plane < kPlanes; ++plane)
              for (int t = t0; ok && t < t1; t += 2) {
                const uint32_t to = next_slot(min(2, t1 - t));
                if (!ok) break;
                for (int k = 0; k < min(2, t1 - t); ++k)
                  load(to + k * kTileBytes, &col_map, plane * a.kb + t + k,
                       (item.first + j) * Shape::kCols);
                loaded_one();
              }
          };
          if (MODE == kLoss) {
            for (int j = 0; ok && j < item.steps; ++j) load_s(j);
          } else {
            const int ahead = min(a.buffers - 1, item.steps);
            for (int j = 0; ok && j < ahead; ++j) load_s(j);
            for (int j = 0; ok && j < item.steps; ++j) {
              if (j + ahead < item.steps) load_s(j + ahead);
              if (ok) load_o(j);
            }
          }
        }
      }
      if (!ok) {  // give up only once nothing is in flight into this CTA's shared memory
        report(a.status, FG_STATUS_WAIT_EXPIRED);
        if (rows.any()) tc::bar_wait(rows_full, rows.last_parity());
        for (uint32_t k = 0; k < min(loaded, (uint32_t)a.slots); ++k)
          tc::bar_wait(full + 8 * k, last_round(slot, k));
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = tc::elect_one();
    const uint32_t s_desc = tc::mma_desc(kBf16, Shape::kCols, a.negate != 0, false);
    Place slot, o_slot, buf, o_buf;     // of S, and of the second product
    uint32_t used = 0, it = 0, segments = 0;
    bool ok = true;
    const uint64_t rows_desc = tc::tile_desc(rows_at, 16);
    const uint64_t ring_desc = tc::tile_desc(ring_at, 16);        // K-major
    const uint64_t ring_desc_mn = tc::tile_desc(ring_at, kTileBytes);  // 64 n per tile
    // 64 k of S
    auto product = [&](uint32_t d, uint64_t da, uint64_t db, bool add) {
#pragma unroll
      for (int k = 0; k < 4; ++k) tc::mma_ss(leader, d, da + 2 * k, db + 2 * k, s_desc, add || k > 0);
    };
    auto slot_ready = [&](const Place& p) {
      if (!warp_wait(full + 8 * p.at, p.parity)) return ok = false;
      tc::fence_after();
      return true;
    };
    // S of one step into its buffer, then its barrier; frees the slots only where the second
    // product does not need them
    auto issue_s = [&]() {
      const uint32_t d = tmem + buf.at * Shape::kCols;
      if (!STREAM) {
        for (int q = 0; q < tiles; ++q) {
          if (!slot_ready(slot)) return;
          const uint64_t db = ring_desc + slot.at * (kSlotBytes >> 4);
          if (!Shape::kSplit) {
            product(d, rows_desc + q * (kTileBytes >> 4), db, q > 0);
          } else if (q < a.kb) {           // high x high, low x high
            product(d, rows_desc + q * (kTileBytes >> 4), db, q > 0);
            product(d, rows_desc + (a.kb + q) * (kTileBytes >> 4), db, true);
          } else {                         // high x low
            product(d, rows_desc + (q - a.kb) * (kTileBytes >> 4), db, true);
          }
          if (MODE == kLoss) tc::mma_commit(leader, empty + 8 * slot.at);
          slot.next(a.slots);
        }
      } else {
        for (int q = 0; q < a.kb * (Shape::kSplit ? 3 : 1); ++q) {
          if (!slot_ready(slot)) return;
          const uint64_t da = ring_desc + slot.at * (kSlotBytes >> 4);
          product(d, da, da + (kTileBytes >> 4), q > 0);
          tc::mma_commit(leader, empty + 8 * slot.at);
          slot.next(a.slots);
        }
      }
      tc::mma_commit(leader, s_full + 8 * buf.at);
      buf.next(a.buffers);
    };
    for (int i = blockIdx.x; ok && i < items; i += gridDim.x, ++it) {
      const Item item = item_at(a, i);
      if (!STREAM && !(ok = warp_wait(rows_full, it & 1))) break;
      if (MODE == kLoss) {
        for (int j = 0; ok && j < item.steps; ++j, ++used) {
          if (used >= (uint32_t)a.buffers && !(ok = warp_wait(s_done + 8 * buf.at, buf.parity ^ 1)))
            break;
          tc::fence_after();
          issue_s();
        }
        if (ok && !STREAM) tc::mma_commit(leader, rows_empty);
      } else {
        // S of the next steps is issued before the second product of step j, so that the
        // tensor cores work on it while the epilogue warps turn S of step j into P.  The
        // products run in the order of their issue: a later S may overwrite P of step j.
        const int c0 = item.chunk * Shape::kChunkTiles * 64;
        const int cols = min(a.out_cols - c0, Shape::kChunkTiles * 64);
        // columns n0 ... of the results += P (of one step) x the tiles at `db`
        auto product_o = [&](int n0, int n, uint32_t p, uint64_t db, bool low, bool begin) {
          const uint32_t d = out_at + n0;
          const uint32_t o_desc = tc::mma_desc(kBf16, n, false, true);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            // 16 k are eight columns; float32's second pieces lie behind the first
            const uint32_t hi = Shape::kSplit ? p + 16 * k : p + 32 * (k >> 1) + 8 * (k & 1);
            if (!Shape::kSplit) {
              tc::mma_ts(leader, d, hi, db + 128 * k, o_desc, !begin || k > 0);
            } else {                       // each half of the k into accumulators of its own
              const uint32_t dk = d + (k >> 2) * Shape::kHalfOut;
              if (!low) {                  // high x high; low x high
                tc::mma_ts(leader, dk, hi, db + 128 * k, o_desc, !begin || (k & 3) > 0);
                tc::mma_ts(leader, dk, hi + 8, db + 128 * k, o_desc, true);
              } else {                     // high x low
                tc::mma_ts(leader, dk, hi, db + 128 * k, o_desc, true);
              }
            }
          }
        };
        auto issue_o = [&](int j) {
          const bool begin = j % Shape::kSegment == 0;
          if (begin && segments > 0 && !(ok = warp_wait(out_empty, (segments - 1) & 1))) return;
          if (!(ok = warp_wait(s_done + 8 * o_buf.at, o_buf.parity))) return;
          tc::fence_after();
          const uint32_t p = tmem + o_buf.at * Shape::kCols;
          if (!STREAM) {
            const int step_tiles = a.paired ? 2 : 1;
            for (int q = 0; q < tiles; q += step_tiles) {
              const int t = q < a.kb ? q : q - a.kb;
              product_o(t * 64, min(64 * step_tiles, cols - t * 64), p,
                        ring_desc_mn + o_slot.at * (kSlotBytes >> 4), q >= a.kb, begin);
              for (int k = 0; k < step_tiles; ++k) {
                tc::mma_commit(leader, empty + 8 * o_slot.at);
                o_slot.next(a.slots);
              }
            }
          } else {
            for (int plane = 0; plane < kPlanes; ++plane)
              for (int n0 = 0; n0 < cols; n0 += 128) {
                if (!slot_ready(slot)) return;
                product_o(n0, min(128, cols - n0), p, ring_desc_mn + slot.at * (kSlotBytes >> 4),
                          plane == 1, begin);
                tc::mma_commit(leader, empty + 8 * slot.at);
                slot.next(a.slots);
              }
          }
          o_buf.next(a.buffers);
          if (j + 1 == item.steps || (j + 1) % Shape::kSegment == 0) {
            tc::mma_commit(leader, out_full);
            ++segments;
          }
        };
        const int ahead = min(a.buffers - 1, item.steps);
        for (int j = 0; ok && j < ahead; ++j) issue_s();
        for (int j = 0; ok && j < item.steps; ++j) {
          if (j + ahead < item.steps) issue_s();
          if (ok && j + ahead + 1 == item.steps && !STREAM) tc::mma_commit(leader, rows_empty);
          if (ok) issue_o(j);
        }
        if (!STREAM && ok && ahead == item.steps) tc::mma_commit(leader, rows_empty);
      }
    }
    // the last barrier arrivals of the tensor cores land before this CTA's memory is freed
    tc::mma_commit(leader, drained);
    if (!warp_wait(drained, 0) || !ok) report(a.status, FG_STATUS_WAIT_EXPIRED);
  } else if (warp >= kEpilogueWarp) {
    const int group = (warp - kEpilogueWarp) >> 2;
    const int quarter = warp & 3;                         // TMEM lanes 32 * quarter ...
    const uint32_t lanes_at = (uint32_t)(quarter * 32) << 16;
    // float32 logits get their factors row by row and column by column instead
    const float scale = Shape::kSplit ? 1.f : fmaxf(a.logit_scale, 1.17549435e-38f);
    const int my_warp = Shape::kColArrays > 0 ? warp - kEpilogueWarp : 0;
    auto& my_cols = col_s[0][my_warp];                  // float32: the factor of a column's scaling
    auto& my_biases = col_s[kColArrays - 1][my_warp];   // gradients: what is added to its logits
    Place buf;
    uint32_t step = 0, segments = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
      const Item item = item_at(a, i);
      const int64_t row0 = (int64_t)item.row_tile * kTileRows;
      const int64_t row = row0 + quarter * 32 + lane;
      float row_mul = 1.f;
      bool row_odd = false;
      if (Shape::kSplit && row < a.n_rows) {
        row_mul = a.row_mul[row];
        row_odd = row_mul != row_mul;
        row_mul = fminf(row_mul * a.logit_scale, 0x1p127f);
      }
      const bool odd_rows = Shape::kSplit && MODE == kWeightGrad && __any_sync(0xffffffffu, row_odd);
      if (MODE == kLoss) {
        // Each group takes 64 of a step's 256 columns.  The exponentials are taken relative to
        // `top`, a value of the row that an earlier step had as its maximum, so that they do
        // not wait for this step's maximum; only where that turns out 2^60 above it (or there
        // is none yet) is the step looked through again with the new one.
        constexpr int kMine = Shape::kCols / Shape::kGroups;
        const bool warp_live = row0 + quarter * 32 < a.n_rows;
        float top = -INFINITY, sum = 0.f;
        // float32: the next step's factors are on the way while this one is worked on
        float next_mul[Shape::kSplit ? kMine / 32 : 1];
        auto fetch = [&](int j) {
          const int64_t col = (int64_t)(item.first + j) * Shape::kCols + group * kMine + lane;
#pragma unroll
          for (int c = 0; c < kMine / 32; ++c)
            next_mul[Shape::kSplit ? c : 0] = col + c * 32 < a.n_cols ? __ldg(a.col_mul + col + c * 32) : 1.f;
        };
        if (Shape::kSplit && warp_live) fetch(0);
        for (int j = 0; j < item.steps; ++j) {
          uint32_t odd[kMine / 32] = {};   // columns that hold an infinity or a NaN
          if (Shape::kSplit && warp_live) {
            __syncwarp();
#pragma unroll
            for (int c = 0; c < kMine / 32; ++c) {
              const float m = next_mul[Shape::kSplit ? c : 0];
              my_cols[c * 32 + lane] = m;
              odd[c] = __ballot_sync(0xffffffffu, m != m);
            }
            __syncwarp();
            if (j + 1 < item.steps) fetch(j + 1);
          }
          if (!(ok = warp_wait(s_full + 8 * buf.at, buf.parity))) break;
          if (warp_live) {
            tc::fence_after();
            const uint32_t s_at = lanes_at + tmem + buf.at * Shape::kCols + group * kMine;
            const int64_t left = a.n_cols - (int64_t)(item.first + j) * Shape::kCols - group * kMine;
            float2 part[2];
            auto pass = [&](bool with_sum) {
              const float off = top == -INFINITY ? 0.f : -top * scale;
              float largest[2] = {-INFINITY, -INFINITY};
              part[0] = part[1] = make_float2(0.f, 0.f);
#pragma unroll
              for (int c = 0; c < kMine / 32; ++c) {
                float v[32];
                tc::tmem_load32(s_at + c * 32, v);
                tc::wait_ld32(v);
                if constexpr (Shape::kSplit) {
                  for (uint32_t which = odd[c]; which; which &= which - 1) {
                    const int from = __ffs(which) - 1;
                    const int64_t col = (int64_t)(item.first + j) * Shape::kCols + group * kMine + c * 32 + from;
                    float z = 0.f;
                    if (row < a.n_rows)
                      z = plain_logit(a.row_src + row * a.row_src_ld, a.col_src + col * a.col_src_ld,
                                      my_cols[c * 32 + from], a.feat_len);
                    if (a.negate) z = -z;
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                      if (k == from) v[k] = z;
                  }
#pragma unroll
                  for (int k = 0; k < 32; k += 4) {
                    const float4 e = *reinterpret_cast<const float4*>(&my_cols[c * 32 + k]);
                    const float2 lo = __fmul2_rn(make_float2(v[k], v[k + 1]), logit_factors(row_mul, e.x, e.y));
                    const float2 hi = __fmul2_rn(make_float2(v[k + 2], v[k + 3]), logit_factors(row_mul, e.z, e.w));
                    v[k] = lo.x, v[k + 1] = lo.y, v[k + 2] = hi.x, v[k + 3] = hi.y;
                  }
                }
                if (left < (c + 1) * 32) {
#pragma unroll
                  for (int k = 0; k < 32; ++k)
                    if (c * 32 + k >= left) v[k] = -INFINITY;
                }
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                  largest[0] = fmaxf(largest[0], fmaxf(v[k], v[k + 1]));
                  largest[1] = fmaxf(largest[1], fmaxf(v[k + 2], v[k + 3]));
                }
                if (with_sum) {
#pragma unroll
                  for (int k = 0; k < 32; k += 2) {
                    float2 x = __ffma2_rn(make_float2(v[k], v[k + 1]), make_float2(scale, scale),
                                          make_float2(off, off));
                    x.x = exp2_fast(x.x);
                    x.y = exp2_fast(x.y);
                    part[k >> 1 & 1] = __fadd2_rn(part[k >> 1 & 1], x);
                  }
                }
              }
              return fmaxf(largest[0], largest[1]);
            };
            if (__any_sync(0xffffffffu, top == -INFINITY)) {
              const float m = pass(false);
              if (top == -INFINITY) top = m;
            }
            const float m = pass(true);
            const bool far = (m - top) * scale > 60.f;
            if (__any_sync(0xffffffffu, far)) {
              if (far) {
                sum *= exp2_fast((top - m) * scale);
                top = m;
              }
              pass(true);
            }
            sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
            tc::fence_before();
          }
          tc::bar_arrive(s_done + 8 * buf.at);
          buf.next(a.buffers);
        }
        if (row_odd) sum = __int_as_float(0x7fc00000);
        if (row < a.n_rows)
          a.stats[(row * a.splits + item.split) * Shape::kGroups + group] =
              make_float2(top == -INFINITY ? -INFINITY : top * scale, sum);
      } else if constexpr (Shape::kSplit) {
        // float32: the left operand of the second product is P times the power of two that the
        // streamed row is scaled by, and those of rows far apart do not fit fp16 together.  So
        // every row has an exponent that brings the largest of its entries so far to (2^13, 2^15].
        // Where one would be larger, the exponent is lowered, and what has been stored of this step
        // with it; each step's is undone when its products are added up.  An entry is off by 2^-22
        // of itself and 2^-36 of the row's largest.
        //
        // A group has half of a step's columns, with exponents and accumulators of their own; two
        // pairs of groups take turns with the steps.
        constexpr int kMine = Shape::kMyCols;
        const int pair = group >> 1, half = group & 1;
        const int32_t warp_row0 = (int32_t)row0 + quarter * 32;
        float bias = -INFINITY, factor = MODE == kFeatGrad ? 0.f : a.out_factor;
        int32_t label = -1;
        if (MODE == kFeatGrad && row < a.n_rows) {
          bias = a.row_bias[row];
          label = a.row_label[row];
          factor = a.row_factor[row];
        }
        const bool live = MODE != kFeatGrad || label >= 0;
        const int c0 = item.chunk * Shape::kChunkTiles * 64;
        float acc[2][16];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int k = 0; k < 16; ++k) acc[q][k] = 0.f;
        // adds a step's accumulators up in registers and lets the tensor cores go on; a group takes
        // every fourth 16-column piece
        int flushed = 0;
        auto flush = [&]() {
          if (!(ok = warp_wait(out_full, segments & 1))) return;
          tc::fence_after();
          const float undo[2] = {undo_s[segments & 3][0][quarter * 32 + lane],
                                 undo_s[segments & 3][1][quarter * 32 + lane]};
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int c = group * 16 + q * 64;
            if (c0 + c >= a.out_cols) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v[16];
              tc::tmem_load16(lanes_at + out_at + h * Shape::kHalfOut + c, v);
              tc::wait_ld16(v);
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                const float2 sum = __ffma2_rn(make_float2(v[k], v[k + 1]), make_float2(undo[h], undo[h]),
                                              make_float2(acc[q][k], acc[q][k + 1]));
                acc[q][k] = sum.x, acc[q][k + 1] = sum.y;
              }
            }
          }
          tc::fence_before();
          tc::bar_arrive(out_empty);
          ++segments;
          ++flushed;
        };
        // What belongs to the group's columns, on the way before the step is: lane c fetches those
        // of c and 32 + c.
        float next_mul[2], next_bias[2], next_weight[2];
        int32_t next_label[2];
        auto fetch = [&](int j) {
          const int64_t first = (int64_t)(item.first + j) * Shape::kCols + half * kMine + lane;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int64_t col = first + c * 32;
            // behind the last column there is no probability, whatever lse
            const bool in = col < a.n_cols;
            next_mul[c] = in ? __ldg(a.col_mul + col) : 1.f;
            next_bias[c] = in ? 0.f : -INFINITY;
            if (MODE == kWeightGrad) {
              next_bias[c] = a.col_bias[col];
              next_weight[c] = a.col_weight[col];
              next_label[c] = a.col_label[col];
            }
          }
        };
        float top = -1000.f;               // of the exponents of the row's entries; less counts as 0
        int lift = 14 + 1000;
        auto too_large = [&]() { return top + (float)lift > 15.f; };
        auto fit = [&]() { lift = 14 - (int)ceilf(fminf(top, 1000.f)); };
        bool fetched = false;
        for (int j = 0; j < item.steps; ++j, ++step) {
          const Place at = buf;
          buf.next(a.buffers);
          if ((step & 1) != pair) continue;
          const int64_t col0 = (int64_t)(item.first + j) * Shape::kCols + half * kMine;
          const int64_t hot_at = MODE == kFeatGrad ? label - col0 : -1;
          const bool hot_here = hot_at >= 0 && hot_at < kMine;
          // In `odd` the columns that hold an infinity or a NaN, in `hits` those whose label is one
          // of this warp's rows, in `negative` those of a negative weight.
          uint32_t odd[2] = {0, 0}, hits[2] = {0, 0}, negative[2] = {0, 0};
          if (!fetched) fetch(j);
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float m = next_mul[c];
            my_cols[c * 32 + lane] = m;
            my_biases[c * 32 + lane] = next_bias[c] + exponent_of(m);
            if (MODE == kFeatGrad) odd[c] = __ballot_sync(0xffffffffu, m != m);
            if (MODE == kWeightGrad) {
              hits[c] = __ballot_sync(0xffffffffu, next_label[c] >= warp_row0 && next_label[c] < warp_row0 + 32);
              negative[c] = __ballot_sync(0xffffffffu, next_weight[c] < 0.f);
            }
          }
          __syncwarp();
          if (hot_here) top = fmaxf(top, my_biases[hot_at]);
          const int hot_col = hot_here ? (int)hot_at : -1;
          const bool any_hot = __any_sync(0xffffffffu, hot_here);
          // weight_grad: which row the hit from column `from` is, and the label's 1 there
          auto hit_row = [&](int c, int from) {
            return a.col_label[col0 + c * 32 + from] - warp_row0;
          };
          auto hit_weight = [&](int c, int from) { return a.col_weight[col0 + c * 32 + from]; };
#pragma unroll
          for (int c = 0; c < 2; ++c)
            for (uint32_t left = hits[c]; left; left &= left - 1) {
              const int from = __ffs(left) - 1;
              if (lane == hit_row(c, from))
                top = fmaxf(top, log2f(fabsf(hit_weight(c, from))) + exponent_of(my_cols[c * 32 + from]));
            }
          if (too_large()) fit();
          if (!(ok = warp_wait(s_full + 8 * at.at, at.parity))) break;
          tc::fence_after();
          const uint32_t s_at = lanes_at + tmem + at.at * Shape::kCols + half * kMine;
#pragma unroll 1
          for (int c = 0; c < kMine / 16; ++c) {
            float v[16];
            tc::tmem_load16(s_at + c * 16, v);
            tc::wait_ld16(v);
            const int of32 = (c & 1) * 16, c32 = c >> 1;
            uint32_t which = (c32 ? odd[1] : odd[0]) >> of32 & 0xffff;
            if (odd_rows) which = 0xffff;
            for (; which; which &= which - 1) {
              const int from = __ffs(which) - 1;
              // a sample that takes no part (or is none) is not looked at
              const bool mine = row < a.n_rows && (MODE == kFeatGrad || row_odd);
              float z = 0.f;
              if (mine && my_biases[c * 16 + from] != -INFINITY)
                z = plain_logit(a.row_src + row * a.row_src_ld, a.col_src + (col0 + c * 16 + from) * a.col_src_ld,
                                MODE == kFeatGrad ? my_cols[c * 16 + from] : a.row_mul[row], a.feat_len);
              if (a.negate) z = -z;
#pragma unroll
              for (int k = 0; k < 16; ++k)
                if (k == from && mine) v[k] = z;
            }
            // the entries' logarithms
            float largest = -INFINITY;
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              const float4 m = *reinterpret_cast<const float4*>(&my_cols[c * 16 + k]);
              const float4 e = *reinterpret_cast<const float4*>(&my_biases[c * 16 + k]);
              float2 e0 = make_float2(e.x, e.y), e1 = make_float2(e.z, e.w);
              if (MODE == kFeatGrad) {
                e0 = __fadd2_rn(e0, make_float2(bias, bias));
                e1 = __fadd2_rn(e1, make_float2(bias, bias));
              }
              const float2 q0 = __ffma2_rn(make_float2(v[k], v[k + 1]), logit_factors(row_mul, m.x, m.y), e0);
              const float2 q1 = __ffma2_rn(make_float2(v[k + 2], v[k + 3]), logit_factors(row_mul, m.z, m.w), e1);
              v[k] = q0.x, v[k + 1] = q0.y, v[k + 2] = q1.x, v[k + 3] = q1.y;
              largest = fmaxf(largest, fmaxf(q0.x, q0.y));
              largest = fmaxf(largest, fmaxf(q1.x, q1.y));
            }
            top = fmaxf(top, largest);
            if (__any_sync(0xffffffffu, too_large())) {
              const int before = lift;
              if (too_large()) fit();
              tc::wait_st();
              const __half2 by = __float2half2_rn(ldexpf(1.f, max(lift - before, -126)));
#pragma unroll 1
              for (int done = 0; done < c; ++done) {
                float r[16];
                tc::tmem_load16(s_at + done * 16, r);
                tc::wait_ld16(r);
                uint32_t w[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  w[k] = __float_as_uint(r[k]);
                  __half2 h;
                  memcpy(&h, &w[k], 4);
                  h = __hmul2(h, by);
                  memcpy(&w[k], &h, 4);
                }
                tc::tmem_store16(s_at + done * 16, w);
              }
            }
            const float lifted = (float)lift;
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              const float2 q = __fadd2_rn(make_float2(v[k], v[k + 1]), make_float2(lifted, lifted));
              v[k] = exp2_fast(q.x), v[k + 1] = exp2_fast(q.y);
            }
            if (MODE == kFeatGrad) {
              if (any_hot) {
                const float hot = hot_here ? ldexpf(1.f, (int)my_biases[hot_col] + lift) : 0.f;
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if (hot_col == c * 16 + k) v[k] -= hot;
              }
            } else {
              const uint32_t minus = (c32 ? negative[1] : negative[0]) >> of32 & 0xffff;
              if (minus) {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if (minus >> k & 1) v[k] = -v[k];
              }
              uint32_t left = (c32 ? hits[1] : hits[0]) >> of32 & 0xffff;
              for (; left; left &= left - 1) {
                const int from = __ffs(left) - 1;
                const float weight = ldexpf(hit_weight(c32, of32 + from),
                                            (int)exponent_of(my_cols[c * 16 + from]) + lift);
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if (k == from && lane == hit_row(c32, of32 + from)) v[k] -= weight;
              }
            }
            store_p_pieces(s_at + c * 16, v);
          }
          float undo = ldexpf(factor, -lift);
          // 0 times it stays 0 where the sums are beyond float32
          if (isinf(undo) && !isinf(factor)) undo = copysignf(3.4028235e38f, factor);
          undo_s[step & 3][half][quarter * 32 + lane] = undo;
          tc::wait_st();
          tc::fence_before();
          tc::bar_arrive(s_done + 8 * at.at);
          fetched = j + 2 < item.steps;
          if (fetched) fetch(j + 2);
          while (ok && flushed <= j) flush();
          if (!ok) break;
        }
        if (!ok) break;
        while (ok && flushed < item.steps) flush();
        if (!ok) break;
        if (row < a.n_rows) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            store_out<MODE, T>(a, item, row, c0 + group * 16 + q * 64, acc[q], 1.f, live);
        }
      } else {
        // The groups take turns with the steps.
        const int32_t warp_row0 = (int32_t)row0 + quarter * 32;
        float bias = -INFINITY;
        int32_t label = -1;
        if (MODE == kFeatGrad && row < a.n_rows) {
          bias = a.row_bias[row];
          label = a.row_label[row];
        }
        const int c0 = item.chunk * Shape::kChunkTiles * 64;
        float factor = 0.f;
        if (a.splits == 1 && row < a.n_rows)
          factor = MODE == kFeatGrad ? a.row_factor[row] : *a.out_scale;
        const bool live = MODE != kFeatGrad || label >= 0;
        for (int j = 0; j < item.steps; ++j, ++step) {
          const Place at = buf;
          buf.next(a.buffers);
          if ((step & 1) != group) continue;
          const int64_t col0 = (int64_t)(item.first + j) * Shape::kCols;
          // weight_grad: lane c holds columns c, 32 + c, ... of the step; in `hits` those whose
          // label is one of this warp's rows, in `negative` those of a negative weight
          int32_t col_label[4];
          float col_weight[4];
          uint32_t hits[4] = {0, 0, 0, 0}, negative[4] = {0, 0, 0, 0};
          if (MODE == kWeightGrad) {
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              col_label[c] = a.col_label[col0 + c * 32 + lane];
              col_weight[c] = a.col_weight[col0 + c * 32 + lane];
              my_biases[c * 32 + lane] = a.col_bias[col0 + c * 32 + lane];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              hits[c] = __ballot_sync(0xffffffffu, col_label[c] >= warp_row0 && col_label[c] < warp_row0 + 32);
              negative[c] = __ballot_sync(0xffffffffu, col_weight[c] < 0.f);
            }
            __syncwarp();
          }
          const int64_t left = a.n_cols - col0;
          if (!(ok = warp_wait(s_full + 8 * at.at, at.parity))) break;
          tc::fence_after();
          const uint32_t s_at = lanes_at + tmem + at.at * Shape::kCols;
          float x[2][32];
          bool not_finite = false;   // a row that holds an infinity or a NaN has no finite logit
          tc::tmem_load32(s_at, x[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float(&v)[32] = x[c & 1];
            tc::wait_ld32(v);
            if (c < 3) tc::tmem_load32(s_at + (c + 1) * 32, x[(c + 1) & 1]);
            if (MODE == kWeightGrad && c == 0) not_finite = __any_sync(0xffffffffu, !(fabsf(v[0]) < INFINITY));
            if (MODE == kFeatGrad) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = exp2_fast(fmaf(v[k], scale, bias));
              const int64_t at_label = label - (col0 + c * 32);
              if (__any_sync(0xffffffffu, at_label >= 0 && at_label < 32)) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (at_label == k) v[k] -= a.hot;
              }
              if (left < (c + 1) * 32) {  // behind the vocabulary: no probability, whatever lse
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (c * 32 + k >= left) v[k] = 0.f;
              }
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 e = *reinterpret_cast<const float4*>(&my_biases[c * 32 + k]);
                v[k] = exp2_fast(fmaf(v[k], scale, e.x));
                v[k + 1] = exp2_fast(fmaf(v[k + 1], scale, e.y));
                v[k + 2] = exp2_fast(fmaf(v[k + 2], scale, e.z));
                v[k + 3] = exp2_fast(fmaf(v[k + 3], scale, e.w));
              }
              if (not_finite) {  // samples that take no part are zeros, which meet an infinity as NaN
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (my_biases[c * 32 + k] == -INFINITY) v[k] = 0.f;
              }
              if (negative[c]) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (negative[c] >> k & 1) v[k] = -v[k];
              }
              for (uint32_t left_hits = hits[c]; left_hits; left_hits &= left_hits - 1) {
                const int from = __ffs(left_hits) - 1;
                const int32_t hit = __shfl_sync(0xffffffffu, col_label[c], from) - warp_row0;
                const float weight = __shfl_sync(0xffffffffu, col_weight[c], from) * a.hot;
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (k == from && lane == hit) v[k] -= weight;
              }
            }
            store_p<T>(s_at + c * 32, v);
          }
          tc::wait_st();
          tc::fence_before();
          tc::bar_arrive(s_done + 8 * at.at);
        }
        if (!ok) break;
        // the two groups take alternate 16-column pieces of the accumulators
        if (!(ok = warp_wait(out_full, segments & 1))) break;
        tc::fence_after();
        ++segments;
        const int cols = min(a.out_cols - c0, Shape::kChunkTiles * 64);
        for (int c = group * 16; c < cols; c += 32) {
          float v[16];
          __syncwarp();
          tc::tmem_load16(lanes_at + out_at + c, v);
          tc::wait_ld16(v);
          if (row < a.n_rows) store_out<MODE, T>(a, item, row, c0 + c, v, factor, live);
        }
        __syncwarp();
        tc::fence_before();
        tc::bar_arrive(out_empty);
      }
    }
    if (!ok && lane == 0) report(a.status, FG_STATUS_WAIT_EXPIRED);
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == 2) tc::tmem_free(tmem_where, 512);
}

// ------------------------------------------------------------ around the kernel --
// Scalars of a call in 16 bits, on the device.
struct Consts {
  float out_weight;                 // factor of weight_grad
  float inv_weight_max;             // 1 / the largest |loss_grad|
};

__device__ __forceinline__ float block_max(float v, float* shared) {
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < (int)blockDim.x / 32; ++w) v = fmaxf(v, shared[w]);
  return v;
}
// The power of two that brings `top`, the largest magnitude of a float32 row, to [2^12, 2^13): the
// two fp16 pieces of a value are then off by 2^-22 of it and 2^-37 of the row's largest.
__device__ __forceinline__ int row_exponent(float top) {
  if (!(top > 0.f)) return 0;
  int e;
  frexpf(top, &e);
  return min(126, 13 - e);
}

// What the gradients' kernels need of a sample, and of the padding up to a whole tile.
struct SampleArrays {
  const float *lse, *loss_grad;
  float *row_bias, *row_factor, *col_bias, *col_weight;
  int32_t* label;
  int64_t padded;
  float hot;
  int32_t* status;
};
__device__ __forceinline__ void sample(const Batch& b, const SampleArrays& s, float inv_weight_max,
                                       int64_t t) {
  const int32_t y = live_label(b, t, s.status);
  float bias = -INFINITY, weight = 0.f, g = 0.f;
  if (y >= 0) {
    g = s.loss_grad[t];
    weight = g * inv_weight_max;
    bias = log2f(s.hot) - s.lse[t] * kLog2e;
  }
  s.label[t] = y;
  s.row_bias[t] = bias;
  s.row_factor[t] = g * b.scale / s.hot;
  s.col_weight[t] = weight;
  s.col_bias[t] = weight == 0.f ? -INFINITY : bias + log2f(fabsf(weight));
}

// 16 bits: the scalars, by one CTA; it also makes the sample arrays of a batch of up to
// kSetupSamples.
constexpr int64_t kSetupSamples = 8192;
__device__ __forceinline__ void setup(const Batch& b, const SampleArrays& s, Consts* consts) {
  __shared__ float shared[32];
  float top = 0.f;
  for (int64_t t = threadIdx.x; t < b.n; t += blockDim.x)
    if (live_label(b, t) >= 0) top = fmaxf(top, fabsf(s.loss_grad[t]));
  top = block_max(top, shared);
  const float inv = top >= 1.17549435e-38f ? 1.f / top : 0.f;
  if (threadIdx.x == 0) *consts = {top * b.scale / s.hot, inv};
  if (s.padded <= kSetupSamples)
    for (int64_t t = threadIdx.x; t < s.padded; t += blockDim.x) sample(b, s, inv, t);
}
__global__ void __launch_bounds__(256)
sample_kernel(Batch b, SampleArrays s, const Consts* __restrict__ consts) {
  begin_chained();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t < s.padded) sample(b, s, consts->inv_weight_max, t);
}

// Operands as the tensor maps want them: rows of `pitch` 16-bit elements, zero behind feat_len.
// float32 becomes two fp16 pieces of the row scaled by its own power of two, the second behind the
// first; `mul` gets what undoes the scaling, or NaN for a row with an infinity or a NaN, whose
// pieces keep these in their places.  A row whose label is out of play (`masked`) becomes zero,
// whatever it held.  The first `blocks` CTAs pack one operand, the others the second.  In 16 bits
// the last CTA makes the scalars (`with_setup`); in float32 the samples' arrays need none and are
// made along with the samples' rows.
template <typename T>
struct PackJob {
  const T* from;
  int64_t ld, rows;
  int blocks, masked;
  float* mul;
  uint16_t* to;
};
template <typename T>
__global__ void __launch_bounds__(256)
pack_kernel(Batch b, PackJob<T> first, PackJob<T> second, int64_t pitch, int with_setup, SampleArrays s,
            Consts* consts) {
  begin_chained();
  if (with_setup && blockIdx.x == gridDim.x - 1) {
    setup(b, s, consts);
    return;
  }
  const bool is_second = (int)blockIdx.x >= first.blocks;
  const PackJob<T> j = is_second ? second : first;
  const int64_t block = is_second ? blockIdx.x - first.blocks : blockIdx.x;
  const int64_t piece = sizeof(T) == 4 ? pitch / 2 : pitch;
  const int lane = threadIdx.x & 31;
  const bool with_samples = sizeof(T) == 4 && !is_second && s.loss_grad;
  const int64_t rows = with_samples ? s.padded : j.rows;
  for (int64_t r = block * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)j.blocks * 8) {
    if (with_samples && lane == 0) sample(b, s, 1.f, r);
    if (r >= j.rows) continue;
    const bool live = !j.masked || live_label(b, r) >= 0;
    float f = 1.f;
    if constexpr (sizeof(T) == 4) {
      float top = 0.f;
      bool odd = false;
      if (live) {
#pragma unroll 4
        for (int64_t c = lane; c < b.feat_len; c += 32) {
          const float x = fabsf(j.from[r * j.ld + c]);
          if (x < INFINITY) top = fmaxf(top, x); else odd = true;
        }
      }
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      uint32_t mark = 0;                 // of a row with an infinity or a NaN
      if (__any_sync(0xffffffffu, odd)) {
        uint32_t first = kOddColumn, count = 0;
        for (int64_t c = lane; c < b.feat_len; c += 32)
          if (!(fabsf(j.from[r * j.ld + c]) < INFINITY)) {
            first = min(first, (uint32_t)c);
            ++count;
          }
        first = __reduce_min_sync(0xffffffffu, first);
        count = __reduce_add_sync(0xffffffffu, count);
        mark = kOddNan | first | (count == 1 ? kOddAlone : 0);
      }
      const int e = row_exponent(top);
      f = ldexpf(1.f, e);
      // a row of zeros adds nothing, and its scaling is the least of all, so that its probabilities
      // do not set the exponents of the second products
      const float undo = top > 0.f ? ldexpf(1.f, -e) : 0x1p-126f;
      if (lane == 0) j.mul[r] = mark ? __uint_as_float(mark) : undo;
    }
    // two neighbouring elements a lane, so that the 16-bit pieces are written as 32 bits
#pragma unroll 2
    for (int64_t c = lane * 2; c < piece; c += 64) {
      T x[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        x[k] = live && c + k < b.feat_len ? j.from[r * j.ld + c + k] : from_float<T>(0.f);
      if constexpr (sizeof(T) == 4) {
        const float y0 = x[0] * f, y1 = x[1] * f;
        const __half2 hi = __floats2half2_rn(y0, y1);
        const float2 back = __half22float2(hi);
        const __half2 lo = __floats2half2_rn(isinf(y0) ? 0.f : y0 - back.x, isinf(y1) ? 0.f : y1 - back.y);
        *reinterpret_cast<__half2*>(j.to + r * pitch + c) = hi;
        *reinterpret_cast<__half2*>(j.to + r * pitch + piece + c) = lo;
      } else {
        uint32_t raw;
        memcpy(&raw, x, 4);
        *reinterpret_cast<uint32_t*>(j.to + r * pitch + c) = raw;
      }
    }
  }
}

// loss and lse of a sample from its partial maxima and sums (base 2); the label's logit is
// computed here once more, one warp a sample, so that 16-bit and float32 samples alike lose nothing
// of it to tensor core sums.
template <typename T>
__global__ void __launch_bounds__(256)
join_loss_kernel(Batch b, const T* __restrict__ feat, int64_t feat_ld, const T* __restrict__ weight,
                 int64_t weight_ld, const float2* __restrict__ stats, int parts,
                 float* __restrict__ loss, float* __restrict__ lse, int32_t* status) {
  begin_chained();
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
    report(status, FG_STATUS_BAD_INDEX);
    loss[t] = __int_as_float(0x7fc00000);
  } else {
    // not below zero: l is a sum that the tensor cores have cut, z one in another order, and where
    // the label has all the probability their difference is the rounding of either sign
    const float d = l - z * b.scale;
    loss[t] = d < 0.f ? 0.f : d;
  }
}

// A gradient from the partial sums of its splits.  A thread adds every kJoinParts-th of them,
// and the first thread of a result those sums in order.
constexpr int kJoinParts = 8;
template <typename T>
__global__ void __launch_bounds__(256)
join_partial_kernel(const float* __restrict__ partial, int splits, int64_t rows, int out_cols,
                    int feat_len, const float* __restrict__ row_factor,
                    const int32_t* __restrict__ row_label, const float* __restrict__ out_scale,
                    T* __restrict__ out) {
  begin_chained();
  constexpr int kQuads = 256 / kJoinParts;
  __shared__ float4 sums[kJoinParts][kQuads];
  const int quads = out_cols / 4;
  const int part = threadIdx.x / kQuads, at = threadIdx.x % kQuads;
  const int64_t i = (int64_t)blockIdx.x * kQuads + at;
  const int64_t row = i / quads;
  const int c = (int)(i - row * quads) * 4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row < rows)
#pragma unroll 4
    for (int k = part; k < splits; k += kJoinParts) {
      const float4 p = *reinterpret_cast<const float4*>(partial + (k * rows + row) * out_cols + c);
      sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
    }
  sums[part][at] = sum;
  __syncthreads();
  if (part != 0 || row >= rows) return;
#pragma unroll
  for (int k = 1; k < kJoinParts; ++k) {
    const float4 p = sums[k][at];
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
constexpr int kLossGroups = MmaShape<kLoss, float, false>::kGroups;
constexpr int kSms = 148;  // the grids below are sized for B200's 148 SMs, one CTA each

// How often the streamed operand is cut so that row_tiles x splits CTAs fill the machine: the
// count that ends first when every item costs its steps plus `item_steps` of start and end.
struct Cut {
  int splits, steps_per_split;
};
Cut cut_steps(int64_t row_tiles, int64_t steps, int item_steps, int64_t most_steps) {
  const int64_t least = (steps + most_steps - 1) / most_steps;
  Cut best = {1, (int)steps};
  int64_t best_time = INT64_MAX;
  // of the counts that give as many waves, the largest ends first: five numbers of waves
  const int64_t waves0 = std::max<int64_t>(1, (row_tiles * least + kSms - 1) / kSms);
  for (int64_t w = waves0; w < waves0 + 5; ++w) {
    // but no more than four waves' worth: partial sums are written and read once more
    const int64_t fit = std::min(w, (int64_t)4) * kSms / std::max<int64_t>(row_tiles, 1);
    const int64_t s = std::min(steps, std::max({least, (int64_t)1, fit}));
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
  int kb, tiles;                // 64-element tiles of a row: of one piece, of all
  int64_t pitch;                // elements of a packed row
  int64_t padded;               // n up to a whole tile
  int64_t t_tiles, v_tiles;
  int out_cols;
  Cut loss, feat, weight;
  size_t consts, feat_mul, weight_mul, packed_feat, packed_weight;
  size_t stats, row_bias, row_factor, col_bias, col_weight, label, partial;
  size_t total, total_in_place;
};

XentLayout xent_layout(int32_t dtype, int64_t n, int64_t vocab, int64_t feat_len, bool with_grad) {
  XentLayout l = {};
  const int planes = dtype == FG_FLOAT32 ? 2 : 1;
  l.kb = (int)((feat_len + 63) / 64);
  l.tiles = l.kb * planes;
  l.pitch = (int64_t)l.tiles * 64;
  l.t_tiles = (n + kTileRows - 1) / kTileRows;
  l.v_tiles = (vocab + kTileRows - 1) / kTileRows;
  l.padded = l.t_tiles * kTileRows;
  l.out_cols = (int)((feat_len + 15) / 16 * 16);
  // 1024 steps of the 16-bit gradients are 8192 additions into the same accumulators, which
  // cut (see kSegment) by 2^-26 of the sum: 1.2e-4 at most, a quarter of float16's half step
  // (2^-11 = 4.9e-4); the pieces are joined in fp32
  const int64_t most_steps = dtype == FG_FLOAT32 ? INT32_MAX : 1024;
  const int chunk_tiles = dtype == FG_FLOAT32 ? 2 : 4;
  const int64_t chunks = (l.kb + chunk_tiles - 1) / chunk_tiles;
  l.loss = cut_steps(l.t_tiles, (vocab + 255) / 256, 2, INT32_MAX);
  l.feat = cut_steps(l.t_tiles * chunks, l.v_tiles, 4, most_steps);
  l.weight = cut_steps(l.v_tiles * chunks, l.t_tiles, 4, most_steps);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.consts = take(sizeof(Consts));
  if (dtype == FG_FLOAT32) {
    l.feat_mul = take((size_t)n * 4);
    l.weight_mul = take((size_t)vocab * 4);
  }
  l.packed_feat = take((size_t)n * l.pitch * 2);
  l.stats = take((size_t)n * l.loss.splits * kLossGroups * sizeof(float2));
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
  // last: a table that is read where it lies needs no room for it
  l.total_in_place = at;
  l.packed_weight = take((size_t)vocab * l.pitch * 2);
  l.total = at;
  return l;
}

int check_xent(const void* feat, const void* weight, int32_t dtype, int64_t feat_ld,
               int64_t weight_ld, const void* labels, int32_t index_type, int64_t n, int64_t vocab,
               int64_t feat_len, float scale, const int32_t* status) {
  if (!std::isfinite(scale))
    return fail(FG_ERR_INVALID_ARGUMENT, "scale=%g is not finite", (double)scale);
  if (!dtype_known(dtype) || !index_known(index_type))
    return fail(FG_ERR_INVALID_ARGUMENT, "unknown dtype=%d or index_type=%d", (int)dtype,
                (int)index_type);
  if (n < 0 || vocab < 1 || feat_len < 1 || feat_ld < feat_len || weight_ld < feat_len)
    return fail(FG_ERR_INVALID_ARGUMENT,
                "bad shape: n=%lld vocab=%lld feat_len=%lld feat_ld=%lld weight_ld=%lld",
                (long long)n, (long long)vocab, (long long)feat_len, (long long)feat_ld,
                (long long)weight_ld);
  if (n >= INT32_MAX / 2 || vocab >= INT32_MAX / 2 || feat_len > kMostFeatures)
    return fail(FG_ERR_UNSUPPORTED, "n and vocab must be below 2^30, feat_len at most 2^20");
  if (!weight || (n > 0 && (!feat || !labels || !status)))
    return fail(FG_ERR_INVALID_ARGUMENT, "null pointer");
  const size_t es = dtype_size(dtype);
  if (((uintptr_t)feat | (uintptr_t)weight) % es != 0)
    return fail(FG_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its type");
  if (((uintptr_t)labels & (index_type == FG_INDEX_INT64 ? 7 : 3)) != 0 || ((uintptr_t)status & 3) != 0)
    return fail(FG_ERR_INVALID_ARGUMENT, "labels or status are not aligned to their type");
  return FG_OK;
}

// Whether one of the results shares memory with one of the inputs or another result.
bool results_overlap(std::initializer_list<Array2d> results, std::initializer_list<Array2d> inputs) {
  for (const Array2d* r = results.begin(); r != results.end(); ++r) {
    for (const Array2d& in : inputs)
      if (overlap(*r, in)) return true;
    for (const Array2d* q = results.begin(); q != r; ++q)
      if (overlap(*r, *q)) return true;
  }
  return false;
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

// Packed copies of the operands where they are needed and, with loss_grad, the samples' arrays
// (in 16 bits the scalars too).  `chained`: whether this call has launched something.
template <typename T>
int prepare_operands(const Batch& b, const XentLayout& l, char* ws, const T* feat, int64_t feat_ld,
                     const T* weight, int64_t weight_ld, int32_t dtype, const SampleArrays& samples,
                     cudaStream_t s, Operands* o, bool* chained) {
  Consts* consts = reinterpret_cast<Consts*>(ws + l.consts);
  const bool grad = samples.loss_grad != nullptr;
  // gradients always pack the features, 16-bit ones make the scalars beside that
  const bool with_setup = sizeof(T) == 2 && grad;
  *o = {feat, weight, feat_ld, weight_ld};
  auto blocks = [](int64_t rows) { return (int)std::min<int64_t>((rows + 7) / 8, 8 * kSms); };
  PackJob<T> jobs[2] = {};
  if (grad || !fits_map(dtype, feat, feat_ld)) {
    jobs[0] = {feat, feat_ld, b.n, blocks(b.n), grad, reinterpret_cast<float*>(ws + l.feat_mul),
               reinterpret_cast<uint16_t*>(ws + l.packed_feat)};
    o->feat = ws + l.packed_feat;
    o->feat_ld = l.pitch;
  }
  if (!fits_map(dtype, weight, weight_ld)) {
    jobs[1] = {weight, weight_ld, b.vocab, blocks(b.vocab), 0, reinterpret_cast<float*>(ws + l.weight_mul),
               reinterpret_cast<uint16_t*>(ws + l.packed_weight)};
    o->weight = ws + l.packed_weight;
    o->weight_ld = l.pitch;
  }
  if (jobs[0].blocks + jobs[1].blocks > 0) {
    FG_CUDA_TRY(launch(*chained, pack_kernel<T>, jobs[0].blocks + jobs[1].blocks + with_setup, 256, 0, s, b,
                       jobs[0], jobs[1], l.pitch, with_setup, samples, consts));
    *chained = true;
  }
  if (with_setup && samples.padded > kSetupSamples)
    FG_CUDA_TRY(launch(true, sample_kernel, (unsigned)((samples.padded + 255) / 256), 256, 0, s, b, samples,
                       consts));
  return FG_OK;
}
// float32: the rows' scalings and the operands they belong to, for the kernel.
template <typename T>
void set_row_scalings(MmaArgs* a, const XentLayout& l, char* ws, bool rows_are_samples, const T* feat,
                      int64_t feat_ld, const T* weight, int64_t weight_ld) {
  if constexpr (sizeof(T) == 4) {
    const float* mul[2] = {reinterpret_cast<float*>(ws + l.feat_mul), reinterpret_cast<float*>(ws + l.weight_mul)};
    const float* src[2] = {feat, weight};
    const int64_t ld[2] = {feat_ld, weight_ld};
    const int row = rows_are_samples ? 0 : 1;
    a->row_mul = mul[row];
    a->row_src = src[row];
    a->row_src_ld = ld[row];
    a->col_mul = mul[1 - row];
    a->col_src = src[1 - row];
    a->col_src_ld = ld[1 - row];
  }
}

template <int MODE, typename T, bool STREAM>
int launch_mma_as(const Batch& b, const XentLayout& l, const Operands& o, const Cut& cut, MmaArgs a,
                  bool chained, int device, cudaStream_t s) {
  using Shape = MmaShape<MODE, T, STREAM>;
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
  constexpr int kCols = Shape::kCols;
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
  a.out_vec = common_vector_bytes({(uint64_t)(uintptr_t)a.out, (uint64_t)b.feat_len * sizeof(T)});
  a.logit_scale = std::min(std::fabs(b.scale) * kLog2e, std::numeric_limits<float>::max());
  // shared memory: 14 tiles of 16 KB at most, 13 where what belongs to columns needs some of it
  const int room = Shape::kColArrays > 0 ? 13 : 14;
  const int resident = STREAM ? 0 : l.tiles;
  a.slots = std::min(kMaxSlots, (room - resident) / Shape::kSlotTiles);
  // Two neighbouring slots are one operand of 128 columns where a step's tiles come in pairs and
  // no pair goes around the end of the ring: half the mma of the second product (feat_grad of
  // 4096 x 65 536 x 128: 131 -> 126 us).  Not where the odd slot that goes for it leaves less
  // than half a step of lead (weight_grad at 256 columns: 226 us against 218), except float32,
  // whose second product is three times as many mma (xent_train 2048 x 50 021 x 128: 418 -> 390).
  a.paired = !STREAM && l.kb % 2 == 0 &&
             (Shape::kSplit || (a.slots & ~1) * Shape::kSlotTiles >= 2 * l.tiles + 2);
  if (a.paired) a.slots &= ~1;
  const size_t smem = (size_t)(resident + a.slots * Shape::kSlotTiles) * kTileBytes + 1024;
  // TMEM: 512 columns, two S tiles, three where the accumulators need only 128 columns
  a.buffers = MODE != kLoss && !Shape::kSplit && l.out_cols <= 128 ? 3 : 2;
  a.chunks = MODE == kLoss ? 1 : (l.kb + Shape::kChunkTiles - 1) / Shape::kChunkTiles;
  auto kernel = xent_mma_kernel<MODE, T, STREAM>;
  FG_CUDA_TRY(allow_shared((const void*)kernel, room * kTileBytes + 1024, device));
  const int64_t items = (int64_t)a.row_tiles * a.splits * a.chunks;
  if (items > INT32_MAX) return fail(FG_ERR_UNSUPPORTED, "too many tiles");
  FG_CUDA_TRY(launch(chained, kernel, (unsigned)std::min<int64_t>(items, kSms), Shape::kThreads, smem, s,
                     row_map, col_map, a));
  return FG_OK;
}

template <int MODE, typename T>
int launch_mma(const Batch& b, const XentLayout& l, const Operands& o, const Cut& cut, const MmaArgs& a,
               bool chained, int device, cudaStream_t s) {
  return l.tiles <= kMaxResidentTiles ? launch_mma_as<MODE, T, false>(b, l, o, cut, a, chained, device, s)
                                      : launch_mma_as<MODE, T, true>(b, l, o, cut, a, chained, device, s);
}

template <typename T>
int loss_mma(const Batch& b, const XentLayout& l, char* ws, const T* feat, int64_t feat_ld,
             const T* weight, int64_t weight_ld, int32_t dtype, float* loss, float* lse,
             int32_t* status, int device, cudaStream_t s) {
  Operands o;
  SampleArrays none = {};
  none.hot = 1.f;
  bool chained = false;
  if (int rc = prepare_operands<T>(b, l, ws, feat, feat_ld, weight, weight_ld, dtype, none, s, &o, &chained))
    return rc;
  MmaArgs a = {};
  set_row_scalings<T>(&a, l, ws, true, feat, feat_ld, weight, weight_ld);
  a.stats = reinterpret_cast<float2*>(ws + l.stats);
  a.status = status;
  if (int rc = launch_mma<kLoss, T>(b, l, o, l.loss, a, chained, device, s)) return rc;
  FG_CUDA_TRY(launch(true, join_loss_kernel<T>, (unsigned)((b.n + 7) / 8), 256, 0, s, b, feat, feat_ld,
                     weight, weight_ld, a.stats, l.loss.splits * kLossGroups, loss, lse, status));
  return FG_OK;
}

template <typename T>
int grad_mma(const Batch& b, const XentLayout& l, char* ws, const float* loss_grad, const T* feat,
             int64_t feat_ld, const T* weight, int64_t weight_ld, int32_t dtype, const float* lse,
             T* feat_grad, T* weight_grad, int32_t* status, int device, cudaStream_t s) {
  // fp16 holds down to 2^-24: a probability of 1 is held as 2^14, so that the smallest that
  // count are 2^-38 (float32's have their own exponents)
  const float hot = dtype == FG_FLOAT16 ? 16384.f : 1.f;
  const SampleArrays arrays = {lse, loss_grad,
                               reinterpret_cast<float*>(ws + l.row_bias),
                               reinterpret_cast<float*>(ws + l.row_factor),
                               reinterpret_cast<float*>(ws + l.col_bias),
                               reinterpret_cast<float*>(ws + l.col_weight),
                               reinterpret_cast<int32_t*>(ws + l.label), l.padded, hot, status};
  Operands o;
  bool chained = false;
  if (int rc = prepare_operands<T>(b, l, ws, feat, feat_ld, weight, weight_ld, dtype, arrays, s, &o, &chained))
    return rc;
  Consts* consts = reinterpret_cast<Consts*>(ws + l.consts);
  MmaArgs a = {};
  a.row_bias = arrays.row_bias;
  a.row_factor = arrays.row_factor;
  a.row_label = a.col_label = arrays.label;
  a.col_bias = arrays.col_bias;
  a.col_weight = arrays.col_weight;
  a.hot = hot;
  a.partial = reinterpret_cast<float*>(ws + l.partial);
  a.status = status;
  auto join = [&](const Cut& cut, int64_t rows, const float* row_factor, const int32_t* row_label,
                  const float* out_scale, T* out) -> cudaError_t {
    if (cut.splits == 1) return cudaSuccess;
    const int64_t quads = rows * (l.out_cols / 4), per_block = 256 / kJoinParts;
    if ((quads + per_block - 1) / per_block > INT32_MAX) return cudaErrorInvalidConfiguration;
    return launch(true, join_partial_kernel<T>, (unsigned)((quads + per_block - 1) / per_block), 256, 0, s,
                  a.partial, cut.splits, rows, l.out_cols, (int)b.feat_len, row_factor, row_label,
                  out_scale, out);
  };
  constexpr bool kSplit = sizeof(T) == 4;   // whose sums have their factors already
  if (feat_grad) {
    a.out = feat_grad;
    set_row_scalings<T>(&a, l, ws, true, feat, feat_ld, weight, weight_ld);
    if (int rc = launch_mma<kFeatGrad, T>(b, l, o, l.feat, a, true, device, s)) return rc;
    FG_CUDA_TRY(join(l.feat, b.n, kSplit ? nullptr : arrays.row_factor, arrays.label, nullptr, feat_grad));
  }
  if (weight_grad) {
    a.out = weight_grad;
    a.out_scale = &consts->out_weight;
    a.out_factor = b.scale;
    set_row_scalings<T>(&a, l, ws, false, feat, feat_ld, weight, weight_ld);
    if (int rc = launch_mma<kWeightGrad, T>(b, l, o, l.weight, a, true, device, s)) return rc;
    FG_CUDA_TRY(join(l.weight, b.vocab, nullptr, nullptr, kSplit ? nullptr : a.out_scale, weight_grad));
  }
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" int64_t fg_softmax_xent_workspace_bytes(int32_t dtype, int64_t n, int64_t vocab,
                                                   int64_t feat_len, int32_t with_grad) {
  if (n <= 0 || vocab < 1 || feat_len < 1) return 0;
  const fg::XentLayout l = fg::xent_layout(dtype, n, vocab, feat_len, (with_grad & ~FG_XENT_TABLE_IN_PLACE) != 0);
  return (int64_t)((with_grad & FG_XENT_TABLE_IN_PLACE) && dtype != FG_FLOAT32 ? l.total_in_place : l.total);
}

extern "C" int fg_softmax_xent(const void* feat_dev, int64_t feat_ld, const void* weight_dev,
                               int64_t weight_ld, int32_t dtype, const void* labels_dev,
                               int32_t index_type, int64_t n, int64_t vocab, int64_t feat_len,
                               float scale, int64_t ignore_index, float* loss_dev, float* lse_dev,
                               void* workspace_dev, int64_t workspace_bytes, int32_t* status_dev,
                               int32_t device, void* stream) {
  using namespace fg;
  if (int rc = check_xent(feat_dev, weight_dev, dtype, feat_ld, weight_ld, labels_dev, index_type,
                          n, vocab, feat_len, scale, status_dev))
    return rc;
  if (n == 0) return FG_OK;
  if (!loss_dev || !lse_dev || (((uintptr_t)loss_dev | (uintptr_t)lse_dev) & 3) != 0)
    return fail(FG_ERR_INVALID_ARGUMENT, "null loss or lse, or not aligned to float");
  const XentLayout l = xent_layout(dtype, n, vocab, feat_len, false);
  const int64_t need = (int64_t)(fits_map(dtype, weight_dev, weight_ld) ? l.total_in_place : l.total);
  if (!workspace_dev || ((uintptr_t)workspace_dev & 255) != 0 || workspace_bytes < need)
    return fail(FG_ERR_INVALID_ARGUMENT, "the workspace needs %lld bytes at a 256-byte boundary",
                (long long)need);
  const size_t es = dtype_size(dtype);
  if (results_overlap({array1d(loss_dev, n, 4), array1d(lse_dev, n, 4)},
                      {{feat_dev, n, feat_len, feat_ld, es}, {weight_dev, vocab, feat_len, weight_ld, es},
                       array1d(labels_dev, n, index_type == FG_INDEX_INT64 ? 8 : 4)}))
    return fail(FG_ERR_INVALID_ARGUMENT, "a result shares memory with an input or the other one");
  DeviceGuard guard(device);
  FG_CUDA_TRY(guard.status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace_dev);
  const Batch b = {labels_dev, index_type == FG_INDEX_INT64, n, vocab, feat_len, ignore_index, scale};
  int rc = FG_OK;
#define FG_LOSS(T)                                                                               \
  rc = loss_mma<T>(b, l, ws, static_cast<const T*>(feat_dev), feat_ld,                           \
                   static_cast<const T*>(weight_dev), weight_ld, dtype, loss_dev, lse_dev, status_dev, device, s)
  FG_DISPATCH_DTYPE(dtype, FG_LOSS)
#undef FG_LOSS
  return rc;
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
                          n, vocab, feat_len, scale, status_dev))
    return rc;
  if (!feat_grad_dev && !weight_grad_dev)
    return fail(FG_ERR_INVALID_ARGUMENT, "neither gradient is asked for");
  if ((((uintptr_t)feat_grad_dev | (uintptr_t)weight_grad_dev) % dtype_size(dtype)) != 0)
    return fail(FG_ERR_INVALID_ARGUMENT, "a gradient is not aligned to its type");
  if (n > 0) {
    if (!loss_grad_dev || !lse_dev || (((uintptr_t)loss_grad_dev | (uintptr_t)lse_dev) & 3) != 0)
      return fail(FG_ERR_INVALID_ARGUMENT, "null loss_grad or lse, or not aligned to float");
    const int64_t need = fg_softmax_xent_workspace_bytes(
        dtype, n, vocab, feat_len, 1 | (fits_map(dtype, weight_dev, weight_ld) ? FG_XENT_TABLE_IN_PLACE : 0));
    if (!workspace_dev || ((uintptr_t)workspace_dev & 255) != 0 || workspace_bytes < need)
      return fail(FG_ERR_INVALID_ARGUMENT, "the workspace needs %lld bytes at a 256-byte boundary",
                  (long long)need);
  }
  const size_t es = dtype_size(dtype);
  if (results_overlap({{feat_grad_dev, n, feat_len, feat_len, es}, {weight_grad_dev, vocab, feat_len, feat_len, es}},
                      {{feat_dev, n, feat_len, feat_ld, es}, {weight_dev, vocab, feat_len, weight_ld, es},
                       array1d(labels_dev, n, index_type == FG_INDEX_INT64 ? 8 : 4),
                       array1d(loss_grad_dev, n, 4), array1d(lse_dev, n, 4)}))
    return fail(FG_ERR_INVALID_ARGUMENT, "a result shares memory with an input or the other one");
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
  int rc = FG_OK;
#define FG_GRAD(T)                                                                              \
  rc = grad_mma<T>(b, l, ws, loss_grad_dev, static_cast<const T*>(feat_dev), feat_ld,           \
                   static_cast<const T*>(weight_dev), weight_ld, dtype, lse_dev,                \
                   static_cast<T*>(feat_grad_dev), static_cast<T*>(weight_grad_dev), status_dev, device, s)
  FG_DISPATCH_DTYPE(dtype, FG_GRAD)
#undef FG_GRAD
  return rc;
}
