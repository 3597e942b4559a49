// lcr_batch_attention: causal GQA attention of many sequences' rows over one
// paged cache.
//
// Work. The query heads of a kv head share its keys, so the heads of a
// sequence's rows are packed: packed row r of a kv head is token r / group,
// head r % group. A unit is a tile of packed rows of one (kv head, sequence)
// over the keys they see: the whole sequence where that is at most 32 rows (one
// token, drafted tokens), else whole tokens up to 32 rows a wave. The units'
// keys, laid end to end in (kv head, sequence, tile) order, are cut into equal
// shares, one a block: every block has the same keys to read, whatever the
// sequences' lengths, and a unit that lies over a cut leaves a partial result
// (its exponent's base, sum and unnormalised output) in the workspace, at most
// two a block, which a second kernel joins. Each block finds its share from the
// sequences' lengths by itself (a prefix sum over the batch), so nothing is
// planned on the host and a captured call replays for other lengths. Blocks of
// one XCD (block id mod 8) take neighbouring shares: with eight kv heads an
// XCD's L2 holds one head's keys.
//
// Arithmetic. S^T = K . Q^T on 16x16x32 matrix instructions: a lane holds one
// packed row and four keys of each sixteen. One pass over the keys:
//   p = exp2(c s + b), c = scale log2 e, b = -(c m) for a running maximum m
//   l += p;  O^T += V^T . P^T
// A new m is taken when some p would pass 2^8, and l and O then move to the new
// base by exp2(b_new - b); a row's l and O always share one base, so its
// rounding cancels in O / l. p is rounded to the element type for the value
// product (the matrix cores take no wider operand beside 16-bit values: half a
// step of each weight, against two more products for a second half of p);
// everything else is fp32.
//
// Few rows (at most 32): bound by the cache's bytes. The waves of a block share
// the rows and split the keys, 32 a step, each streaming its own keys and
// values into its own part of LDS with direct loads (no registers, no barrier):
// the next step's keys are requested as soon as the scores are taken, its values
// when the products are. Their results meet in LDS.
// Many rows: bound by the exponentials and, at head_dim 128, by LDS reads and
// the matrix cores. The waves share 64-key tiles, staged four deep, and split
// the rows, 32 each.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "../kv_cache.h"
#include "device_common.h"
#include "kv_tiles.h"

namespace lcr {
namespace {

struct BatchAttnArgs {
  elem_t* out;
  const elem_t* q;
  KvCacheView view;
  const int32_t* row_starts;
  const int32_t* lengths;
  int batch;
  int tokens;
  int max_new;
  int num_heads;
  int group;
  int table_stride;
  int pool_pages;
  int q_row_stride;
  float scale;
};

// ---------------------------------------------------------------------------
// Work division
// ---------------------------------------------------------------------------

// What the matrix-core kernels need besides.
struct FlashPlan {
  uint32_t group_magic;   // r / group = r * group_magic >> 16 for r < 256
  uint32_t page_magic;    // key / page_size = mulhi(key, page_magic) >> page_shift
  int page_shift;
  int whole_pages;        // page_size is a multiple of a load's rows
  int tile_tokens;        // tokens of a tile of many rows
  int shares;             // blocks the keys are cut for; 0: a unit a block
  int min_share;          // keys
  float scale_log2e;
  long long* starts;      // [batch + 2] keys before each sequence, their total, and the share
  float* partials;        // [2 * shares][rows][head_dim], then [2 * shares][rows][2] bases and sums
};

constexpr int kFewRows = 32;
// Keys that a unit counts for besides its own: its queries, the join of the
// waves, the output.
constexpr int kUnitKeys = 64;
constexpr int kStepKeys = 64;  // shares are cut at multiples of this within a unit

// A sequence's share of the work, in tokens and keys of one kv head.
struct Sequence {
  int row0;      // first row
  int rows;      // as row_starts says
  int tokens;    // at most max_new
  int tiles;
  long long before;  // positions before its first row (may be negative)
  int visible;   // keys its last token sees
};

// Keys that token i of a sequence sees.
__device__ __forceinline__ int keys_seen(const BatchAttnArgs& a, long long before, int i) {
  const long long held = static_cast<long long>(a.table_stride) * a.view.page_size;
  return static_cast<int>(max(0ll, min(before + i + 1, held)));
}

__device__ __forceinline__ Sequence load_sequence(const BatchAttnArgs& a, const FlashPlan& plan, int b) {
  const int lo = a.row_starts[b], hi = a.row_starts[b + 1];
  const int length = a.lengths[b];
  Sequence s;
  s.row0 = lo;
  // starts that are no ascending rows of the buffer name no rows
  s.rows = lo >= 0 && hi > lo && hi <= a.tokens ? hi - lo : 0;
  s.tokens = min(s.rows, a.max_new);
  s.tiles = s.tokens * a.group <= kFewRows ? (s.rows > 0 ? 1 : 0) : (s.tokens - 1) / plan.tile_tokens + 1;
  s.before = static_cast<long long>(length) - s.rows;
  s.visible = s.tokens > 0 ? keys_seen(a, s.before, s.tokens - 1) : 0;
  return s;
}

// Keys the tiles before tile i count for: tile j sees up to
// visible - tokens + (j + 1) tile_tokens keys. An estimate above the keys that
// are seen (negative positions, the table's end) only leaves a share short.
__device__ __forceinline__ long long keys_before_tile(const FlashPlan& plan, const Sequence& s, int i) {
  if (plan.shares == 0) return i;
  const long long first = max(s.visible - s.tokens, 0);
  return i * (first + kUnitKeys) + static_cast<long long>(plan.tile_tokens) * i * (i + 1) / 2;
}

__device__ __forceinline__ long long sequence_keys(const FlashPlan& plan, const Sequence& s) {
  if (plan.shares == 0 || s.tiles == 0) return s.tiles;
  const int last = s.tiles - 1;
  return keys_before_tile(plan, s, last) + max(s.visible - s.tokens, 0) + s.tokens + kUnitKeys;
}

__device__ __forceinline__ long long share_of(const FlashPlan& plan, long long total, int kv_heads) {
  if (plan.shares == 0) return 1;
  const long long even = (total * kv_heads + plan.shares - 1) / plan.shares;
  return (max(even, static_cast<long long>(plan.min_share)) + kStepKeys - 1) / kStepKeys * kStepKeys;
}

struct ShareStart {
  long long total;      // keys of one kv head
  long long share;
  long long before;     // keys before the sequence
  int sequence;
};

// Where share `index` begins: the prefix sums of the sequences' keys, taken by
// the whole block. With `starts` they are written out for the join.
template <int kThreads>
__device__ __forceinline__ ShareStart find_share(const BatchAttnArgs& a, const FlashPlan& plan, long long index,
                                                 long long* starts, long long* lds_sums, ShareStart* lds_found) {
  constexpr int kWaves = kThreads / 64;
  const int t = threadIdx.x;
  const int per = (a.batch + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int k = 0; k < per; ++k) {
    const int b = t * per + k;
    if (b < a.batch) mine += sequence_keys(plan, load_sequence(a, plan, b));
  }
  long long to = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long other = __shfl_up(to, o, 64);
    if (lane_id() >= o) to += other;
  }
  if (lane_id() == 63) lds_sums[t >> 6] = to;
  if (t == 0) lds_found->sequence = -1;
  __syncthreads();
  long long total = 0, before = to - mine;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < (t >> 6)) before += lds_sums[w];
    total += lds_sums[w];
  }
  const long long share = share_of(plan, total, a.view.num_kv_heads);
  const long long at = index * share;
  const long long within = total > 0 && at < total * a.view.num_kv_heads ? at % total : -1;
  if (starts != nullptr || (within >= before && within < before + mine)) {
    for (int k = 0; k < per; ++k) {
      const int b = t * per + k;
      if (b >= a.batch) break;
      const long long keys = sequence_keys(plan, load_sequence(a, plan, b));
      if (starts != nullptr) starts[b] = before;
      if (within >= before && within < before + keys) *lds_found = ShareStart{total, share, before, b};
      before += keys;
    }
  }
  if (starts != nullptr && t == 0) {
    starts[a.batch] = total;
    starts[a.batch + 1] = share;
  }
  __syncthreads();
  return *lds_found;
}

// Waits for direct loads and for LDS reads, across which the compiler moves no
// memory access.
template <int kCount>
__device__ __forceinline__ void loads_landed() {
  asm volatile("" : : : "memory");
  wait_stage_landed<kCount>();
  asm volatile("" : : : "memory");
}
__device__ __forceinline__ void reads_returned() { loads_landed<63>(); }

// One block's part of a unit.
struct Piece {
  Sequence seq;
  const int32_t* table;
  int kv;
  int token0;      // first token of the tile
  int rows;        // packed rows
  int seen_first;  // keys that the tile's first and last token see
  int seen_last;
  int key0;        // keys [key0, key1)
  int key1;
  int slot;        // partial slot, or -1: the unit is whole
};

// ---------------------------------------------------------------------------
// Matrix-core kernels
// ---------------------------------------------------------------------------

template <int kHeadDim>
struct FlashShape {
  static constexpr int kWaves = kHeadDim == 64 ? 4 : 8;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kTileRows = 32 * kWaves;               // packed rows of a tile of many rows
  static constexpr int kSlots = kHeadDim == 64 ? 2 : 1;       // few rows: steps in flight a wave
  static constexpr int kStages = 4;                           // many rows: tiles staged
  static constexpr int kRowChunks = kHeadDim / 8;             // 16-byte chunks of a key
  static constexpr int kLoadRows = 64 / kRowChunks;           // keys of one 1 KiB direct load
  static constexpr int kSteps = kHeadDim / 32;                // k-steps of a score
  static constexpr int kDFrags = kHeadDim / 16;               // output fragments
  // elements of LDS: a wave's slots (few) or a block's stages (many)
  static constexpr int kWaveElems = kSlots * 2 * 32 * kHeadDim;
  static constexpr int kRingElems = kStages * 2 * 64 * kHeadDim;
  static_assert(kRingElems == kWaves * kWaveElems, "both use the same LDS");
};

template <int kHeadDim>
struct FlashLds {
  elem_t ring[FlashShape<kHeadDim>::kRingElems];
  float stats[FlashShape<kHeadDim>::kWaves][kFewRows][2];  // few rows: a wave's bases and sums
  long long sums[FlashShape<kHeadDim>::kWaves];
  ShareStart found;
  int bad;  // a page outside the pool was read
};

// A packed-row fragment's accumulators: rows 16 rf + col, per lane.
template <int kHeadDim, int kRF>
struct FlashRows {
  mfma_in8 q[kRF][FlashShape<kHeadDim>::kSteps];
  mfma_acc4 o[kRF][FlashShape<kHeadDim>::kDFrags];
  float base[kRF];  // +inf: no visible key yet
  float sum[kRF];   // of this lane's keys
  int seen[kRF];    // keys the row sees, at most key1

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      base[rf] = __builtin_huge_valf();
      sum[rf] = 0.0f;
#pragma unroll
      for (int df = 0; df < FlashShape<kHeadDim>::kDFrags; ++df) o[rf][df] = mfma_acc4{0.f, 0.f, 0.f, 0.f};
    }
  }
};

__device__ __forceinline__ int packed_token(const FlashPlan& plan, int r) {
  return static_cast<int>((static_cast<uint32_t>(r) * plan.group_magic) >> 16);
}

// Queries of packed rows row0 + 16 rf + col (those past the unit's rows repeat
// its last, are never stored and see what that one sees).
template <int kHeadDim, int kRF>
__device__ __forceinline__ void load_rows(FlashRows<kHeadDim, kRF>& rows, const BatchAttnArgs& a, const FlashPlan& plan,
                                          const Piece& p, int row0) {
  const int col = lane_id() & 15;
  const int grp = lane_id() >> 4;
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const int r = min(row0 + 16 * rf + col, p.rows - 1);
    const int token = packed_token(plan, r);
    const int head = p.kv * a.group + r - token * a.group;
    const elem_t* q = a.q + static_cast<size_t>(p.seq.row0 + p.token0 + token) * a.q_row_stride +
                      static_cast<size_t>(head) * kHeadDim + 8 * grp;
#pragma unroll
    for (int ks = 0; ks < FlashShape<kHeadDim>::kSteps; ++ks) rows.q[rf][ks] = as_operand(load16(q + 32 * ks));
    rows.seen[rf] = min(keys_seen(a, p.seq.before, p.token0 + token), p.key1);
  }
}

// 16 kKF keys of a tile against the rows: scores, weights, values.
//   keys, values  the tile in LDS
//   key0          its first key
//   all_seen      keys that every row of the wave sees
template <int kHeadDim, int kRF, int kKF>
struct TileWork {
  using Shape = FlashShape<kHeadDim>;
  mfma_acc4 s[kRF][kKF];
  uint32_t packed[kRF][kKF][2];

  __device__ __forceinline__ void scores(const FlashRows<kHeadDim, kRF>& rows, const elem_t* keys) {
    const int col = lane_id() & 15;
    const int grp = lane_id() >> 4;
#pragma unroll
    for (int kf = 0; kf < kKF; ++kf) {
#pragma unroll
      for (int rf = 0; rf < kRF; ++rf) s[rf][kf] = mfma_acc4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < Shape::kSteps; ++ks) {
        const mfma_in8 k =
            lds_operand(keys + (kf * 16 + col) * kHeadDim + (((ks * 4 + grp) ^ key_swizzle<kHeadDim>(col)) << 3));
#pragma unroll
        for (int rf = 0; rf < kRF; ++rf) s[rf][kf] = mfma16x16x32(k, rows.q[rf][ks], s[rf][kf]);
      }
    }
  }

  __device__ __forceinline__ void mask(const FlashRows<kHeadDim, kRF>& rows, int key0) {
    const int grp = lane_id() >> 4;
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      const int left = rows.seen[rf] - key0 - 4 * grp;
#pragma unroll
      for (int kf = 0; kf < kKF; ++kf) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (16 * kf + v >= left) s[rf][kf][v] = -__builtin_huge_valf();
        }
      }
    }
  }

  // The running statistics, and the weights rounded to the element type.
  __device__ __forceinline__ void weights(FlashRows<kHeadDim, kRF>& rows, float c) {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      float top = s[rf][0][0];
#pragma unroll
      for (int kf = 0; kf < kKF; ++kf) {
#pragma unroll
        for (int v = 0; v < 4; ++v) top = fmaxf(top, s[rf][kf][v]);
      }
      // c top + base: the largest weight's exponent (inf for a first visible
      // key, NaN, which compares false, while there is none)
      if (__any(__builtin_fmaf(top, c, rows.base[rf]) > 8.0f)) {
        top = fmaxf(top, xor_lane<16>(top));
        top = fmaxf(top, xor_lane<32>(top));
        if (__builtin_fmaf(top, c, rows.base[rf]) > 0.0f) {
          const float base = -(top * c);
          const float move = __builtin_amdgcn_exp2f(base - rows.base[rf]);
          rows.base[rf] = base;
          rows.sum[rf] *= move;
#pragma unroll
          for (int df = 0; df < Shape::kDFrags; ++df) rows.o[rf][df] *= move;
        }
      }
      // before the first visible key every score is -inf: against base 0
      const float base = rows.base[rf] == __builtin_huge_valf() ? 0.0f : rows.base[rf];
      float sum = 0.0f;
#pragma unroll
      for (int kf = 0; kf < kKF; ++kf) {
        float p[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rf][kf][v], c, base));
          sum += p[v];
        }
        packed[rf][kf][0] = pack_rounded(p[0], p[1]);
        packed[rf][kf][1] = pack_rounded(p[2], p[3]);
      }
      rows.sum[rf] += sum;
    }
  }

  __device__ __forceinline__ mfma_in8 weight_operand(int rf, int half) const {
    return as_operand(vec16{{packed[rf][2 * half][0], packed[rf][2 * half][1], packed[rf][2 * half + 1][0],
                             packed[rf][2 * half + 1][1]}});
  }

  __device__ __forceinline__ void products(FlashRows<kHeadDim, kRF>& rows, const elem_t* values, bool whole) {
#pragma unroll
    for (int half = 0; half < kKF / 2; ++half) {
#pragma unroll
      for (int df = 0; df < Shape::kDFrags; ++df) {
        mfma_in8 v = transposed_values<kHeadDim>(values, half, df, lane_id());
        if (!whole) v = without_special(rows, v, half, df);
#pragma unroll
        for (int rf = 0; rf < kRF; ++rf) rows.o[rf][df] = mfma16x16x32(v, weight_operand(rf, half), rows.o[rf][df]);
      }
    }
  }

  // For a tile that some row does not see whole. An infinity or NaN among its
  // values would reach, as 0 * inf in the matrix product, the rows that do not
  // see it. It is taken as 0 there, and a product with 1 in its place shows the
  // rows that do see it (weight above 0), which get it added; a NaN is added as
  // both infinities.
  __device__ __forceinline__ mfma_in8 without_special(FlashRows<kHeadDim, kRF>& rows, const mfma_in8& operand, int half,
                                                      int df) {
#if defined(LCR_ELEM_FP16)
    constexpr uint32_t kInf = 0x7c00u, kOne = 0x3c00u;
#else
    constexpr uint32_t kInf = 0x7f80u, kOne = 0x3f80u;
#endif
    vec16 v = __builtin_bit_cast(vec16, operand);
    bool special = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) special |= (v.w[i] & kInf) == kInf || ((v.w[i] >> 16) & kInf) == kInf;
    if (!__any(special)) return operand;
    vec16 up, down;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t kept = 0, plus = 0, minus = 0;
#pragma unroll
      for (int h = 0; h < 32; h += 16) {
        const uint32_t x = (v.w[i] >> h) & 0xffffu;
        const bool out = (x & kInf) == kInf;
        kept |= (out ? 0u : x) << h;
        plus |= (out && x != (0x8000u | kInf) ? kOne : 0u) << h;
        minus |= (out && x != kInf ? kOne : 0u) << h;
      }
      v.w[i] = kept;
      up.w[i] = plus;
      down.w[i] = minus;
    }
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      const mfma_acc4 zero{0.f, 0.f, 0.f, 0.f};
      const mfma_acc4 a = mfma16x16x32(as_operand(up), weight_operand(rf, half), zero);
      const mfma_acc4 b = mfma16x16x32(as_operand(down), weight_operand(rf, half), zero);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (a[e] > 0.0f) rows.o[rf][df][e] += __builtin_huge_valf();
        if (b[e] > 0.0f) rows.o[rf][df][e] -= __builtin_huge_valf();
      }
    }
    return as_operand(v);
  }
};

// Direct loads of kLoads groups of kLoadRows keys: group n of a call holds
// keys key_of(n) .. + kLoadRows - 1 (those past `last` repeat it). With whole
// pages a group lies in one page, whose table entry is a scalar load; a vector
// load of it would be waited for with every tile load in flight.
template <int kLoads>
struct LoadPages {
  int page[kLoads];
  int slot[kLoads];  // of the group's first key, within its page
};

template <int kHeadDim, int kLoads, typename KeyOf>
__device__ __forceinline__ LoadPages<kLoads> find_pages(const BatchAttnArgs& a, const FlashPlan& plan, const Piece& p,
                                                        int last, bool& bad, KeyOf key_of) {
  LoadPages<kLoads> pages;
  typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
  const constant_ptr table = (constant_ptr)(reinterpret_cast<uintptr_t>(p.table));
  constexpr int kLoadRows = FlashShape<kHeadDim>::kLoadRows;
#pragma unroll
  for (int n = 0; n < kLoads; ++n) {
    if (plan.whole_pages) {
      const int key = __builtin_amdgcn_readfirstlane(min(key_of(n), last / kLoadRows * kLoadRows));
      const int index = static_cast<int>(__umulhi(static_cast<uint32_t>(key), plan.page_magic) >> plan.page_shift);
      const int page = table[index];
      const bool inside = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pool_pages);
      bad |= !inside;
      pages.page[n] = inside ? page : 0;
      pages.slot[n] = key - index * a.view.page_size;
    } else {
      pages.page[n] = pages.slot[n] = 0;
    }
  }
  return pages;
}

template <int kHeadDim, int kLoads, bool kKeys, typename KeyOf, typename RowOf>
__device__ __forceinline__ void issue_loads(const BatchAttnArgs& a, const FlashPlan& plan, const Piece& p, int last,
                                            const LoadPages<kLoads>& pages, bool& bad, elem_t* tile, KeyOf key_of,
                                            RowOf row_of) {
  using Shape = FlashShape<kHeadDim>;
  const int load_row = lane_id() / Shape::kRowChunks;
  const int load_slot = lane_id() % Shape::kRowChunks;
  const elem_t* pool = kKeys ? a.view.keys : a.view.values;
  const size_t head_at = static_cast<size_t>(p.kv) * static_cast<size_t>(a.view.head_stride);
#pragma unroll
  for (int n = 0; n < kLoads; ++n) {
    const int row = row_of(n);  // of the tile, the group's first
    const int swizzle = kKeys ? key_swizzle<kHeadDim>(row + load_row) : value_swizzle<kHeadDim>(row + load_row);
    size_t at;
    if (plan.whole_pages) {
      const int first = min(key_of(n), last / Shape::kLoadRows * Shape::kLoadRows);
      at = static_cast<size_t>(pages.page[n]) * static_cast<size_t>(a.view.page_stride) + head_at +
           static_cast<size_t>((pages.slot[n] + min(load_row, last - first)) * kHeadDim);
    } else {
      const int key = min(key_of(n) + load_row, last);
      const int index = key / a.view.page_size;
      int page = p.table[index];
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pool_pages)) {
        bad = true;
        page = 0;
      }
      at = static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) + head_at +
           static_cast<size_t>(key - index * a.view.page_size) * kHeadDim;
    }
    load_to_lds16(pool + at + 8 * (load_slot ^ swizzle), lds_address_of(tile + row * kHeadDim));
  }
}

// One element's place in the output, from a packed row.
template <int kHeadDim>
__device__ __forceinline__ size_t out_at(const BatchAttnArgs& a, const FlashPlan& plan, const Piece& p, int r) {
  const int token = packed_token(plan, r);
  return (static_cast<size_t>(p.seq.row0 + p.token0 + token) * a.num_heads + p.kv * a.group + (r - token * a.group)) *
         kHeadDim;
}

template <int kHeadDim>
__device__ __forceinline__ float* partial_stats(const FlashPlan& plan, int tile_rows) {
  return plan.partials + static_cast<size_t>(2 * plan.shares) * tile_rows * kHeadDim;
}

// At most 32 rows: the waves split the keys.
template <int kHeadDim, int kRF, int kTileRows>
__device__ __forceinline__ void few_rows(FlashLds<kHeadDim>& lds, const BatchAttnArgs& a, const FlashPlan& plan,
                                         const Piece& p) {
  using Shape = FlashShape<kHeadDim>;
  constexpr int kLoads = 32 / Shape::kLoadRows;
  constexpr int kSlots = Shape::kSlots;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id();
  const int col = lane & 15;
  const int grp = lane >> 4;
  elem_t* mine = lds.ring + wave * Shape::kWaveElems;
  auto key_tile = [&](int t) { return mine + (t % kSlots) * (2 * 32 * kHeadDim); };
  auto value_tile = [&](int t) { return key_tile(t) + 32 * kHeadDim; };
  const int tiles = (p.key1 - p.key0 + 31) / 32;
  const int count = tiles > wave ? (tiles - wave - 1) / Shape::kWaves + 1 : 0;
  const int last = p.key1 - 1;
  bool bad = false;
  auto first_key = [&](int t) { return p.key0 + 32 * (wave + Shape::kWaves * t); };
  auto pages_of = [&](int t) {
    return find_pages<kHeadDim, kLoads>(a, plan, p, last, bad, [&](int n) { return first_key(t) + Shape::kLoadRows * n; });
  };
  auto issue = [&](auto is_keys, int t, const LoadPages<kLoads>& pages) {
    constexpr bool kKeys = decltype(is_keys)::value;
    issue_loads<kHeadDim, kLoads, kKeys>(a, plan, p, last, pages, bad, kKeys ? key_tile(t) : value_tile(t),
                                         [&](int n) { return first_key(t) + Shape::kLoadRows * n; },
                                         [&](int n) { return Shape::kLoadRows * n; });
  };
  using Keys = std::integral_constant<bool, true>;
  using Values = std::integral_constant<bool, false>;

  FlashRows<kHeadDim, kRF> rows;
  rows.clear();
  if (count > 0) {
    load_rows<kHeadDim, kRF>(rows, a, plan, p, 0);
#pragma unroll
    for (int t = 0; t < kSlots; ++t) {
      if (t < count) {
        const LoadPages<kLoads> pages = pages_of(t);
        issue(Keys{}, t, pages);
        issue(Values{}, t, pages);
      }
    }
  }
  const int all_seen = min(p.seen_first, p.key1);
  for (int t = 0; t < count; ++t) {
    const int left = count - 1 - t;
    const bool more = left >= kSlots;
    LoadPages<kLoads> pages{};
    if (more) pages = pages_of(t + kSlots);
    // In flight behind step t's keys: its values, and the later steps' both.
    if (kSlots > 1 && left > 0) {
      loads_landed<3 * kLoads>();
    } else {
      loads_landed<kLoads>();
    }
    const int key0 = first_key(t);
    const bool whole = key0 + 32 <= all_seen;
    TileWork<kHeadDim, kRF, 2> work;
    work.scores(rows, key_tile(t));
    reads_returned();  // the keys have been read
    if (more) issue(Keys{}, t + kSlots, pages);
    if (!whole) work.mask(rows, key0);
    work.weights(rows, plan.scale_log2e);
    // Behind step t's values: the later steps' keys and values.
    if (more) {
      loads_landed<(2 * (kSlots - 1) + 1) * kLoads>();
    } else if (kSlots > 1 && left > 0) {
      loads_landed<2 * kLoads>();
    } else {
      loads_landed<0>();
    }
    work.products(rows, value_tile(t), whole);
    reads_returned();
    if (more) issue(Values{}, t + kSlots, pages);
  }

  // The waves' results meet in LDS, each in its own (now free) part.
  if (__any(bad)) {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) rows.sum[rf] = __builtin_nanf("");
  }
  float* outputs = reinterpret_cast<float*>(mine);
  static_assert(Shape::kWaveElems * sizeof(elem_t) >= kFewRows * kHeadDim * sizeof(float), "a wave's outputs fit");
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    float sum = rows.sum[rf];
    sum += xor_lane<16>(sum);
    sum += xor_lane<32>(sum);
    if (grp == 0) {
      lds.stats[wave][16 * rf + col][0] = rows.base[rf];
      lds.stats[wave][16 * rf + col][1] = sum;
    }
#pragma unroll
    for (int df = 0; df < Shape::kDFrags; ++df) {
      *reinterpret_cast<mfma_acc4*>(outputs + (16 * rf + col) * kHeadDim + 16 * df + 4 * grp) = rows.o[rf][df];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.rows * (kHeadDim / 4); i += Shape::kThreads) {
    const int r = i / (kHeadDim / 4);
    const int d = i % (kHeadDim / 4) * 4;
    float base = lds.stats[0][r][0];
#pragma unroll
    for (int w = 1; w < Shape::kWaves; ++w) base = fminf(base, lds.stats[w][r][0]);
    float sum = 0.0f;
    mfma_acc4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < Shape::kWaves; ++w) {
      const float from = lds.stats[w][r][0];
      // a wave that saw no key has base +inf and nothing to add
      const float move = from == __builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(base - from);
      sum = __builtin_fmaf(lds.stats[w][r][1], move, sum);
      const mfma_acc4 x =
          *reinterpret_cast<const mfma_acc4*>(reinterpret_cast<const float*>(lds.ring + w * Shape::kWaveElems) +
                                              r * kHeadDim + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], move, o[e]);
    }
    if (p.slot >= 0) {
      *reinterpret_cast<mfma_acc4*>(plan.partials + (static_cast<size_t>(p.slot) * kTileRows + r) * kHeadDim + d) = o;
      if (d == 0) {
        float* stats = partial_stats<kHeadDim>(plan, kTileRows) + (static_cast<size_t>(p.slot) * kTileRows + r) * 2;
        stats[0] = base;
        stats[1] = sum;
      }
    } else {
      const int token = packed_token(plan, r);
      const bool any = keys_seen(a, p.seq.before, p.token0 + token) > 0;
      const float inv = any ? 1.0f / sum : 0.0f;
      uint2 words;
      words.x = any ? pack_elems(o[0] * inv, o[1] * inv) : 0u;
      words.y = any ? pack_elems(o[2] * inv, o[3] * inv) : 0u;
      *reinterpret_cast<uint2*>(a.out + out_at<kHeadDim>(a, plan, p, r) + d) = words;
    }
  }
  __syncthreads();  // the parts may be loaded into again
}

// Many rows: the waves split them, 32 each, and share the tiles.
template <int kHeadDim>
__device__ __forceinline__ void many_rows(FlashLds<kHeadDim>& lds, const BatchAttnArgs& a, const FlashPlan& plan,
                                          const Piece& p) {
  using Shape = FlashShape<kHeadDim>;
  constexpr int kRF = 2;
  constexpr int kLoads = 64 / Shape::kLoadRows / Shape::kWaves;  // a wave's, of keys or of values
  static_assert(kLoads * Shape::kLoadRows * Shape::kWaves == 64, "a tile splits over the waves");
  constexpr int kTileRows = Shape::kTileRows;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id();
  const int col = lane & 15;
  const int grp = lane >> 4;
  auto key_tile = [&](int t) { return lds.ring + (t % Shape::kStages) * (2 * 64 * kHeadDim); };
  auto value_tile = [&](int t) { return key_tile(t) + 64 * kHeadDim; };
  const int tiles = (p.key1 - p.key0 + 63) / 64;
  const int last = p.key1 - 1;
  bool bad = false;
  auto group_row = [&](int n) { return Shape::kLoadRows * (wave + Shape::kWaves * n); };
  auto pages_of = [&](int t) {
    return find_pages<kHeadDim, kLoads>(a, plan, p, last, bad, [&](int n) { return p.key0 + 64 * t + group_row(n); });
  };
  auto issue = [&](int t, const LoadPages<kLoads>& pages) {
    auto key_of = [&](int n) { return p.key0 + 64 * t + group_row(n); };
    issue_loads<kHeadDim, kLoads, true>(a, plan, p, last, pages, bad, key_tile(t), key_of, group_row);
    issue_loads<kHeadDim, kLoads, false>(a, plan, p, last, pages, bad, value_tile(t), key_of, group_row);
  };
  if (threadIdx.x == 0) lds.bad = 0;

  const int row0 = 32 * wave;
  const bool active = row0 < p.rows;
  FlashRows<kHeadDim, kRF> rows;
  rows.clear();
  int all_seen = 0, any_seen = 0;
  if (active) {
    load_rows<kHeadDim, kRF>(rows, a, plan, p, row0);
    all_seen = min(keys_seen(a, p.seq.before, p.token0 + packed_token(plan, row0)), p.key1);
    any_seen = min(keys_seen(a, p.seq.before, p.token0 + packed_token(plan, min(row0 + 31, p.rows - 1))), p.key1);
  }
  constexpr int kAhead = Shape::kStages - 1;
  if (tiles > 0) {
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      if (t < tiles) issue(t, pages_of(t));
    }
  }
  LoadPages<kLoads> pages{};
  if (kAhead < tiles) pages = pages_of(kAhead);
  for (int t = 0; t < tiles; ++t) {
    // This wave's loads of the tile have landed (the later tiles' remain);
    // behind the barrier every wave's have, and the tile before is free.
    if (t + kAhead - 1 < tiles) {
      wait_stage_landed<(kAhead - 1) * 2 * kLoads>();
    } else {
      wait_stage_landed<0>();
    }
    plain_barrier();
    if (t + kAhead < tiles) issue(t + kAhead, pages);
    if (t + kAhead + 1 < tiles) pages = pages_of(t + kAhead + 1);
    const int key0 = p.key0 + 64 * t;
    if (key0 < any_seen) {
      const bool whole = key0 + 64 <= all_seen;
      TileWork<kHeadDim, kRF, 4> work;
      work.scores(rows, key_tile(t));
      if (!whole) work.mask(rows, key0);
      work.weights(rows, plan.scale_log2e);
      work.products(rows, value_tile(t), whole);
    }
  }
  if (__any(bad) && lane == 0) lds.bad = 1;
  __syncthreads();  // every wave is done with the tiles; the flag is set
  if (!active) return;
  const bool spoilt = lds.bad != 0;
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const int r = row0 + 16 * rf + col;
    float sum = rows.sum[rf];
    sum += xor_lane<16>(sum);
    sum += xor_lane<32>(sum);
    if (spoilt) sum = __builtin_nanf("");
    if (r >= p.rows) continue;
    if (p.slot >= 0) {
      const size_t at = static_cast<size_t>(p.slot) * kTileRows + r;
#pragma unroll
      for (int df = 0; df < Shape::kDFrags; ++df) {
        *reinterpret_cast<mfma_acc4*>(plan.partials + at * kHeadDim + 16 * df + 4 * grp) = rows.o[rf][df];
      }
      if (grp == 0) {
        float* stats = partial_stats<kHeadDim>(plan, kTileRows) + at * 2;
        stats[0] = rows.base[rf];
        stats[1] = sum;
      }
    } else {
      const bool any = keys_seen(a, p.seq.before, p.token0 + packed_token(plan, r)) > 0;
      const float inv = any ? 1.0f / sum : 0.0f;
      elem_t* out = a.out + out_at<kHeadDim>(a, plan, p, r) + 4 * grp;
#pragma unroll
      for (int df = 0; df < Shape::kDFrags; ++df) {
        uint2 words;
        words.x = any ? pack_elems(rows.o[rf][df][0] * inv, rows.o[rf][df][1] * inv) : 0u;
        words.y = any ? pack_elems(rows.o[rf][df][2] * inv, rows.o[rf][df][3] * inv) : 0u;
        *reinterpret_cast<uint2*>(out + 16 * df) = words;
      }
    }
  }
}

// kMany: a sequence may have more than 32 packed rows.
template <int kHeadDim, bool kMany>
__global__ __launch_bounds__(FlashShape<kHeadDim>::kThreads, 2) void batch_attention_kernel(BatchAttnArgs a, FlashPlan plan) {
  using Shape = FlashShape<kHeadDim>;
  constexpr int kTileRows = kMany ? Shape::kTileRows : kFewRows;
  __shared__ __attribute__((aligned(1024))) FlashLds<kHeadDim> lds;
  // Share: neighbours on one XCD (a grid of shares is a multiple of 8).
  const long long index = plan.shares > 0
      ? static_cast<long long>(blockIdx.x % 8u) * (gridDim.x / 8u) + blockIdx.x / 8u
      : static_cast<long long>(blockIdx.x);
  const ShareStart found = find_share<Shape::kThreads>(
      a, plan, index, plan.shares > 0 && blockIdx.x == 0 ? plan.starts : nullptr, lds.sums, &lds.found);
  if (found.sequence < 0) return;
  const int kv_heads = a.view.num_kv_heads;
  const long long end = min((index + 1) * found.share, found.total * kv_heads);
  long long at = index * found.share;
  int kv = __builtin_amdgcn_readfirstlane(static_cast<int>(at / found.total));
  int b = __builtin_amdgcn_readfirstlane(found.sequence);
  Sequence seq = load_sequence(a, plan, b);
  long long before = kv * found.total + found.before;  // keys before the sequence
  // The tile that the share begins in: the last that starts at or before it.
  int tile = 0;
  for (int lo = 0, hi = seq.tiles - 1; lo < hi;) {
    const int mid = (lo + hi + 1) >> 1;
    if (before + keys_before_tile(plan, seq, mid) <= at) {
      lo = mid;
      tile = mid;
    } else {
      hi = mid - 1;
    }
  }
  while (at < end) {
    const long long start = before + keys_before_tile(plan, seq, tile);
    const long long keys = sequence_keys(plan, seq);
    const long long stop = tile + 1 < seq.tiles ? before + keys_before_tile(plan, seq, tile + 1) : before + keys;
    Piece p;
    p.seq = seq;
    p.table = a.view.page_table + static_cast<size_t>(b) * a.table_stride;
    p.kv = kv;
    const bool single = seq.tokens * a.group <= kFewRows;
    p.token0 = tile * plan.tile_tokens;
    const int tokens = single ? seq.tokens : min(plan.tile_tokens, seq.tokens - p.token0);
    p.rows = tokens * a.group;
    p.seen_first = keys_seen(a, seq.before, p.token0);
    p.seen_last = tokens > 0 ? keys_seen(a, seq.before, p.token0 + tokens - 1) : 0;
    // Cuts within the unit round up to whole steps, both shares alike.
    auto cut = [&](long long x) {
      const long long k = x <= start ? 0 : (x - start + kStepKeys - 1) / kStepKeys * kStepKeys;
      return static_cast<int>(min(k, static_cast<long long>(p.seen_last)));
    };
    p.slot = -1;
    if (plan.shares > 0 && (start < at || stop > end)) {
      p.slot = 2 * static_cast<int>(index) + (start < at ? 0 : 1);
      p.key0 = cut(at);
      p.key1 = stop > end ? cut(end) : p.seen_last;
    } else {
      p.key0 = 0;
      p.key1 = p.seen_last;
    }
    // Rows past max_new are zeros, written with the sequence's first tile's
    // first keys.
    if (tile == 0 && start >= at && seq.rows > seq.tokens) {
      const long long words = static_cast<long long>(seq.rows - seq.tokens) * a.group * (kHeadDim / 4);
      for (long long i = threadIdx.x; i < words; i += Shape::kThreads) {
        const long long r = i / (kHeadDim / 4);
        const long long token = r / a.group;
        const size_t row = static_cast<size_t>(seq.row0 + seq.tokens + token) * a.num_heads + kv * a.group +
                           static_cast<size_t>(r - token * a.group);
        *reinterpret_cast<uint2*>(a.out + row * kHeadDim + i % (kHeadDim / 4) * 4) = make_uint2(0u, 0u);
      }
    }
    if (p.rows > 0) {
      if (!single) {
        if constexpr (kMany) many_rows<kHeadDim>(lds, a, plan, p);
      } else if (p.rows <= 16) {
        few_rows<kHeadDim, 1, kTileRows>(lds, a, plan, p);
      } else {
        few_rows<kHeadDim, 2, kTileRows>(lds, a, plan, p);
      }
    }
    at = stop;
    if (at >= end) break;
    if (++tile >= seq.tiles) {
      tile = 0;
      before += keys;
      do {  // the next sequence that has rows, in this kv head or the next
        if (++b == a.batch) {
          b = 0;
          if (++kv == kv_heads) return;
        }
        seq = load_sequence(a, plan, b);
      } while (seq.tiles == 0);
    }
    if constexpr (kMany) __syncthreads();  // the tiles and the flag are free again
  }
}

// Joins the partials of each row whose unit lies over a cut: a block per token,
// a wave per head.
constexpr int kJoinThreads = 256;

template <int kHeadDim>
__global__ __launch_bounds__(kJoinThreads) void batch_attention_join_kernel(BatchAttnArgs a, FlashPlan plan,
                                                                           int tile_rows) {
  __shared__ int lds_count[kJoinThreads / 64];
  const int row = blockIdx.x;
  const int lane = lane_id();
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  // The row's sequence: the starts at or before it, counted.
  int below = 0;
  for (int i = threadIdx.x; i <= a.batch; i += kJoinThreads) below += a.row_starts[i] <= row ? 1 : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) lds_count[wave] = below;
  __syncthreads();
  below = 0;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 64; ++w) below += lds_count[w];
  const int b = below - 1;
  if (b < 0 || b >= a.batch) return;
  const Sequence seq = load_sequence(a, plan, b);
  const int i = row - seq.row0;
  if (i < 0 || i >= seq.tokens) return;
  const int seen = keys_seen(a, seq.before, i);
  const bool single = seq.tokens * a.group <= kFewRows;
  const int tile = single ? 0 : i / plan.tile_tokens;
  const int in_tile = single ? i : i - tile * plan.tile_tokens;
  const long long total = plan.starts[a.batch];
  const long long share = plan.starts[a.batch + 1];
  const long long first = plan.starts[b] + keys_before_tile(plan, seq, tile);
  const long long next = tile + 1 < seq.tiles ? plan.starts[b] + keys_before_tile(plan, seq, tile + 1)
                                              : plan.starts[b] + sequence_keys(plan, seq);
  const float* all_stats = partial_stats<kHeadDim>(plan, tile_rows);
  int last_kv = -1, from = 0, to = 0;
  for (int head = wave; head < a.num_heads; head += kJoinThreads / 64) {
    const int kv = head / a.group;
    if (kv != last_kv) {
      from = static_cast<int>((kv * total + first) / share);
      to = static_cast<int>((kv * total + next - 1) / share);
      last_kv = kv;
    }
    if (from == to) continue;
    const int r = in_tile * a.group + head - kv * a.group;
    auto slot = [&](int s) { return static_cast<size_t>(s == from ? 2 * s + 1 : 2 * s) * tile_rows + r; };
    float base = __builtin_huge_valf();
    for (int s = from + lane; s <= to; s += 64) base = fminf(base, all_stats[2 * slot(s)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) base = fminf(base, __shfl_xor(base, o, 64));
    float sum = 0.0f;
    float o[kHeadDim / 64] = {};
    for (int s = from; s <= to; ++s) {
      const float b_s = all_stats[2 * slot(s)], l_s = all_stats[2 * slot(s) + 1];
      const float move = b_s == __builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(base - b_s);
      sum = __builtin_fmaf(l_s, move, sum);
#pragma unroll
      for (int j = 0; j < kHeadDim / 64; ++j) {
        o[j] = __builtin_fmaf(plan.partials[slot(s) * kHeadDim + 64 * j + lane], move, o[j]);
      }
    }
    const float inv = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < kHeadDim / 64; ++j) {
      a.out[(static_cast<size_t>(row) * a.num_heads + head) * kHeadDim + 64 * j + lane] =
          float_to_elem(seen > 0 ? o[j] * inv : 0.0f);
    }
  }
}

// ---------------------------------------------------------------------------
// Any head_dim up to 256, any alignment: a wave per (row, query head).
// ---------------------------------------------------------------------------

constexpr int kGenericWaves = 4;
constexpr int kGenericThreads = 64 * kGenericWaves;
constexpr int kGenericMaxDim = 256;

// Lane L of a 64-key tile takes key L's whole dot product; the tile's weights
// go through LDS, and lane L then holds elements L, L + 64, ... of the output.
__global__ __launch_bounds__(kGenericThreads) void batch_attention_generic_kernel(BatchAttnArgs a) {
  constexpr int kDims = kGenericMaxDim / 64;
  __shared__ float q_lds[kGenericWaves][kGenericMaxDim];
  __shared__ float weights[kGenericWaves][64];
  __shared__ int32_t offsets_page[kGenericWaves][64];
  const int lane = lane_id();
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const long long unit = static_cast<long long>(blockIdx.x) * kGenericWaves + wave;
  const int row = static_cast<int>(unit / a.num_heads);
  const int head = static_cast<int>(unit - static_cast<long long>(row) * a.num_heads);
  if (row >= a.tokens) return;  // the wave; no block-wide barrier below
  int lo = 0, hi = a.batch;     // the last start at or before the row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.row_starts[mid] <= row) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  if (lo == a.batch) return;  // behind the last sequence
  const int b = lo;
  const int in_sequence = row - a.row_starts[b];
  const int head_dim = a.view.head_dim;
  const int kv = head / a.group;
  const long long position = static_cast<long long>(a.lengths[b]) - (a.row_starts[b + 1] - row);
  const long long held = static_cast<long long>(a.table_stride) * a.view.page_size;
  const int limit = in_sequence < a.max_new ? static_cast<int>(max(0ll, min(position + 1, held))) : 0;
  const int32_t* table = a.view.page_table + static_cast<size_t>(b) * a.table_stride;
  const elem_t* q = a.q + static_cast<size_t>(row) * a.q_row_stride + static_cast<size_t>(head) * head_dim;
  for (int i = lane; i < head_dim; i += 64) q_lds[wave][i] = elem_to_float(q[i]) * a.scale;
  const size_t head_at = static_cast<size_t>(kv) * static_cast<size_t>(a.view.head_stride);
  auto row_of = [&](int page, int key) {
    return static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) + head_at +
           static_cast<size_t>(key % a.view.page_size) * static_cast<size_t>(head_dim);
  };
  float m = kSoftmaxIdentity, l = 0.0f;
  float acc[kDims] = {};
  bool bad = false;
  for (int base = 0; base < limit; base += 64) {
    const int n = min(64, limit - base);
    float s = -__builtin_huge_valf();
    int page = 0;
    if (lane < n) {
      page = table[(base + lane) / a.view.page_size];
      if (page < 0 || page >= a.pool_pages) {
        bad = true;
        page = 0;
      }
    }
    offsets_page[wave][lane] = page;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (a.pool_pages > 0 && lane < n) {
      const elem_t* k = a.view.keys + row_of(page, base + lane);
      float d = 0.0f;
      for (int i = 0; i < head_dim; ++i) d = __builtin_fmaf(q_lds[wave][i], elem_to_float(k[i]), d);
      s = d;
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float keep = lcr_expf(m - m_new);
    const float p = lane < n ? lcr_expf(s - m_new) : 0.0f;
    m = m_new;
    l = l * keep + p;
    weights[wave][lane] = elem_to_float(float_to_elem(p));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int j = 0; j < kDims; ++j) acc[j] *= keep;
    for (int i = 0; i < n && a.pool_pages > 0; ++i) {
      const float w = weights[wave][i];
      const elem_t* v = a.view.values + row_of(offsets_page[wave][i], base + i);
#pragma unroll
      for (int j = 0; j < kDims; ++j) {
        if (lane + 64 * j < head_dim) acc[j] = __builtin_fmaf(w, elem_to_float(v[lane + 64 * j]), acc[j]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  l = wave_sum(l);
  float inv = limit > 0 ? 1.0f / l : 0.0f;
  if (__any(bad)) inv = __builtin_nanf("");
  elem_t* out = a.out + (static_cast<size_t>(row) * a.num_heads + head) * head_dim;
#pragma unroll
  for (int j = 0; j < kDims; ++j) {
    if (lane + 64 * j < head_dim) out[lane + 64 * j] = float_to_elem(acc[j] * inv);
  }
}

// The matrix-core kernels' shares: as many blocks as are resident at once.
template <int kHeadDim>
int flash_shares() {
  constexpr int kBlocksPerUnit = kHeadDim == 64 ? 2 : 1;
  return std::max(8, device_compute_units() * kBlocksPerUnit / 8 * 8);
}

bool many_rows_possible(int max_new, int group) { return static_cast<long long>(max_new) * group > kFewRows; }

template <int kHeadDim>
size_t flash_workspace(int batch, int max_new, int group) {
  const size_t rows = many_rows_possible(max_new, group) ? FlashShape<kHeadDim>::kTileRows : kFewRows;
  const size_t starts = align_up((static_cast<size_t>(batch) + 2) * sizeof(long long), 256);
  return starts + 2 * static_cast<size_t>(flash_shares<kHeadDim>()) * rows * (kHeadDim + 2) * sizeof(float);
}

template <int kHeadDim, bool kMany>
void launch_flash_kernels(const BatchAttnArgs& a, FlashPlan plan, hipStream_t s) {
  using Shape = FlashShape<kHeadDim>;
  if (plan.shares > 0) {
    batch_attention_kernel<kHeadDim, kMany><<<static_cast<unsigned>(plan.shares), Shape::kThreads, 0, s>>>(a, plan);
    batch_attention_join_kernel<kHeadDim>
        <<<static_cast<unsigned>(a.tokens), kJoinThreads, 0, s>>>(a, plan, kMany ? Shape::kTileRows : kFewRows);
    return;
  }
  // A unit a block: at most one short tile a sequence beside the full ones.
  const long long units = static_cast<long long>(a.tokens) / plan.tile_tokens + a.batch;
  batch_attention_kernel<kHeadDim, kMany>
      <<<static_cast<unsigned>(units * a.view.num_kv_heads), Shape::kThreads, 0, s>>>(a, plan);
}

template <int kHeadDim>
void launch_flash(const BatchAttnArgs& a, void* workspace, size_t workspace_bytes, hipStream_t s) {
  using Shape = FlashShape<kHeadDim>;
  FlashPlan plan{};
  plan.group_magic = static_cast<uint32_t>((65536 + a.group - 1) / a.group);
  const uint32_t page = static_cast<uint32_t>(a.view.page_size);
  plan.whole_pages = page % Shape::kLoadRows == 0 ? 1 : 0;
  if (plan.whole_pages) {
    // ceil(2^(31 + l) / page) with 2^l >= page: exact for keys below 2^31
    int l = 0;
    while ((1ull << l) < page) ++l;
    plan.page_magic = static_cast<uint32_t>(((1ull << (31 + l)) + page - 1) / page);
    plan.page_shift = l - 1;
  }
  plan.tile_tokens = std::max(1, Shape::kTileRows / a.group);
  plan.scale_log2e = static_cast<float>(static_cast<double>(a.scale) * 1.4426950408889634);
  plan.min_share = 256;
  const bool many = many_rows_possible(a.max_new, a.group);
  if (workspace != nullptr && workspace_bytes >= flash_workspace<kHeadDim>(a.batch, a.max_new, a.group)) {
    plan.shares = flash_shares<kHeadDim>();
    plan.starts = static_cast<long long*>(workspace);
    plan.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                             align_up((static_cast<size_t>(a.batch) + 2) * sizeof(long long), 256));
  }
  if (many) {
    launch_flash_kernels<kHeadDim, true>(a, plan, s);
  } else {
    launch_flash_kernels<kHeadDim, false>(a, plan, s);
  }
}

bool on_bytes(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The matrix-core kernels take a positive scale (the running maximum is the
// scores') and a group that fits a tile.
bool flash_takes(const BatchAttnArgs& a) {
  return (a.view.head_dim == 64 || a.view.head_dim == 128) &&
         a.group <= (a.view.head_dim == 64 ? FlashShape<64>::kTileRows : FlashShape<128>::kTileRows) &&
         a.scale > 0.0f && a.scale < 1e30f && a.q_row_stride % 8 == 0 && a.view.page_stride % 8 == 0 &&
         a.view.head_stride % 8 == 0 && on_bytes(a.q, 16) && on_bytes(a.out, 8) && on_bytes(a.view.keys, 16) &&
         on_bytes(a.view.values, 16);
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" size_t lcr_batch_attention_workspace_bytes(int batch, int tokens, int max_new, int num_heads,
                                                      int heads_per_kv, int head_dim) {
  if (batch <= 0 || tokens <= 0 || max_new <= 0 || num_heads <= 0 || heads_per_kv <= 0) return 0;
  if (head_dim == 64) return flash_workspace<64>(batch, max_new, heads_per_kv);
  if (head_dim == 128) return flash_workspace<128>(batch, max_new, heads_per_kv);
  return 0;
}

extern "C" int lcr_batch_attention(void* out, const void* q, const lcr_kv_view* view, const int32_t* row_starts,
                                   const int32_t* lengths, int batch, int tokens, int max_new, int num_heads,
                                   int heads_per_kv, int table_stride, int pool_pages, int q_row_stride, float scale,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  CAPI_CHECK(view != nullptr, "batch attention needs a cache view");
  CAPI_CHECK(batch >= 0 && tokens >= 0 && max_new >= 0 && num_heads >= 0, "batch attention needs non-negative sizes");
  CAPI_CHECK(batch <= LCR_BATCH_MAX_SEQUENCES,
             "batch attention takes up to " << LCR_BATCH_MAX_SEQUENCES << " sequences, got " << batch);
  if (batch == 0 || tokens == 0 || num_heads == 0) return LCR_OK;
  CAPI_CHECK(view->head_dim > 0 && view->head_dim <= kGenericMaxDim,
             "batch attention supports head_dim up to " << kGenericMaxDim << ", got " << view->head_dim);
  CAPI_CHECK(heads_per_kv > 0 && num_heads % heads_per_kv == 0 && num_heads / heads_per_kv == view->num_kv_heads,
             "num_heads (" << num_heads << ") must equal num_kv_heads (" << view->num_kv_heads
                           << ") times heads_per_kv (" << heads_per_kv << ")");
  CAPI_CHECK(view->page_table != nullptr, "a paged cache view needs a page table");
  CAPI_CHECK(view->page_size > 0, "a paged cache view needs a positive page size");
  CAPI_CHECK(table_stride > 0 && pool_pages > 0, "batch attention needs page tables and a pool of at least one page");
  CAPI_CHECK(static_cast<long long>(table_stride) * view->page_size <= INT32_MAX,
             "tables of " << table_stride << " pages of " << view->page_size << " hold positions past 32 bits");
  CAPI_CHECK(view->page_stride >= 0 && view->head_stride >= 0, "batch attention needs non-negative cache strides");
  CAPI_CHECK(q_row_stride >= static_cast<long long>(num_heads) * view->head_dim,
             "query rows of " << num_heads << " heads cannot lie " << q_row_stride << " elements apart");
  CAPI_CHECK(static_cast<long long>(tokens) * num_heads <= INT32_MAX,
             "batch attention takes up to 2^31 - 1 query heads in all");
  CAPI_CHECK(out != nullptr && q != nullptr && view->keys != nullptr && view->values != nullptr &&
                 row_starts != nullptr && lengths != nullptr,
             "batch attention needs its arrays");
  CAPI_CHECK(workspace != nullptr || workspace_bytes == 0,
             "batch attention workspace of " << workspace_bytes << " bytes has no pointer");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch attention workspace must be 16-byte aligned");
  BatchAttnArgs a{static_cast<elem_t*>(out), static_cast<const elem_t*>(q), KvCacheView::from_c(*view), row_starts,
                  lengths, batch, tokens, max_new, num_heads, heads_per_kv, table_stride, pool_pages, q_row_stride, scale};
  auto s = static_cast<hipStream_t>(stream);
  if (flash_takes(a)) {
    if (view->head_dim == 64) {
      launch_flash<64>(a, workspace, workspace_bytes, s);
    } else {
      launch_flash<128>(a, workspace, workspace_bytes, s);
    }
    CAPI_LAUNCHED();
    return LCR_OK;
  }
  const long long units = static_cast<long long>(tokens) * num_heads;
  batch_attention_generic_kernel<<<static_cast<unsigned>((units + kGenericWaves - 1) / kGenericWaves), kGenericThreads,
                                   0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
