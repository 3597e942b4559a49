// lcr_batch_attention: causal GQA attention of many sequences' rows over one
// paged cache. Work division and arithmetic are batch_attention.h's.
//
// Sizes in the measurements below are the largest of a ragged batch: the first
// chunk has all of the tokens named, others half to all, and caches have a third
// to all of the positions named.
//
// Few rows (at most 32): bound by the cache's bytes. The waves of a block share
// the rows and split the keys, 32 a step, each streaming its own keys and
// values into its own part of LDS with direct loads (no registers, no barrier):
// the next step's keys are requested as soon as the scores are taken, its values
// when the products are. Their results meet in LDS. 64 sequences over 0.7 GB of
// cache (head_dim 64, bf16) 115 us, 6.2 TB/s; a streaming read reaches 7.0.
// Many rows: bound by the exponentials (16 cycles each on the vector units) and,
// at head_dim 128, by LDS reads and the matrix cores. The waves share 64-key
// tiles, staged three or four deep, and split the rows, 32 each. A tile's scores
// are all taken before its first weights, so that products and exponentials of
// its halves overlap in a wave: 32 keys at a time were 3 to 15 % slower. Four
// chunks of 1000 tokens behind 4000 positions (110 GFLOP) 163 us, 0.68 PFLOP/s; the
// vector units are then busy for three quarters of it. Short prompts lose to
// the pieces' first loads and to partials: one of 2048 takes 47 us, 0.37.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "../kv_cache.h"
#include "batch_attention.h"

namespace lcr {
namespace {

using Args = BatchAttnArgs<KvCacheView>;
using KvPiece = Piece<elem_t>;

// ---------------------------------------------------------------------------
// Matrix-core kernels
// ---------------------------------------------------------------------------

// Blocks a compute unit, and waves a SIMD, follow from LDS and registers. At
// head_dim 64, three blocks of four waves (168 registers a lane); at 128, one of
// eight (256).
template <int kDim>
struct TiledShape {
  static constexpr int kHeadDim = kDim;
  static constexpr int kWaves = kHeadDim == 64 ? 4 : 8;
  static constexpr int kBlocks = kHeadDim == 64 ? 3 : 1;      // resident a compute unit
  // Of few rows, two: 64 sequences of 8000 positions 115 us, with three 116, and
  // shorter caches have fewer cuts (32 of 1000 in 16.0, 16.1).
  static constexpr int kFewBlocks = kHeadDim == 64 ? 2 : 1;
  static constexpr int kSimdWaves = kWaves * kBlocks / 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kTileRows = 32 * kWaves;               // packed rows of a tile of many rows
  static constexpr int kStages = kHeadDim == 64 ? 3 : 4;      // many rows: tiles staged
  static constexpr int kRowChunks = kHeadDim / 8;             // 16-byte chunks of a key
  static constexpr int kLoadRows = 64 / kRowChunks;           // keys of one 1 KiB direct load
  static constexpr int kSteps = kHeadDim / 32;                // k-steps of a score
  static constexpr int kDFrags = kHeadDim / 16;               // output fragments
  // elements of LDS: a wave's step (few) or a block's stages (many)
  static constexpr int kWaveElems = 2 * 32 * kHeadDim;
  static constexpr int kRingElems = kStages * 2 * 64 * kHeadDim;
  static_assert(kRingElems >= kWaves * kWaveElems, "both use the same LDS");
  // Few rows beside many: a step of 64 keys takes less than one of many rows, which
  // keeps the vector units busy while the cache is read. 16 sequences of one token
  // beside two chunks of 1000, with 64, 96, 128 and 192 keys a step: heads of 64 77,
  // 74, 74 and 79 us, of 128 121, 105, 95 and 90; 64 beside two of 512: 102, 95, 99
  // and 97, and 248, 184, 156 and 147.
  static constexpr int kFewStepKeys = kHeadDim == 64 ? 96 : 192;
  static constexpr bool kNeighbours = true;

  // A lane's first dim of k-step ks of a query, and of four neighbouring dims of its
  // outputs.
  static __device__ __forceinline__ int q_dim(int ks, int grp) { return 32 * ks + 8 * grp; }
  static __device__ __forceinline__ int out_dim(int n, int grp) { return 16 * n + 4 * grp; }
  static __device__ __forceinline__ mfma_acc4 out_piece(const mfma_acc4* o, int n) { return o[n]; }
};

template <int kHeadDim>
struct TiledLds {
  elem_t ring[TiledShape<kHeadDim>::kRingElems];
  float stats[TiledShape<kHeadDim>::kWaves][kFewRows][2];  // few rows: a wave's bases and sums
  uint32_t sums[TiledShape<kHeadDim>::kWaves];
  ShareStart found;
  int bad;  // a page outside the pool was read
  int special[2];  // many rows: the last tile of even and of odd number whose values hold infinities or NaN
};

// Keys and values in LDS.
template <int kHeadDim>
struct LdsTile {
  const elem_t* keys;
  const elem_t* values;

  __device__ __forceinline__ mfma_in8 key(int kf, int ks) const {
    const int col = lane_id() & 15;
    const int grp = lane_id() >> 4;
    return lds_operand(keys + (kf * 16 + col) * kHeadDim + (((ks * 4 + grp) ^ key_swizzle<kHeadDim>(col)) << 3));
  }
  __device__ __forceinline__ mfma_in8 value(int half, int df) const {
    return transposed_values<kHeadDim>(values, half, df, lane_id());
  }
};

// Keys are loaded in runs: kRun keys from a multiple of kRun on, by direct loads
// of kLoadRows keys each. With whole pages (page_size a multiple of 16) a run
// lies in one page, whose table entry is a scalar load; otherwise each lane reads
// its own key's, and waits for it with every tile load in flight. Keys past the
// last repeat it.
struct RunPage {
  int page;
  int slot;  // of the run's first key, within its page
};

template <int kRun>
__device__ __forceinline__ int run_start(int key, int last) {
  return min(key, last / kRun * kRun);
}

template <bool kWholePages, int kRun>
__device__ __forceinline__ RunPage find_run(const Args& a, const TiledPlan& plan, const KvPiece& p, int last,
                                            int key) {
  if constexpr (kWholePages) {
    typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
    const constant_ptr table = (constant_ptr)(reinterpret_cast<uintptr_t>(p.table));
    const int first = uniform(run_start<kRun>(key, last));
    const int index = plan.by_page(first);
    return RunPage{table[index], first - index * a.view.page_size};
  } else {
    return RunPage{0, 0};
  }
}

// The run of keys (or values) from key `key` on into rows row0 .. of a tile. Row
// r of LDS starts r rows behind the tile, in memory as in LDS, so the loads of a
// run differ by one offset that counts in both.
template <int kHeadDim, bool kWholePages, int kRun, bool kKeys, bool kStream>
__device__ __forceinline__ void load_run(const Args& a, const TiledPlan& plan, const KvPiece& p, int last,
                                         const RunPage& run, int& bad, elem_t* tile, int key, int row0) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kLoads = kRun / Shape::kLoadRows;
  constexpr int kLoadBytes = Shape::kLoadRows * kHeadDim * 2;
  static_assert(kLoadBytes == 1024 && kLoads <= 4, "offsets of 12 bits");
  const int load_row = lane_id() / Shape::kRowChunks;
  const int load_slot = lane_id() % Shape::kRowChunks;
  const elem_t* pool = kKeys ? p.keys : p.values;
  auto chunk = [&](int n) {
    const int row = row0 + n * Shape::kLoadRows + load_row;
    return 16u * static_cast<uint32_t>(load_slot ^ (kKeys ? key_swizzle<kHeadDim>(row) : value_swizzle<kHeadDim>(row)));
  };
  const uint32_t to = lds_address_of(tile + row0 * kHeadDim);
  if constexpr (kWholePages) {
    const int first = run_start<kRun>(key, last);
    const int page = pool_page(a, run.page, bad);
    const elem_t* from = pool + static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) +
                         static_cast<size_t>(static_cast<uint32_t>(run.slot)) * kHeadDim;
    if (last - first >= kRun - 1) {
      const uint32_t row_at = static_cast<uint32_t>(load_row * kHeadDim * 2);
      load_to_lds16<0, kStream>(from, row_at + chunk(0), to);
      if constexpr (kLoads > 1) load_to_lds16<kLoadBytes, kStream>(from, row_at + chunk(1), to);
      if constexpr (kLoads > 2) load_to_lds16<2 * kLoadBytes, kStream>(from, row_at + chunk(2), to);
      if constexpr (kLoads > 3) load_to_lds16<3 * kLoadBytes, kStream>(from, row_at + chunk(3), to);
    } else {
#pragma unroll 1
      for (int n = 0; n < kLoads; ++n) {
        const int row = min(n * Shape::kLoadRows + load_row, last - first);
        load_to_lds16<0, kStream>(from, static_cast<uint32_t>(row * kHeadDim * 2) + chunk(n), to + n * kLoadBytes);
      }
    }
  } else {
#pragma unroll 1
    for (int n = 0; n < kLoads; ++n) {
      const int at_key = min(key + n * Shape::kLoadRows + load_row, last);
      const int index = plan.by_page(at_key);
      const int page = pool_page(a, p.table[index], bad);
      const size_t at = static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) +
                        static_cast<size_t>(at_key - index * a.view.page_size) * kHeadDim;
      load_to_lds16(reinterpret_cast<const char*>(pool + at) + chunk(n), to + n * kLoadBytes);
    }
  }
}

// At most 32 rows: the waves split the keys.
template <int kHeadDim, bool kWholePages, int kRF, int kTileRows>
__device__ __forceinline__ void few_rows(TiledLds<kHeadDim>& lds, const Args& a, const TiledPlan& plan,
                                         const KvPiece& p) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kLoads = 32 / Shape::kLoadRows;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  elem_t* mine = lds.ring + wave * Shape::kWaveElems;
  elem_t* const key_tile = mine;
  elem_t* const value_tile = mine + 32 * kHeadDim;
  const LdsTile<kHeadDim> tile{key_tile, value_tile};
  const int tiles = (p.key1 - p.key0 + 31) / 32;
  const int count = tiles > wave ? (tiles - wave - 1) / Shape::kWaves + 1 : 0;
  const int last = p.key1 - 1;
  int bad = 0;
  auto first_key = [&](int t) { return p.key0 + 32 * (wave + Shape::kWaves * t); };
  struct StepPages {
    RunPage run[2];
  };
  auto pages_of = [&](int t) {
    return StepPages{{find_run<kWholePages, 16>(a, plan, p, last, first_key(t)),
                      find_run<kWholePages, 16>(a, plan, p, last, first_key(t) + 16)}};
  };
  auto issue = [&](auto is_keys, int t, const StepPages& pages) {
    constexpr bool kKeys = decltype(is_keys)::value;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      load_run<kHeadDim, kWholePages, 16, kKeys, true>(a, plan, p, last, pages.run[n], bad,
                                                       kKeys ? key_tile : value_tile, first_key(t) + 16 * n, 16 * n);
    }
  };
  using Keys = std::integral_constant<bool, true>;
  using Values = std::integral_constant<bool, false>;

  TiledRows<Shape, kRF> rows;
  rows.clear();
  if (count > 0) {
    load_rows(rows, a, plan, p, 0);
    const StepPages pages = pages_of(0);
    issue(Keys{}, 0, pages);
    issue(Values{}, 0, pages);
  }
  hold_rows(rows);
  const int all_seen = min(p.seen_first, p.key1);
  for (int t = 0; t < count; ++t) {
    const bool more = t + 1 < count;
    StepPages pages{};
    if (more) pages = pages_of(t + 1);
    loads_landed<kLoads>();  // step t's keys; behind them its values are in flight
    const int key0 = first_key(t);
    const bool whole = key0 + 32 <= all_seen;
    TileWork<Shape, kRF, 2> work;
    work.scores(rows, tile);
    lds_settled();  // the keys have been read
    if (more) issue(Keys{}, t + 1, pages);
    if (!whole) work.mask(rows, key0);
    work.raise_base(rows, plan.scale_log2e);
    work.weights(rows, plan.scale_log2e, 0);
    if (more) {
      loads_landed<kLoads>();  // step t's values; behind them the next keys
    } else {
      loads_landed<0>();
    }
    if (!whole && any_special(value_tile, 32 * kHeadDim / 512)) {
      work.mark_special(rows, tile, key0);
      clear_special(value_tile, 32 * kHeadDim / 512);
    }
    work.products(rows, tile, 0);
    lds_settled();
    if (more) issue(Values{}, t + 1, pages);
  }

  join_waves<Shape, kTileRows, Shape::kWaveElems / 2>(rows, bad, reinterpret_cast<float*>(lds.ring), lds.stats, a, plan,
                                                      p);
}

// Many rows: the waves split them, 32 each, and share the tiles. `tiles_done`:
// of the block's pieces before, so that a tile's number is its own.
template <int kHeadDim, bool kWholePages>
__device__ __forceinline__ void many_rows(TiledLds<kHeadDim>& lds, const Args& a, const TiledPlan& plan,
                                          const KvPiece& p, int& tiles_done) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kRF = 2;
  constexpr int kRun = 64 / Shape::kWaves;          // a wave's keys of a tile
  constexpr int kLoads = kRun / Shape::kLoadRows;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id();
  constexpr int kStageElems = 2 * 64 * kHeadDim;    // a tile's keys, then its values
  const int tiles = (p.key1 - p.key0 + 63) / 64;
  const int last = p.key1 - 1;
  int bad = 0;
  auto page_of = [&](int t) {
    return find_run<kWholePages, kRun>(a, plan, p, last, p.key0 + 64 * t + kRun * wave);
  };
  auto issue = [&](int t, elem_t* stage, const RunPage& page) {
    const int key = p.key0 + 64 * t + kRun * wave;
    load_run<kHeadDim, kWholePages, kRun, true, false>(a, plan, p, last, page, bad, stage, key, kRun * wave);
    load_run<kHeadDim, kWholePages, kRun, false, false>(a, plan, p, last, page, bad, stage + 64 * kHeadDim, key, kRun * wave);
  };
  if (threadIdx.x == 0) lds.bad = 0;

  const int row0 = 32 * wave;
  const bool active = row0 < p.rows;
  TiledRows<Shape, kRF> rows;
  rows.clear();
  int all_seen = 0, any_seen = 0;
  if (active) {
    load_rows(rows, a, plan, p, row0);
    all_seen = min(keys_seen(a, p.before, packed_token(plan, row0)), p.key1);
    any_seen = min(keys_seen(a, p.before, packed_token(plan, min(row0 + 31, p.rows - 1))), p.key1);
  }
  constexpr int kAhead = Shape::kStages - 1;
  if (tiles > 0) {
    RunPage first[kAhead];
#pragma unroll
    for (int t = 0; t < kAhead; ++t) first[t] = page_of(t);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      if (t < tiles) issue(t, lds.ring + t * kStageElems, first[t]);
    }
  }
  hold_rows(rows);
  elem_t* stage = lds.ring;                            // tile t's
  elem_t* next_stage = lds.ring + kAhead * kStageElems;  // tile t + kAhead's: the one before tile t's
  auto step = [&](elem_t* at) { return at == lds.ring + kAhead * kStageElems ? lds.ring : at + kStageElems; };
  for (int t = 0; t < tiles; ++t, stage = step(stage), next_stage = step(next_stage)) {
    RunPage page{0, 0};
    if (t + kAhead < tiles) page = page_of(t + kAhead);
    // This wave's loads of the tile have landed (the later tiles' remain);
    // behind the barrier every wave's have, and the tile before is free.
    if (t + kAhead - 1 < tiles) {
      loads_landed<(kAhead - 1) * 2 * kLoads>();
    } else {
      loads_landed<0>();
    }
    // A tile that some row of the unit does not see whole: each wave looks for
    // infinities and NaN among the values that it loaded. (In all of the tile's,
    // heads of 128 and a prompt of 133 tokens took 18.4 us for 14.6.) The next tile
    // of this tile's slot is looked at behind the next barrier, when every wave
    // has read the slot.
    const int tile0 = p.key0 + 64 * t;
    const bool partly = tile0 + 64 > p.seen_first;
    int* const slot = lds.special + ((tiles_done + t) & 1);
    if (partly) {
      const bool found = any_special(stage + (64 + kRun * wave) * kHeadDim, kRun * kHeadDim / 512);
      if (found && lane == 0) *slot = tiles_done + t;
      lds_settled();
    }
    plain_barrier();
    if (t + kAhead < tiles) issue(t + kAhead, next_stage, page);
    const bool special = partly && uniform(*slot) == tiles_done + t;
    const bool mine = tile0 < any_seen;
    const bool whole = tile0 + 64 <= all_seen;
    elem_t* values = stage + 64 * kHeadDim;
    const LdsTile<kHeadDim> tile{stage, values};
    if (mine) {
      TileWork<Shape, kRF, 4> work;
      work.scores(rows, tile);
      if (!whole) work.mask(rows, tile0);
      work.raise_base(rows, plan.scale_log2e);
      if (!special) {
        work.weights(rows, plan.scale_log2e, 0);
        work.products(rows, tile, 0);
        work.weights(rows, plan.scale_log2e, 1);
        work.products(rows, tile, 1);
      }
    }
    if (!special) continue;
    // Half a tile at a time, its scores once more: registers for the marks.
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      elem_t* at = values + half * 32 * kHeadDim;
      const LdsTile<kHeadDim> part{stage + half * 32 * kHeadDim, at};
      TileWork<Shape, kRF, 2> work;
      if (mine) {
        work.scores(rows, part);
        if (!whole) work.mask(rows, tile0 + 32 * half);
        work.weights(rows, plan.scale_log2e, 0);
        work.mark_special(rows, part, tile0 + 32 * half);
      }
      lds_settled();
      plain_barrier();
      static_assert(kHeadDim / 16 <= Shape::kWaves, "a wave clears one group of chunks at most");
      if (wave < kHeadDim / 16) clear_special(at + wave * 512, 1);
      lds_settled();
      plain_barrier();
      if (mine) work.products(rows, part, 0);
    }
  }
  tiles_done += max(tiles, 0);
  if (__any(bad != 0) && lane == 0) lds.bad = 1;
  __syncthreads();  // every wave is done with the tiles; the flag is set
  if (!active) return;
  rows.add_special();
  const bool spoilt = lds.bad != 0;
  store_rows(rows, spoilt, row0, a, plan, p);
}

// kMaxRows: packed rows a sequence may have, 16, 32 or any number (0).
template <int kHeadDim, int kMaxRows, bool kWholePages>
__global__ __launch_bounds__(TiledShape<kHeadDim>::kThreads, TiledShape<kHeadDim>::kSimdWaves) void batch_attention_kernel(
    Args args, TiledPlan tiled_plan) {
  using Shape = TiledShape<kHeadDim>;
  constexpr bool kMany = kMaxRows == 0;
  constexpr int kTileRows = kMany ? Shape::kTileRows : kFewRows;
  __shared__ __attribute__((aligned(1024))) TiledLds<kHeadDim> lds;
  Args a = args;
  a.view.page_size = own_register(a.view.page_size);
  a.view.page_stride = own_register(a.view.page_stride);
  a.pool_pages = own_register(a.pool_pages);
  a.held = own_register(a.held);
  a.group = own_register(a.group);
  TiledPlan plan = tiled_plan;
  plan.by_page.magic = own_register(plan.by_page.magic);
  plan.by_page.shift = own_register(plan.by_page.shift);
  plan.group_magic = own_register(plan.group_magic);
  plan.scale_log2e = own_register(plan.scale_log2e);

  // seen by every wave behind the barriers of the search for the share
  if (threadIdx.x == 0) lds.special[0] = lds.special[1] = -1;
  int tiles_done = 0;
  walk_share<Shape, kMany, elem_t>(
      a, plan, lds.sums, &lds.found, [](int) {},
      [&](const KvPiece& p) {
        few_rows<kHeadDim, kWholePages, kMaxRows == 16 ? 1 : 2, kTileRows>(lds, a, plan, p);
      },
      [&](const KvPiece& p) {
        if constexpr (kMany) many_rows<kHeadDim, kWholePages>(lds, a, plan, p, tiles_done);
      });
}

// ---------------------------------------------------------------------------
// Any head_dim up to 256, any alignment: a wave per (row, query head).
// ---------------------------------------------------------------------------

constexpr int kGenericWaves = 4;
constexpr int kGenericThreads = 64 * kGenericWaves;
constexpr int kGenericMaxDim = 256;

// Lane L of a 64-key tile takes key L's whole dot product; the tile's weights
// go through LDS, and lane L then holds elements L, L + 64, ... of the output.
// Nothing is shared between heads or rows and nothing split: the way for what the
// tiles above do not take, not for speed (64 sequences of up to 8000 positions,
// heads of 64: 4.2 ms).
__global__ __launch_bounds__(kGenericThreads) void batch_attention_generic_kernel(Args a) {
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
  // before the first sequence, or of one whose rows the buffer does not hold
  if (in_sequence < 0 || a.row_starts[b + 1] > a.tokens) return;
  const int head_dim = a.view.head_dim;
  const int kv = head / a.group;
  const long long position = static_cast<long long>(a.lengths[b]) - (a.row_starts[b + 1] - row);
  const int limit = in_sequence < a.max_new ? static_cast<int>(max(0ll, min(position + 1, static_cast<long long>(a.held)))) : 0;
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
    weights[wave][lane] = p;
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

template <int kHeadDim, int kMaxRows, bool kWholePages>
void launch_tiled_kernels(const Args& a, const TiledPlan& plan, hipStream_t s) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kTileRows = kMaxRows == 0 ? Shape::kTileRows : kFewRows;
  const unsigned blocks = static_cast<unsigned>(plan.shares) * static_cast<unsigned>(a.view.num_kv_heads);
  batch_attention_kernel<kHeadDim, kMaxRows, kWholePages><<<blocks, Shape::kThreads, 0, s>>>(a, plan);
  if (!plan.split) return;
  // A row is a chain of loads, so few follow each other: one time round for
  // many rows, two for few.
  constexpr bool kRowEach = kMaxRows == 0;
  const dim3 join(blocks, kRowEach ? kTileRows / (4 * 256 / kHeadDim) : kTileRows / 8);
  batch_attention_join_kernel<kHeadDim, kRowEach, Args><<<join, kJoinThreads, 0, s>>>(a, plan, kTileRows);
}

template <int kHeadDim>
void launch_tiled(const Args& a, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const TiledPlan plan = plan_tiled<TiledShape<kHeadDim>>(a, workspace, workspace_bytes);
  const long long most = static_cast<long long>(a.max_new) * a.group;
  if (a.view.page_size % 16 == 0) {
    if (most <= 16) {
      launch_tiled_kernels<kHeadDim, 16, true>(a, plan, s);
    } else if (most <= kFewRows) {
      launch_tiled_kernels<kHeadDim, 32, true>(a, plan, s);
    } else {
      launch_tiled_kernels<kHeadDim, 0, true>(a, plan, s);
    }
  } else if (most <= kFewRows) {
    launch_tiled_kernels<kHeadDim, 32, false>(a, plan, s);
  } else {
    launch_tiled_kernels<kHeadDim, 0, false>(a, plan, s);
  }
}

// The matrix-core kernels take a positive scale (the running maximum is the
// scores') and a group that fits a tile.
bool tiled_takes(const Args& a) {
  return (a.view.head_dim == 64 || a.view.head_dim == 128) &&
         a.group <= (a.view.head_dim == 64 ? TiledShape<64>::kTileRows : TiledShape<128>::kTileRows) &&
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
  const int kv_heads = std::max(1, num_heads / heads_per_kv);
  if (head_dim == 64) return tiled_workspace<TiledShape<64>>(max_new, kv_heads, heads_per_kv);
  if (head_dim == 128) return tiled_workspace<TiledShape<128>>(max_new, kv_heads, heads_per_kv);
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
  CAPI_CHECK(static_cast<long long>(table_stride) * view->page_size <= (1 << 30),
             "batch attention takes tables of up to 2^30 positions");
  CAPI_CHECK(view->page_stride >= 0 && view->head_stride >= 0, "batch attention needs non-negative cache strides");
  CAPI_CHECK(q_row_stride >= static_cast<long long>(num_heads) * view->head_dim,
             "query rows of " << num_heads << " heads cannot lie " << q_row_stride << " elements apart");
  CAPI_CHECK(tokens <= (1 << 30) && static_cast<long long>(tokens) * num_heads <= INT32_MAX,
             "batch attention takes up to 2^30 rows and 2^31 - 1 query heads in all");
  CAPI_CHECK(out != nullptr && q != nullptr && view->keys != nullptr && view->values != nullptr &&
                 row_starts != nullptr && lengths != nullptr,
             "batch attention needs its arrays");
  CAPI_CHECK(workspace != nullptr || workspace_bytes == 0,
             "batch attention workspace of " << workspace_bytes << " bytes has no pointer");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch attention workspace must be 16-byte aligned");
  Args a{static_cast<elem_t*>(out), static_cast<const elem_t*>(q), KvCacheView::from_c(*view), row_starts,
                  lengths, batch, tokens, max_new, num_heads, heads_per_kv, table_stride, pool_pages, q_row_stride,
                  table_stride * view->page_size, scale};
  auto s = static_cast<hipStream_t>(stream);
  const bool tiled = tiled_takes(a);
  // A launch has fewer than 2^32 threads in all.
  const long long units = static_cast<long long>(tokens) * num_heads;
  const long long blocks = !tiled ? (units + kGenericWaves - 1) / kGenericWaves
                           : view->num_kv_heads * (view->head_dim == 64 ? most_tiled_units<TiledShape<64>>(a) : most_tiled_units<TiledShape<128>>(a));
  const int threads = !tiled ? kGenericThreads : view->head_dim == 64 ? TiledShape<64>::kThreads : TiledShape<128>::kThreads;
  CAPI_CHECK(blocks * threads <= UINT32_MAX, "batch attention of " << tokens << " rows of " << num_heads
                                                                   << " heads needs more than 2^32 threads");
  if (tiled) {
    if (view->head_dim == 64) {
      launch_tiled<64>(a, workspace, workspace_bytes, s);
    } else {
      launch_tiled<128>(a, workspace, workspace_bytes, s);
    }
    CAPI_LAUNCHED();
    return LCR_OK;
  }
  batch_attention_generic_kernel<<<static_cast<unsigned>(blocks), kGenericThreads, 0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
