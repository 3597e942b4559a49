// lcr_batch_attention_kv8: causal GQA attention of many sequences' rows over one
// paged cache of 8-bit numbers. Work division and arithmetic are
// batch_attention.h's; this is how the cache's numbers become operands.
//
// A number times its block's scale is a value of the element type (kv8.h), and one
// instruction makes two of them, so nothing is rounded on the way and the products
// are those of a 16-bit cache. The layout gives a lane what its operands need in
// 16 contiguous bytes: of keys 16 dims of one position, two k-steps' worth (queries
// are loaded in the same order of dims); of values four positions of four dims.
//
// Few rows (at most 32): bound by the cache's bytes. The waves of a block share the
// rows and split the keys, 32 a step. Keys and values go from memory to registers,
// where they are widened: no LDS and no barrier until the waves' results meet. A
// step's keys are loaded again as soon as its scores are taken, its values when the
// products are; more steps in flight were no faster. The loads are marked as read once:
// without that 64 sequences of 8000 positions took 73 us for 65. They take 62 for 0.36 GB
// (head_dim 64, bf16): 5.8 TB/s with the join of the cut units, and twice the bytes
// come at 7.4: 14 us are the launches, the search for the share, the first loads, and
// blocks that end 45 to 59 us in. Five sequences of 90000, heads of 128: 0.69 GB in
// 109 us, 6.4 TB/s; a streaming read reaches 7.0.
// Many rows: bound by the vector units (exponentials, their arguments and rounding).
// The waves share 64-key tiles and split the rows, 32 each. A wave loads its part of a
// tile, widens it and leaves it in LDS as the operands that all waves read, two tiles
// in turn. Four chunks of 1000 tokens behind 4000 positions (110 GFLOP) 147 us,
// 0.75 PFLOP/s.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../capi_util.h"
#include "batch_attention.h"
#include "kv8.h"

namespace lcr {
namespace {

using Args = BatchAttnArgs<Kv8View>;
using KvPiece = Piece<uint8_t>;

// ---------------------------------------------------------------------------
// Matrix-core kernels
// ---------------------------------------------------------------------------

// kMaxRows: packed rows a sequence may have, 16, 32 or any number (0).
template <int kDim, int kMaxRows>
struct Shape8 {
  // Few rows: two blocks of eight waves (head_dim 128: one). Four of four have more
  // cuts to join: 64 sequences of 8000 positions 63.2 and 61.8 us, 8 of 2000 13.8 and
  // 12.3; one of sixteen leaves 64 of 600 with 13.3 for 9.1. With more than 16 rows,
  // two of four, by registers.
  static constexpr bool kMany = kMaxRows == 0;
  static constexpr int kHeadDim = kDim;
  static constexpr int kWaves = kMaxRows == 16 || (kMany && kHeadDim == 128) ? 8 : 4;
  static constexpr int kThreads = 64 * kWaves;
  // resident a compute unit
  static constexpr int kBlocks = kHeadDim == 64 ? 3 : 1;
  static constexpr int kFewBlocks = kMaxRows == 16 && kHeadDim == 128 ? 1 : 2;
  static constexpr int kSimdWaves = kWaves * (kMany ? kBlocks : kFewBlocks) / 4;
  static constexpr int kTileRows = 32 * kWaves;     // packed rows of a tile of many rows
  static constexpr int kSteps = kHeadDim / 32;      // k-steps of a score
  static constexpr int kDFrags = kHeadDim / 16;     // output fragments
  static constexpr int kChunks = kHeadDim / 64;     // 16-byte chunks of a lane's in a block
  static constexpr int kBlockBytes = kKv8Block * kHeadDim;
  static constexpr int kTileElems = 2 * 64 * kHeadDim;  // many rows: a tile's keys, then its values
  static constexpr int kFewStepKeys = kHeadDim == 64 ? 96 : 192;
  // Few rows read each key once, and an XCD that reads one head alone loads some
  // memory channels more than others: 64 sequences of 8000 positions 65.5 us with
  // neighbouring shares on an XCD, 63.8 without.
  static constexpr bool kNeighbours = kMany;
  static constexpr bool kPaced = kMany && kBlocks > 1;  // blocks of a compute unit take turns (Pace)
  static constexpr int kFewStepBlocks = 2;          // few rows: blocks of a wave's step
  static constexpr int kFewFrags = kMaxRows == 16 ? 1 : 2;
  static constexpr int kWaveOutputs = 16 * kFewFrags * kHeadDim;

  // Chunk h of keys has dims 64 h + 16 grp .. + 15, k-steps 2 h and 2 h + 1.
  static __device__ __forceinline__ int q_dim(int ks, int grp) { return 64 * (ks >> 1) + 16 * grp + 8 * (ks & 1); }
  // Row m of output fragment 4 h + j is dim 64 h + 4 m + j, so that a lane's
  // 4 grp + e of four fragments are neighbours.
  static __device__ __forceinline__ int out_dim(int n, int grp) { return 64 * (n >> 2) + 16 * grp + 4 * (n & 3); }
  static __device__ __forceinline__ mfma_acc4 out_piece(const mfma_acc4* o, int n) {
    const mfma_acc4* f = o + (n & ~3);
    const int e = n & 3;
    return mfma_acc4{f[0][e], f[1][e], f[2][e], f[3][e]};
  }
};

template <typename Shape>
struct Lds8 {
  union {
    float outputs[Shape::kWaves * Shape::kWaveOutputs];  // few rows: the waves' results
    elem_t tiles[Shape::kMany ? 2 : 1][Shape::kMany ? Shape::kTileElems : 8];
  };
  // many rows: the NaN of a tile's values, a lane's words as it loaded them
  vec16 marks[Shape::kMany ? 2 : 1][Shape::kMany ? Shape::kThreads : 1];
  float stats[Shape::kWaves][kFewRows][2];  // few rows: a wave's bases and sums
  uint32_t sums[Shape::kWaves];
  ShareStart found;
  int bad;         // a page outside the pool was read
  int special[2];  // many rows: the last tile of even and of odd number whose values hold NaN
};

// The blocks of a compute unit take turns by how far they are. Waves that were there
// first are served first, so that of three blocks with equal shares the oldest was
// done after 107 us, the second after 137 and the third, at last alone, after 170
// (four chunks of 1000 tokens behind 4000 positions). A wave's priority falls when
// half of its share is done, and half of the rest, and half of that: the same
// chunks take 147 us for 158, and two of them beside 16 single tokens 66 for 72;
// falling by quarters 150 and 68.
struct Pace {
  int left = 0;   // steps of the share
  int next = 0;   // steps done at which the priority falls
  int level = 0;  // the priority; at 0 it stays

  __device__ __forceinline__ void begin(int steps) {
    left = steps;
    next = steps - (left >>= 1);
    level = 3;
    __builtin_amdgcn_s_setprio(3);
  }
  __device__ __forceinline__ void reached(int steps) {
    while (steps >= next && level > 0) {
      next += left - (left >> 1);
      left >>= 1;
      --level;
      if (level == 2) {
        __builtin_amdgcn_s_setprio(2);
      } else if (level == 1) {
        __builtin_amdgcn_s_setprio(1);
      } else {
        __builtin_amdgcn_s_setprio(0);
      }
    }
  }
};
// Of a call whose units are not cut, which begins none: a constant, so that it does
// not compile with a member left without a value.
constexpr Pace kUnpaced;

// Two neighbouring numbers of a word as elements.
template <bool kHigh>
__device__ __forceinline__ uint32_t widen_pair(uint32_t numbers, float scale) {
#if defined(LCR_ELEM_FP16)
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(numbers, scale, kHigh));
#else
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(numbers, scale, kHigh));
#endif
}

__device__ __forceinline__ mfma_in8 widen(uint32_t a, float scale_a, uint32_t b, float scale_b) {
  return as_operand(vec16{{widen_pair<false>(a, scale_a), widen_pair<true>(a, scale_a), widen_pair<false>(b, scale_b),
                           widen_pair<true>(b, scale_b)}});
}

// All bits of the bytes of a word of numbers that are NaN (0x7f, 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t marks = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (marks >> 7) * 0xffu;
}

// A word of four positions' numbers without those from `count` on.
__device__ __forceinline__ uint32_t first_numbers(int count) {
  return count >= 4 ? ~0u : (1u << (8 * max(count, 0))) - 1u;
}

typedef const __attribute__((address_space(4))) int32_t* constant_ints;
typedef const __attribute__((address_space(4))) float* constant_floats;

// Where 16 positions of a sequence lie: the same for the whole wave.
struct BlockPlace {
  int page;   // as the table has it
  int block;  // within the page
};

// Of the piece's keys 16 n .. 16 n + 15; blocks past the last repeat it.
__device__ __forceinline__ BlockPlace find_block(const Args& a, const TiledPlan& plan, const KvPiece& p, int n) {
  const constant_ints table = (constant_ints)(reinterpret_cast<uintptr_t>(p.table));
  const int at = uniform(min(n, (p.key1 - 1) / kKv8Block));
  const int index = plan.by_page(at * kKv8Block);
  return BlockPlace{table[index], at - index * (a.view.page_size / kKv8Block)};
}

// One chunk of a block's keys and values, as a lane loads them, and their scales.
struct BlockScales {
  float key;
  float value;
};

template <bool kStream>
__device__ __forceinline__ vec16 load_numbers(const uint8_t* base, uint32_t at) {
  if constexpr (kStream) {
    return load16_stream(base + at);
  } else {
    return load16(base + at);
  }
}

__device__ __forceinline__ BlockScales load_scales(const Args& a, const KvPiece& p, int page, int block) {
  const size_t at = a.view.scale_at(page, p.kv, block);
  return BlockScales{((constant_floats)(reinterpret_cast<uintptr_t>(a.view.key_scales)))[at],
                     ((constant_floats)(reinterpret_cast<uintptr_t>(a.view.value_scales)))[at]};
}

// A block's first byte in its page: in 64 bits, as a page may have more than 2^32.
template <typename Shape>
__device__ __forceinline__ size_t block_in_page(int block) {
  return static_cast<size_t>(static_cast<uint32_t>(block)) * Shape::kBlockBytes;
}

template <typename Shape>
__device__ __forceinline__ uint32_t key_chunk_at(int h) {
  return static_cast<uint32_t>((lane_id() & 15) * Shape::kHeadDim + 64 * h + 16 * (lane_id() >> 4));
}
template <typename Shape>
__device__ __forceinline__ uint32_t value_chunk_at(int h) {
  return static_cast<uint32_t>((lane_id() >> 4) * 4 * Shape::kHeadDim + 256 * h + 16 * (lane_id() & 15));
}

// A step's keys and their values in registers, a block of 16 beside the other.
template <typename Shape>
struct RawTile {
  static constexpr int kBlocks = Shape::kFewStepBlocks;
  vec16 keys[kBlocks][Shape::kChunks];
  vec16 values[kBlocks][Shape::kChunks];
  float key_scales[kBlocks];
  float value_scales[kBlocks];

  __device__ __forceinline__ mfma_in8 key(int kf, int ks) const {
    const vec16& c = keys[kf][ks >> 1];
    const int w = 2 * (ks & 1);
    return widen(c.w[w], key_scales[kf], c.w[w + 1], key_scales[kf]);
  }
  __device__ __forceinline__ mfma_in8 value(int half, int df) const {
    const int n = 2 * half;
    return widen(values[n][df >> 2].w[df & 3], value_scales[n], values[n + 1][df >> 2].w[df & 3], value_scales[n + 1]);
  }
};

// The values of a RawTile in LDS, a word of four positions at a time, for loops that
// are not unrolled.
template <typename Shape>
struct StashedValues {
  static constexpr int kBlocks = Shape::kFewStepBlocks;
  uint32_t* words;
  float scales[kBlocks];

  __device__ __forceinline__ StashedValues(const RawTile<Shape>& tile, float* lds)
      : words(reinterpret_cast<uint32_t*>(lds)) {
    static_assert(Shape::kWaveOutputs >= 64 * kBlocks * Shape::kDFrags, "a wave's values fit");
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      scales[n] = tile.value_scales[n];
#pragma unroll
      for (int df = 0; df < Shape::kDFrags; ++df) words[at(n, df)] = tile.values[n][df >> 2].w[df & 3];
    }
    lds_settled();
  }
  static __device__ __forceinline__ int at(int n, int df) { return (n * Shape::kDFrags + df) * 64 + lane_id(); }
  __device__ __forceinline__ mfma_in8 value(int half, int df) const {
    return widen(words[at(2 * half, df)], scales[2 * half], words[at(2 * half + 1, df)], scales[2 * half + 1]);
  }
};

// At most 32 rows: the waves split the keys.
template <typename Shape, int kTileRows>
__device__ __forceinline__ void few_rows(Lds8<Shape>& lds, const Args& a, const TiledPlan& plan, const KvPiece& p,
                                         Pace& pace) {
  constexpr int kRF = Shape::kFewFrags;
  constexpr int kBlocks = Shape::kFewStepBlocks;
  constexpr int kKeys = kKv8Block * kBlocks;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int tiles = (p.key1 - p.key0 + kKeys - 1) / kKeys;
  const int count = tiles > wave ? (tiles - wave - 1) / Shape::kWaves + 1 : 0;
  int bad = 0;
  auto first_key = [&](int t) { return p.key0 + kKeys * (wave + Shape::kWaves * t); };
  const size_t scales_at = static_cast<size_t>(p.kv) * static_cast<size_t>(a.view.scale_head_stride);
  const constant_floats key_scales = (constant_floats)(reinterpret_cast<uintptr_t>(a.view.key_scales + scales_at));
  const constant_floats value_scales = (constant_floats)(reinterpret_cast<uintptr_t>(a.view.value_scales + scales_at));
  struct Places {
    BlockPlace of[kBlocks];
  };
  auto places_of = [&](int t) {
    const int n0 = first_key(t) / kKv8Block;
    Places places;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) places.of[n] = find_block(a, plan, p, n0 + n);
    return places;
  };
  // Bytes from the kv head's first to each block, and its values' scale.
  struct ValuesAt {
    size_t of[kBlocks];
    float scales[kBlocks];
  };
  auto load_keys = [&](RawTile<Shape>& tile, const Places& places) {
    ValuesAt at;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const int page = pool_page(a, places.of[n].page, bad);
      const int block = places.of[n].block;
      at.of[n] = static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) + block_in_page<Shape>(block);
#pragma unroll
      for (int h = 0; h < Shape::kChunks; ++h) {
        tile.keys[n][h] = load_numbers<true>(p.keys + at.of[n], key_chunk_at<Shape>(h));
      }
      const size_t scale = static_cast<size_t>(page) * static_cast<size_t>(a.view.scale_page_stride) +
                           static_cast<size_t>(static_cast<uint32_t>(block));
      tile.key_scales[n] = key_scales[scale];
      at.scales[n] = value_scales[scale];
    }
    return at;
  };
  auto load_values = [&](RawTile<Shape>& tile, const ValuesAt& at) {
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      tile.value_scales[n] = at.scales[n];
#pragma unroll
      for (int h = 0; h < Shape::kChunks; ++h) {
        tile.values[n][h] = load_numbers<true>(p.values + at.of[n], value_chunk_at<Shape>(h));
      }
    }
  };

  TiledRows<Shape, kRF> rows;
  rows.clear();
  RawTile<Shape> tile;
  Places next{};
  if (count > 0) {
    const Places places = places_of(0);
    load_rows(rows, a, plan, p, 0);
    const ValuesAt at = load_keys(tile, places);
    load_values(tile, at);
    next = places_of(min(1, count - 1));
  }
  hold_rows(rows);
  const int all_seen = min(p.seen_first, p.key1);
  for (int t = 0; t < count; ++t) {
    const bool more = t + 1 < count;
    const int key0 = first_key(t);
    const bool whole = key0 + kKeys <= all_seen;
    if constexpr (Shape::kPaced) pace.reached(p.done + (key0 - p.key0) / Shape::kFewStepKeys);
    TileWork<Shape, kRF, kBlocks> work;
    work.scores(rows, tile);
    ValuesAt at{};
    if (more) {
      at = load_keys(tile, next);
      next = places_of(min(t + 2, count - 1));
    }
    if (!whole) work.mask(rows, key0);
    work.raise_base(rows, plan.scale_log2e);
#pragma unroll
    for (int half = 0; half < kBlocks / 2; ++half) work.weights(rows, plan.scale_log2e, half);
    if (!whole) {
      // numbers behind the last key that counts may be any
      bool found = false;
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) {
        const uint32_t keep = first_numbers(p.key1 - key0 - 16 * n - 4 * (lane_id() >> 4));
#pragma unroll
        for (int h = 0; h < Shape::kChunks; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            tile.values[n][h].w[i] &= keep;
            found |= nan_bytes(tile.values[n][h].w[i]) != 0;
          }
        }
      }
      if (__any(found)) {
        const StashedValues<Shape> values(tile, lds.outputs + wave * Shape::kWaveOutputs);
        work.mark_special(rows, values, key0);  // rows that see them get them at the end
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
          for (int h = 0; h < Shape::kChunks; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) tile.values[n][h].w[i] &= ~nan_bytes(tile.values[n][h].w[i]);
          }
        }
      }
    }
#pragma unroll
    for (int half = 0; half < kBlocks / 2; ++half) work.products(rows, tile, half);
    if (more) load_values(tile, at);
  }
  join_waves<Shape, kTileRows, Shape::kWaveOutputs>(rows, bad, lds.outputs, lds.stats, a, plan, p);
}

// 64 keys and their values as operands in LDS: lane by lane, 16 bytes each.
template <typename Shape>
struct OperandTile {
  const elem_t* tile;

  static __device__ __forceinline__ int key_at(int kf, int ks) { return ((kf * Shape::kSteps + ks) * 64 + lane_id()) * 8; }
  static __device__ __forceinline__ int value_at(int half, int df) {
    return 64 * Shape::kHeadDim + ((half * Shape::kDFrags + df) * 64 + lane_id()) * 8;
  }
  __device__ __forceinline__ mfma_in8 key(int kf, int ks) const { return lds_operand(tile + key_at(kf, ks)); }
  __device__ __forceinline__ mfma_in8 value(int half, int df) const { return lds_operand(tile + value_at(half, df)); }
};

// A tile's NaN as values, 0 elsewhere, from the waves' marks.
template <typename Shape>
struct MarkedValues {
  const vec16* marks;

  __device__ __forceinline__ mfma_in8 value(int half, int df) const {
    auto words = [&](int block) {
      return reinterpret_cast<const uint32_t*>(marks + (block * Shape::kChunks + (df >> 2)) * 64 + lane_id())[df & 3];
    };
    return widen(words(2 * half), 1.0f, words(2 * half + 1), 1.0f);
  }
};

// Many rows: the waves split them, 32 each, and share the tiles. `tiles_done`:
// of the block's pieces before, so that a tile's number is its own.
template <typename Shape>
__device__ __forceinline__ void many_rows(Lds8<Shape>& lds, const Args& a, const TiledPlan& plan, const KvPiece& p,
                                          Pace& pace, int& tiles_done) {
  constexpr int kRF = 2;
  static_assert(Shape::kWaves == 4 * Shape::kChunks, "a wave stages one chunk of one block of a tile");
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int my_block = wave / Shape::kChunks;
  const int my_chunk = wave % Shape::kChunks;
  const int tiles = (p.key1 - p.key0 + 63) / 64;
  int bad = 0;
  if (threadIdx.x == 0) lds.bad = 0;

  struct Raw {
    vec16 keys;
    vec16 values;
    BlockScales scales;
  };
  auto place_of = [&](int t) { return find_block(a, plan, p, (p.key0 + 64 * t) / kKv8Block + my_block); };
  auto load = [&](const BlockPlace& place) {
    const int page = pool_page(a, place.page, bad);
    const size_t at =
        static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) + block_in_page<Shape>(place.block);
    Raw raw;
    raw.keys = load_numbers<false>(p.keys + at, key_chunk_at<Shape>(my_chunk));
    raw.values = load_numbers<false>(p.values + at, value_chunk_at<Shape>(my_chunk));
    raw.scales = load_scales(a, p, page, place.block);
    return raw;
  };
  // Widens a wave's part of tile t and leaves it in LDS.
  auto stage = [&](int t, Raw& raw) {
    elem_t* tile = lds.tiles[t & 1];
    const int key0 = p.key0 + 64 * t + 16 * my_block;
    if (p.key0 + 64 * t + 64 > p.seen_first) {
      // A tile that some row of the unit does not see whole. Numbers behind the
      // last key that counts may be any; NaN would reach, as 0 * NaN, rows that do
      // not see them, and are left beside the tile for those that do.
      const uint32_t keep = first_numbers(p.key1 - key0 - 4 * (lane_id() >> 4));
      vec16 marks;
      bool found = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        marks.w[i] = nan_bytes(raw.values.w[i] & keep);
        raw.values.w[i] &= keep & ~marks.w[i];
        found |= marks.w[i] != 0;
      }
      lds.marks[t & 1][threadIdx.x] = marks;
      if (__any(found) && lane_id() == 0) lds.special[(tiles_done + t) & 1] = tiles_done + t;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<mfma_in8*>(tile + OperandTile<Shape>::key_at(my_block, 2 * my_chunk + i)) =
          widen(raw.keys.w[2 * i], raw.scales.key, raw.keys.w[2 * i + 1], raw.scales.key);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 four = make_uint2(widen_pair<false>(raw.values.w[i], raw.scales.value),
                                    widen_pair<true>(raw.values.w[i], raw.scales.value));
      *reinterpret_cast<uint2*>(tile + OperandTile<Shape>::value_at(my_block >> 1, 4 * my_chunk + i) +
                                4 * (my_block & 1)) = four;
    }
  };

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
  Raw raw{};
  BlockPlace next{};
  if (tiles > 0) {
    raw = load(place_of(0));
    const BlockPlace second = place_of(min(1, tiles - 1));
    next = place_of(min(2, tiles - 1));
    stage(0, raw);
    if (tiles > 1) raw = load(second);
  }
  hold_rows(rows);
  for (int t = 0; t < tiles; ++t) {
    // Behind the barrier tile t is staged, and the tile before has been read.
    lds_settled();
    plain_barrier();
    if constexpr (Shape::kPaced) pace.reached(p.done + t);
    if (t + 1 < tiles) {
      stage(t + 1, raw);
      if (t + 2 < tiles) {
        raw = load(next);
        next = place_of(min(t + 3, tiles - 1));
      }
    }
    const int tile0 = p.key0 + 64 * t;
    if (tile0 >= any_seen) continue;
    const bool whole = tile0 + 64 <= all_seen;
    const bool special = tile0 + 64 > p.seen_first && uniform(lds.special[(tiles_done + t) & 1]) == tiles_done + t;
    const OperandTile<Shape> tile{lds.tiles[t & 1]};
    TileWork<Shape, kRF, 4> work;
    work.scores(rows, tile);
    if (!whole) work.mask(rows, tile0);
    work.raise_base(rows, plan.scale_log2e);
    if (special) work.mark_special(rows, MarkedValues<Shape>{lds.marks[t & 1]}, tile0);
    work.weights(rows, plan.scale_log2e, 0);
    work.products(rows, tile, 0);
    work.weights(rows, plan.scale_log2e, 1);
    work.products(rows, tile, 1);
  }
  tiles_done += max(tiles, 0);
  if (__any(bad != 0) && lane_id() == 0) lds.bad = 1;
  __syncthreads();  // every wave is done with the tiles; the flag is set
  if (!active) return;
  rows.add_special();
  store_rows(rows, lds.bad != 0, row0, a, plan, p);
}

template <typename Shape>
__global__ __launch_bounds__(Shape::kThreads, Shape::kSimdWaves) void batch_attention_kv8_kernel(Args args,
                                                                                               TiledPlan tiled_plan) {
  constexpr bool kMany = Shape::kMany;
  constexpr int kTileRows = kMany ? Shape::kTileRows : kFewRows;
  __shared__ __attribute__((aligned(1024))) Lds8<Shape> lds;
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
  Pace pace = kUnpaced;
  walk_share<Shape, kMany, uint8_t>(
      a, plan, lds.sums, &lds.found, [&](int steps) { if (Shape::kPaced && plan.split) pace.begin(steps); },
      [&](const KvPiece& p) { few_rows<Shape, kTileRows>(lds, a, plan, p, pace); },
      [&](const KvPiece& p) {
        if constexpr (kMany) many_rows<Shape>(lds, a, plan, p, pace, tiles_done);
      });
}

// ---------------------------------------------------------------------------
// Any head_dim that is a multiple of 16 up to 256: a wave per (row, query head).
// ---------------------------------------------------------------------------

constexpr int kGenericWaves = 4;
constexpr int kGenericThreads = 64 * kGenericWaves;
constexpr int kGenericMaxDim = 256;

// Lane L of a 64-key tile takes key L's whole dot product; the tile's weights, with
// their scales, go through LDS, and lane L then holds elements L, L + 64, ... of
// the output. Nothing is shared between heads or rows and nothing split: the way
// for what the tiles above do not take, not for speed.
__global__ __launch_bounds__(kGenericThreads) void batch_attention_kv8_generic_kernel(Args a) {
  constexpr int kDims = kGenericMaxDim / 64;
  __shared__ float q_lds[kGenericWaves][kGenericMaxDim];
  __shared__ float weights[kGenericWaves][64];
  __shared__ int32_t pages[kGenericWaves][64];
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
  const int d = a.view.head_dim;
  const int kv = head / a.group;
  const long long position = static_cast<long long>(a.lengths[b]) - (a.row_starts[b + 1] - row);
  const int limit = in_sequence < a.max_new ? static_cast<int>(max(0ll, min(position + 1, static_cast<long long>(a.held)))) : 0;
  const int32_t* table = a.view.page_table + static_cast<size_t>(b) * a.table_stride;
  const elem_t* q = a.q + static_cast<size_t>(row) * a.q_row_stride + static_cast<size_t>(head) * d;
  for (int i = lane; i < d; i += 64) q_lds[wave][i] = elem_to_float(q[i]) * a.scale;
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
    pages[wave][lane] = page;
    wave_settled();
    const int slot = (base + lane) % a.view.page_size;
    if (lane < n) {
      const uint8_t* k = a.view.keys + a.view.block_at(page, kv, slot / kKv8Block);
      float dot = 0.0f;
      for (int i = 0; i < d; ++i) {
        dot = __builtin_fmaf(q_lds[wave][i], kv8_number(k[kv8_key_byte(d, slot % kKv8Block, i)]), dot);
      }
      s = dot * a.view.key_scales[a.view.scale_at(page, kv, slot / kKv8Block)];
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float keep = lcr_expf(m - m_new);
    const float p = lane < n ? lcr_expf(s - m_new) : 0.0f;
    m = m_new;
    l = l * keep + p;
    weights[wave][lane] = lane < n ? p * a.view.value_scales[a.view.scale_at(page, kv, slot / kKv8Block)] : 0.0f;
    wave_settled();
#pragma unroll
    for (int j = 0; j < kDims; ++j) acc[j] *= keep;
    for (int i = 0; i < n; ++i) {
      const float w = weights[wave][i];
      const int at = (base + i) % a.view.page_size;
      const uint8_t* v = a.view.values + a.view.block_at(pages[wave][i], kv, at / kKv8Block);
#pragma unroll
      for (int j = 0; j < kDims; ++j) {
        if (lane + 64 * j < d) {
          acc[j] = __builtin_fmaf(w, kv8_number(v[kv8_value_byte(d, at % kKv8Block, lane + 64 * j)]), acc[j]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  l = wave_sum(l);
  float inv = limit > 0 ? 1.0f / l : 0.0f;
  if (__any(bad)) inv = __builtin_nanf("");
  elem_t* out = a.out + (static_cast<size_t>(row) * a.num_heads + head) * d;
#pragma unroll
  for (int j = 0; j < kDims; ++j) {
    if (lane + 64 * j < d) out[lane + 64 * j] = float_to_elem(acc[j] * inv);
  }
}

// A launch has fewer than 2^32 threads in all.
int check_threads(const Args& a, long long blocks, int threads) {
  CAPI_CHECK(blocks * threads <= UINT32_MAX, "batch attention of " << a.tokens << " rows of " << a.num_heads
                                                                   << " heads needs more than 2^32 threads");
  return LCR_OK;
}

template <int kHeadDim, int kMaxRows>
int launch_tiled(const Args& a, void* workspace, size_t workspace_bytes, hipStream_t s) {
  using Shape = Shape8<kHeadDim, kMaxRows>;
  constexpr int kTileRows = kMaxRows == 0 ? Shape::kTileRows : kFewRows;
  const TiledPlan plan = plan_tiled<Shape>(a, workspace, workspace_bytes);
  const int status = check_threads(a, static_cast<long long>(plan.shares) * a.view.num_kv_heads, Shape::kThreads);
  if (status != LCR_OK) return status;
  const unsigned blocks = static_cast<unsigned>(plan.shares) * static_cast<unsigned>(a.view.num_kv_heads);
  batch_attention_kv8_kernel<Shape><<<blocks, Shape::kThreads, 0, s>>>(a, plan);
  if (!plan.split) return LCR_OK;
  // A row is a chain of loads, so none follows another.
  constexpr bool kRowEach = kMaxRows == 0;
  const int few_rows = static_cast<int>(std::min<long long>(static_cast<long long>(a.max_new) * a.group, kFewRows));
  const dim3 join(blocks, kRowEach ? kTileRows / (4 * 256 / kHeadDim) : (few_rows + 3) / 4);
  batch_attention_join_kernel<kHeadDim, kRowEach, Args><<<join, kJoinThreads, 0, s>>>(a, plan, kTileRows);
  return LCR_OK;
}

template <int kHeadDim>
int launch_tiled(const Args& a, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const long long most = static_cast<long long>(a.max_new) * a.group;
  if (most <= 16) return launch_tiled<kHeadDim, 16>(a, workspace, workspace_bytes, s);
  if (most <= kFewRows) return launch_tiled<kHeadDim, 32>(a, workspace, workspace_bytes, s);
  return launch_tiled<kHeadDim, 0>(a, workspace, workspace_bytes, s);
}

// The matrix-core kernels take a positive scale (the running maximum is the
// scores') and a group that fits a tile.
bool tiled_takes(const Args& a) {
  return (a.view.head_dim == 64 || a.view.head_dim == 128) &&
         a.group <= (a.view.head_dim == 64 ? Shape8<64, 0>::kTileRows : Shape8<128, 0>::kTileRows) && a.scale > 0.0f &&
         a.scale < 1e30f && a.q_row_stride % 8 == 0 && on_bytes(a.q, 16) && on_bytes(a.out, 8);
}

template <int kHeadDim>
size_t workspace_for(int max_new, int kv_heads, int group) {
  const long long most = static_cast<long long>(max_new) * group;
  if (most <= 16) return tiled_workspace<Shape8<kHeadDim, 16>>(max_new, kv_heads, group);
  if (most <= kFewRows) return tiled_workspace<Shape8<kHeadDim, 32>>(max_new, kv_heads, group);
  return tiled_workspace<Shape8<kHeadDim, 0>>(max_new, kv_heads, group);
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" size_t lcr_batch_attention_kv8_workspace_bytes(int batch, int tokens, int max_new, int num_heads,
                                                          int heads_per_kv, int head_dim) {
  if (batch <= 0 || tokens <= 0 || max_new <= 0 || num_heads <= 0 || heads_per_kv <= 0) return 0;
  const int kv_heads = std::max(1, num_heads / heads_per_kv);
  if (head_dim == 64) return workspace_for<64>(max_new, kv_heads, heads_per_kv);
  if (head_dim == 128) return workspace_for<128>(max_new, kv_heads, heads_per_kv);
  return 0;
}

extern "C" int lcr_batch_attention_kv8(void* out, const void* q, const lcr_kv8_view* view, const int32_t* row_starts,
                                       const int32_t* lengths, int batch, int tokens, int max_new, int num_heads,
                                       int heads_per_kv, int table_stride, int pool_pages, int q_row_stride,
                                       float scale, void* workspace, size_t workspace_bytes, void* stream) {
  CAPI_CHECK(view != nullptr, "batch attention needs a cache view");
  CAPI_CHECK(batch >= 0 && tokens >= 0 && max_new >= 0 && num_heads >= 0, "batch attention needs non-negative sizes");
  CAPI_CHECK(batch <= LCR_BATCH_MAX_SEQUENCES,
             "batch attention takes up to " << LCR_BATCH_MAX_SEQUENCES << " sequences, got " << batch);
  if (batch == 0 || tokens == 0 || num_heads == 0) return LCR_OK;
  CAPI_CHECK(view->head_dim > 0 && view->head_dim % 16 == 0 && view->head_dim <= kGenericMaxDim,
             "an 8-bit cache has a head_dim that is a multiple of 16 up to " << kGenericMaxDim << ", got "
                                                                             << view->head_dim);
  CAPI_CHECK(heads_per_kv > 0 && num_heads % heads_per_kv == 0 && num_heads / heads_per_kv == view->num_kv_heads,
             "num_heads (" << num_heads << ") must equal num_kv_heads (" << view->num_kv_heads
                           << ") times heads_per_kv (" << heads_per_kv << ")");
  CAPI_CHECK(view->page_table != nullptr, "a paged cache view needs a page table");
  CAPI_CHECK(view->page_size > 0 && view->page_size % kKv8Block == 0,
             "an 8-bit cache view needs pages of a multiple of " << kKv8Block << " positions, got " << view->page_size);
  CAPI_CHECK(table_stride > 0 && pool_pages > 0, "batch attention needs page tables and a pool of at least one page");
  CAPI_CHECK(static_cast<long long>(table_stride) * view->page_size <= (1 << 30),
             "batch attention takes tables of up to 2^30 positions");
  CAPI_CHECK(view->page_stride >= 0 && view->head_stride >= 0 && view->scale_page_stride >= 0 &&
                 view->scale_head_stride >= 0 && view->page_stride % 16 == 0 && view->head_stride % 16 == 0,
             "an 8-bit cache has non-negative strides, of its numbers in multiples of 16 bytes");
  CAPI_CHECK(q_row_stride >= static_cast<long long>(num_heads) * view->head_dim,
             "query rows of " << num_heads << " heads cannot lie " << q_row_stride << " elements apart");
  CAPI_CHECK(tokens <= (1 << 30) && static_cast<long long>(tokens) * num_heads <= INT32_MAX,
             "batch attention takes up to 2^30 rows and 2^31 - 1 query heads in all");
  CAPI_CHECK(out != nullptr && q != nullptr && view->keys != nullptr && view->values != nullptr &&
                 view->key_scales != nullptr && view->value_scales != nullptr && row_starts != nullptr &&
                 lengths != nullptr,
             "batch attention needs its arrays");
  CAPI_CHECK(((reinterpret_cast<uintptr_t>(view->keys) | reinterpret_cast<uintptr_t>(view->values)) & 15u) == 0,
             "an 8-bit cache's numbers must be 16-byte aligned");
  CAPI_CHECK(workspace != nullptr || workspace_bytes == 0,
             "batch attention workspace of " << workspace_bytes << " bytes has no pointer");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch attention workspace must be 16-byte aligned");
  Args a{static_cast<elem_t*>(out), static_cast<const elem_t*>(q), Kv8View::from_c(*view), row_starts,
                   lengths, batch, tokens, max_new, num_heads, heads_per_kv, table_stride, pool_pages, q_row_stride,
                   table_stride * view->page_size, scale};
  auto s = static_cast<hipStream_t>(stream);
  if (tiled_takes(a)) {
    const int status = view->head_dim == 64 ? launch_tiled<64>(a, workspace, workspace_bytes, s)
                                            : launch_tiled<128>(a, workspace, workspace_bytes, s);
    if (status != LCR_OK) return status;
  } else {
    const long long units = static_cast<long long>(tokens) * num_heads;
    const long long blocks = (units + kGenericWaves - 1) / kGenericWaves;
    const int status = check_threads(a, blocks, kGenericThreads);
    if (status != LCR_OK) return status;
    batch_attention_kv8_generic_kernel<<<static_cast<unsigned>(blocks), kGenericThreads, 0, s>>>(a);
  }
  CAPI_LAUNCHED();
  return LCR_OK;
}
