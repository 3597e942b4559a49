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
// one XCD (block id mod 8) take neighbouring shares: with eight kv heads an XCD
// reads one head's keys, which short caches keep in its L2.
//
// Sizes in the measurements below are the largest of a ragged batch: the first
// chunk has all of the tokens named, others half to all, and caches have a third
// to all of the positions named.
//
// Arithmetic. S^T = K . Q^T on 16x16x32 matrix instructions: a lane holds one
// packed row and four keys of each sixteen. One pass over the keys:
//   p = exp2(c s + b), c = scale log2 e, b = e - c m for a running maximum m (e is
//   0, and 7 in fp16)
//   l += 1 . P^T;  O^T += V^T . P^T
// A new m is taken when some p would pass 2^(e + 8), and l and O then move to the
// new base by exp2(b_new - b); a row's l and O always share one base, so its
// rounding cancels in O / l. p is rounded to the element type for the products
// (the matrix cores take no wider operand beside 16-bit values: half a step of
// each weight, against two more products for a second half of p); everything else
// is fp32.
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
  int held;  // positions that a table has pages for
  float scale;
};

// ---------------------------------------------------------------------------
// Work division
// ---------------------------------------------------------------------------

// n / d for 0 <= n < 2^31: n * magic >> shift with magic = ceil(2^shift / d) and
// 2^(shift - 31) >= d. magic * d is past 2^shift by less than d, so the error,
// n / 2^shift of that, stays under 1 / d.
struct FastDivide {
  uint32_t magic;
  uint32_t shift;

  static FastDivide by(uint32_t d) {
    uint32_t shift = 31;
    while ((1ull << (shift - 31)) < d) ++shift;
    return FastDivide{static_cast<uint32_t>(((1ull << shift) + d - 1) / d), shift};
  }
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((static_cast<unsigned long long>(static_cast<uint32_t>(n)) * magic) >> shift);
  }
};

// A unit that lies over a cut, for the join: written by the share it begins in.
struct alignas(16) CutUnit {
  int rows;             // packed rows; 0: the share leaves no unit unfinished
  int last_share;
  int first_row;        // of the buffer
  int kv;
  int position;         // of the first token
};

// A value that is the same in every lane, held once for the wave.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A kernel argument in registers of its own. Left in the sixteen that one load
// brings, it is spilled and restored with all of them.
template <typename T>
__device__ __forceinline__ T own_register(T v) {
  asm volatile("" : "+s"(v));
  return v;
}

// What the matrix-core kernels need besides. Work is counted in steps of 64
// keys.
struct TiledPlan {
  uint32_t group_magic;   // r / group = r * group_magic >> 16 for r < 256
  FastDivide by_page;     // by page_size
  FastDivide by_tile;     // by tile_tokens
  FastDivide by_shares;   // by shares
  int tile_tokens;        // tokens of a tile of many rows
  int shares;             // of each kv head
  int split;              // 0: a share is a unit
  int min_share;          // steps
  float scale_log2e;
  CutUnit* cuts;          // [shares of all heads] the unit that each share leaves unfinished
  float* partials;        // [2 * shares of all heads][rows][head_dim], then [...][rows][2] bases and sums
};

constexpr int kFewRows = 32;
// Steps that a unit counts for besides its keys': its queries, the join of the
// waves, the output.
constexpr int kUnitSteps = 3;
constexpr int kStepKeys = 64;
// Few rows beside many: a step of 64 keys takes less than one of many rows, which
// keeps the vector units busy while the cache is read. 16 sequences of one token
// beside two chunks of 1000, with 64, 96, 128 and 192 keys a step: heads of 64 77,
// 74, 74 and 79 us, of 128 121, 105, 95 and 90; 64 beside two of 512: 102, 95, 99
// and 97, and 248, 184, 156 and 147.
template <int kHeadDim>
constexpr int kFewStepKeys = kHeadDim == 64 ? 96 : 192;
// A unit of at most so many steps is not cut: its partials and their join cost
// more than the share it lengthens. With 0, 4, 8 and 16: eight prompts of 256
// tokens 28, 26, 20 and 20 us, one of 2048 49, -, 48 and 47, two of 2048 65, -, 65
// and 67; few rows, which have less to join, 64 of 600 positions 18.2, 17.9, 19.1
// and 20.3, 32 of 1000 16.2, 16.3, 16.8 and 19.6.
template <bool kMany>
constexpr int kWholeSteps = kMany ? 8 : 4;

// A sequence's share of the work, in tokens and steps of one kv head.
struct Sequence {
  int row0;      // first row
  int rows;      // as row_starts says
  int tokens;    // at most max_new
  int tiles;
  int before;    // positions before its first row (may be negative)
  int visible;   // keys its last token sees
  int steps;     // what it counts for
};

// Keys that token i of a sequence sees.
__device__ __forceinline__ int keys_seen(const BatchAttnArgs& a, int before, int i) {
  return max(0, min(before + i + 1, a.held));
}

// Steps the tiles before tile i count for: tile j sees up to
// visible - tokens + (j + 1) tile_tokens keys. An estimate besides what is seen
// (negative positions, the table's end) only makes a share longer or shorter.
__device__ __forceinline__ int steps_before_tile(const TiledPlan& plan, const Sequence& s, int i) {
  if (!plan.split) return i;
  const long long tiles = i;
  const long long keys = tiles * max(s.visible - s.tokens, 0) + plan.tile_tokens * (tiles * (tiles + 1) / 2);
  return i * kUnitSteps + static_cast<int>(keys / kStepKeys);
}

// kMany: sequences may have more rows than a tile of few.
template <int kHeadDim, bool kMany>
__device__ __forceinline__ Sequence load_sequence(const BatchAttnArgs& a, const TiledPlan& plan, int b) {
  const int lo = a.row_starts[b], hi = a.row_starts[b + 1];
  const int length = a.lengths[b];
  Sequence s;
  s.row0 = lo;
  // starts that are no ascending rows of the buffer name no rows
  s.rows = lo >= 0 && hi > lo && hi <= a.tokens ? hi - lo : 0;
  s.tokens = min(s.rows, a.max_new);
  s.tiles = s.rows > 0 ? 1 : 0;
  if (kMany && s.tokens * a.group > kFewRows) s.tiles = plan.by_tile(s.tokens - 1) + 1;
  // lengths below -2^30 see nothing, as -2^30 does; rows are at most 2^30
  s.before = max(length, -(1 << 30)) - s.rows;
  s.visible = s.tokens > 0 ? keys_seen(a, s.before, s.tokens - 1) : 0;
  // up to the last tile, and that
  s.steps = s.tiles;
  if (plan.split && s.tiles > 0) {
    const int keys = max(s.visible, s.tokens);
    const bool few = s.tokens * a.group <= kFewRows;
    s.steps = kUnitSteps + (kMany && few ? keys / kFewStepKeys<kHeadDim> : keys / kStepKeys);
    if (kMany && s.tiles > 1) s.steps += steps_before_tile(plan, s, s.tiles - 1);
  }
  return s;
}

__device__ __forceinline__ Sequence uniform(const Sequence& s) {
  return Sequence{uniform(s.row0),   uniform(s.rows),    uniform(s.tokens), uniform(s.tiles),
                  uniform(s.before), uniform(s.visible), uniform(s.steps)};
}

struct ShareStart {
  int total;      // steps of a kv head
  int share;
  int before;     // steps before the sequence
  int sequence;   // -1: there is nothing left for this share
  Sequence seq;
};

// Steps that a kv head may count for: what the host allows of a call whose
// sequences have rows of their own. Row starts that overlap can count for more,
// past what the steps' arithmetic holds; such a call has no work.
constexpr int kMostSteps = INT32_MAX / 2;

// Sums of steps, which stay at the largest number instead of wrapping.
__device__ __forceinline__ uint32_t add_steps(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Where a kv head's share `index` begins: the prefix sums of the sequences'
// steps, taken by the whole block.
template <int kHeadDim, bool kMany, int kThreads>
__device__ __forceinline__ ShareStart find_share(const BatchAttnArgs& a, const TiledPlan& plan, int index,
                                                 uint32_t* lds_sums, ShareStart* lds_found) {
  constexpr int kWaves = kThreads / 64;
  const int t = threadIdx.x;
  const int per = (a.batch + kThreads - 1) / kThreads;
  uint32_t mine = 0;
  Sequence seq{};
  for (int k = 0; k < per; ++k) {
    const int b = t * per + k;
    if (b < a.batch) {
      seq = load_sequence<kHeadDim, kMany>(a, plan, b);
      mine = add_steps(mine, static_cast<uint32_t>(seq.steps));
    }
  }
  uint32_t to = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t other = __shfl_up(to, o, 64);
    if (lane_id() >= o) to = add_steps(to, other);
  }
  if (lane_id() == 63) lds_sums[t >> 6] = to;
  if (t == 0) lds_found->sequence = -1;
  __syncthreads();
  uint32_t all = 0, ahead = to - mine;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < (t >> 6)) ahead = add_steps(ahead, lds_sums[w]);
    all = add_steps(all, lds_sums[w]);
  }
  const int total = all <= kMostSteps ? static_cast<int>(all) : 0;
  int before = static_cast<int>(ahead);
  const int share = plan.split ? max(plan.by_shares(total + plan.shares - 1), plan.min_share) : 1;
  const int at = index * share;
  if (total > 0 && at >= before && at < before + static_cast<int>(mine)) {
    for (int k = 0; k < per; ++k) {
      const int b = t * per + k;
      if (b >= a.batch) break;
      if (per > 1) seq = load_sequence<kHeadDim, kMany>(a, plan, b);
      if (at < before + seq.steps) {
        *lds_found = ShareStart{total, share, before, b, seq};
        break;
      }
      before += seq.steps;
    }
  }
  __syncthreads();
  const ShareStart found = *lds_found;
  return ShareStart{uniform(found.total), uniform(found.share), uniform(found.before), uniform(found.sequence),
                    uniform(found.seq)};
}

// Waits for direct loads, and for LDS reads and writes, across which the compiler
// moves no memory access.
template <int kCount>
__device__ __forceinline__ void loads_landed() {
  asm volatile("" : : : "memory");
  wait_stage_landed<kCount>();
  asm volatile("" : : : "memory");
}
__device__ __forceinline__ void lds_settled() { loads_landed<63>(); }

// One block's part of a unit.
struct Piece {
  const int32_t* table;
  const elem_t* keys;    // the kv head's, of page 0
  const elem_t* values;
  int kv;
  int before;      // positions before the tile's first token
  int row0;        // the tile's first row
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

// Blocks a compute unit, and waves a SIMD, follow from LDS and registers. At
// head_dim 64, three blocks of four waves (168 registers a lane); at 128, one of
// eight (256).
template <int kHeadDim>
struct TiledShape {
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

// kTop: the exponent of a row's largest weight when its base is taken. The base is
// kept until a weight would pass 8 more. In fp16 weights are held as high as that
// leaves them (2^15), as they round coarsely below 2^-14 and to 0 below 2^-25:
// with kTop 0, 9000 keys of e^-18 of the largest each counted for nothing.
#if defined(LCR_ELEM_FP16)
constexpr uint32_t kInfBits = 0x7c00u, kOneBits = 0x3c00u;
constexpr float kTop = 7.0f;
#else
constexpr uint32_t kInfBits = 0x7f80u, kOneBits = 0x3f80u;
constexpr float kTop = 0.0f;
#endif

// A packed-row fragment's accumulators: rows 16 rf + col, per lane.
template <int kHeadDim, int kRF>
struct TiledRows {
  mfma_in8 q[kRF][TiledShape<kHeadDim>::kSteps];
  mfma_acc4 o[kRF][TiledShape<kHeadDim>::kDFrags];
  float base[kRF];  // +inf: no visible key yet
  mfma_acc4 sum[kRF];  // of the row's weights, four times
  int seen[kRF];    // keys the row sees, at most key1
  uint32_t up[kRF], down[kRF];  // bit 4 df + e: o[rf][df][e] sees +inf, -inf (both: NaN)

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      base[rf] = __builtin_huge_valf();
      sum[rf] = mfma_acc4{0.f, 0.f, 0.f, 0.f};
      up[rf] = down[rf] = 0;
#pragma unroll
      for (int df = 0; df < TiledShape<kHeadDim>::kDFrags; ++df) o[rf][df] = mfma_acc4{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ __forceinline__ void add_special() {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      if (!__any((up[rf] | down[rf]) != 0)) continue;
#pragma unroll
      for (int df = 0; df < TiledShape<kHeadDim>::kDFrags; ++df) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool plus = (up[rf] >> (4 * df + e) & 1) != 0, minus = (down[rf] >> (4 * df + e) & 1) != 0;
          if (plus) o[rf][df][e] += __builtin_huge_valf();
          if (minus) o[rf][df][e] -= __builtin_huge_valf();
        }
      }
    }
  }
};

__device__ __forceinline__ int packed_token(const TiledPlan& plan, int r) {
  return static_cast<int>((static_cast<uint32_t>(r) * plan.group_magic) >> 16);
}

// Queries of packed rows row0 + 16 rf + col (those past the unit's rows repeat
// its last, are never stored and see what that one sees).
template <int kHeadDim, int kRF>
__device__ __forceinline__ void load_rows(TiledRows<kHeadDim, kRF>& rows, const BatchAttnArgs& a, const TiledPlan& plan,
                                          const Piece& p, int row0) {
  const int col = lane_id() & 15;
  const int grp = lane_id() >> 4;
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const int r = min(row0 + 16 * rf + col, p.rows - 1);
    const int token = packed_token(plan, r);
    const int head = p.kv * a.group + r - token * a.group;
    const elem_t* q = a.q + static_cast<size_t>(p.row0 + token) * a.q_row_stride +
                      static_cast<size_t>(head) * kHeadDim + 8 * grp;
#pragma unroll
    for (int ks = 0; ks < TiledShape<kHeadDim>::kSteps; ++ks) rows.q[rf][ks] = as_operand(load16(q + 32 * ks));
    rows.seen[rf] = min(keys_seen(a, p.before, token), p.key1);
  }
}

// Waits for the queries here. Left to their first use, inside the loop over the
// tiles, the compiler's wait for them there is one for every direct load in
// flight, each time round.
template <int kHeadDim, int kRF>
__device__ __forceinline__ void hold_rows(TiledRows<kHeadDim, kRF>& rows) {
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
#pragma unroll
    for (int ks = 0; ks < TiledShape<kHeadDim>::kSteps; ++ks) asm volatile("" : "+v"(rows.q[rf][ks]));
  }
}

// 16 kKF keys of a tile against the rows: scores, weights, values.
//   keys, values  the tile in LDS
//   key0          its first key
//   all_seen      keys that every row of the wave sees
template <int kHeadDim, int kRF, int kKF>
struct TileWork {
  using Shape = TiledShape<kHeadDim>;
  mfma_acc4 s[kRF][kKF];
  uint32_t packed[kRF][kKF][2];

  __device__ __forceinline__ void scores(const TiledRows<kHeadDim, kRF>& rows, const elem_t* keys) {
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

  __device__ __forceinline__ void mask(const TiledRows<kHeadDim, kRF>& rows, int key0) {
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

  // The running statistics: a larger base where a score needs one.
  __device__ __forceinline__ void raise_base(TiledRows<kHeadDim, kRF>& rows, float c) {
    float top[kRF];
    bool raise = false;
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      top[rf] = s[rf][0][0];
#pragma unroll
      for (int kf = 0; kf < kKF; ++kf) {
#pragma unroll
        for (int v = 0; v < 4; ++v) top[rf] = fmaxf(top[rf], s[rf][kf][v]);
      }
      // c top + base: the largest weight's exponent (inf for a first visible
      // key, NaN, which compares false, while there is none)
      raise |= __builtin_fmaf(top[rf], c, rows.base[rf]) > kTop + 8.0f;
    }
    if (!__any(raise)) return;
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      float most = fmaxf(top[rf], xor_lane<16>(top[rf]));
      most = fmaxf(most, xor_lane<32>(most));
      if (__builtin_fmaf(most, c, rows.base[rf]) > kTop) {
        const float base = kTop - most * c;
        const float move = __builtin_amdgcn_exp2f(base - rows.base[rf]);
        rows.base[rf] = base;
        rows.sum[rf] *= move;
#pragma unroll
        for (int df = 0; df < Shape::kDFrags; ++df) rows.o[rf][df] *= move;
      }
    }
  }

  // The weights of the scores of 32 keys, rounded to the element type.
  __device__ __forceinline__ void weights(const TiledRows<kHeadDim, kRF>& rows, float c, int half) {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      // before the first visible key every score is -inf: against base 0
      const float base = rows.base[rf] == __builtin_huge_valf() ? 0.0f : rows.base[rf];
#pragma unroll
      for (int kf = 2 * half; kf < 2 * half + 2; ++kf) {
        float p[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rf][kf][v], c, base));
        packed[rf][kf][0] = pack_rounded(p[0], p[1]);
        packed[rf][kf][1] = pack_rounded(p[2], p[3]);
      }
    }
  }

  __device__ __forceinline__ mfma_in8 weight_operand(int rf, int half) const {
    return as_operand(vec16{{packed[rf][2 * half][0], packed[rf][2 * half][1], packed[rf][2 * half + 1][0],
                             packed[rf][2 * half + 1][1]}});
  }

  // The weights' sum is a product with ones: of what the values are weighted
  // with, rounded as they are, and off the vector units, which the exponentials
  // keep busy.
  __device__ __forceinline__ void products(TiledRows<kHeadDim, kRF>& rows, const elem_t* values, int half) {
    constexpr uint32_t kOnes = kOneBits << 16 | kOneBits;
    const mfma_in8 ones = as_operand(vec16{{kOnes, kOnes, kOnes, kOnes}});
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) rows.sum[rf] = mfma16x16x32(ones, weight_operand(rf, half), rows.sum[rf]);
#pragma unroll
    for (int df = 0; df < Shape::kDFrags; ++df) {
      const mfma_in8 v = transposed_values<kHeadDim>(values, half, df, lane_id());
#pragma unroll
      for (int rf = 0; rf < kRF; ++rf) rows.o[rf][df] = mfma16x16x32(v, weight_operand(rf, half), rows.o[rf][df]);
    }
  }

  // 1 for each of 32 keys that a lane's row sees, in the order of weight_operand.
  __device__ __forceinline__ mfma_in8 seen_operand(const TiledRows<kHeadDim, kRF>& rows, int rf, int half, int key0) const {
    int left = rows.seen[rf] - key0 - 32 * half - 4 * (lane_id() >> 4);
    asm volatile("" : "+v"(left));  // made again each time: kept, they cost registers in every tile
    vec16 seen;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 16 * (i >> 1) + 2 * (i & 1);
      seen.w[i] = (key < left ? kOneBits : 0u) | (key + 1 < left ? kOneBits << 16 : 0u);
    }
    return as_operand(seen);
  }

  // Which rows see an infinity or NaN of the tile, by a product of ones in place
  // of it and of what they see; a NaN counts as both infinities. (With the weights
  // instead, one that rounds to 0 would lose it: in fp16, of any key 17 below the
  // largest score.)
  __device__ __forceinline__ void mark_special(TiledRows<kHeadDim, kRF>& rows, const elem_t* values, int key0) {
#pragma unroll
    for (int half = 0; half < kKF / 2; ++half) {
#pragma unroll 1
      for (int df = 0; df < Shape::kDFrags; ++df) {
        const vec16 v = __builtin_bit_cast(vec16, transposed_values<kHeadDim>(values, half, df, lane_id()));
        vec16 up, down;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t plus = 0, minus = 0;
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            const uint32_t x = (v.w[i] >> h) & 0xffffu;
            const bool special = (x & kInfBits) == kInfBits;
            plus |= (special && x != (0x8000u | kInfBits) ? kOneBits : 0u) << h;
            minus |= (special && x != kInfBits ? kOneBits : 0u) << h;
          }
          up.w[i] = plus;
          down.w[i] = minus;
        }
#pragma unroll
        for (int rf = 0; rf < kRF; ++rf) {
          const mfma_acc4 zero{0.f, 0.f, 0.f, 0.f};
          const mfma_acc4 a = mfma16x16x32(as_operand(up), seen_operand(rows, rf, half, key0), zero);
          const mfma_acc4 b = mfma16x16x32(as_operand(down), seen_operand(rows, rf, half, key0), zero);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            rows.up[rf] |= (a[e] > 0.0f ? 1u : 0u) << (4 * df + e);
            rows.down[rf] |= (b[e] > 0.0f ? 1u : 0u) << (4 * df + e);
          }
        }
      }
    }
  }
};

// Infinities and NaN among the values of a tile that some row does not see
// whole. In the matrix product they would reach, as 0 * inf, rows that do not
// see them: such a tile's are marked in the rows that do, which get them added
// at the end, and then cleared.
__device__ __forceinline__ bool pair_special(uint32_t w) {
  return (w & kInfBits) == kInfBits || ((w >> 16) & kInfBits) == kInfBits;
}

// Whether `chunks` groups of 64 16-byte chunks hold any.
__device__ __forceinline__ bool any_special(const elem_t* values, int chunks) {
  bool special = false;
#pragma unroll 4
  for (int n = 0; n < chunks; ++n) {
    const vec16 v = load16(values + 8 * (64 * n + lane_id()));
#pragma unroll
    for (int i = 0; i < 4; ++i) special |= pair_special(v.w[i]);
  }
  return __any(special);
}

__device__ __forceinline__ void clear_special(elem_t* values, int chunks) {
#pragma unroll 1
  for (int n = 0; n < chunks; ++n) {
    elem_t* at = values + 8 * (64 * n + lane_id());
    vec16 v = load16(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((v.w[i] & kInfBits) == kInfBits) v.w[i] &= 0xffff0000u;
      if (((v.w[i] >> 16) & kInfBits) == kInfBits) v.w[i] &= 0xffffu;
    }
    store16(at, v);
  }
}

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
__device__ __forceinline__ RunPage find_run(const BatchAttnArgs& a, const TiledPlan& plan, const Piece& p, int last,
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

// A page outside the pool is read as page 0, and `bad` set.
__device__ __forceinline__ int pool_page(const BatchAttnArgs& a, int page, int& bad) {
  const bool inside = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pool_pages);
  bad |= inside ? 0 : 1;
  return inside ? page : 0;
}

// The run of keys (or values) from key `key` on into rows row0 .. of a tile. Row
// r of LDS starts r rows behind the tile, in memory as in LDS, so the loads of a
// run differ by one offset that counts in both.
template <int kHeadDim, bool kWholePages, int kRun, bool kKeys, bool kStream>
__device__ __forceinline__ void load_run(const BatchAttnArgs& a, const TiledPlan& plan, const Piece& p, int last,
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

// One element's place in the output, from a packed row.
template <int kHeadDim>
__device__ __forceinline__ size_t out_at(const BatchAttnArgs& a, const TiledPlan& plan, const Piece& p, int r) {
  const int token = packed_token(plan, r);
  return (static_cast<size_t>(p.row0 + token) * a.num_heads + p.kv * a.group + (r - token * a.group)) *
         kHeadDim;
}

template <int kHeadDim>
__device__ __forceinline__ float* partial_stats(const TiledPlan& plan, int kv_heads, int tile_rows) {
  return plan.partials + static_cast<size_t>(2 * plan.shares) * kv_heads * tile_rows * kHeadDim;
}

// At most 32 rows: the waves split the keys.
template <int kHeadDim, bool kWholePages, int kRF, int kTileRows>
__device__ __forceinline__ void few_rows(TiledLds<kHeadDim>& lds, const BatchAttnArgs& a, const TiledPlan& plan,
                                         const Piece& p) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kLoads = 32 / Shape::kLoadRows;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id();
  const int col = lane & 15;
  const int grp = lane >> 4;
  elem_t* mine = lds.ring + wave * Shape::kWaveElems;
  elem_t* const key_tile = mine;
  elem_t* const value_tile = mine + 32 * kHeadDim;
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

  TiledRows<kHeadDim, kRF> rows;
  rows.clear();
  if (count > 0) {
    load_rows<kHeadDim, kRF>(rows, a, plan, p, 0);
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
    TileWork<kHeadDim, kRF, 2> work;
    work.scores(rows, key_tile);
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
      work.mark_special(rows, value_tile, key0);
      clear_special(value_tile, 32 * kHeadDim / 512);
    }
    work.products(rows, value_tile, 0);
    lds_settled();
    if (more) issue(Values{}, t + 1, pages);
  }

  rows.add_special();
  // The waves' results meet in LDS, each in its own (now free) part.
  if (__any(bad != 0)) {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) rows.sum[rf][0] = __builtin_nanf("");
  }
  float* outputs = reinterpret_cast<float*>(mine);
  static_assert(Shape::kWaveElems * sizeof(elem_t) >= kFewRows * kHeadDim * sizeof(float), "a wave's outputs fit");
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const float sum = rows.sum[rf][0];
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
        float* stats = partial_stats<kHeadDim>(plan, a.view.num_kv_heads, kTileRows) + (static_cast<size_t>(p.slot) * kTileRows + r) * 2;
        stats[0] = base;
        stats[1] = sum;
      }
    } else {
      const int token = packed_token(plan, r);
      const bool any = keys_seen(a, p.before, token) > 0;
      const float inv = any ? 1.0f / sum : 0.0f;
      uint2 words;
      words.x = any ? pack_elems(o[0] * inv, o[1] * inv) : 0u;
      words.y = any ? pack_elems(o[2] * inv, o[3] * inv) : 0u;
      *reinterpret_cast<uint2*>(a.out + out_at<kHeadDim>(a, plan, p, r) + d) = words;
    }
  }
  __syncthreads();  // the parts may be loaded into again
}

// Many rows: the waves split them, 32 each, and share the tiles. `tiles_done`:
// of the block's pieces before, so that a tile's number is its own.
template <int kHeadDim, bool kWholePages>
__device__ __forceinline__ void many_rows(TiledLds<kHeadDim>& lds, const BatchAttnArgs& a, const TiledPlan& plan,
                                          const Piece& p, int& tiles_done) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kRF = 2;
  constexpr int kRun = 64 / Shape::kWaves;          // a wave's keys of a tile
  constexpr int kLoads = kRun / Shape::kLoadRows;
  constexpr int kTileRows = Shape::kTileRows;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id();
  const int col = lane & 15;
  const int grp = lane >> 4;
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
  TiledRows<kHeadDim, kRF> rows;
  rows.clear();
  int all_seen = 0, any_seen = 0;
  if (active) {
    load_rows<kHeadDim, kRF>(rows, a, plan, p, row0);
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
    if (mine) {
      TileWork<kHeadDim, kRF, 4> work;
      work.scores(rows, stage);
      if (!whole) work.mask(rows, tile0);
      work.raise_base(rows, plan.scale_log2e);
      if (!special) {
        work.weights(rows, plan.scale_log2e, 0);
        work.products(rows, values, 0);
        work.weights(rows, plan.scale_log2e, 1);
        work.products(rows, values, 1);
      }
    }
    if (!special) continue;
    // Half a tile at a time, its scores once more: registers for the marks.
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      elem_t* at = values + half * 32 * kHeadDim;
      TileWork<kHeadDim, kRF, 2> work;
      if (mine) {
        work.scores(rows, stage + half * 32 * kHeadDim);
        if (!whole) work.mask(rows, tile0 + 32 * half);
        work.weights(rows, plan.scale_log2e, 0);
        work.mark_special(rows, at, tile0 + 32 * half);
      }
      lds_settled();
      plain_barrier();
      static_assert(kHeadDim / 16 <= Shape::kWaves, "a wave clears one group of chunks at most");
      if (wave < kHeadDim / 16) clear_special(at + wave * 512, 1);
      lds_settled();
      plain_barrier();
      if (mine) work.products(rows, at, 0);
    }
  }
  tiles_done += max(tiles, 0);
  if (__any(bad != 0) && lane == 0) lds.bad = 1;
  __syncthreads();  // every wave is done with the tiles; the flag is set
  if (!active) return;
  rows.add_special();
  const bool spoilt = lds.bad != 0;
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const int r = row0 + 16 * rf + col;
    float sum = rows.sum[rf][0];
    if (spoilt) sum = __builtin_nanf("");
    if (r >= p.rows) continue;
    if (p.slot >= 0) {
      const size_t at = static_cast<size_t>(p.slot) * kTileRows + r;
#pragma unroll
      for (int df = 0; df < Shape::kDFrags; ++df) {
        *reinterpret_cast<mfma_acc4*>(plan.partials + at * kHeadDim + 16 * df + 4 * grp) = rows.o[rf][df];
      }
      if (grp == 0) {
        float* stats = partial_stats<kHeadDim>(plan, a.view.num_kv_heads, kTileRows) + at * 2;
        stats[0] = rows.base[rf];
        stats[1] = sum;
      }
    } else {
      const bool any = keys_seen(a, p.before, packed_token(plan, r)) > 0;
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

// kMaxRows: packed rows a sequence may have, 16, 32 or any number (0).
template <int kHeadDim, int kMaxRows, bool kWholePages>
__global__ __launch_bounds__(TiledShape<kHeadDim>::kThreads, TiledShape<kHeadDim>::kSimdWaves) void batch_attention_kernel(
    BatchAttnArgs args, TiledPlan tiled_plan) {
  using Shape = TiledShape<kHeadDim>;
  constexpr bool kMany = kMaxRows == 0;
  constexpr int kTileRows = kMany ? Shape::kTileRows : kFewRows;
  __shared__ __attribute__((aligned(1024))) TiledLds<kHeadDim> lds;
  BatchAttnArgs a = args;
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

  // Share: neighbours on one XCD where the grid is a multiple of 8.
  const unsigned blocks = gridDim.x;
  const int block = static_cast<int>(blocks % 8u == 0 ? blockIdx.x % 8u * (blocks / 8u) + blockIdx.x / 8u : blockIdx.x);
  const int kv = plan.by_shares(block);
  // seen by every wave behind the barriers of the search
  if (threadIdx.x == 0) lds.special[0] = lds.special[1] = -1;
  const ShareStart found =
      find_share<kHeadDim, kMany, Shape::kThreads>(a, plan, block - kv * plan.shares, lds.sums, &lds.found);
  if (plan.split && threadIdx.x == 0) plan.cuts[block].rows = 0;
  if (found.sequence < 0) return;
  int b = found.sequence;
  Sequence seq = found.seq;
  int at = (block - kv * plan.shares) * found.share;
  const int end = min(at + found.share, found.total);
  int before = found.before;  // steps before the sequence
  // The tile that the share begins in: the last that starts at or before it.
  int tile = 0;
  if constexpr (kMany) {
    for (int lo = 0, hi = seq.tiles - 1; lo < hi;) {
      const int mid = (lo + hi + 1) >> 1;
      if (before + steps_before_tile(plan, seq, mid) <= at) {
        lo = mid;
        tile = mid;
      } else {
        hi = mid - 1;
      }
    }
  }
  int tiles_done = 0;
  Piece p;
  p.kv = kv;
  p.keys = a.view.keys + static_cast<size_t>(kv) * static_cast<size_t>(a.view.head_stride);
  p.values = a.view.values + static_cast<size_t>(kv) * static_cast<size_t>(a.view.head_stride);
  while (true) {
    const int start = before + (kMany ? steps_before_tile(plan, seq, tile) : 0);
    const int stop = before + (kMany && tile + 1 < seq.tiles ? steps_before_tile(plan, seq, tile + 1) : seq.steps);
    const bool single = !kMany || seq.tokens * a.group <= kFewRows;
    const int token0 = single ? 0 : tile * plan.tile_tokens;
    const int tokens = single ? seq.tokens : min(plan.tile_tokens, seq.tokens - token0);
    p.table = a.view.page_table + static_cast<size_t>(b) * a.table_stride;
    p.row0 = seq.row0 + token0;
    p.before = seq.before + token0;
    p.rows = tokens * a.group;
    p.seen_first = keys_seen(a, p.before, 0);
    p.seen_last = tokens > 0 ? keys_seen(a, p.before, tokens - 1) : 0;
    p.key0 = 0;
    p.key1 = p.seen_last;
    p.slot = -1;
    // A short unit is not cut: it goes to the share that it begins in.
    const bool whole = !plan.split || stop - start <= kWholeSteps<kMany>;
    if (!whole && (start < at || stop > end)) {
      // steps into the unit, in keys
      const int keys = kMany && single ? kFewStepKeys<kHeadDim> : kStepKeys;
      auto cut = [&](int steps) { return steps >= (p.seen_last + keys - 1) / keys ? p.seen_last : steps * keys; };
      p.slot = 2 * block + (start < at ? 0 : 1);
      if (start < at) p.key0 = cut(at - start);
      if (stop > end) p.key1 = cut(end - start);
      if (start >= at && threadIdx.x == 0) {
        plan.cuts[block] = CutUnit{p.rows, kv * plan.shares + static_cast<int>(static_cast<unsigned>(stop - 1) /
                                                                               static_cast<unsigned>(found.share)),
                                   p.row0, kv, p.before};
      }
    }
    // Rows past max_new are zeros, written where the sequence begins.
    if (tile == 0 && start >= at && seq.rows > seq.tokens) {
      for (int i = seq.tokens; i < seq.rows; ++i) {
        elem_t* row = a.out + (static_cast<size_t>(seq.row0 + i) * a.num_heads + kv * a.group) * kHeadDim;
        for (int e = 4 * static_cast<int>(threadIdx.x); e < a.group * kHeadDim; e += 4 * Shape::kThreads) {
          *reinterpret_cast<uint2*>(row + e) = make_uint2(0u, 0u);
        }
      }
    }
    if (p.rows > 0 && !(whole && start < at)) {
      if (!single) {
        if constexpr (kMany) many_rows<kHeadDim, kWholePages>(lds, a, plan, p, tiles_done);
      } else {
        few_rows<kHeadDim, kWholePages, kMaxRows == 16 ? 1 : 2, kTileRows>(lds, a, plan, p);
      }
    }
    at = stop;
    if (at >= end) break;
    if (!kMany || ++tile >= seq.tiles) {
      tile = 0;
      before += seq.steps;
      do {  // the next sequence that has rows
        if (++b == a.batch) return;
        seq = uniform(load_sequence<kHeadDim, kMany>(a, plan, b));
      } while (seq.tiles == 0);
    }
    if constexpr (kMany) __syncthreads();  // the tiles and the flag are free again
  }
}

// Joins the partials of the units that lie over a cut: gridDim.y blocks for the
// unit that share blockIdx.x leaves unfinished (most often none), four elements
// of a packed row a lane, so that a wave has room for kGroups rows. Tiles of
// many rows have few partials each, and the groups take a row each; few rows
// have many, and the groups take the row's partials in turn. A launch and a chain
// of three reads, 4 us for few rows, 9 for many (up to 25 MB of partials).
constexpr int kJoinThreads = 256;

template <int kHeadDim, bool kRowEach>
__global__ __launch_bounds__(kJoinThreads) void batch_attention_join_kernel(BatchAttnArgs a, TiledPlan plan,
                                                                           int tile_rows) {
  constexpr int kRowLanes = kHeadDim / 4;
  constexpr int kGroups = 64 / kRowLanes;
  const CutUnit unit = plan.cuts[blockIdx.x];
  if (unit.rows == 0) return;
  const int lane = lane_id();
  const int d = 4 * (lane % kRowLanes);
  const int group = lane / kRowLanes;
  const float* all_stats = partial_stats<kHeadDim>(plan, a.view.num_kv_heads, tile_rows);
  const int waves = static_cast<int>(gridDim.y) * (kJoinThreads / 64);
  const int wave = static_cast<int>(blockIdx.y) * (kJoinThreads / 64) + (static_cast<int>(threadIdx.x) >> 6);
  constexpr int kWaveRows = kRowEach ? kGroups : 1;
  const int first = static_cast<int>(blockIdx.x) + (kRowEach ? 0 : group);
  for (int r0 = wave * kWaveRows; r0 < unit.rows; r0 += waves * kWaveRows) {
    const int r = min(r0 + (kRowEach ? group : 0), unit.rows - 1);
    float base = __builtin_huge_valf(), sum = 0.0f;
    mfma_acc4 o{0.f, 0.f, 0.f, 0.f};
    // (from, sum, x) joins (base, sum, o): both move to the smaller base. No
    // keys: base +inf, nothing to add.
    auto join = [&](float from, float part, const mfma_acc4& x) {
      const float to = fminf(base, from);
      const float keep = base == __builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(to - base);
      const float move = from == __builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(to - from);
      base = to;
      sum = __builtin_fmaf(part, move, sum * keep);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], move, o[e] * keep);
    };
#pragma unroll 4
    for (int s = first; s <= unit.last_share; s += kRowEach ? 1 : kGroups) {
      // a share's first partial continues a unit, its second begins one
      const size_t at = static_cast<size_t>(s == static_cast<int>(blockIdx.x) ? 2 * s + 1 : 2 * s) * tile_rows + r;
      const float2 stats = *reinterpret_cast<const float2*>(all_stats + 2 * at);
      join(stats.x, stats.y, *reinterpret_cast<const mfma_acc4*>(plan.partials + at * kHeadDim + d));
    }
    auto join_lane = [&](auto distance) {
      constexpr int kDistance = decltype(distance)::value;
      mfma_acc4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = xor_lane<kDistance>(o[e]);
      join(xor_lane<kDistance>(base), xor_lane<kDistance>(sum), x);
    };
    if constexpr (!kRowEach) {
      join_lane(std::integral_constant<int, 32>{});
      if constexpr (kGroups == 4) join_lane(std::integral_constant<int, 16>{});
    }
    if (kRowEach ? r0 + group < unit.rows : group == 0) {
      const int token = packed_token(plan, r);
      const bool any = unit.position + token >= 0;
      const float inv = any ? 1.0f / sum : 0.0f;
      uint2 words;
      words.x = any ? pack_elems(o[0] * inv, o[1] * inv) : 0u;
      words.y = any ? pack_elems(o[2] * inv, o[3] * inv) : 0u;
      const size_t row = static_cast<size_t>(unit.first_row + token) * a.num_heads + unit.kv * a.group +
                         (r - token * a.group);
      *reinterpret_cast<uint2*>(a.out + row * kHeadDim + d) = words;
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
// Nothing is shared between heads or rows and nothing split: the way for what the
// tiles above do not take, not for speed (64 sequences of up to 8000 positions,
// heads of 64: 4.2 ms).
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

// A kv head's shares: all heads' together are the blocks resident at once.
template <int kHeadDim>
int tiled_shares(int kv_heads, bool many) {
  const int blocks = many ? TiledShape<kHeadDim>::kBlocks : TiledShape<kHeadDim>::kFewBlocks;
  return std::max(1, device_compute_units() * blocks / kv_heads);
}

bool many_rows_possible(int max_new, int group) { return static_cast<long long>(max_new) * group > kFewRows; }

template <int kHeadDim>
size_t tiled_workspace(int max_new, int kv_heads, int group) {
  const bool many = many_rows_possible(max_new, group);
  const size_t rows = many ? TiledShape<kHeadDim>::kTileRows : kFewRows;
  const size_t shares = static_cast<size_t>(tiled_shares<kHeadDim>(kv_heads, many)) * static_cast<size_t>(kv_heads);
  return shares * (sizeof(CutUnit) + 2 * rows * (kHeadDim + 2) * sizeof(float));
}

template <int kHeadDim, int kMaxRows, bool kWholePages>
void launch_tiled_kernels(const BatchAttnArgs& a, const TiledPlan& plan, hipStream_t s) {
  using Shape = TiledShape<kHeadDim>;
  constexpr int kTileRows = kMaxRows == 0 ? Shape::kTileRows : kFewRows;
  const unsigned blocks = static_cast<unsigned>(plan.shares) * static_cast<unsigned>(a.view.num_kv_heads);
  batch_attention_kernel<kHeadDim, kMaxRows, kWholePages><<<blocks, Shape::kThreads, 0, s>>>(a, plan);
  if (!plan.split) return;
  // A row is a chain of loads, so few follow each other: one time round for
  // many rows, two for few.
  constexpr bool kRowEach = kMaxRows == 0;
  const dim3 join(blocks, kRowEach ? kTileRows / (4 * 256 / kHeadDim) : kTileRows / 8);
  batch_attention_join_kernel<kHeadDim, kRowEach><<<join, kJoinThreads, 0, s>>>(a, plan, kTileRows);
}

template <int kHeadDim>
int tiled_tile_tokens(int group) {
  return std::max(1, TiledShape<kHeadDim>::kTileRows / group);
}

// A unit a block: at most one short tile a sequence beside the full ones.
template <int kHeadDim>
long long most_tiled_units(const BatchAttnArgs& a) {
  return a.tokens / tiled_tile_tokens<kHeadDim>(a.group) + static_cast<long long>(a.batch);
}

template <int kHeadDim>
void launch_tiled(const BatchAttnArgs& a, void* workspace, size_t workspace_bytes, hipStream_t s) {
  TiledPlan plan{};
  const int kv_heads = a.view.num_kv_heads;
  plan.group_magic = static_cast<uint32_t>((65536 + a.group - 1) / a.group);
  plan.tile_tokens = tiled_tile_tokens<kHeadDim>(a.group);
  plan.by_page = FastDivide::by(static_cast<uint32_t>(a.view.page_size));
  plan.by_tile = FastDivide::by(static_cast<uint32_t>(plan.tile_tokens));
  plan.scale_log2e = static_cast<float>(static_cast<double>(a.scale) * 1.4426950408889634);
  plan.min_share = 4;
  // Tables of at most 1024 positions: no unit is long enough for a cut and its
  // second launch to pay. By the number of sequences and positions, one token
  // each, cut and not: 8 of 1000 14.4 and 11.7 us, 64 of 600 18.2 and 13.1, 128 of
  // 1000 36.4 and 35.0; 8 of 2000 14.3 and 18.0. Where the tiles of many rows
  // leave half of the device without work, 768: heads of 128, 8 on 4, a prompt of
  // 837 tokens with others (76 units) 33.4 and 37.9, 16 on 8, one of 1000 (64)
  // 39.3 and 43.9; heads of 64, 8 on 8, one of 900 (64) 19.7 and 22.9, but 8 on 2,
  // two of 800 (78) 24.2 and 21.3, and 32 on 8, one of 500 (128) 20.1 and 16.1.
  const bool many = many_rows_possible(a.max_new, a.group);
  const bool half_idle = many && 2 * most_tiled_units<kHeadDim>(a) * kv_heads <= device_compute_units();
  const int cut_positions = half_idle ? 768 : 1024;
  // Steps are counted in 32 bits. Where a call's could pass them, it has units
  // enough to fill the device uncut.
  const long long most_units = many ? most_tiled_units<kHeadDim>(a) : a.batch;
  const long long most_steps = kUnitSteps + 1 + std::max(a.held, std::min(a.max_new, a.tokens)) / kStepKeys;
  if (a.held > cut_positions && most_units * most_steps <= kMostSteps && workspace != nullptr &&
      workspace_bytes >= tiled_workspace<kHeadDim>(a.max_new, kv_heads, a.group)) {
    plan.split = 1;
    plan.shares = tiled_shares<kHeadDim>(kv_heads, many);
    plan.cuts = static_cast<CutUnit*>(workspace);
    plan.partials = reinterpret_cast<float*>(plan.cuts + static_cast<size_t>(plan.shares) * kv_heads);
  } else {
    plan.shares = static_cast<int>(most_tiled_units<kHeadDim>(a));
  }
  plan.by_shares = FastDivide::by(static_cast<uint32_t>(plan.shares));
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

bool on_bytes(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The matrix-core kernels take a positive scale (the running maximum is the
// scores') and a group that fits a tile.
bool tiled_takes(const BatchAttnArgs& a) {
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
  if (head_dim == 64) return tiled_workspace<64>(max_new, kv_heads, heads_per_kv);
  if (head_dim == 128) return tiled_workspace<128>(max_new, kv_heads, heads_per_kv);
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
  BatchAttnArgs a{static_cast<elem_t*>(out), static_cast<const elem_t*>(q), KvCacheView::from_c(*view), row_starts,
                  lengths, batch, tokens, max_new, num_heads, heads_per_kv, table_stride, pool_pages, q_row_stride,
                  table_stride * view->page_size, scale};
  auto s = static_cast<hipStream_t>(stream);
  const bool tiled = tiled_takes(a);
  // A launch has fewer than 2^32 threads in all.
  const long long units = static_cast<long long>(tokens) * num_heads;
  const long long blocks = !tiled ? (units + kGenericWaves - 1) / kGenericWaves
                           : view->num_kv_heads * (view->head_dim == 64 ? most_tiled_units<64>(a) : most_tiled_units<128>(a));
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
