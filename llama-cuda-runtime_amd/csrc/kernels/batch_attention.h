// What the batched attention's kernels share, whatever their cache holds: how the
// work is divided, the arithmetic on the matrix cores, the joining of partials.
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
// one XCD (block id mod 8) take neighbouring shares (kNeighbours): with eight kv
// heads an XCD reads one head's keys, which short caches keep in its L2.
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
// A kernel's Shape says how many waves a block has (kWaves, kThreads) and rows a
// tile of many (kTileRows), how its lanes hold dims (q_dim, out_dim, out_piece),
// what a step of few rows weighs beside one of many (kFewStepKeys), and which
// blocks take neighbouring shares (kNeighbours).
#pragma once

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "device_common.h"
#include "kv_tiles.h"

namespace lcr {
namespace {

template <typename CacheView>
struct BatchAttnArgs {
  elem_t* out;
  const elem_t* q;
  CacheView view;
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
template <typename Args>
__device__ __forceinline__ int keys_seen(const Args& a, int before, int i) {
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
template <typename Shape, bool kMany, typename Args>
__device__ __forceinline__ Sequence load_sequence(const Args& a, const TiledPlan& plan, int b) {
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
    s.steps = kUnitSteps + (kMany && few ? keys / Shape::kFewStepKeys : keys / kStepKeys);
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
template <typename Shape, bool kMany, typename Args>
__device__ __forceinline__ ShareStart find_share(const Args& a, const TiledPlan& plan, int index,
                                                 uint32_t* lds_sums, ShareStart* lds_found) {
  constexpr int kThreads = Shape::kThreads;
  constexpr int kWaves = kThreads / 64;
  const int t = threadIdx.x;
  const int per = (a.batch + kThreads - 1) / kThreads;
  uint32_t mine = 0;
  Sequence seq{};
  for (int k = 0; k < per; ++k) {
    const int b = t * per + k;
    if (b < a.batch) {
      seq = load_sequence<Shape, kMany>(a, plan, b);
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
      if (per > 1) seq = load_sequence<Shape, kMany>(a, plan, b);
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
template <typename Number>
struct Piece {
  const int32_t* table;
  const Number* keys;    // the kv head's, of page 0
  const Number* values;
  int kv;
  int before;      // positions before the tile's first token
  int row0;        // the tile's first row
  int rows;        // packed rows
  int seen_first;  // keys that the tile's first and last token see
  int seen_last;
  int key0;        // keys [key0, key1)
  int key1;
  int slot;        // partial slot, or -1: the unit is whole
  int done;        // steps of the share before it
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
template <typename Shape, int kRF>
struct TiledRows {
  mfma_in8 q[kRF][Shape::kSteps];
  mfma_acc4 o[kRF][Shape::kDFrags];
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
      for (int df = 0; df < Shape::kDFrags; ++df) o[rf][df] = mfma_acc4{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ __forceinline__ void add_special() {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) {
      if (!__any((up[rf] | down[rf]) != 0)) continue;
#pragma unroll
      for (int df = 0; df < Shape::kDFrags; ++df) {
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
template <typename Shape, int kRF, typename Args, typename PieceT>
__device__ __forceinline__ void load_rows(TiledRows<Shape, kRF>& rows, const Args& a, const TiledPlan& plan,
                                          const PieceT& p, int row0) {
  const int col = lane_id() & 15;
  const int grp = lane_id() >> 4;
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const int r = min(row0 + 16 * rf + col, p.rows - 1);
    const int token = packed_token(plan, r);
    const int head = p.kv * a.group + r - token * a.group;
    const elem_t* q = a.q + static_cast<size_t>(p.row0 + token) * a.q_row_stride +
                      static_cast<size_t>(head) * Shape::kHeadDim;
#pragma unroll
    for (int ks = 0; ks < Shape::kSteps; ++ks) rows.q[rf][ks] = as_operand(load16(q + Shape::q_dim(ks, grp)));
    rows.seen[rf] = min(keys_seen(a, p.before, token), p.key1);
  }
}

// Waits for the queries here. Left to their first use, inside the loop over the
// tiles, the compiler's wait for them there is one for every direct load in
// flight, each time round.
template <typename Shape, int kRF>
__device__ __forceinline__ void hold_rows(TiledRows<Shape, kRF>& rows) {
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
#pragma unroll
    for (int ks = 0; ks < Shape::kSteps; ++ks) asm volatile("" : "+v"(rows.q[rf][ks]));
  }
}

// 16 kKF keys of a tile against the rows: scores, weights, values.
// A Tile gives the operands:
//   key(kf, ks)       of 16 keys and a k-step of their dims
//   value(half, df)   of 16 dims and 32 keys
template <typename Shape, int kRF, int kKF>
struct TileWork {
  using Rows = TiledRows<Shape, kRF>;
  mfma_acc4 s[kRF][kKF];
  uint32_t packed[kRF][kKF][2];

  template <typename Tile>
  __device__ __forceinline__ void scores(const Rows& rows, const Tile& tile) {
#pragma unroll
    for (int kf = 0; kf < kKF; ++kf) {
#pragma unroll
      for (int rf = 0; rf < kRF; ++rf) s[rf][kf] = mfma_acc4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < Shape::kSteps; ++ks) {
        const mfma_in8 k = tile.key(kf, ks);
#pragma unroll
        for (int rf = 0; rf < kRF; ++rf) s[rf][kf] = mfma16x16x32(k, rows.q[rf][ks], s[rf][kf]);
      }
    }
  }

  __device__ __forceinline__ void mask(const Rows& rows, int key0) {
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
  __device__ __forceinline__ void raise_base(Rows& rows, float c) {
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
  __device__ __forceinline__ void weights(const Rows& rows, float c, int half) {
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
  template <typename Tile>
  __device__ __forceinline__ void products(Rows& rows, const Tile& tile, int half) {
    constexpr uint32_t kOnes = kOneBits << 16 | kOneBits;
    const mfma_in8 ones = as_operand(vec16{{kOnes, kOnes, kOnes, kOnes}});
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) rows.sum[rf] = mfma16x16x32(ones, weight_operand(rf, half), rows.sum[rf]);
#pragma unroll
    for (int df = 0; df < Shape::kDFrags; ++df) {
      const mfma_in8 v = tile.value(half, df);
#pragma unroll
      for (int rf = 0; rf < kRF; ++rf) rows.o[rf][df] = mfma16x16x32(v, weight_operand(rf, half), rows.o[rf][df]);
    }
  }

  // 1 for each of 32 keys that a lane's row sees, in the order of weight_operand.
  __device__ __forceinline__ mfma_in8 seen_operand(const Rows& rows, int rf, int half, int key0) const {
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
  template <typename Tile>
  __device__ __forceinline__ void mark_special(Rows& rows, const Tile& tile, int key0) {
#pragma unroll
    for (int half = 0; half < kKF / 2; ++half) {
#pragma unroll 1
      for (int df = 0; df < Shape::kDFrags; ++df) {
        const vec16 v = __builtin_bit_cast(vec16, tile.value(half, df));
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

// A page outside the pool is read as page 0, and `bad` set.
template <typename Args>
__device__ __forceinline__ int pool_page(const Args& a, int page, int& bad) {
  const bool inside = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pool_pages);
  bad |= inside ? 0 : 1;
  return inside ? page : 0;
}

// One element's place in the output, from a packed row.
template <int kHeadDim, typename Args, typename PieceT>
__device__ __forceinline__ size_t out_at(const Args& a, const TiledPlan& plan, const PieceT& p, int r) {
  const int token = packed_token(plan, r);
  return (static_cast<size_t>(p.row0 + token) * a.num_heads + p.kv * a.group + (r - token * a.group)) *
         kHeadDim;
}

template <int kHeadDim>
__device__ __forceinline__ float* partial_stats(const TiledPlan& plan, int kv_heads, int tile_rows) {
  return plan.partials + static_cast<size_t>(2 * plan.shares) * kv_heads * tile_rows * kHeadDim;
}

// The waves' results of at most 32 rows meet in LDS, each in a part of kPitch floats
// of `outputs` that the wave alone used before, their bases and sums in `stats`.
template <typename Shape, int kTileRows, int kPitch, int kRF, typename Args, typename PieceT>
__device__ __forceinline__ void join_waves(TiledRows<Shape, kRF>& rows, int bad, float* all_outputs,
                                           float (*all_stats)[kFewRows][2], const Args& a, const TiledPlan& plan,
                                           const PieceT& p) {
  constexpr int kHeadDim = Shape::kHeadDim;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int col = lane_id() & 15;
  const int grp = lane_id() >> 4;
  rows.add_special();
  if (__any(bad != 0)) {
#pragma unroll
    for (int rf = 0; rf < kRF; ++rf) rows.sum[rf][0] = __builtin_nanf("");
  }
  float* outputs = all_outputs + wave * kPitch;
  static_assert(kPitch >= 16 * kRF * kHeadDim, "a wave's outputs fit");
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const float sum = rows.sum[rf][0];
    if (grp == 0) {
      all_stats[wave][16 * rf + col][0] = rows.base[rf];
      all_stats[wave][16 * rf + col][1] = sum;
    }
#pragma unroll
    for (int n = 0; n < Shape::kDFrags; ++n) {
      *reinterpret_cast<mfma_acc4*>(outputs + (16 * rf + col) * kHeadDim + Shape::out_dim(n, grp)) =
          Shape::out_piece(rows.o[rf], n);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.rows * (kHeadDim / 4); i += Shape::kThreads) {
    const int r = i / (kHeadDim / 4);
    const int d = i % (kHeadDim / 4) * 4;
    float base = all_stats[0][r][0];
#pragma unroll
    for (int w = 1; w < Shape::kWaves; ++w) base = fminf(base, all_stats[w][r][0]);
    float sum = 0.0f;
    mfma_acc4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < Shape::kWaves; ++w) {
      const float from = all_stats[w][r][0];
      // a wave that saw no key has base +inf and nothing to add
      const float move = from == __builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(base - from);
      sum = __builtin_fmaf(all_stats[w][r][1], move, sum);
      const mfma_acc4 x =
          *reinterpret_cast<const mfma_acc4*>(all_outputs + w * kPitch + r * kHeadDim + d);
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

// A wave's 32 of many rows, from packed row row0 on: stored, or left as a partial.
template <typename Shape, int kRF, typename Args, typename PieceT>
__device__ __forceinline__ void store_rows(const TiledRows<Shape, kRF>& rows, bool spoilt, int row0, const Args& a,
                                           const TiledPlan& plan, const PieceT& p) {
  constexpr int kHeadDim = Shape::kHeadDim;
  constexpr int kTileRows = Shape::kTileRows;
  const int col = lane_id() & 15;
  const int grp = lane_id() >> 4;
#pragma unroll
  for (int rf = 0; rf < kRF; ++rf) {
    const int r = row0 + 16 * rf + col;
    float sum = rows.sum[rf][0];
    if (spoilt) sum = __builtin_nanf("");
    if (r >= p.rows) continue;
    if (p.slot >= 0) {
      const size_t at = static_cast<size_t>(p.slot) * kTileRows + r;
#pragma unroll
      for (int n = 0; n < Shape::kDFrags; ++n) {
        *reinterpret_cast<mfma_acc4*>(plan.partials + at * kHeadDim + Shape::out_dim(n, grp)) =
            Shape::out_piece(rows.o[rf], n);
      }
      if (grp == 0) {
        float* stats = partial_stats<kHeadDim>(plan, a.view.num_kv_heads, kTileRows) + at * 2;
        stats[0] = rows.base[rf];
        stats[1] = sum;
      }
    } else {
      const bool any = keys_seen(a, p.before, packed_token(plan, r)) > 0;
      const float inv = any ? 1.0f / sum : 0.0f;
      elem_t* out = a.out + out_at<kHeadDim>(a, plan, p, r);
#pragma unroll
      for (int n = 0; n < Shape::kDFrags; ++n) {
        const mfma_acc4 o = Shape::out_piece(rows.o[rf], n);
        uint2 words;
        words.x = any ? pack_elems(o[0] * inv, o[1] * inv) : 0u;
        words.y = any ? pack_elems(o[2] * inv, o[3] * inv) : 0u;
        *reinterpret_cast<uint2*>(out + Shape::out_dim(n, grp)) = words;
      }
    }
  }
}

// A block's share, piece by piece: few(piece) for pieces of at most 32 rows,
// many(piece) for others (kMany).
// begin(steps) is told the share's length.
template <typename Shape, bool kMany, typename Number, typename Args, typename Begin, typename Few, typename Many>
__device__ __forceinline__ void walk_share(const Args& a, const TiledPlan& plan, uint32_t* sums, ShareStart* found_at,
                                           const Begin& begin, const Few& few, const Many& many) {
  constexpr int kHeadDim = Shape::kHeadDim;
  // Share: neighbours on one XCD where the grid is a multiple of 8.
  const unsigned blocks = gridDim.x;
  const int block = static_cast<int>(Shape::kNeighbours && blocks % 8u == 0
                                         ? blockIdx.x % 8u * (blocks / 8u) + blockIdx.x / 8u
                                         : blockIdx.x);
  const int kv = plan.by_shares(block);
  const ShareStart found =
      find_share<Shape, kMany>(a, plan, block - kv * plan.shares, sums, found_at);
  if (plan.split && threadIdx.x == 0) plan.cuts[block].rows = 0;
  if (found.sequence < 0) return;
  int b = found.sequence;
  Sequence seq = found.seq;
  int at = (block - kv * plan.shares) * found.share;
  const int first = at;
  const int end = min(at + found.share, found.total);
  begin(end - first);
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
  Piece<Number> p;
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
    p.done = max(start, at) - first;
    // A short unit is not cut: it goes to the share that it begins in.
    const bool whole = !plan.split || stop - start <= kWholeSteps<kMany>;
    if (!whole && (start < at || stop > end)) {
      // steps into the unit, in keys
      const int keys = kMany && single ? Shape::kFewStepKeys : kStepKeys;
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
        if constexpr (kMany) many(p);
      } else {
        few(p);
      }
    }
    at = stop;
    if (at >= end) break;
    if (!kMany || ++tile >= seq.tiles) {
      tile = 0;
      before += seq.steps;
      do {  // the next sequence that has rows
        if (++b == a.batch) return;
        seq = uniform(load_sequence<Shape, kMany>(a, plan, b));
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

template <int kHeadDim, bool kRowEach, typename Args>
__global__ __launch_bounds__(kJoinThreads) void batch_attention_join_kernel(Args a, TiledPlan plan, int tile_rows) {
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

// A kv head's shares: all heads' together are the blocks resident at once.
template <typename Shape>
int tiled_shares(int kv_heads, bool many) {
  const int blocks = many ? Shape::kBlocks : Shape::kFewBlocks;
  return std::max(1, device_compute_units() * blocks / kv_heads);
}

bool many_rows_possible(int max_new, int group) { return static_cast<long long>(max_new) * group > kFewRows; }

template <typename Shape>
size_t tiled_workspace(int max_new, int kv_heads, int group) {
  const bool many = many_rows_possible(max_new, group);
  const size_t rows = many ? Shape::kTileRows : kFewRows;
  const size_t shares = static_cast<size_t>(tiled_shares<Shape>(kv_heads, many)) * static_cast<size_t>(kv_heads);
  return shares * (sizeof(CutUnit) + 2 * rows * (Shape::kHeadDim + 2) * sizeof(float));
}

template <typename Shape>
int tiled_tile_tokens(int group) {
  return std::max(1, Shape::kTileRows / group);
}

// A unit a block: at most one short tile a sequence beside the full ones.
template <typename Shape, typename Args>
long long most_tiled_units(const Args& a) {
  return a.tokens / tiled_tile_tokens<Shape>(a.group) + static_cast<long long>(a.batch);
}

template <typename Shape, typename Args>
TiledPlan plan_tiled(const Args& a, void* workspace, size_t workspace_bytes) {
  TiledPlan plan{};
  const int kv_heads = a.view.num_kv_heads;
  plan.group_magic = static_cast<uint32_t>((65536 + a.group - 1) / a.group);
  plan.tile_tokens = tiled_tile_tokens<Shape>(a.group);
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
  const bool half_idle = many && 2 * most_tiled_units<Shape>(a) * kv_heads <= device_compute_units();
  const int cut_positions = half_idle ? 768 : 1024;
  // Steps are counted in 32 bits. Where a call's could pass them, it has units
  // enough to fill the device uncut.
  const long long most_units = many ? most_tiled_units<Shape>(a) : a.batch;
  const long long most_steps = kUnitSteps + 1 + std::max(a.held, std::min(a.max_new, a.tokens)) / kStepKeys;
  if (a.held > cut_positions && most_units * most_steps <= kMostSteps && workspace != nullptr &&
      workspace_bytes >= tiled_workspace<Shape>(a.max_new, kv_heads, a.group)) {
    plan.split = 1;
    plan.shares = tiled_shares<Shape>(kv_heads, many);
    plan.cuts = static_cast<CutUnit*>(workspace);
    plan.partials = reinterpret_cast<float*>(plan.cuts + static_cast<size_t>(plan.shares) * kv_heads);
  } else {
    plan.shares = static_cast<int>(most_tiled_units<Shape>(a));
  }
  plan.by_shares = FastDivide::by(static_cast<uint32_t>(plan.shares));
  return plan;
}

}  // namespace
}  // namespace lcr
