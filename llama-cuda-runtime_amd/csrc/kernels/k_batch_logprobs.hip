// lcr_batch_logprobs: log probabilities of given tokens, with their rows'
// entropies and likeliest ids.
//
// One pass over the logits: with m the largest so far, a lane keeps
//   s = sum e^(l - m),  t = sum e^(l - m) (l - m)
// and moves both when m rises by d: s' = s e^-d, t' = (t - d s) e^-d. From a row's,
//   log p = l - m - log s,  entropy = log s - t / s.
// Sixteen logits at a time are summed in fp32, and those sums in fp64.
//
// The likeliest ids need no order of all logits: the k-th largest of 64 columns'
// largest logits is one that at least k logits reach, and few others do. The tiles in
// which a lane reaches it are read again, and logits at least as large (few more than
// k) are ranked by counting. The streaming pass does nothing for it but keep the largest.
//
// Bound by memory: 11 operations a logit, the exponential four times as long as the
// others, are half of the vector units' time at the rate that logits arrive. 1500 rows
// of 50001 logits 49 us, 6.1 TB/s of a streaming read's 7.0; 700 of 128256 with 8 ids
// 62 us, 5.8, without ids 56. One row, in 16 parts: 5 us for the parts, 7.5 to join them
// and choose, chains of some ten reads and exchanges.
#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "device_common.h"

namespace lcr {
namespace {

// Threads of a block. A row of few tiles has little for many waves, and its choice of
// likeliest ids, a chain of short steps, wants more blocks beside it: 4000 rows of
// 8000 logits 46 us by blocks of 512 threads, 33 by 256; 256 rows of 128256 28 and 33.
constexpr int kManyThreads = 512;
constexpr int kFewThreads = 256;
constexpr int kFewThreadTiles = 16;
constexpr int kTile = 1024;            // logits of a wave's step: four times four a lane
constexpr int kMostCandidates = 1024;
constexpr int kMostTop = LCR_BATCH_MAX_ALTERNATIVES;
constexpr float kLog2e = 1.44269504088896340736f;

// What a part of a row comes to.
struct alignas(16) PartSums {
  double sum;
  double weighted;
  float max;
  int above;   // logits larger than the given token's
  int hot;     // the lowest index of the largest logit, where it is not finite
};

struct LogprobArgs {
  float* logprobs;
  int32_t* ranks;
  float* entropies;
  int32_t* top_ids;
  float* top_logprobs;
  const float* logits;
  const int32_t* token_ids;
  int top;
  int vocab;
  int logits_stride;
  int parts;
  PartSums* sums;   // [rows][parts]
  float* largest;   // [rows][parts][kManyThreads]: of each thread's logits
};

__device__ __forceinline__ float infinity() { return __builtin_huge_valf(); }
__device__ __forceinline__ float clean(float l) { return l == l ? l : -infinity(); }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < infinity(); }

// A logit's order: by value (zeros of both signs are equal), equal ones by ascending
// id. A larger key is before a smaller.
__device__ __forceinline__ unsigned long long key_of(float l, int id) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, l + 0.0f);
  const uint32_t ordered = bits ^ (static_cast<uint32_t>(static_cast<int>(bits) >> 31) | 0x80000000u);
  return static_cast<unsigned long long>(ordered) << 32 | (0xffffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t ordered = static_cast<uint32_t>(key >> 32);
  return __builtin_bit_cast(float, ordered & 0x80000000u ? ordered ^ 0x80000000u : ~ordered);
}
__device__ __forceinline__ int id_of(unsigned long long key) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}

// The largest of three, or NaN if one is. (Of a signalling NaN the other maximum
// makes a quiet one, which the next takes for none: what it was compared with is
// lost.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// e^d of a difference to the largest, d clamped so that -inf and NaN weigh nothing
// (and 0 times them is 0).
__device__ __forceinline__ float below(float l, float max) { return fmaxf(l - max, -3.0e38f); }
__device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// A row in tiles of kTile places, cut into parts. Loads are 16-byte aligned, so that
// index i of the row is place i + shift of them; places outside the row hold -inf.
struct RowTiles {
  const float* row;
  int shift;   // 0 .. 3
  int places;  // shift + vocab
  int tiles;
  int parts;

  __device__ __forceinline__ RowTiles(const LogprobArgs& a, int r)
      : row(a.logits + static_cast<size_t>(r) * static_cast<size_t>(a.logits_stride)),
        shift(static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 2 & 3u)),
        places(shift + a.vocab),
        tiles((places + kTile - 1) / kTile),
        parts(a.parts) {}

  // The first tile of a part (tiles are at most 2^20 + 1, parts 32).
  __device__ __forceinline__ int first_tile(int part) const { return tiles * part / parts; }

  // Places 4 g .. 4 g + 3.
  __device__ __forceinline__ float4 load(int g) const {
    const int at = 4 * g - shift;
    if (at >= 0 && at <= places - shift - 4) return *reinterpret_cast<const float4*>(row + at);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = at + i >= 0 && at + i < places - shift ? row[at + i] : -infinity();
    return make_float4(v[0], v[1], v[2], v[3]);
  }
};

// A lane's four times four places of a tile.
struct Tile {
  float l[16];

  __device__ __forceinline__ void load(const RowTiles& p, int tile) {
    const int g = tile * (kTile / 4) + lane_id();
    // whole tiles without a test of each load
    const bool whole = 1024 * tile >= p.shift && 1024 * tile + 1023 < p.places;
    if (whole) {
      const float* from = p.row + (4 * g - p.shift);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        typedef float f32x4 __attribute__((ext_vector_type(4)));
        const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(from + 256 * j));
        l[4 * j] = v.x;
        l[4 * j + 1] = v.y;
        l[4 * j + 2] = v.z;
        l[4 * j + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 v = p.load(g + 64 * j);
        l[4 * j] = v.x;
        l[4 * j + 1] = v.y;
        l[4 * j + 2] = v.z;
        l[4 * j + 3] = v.w;
      }
    }
  }
};

constexpr int kMostParts = 32;

constexpr int kMostSlots = 16;
constexpr int kMostReads = 1024;

// What the choice of likeliest ids needs.
template <int kThreads>
struct ChoiceLds {
  static constexpr int kWaves = kThreads / 64;
  float largest[kWaves][64];
  unsigned long long candidates[kMostCandidates];
  uint16_t reads[kMostReads];   // what is read again, as the Source names it
  int found[kWaves];
  int read_count;
  int count;   // of candidates
};

template <int kWaves>
struct SumsLds {
  double sums[kWaves][2];
  float max[kWaves];
  int above[kWaves];
  int hot[kWaves];
};

// A place in a list for each lane that `wants` one: one count a wave, not a lane.
__device__ __forceinline__ int take_place(int* count, bool wants) {
  const unsigned long long mask = __ballot(wants);
  if (mask == 0) return 0;
  int base = 0;
  if (lane_id() == 0) base = atomicAdd(count, __popcll(mask));
  return __builtin_amdgcn_readfirstlane(base) + __popcll(mask & ((1ull << lane_id()) - 1));
}

// A compare and exchange over lanes kMask apart: the larger to the lower lane where
// `down`.
template <int kMask>
__device__ __forceinline__ float exchange(float v, bool down) {
  const float other = xor_lane<kMask>(v);
  const bool lower = (lane_id() & kMask) == 0;
  return lower == down ? fmaxf(v, other) : fminf(v, other);
}

// A wave's 64 values in descending order.
__device__ __forceinline__ float sort_wave(float v) {
  const int lane = lane_id();
  v = exchange<1>(v, (lane & 2) == 0);
  v = exchange<2>(v, (lane & 4) == 0);
  v = exchange<1>(v, (lane & 4) == 0);
  v = exchange<4>(v, (lane & 8) == 0);
  v = exchange<2>(v, (lane & 8) == 0);
  v = exchange<1>(v, (lane & 8) == 0);
  v = exchange<8>(v, (lane & 16) == 0);
  v = exchange<4>(v, (lane & 16) == 0);
  v = exchange<2>(v, (lane & 16) == 0);
  v = exchange<1>(v, (lane & 16) == 0);
  v = exchange<16>(v, (lane & 32) == 0);
  v = exchange<8>(v, (lane & 32) == 0);
  v = exchange<4>(v, (lane & 32) == 0);
  v = exchange<2>(v, (lane & 32) == 0);
  v = exchange<1>(v, (lane & 32) == 0);
  v = exchange<32>(v, true);
  v = exchange<16>(v, true);
  v = exchange<8>(v, true);
  v = exchange<4>(v, true);
  v = exchange<2>(v, true);
  return exchange<1>(v, true);
}

// The top-th largest of 64 values, each the largest that one lane of all waves has: a
// bound that at least `top` logits of the block reach, and not many more. (With 20 of
// 64, some 24. The exact one of all the lanes' takes three more merges and barriers.)
template <int kThreads>
__device__ __forceinline__ float largest_reached(ChoiceLds<kThreads>& lds, float v, int top) {
  constexpr int kWaves = kThreads / 64;
  lds.largest[threadIdx.x >> 6][lane_id()] = v;
  __syncthreads();
  v = lds.largest[0][lane_id()];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = fmaxf(v, lds.largest[w][lane_id()]);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sort_wave(v)), top - 1));
}

// Upper bits of a value's place in the order of values.
__device__ __forceinline__ uint32_t order16(float l) { return static_cast<uint32_t>(key_of(l, 0) >> 48); }

// Where a thread's logits of a whole row were: its tiles in up to kMostSlots groups,
// with the upper bits of each group's largest.
template <int kThreads>
struct RowSource {
  static constexpr int kWaves = kThreads / 64;
  uint16_t (*most)[kThreads];
  float largest;
  int steps;   // a wave's tiles, at most
  int group;   // steps of a slot

  // Names to `take` what may hold logits that `counts` (at or above reach) takes.
  template <typename Counts, typename Take>
  __device__ __forceinline__ void find(float reach, const Counts& counts, const Take& take) const {
    const bool mine = counts(largest);
    if (!__any(mine)) return;
    const uint32_t least = max(order16(reach), order16(-infinity()) + 1);
    for (int slot = 0; slot * group < steps; ++slot) {
      take(mine && most[slot][threadIdx.x] >= least, static_cast<int>(threadIdx.x) * kMostSlots + slot);
    }
  }
  // Fours of logits behind a name, and the place of one, or -1.
  __device__ __forceinline__ int fours() const { return 4 * group; }
  __device__ __forceinline__ int four_at(const RowTiles& p, int name, int four) const {
    const int thread = name / kMostSlots;
    const int tile = (thread >> 6) + kWaves * (name % kMostSlots * group + (four >> 2));
    return tile < p.tiles ? tile * (kTile / 4) + 64 * (four & 3) + (thread & 63) : -1;
  }
};

// Of a row in parts: a thread's largest of each.
template <int kThreads>
struct PartsSource {
  static constexpr int kWaves = kThreads / 64;
  const float (&largest)[kMostParts];
  int parts;
  int steps;

  template <typename Counts, typename Take>
  __device__ __forceinline__ void find(float, const Counts& counts, const Take& take) const {
#pragma unroll
    for (int part = 0; part < kMostParts; ++part) {
      if (part < parts) take(counts(largest[part]), part * kThreads + static_cast<int>(threadIdx.x));
    }
  }
  __device__ __forceinline__ int fours() const { return 4 * steps; }
  __device__ __forceinline__ int four_at(const RowTiles& p, int name, int four) const {
    const int part = name / kThreads, thread = name % kThreads;
    const int tile = p.first_tile(part) + (thread >> 6) + kWaves * (four >> 2);
    return tile < p.first_tile(part + 1) ? tile * (kTile / 4) + 64 * (four & 3) + (thread & 63) : -1;
  }
};

// The row's logits at or above (kAbove: above) `reach` as candidates; -inf is none.
// What the lanes that reach it had is read again, four logits at a time, by the whole
// block. 256 rows of 128256, 20 ids: with those lanes reading theirs, one step behind
// the other, 60 us; all that they had by the block 30; the tiles that reach it 28; no
// ids at all 22.
template <bool kAbove, int kThreads, typename Source>
__device__ __forceinline__ int gather(ChoiceLds<kThreads>& lds, const RowTiles& p, float reach, const Source& source) {
  auto counts = [&](float l) { return (kAbove ? l > reach : l >= reach) && l > -infinity(); };
  if (threadIdx.x == 0) lds.count = lds.read_count = 0;
  __syncthreads();
  source.find(reach, counts, [&](bool wanted, int name) {
    const int at = take_place(&lds.read_count, wanted);
    if (wanted && at < kMostReads) lds.reads[at] = static_cast<uint16_t>(name);
  });
  __syncthreads();
  if (lds.read_count > kMostReads) {
    __syncthreads();  // it may be counted in again
    return kMostCandidates + 1;
  }
  const uint32_t fours = static_cast<uint32_t>(source.fours());
  const uint32_t items = static_cast<uint32_t>(lds.read_count) * fours;  // under 2^30
  constexpr int kAtOnce = 2;
  for (uint32_t first = 0; first < items; first += kAtOnce * kThreads) {
    float4 v[kAtOnce];
    int g[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const uint32_t item = first + n * kThreads + threadIdx.x;
      const uint32_t read = item < items ? item / fours : 0;
      g[n] = item < items ? source.four_at(p, lds.reads[read], static_cast<int>(item - read * fours)) : -1;
      v[n] = g[n] >= 0 ? p.load(g[n]) : make_float4(-infinity(), -infinity(), -infinity(), -infinity());
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const float l[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool wanted = counts(l[i]);
        const int at = take_place(&lds.count, wanted);
        if (wanted && at < kMostCandidates) lds.candidates[at] = key_of(l[i], 4 * g[n] + i - p.shift);
      }
    }
    // more than there is room for: counted no further
    if (lds.count > kMostCandidates) break;
  }
  __syncthreads();
  const int n = lds.count;
  __syncthreads();  // it may be counted in again
  return n;
}

// Adds the first `want` of the row's logits that equal `reach`, in the order of
// their ids, behind `have` candidates.
template <int kThreads>
__device__ __forceinline__ void gather_equal(ChoiceLds<kThreads>& lds, const RowTiles& p, float reach, int have,
                                             int want) {
  constexpr int kWaves = kThreads / 64;
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int vocab = p.places - p.shift;
  for (int base = 0; base < vocab && want > 0; base += kThreads) {
    const int i = base + static_cast<int>(threadIdx.x);
    const bool equal = i < vocab && p.row[i] == reach;
    const unsigned long long mask = __ballot(equal);
    if (lane_id() == 0) lds.found[wave] = __popcll(mask);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += lds.found[w];
      all += lds.found[w];
    }
    before += __popcll(mask & ((1ull << lane_id()) - 1));
    if (equal && before < want) lds.candidates[have + before] = key_of(reach, i);
    have += min(all, want);
    want -= min(all, want);
    __syncthreads();
  }
}

// The row's `top` largest, one pass over it for each: for rows with too many
// candidates, whose large logits all lie with few lanes.
template <int kThreads>
__device__ __forceinline__ int gather_slowly(ChoiceLds<kThreads>& lds, const RowTiles& p, int top) {
  constexpr int kWaves = kThreads / 64;
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int vocab = p.places - p.shift;
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const float l = p.row[i];
      if (!(l > -infinity())) continue;
      const unsigned long long key = key_of(l, i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long other = __shfl_xor(best, o, 64);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane_id() == 0) lds.candidates[kMostTop + wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
      const unsigned long long other = lds.candidates[kMostTop + w];
      best = other > best ? other : best;
    }
    if (best == 0) {
      __syncthreads();
      return k;
    }
    if (threadIdx.x == 0) lds.candidates[k] = best;
    last = best;
  }
  __syncthreads();
  return top;
}

// Hands (rank, key) of the `top` first of n candidates to `out`.
template <int kThreads, typename Out>
__device__ __forceinline__ void rank(const unsigned long long* candidates, int n, int top, const Out& out) {
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const unsigned long long key = candidates[c];
    int ahead = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) ahead += candidates[i] > key ? 1 : 0;
    if (ahead < top) out(ahead, key);
  }
}

// A row's distribution, and what is written of it.
struct RowResult {
  double log_sum;
  float max;
  int hot;   // p is 1 there; -1: the largest logit is finite

  __device__ __forceinline__ float logprob(float l, int id) const {
    if (hot >= 0) return id == hot ? 0.0f : -infinity();
    return static_cast<float>(static_cast<double>(l) - static_cast<double>(max) - log_sum);
  }
};

__device__ __forceinline__ RowResult result_of(const PartSums& s) {
  const bool hot = !finite(s.max);
  return RowResult{hot ? 0.0 : log(s.sum), s.max, hot ? s.hot : -1};
}

// Thread 0's part of a row's answer.
__device__ __forceinline__ void write_row(const LogprobArgs& a, int row, int token, float given, const PartSums& s,
                                          const RowResult& r) {
  if (token >= 0) {
    const bool inside = token < a.vocab;
    if (a.logprobs != nullptr) a.logprobs[row] = inside ? r.logprob(given, token) : -infinity();
    if (a.ranks != nullptr) a.ranks[row] = inside ? s.above : a.vocab;
  }
  if (a.entropies != nullptr) a.entropies[row] = r.hot >= 0 ? 0.0f : static_cast<float>(r.log_sum - s.weighted / s.sum);
}

__device__ __forceinline__ void write_top(const LogprobArgs& a, int row, int place, float logprob, int id) {
  const size_t at = static_cast<size_t>(row) * a.top + place;
  a.top_ids[at] = id;
  a.top_logprobs[at] = logprob;
}

// A row's likeliest ids.
template <int kThreads, typename Source>
__device__ __forceinline__ void choose(ChoiceLds<kThreads>& lds, const LogprobArgs& a, const RowTiles& p, int row,
                                       float thread_largest, const Source& source, const RowResult& result) {
  const float reach = largest_reached(lds, thread_largest, a.top);
  int n = gather<false>(lds, p, reach, source);
  if (n > kMostCandidates) {
    // Many equal ones (a mask of the type's lowest value), or many in few lanes.
    n = gather<true>(lds, p, reach, source);
    if (n <= kMostCandidates - kMostTop) {
      const int want = max(a.top - n, 0);
      gather_equal(lds, p, reach, n, want);
      n += want;
    } else {
      n = gather_slowly(lds, p, a.top);
    }
  }
  rank<kThreads>(lds.candidates, n, a.top, [&](int place, unsigned long long key) {
    write_top(a, row, place, result.logprob(value_of(key), id_of(key)), id_of(key));
  });
  for (int place = min(n, a.top) + static_cast<int>(threadIdx.x); place < a.top; place += kThreads) {
    write_top(a, row, place, -infinity(), -1);
  }
}

struct Nothing {};

// A row (kPart: a part of one) a block.
template <bool kTop, bool kPart, int kThreads>
__global__ __launch_bounds__(kThreads, 4) void logprobs_kernel(LogprobArgs a) {
  constexpr int kWaves = kThreads / 64;
  __shared__ SumsLds<kWaves> lds;
  __shared__ std::conditional_t<kTop && !kPart, ChoiceLds<kThreads>, Nothing> choice;
  __shared__ std::conditional_t<kTop && !kPart, uint16_t[kMostSlots][kThreads], Nothing> slot_most;
  const int row = kPart ? blockIdx.y : blockIdx.x;
  const int part = kPart ? blockIdx.x : 0;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int token = a.token_ids != nullptr ? a.token_ids[row] : -1;
  if (a.token_ids != nullptr && token < 0) return;  // the row is left out
  const RowTiles p(a, row);
  const int tile0 = kPart ? p.first_tile(part) : 0;
  const int tile1 = kPart ? p.first_tile(part + 1) : p.tiles;

  Tile next;
  int tile = tile0 + wave;
  if (tile < tile1) next.load(p, tile);
  const float given = token >= 0 && token < a.vocab ? clean(p.row[token]) : infinity();
  float largest = -infinity();
  double sum = 0.0, weighted = 0.0;
  int above = 0;
  const int steps = (p.tiles + kWaves - 1) / kWaves;  // of a whole row
  const int group = (steps + kMostSlots - 1) / kMostSlots;
  float group_most = -infinity();
  int slot = 0, in_group = 0;
  if constexpr (kTop && !kPart) {
#pragma unroll
    for (int n = 0; n < kMostSlots; ++n) slot_most[n][threadIdx.x] = 0;
  }
  for (; tile < tile1; tile += kWaves) {
    Tile now = next;
    if (tile + kWaves < tile1) next.load(p, tile + kWaves);
    float most = max3(now.l[0], now.l[1], now.l[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) most = max3(most, now.l[i], now.l[i + 1]);
    most = max3(most, now.l[15], -infinity());
    if (__any(most != most)) {
      most = -infinity();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        now.l[i] = clean(now.l[i]);
        most = fmaxf(most, now.l[i]);
      }
    }
    // the token's rank: tiles without a larger logit are most
    if (__any(most > given)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) above += __popcll(__ballot(now.l[i] > given));
    }
    if constexpr (kTop && !kPart) {
      group_most = in_group == 0 ? most : fmaxf(group_most, most);
      slot_most[slot][threadIdx.x] = static_cast<uint16_t>(order16(group_most));
      if (++in_group == group) {
        in_group = 0;
        ++slot;
      }
    }
    const float raised = fmaxf(largest, most);
    const float fall = below(largest, raised);
    const double keep = weight(fall);
    float s[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = below(now.l[i], raised);
      const float w = weight(d);
      s[i & 1] += w;
      t[i & 1] = __builtin_fmaf(w, d, t[i & 1]);
    }
    weighted = __builtin_fma(keep, __builtin_fma(sum, static_cast<double>(fall), weighted), static_cast<double>(t[0] + t[1]));
    sum = __builtin_fma(sum, keep, static_cast<double>(s[0] + s[1]));
    largest = raised;
  }
  if constexpr (kTop && kPart) {
    a.largest[(static_cast<size_t>(row) * a.parts + part) * kThreads + threadIdx.x] = largest;
  }

  // The lanes' sums against the block's largest logit, in a fixed order.
  const float wave_most = wave_max(largest);
  if (lane_id() == 0) lds.max[wave] = wave_most;
  __syncthreads();
  float most = lds.max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) most = fmaxf(most, lds.max[w]);
  const float fall = below(largest, most);
  const double keep = weight(fall);
  weighted = wave_sum_f64(keep * __builtin_fma(sum, static_cast<double>(fall), weighted));
  sum = wave_sum_f64(sum * keep);
  int hot = INT_MAX;
  if (!finite(most)) {
    for (int i = tile0 * kTile + static_cast<int>(threadIdx.x); i < min(tile1 * kTile, p.places); i += kThreads) {
      if (i >= p.shift && clean(p.row[i - p.shift]) == most) {
        hot = i - p.shift;
        break;
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) hot = min(hot, __shfl_xor(hot, o, 64));
  }
  if (lane_id() == 0) {
    lds.sums[wave][0] = sum;
    lds.sums[wave][1] = weighted;
    lds.above[wave] = above;
    lds.hot[wave] = hot;
  }
  __syncthreads();
  PartSums all{0.0, 0.0, most, 0, INT_MAX};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    all.sum += lds.sums[w][0];
    all.weighted += lds.sums[w][1];
    all.above += lds.above[w];
    all.hot = min(all.hot, lds.hot[w]);
  }
  if constexpr (kPart) {
    if (threadIdx.x == 0) a.sums[static_cast<size_t>(row) * a.parts + part] = all;
  } else {
    const RowResult result = result_of(all);
    if (threadIdx.x == 0) write_row(a, row, token, given, all, result);
    if constexpr (kTop) choose(choice, a, p, row, largest, RowSource<kThreads>{slot_most, largest, steps, group}, result);
  }
}

// Joins the parts of a row, a block each.
template <bool kTop>
__global__ __launch_bounds__(kManyThreads) void logprobs_join_kernel(LogprobArgs a) {
  constexpr int kThreads = kManyThreads;
  constexpr int kWaves = kThreads / 64;
  __shared__ std::conditional_t<kTop, ChoiceLds<kThreads>, Nothing> choice;
  const int row = blockIdx.x;
  const int token = a.token_ids != nullptr ? a.token_ids[row] : -1;
  if (a.token_ids != nullptr && token < 0) return;
  const RowTiles p(a, row);
  const int lane = lane_id();
  // Every wave joins the sums for itself, a part a lane.
  PartSums mine{0.0, 0.0, -infinity(), 0, INT_MAX};
  if (lane < a.parts) mine = a.sums[static_cast<size_t>(row) * a.parts + lane];
  const float given = token >= 0 && token < a.vocab ? clean(p.row[token]) : infinity();
  float each[kMostParts];
  float largest = -infinity();
  if constexpr (kTop) {
    const float* from = a.largest + static_cast<size_t>(row) * a.parts * kThreads + threadIdx.x;
#pragma unroll
    for (int part = 0; part < kMostParts; ++part) each[part] = part < a.parts ? from[part * kThreads] : -infinity();
#pragma unroll
    for (int part = 0; part < kMostParts; ++part) largest = fmaxf(largest, each[part]);
  }
  PartSums all;
  all.max = wave_max(mine.max);
  const float fall = below(mine.max, all.max);
  const double keep = weight(fall);
  all.sum = wave_sum_f64(mine.sum * keep);
  all.weighted = wave_sum_f64(keep * __builtin_fma(mine.sum, static_cast<double>(fall), mine.weighted));
  all.above = mine.above;
  all.hot = mine.max == all.max ? mine.hot : INT_MAX;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    all.above += __shfl_xor(all.above, o, 64);
    all.hot = min(all.hot, __shfl_xor(all.hot, o, 64));
  }
  const RowResult result = result_of(all);
  if (threadIdx.x == 0) write_row(a, row, token, given, all, result);
  if constexpr (kTop) {
    const int part_tiles = (p.tiles + p.parts - 1) / p.parts;  // at most
    choose(choice, a, p, row, largest, PartsSource<kThreads>{each, p.parts, (part_tiles + kWaves - 1) / kWaves}, result);
  }
}

// Parts that a row is cut into: as many as give each compute unit two, of no less
// than a step of each wave. With a row for every second compute unit the second
// launch and the reads of its own cost as much as they save: 64 rows of 128256 in
// parts 17.7 us, 128 as long either way, 200 in parts 28.5, whole 23.3.
int parts_for(int rows, int vocab) {
  const int compute_units = device_compute_units();
  if (2 * rows > compute_units) return 1;
  constexpr int kStep = kTile * kManyThreads / 64;
  const int steps = (vocab + kStep - 1) / kStep;
  return std::max(1, std::min({kMostParts, (2 * compute_units + rows - 1) / rows, steps}));
}

size_t workspace_for(int rows, int parts, int top) {
  return static_cast<size_t>(rows) * static_cast<size_t>(parts) *
         (sizeof(PartSums) + (top > 0 ? kManyThreads * sizeof(float) : 0));
}

template <bool kTop>
void launch_parts(const LogprobArgs& a, int rows, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.parts), static_cast<unsigned>(rows));
  logprobs_kernel<kTop, true, kManyThreads><<<grid, kManyThreads, 0, s>>>(a);
  logprobs_join_kernel<kTop><<<static_cast<unsigned>(rows), kManyThreads, 0, s>>>(a);
}

template <int kThreads>
void launch_rows(const LogprobArgs& a, int rows, hipStream_t s) {
  const unsigned blocks = static_cast<unsigned>(rows);
  if (a.top > 0) {
    logprobs_kernel<true, false, kThreads><<<blocks, kThreads, 0, s>>>(a);
  } else {
    logprobs_kernel<false, false, kThreads><<<blocks, kThreads, 0, s>>>(a);
  }
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" size_t lcr_batch_logprobs_workspace_bytes(int rows, int top, int vocab) {
  if (rows <= 0 || top < 0 || vocab <= 0) return 0;
  const int parts = parts_for(rows, vocab);
  return parts > 1 ? workspace_for(rows, parts, top) : 0;
}

extern "C" int lcr_batch_logprobs(float* logprobs, int32_t* ranks, float* entropies, int32_t* top_ids,
                                  float* top_logprobs, const float* logits, const int32_t* token_ids, int rows, int top,
                                  int vocab, int logits_stride, void* workspace, size_t workspace_bytes, void* stream) {
  CAPI_CHECK(rows >= 0 && top >= 0, "batch_logprobs needs non-negative sizes");
  CAPI_CHECK(top <= LCR_BATCH_MAX_ALTERNATIVES,
             "batch_logprobs takes up to " << LCR_BATCH_MAX_ALTERNATIVES << " alternatives, got " << top);
  if (rows == 0) return LCR_OK;
  CAPI_CHECK(vocab > 0, "batch_logprobs needs a vocabulary, got " << vocab);
  CAPI_CHECK(vocab <= (1 << 30), "batch_logprobs takes up to 2^30 ids, got " << vocab);
  CAPI_CHECK(logits_stride >= vocab, "rows of " << vocab << " logits cannot lie " << logits_stride << " apart");
  CAPI_CHECK(logits != nullptr, "batch_logprobs needs logits");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(logits) & 3u) == 0, "batch_logprobs needs logits on 4-byte boundaries");
  CAPI_CHECK(top == 0 || (top_ids != nullptr && top_logprobs != nullptr),
             "batch_logprobs needs room for its alternatives");
  CAPI_CHECK(token_ids != nullptr || (logprobs == nullptr && ranks == nullptr),
             "batch_logprobs needs the tokens whose probabilities it writes");
  CAPI_CHECK(workspace != nullptr || workspace_bytes == 0,
             "batch_logprobs workspace of " << workspace_bytes << " bytes has no pointer");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch_logprobs workspace must be 16-byte aligned");
  CAPI_CHECK(static_cast<long long>(rows) * kManyThreads <= UINT32_MAX,
             "batch_logprobs of " << rows << " rows needs more than 2^32 threads");
  LogprobArgs a{logprobs, ranks, entropies, top_ids, top_logprobs, logits, token_ids, top, vocab, logits_stride,
                1, nullptr, nullptr};
  auto s = static_cast<hipStream_t>(stream);
  const int parts = parts_for(rows, vocab);
  if (parts > 1 && workspace != nullptr && workspace_bytes >= workspace_for(rows, parts, top)) {
    a.parts = parts;
    a.sums = static_cast<PartSums*>(workspace);
    a.largest = reinterpret_cast<float*>(a.sums + static_cast<size_t>(rows) * parts);
    if (top > 0) {
      launch_parts<true>(a, rows, s);
    } else {
      launch_parts<false>(a, rows, s);
    }
  } else if (vocab <= kFewThreadTiles * kTile) {
    launch_rows<kFewThreads>(a, rows, s);
  } else {
    launch_rows<kManyThreads>(a, rows, s);
  }
  CAPI_LAUNCHED();
  return LCR_OK;
}
