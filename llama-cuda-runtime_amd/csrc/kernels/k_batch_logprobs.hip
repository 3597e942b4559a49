// lcr_batch_logprobs: log probabilities of given tokens, with their rows'
// entropies and likeliest ids.
//
// One pass over the logits: with m the largest so far, a lane keeps
//   s = sum e^(l - m),  t = sum e^(l - m) (l - m)
// and moves both when m rises by d: s' = s e^-d, t' = (t - d s) e^-d. From a row's,
//   log p = l - m - log s,  entropy = log s - t / s.
// Sixteen logits at a time are summed in fp32, and those sums in fp64.
//
// The likeliest ids need no second order of all logits: the k-th largest of the
// lanes' largest logits is one that at least k logits reach, and few others do. The
// lanes that hold one read theirs again, and those at least as large (about k) are
// ranked by counting. The streaming pass does nothing for it but keep the largest.
//
// Bound by memory: 11 operations a logit, the exponential four times as long as the
// others, are half of the vector units' time at the rate that logits arrive.
#include <algorithm>
#include <climits>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "device_common.h"

namespace lcr {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
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
  int count;   // of its likeliest ids
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
  PartSums* sums;            // [rows][parts]
  unsigned long long* keys;  // [rows][parts][top]
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

template <int kMask>
__device__ __forceinline__ double xor_lane_f64(double v) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = static_cast<uint32_t>(xor_lane_bits<kMask>(static_cast<int>(static_cast<uint32_t>(bits))));
  const uint32_t hi = static_cast<uint32_t>(xor_lane_bits<kMask>(static_cast<int>(static_cast<uint32_t>(bits >> 32))));
  return __builtin_bit_cast(double, (static_cast<unsigned long long>(hi) << 32) | lo);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
  v += xor_lane_f64<32>(v);
  v += xor_lane_f64<16>(v);
  v += xor_lane_f64<8>(v);
  v += xor_lane_f64<4>(v);
  v += xor_lane_f64<2>(v);
  return v + xor_lane_f64<1>(v);
}

// A part of a row. Loads are 16-byte aligned, so that index i of the row is place
// i + shift of them; places outside the row hold -inf.
struct RowPart {
  const float* row;
  int shift;   // 0 .. 3
  int places;  // shift + vocab
  int tile0;   // [tile0, tile1) of kTile places
  int tile1;

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

  __device__ __forceinline__ void load(const RowPart& p, int tile) {
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

struct Lds {
  float lists[kWaves][64];
  unsigned long long candidates[kMostCandidates];
  double sums[kWaves][2];
  float max[kWaves];
  int above[kWaves];
  int hot[kWaves];
  int count;
  float reach;
};

// A compare and exchange over lanes kMask apart: the larger to the lower lane where
// `down`.
template <int kMask>
__device__ __forceinline__ float exchange(float v, bool down) {
  const float other = xor_lane<kMask>(v);
  const bool lower = (lane_id() & kMask) == 0;
  return lower == down ? fmaxf(v, other) : fminf(v, other);
}

// 64 values that rise and then fall, or the reverse, in descending order.
__device__ __forceinline__ float sort_bitonic(float v) {
  v = exchange<32>(v, true);
  v = exchange<16>(v, true);
  v = exchange<8>(v, true);
  v = exchange<4>(v, true);
  v = exchange<2>(v, true);
  return exchange<1>(v, true);
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
  return sort_bitonic(v);
}

// The top-th largest of the block's 64 kWaves values, for all of it.
__device__ __forceinline__ float largest_reached(Lds& lds, float v, int top) {
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  v = sort_wave(v);
#pragma unroll
  for (int step = 1; step < kWaves; step <<= 1) {
    if ((wave & (2 * step - 1)) == step) lds.lists[wave][lane_id()] = v;
    __syncthreads();
    // the larger of two lists' 64 values, one read backwards: they rise and fall
    if ((wave & (2 * step - 1)) == 0) v = sort_bitonic(fmaxf(v, lds.lists[wave + step][63 - lane_id()]));
  }
  if (threadIdx.x == static_cast<unsigned>(top - 1)) lds.reach = v;
  __syncthreads();
  return lds.reach;
}

// The part's logits at or above (kAbove: above) `reach` as candidates, by the lanes
// whose largest reaches it; -inf is none.
template <bool kAbove>
__device__ __forceinline__ int gather(Lds& lds, const RowPart& p, float reach, float lane_max) {
  if (threadIdx.x == 0) lds.count = 0;
  __syncthreads();
  auto counts = [&](float l) { return (kAbove ? l > reach : l >= reach) && l > -infinity(); };
  const bool mine = counts(lane_max);
  if (__any(mine)) {
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    for (int tile = p.tile0 + wave; tile < p.tile1; tile += kWaves) {
      if (!mine) continue;
      const int g = tile * (kTile / 4) + lane_id();
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = p.load(g + 64 * j);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float l[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!counts(l[i])) continue;
          const int at = atomicAdd(&lds.count, 1);
          if (at < kMostCandidates) lds.candidates[at] = key_of(l[i], 4 * (g + 64 * j) + i - p.shift);
        }
      }
    }
  }
  __syncthreads();
  const int n = lds.count;
  __syncthreads();  // it may be counted in again
  return n;
}

// Adds the first `want` of the part's logits that equal `reach`, in the order of
// their ids, behind `have` candidates.
__device__ __forceinline__ void gather_equal(Lds& lds, const RowPart& p, float reach, int have, int want) {
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int end = min(p.tile1 * kTile, p.places);
  for (int base = p.tile0 * kTile; base < end && want > 0; base += kThreads) {
    const int i = base + static_cast<int>(threadIdx.x) - p.shift;
    const bool equal = i >= 0 && i + p.shift < end && p.row[i] == reach;
    const unsigned long long mask = __ballot(equal);
    if (lane_id() == 0) lds.above[wave] = __popcll(mask);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += lds.above[w];
      all += lds.above[w];
    }
    before += __popcll(mask & ((1ull << lane_id()) - 1));
    if (equal && before < want) lds.candidates[have + before] = key_of(reach, i);
    have += min(all, want);
    want -= min(all, want);
    __syncthreads();
  }
}

// The part's `top` largest, one pass over it for each: for parts with too many
// candidates, whose large logits all lie with few lanes.
__device__ __forceinline__ int gather_slowly(Lds& lds, const RowPart& p, int top) {
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int end = min(p.tile1 * kTile, p.places);
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int at = p.tile0 * kTile + static_cast<int>(threadIdx.x); at < end; at += kThreads) {
      if (at < p.shift) continue;
      const float l = p.row[at - p.shift];
      if (!(l > -infinity())) continue;
      const unsigned long long key = key_of(l, at - p.shift);
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
template <typename Out>
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

// A row (kPart: a part of one) a block.
template <bool kTop, bool kPart>
__global__ __launch_bounds__(kThreads, 4) void logprobs_kernel(LogprobArgs a) {
  __shared__ Lds lds;
  const int row = kPart ? blockIdx.y : blockIdx.x;
  const int part = kPart ? blockIdx.x : 0;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int token = a.token_ids != nullptr ? a.token_ids[row] : -1;
  if (a.token_ids != nullptr && token < 0) return;  // the row is left out
  RowPart p;
  p.row = a.logits + static_cast<size_t>(row) * static_cast<size_t>(a.logits_stride);
  p.shift = static_cast<int>(reinterpret_cast<uintptr_t>(p.row) >> 2 & 3u);
  p.places = p.shift + a.vocab;
  const int tiles = (p.places + kTile - 1) / kTile;
  p.tile0 = kPart ? static_cast<int>(static_cast<long long>(tiles) * part / a.parts) : 0;
  p.tile1 = kPart ? static_cast<int>(static_cast<long long>(tiles) * (part + 1) / a.parts) : tiles;

  Tile next;
  int tile = p.tile0 + wave;
  if (tile < p.tile1) next.load(p, tile);
  const float given = token >= 0 && token < a.vocab ? clean(p.row[token]) : infinity();
  float largest = -infinity();
  double sum = 0.0, weighted = 0.0;
  int above = 0;
  for (; tile < p.tile1; tile += kWaves) {
    Tile now = next;
    if (tile + kWaves < p.tile1) next.load(p, tile + kWaves);
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
    for (int i = p.tile0 * kTile + static_cast<int>(threadIdx.x); i < min(p.tile1 * kTile, p.places); i += kThreads) {
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
  PartSums all{0.0, 0.0, most, 0, INT_MAX, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    all.sum += lds.sums[w][0];
    all.weighted += lds.sums[w][1];
    all.above += lds.above[w];
    all.hot = min(all.hot, lds.hot[w]);
  }
  const RowResult result = kPart ? RowResult{} : result_of(all);
  if constexpr (!kPart) {
    if (threadIdx.x == 0) write_row(a, row, token, given, all, result);
  }
  PartSums* sums = kPart ? a.sums + static_cast<size_t>(row) * a.parts + part : nullptr;
  if constexpr (kTop) {
    const float reach = largest_reached(lds, largest, a.top);
    int n = gather<false>(lds, p, reach, largest);
    if (n > kMostCandidates) {
      // Many equal ones (a mask of the type's lowest value), or many in few lanes.
      n = gather<true>(lds, p, reach, largest);
      if (n <= kMostCandidates - kMostTop) {
        const int want = max(a.top - n, 0);
        gather_equal(lds, p, reach, n, want);
        n += want;
      } else {
        n = gather_slowly(lds, p, a.top);
      }
    }
    const int top = min(n, a.top);
    if constexpr (kPart) {
      unsigned long long* keys = a.keys + (static_cast<size_t>(row) * a.parts + part) * a.top;
      rank(lds.candidates, n, a.top, [&](int place, unsigned long long key) { keys[place] = key; });
      all.count = top;
    } else {
      rank(lds.candidates, n, a.top, [&](int place, unsigned long long key) {
        write_top(a, row, place, result.logprob(value_of(key), id_of(key)), id_of(key));
      });
      for (int place = top + static_cast<int>(threadIdx.x); place < a.top; place += kThreads) {
        write_top(a, row, place, -infinity(), -1);
      }
    }
  }
  if (kPart && threadIdx.x == 0) *sums = all;
}

constexpr int kMostParts = 32;

// Joins the parts of a row, a block each.
template <bool kTop>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ unsigned long long keys[kMostParts * kMostTop];
  __shared__ unsigned long long candidates[kMostParts * kMostTop];
  __shared__ int lds_count;
  const int row = blockIdx.x;
  const int token = a.token_ids != nullptr ? a.token_ids[row] : -1;
  if (a.token_ids != nullptr && token < 0) return;
  const float* logits = a.logits + static_cast<size_t>(row) * static_cast<size_t>(a.logits_stride);
  const float given = token >= 0 && token < a.vocab ? clean(logits[token]) : infinity();
  const int lane = lane_id();
  // Every wave joins the sums for itself, a part a lane.
  PartSums mine{0.0, 0.0, -infinity(), 0, INT_MAX, 0};
  if (lane < a.parts) mine = a.sums[static_cast<size_t>(row) * a.parts + lane];
  if constexpr (kTop) {
    const unsigned long long* from = a.keys + static_cast<size_t>(row) * a.parts * a.top;
    for (int i = threadIdx.x; i < a.parts * a.top; i += kThreads) keys[i] = from[i];
    if (threadIdx.x == 0) lds_count = 0;
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
    __syncthreads();
    // What some part has as many of is a bound for the others.
    unsigned long long reach = lane < a.parts && mine.count == a.top ? keys[lane * a.top + a.top - 1] : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long other = __shfl_xor(reach, o, 64);
      reach = other > reach ? other : reach;
    }
    for (int base = 0; base < a.parts * a.top; base += kThreads) {
      const int i = base + static_cast<int>(threadIdx.x);
      const int part = min(i / a.top, a.parts - 1);
      const int count = __shfl(mine.count, part, 64);
      if (i < a.parts * a.top && i - part * a.top < count && keys[i] >= reach) {
        candidates[atomicAdd(&lds_count, 1)] = keys[i];
      }
    }
    __syncthreads();
    const int n = lds_count;
    rank(candidates, n, a.top, [&](int place, unsigned long long key) {
      write_top(a, row, place, result.logprob(value_of(key), id_of(key)), id_of(key));
    });
    for (int place = min(n, a.top) + static_cast<int>(threadIdx.x); place < a.top; place += kThreads) {
      write_top(a, row, place, -infinity(), -1);
    }
  }
}

// Parts that a row is cut into: as many as give each compute unit two, of no less
// than a step of each wave.
int parts_for(int rows, int vocab) {
  const int compute_units = device_compute_units();
  if (rows >= compute_units) return 1;
  const int steps = (vocab + kTile * kWaves - 1) / (kTile * kWaves);
  return std::max(1, std::min({kMostParts, (2 * compute_units + rows - 1) / rows, steps}));
}

size_t workspace_for(int rows, int parts, int top) {
  return static_cast<size_t>(rows) * static_cast<size_t>(parts) *
         (sizeof(PartSums) + static_cast<size_t>(top) * sizeof(unsigned long long));
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
  CAPI_CHECK(static_cast<long long>(rows) * kThreads <= UINT32_MAX,
             "batch_logprobs of " << rows << " rows needs more than 2^32 threads");
  LogprobArgs a{logprobs, ranks, entropies, top_ids, top_logprobs, logits, token_ids, top, vocab, logits_stride,
                1, nullptr, nullptr};
  auto s = static_cast<hipStream_t>(stream);
  const int parts = parts_for(rows, vocab);
  if (parts > 1 && workspace != nullptr && workspace_bytes >= workspace_for(rows, parts, top)) {
    a.parts = parts;
    a.sums = static_cast<PartSums*>(workspace);
    a.keys = reinterpret_cast<unsigned long long*>(a.sums + static_cast<size_t>(rows) * parts);
    const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(rows));
    if (top > 0) {
      logprobs_kernel<true, true><<<grid, kThreads, 0, s>>>(a);
      CAPI_LAUNCHED();
      logprobs_join_kernel<true><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(a);
    } else {
      logprobs_kernel<false, true><<<grid, kThreads, 0, s>>>(a);
      CAPI_LAUNCHED();
      logprobs_join_kernel<false><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(a);
    }
  } else if (top > 0) {
    logprobs_kernel<true, false><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(a);
  } else {
    logprobs_kernel<false, false><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(a);
  }
  CAPI_LAUNCHED();
  return LCR_OK;
}
