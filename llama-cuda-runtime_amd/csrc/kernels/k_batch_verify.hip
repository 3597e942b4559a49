// lcr_batch_verify: drafted tokens kept or not, and the token behind them.
//
// Two launches:
//   verify_stats  1024 logits (a part) of a row of target or draft a wave: the
//                 largest and the sum of exp((l - largest) / T) against it
//   verify_draw   four parts of the vocabulary of one sequence a block: the
//                 parts of its rows joined, the drafts kept or not in order, and
//                 the id behind them. Behind drafts that were all kept it is
//                 drawn from the last row's p, whose parts' sums are there
//                 already: the first block finds the part, then the index, at
//                 which the running sum passes the draw. Behind a draft not
//                 kept, the blocks sum max(p - q, 0) over their parts of its
//                 row, and the block whose sum arrives last finds them.
// Every logit is read once in the first launch, and the row of a draft not kept
// again in the second. The exponentials and sums are fp64: the running sum over
// 128256 weights has intervals of 1e-5 and less, of which fp32 weights (6e-8
// each, and as much in p's and q's normalisers) would give some draws to a
// neighbour. gfx950 runs fp64 fma at the fp32 rate, so that a logit's 17
// operations (10 of them fp64) take about as long as its 4 bytes: 332 rows of
// 128256 logits (170 MB) in 40 us, of which the vector units are busy for 25 and
// the memory, at 7 TB/s, for 24. A wave loads its part, waits, and computes, so
// that the two overlap only where other waves of its compute unit are at the other.
// The draw of 64 sequences takes 23 us, the rows of rejected drafts (half of
// them, 1 MB each) and a chain of a dozen dependent reads and exchanges; alone,
// one sequence's takes 8 where all drafts are kept and 13 where one is not. Blocks
// of eight waves, which look at eight rows at once, were slower (25 us for 64
// sequences): more waves wait for the slowest.
// Which block arrives last decides who computes, not what: all sums have a fixed
// order.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "sampling.h"

namespace lcr {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kPart = 1024;                         // logits of a wave
constexpr int kPerLane = kPart / 64;

// A part of a row: its largest logit, its sum of exp((l - max) / T), and the
// lowest index of the largest logit (only of greedy rows and where it is not
// finite).
struct alignas(16) PartStats {
  double sum;
  float max;
  int index;
};

// What a row's distribution is: exp((l - max) / T) / sum where max is finite,
// else (sum = 0) one at the index `hot`.
struct RowStats {
  double sum;
  float max;
  int hot;
};

struct VerifyArgs {
  const float* target;
  const float* draft;
  const int32_t* draft_ids;
  const int32_t* row_starts;
  const float* temperatures;
  const float* accept_uniforms;
  const float* sample_uniforms;
  int32_t* out_ids;
  int32_t* out_counts;
  PartStats* stats;     // [rows][2][parts]
  double* totals;       // [batch][parts]: sums of max(p - q, 0)
  int* arrived;         // [batch] parts of `totals` that are there
  int batch;
  int rows;
  int max_draft;
  int vocab;
  int parts;
  int logits_stride;
  bool vectors;         // rows on 16-byte boundaries
};

// 2^(j / 32), by a thread of the table's 32: 2^x on [-1/2, 1/2] by its Chebyshev
// interpolation of degree 10 (off by 3e-16), doubled for j of 16 and more. The
// table holds it with j << 15 taken off the high word, which the exponent's
// addition below puts back.
constexpr int kExp2Entries = 32;

__device__ __forceinline__ uint2 exp2_entry(int j) {
  const double x = (j < 16 ? j : j - 32) * (1.0 / 32.0);
  double p = 7.072585949269223e-09;
  p = __builtin_fma(p, x, 1.0208690299958306e-07);
  p = __builtin_fma(p, x, 1.321544258792169e-06);
  p = __builtin_fma(p, x, 1.5252657260200837e-05);
  p = __builtin_fma(p, x, 0.0001540353044173605);
  p = __builtin_fma(p, x, 0.0013333558230164974);
  p = __builtin_fma(p, x, 0.009618129107606888);
  p = __builtin_fma(p, x, 0.05550410866444772);
  p = __builtin_fma(p, x, 0.24022650695910097);
  p = __builtin_fma(p, x, 0.69314718055995);
  p = __builtin_fma(p, x, 1.0);
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, j < 16 ? p : 2.0 * p);
  return make_uint2(static_cast<uint32_t>(bits), static_cast<uint32_t>(bits >> 32) - (static_cast<uint32_t>(j) << 15));
}

constexpr double kLog2e = 1.44269504088896340736;

// The scale of a temperature: z = (l - max) c is the power of two that a logit
// weighs, and logits more than `span` below the largest weigh nothing: z below
// -1020 would leave the normal range.
struct Scale {
  double c, span;
};

__device__ __forceinline__ Scale scale_of(float temperature) {
  const double t = temperature;
  return Scale{kLog2e / t, t * (1020.0 / kLog2e)};
}

// The lowest logit that weighs anything beside `max`.
__device__ __forceinline__ double lowest_of(float max, const Scale& scale) {
  return static_cast<double>(max) - scale.span;
}

// The next float at or above a double, -FLT_MAX at least.
__device__ __forceinline__ float float_above(double v) {
  const float f = fmaxf(static_cast<float>(v), -FLT_MAX);
  if (static_cast<double>(f) >= v) return f;
  const int bits = __float_as_int(f);
  return f == 0.0f ? __int_as_float(1) : __int_as_float(bits + (bits < 0 ? -1 : 1));
}

// exp((l - max) / T) = 2^z in fp64: z = k / 32 + f with k whole, by adding and
// taking off 1.5 * 2^47 (k then also stands in the sum's low word); 2^f = 1 + f
// Q(f) on [-1/64, 1/64], Q by Chebyshev interpolation (off by 1.6e-13, of which
// a running sum over a vocabulary hands a draw of 1e-8 to a neighbour), times the
// table's 2^((k mod 32) / 32), and k / 32 added to the exponent. 32 entries of 8
// bytes lie on banks of their own, so that 64 lanes with an entry each read them
// without conflicts. The statistics of 332 rows of 128256 take 40 us, with 64
// entries 42, with a polynomial over [-1/2, 1/2] and no table 48.
// The coefficients are kept in registers, scalar but for one (an instruction
// takes one scalar): left to the compiler, each is moved before each use.
struct Exp2 {
  double c0, c1, c2, c3;
  const uint2* table;

  __device__ __forceinline__ explicit Exp2(const uint2* table_lds)
      : c0(0.693147180550011), c1(0.24022650695795306), c2(0.055504434191939005), c3(0.009618166713972776),
        table(table_lds) {
    asm volatile("" : "+s"(c0), "+s"(c1), "+v"(c2), "+s"(c3));
  }

  // Of a logit no lower than lowest_of(max).
  __device__ __forceinline__ double inside(float l, double max, const Scale& scale) const {
    constexpr double kRound = 211106232532992.0;
    const double below = static_cast<double>(l) - max;
    const double shifted = __builtin_fma(below, scale.c, kRound);
    const double f = __builtin_fma(below, scale.c, kRound - shifted);
    const uint32_t k = static_cast<uint32_t>(__builtin_bit_cast(unsigned long long, shifted));
    const uint2 entry = table[k & (kExp2Entries - 1)];
    const uint32_t high = entry.y + (k << 15);
    const double t = __builtin_bit_cast(double, (static_cast<unsigned long long>(high) << 32) | entry.x);
    double q = __builtin_fma(c3, f, c2);
    q = __builtin_fma(q, f, c1);
    q = __builtin_fma(q, f, c0);
    return __builtin_fma(t * f, q, t);
  }

  // Of any logit but infinity: 0 below the lowest and for NaN.
  __device__ __forceinline__ double operator()(float l, float max, const Scale& scale) const {
    const double lowest = fmax(lowest_of(max, scale), -static_cast<double>(FLT_MAX));
    const bool weighs = static_cast<double>(l) >= lowest;
    const double w = inside(weighs ? l : max, max, scale);
    return weighs ? w : 0.0;
  }
};

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

// v of another lane by DPP, 0 in lanes that get none.
template <int kControl, int kRowMask, bool kBoundZero>
__device__ __forceinline__ double dpp_f64(double v) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const int lo = static_cast<int>(static_cast<uint32_t>(bits)), hi = static_cast<int>(static_cast<uint32_t>(bits >> 32));
  const uint32_t l = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, lo, kControl, kRowMask, 0xF, kBoundZero));
  const uint32_t h = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, hi, kControl, kRowMask, 0xF, kBoundZero));
  return __builtin_bit_cast(double, (static_cast<unsigned long long>(h) << 32) | l);
}

// Inclusive sums over the wave: within rows of 16 lanes by shifts, then the
// total of row 0 into row 1 and of row 2 into row 3, then of rows 0-1 into 2-3.
__device__ __forceinline__ double wave_inclusive_scan_f64(double v) {
  v += dpp_f64<0x111, 0xF, true>(v);   // row_shr:1
  v += dpp_f64<0x112, 0xF, true>(v);   // row_shr:2
  v += dpp_f64<0x114, 0xF, true>(v);   // row_shr:4
  v += dpp_f64<0x118, 0xF, true>(v);   // row_shr:8
  v += dpp_f64<0x142, 0xA, false>(v);  // row_bcast:15
  v += dpp_f64<0x143, 0xC, false>(v);  // row_bcast:31
  return v;
}

__device__ __forceinline__ double read_lane_f64(double v, int lane) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const uint32_t l = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(bits)), lane));
  const uint32_t h =
      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(bits >> 32)), lane));
  return __builtin_bit_cast(double, (static_cast<unsigned long long>(h) << 32) | l);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

// Probability of index i with logit l in a row's distribution.
__device__ __forceinline__ double probability(const Exp2& exp2, const RowStats& r, double inv_sum, float l, int i,
                                              const Scale& scale) {
  return r.sum > 0.0 ? exp2(l, r.max, scale) * inv_sum : (i == r.hot ? 1.0 : 0.0);
}

// Four logits of a row from index `first`; -inf behind the vocabulary's end.
__device__ __forceinline__ void load_logits(float* out, const float* row, int first, int vocab, bool vectors) {
  if (vectors && first <= vocab - 4) {
    const float4 v = *reinterpret_cast<const float4*>(row + first);
    out[0] = v.x;
    out[1] = v.y;
    out[2] = v.z;
    out[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = j < vocab - first ? row[first + j] : -__builtin_huge_valf();
  }
}

// A row's sequence: its first row, the next sequence's, its temperature.
struct RowPlace {
  int start;     // -1: the row is behind the last sequence
  int next;
  float temperature;
};

// 64 starts and temperatures at once, each wave for itself: the last start at
// or before the row, and the one behind it. A bisection would be a chain of
// loads.
__device__ __forceinline__ RowPlace place_row(const VerifyArgs& a, int row, int starts, float temperatures) {
  RowPlace place{-1, 0, 0.0f};
  for (int base = 0;; base += 64) {
    const int b = base + lane_id();
    const unsigned long long below = __ballot(b <= a.batch && starts <= row);
    const int count = __popcll(below);
    if (count > 0) {
      place.start = __builtin_amdgcn_readlane(starts, count - 1);
      place.temperature = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(temperatures), count - 1));
    }
    if (count < 64 || base + 64 > a.batch) {
      // count - 1 is the last start at or before the row: batch's own says that
      // the row is behind the last sequence
      if (base + count > a.batch || place.start < 0) return RowPlace{-1, 0, 0.0f};
      place.next = __builtin_amdgcn_readlane(starts, min(count, 63));
      return place;
    }
    starts = a.row_starts[min(b + 64, a.batch)];
    temperatures = a.temperatures[min(b + 64, a.batch - 1)];
    // the next 64 may begin behind the row
    if (__builtin_amdgcn_readfirstlane(starts) > row) {
      place.next = __builtin_amdgcn_readfirstlane(starts);
      return place;
    }
  }
}

__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyArgs a) {
  __shared__ uint2 lds_table[kExp2Entries];
  const int part = static_cast<int>(blockIdx.x) * kVerifyWaves + (static_cast<int>(threadIdx.x) >> 6);
  const int row = blockIdx.y;
  const bool is_draft = blockIdx.z != 0;
  const int lane = lane_id();
  const float* logits = (is_draft ? a.draft : a.target) + static_cast<size_t>(row) * a.logits_stride;
  // Four of each 256 neighbouring logits a lane.
  const int first = min(part, a.parts - 1) * kPart + 4 * lane;
  if (blockIdx.x == 0 && row == 0 && !is_draft) {
    for (int b = threadIdx.x; b < a.batch; b += kVerifyThreads) a.arrived[b] = 0;
  }
  const int starts = a.row_starts[min(lane, a.batch)];
  const float temperatures = a.temperatures[min(lane, a.batch - 1)];
  float l[kPerLane];
  auto load = [&] {
#pragma unroll
    for (int j = 0; j < kPerLane / 4; ++j) load_logits(l + 4 * j, logits, first + 256 * j, a.vocab, a.vectors);
  };
  // Nearly every target row counts: its logits are requested before the wave
  // knows (and behind what it has to know, as loads return in order). Every
  // sequence has a draft row that does not.
  if (!is_draft) load();
  if (threadIdx.x < kExp2Entries) lds_table[threadIdx.x] = exp2_entry(static_cast<int>(threadIdx.x));
  __syncthreads();
  if (part >= a.parts) return;  // the waves have no more to do with each other
  const RowPlace place = place_row(a, row, starts, temperatures);
  if (place.start < 0) return;
  const int in_sequence = row - place.start;
  const int drafts = min(place.next - place.start - 1, a.max_draft);
  const float t = place.temperature;
  const bool greedy = !(t > 0.0f);
  if (in_sequence > drafts || (is_draft && (greedy || in_sequence == drafts))) return;
  if (is_draft) load();
  float max = -__builtin_huge_valf();
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) max = fmaxf(max, l[j]);  // NaN counts as -inf
  max = wave_max(max);
  double sum = 0.0;
  int index = INT_MAX;
  if (greedy || !finite(max)) {
#pragma unroll
    for (int j = kPerLane - 1; j >= 0; --j) {
      const int i = first + 256 * (j / 4) + (j & 3);
      if (fmaxf(l[j], -__builtin_huge_valf()) == max && i < a.vocab) index = i;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) index = min(index, __shfl_xor(index, o, 64));
  } else {
    const Scale scale = scale_of(t);
    const double m = max;
    const double lowest = lowest_of(max, scale);
    const Exp2 exp2(lds_table);
    const float low = float_above(lowest);
    if (lowest >= -static_cast<double>(FLT_MAX) && low < max) {
      // Clamped to the next float above the lowest, a logit weighs nothing beside
      // the 1 of the largest: it is below that by at least the spacing of floats
      // above `low`, and short of `span` by less than the spacing below it (twice
      // the other at most), so below by more than span / 3: 2^-340 at most. One
      // operation, where a choice of 0 takes three.
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) {
        sum += exp2.inside(__builtin_amdgcn_fmed3f(l[j], low, max), m, scale);  // NaN is the lowest
      }
    } else {
      // A temperature so high that every finite logit weighs something, and -inf
      // nothing; or so low that no float lies between the lowest and the largest.
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) sum += exp2(l[j], max, scale);
    }
    sum = wave_sum_f64(sum);
  }
  if (lane == 0) {
    a.stats[(static_cast<size_t>(row) * 2 + (is_draft ? 1 : 0)) * a.parts + part] = PartStats{sum, max, index};
  }
}

// A row's parts joined, by one wave; every lane gets the result.
__device__ __forceinline__ RowStats join_row(const Exp2& exp2, const PartStats* stats, int parts,
                                             const Scale& scale) {
  // Two parts a lane at once, which is all of a vocabulary up to 131072.
  PartStats s[2];
  float max = -__builtin_huge_valf();
  double sum = 0.0;
  int index = INT_MAX;
  for (int base = 0; base < parts; base += 128) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = base + 64 * k + lane_id();
      s[k] = i < parts ? stats[i] : PartStats{0.0, -__builtin_huge_valf(), INT_MAX};
    }
    const float to = fmaxf(max, wave_max(fmaxf(s[0].max, s[1].max)));
    index = max == to ? index : INT_MAX;
#pragma unroll
    for (int k = 0; k < 2; ++k) index = s[k].max == to ? min(index, s[k].index) : index;
    if (finite(to)) {
      if (max != to) sum = finite(max) ? sum * exp2(max, to, scale) : 0.0;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (finite(s[k].max)) sum += s[k].sum * exp2(s[k].max, to, scale);
      }
    }
    max = to;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) index = min(index, __shfl_xor(index, o, 64));
  return RowStats{finite(max) ? wave_sum_f64(sum) : 0.0, max, index};
}

struct DrawLds {
  int stop[kVerifyWaves];
  RowStats target[kVerifyWaves], draft[kVerifyWaves];
  uint2 table[kExp2Entries];
  int last;          // this block's sum was the last
  int part;          // of the drawn index; -1: no part has a weight
  double before;     // running sum before that part
  double goal;
  double wave_total[kVerifyWaves];
  int wave_first[kVerifyWaves], wave_last[kVerifyWaves];
};

// The first index whose running sum of weights passes u times their whole sum,
// by the block: the part by its parts' sums total_of(part), then the index by
// the weights weight_of(logits of target, logits of draft, index) in it.
// Rounding may leave no sum past the goal: then the last index with a weight.
// -1 where there is no weight.
template <typename TotalOf, typename WeightOf>
__device__ __forceinline__ int draw_index(DrawLds& lds, const VerifyArgs& a, float u, const float* target_row,
                                          const float* draft_row, TotalOf total_of, WeightOf weight_of) {
  const int lane = lane_id();
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  if (wave == 0) {
    // 256 parts at once, so that their reads do not wait for each other; all of
    // a vocabulary up to 262144 is read once.
    double v[4];
    auto load = [&](int base) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = base + 64 * k + lane;
        v[k] = i < a.parts ? total_of(i) : 0.0;
      }
    };
    double whole = 0.0;
    for (int base = 0; base < a.parts; base += 256) {
      load(base);
#pragma unroll
      for (int k = 0; k < 4; ++k) whole += read_lane_f64(wave_inclusive_scan_f64(v[k]), 63);
    }
    const double goal = static_cast<double>(u) * whole;
    double before = 0.0, part_before = 0.0;
    int part = -1;
    bool hit = false;
    for (int base = 0; base < a.parts && !hit; base += 256) {
      if (a.parts > 256) load(base);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (hit) continue;
        const double incl = wave_inclusive_scan_f64(v[k]);
        const unsigned long long past = __ballot(v[k] > 0.0 && before + incl > goal);
        const unsigned long long weighty = __ballot(v[k] > 0.0);
        const int at = past != 0 ? __ffsll(past) - 1 : (weighty != 0 ? 63 - __clzll(weighty) : -1);
        if (at >= 0) {
          part = base + 64 * k + at;
          part_before = before + read_lane_f64(incl - v[k], at);
          hit = past != 0;
        }
        before += read_lane_f64(incl, 63);
      }
    }
    if (lane == 0) {
      lds.part = part;
      lds.before = part_before;
      lds.goal = goal;
    }
  }
  __syncthreads();
  const int part = lds.part;
  if (part < 0) {
    __syncthreads();  // every wave has read it: `lds` may be drawn with again
    return -1;
  }
  // Four neighbouring weights a thread.
  static_assert(kPart == 4 * kVerifyThreads, "one 16-byte load a thread");
  const int i0 = part * kPart + 4 * static_cast<int>(threadIdx.x);
  float lp[4], lq[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  load_logits(lp, target_row, i0, a.vocab, a.vectors);
  if (draft_row != nullptr) load_logits(lq, draft_row, i0, a.vocab, a.vectors);
  double run[4];
  double sum = 0.0;
  bool weighty[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double w = e < a.vocab - i0 ? weight_of(lp[e], lq[e], i0 + e) : 0.0;
    sum += w;
    run[e] = sum;
    weighty[e] = w > 0.0;
  }
  const double incl = wave_inclusive_scan_f64(sum);
  if (lane == 63) lds.wave_total[wave] = incl;
  __syncthreads();
  double before = lds.before;
  for (int w = 0; w < wave; ++w) before += lds.wave_total[w];
  before += incl - sum;
  int first = INT_MAX, last = -1;
#pragma unroll
  for (int e = 3; e >= 0; --e) {
    if (weighty[e]) {
      last = max(last, i0 + e);
      if (before + run[e] > lds.goal) first = i0 + e;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    first = min(first, __shfl_xor(first, o, 64));
    last = max(last, __shfl_xor(last, o, 64));
  }
  if (lane == 0) {
    lds.wave_first[wave] = first;
    lds.wave_last[wave] = last;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerifyWaves; ++w) {
    first = min(first, lds.wave_first[w]);
    last = max(last, lds.wave_last[w]);
  }
  __syncthreads();  // `lds` may be drawn with again
  return first != INT_MAX ? first : max(last, 0);
}

// A sum handed to other blocks of the grid. Atomic accesses of device scope go
// past the caches of one XCD; that the exchange has returned says that its value
// is where they all look, so that a count taken after it counts it. (Releasing
// and acquiring with the count instead writes back and drops the whole L2, once
// a block: 68 us against 24 for 64 sequences of 128256 logits.)
__device__ __forceinline__ void publish(double* at, double value) {
  const unsigned long long before =
      __hip_atomic_exchange(reinterpret_cast<unsigned long long*>(at), __builtin_bit_cast(unsigned long long, value),
                            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("" : : "v"(before) : "memory");  // waits for it
}
__device__ __forceinline__ double published(const double* at) {
  return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(at), __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_AGENT));
}

__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ DrawLds lds;
  const int b = blockIdx.y;
  const int lane = lane_id();
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int first = a.row_starts[b];
  const int count = a.row_starts[b + 1] - first;
  const float t = a.temperatures[b];
  if (threadIdx.x < kExp2Entries) lds.table[threadIdx.x] = exp2_entry(static_cast<int>(threadIdx.x));
  if (threadIdx.x == 0) lds.last = 0;
  __syncthreads();
  int32_t* ids = a.out_ids + static_cast<size_t>(b) * (a.max_draft + 1);
  // Rows of a table that is no ascending list of rows are not read.
  if (count <= 0 || first < 0 || first > a.rows - count) {
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i <= a.max_draft; i += kVerifyThreads) ids[i] = -1;
      if (threadIdx.x == 0) a.out_counts[b] = 0;
    }
    return;
  }
  const int drafts = min(count - 1, a.max_draft);
  const bool greedy = !(t > 0.0f);
  const Scale scale = scale_of(greedy ? 1.0f : t);
  const Exp2 exp2(lds.table);
  // The first row that stops: its draft is not kept, or it is the last. A wave
  // a row, so that rows do not wait for each other's reads.
  int kept = 0;
  int at = -1;
  for (int base = 0; at < 0; base += kVerifyWaves) {
    const int i = base + wave;
    bool stop = true;
    if (i <= drafts) {
      const int row = first + i;
      const PartStats* stats = a.stats + static_cast<size_t>(row) * 2 * a.parts;
      const bool sampled = i < drafts && !greedy;
      const int x = i < drafts ? a.draft_ids[row] : 0;
      const float u = sampled ? a.accept_uniforms[row] : 0.0f;
      const bool inside = x >= 0 && x < a.vocab;
      const size_t place = static_cast<size_t>(row) * a.logits_stride + (inside ? x : 0);
      const float target_logit = sampled ? a.target[place] : 0.0f;
      const float draft_logit = sampled && a.draft != nullptr ? a.draft[place] : 0.0f;
      const RowStats target = join_row(exp2, stats, a.parts, scale);
      RowStats draft{0.0, 0.0f, x};
      if (sampled && a.draft != nullptr) {
        const RowStats d = join_row(exp2, stats + a.parts, a.parts, scale);
        draft.max = d.max;
        draft.sum = d.sum;
      }
      if (sampled) {
        const double p = probability(exp2, target, 1.0 / target.sum, target_logit, x, scale);
        const double q = draft.sum > 0.0 ? probability(exp2, draft, 1.0 / draft.sum, draft_logit, x, scale) : 1.0;
        stop = !(inside && static_cast<double>(u) * q < p);
      } else {
        stop = i == drafts || x != target.hot;
      }
      if (lane == 0) {
        lds.target[wave] = target;
        lds.draft[wave] = draft;
      }
    }
    if (lane == 0) lds.stop[wave] = stop ? 1 : 0;
    __syncthreads();
#pragma unroll
    for (int w = kVerifyWaves - 1; w >= 0; --w) {
      if (lds.stop[w] != 0) at = w;
    }
    kept = base + at;
    if (at < 0) __syncthreads();  // read before the next rows are written
  }
  const RowStats target = lds.target[at], draft = lds.draft[at];
  const bool subtract = kept < drafts && !greedy;
  if (!subtract && blockIdx.x != 0) return;
  const int row = first + kept;
  const float* target_row = a.target + static_cast<size_t>(row) * a.logits_stride;
  const float* draft_row =
      subtract && draft.sum > 0.0 ? a.draft + static_cast<size_t>(row) * a.logits_stride : nullptr;
  int id = -1;
  if (subtract) {
    const double inv_p = 1.0 / target.sum, inv_q = 1.0 / draft.sum;
    auto weight_of = [&](float p, float q, int i) {
      return fmax(probability(exp2, target, inv_p, p, i, scale) - probability(exp2, draft, inv_q, q, i, scale), 0.0);
    };
    double* totals = a.totals + static_cast<size_t>(b) * a.parts;
    const int part = static_cast<int>(blockIdx.x) * kVerifyWaves + wave;
    if (part < a.parts) {
      double rest = 0.0;
#pragma unroll
      for (int j = 0; j < kPerLane / 4; ++j) {
        const int i0 = part * kPart + 256 * j + 4 * lane;
        float lp[4], lq[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        load_logits(lp, target_row, i0, a.vocab, a.vectors);
        if (draft_row != nullptr) load_logits(lq, draft_row, i0, a.vocab, a.vectors);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e < a.vocab - i0) rest += weight_of(lp[e], lq[e], i0 + e);
        }
      }
      rest = wave_sum_f64(rest);
      if (lane == 0) publish(totals + part, rest);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      const int before = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (before == static_cast<int>(gridDim.x) - 1) lds.last = 1;
    }
    __syncthreads();
    if (lds.last == 0) return;
    id = draw_index(lds, a, a.sample_uniforms[b], target_row, draft_row, [&](int i) { return published(totals + i); }, weight_of);
  }
  if (greedy) {
    id = target.hot;
  } else if (id < 0) {
    // from p: unnormalised, as the parts' sums are
    const PartStats* stats = a.stats + static_cast<size_t>(row) * 2 * a.parts;
    id = draw_index(
        lds, a, a.sample_uniforms[b], target_row, nullptr,
        [&](int i) {
          if (!(target.sum > 0.0)) return target.hot / kPart == i ? 1.0 : 0.0;
          const PartStats s = stats[i];
          return finite(s.max) ? s.sum * exp2(s.max, target.max, scale) : 0.0;
        },
        [&](float p, float, int i) { return probability(exp2, target, 1.0, p, i, scale); });
  }
  for (int i = threadIdx.x; i <= a.max_draft; i += kVerifyThreads) {
    ids[i] = i < kept ? a.draft_ids[first + i] : (i == kept ? id : -1);
  }
  if (threadIdx.x == 0) a.out_counts[b] = kept + 1;
}

int parts_for(int vocab) { return (vocab + kPart - 1) / kPart; }

struct VerifyLayout {
  size_t totals_at, arrived_at, bytes;
};

VerifyLayout layout_for(int batch, int rows, int vocab) {
  const size_t parts = static_cast<size_t>(parts_for(vocab));
  VerifyLayout l;
  l.totals_at = static_cast<size_t>(rows) * 2 * parts * sizeof(PartStats);
  l.arrived_at = l.totals_at + static_cast<size_t>(batch) * parts * sizeof(double);
  l.bytes = l.arrived_at + static_cast<size_t>(batch) * sizeof(int);
  return l;
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" size_t lcr_batch_verify_workspace_bytes(int batch, int rows, int vocab) {
  if (batch <= 0 || rows < 0 || vocab <= 0) return 0;
  return layout_for(batch, rows, vocab).bytes;
}

extern "C" int lcr_batch_verify(int32_t* out_ids, int32_t* out_counts, const float* target_logits,
                                const float* draft_logits, const int32_t* draft_ids, const int32_t* row_starts,
                                const float* temperatures, const float* accept_uniforms, const float* sample_uniforms,
                                int batch, int rows, int max_draft, int vocab, int logits_stride, void* workspace,
                                size_t workspace_bytes, void* stream) {
  CAPI_CHECK(batch >= 0 && rows >= 0 && max_draft >= 0, "batch_verify needs non-negative sizes");
  CAPI_CHECK(batch <= LCR_BATCH_MAX_SEQUENCES,
             "batch_verify takes up to " << LCR_BATCH_MAX_SEQUENCES << " sequences, got " << batch);
  if (batch == 0) return LCR_OK;
  CAPI_CHECK(vocab > 0, "cannot sample from an empty vocabulary");
  // counted in 32 bits, a block's threads at a time
  CAPI_CHECK(max_draft <= (1 << 30), "batch_verify takes up to 2^30 drafts, got " << max_draft);
  CAPI_CHECK(logits_stride >= vocab, "rows of " << vocab << " logits cannot lie " << logits_stride << " apart");
  CAPI_CHECK(rows <= 65535, "batch_verify takes up to 65535 rows, got " << rows);
  CAPI_CHECK(out_ids != nullptr && out_counts != nullptr && row_starts != nullptr && temperatures != nullptr &&
                 sample_uniforms != nullptr,
             "batch_verify needs its arrays");
  CAPI_CHECK(rows == 0 || target_logits != nullptr, "batch_verify needs the target's logits");
  CAPI_CHECK(rows == 0 || max_draft == 0 || (draft_ids != nullptr && accept_uniforms != nullptr),
             "batch_verify needs the drafted tokens and their draws");
  const VerifyLayout layout = layout_for(batch, rows, vocab);
  CAPI_CHECK(workspace != nullptr && workspace_bytes >= layout.bytes,
             "batch_verify needs a workspace of " << layout.bytes << " bytes, got " << workspace_bytes);
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch_verify workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  VerifyArgs a;
  a.target = target_logits;
  a.draft = max_draft > 0 ? draft_logits : nullptr;
  a.draft_ids = draft_ids;
  a.row_starts = row_starts;
  a.temperatures = temperatures;
  a.accept_uniforms = accept_uniforms;
  a.sample_uniforms = sample_uniforms;
  a.out_ids = out_ids;
  a.out_counts = out_counts;
  a.stats = reinterpret_cast<PartStats*>(ws);
  a.totals = reinterpret_cast<double*>(ws + layout.totals_at);
  a.arrived = reinterpret_cast<int*>(ws + layout.arrived_at);
  a.batch = batch;
  a.rows = rows;
  a.max_draft = max_draft;
  a.vocab = vocab;
  a.parts = parts_for(vocab);
  a.logits_stride = logits_stride;
  a.vectors = logits_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(target_logits) & 15u) == 0 &&
              (reinterpret_cast<uintptr_t>(draft_logits) & 15u) == 0;
  auto s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    const dim3 grid(static_cast<unsigned>((a.parts + kVerifyWaves - 1) / kVerifyWaves), static_cast<unsigned>(rows),
                    a.draft != nullptr ? 2u : 1u);
    verify_stats_kernel<<<grid, kVerifyThreads, 0, s>>>(a);
    CAPI_LAUNCHED();
  }
  const dim3 grid(static_cast<unsigned>((a.parts + kVerifyWaves - 1) / kVerifyWaves), static_cast<unsigned>(batch));
  verify_draw_kernel<<<grid, kVerifyThreads, 0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
