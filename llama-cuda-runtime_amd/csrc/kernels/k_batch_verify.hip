// lcr_batch_verify: drafted tokens kept or not, and the token behind them.
//
// Three launches:
//   verify_stats    a slice of one row of target or draft logits a block: its
//                   largest logit (with its index, as argmax's 64-bit key) and
//                   the sum of exp((l - largest) / T) against it
//   verify_residual a slice of the vocabulary of one sequence a block: the
//                   row's slices joined, the drafts kept or not in order, and
//                   the slice's sum of the weights the last token is drawn
//                   with: max(p - q, 0) in the row of the first draft not
//                   kept, or p in the last row
//   verify_pick     one block a sequence: the slice, then the index, at which
//                   the running sum of those weights passes the draw
// Every logit is read once in the first launch, and one row of each sequence
// again in the second: bound by memory. The exponentials and sums are fp64. The
// running sum over 128256 weights has intervals of 1e-5 and less, of which fp32
// weights (6e-8 each, and as much in p's and q's normalisers) would give some
// draws to a neighbour. gfx950 runs fp64 fma at the fp32 rate, so a logit's 20
// fp64 operations stay under its 4 bytes of traffic.
#include <algorithm>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "sampling.h"

namespace lcr {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kSlice = 4096;                        // logits of a block
constexpr int kPerThread = kSlice / kVerifyThreads;  // 16
constexpr int kPickThreads = 1024;
constexpr int kPickPer = kSlice / kPickThreads;

// A row's slice: its sum of exp((l - max) / T), and its argmax key (the maximum
// is the key's value half).
struct SliceStats {
  double sum;
  unsigned long long key;
};

// What a row's distribution is: exp((l - max) / T) / sum where max is finite,
// else (sum = 0) one at the index `hot`.
struct RowStats {
  double max;
  double sum;
  int hot;
};

// What verify_pick needs of a sequence: `kept` drafts, the row and its
// distribution, and whether there is a draft's row to take off.
struct SequencePlan {
  int kept;
  int row;           // -1: the sequence has no rows
  int greedy_id;     // >= 0: the id itself
  int subtract;      // 1: weights max(p - q, 0)
  RowStats target;
  RowStats draft;    // sum = 0: one at the index `hot`
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
  SliceStats* stats;    // [rows][2][slices]
  double2* totals;      // [batch][slices]: sum of max(p - q, 0), sum of p
  SequencePlan* plans;  // [batch]
  int batch;
  int rows;
  int max_draft;
  int vocab;
  int slices;
  int logits_stride;
  bool vectors;         // rows on 16-byte boundaries
};

// exp(x) for x <= 0 in fp64: x = k ln2 + r (ln2 in two parts, the high one with
// 32 significant bits so that k ln2_hi is exact), the Taylor polynomial of
// degree 12 (|r| <= 0.347: truncated by 2e-16), scaled by 2^k. 0 below -708,
// where the result leaves the normal range.
__device__ __forceinline__ double exp_negative(double x) {
  const double y = fmax(x, -708.0);
  const double k = __builtin_rint(y * 1.44269504088896340736);
  double r = __builtin_fma(k, -6.93147180369123816490e-01, y);
  r = __builtin_fma(k, -1.90821492927058770002e-10, r);
  double p = 2.08767569878680989792e-09;
  p = __builtin_fma(p, r, 2.50521083854417187751e-08);
  p = __builtin_fma(p, r, 2.75573192239858906526e-07);
  p = __builtin_fma(p, r, 2.75573192239858906526e-06);
  p = __builtin_fma(p, r, 2.48015873015873015873e-05);
  p = __builtin_fma(p, r, 1.98412698412698412698e-04);
  p = __builtin_fma(p, r, 1.38888888888888888889e-03);
  p = __builtin_fma(p, r, 8.33333333333333333333e-03);
  p = __builtin_fma(p, r, 4.16666666666666666667e-02);
  p = __builtin_fma(p, r, 1.66666666666666666667e-01);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return x < -708.0 ? 0.0 : __builtin_ldexp(p, static_cast<int>(k));
}

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

__device__ __forceinline__ double wave_inclusive_scan_f64(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double other = __shfl_up(v, o, 64);
    if (lane_id() >= o) v += other;
  }
  return v;
}

__device__ __forceinline__ float key_logit(unsigned long long key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return u32_as_f32((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// A logit's key: NaN as -inf, -0 as 0 (equal logits tie on the index alone).
__device__ __forceinline__ float clean_logit(float l) { return l != l ? -__builtin_huge_valf() : l + 0.0f; }

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

// Weight of a logit against a row's maximum.
__device__ __forceinline__ double logit_weight(float l, double max, double inv_t) {
  return l == -__builtin_huge_valf() ? 0.0 : exp_negative((static_cast<double>(l) - max) * inv_t);
}

// Probability of index i with logit l in a row's distribution.
__device__ __forceinline__ double probability(const RowStats& r, double inv_sum, float l, int i, double inv_t) {
  return r.sum > 0.0 ? logit_weight(clean_logit(l), r.max, inv_t) * inv_sum : (i == r.hot ? 1.0 : 0.0);
}

// kCount logits of a row from index `first` (all of the block's at once, so
// they arrive together); -inf behind the vocabulary's end.
template <int kCount>
__device__ __forceinline__ void load_logits(float* out, const float* row, int first, int vocab, bool vectors) {
  static_assert(kCount == 4, "one 16-byte load");
  if (vectors && first + 4 <= vocab) {
    const float4 v = *reinterpret_cast<const float4*>(row + first);
    out[0] = v.x;
    out[1] = v.y;
    out[2] = v.z;
    out[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = first + j < vocab ? row[first + j] : -__builtin_huge_valf();
  }
}

// The sequence of a row (the batch's size for a row behind the last), and its
// first row and row count. Every thread of the block reads its share of the
// starts; a bisection would be a chain of as many loads. `lds` holds 4 ints.
__device__ __forceinline__ int sequence_of(const VerifyArgs& a, int row, int* lds) {
  int below = 0;
  for (int b = threadIdx.x; b <= a.batch; b += kVerifyThreads) below += a.row_starts[b] <= row ? 1 : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane_id() == 0) lds[threadIdx.x >> 6] = below;
  __syncthreads();
  below = 0;
#pragma unroll
  for (int w = 0; w < kVerifyWaves; ++w) below += lds[w];
  __syncthreads();
  return below - 1;
}

__device__ __forceinline__ double block_sum_f64(double v, double* lds) {
  v = wave_sum_f64(v);
  if (lane_id() == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = lds[0];
#pragma unroll
  for (int w = 1; w < kVerifyWaves; ++w) sum += lds[w];
  __syncthreads();
  return sum;
}

__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyArgs a) {
  __shared__ int lds_count[kVerifyWaves];
  __shared__ unsigned long long lds_key[16];
  __shared__ double lds_sum[kVerifyWaves];
  const int slice = blockIdx.x;
  const int row = blockIdx.y;
  const bool is_draft = blockIdx.z != 0;
  const float* logits = (is_draft ? a.draft : a.target) + static_cast<size_t>(row) * a.logits_stride;
  float l[kPerThread];
  auto load = [&] {
#pragma unroll
    for (int j = 0; j < kPerThread / 4; ++j) {
      load_logits<4>(l + 4 * j, logits, slice * kSlice + 4 * (j * kVerifyThreads + static_cast<int>(threadIdx.x)),
                     a.vocab, a.vectors);
    }
  };
  // Nearly every target row counts: its logits are requested before the block
  // knows. Every sequence has a draft row that does not.
  if (!is_draft) load();
  const int b = sequence_of(a, row, lds_count);
  if (b < 0 || b >= a.batch) return;
  const int in_sequence = row - a.row_starts[b];
  const int drafts = min(a.row_starts[b + 1] - a.row_starts[b] - 1, a.max_draft);
  const float t = a.temperatures[b];
  const bool greedy = !(t > 0.0f);
  if (in_sequence > drafts || (is_draft && (greedy || in_sequence == drafts))) return;
  if (is_draft) load();
  unsigned long long key = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int i = slice * kSlice + 4 * ((j / 4) * kVerifyThreads + static_cast<int>(threadIdx.x)) + (j & 3);
    l[j] = clean_logit(l[j]);
    if (i < a.vocab) key = umax64(key, argmax_key(l[j], static_cast<uint32_t>(i)));
  }
  key = block_max_u64(key, lds_key);
  double sum = 0.0;
  const float max = key_logit(key);
  if (!greedy && finite(max)) {
    const double inv_t = 1.0 / static_cast<double>(t);
    const double m = max;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) sum += logit_weight(l[j], m, inv_t);
    sum = block_sum_f64(sum, lds_sum);
  }
  if (threadIdx.x == 0) a.stats[(static_cast<size_t>(row) * 2 + (is_draft ? 1 : 0)) * a.slices + slice] = SliceStats{sum, key};
}

// A row's slices joined, by one wave; every lane gets the result.
__device__ __forceinline__ RowStats join_slices(const SliceStats* s, int slices, double inv_t) {
  unsigned long long key = 0;
  for (int i = lane_id(); i < slices; i += 64) key = umax64(key, s[i].key);
  key = wave_max_u64(key);
  const float max = key_logit(key);
  double sum = 0.0;
  if (finite(max)) {
    for (int i = lane_id(); i < slices; i += 64) {
      const float m = key_logit(s[i].key);
      if (finite(m)) sum += s[i].sum * exp_negative((static_cast<double>(m) - max) * inv_t);
    }
    sum = wave_sum_f64(sum);
  }
  return RowStats{max, sum, argmax_id(key)};
}

__global__ __launch_bounds__(kVerifyThreads) void verify_residual_kernel(VerifyArgs a) {
  __shared__ int shared_kept;
  __shared__ RowStats shared_target, shared_draft;
  __shared__ int shared_subtract;
  __shared__ double lds_sum[kVerifyWaves];
  const int slice = blockIdx.x;
  const int b = blockIdx.y;
  const int lane = lane_id();
  const int first = a.row_starts[b];
  const int count = a.row_starts[b + 1] - first;
  SequencePlan& plan = a.plans[b];
  // Rows of a table that is no ascending list of rows are not read.
  if (count <= 0 || first < 0 || first > a.rows - count) {
    if (slice == 0 && threadIdx.x == 0) plan.row = -1;
    return;
  }
  const int drafts = min(count - 1, a.max_draft);
  const float t = a.temperatures[b];
  const bool greedy = !(t > 0.0f);
  const double inv_t = greedy ? 0.0 : 1.0 / static_cast<double>(t);
  // Drafts kept, in order, by wave 0.
  if (threadIdx.x < 64) {
    int kept = 0;
    RowStats target{}, draft{};
    for (;; ++kept) {
      const int row = first + kept;
      target = join_slices(a.stats + static_cast<size_t>(row) * 2 * a.slices, a.slices, inv_t);
      if (kept == drafts) break;
      const int x = a.draft_ids[row];
      if (greedy) {
        if (x != target.hot) break;
        continue;
      }
      draft = RowStats{0.0, 0.0, x};
      if (a.draft != nullptr) {
        const RowStats d = join_slices(a.stats + (static_cast<size_t>(row) * 2 + 1) * a.slices, a.slices, inv_t);
        draft.max = d.max;
        draft.sum = d.sum;
      }
      if (x < 0 || x >= a.vocab) break;
      const size_t at = static_cast<size_t>(row) * a.logits_stride + x;
      const double p = probability(target, 1.0 / target.sum, a.target[at], x, inv_t);
      const double q = draft.sum > 0.0 ? probability(draft, 1.0 / draft.sum, a.draft[at], x, inv_t) : 1.0;
      if (!(static_cast<double>(a.accept_uniforms[row]) * q < p)) break;
    }
    if (lane == 0) {
      shared_kept = kept;
      shared_target = target;
      shared_draft = draft;
      shared_subtract = kept < drafts ? 1 : 0;
    }
  }
  __syncthreads();
  const int kept = shared_kept;
  const RowStats target = shared_target, draft = shared_draft;
  const int subtract = shared_subtract;
  const int row = first + kept;
  if (slice == 0 && threadIdx.x == 0) {
    plan = SequencePlan{kept, row, greedy ? target.hot : -1, subtract, target, draft};
  }
  if (greedy) return;
  const size_t at = static_cast<size_t>(row) * a.logits_stride;
  const double inv_p = 1.0 / target.sum, inv_q = 1.0 / draft.sum;
  double rest = 0.0, whole = 0.0;
#pragma unroll
  for (int j = 0; j < kPerThread / 4; ++j) {
    const int i0 = slice * kSlice + 4 * (j * kVerifyThreads + static_cast<int>(threadIdx.x));
    float lp[4], lq[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load_logits<4>(lp, a.target + at, i0, a.vocab, a.vectors);
    if (subtract && draft.sum > 0.0) load_logits<4>(lq, a.draft + at, i0, a.vocab, a.vectors);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i0 + e >= a.vocab) continue;
      const double p = probability(target, inv_p, lp[e], i0 + e, inv_t);
      whole += p;
      if (subtract) rest += fmax(p - probability(draft, inv_q, lq[e], i0 + e, inv_t), 0.0);
    }
  }
  rest = block_sum_f64(rest, lds_sum);
  whole = block_sum_f64(whole, lds_sum);
  if (threadIdx.x == 0) a.totals[static_cast<size_t>(b) * a.slices + slice] = make_double2(rest, whole);
}

__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ int shared_slice, shared_subtract;
  __shared__ double shared_before, shared_goal;
  __shared__ double wave_total[kPickThreads / 64];
  __shared__ int wave_first[kPickThreads / 64], wave_last[kPickThreads / 64];
  const int b = blockIdx.x;
  const int lane = lane_id();
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const SequencePlan plan = a.plans[b];
  int32_t* ids = a.out_ids + static_cast<size_t>(b) * (a.max_draft + 1);
  const int kept = plan.row < 0 ? 0 : plan.kept;
  // The kept drafts, and -1 behind the drawn token, which is written last.
  for (int i = threadIdx.x; i <= a.max_draft; i += kPickThreads) {
    if (plan.row < 0 || i != kept) ids[i] = i < kept ? a.draft_ids[plan.row - kept + i] : -1;
  }
  if (threadIdx.x == 0) {
    a.out_counts[b] = plan.row < 0 ? 0 : kept + 1;
    if (plan.row >= 0 && plan.greedy_id >= 0) ids[kept] = plan.greedy_id;
  }
  if (plan.row < 0 || plan.greedy_id >= 0) return;  // the whole block
  // The slice: the first whose running sum passes the draw. Rounding may leave
  // none: then the last slice with a weight.
  if (wave == 0) {
    const double2* totals = a.totals + static_cast<size_t>(b) * a.slices;
    double rest = 0.0;
    for (int s = lane; s < a.slices; s += 64) rest += totals[s].x;
    rest = wave_sum_f64(rest);
    const bool subtract = plan.subtract != 0 && rest > 0.0;
    double whole = 0.0;
    for (int base = 0; base < a.slices; base += 64) {
      const int s = base + lane;
      const double v = s < a.slices ? (subtract ? totals[s].x : totals[s].y) : 0.0;
      whole += __shfl(wave_inclusive_scan_f64(v), 63, 64);
    }
    const double goal = static_cast<double>(a.sample_uniforms[b]) * whole;
    double before = 0.0, last_before = 0.0;
    int found = -1, last = 0;
    for (int base = 0; base < a.slices && found < 0; base += 64) {
      const int s = base + lane;
      const double v = s < a.slices ? (subtract ? totals[s].x : totals[s].y) : 0.0;
      const double incl = wave_inclusive_scan_f64(v);
      const unsigned long long weighty = __ballot(v > 0.0);
      const unsigned long long hit = __ballot(v > 0.0 && before + incl > goal);
      const int pick = hit != 0 ? __ffsll(hit) - 1 : (weighty != 0 ? 63 - __clzll(weighty) : -1);
      if (pick >= 0) {
        last = base + pick;
        last_before = before + __shfl(incl - v, pick, 64);
        if (hit != 0) found = last;
      }
      before += __shfl(incl, 63, 64);
    }
    if (lane == 0) {
      shared_slice = last;
      shared_before = last_before;
      shared_goal = goal;
      shared_subtract = subtract ? 1 : 0;
    }
  }
  __syncthreads();
  const int slice = shared_slice;
  const bool subtract = shared_subtract != 0;
  const double inv_t = 1.0 / static_cast<double>(a.temperatures[b]);
  const double inv_p = 1.0 / plan.target.sum, inv_q = 1.0 / plan.draft.sum;
  const size_t at = static_cast<size_t>(plan.row) * a.logits_stride;
  // Four neighbouring weights a thread, their running sum within the slice.
  static_assert(kPickPer == 4, "one 16-byte load a thread");
  const int i0 = slice * kSlice + 4 * static_cast<int>(threadIdx.x);
  float lp[4], lq[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  load_logits<4>(lp, a.target + at, i0, a.vocab, a.vectors);
  if (subtract && plan.draft.sum > 0.0) load_logits<4>(lq, a.draft + at, i0, a.vocab, a.vectors);
  double run[4];
  double sum = 0.0;
  bool weighty[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    double w = 0.0;
    if (i0 + e < a.vocab) {
      w = probability(plan.target, inv_p, lp[e], i0 + e, inv_t);
      if (subtract) w = fmax(w - probability(plan.draft, inv_q, lq[e], i0 + e, inv_t), 0.0);
    }
    sum += w;
    run[e] = sum;
    weighty[e] = w > 0.0;
  }
  const double incl = wave_inclusive_scan_f64(sum);
  if (lane == 63) wave_total[wave] = incl;
  __syncthreads();
  double before = shared_before;
  for (int w = 0; w < wave; ++w) before += wave_total[w];
  before += incl - sum;
  int hit = INT32_MAX, last = -1;
#pragma unroll
  for (int e = 3; e >= 0; --e) {
    if (weighty[e]) {
      last = max(last, i0 + e);
      if (before + run[e] > shared_goal) hit = i0 + e;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    hit = min(hit, __shfl_xor(hit, o, 64));
    last = max(last, __shfl_xor(last, o, 64));
  }
  if (lane == 0) {
    wave_first[wave] = hit;
    wave_last[wave] = last;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < kPickThreads / 64; ++w) {
      hit = min(hit, wave_first[w]);
      last = max(last, wave_last[w]);
    }
    ids[kept] = hit != INT32_MAX ? hit : max(last, 0);
  }
}

int slices_for(int vocab) { return (vocab + kSlice - 1) / kSlice; }

struct VerifyLayout {
  size_t totals_at, plans_at, bytes;
};

VerifyLayout layout_for(int batch, int rows, int vocab) {
  const size_t slices = static_cast<size_t>(slices_for(vocab));
  VerifyLayout l;
  l.totals_at = static_cast<size_t>(rows) * 2 * slices * sizeof(SliceStats);
  l.plans_at = l.totals_at + static_cast<size_t>(batch) * slices * sizeof(double2);
  l.bytes = l.plans_at + static_cast<size_t>(batch) * sizeof(SequencePlan);
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
  CAPI_CHECK(max_draft < INT32_MAX, "batch_verify takes fewer than 2^31 - 1 drafts");
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
  a.stats = reinterpret_cast<SliceStats*>(ws);
  a.totals = reinterpret_cast<double2*>(ws + layout.totals_at);
  a.plans = reinterpret_cast<SequencePlan*>(ws + layout.plans_at);
  a.batch = batch;
  a.rows = rows;
  a.max_draft = max_draft;
  a.vocab = vocab;
  a.slices = slices_for(vocab);
  a.logits_stride = logits_stride;
  a.vectors = logits_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(target_logits) & 15u) == 0 &&
              (reinterpret_cast<uintptr_t>(draft_logits) & 15u) == 0;
  auto s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    const dim3 grid(static_cast<unsigned>(a.slices), static_cast<unsigned>(rows), a.draft != nullptr ? 2u : 1u);
    verify_stats_kernel<<<grid, kVerifyThreads, 0, s>>>(a);
    CAPI_LAUNCHED();
  }
  const dim3 grid(static_cast<unsigned>(a.slices), static_cast<unsigned>(batch));
  verify_residual_kernel<<<grid, kVerifyThreads, 0, s>>>(a);
  CAPI_LAUNCHED();
  verify_pick_kernel<<<static_cast<unsigned>(batch), kPickThreads, 0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
