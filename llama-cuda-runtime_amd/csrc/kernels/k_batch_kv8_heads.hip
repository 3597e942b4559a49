// lcr_batch_norm_rope_write_kv8: per-head RMSNorm and rotation of a step's rows,
// queries to a buffer, keys and values appended to a cache of 8-bit numbers.
//
// A block of 16 positions of a head shares a scale, so the rows of a call that lie
// in one block have to know each other's largest value: it decides whether the scale
// holds, and where it does not, the numbers held are rounded to the new one. A row is
// its block's first if none of the 15 rows before it lies there, and the block's others
// are among the 15 behind it.
//
// Heads of 64 and 128: a wave takes 16 rows that hold whole blocks, four lanes a row,
// whether they are one sequence's or 16 sequences'; the blocks' largest values meet in
// LDS. Bound by memory and, at many rows, by what it takes to norm and rotate in fp64
// (which the vector units run as fast as fp32): 6779 rows of 32 + 8 + 8 heads of 64
// 18.2 us for 78 MB, 4.3 TB/s of a copy's 5.2; of 16 + 8 + 8 heads of 128 33 us for
// 100 MB (35 with norms, 24 without the keys); 8 rows 4.2 us, a chain of three reads; 64
// sequences of up to five rows, of heads of 128, 6.8.
#include <algorithm>
#include <cstdint>

#include "../capi_util.h"
#include "head_rotation.h"
#include "kv8.h"

namespace lcr {
namespace {

constexpr int kHeadsThreads = 256;
constexpr int kHeadsWaves = kHeadsThreads / 64;
constexpr int kMaxHeadDim = 256;
// Waves a compute unit that a call's keys and values are spread over, more or less:
// with more rows a wave takes several heads of its own, having looked for their blocks
// once. With 64, 32 and a wave a head: 28783 rows of 32 on 8 heads of 64 91, 89 and 98
// us, of 16 on 8 of 128 127, 129 and 133, 10049 of 32 on 32 of 64 62, 62 and 76, 20000
// of sequences of their own 81, 83 and 87.
constexpr int kMostWaves = 64;
// Rows that do not fill a window leave a second set in most: every second one goes to
// waves of its own while that gives no SIMD two (by the waves a compute unit there are
// without). 64 sequences of up to five rows, 16 on 8 heads of 128, 9.7 us in turn, 7.1
// so; 140 of them 10.8 and 10.6, 700 of one row 5.2 and 6.3.
constexpr int kHalvedWaves = 2;

struct Heads8Args {
  elem_t* q_out;
  Kv8View view;
  const elem_t* q;
  const elem_t* k;
  const elem_t* v;
  const elem_t* q_norm;
  const elem_t* k_norm;
  float eps;
  const float2* table;
  int table_positions;
  const int32_t* positions;
  const int32_t* slots;
  int tokens;
  int num_heads;
  int pool_slots;  // pool_pages * page_size
  int src_row_stride;
};

__device__ __forceinline__ bool row_is_live(const Heads8Args& a, int slot, int position) {
  return slot >= 0 && slot < a.pool_slots && position >= 0 && position < a.table_positions;
}

// Which rows of a call write to a block: lanes 0 .. 30 look at rows row - 15 ..
// row + 15.
struct BlockRows {
  int slot;           // this lane's row's, -1: none that counts
  unsigned long long members;  // lanes whose rows lie in the block, from lane 15 (the row itself) on
  bool first;         // the row is live, and the first of its block
};

__device__ __forceinline__ BlockRows find_block_rows(const Heads8Args& a, int row) {
  const int at = row - 15 + lane_id();
  BlockRows r{-1, 0, false};
  if (lane_id() < 31 && at >= 0 && at < a.tokens) {
    const int slot = a.slots[at], position = a.positions[at];
    if (row_is_live(a, slot, position)) r.slot = slot;
  }
  const int mine = __builtin_amdgcn_readlane(r.slot, 15);
  const unsigned long long same = __ballot(r.slot >= 0 && mine >= 0 && (r.slot ^ mine) < kKv8Block);
  r.first = mine >= 0 && (same & 0x7fffull) == 0;
  r.members = same;
  return r;
}

// Any head_dim and any alignment of the rows: a wave per (row, query head) and per
// (row, kv head, keys or values), pairs (i, i + head_dim / 2) spread over the
// lanes, a block's rows one after another.
struct Pairs {
  float lo[kMaxHeadDim / 128];
  float hi[kMaxHeadDim / 128];
};

__device__ __forceinline__ Pairs key_pairs(const Heads8Args& a, const elem_t* src, int position) {
  const int half = a.view.head_dim / 2;
  double x[kMaxHeadDim / 128], y[kMaxHeadDim / 128];
  double square = 0.0;
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 128; ++j) {
    const int i = lane_id() + 64 * j;
    x[j] = y[j] = 0.0;
    if (i < half) {
      x[j] = elem_to_float(src[i]);
      y[j] = elem_to_float(src[half + i]);
    }
    square = __builtin_fma(x[j], x[j], __builtin_fma(y[j], y[j], square));
  }
  if (a.k_norm != nullptr) {
    const double scale = 1.0 / sqrt(wave_sum_f64(square) / a.view.head_dim + static_cast<double>(a.eps));
#pragma unroll
    for (int j = 0; j < kMaxHeadDim / 128; ++j) {
      const int i = lane_id() + 64 * j;
      if (i < half) {
        x[j] = x[j] * scale * elem_to_float(a.k_norm[i]);
        y[j] = y[j] * scale * elem_to_float(a.k_norm[half + i]);
      }
    }
  }
  Pairs p;
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 128; ++j) {
    const int i = lane_id() + 64 * j;
    p.lo[j] = p.hi[j] = 0.0f;
    if (i < half) {
      const float2 cs = a.table[static_cast<size_t>(position) * half + i];
      p.lo[j] = kv8_clamped(static_cast<float>(x[j] * cs.x - y[j] * cs.y));
      p.hi[j] = kv8_clamped(static_cast<float>(y[j] * cs.x + x[j] * cs.y));
    }
  }
  return p;
}

__device__ __forceinline__ Pairs value_pairs(const Heads8Args& a, const elem_t* src) {
  const int half = a.view.head_dim / 2;
  Pairs p;
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 128; ++j) {
    const int i = lane_id() + 64 * j;
    p.lo[j] = i < half ? kv8_clamped(elem_to_float(src[i])) : 0.0f;
    p.hi[j] = i < half ? kv8_clamped(elem_to_float(src[half + i])) : 0.0f;
  }
  return p;
}

__device__ void append_any(const Heads8Args& a, int row, int head, bool is_key) {
  const int d = a.view.head_dim;
  const int half = d / 2;
  const BlockRows rows = find_block_rows(a, row);
  if (!rows.first) return;
  const elem_t* src = (is_key ? a.k : a.v) + static_cast<size_t>(head) * d;
  auto pairs_of = [&](int lane) {
    const int r = row - 15 + lane;
    const elem_t* from = src + static_cast<size_t>(r) * static_cast<size_t>(a.src_row_stride);
    return is_key ? key_pairs(a, from, a.positions[r]) : value_pairs(a, from);
  };
  float largest = 0.0f;
  uint32_t written = 0;  // positions of the block
  for (unsigned long long m = rows.members; m != 0; m &= m - 1) {
    const int lane = __builtin_ctzll(m);
    written |= 1u << (__builtin_amdgcn_readlane(rows.slot, lane) % kKv8Block);
    const Pairs p = pairs_of(lane);
#pragma unroll
    for (int j = 0; j < kMaxHeadDim / 128; ++j) largest = fmaxf(largest, fmaxf(kv8_size(p.lo[j]), kv8_size(p.hi[j])));
  }
  largest = wave_max(largest);
  const int slot = __builtin_amdgcn_readlane(rows.slot, 15);
  const int page = slot / a.view.page_size;
  const int block = (slot - page * a.view.page_size) / kKv8Block;
  uint8_t* bytes = (is_key ? a.view.keys : a.view.values) + a.view.block_at(page, head, block);
  float* scale_at = (is_key ? a.view.key_scales : a.view.value_scales) + a.view.scale_at(page, head, block);
  auto byte_of = [&](int t, int i) { return is_key ? kv8_key_byte(d, t, i) : kv8_value_byte(d, t, i); };
  float scale = power_of_two(kv8_exponent_for(largest));
  if ((written & 1u) == 0) {
    const float held = *scale_at;
    scale = fmaxf(scale, held);
    if (scale > held) {
      const float move = held / scale;
      for (int n = lane_id(); n < kKv8Block * d; n += 64) {
        const int t = n / d, i = n - t * d;
        if ((written >> t & 1u) == 0) {
          uint8_t* b = bytes + byte_of(t, i);
          *b = static_cast<uint8_t>(kv8_pair(kv8_number(*b) * move, 0.0f));
        }
      }
    }
  }
  if (lane_id() == 0) *scale_at = scale;
  const float inverse = 1.0f / scale;
  for (unsigned long long m = rows.members; m != 0; m &= m - 1) {
    const int lane = __builtin_ctzll(m);
    const int t = __builtin_amdgcn_readlane(rows.slot, lane) % kKv8Block;
    const Pairs p = pairs_of(lane);
#pragma unroll
    for (int j = 0; j < kMaxHeadDim / 128; ++j) {
      const int i = lane_id() + 64 * j;
      if (i >= half) continue;
      const uint32_t w = kv8_pair(p.lo[j] * inverse, p.hi[j] * inverse);
      bytes[byte_of(t, i)] = static_cast<uint8_t>(w);
      bytes[byte_of(t, half + i)] = static_cast<uint8_t>(w >> 8);
    }
  }
}

__device__ void query_any(const Heads8Args& a, int row, int head) {
  if (!row_is_live(a, a.slots[row], a.positions[row])) return;
  const int d = a.view.head_dim;
  const int half = d / 2;
  const elem_t* src = a.q + static_cast<size_t>(row) * static_cast<size_t>(a.src_row_stride) + static_cast<size_t>(head) * d;
  elem_t* dst = a.q_out + (static_cast<size_t>(row) * a.num_heads + head) * d;
  float x[kMaxHeadDim / 128], y[kMaxHeadDim / 128];
  float square = 0.0f;
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 128; ++j) {
    const int i = lane_id() + 64 * j;
    x[j] = i < half ? elem_to_float(src[i]) : 0.0f;
    y[j] = i < half ? elem_to_float(src[half + i]) : 0.0f;
    square = __builtin_fmaf(x[j], x[j], __builtin_fmaf(y[j], y[j], square));
  }
  const float scale = 1.0f / sqrtf(wave_sum(square) / static_cast<float>(d) + a.eps);
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 128; ++j) {
    const int i = lane_id() + 64 * j;
    if (i >= half) continue;
    if (a.q_norm != nullptr) {
      x[j] = x[j] * scale * elem_to_float(a.q_norm[i]);
      y[j] = y[j] * scale * elem_to_float(a.q_norm[half + i]);
    }
    const float2 r = rope_rotate(x[j], y[j], a.table[static_cast<size_t>(a.positions[row]) * half + i]);
    dst[i] = float_to_elem(r.x);
    dst[half + i] = float_to_elem(r.y);
  }
}

__global__ __launch_bounds__(kHeadsThreads) void batch_kv8_heads_any_kernel(Heads8Args a) {
  const int heads = a.num_heads + 2 * a.view.num_kv_heads;
  const long long unit = static_cast<long long>(blockIdx.x) * kHeadsWaves + (threadIdx.x >> 6);
  const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(unit / heads));
  const int head = __builtin_amdgcn_readfirstlane(static_cast<int>(unit - static_cast<long long>(row) * heads));
  if (row >= a.tokens) return;
  if (head < a.num_heads) {
    query_any(a, row, head);
  } else {
    const int n = head - a.num_heads;
    append_any(a, row, n % a.view.num_kv_heads, n < a.view.num_kv_heads);
  }
}

// ---------------------------------------------------------------------------
// Heads of 64 and 128, rows on 16 bytes
// ---------------------------------------------------------------------------

// Rows of a window, whose blocks are some waves' work, and the rows about them that
// may lie in the same blocks: lane n looks at row first - 15 + n.
constexpr int kWindowRows = 16;
constexpr int kWindowLanes = kWindowRows + 2 * 15;

struct Window {
  int first;      // row
  int slot;       // this lane's row's, -1: none that counts
  int position;
  int leader;     // the lane of its block's first row
  unsigned long long leaders;  // lanes of the window that are first of their blocks

  __device__ __forceinline__ Window(const Heads8Args& a, int first_row) : first(first_row), slot(-1), position(0) {
    const int lane = lane_id();
    const int row = first - 15 + lane;
    if (lane < kWindowLanes && row >= 0 && row < a.tokens) {
      const int s = a.slots[row];
      position = a.positions[row];
      if (row_is_live(a, s, position)) slot = s;
    }
    // Each lane looks back: a wave shift for each of the 15 lanes before it.
    const int block = slot >> 4;
    int before = block;
    leader = lane;
#pragma unroll
    for (int o = 1; o <= 15; ++o) {
      before = __builtin_amdgcn_update_dpp(-1, before, 0x138, 0xF, 0xF, false);  // wave_shr:1
      if (before == block) leader = lane - o;
    }
    leaders = __ballot(slot >= 0 && leader == lane && lane >= 15 && lane < 15 + kWindowRows);
  }
};
static_assert(kKv8Block == 16, "a slot's block is slot >> 4");

// Up to 16 rows that follow each other, with blocks that lie among them whole: four
// lanes a row. One new token each of 16 sequences, or 16 of one, is one such set.
struct RowSet {
  int row;         // this lane's, -1: none that counts
  int position;
  int t;           // its position in its block
  int first;       // which of the set's rows is the first of its block
  size_t block;    // first byte of the block of the first kv head, and its scale
  size_t scale;
  uint32_t written;  // the block's positions that this call writes

  // Takes a set's leaders out of `left`.
  __device__ __forceinline__ RowSet(const Heads8Args& a, const Window& win, unsigned long long& left,
                                    uint32_t* lds_written) {
    const int start = __builtin_ctzll(left);
    // leaders with rows behind the set wait for one of their own
    unsigned long long cut = __ballot(win.slot >= 0 && lane_id() >= start + 16 && win.leader >= start &&
                                      win.leader < start + 16);
    unsigned long long whole = left & (0xffffull << start);
    for (; cut != 0; cut &= cut - 1) whole &= ~(1ull << __builtin_amdgcn_readlane(win.leader, __builtin_ctzll(cut)));
    left &= ~whole;
    const int group = lane_id() >> 2;
    const int from = start + group;  // at most 30 + 15
    const int slot = __shfl(win.slot, from, 64);
    const int leader = __shfl(win.leader, from, 64);
    position = __shfl(win.position, from, 64);
    row = slot >= 0 && (whole >> leader & 1ull) != 0 ? win.first - 15 + from : -1;
    t = slot & (kKv8Block - 1);
    first = row >= 0 ? leader - start : group;
    const int counted = row >= 0 ? slot : 0;
    const int page = counted / a.view.page_size;
    const int n = (counted - page * a.view.page_size) / kKv8Block;
    block = a.view.block_at(page, 0, n);
    scale = a.view.scale_at(page, 0, n);
    if (lane_id() < 16) lds_written[lane_id()] = 0;
    wave_settled();
    if (row >= 0 && (lane_id() & 3) == 0) atomicOr(&lds_written[first], 1u << t);
    wave_settled();
    written = lds_written[first];
    wave_settled();
  }
  __device__ __forceinline__ bool leads() const { return row >= 0 && first == lane_id() >> 2; }
};

// The scale of a row's block, from the largest of this row's values (of four lanes):
// the larger of what the block's new values need and, unless the block begins, of what
// it has. `move`: what the numbers held are multiplied by, 1 where they stay.
__device__ __forceinline__ float block_scale(const RowSet& set, float held, float largest, uint32_t* lds_largest,
                                             float& move) {
  largest = fmaxf(largest, xor_lane<1>(largest));
  largest = fmaxf(largest, xor_lane<2>(largest));
  if (lane_id() < 16) lds_largest[lane_id()] = 0;
  wave_settled();
  // no less than 0, so that they compare as their bits do
  if (set.row >= 0 && (lane_id() & 3) == 0) atomicMax(&lds_largest[set.first], __builtin_bit_cast(uint32_t, largest));
  wave_settled();
  largest = __builtin_bit_cast(float, lds_largest[set.first]);
  wave_settled();
  const float need = power_of_two(kv8_exponent_for(largest));
  move = 1.0f;
  if (set.written & 1u) return need;
  const float after = fmaxf(need, held);
  if (after > held) move = held / after;
  return after;
}

__device__ __forceinline__ uint32_t moved_numbers(uint32_t w, float move) {
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = kv8_number(static_cast<uint8_t>(w >> (8 * i))) * move;
  return kv8_pair(x[0], x[1]) | kv8_pair(x[2], x[3]) << 16;
}

// Rounds what blocks hold to their larger scales, but for the positions written: block
// after block, by the whole wave. Stores touch only bytes that no others do, so that
// they need no order among the new numbers'.
template <int kHeadDim, bool kKeys>
__device__ __forceinline__ void move_blocks(const RowSet& set, uint8_t* numbers, float move) {
  for (unsigned long long m = __ballot(set.leads() && (lane_id() & 3) == 0 && move != 1.0f); m != 0; m &= m - 1) {
    const int lane = __builtin_ctzll(m);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(set.block), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(set.block >> 32), lane);
    const uint32_t written = __builtin_amdgcn_readlane(set.written, lane);
    const float by = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, move), lane));
    uint8_t* bytes = numbers + (static_cast<size_t>(hi) << 32 | lo);
    constexpr int kChunks = kHeadDim / 64;  // 16 bytes a lane
    vec16 old[kChunks];
#pragma unroll
    for (int h = 0; h < kChunks; ++h) old[h] = load16(bytes + 16 * (lane_id() + 64 * h));
#pragma unroll
    for (int h = 0; h < kChunks; ++h) {
      // 16 dims of one position, or four of four
      const int at = 16 * (lane_id() + 64 * h);
      const uint32_t skip = kKeys ? (written >> (at / kHeadDim) & 1u ? 15u : 0u) : written >> (at / (4 * kHeadDim) * 4) & 15u;
      vec16 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w.w[i] = moved_numbers(old[h].w[i], by);
      if (skip == 0u) {
        store16(bytes + at, w);
      } else if (skip != 15u) {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          if ((skip >> (n & 3) & 1u) == 0) bytes[at + n] = static_cast<uint8_t>(w.w[n / 4] >> (8 * (n & 3)));
        }
      }
    }
  }
}

// What the largest of `n` values is, for their block's scale. Values past the largest
// that is held are clamped and infinities made NaN, where there are any.
template <int n>
__device__ __forceinline__ float largest_of(float* v) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < n; j += 2) {
    most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, fabsf(v[j])), fabsf(v[j + 1]));
  }
  if (__any(!(most <= kKv8Largest))) {
    most = 0.0f;
#pragma unroll
    for (int j = 0; j < n; ++j) {
      v[j] = fabsf(v[j]) < __builtin_huge_valf() ? kv8_clamped(v[j]) : __builtin_nanf("");
      most = fmaxf(most, kv8_size(v[j]));
    }
  }
  return most;
}

__device__ __forceinline__ void unpack4(const uint2& w, float* out) {
  out[0] = elem_lo(w.x);
  out[1] = elem_hi(w.x);
  out[2] = elem_lo(w.y);
  out[3] = elem_hi(w.y);
}

// Four values over their scale as numbers: none is infinite.
__device__ __forceinline__ uint32_t four_numbers(const float* v, float inverse) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, w, true);
  return static_cast<uint32_t>(w);
}

// Keys of a set: a lane has a quarter of both halves of a head, so that pairs stay in
// their lanes and the norm is two exchanges.
template <int kHeadDim>
__device__ __forceinline__ void append_keys(const Heads8Args& a, const RowSet& set, int head, uint32_t* lds_largest) {
  constexpr int kHalf = kHeadDim / 2;
  constexpr int kPairs = kHeadDim / 8;  // of a lane
  const int i0 = kPairs * (lane_id() & 3);
  const size_t scale_at = set.scale + static_cast<size_t>(head) * static_cast<size_t>(a.view.scale_head_stride);
  const float held = a.view.key_scales[scale_at];
  const int row = max(set.row, 0);
  const elem_t* src = a.k + static_cast<size_t>(row) * static_cast<size_t>(a.src_row_stride) +
                      static_cast<size_t>(head) * kHeadDim + i0;
  const float4* cs = reinterpret_cast<const float4*>(a.table + static_cast<size_t>(set.row >= 0 ? set.position : 0) * kHalf + i0);
  float v[2 * kPairs];  // lower halves' elements, then the upper's
  if (set.row >= 0) {
#pragma unroll
    for (int j = 0; j < kPairs; j += 8) {
      unpack8(load16(src + j), v + j);
      unpack8(load16(src + kHalf + j), v + kPairs + j);
    }
    // Without a norm everything is multiplied with ones, as two forms of the loop below
    // cost the registers of both.
    const bool normed = a.k_norm != nullptr;
    const elem_t* weights = normed ? a.k_norm + i0 : src;
    double scale = 1.0;
    if (normed) {
      double square = 0.0;
#pragma unroll
      for (int j = 0; j < 2 * kPairs; ++j) square = __builtin_fma(static_cast<double>(v[j]), static_cast<double>(v[j]), square);
      square += xor_lane_f64<1>(square);
      square += xor_lane_f64<2>(square);
      scale = 1.0 / sqrt(square * (1.0 / kHeadDim) + static_cast<double>(a.eps));
      // widened again below: kept in fp64, they cost twice their registers
#pragma unroll
      for (int j = 0; j < 2 * kPairs; ++j) asm volatile("" : "+v"(v[j]));
    }
#pragma unroll
    for (int j = 0; j < kPairs; j += 4) {
      const float4 angle[2] = {cs[j / 2], cs[j / 2 + 1]};
      float wx[4], wy[4];
      unpack4(*reinterpret_cast<const uint2*>(weights + j), wx);
      unpack4(*reinterpret_cast<const uint2*>(weights + kHalf + j), wy);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const double x = static_cast<double>(v[j + n]) * scale * static_cast<double>(normed ? wx[n] : 1.0f);
        const double y = static_cast<double>(v[kPairs + j + n]) * scale * static_cast<double>(normed ? wy[n] : 1.0f);
        const double c = n & 1 ? angle[n / 2].z : angle[n / 2].x;
        const double s = n & 1 ? angle[n / 2].w : angle[n / 2].y;
        v[j + n] = static_cast<float>(x * c - y * s);
        v[kPairs + j + n] = static_cast<float>(y * c + x * s);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2 * kPairs; ++j) v[j] = 0.0f;
  }
  float move;
  const float scale = block_scale(set, held, largest_of<2 * kPairs>(v), lds_largest, move);
  uint8_t* const numbers = a.view.keys + static_cast<size_t>(head) * static_cast<size_t>(a.view.head_stride);
  if (set.row >= 0) {
    if (set.leads() && (lane_id() & 3) == 0) a.view.key_scales[scale_at] = scale;
    uint8_t* const to = numbers + set.block + kv8_key_byte(kHeadDim, set.t, i0);
    const float inverse = 1.0f / scale;
#pragma unroll
    for (int j = 0; j < kPairs; j += 8) {
      *reinterpret_cast<uint2*>(to + j) = make_uint2(four_numbers(v + j, inverse), four_numbers(v + j + 4, inverse));
      *reinterpret_cast<uint2*>(to + kHalf + j) =
          make_uint2(four_numbers(v + kPairs + j, inverse), four_numbers(v + kPairs + j + 4, inverse));
    }
  }
  move_blocks<kHeadDim, true>(set, numbers, move);
}

// Values of a set: a lane has four neighbouring dims of each 16. A position's bytes
// lie four apart, those of the three beside it between them. A row alone among its
// four reads them and writes all, unless they change their scale; rows together write
// their bytes. (4000 rows of sequences of their own, 16 on 8 heads of 128, 54 us with
// bytes alone.)
template <int kHeadDim>
__device__ __forceinline__ void append_values(const Heads8Args& a, const RowSet& set, int head, uint32_t* lds_largest) {
  constexpr int kFours = kHeadDim / 16;
  const int i0 = 4 * (lane_id() & 3);
  const size_t scale_at = set.scale + static_cast<size_t>(head) * static_cast<size_t>(a.view.scale_head_stride);
  const float held = a.view.value_scales[scale_at];
  const elem_t* src = a.v + static_cast<size_t>(max(set.row, 0)) * static_cast<size_t>(a.src_row_stride) +
                      static_cast<size_t>(head) * kHeadDim + i0;
  uint8_t* const numbers = a.view.values + static_cast<size_t>(head) * static_cast<size_t>(a.view.head_stride);
  uint8_t* const four = numbers + set.block + kv8_value_byte(kHeadDim, set.t & ~3, i0);
  const bool single = set.row >= 0 && __popc(set.written >> (set.t & ~3) & 15u) == 1;
  float v[4 * kFours];
  vec16 beside[kFours];
#pragma unroll
  for (int j = 0; j < kFours; ++j) {
    uint2 w = make_uint2(0u, 0u);
    if (set.row >= 0) w = *reinterpret_cast<const uint2*>(src + 16 * j);
    unpack4(w, v + 4 * j);
    if (single) beside[j] = load16(four + 64 * j);
  }
  float move;
  const float scale = block_scale(set, held, largest_of<4 * kFours>(v), lds_largest, move);
  if (set.row >= 0) {
    if (set.leads() && (lane_id() & 3) == 0) a.view.value_scales[scale_at] = scale;
    const float inverse = 1.0f / scale;
    const int byte = set.t & 3;
#pragma unroll
    for (int j = 0; j < kFours; ++j) {
      const uint32_t w = four_numbers(v + 4 * j, inverse);
      if (single && move == 1.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          beside[j].w[i] = (beside[j].w[i] & ~(0xffu << (8 * byte))) | (w >> (8 * i) & 0xffu) << (8 * byte);
        }
        store16(four + 64 * j, beside[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) four[64 * j + 4 * i + byte] = static_cast<uint8_t>(w >> (8 * i));
      }
    }
  }
  move_blocks<kHeadDim, false>(set, numbers, move);
}

// The first kv_blocks blocks' waves share the windows' kv heads, keys and values,
// `waves` a window (with twice as many as those, each half has every second set); behind
// them come the queries, kHeadDim / 16 lanes a head. The first compute, the others move
// bytes, and so they overlap: 6779 rows of 32 on 8 heads of 64, queries first 23 us, then
// 19; either alone 11 and 13. Heads of 128 take 154 registers, three waves a SIMD: held
// to 128 by loads one behind the other, 200 sequences of up to five rows take 13.0 us for
// 11.6, 500 18.2 for 16.1, prompts of 6779 33.2 for 32.8 without a norm and 34.1 for 35.1
// with one.
template <int kHeadDim>
__global__ __launch_bounds__(kHeadsThreads, 2) void batch_kv8_heads_kernel(Heads8Args a, unsigned kv_blocks, int waves) {
  __shared__ uint32_t lds_words[kHeadsWaves][16];
  if (blockIdx.x >= kv_blocks) {
    const unsigned q_block = blockIdx.x - kv_blocks;
    constexpr int kLanes = kHeadDim / 16;
    constexpr int kHalf = kHeadDim / 2;
    const long long unit = (static_cast<long long>(q_block) * kHeadsThreads + threadIdx.x) / kLanes;
    const int row = static_cast<int>(unit / a.num_heads);
    const int head = static_cast<int>(unit - static_cast<long long>(row) * a.num_heads);
    const int i = 8 * (static_cast<int>(threadIdx.x) % kLanes);
    if (row >= a.tokens) return;  // whole heads leave together
    const int position = a.positions[row];
    if (!row_is_live(a, a.slots[row], position)) return;
    const elem_t* src = a.q + static_cast<size_t>(row) * static_cast<size_t>(a.src_row_stride) +
                        static_cast<size_t>(head) * kHeadDim + i;
    elem_t* dst = a.q_out + (static_cast<size_t>(row) * a.num_heads + head) * kHeadDim + i;
    vec16 lo = load16(src), hi = load16(src + kHalf);
    norm_rotate<kHeadDim>(lo, hi, a.q_norm, a.eps, a.table + static_cast<size_t>(position) * kHalf, i);
    store16(dst, lo);
    store16(dst + kHalf, hi);
    return;
  }
  const int in_block = static_cast<int>(threadIdx.x) >> 6;
  const long long wave = static_cast<long long>(blockIdx.x) * kHeadsWaves + in_block;
  const int window = __builtin_amdgcn_readfirstlane(static_cast<int>(wave / waves));
  const int in_window = __builtin_amdgcn_readfirstlane(static_cast<int>(wave % waves));
  if (window * kWindowRows >= a.tokens) return;
  const Window win(a, window * kWindowRows);
  const int kv = a.view.num_kv_heads;
  const bool halved = waves > 2 * kv;  // then 4 kv
  const int half = halved && in_window >= 2 * kv ? 1 : 0;
  const int share = in_window - half * 2 * kv;
  unsigned long long left = win.leaders;
  for (int at = 0; left != 0; ++at) {
    const RowSet set(a, win, left, lds_words[in_block]);
    if (halved && (at & 1) != half) continue;
    for (int n = share; n < 2 * kv; n += waves) {
      if (n < kv) {
        append_keys<kHeadDim>(a, set, n, lds_words[in_block]);
      } else {
        append_values<kHeadDim>(a, set, n - kv, lds_words[in_block]);
      }
    }
  }
}

template <int kHeadDim>
void launch_heads(const Heads8Args& a, hipStream_t s) {
  const long long q_lanes = static_cast<long long>(a.tokens) * a.num_heads * (kHeadDim / 16);
  const unsigned q_blocks = static_cast<unsigned>((q_lanes + kHeadsThreads - 1) / kHeadsThreads);
  const int windows = (a.tokens + kWindowRows - 1) / kWindowRows;
  const int shares = 2 * a.view.num_kv_heads;
  const int units = device_compute_units();
  const int waves = static_cast<long long>(windows) * shares <= kHalvedWaves * units
                        ? 2 * shares
                        : std::min(shares, (kMostWaves * units + windows - 1) / windows);
  const long long kv_waves = static_cast<long long>(windows) * waves;
  const unsigned kv_blocks = static_cast<unsigned>((kv_waves + kHeadsWaves - 1) / kHeadsWaves);
  batch_kv8_heads_kernel<kHeadDim><<<kv_blocks + q_blocks, kHeadsThreads, 0, s>>>(a, kv_blocks, std::max(waves, 1));
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" int lcr_batch_norm_rope_write_kv8(void* q_out, const lcr_kv8_view* view, const void* q, const void* k,
                                             const void* v, const void* q_norm, const void* k_norm, float eps,
                                             const float* rope_table, int table_positions, const int32_t* positions,
                                             const int32_t* slots, int tokens, int num_heads, int pool_pages,
                                             int src_row_stride, void* stream) {
  CAPI_CHECK(view != nullptr, "batch_norm_rope_write_kv8 needs a cache view");
  CAPI_CHECK(tokens >= 0 && num_heads >= 0 && view->num_kv_heads >= 0,
             "batch_norm_rope_write_kv8 needs non-negative sizes");
  CAPI_CHECK(view->head_dim > 0 && view->head_dim % 16 == 0 && view->head_dim <= kMaxHeadDim,
             "an 8-bit cache has a head_dim that is a multiple of 16 up to " << kMaxHeadDim << ", got "
                                                                             << view->head_dim);
  const long long heads = num_heads + 2ll * view->num_kv_heads;
  if (tokens == 0 || heads == 0) return LCR_OK;
  CAPI_CHECK(view->page_size > 0 && view->page_size % kKv8Block == 0,
             "an 8-bit cache view needs pages of a multiple of " << kKv8Block << " positions, got " << view->page_size);
  CAPI_CHECK(pool_pages >= 0 && table_positions >= 0, "batch_norm_rope_write_kv8 needs a non-negative pool and table");
  CAPI_CHECK(static_cast<long long>(pool_pages) * view->page_size <= INT32_MAX,
             "a pool of " << pool_pages << " pages of " << view->page_size << " positions has slots past 32 bits");
  CAPI_CHECK(view->page_stride >= 0 && view->head_stride >= 0 && view->scale_page_stride >= 0 &&
                 view->scale_head_stride >= 0 && view->page_stride % 16 == 0 && view->head_stride % 16 == 0,
             "an 8-bit cache has non-negative strides, of its numbers in multiples of 16 bytes");
  const long long widest = static_cast<long long>(std::max(num_heads, view->num_kv_heads)) * view->head_dim;
  CAPI_CHECK(src_row_stride >= widest, "rows of " << widest << " elements cannot lie " << src_row_stride << " apart");
  CAPI_CHECK(tokens * heads <= (1ll << 32) / 64 - kHeadsWaves,
             "batch_norm_rope_write_kv8 takes up to 2^26 heads in all, got " << tokens * heads);
  CAPI_CHECK(positions != nullptr && slots != nullptr, "batch_norm_rope_write_kv8 needs positions and slots");
  CAPI_CHECK(num_heads == 0 || (q_out != nullptr && q != nullptr), "batch_norm_rope_write_kv8 needs its queries");
  CAPI_CHECK(view->num_kv_heads == 0 || (k != nullptr && v != nullptr && view->keys != nullptr &&
                                         view->values != nullptr && view->key_scales != nullptr &&
                                         view->value_scales != nullptr),
             "batch_norm_rope_write_kv8 needs its keys and values and a cache with scales to write");
  CAPI_CHECK(((reinterpret_cast<uintptr_t>(view->keys) | reinterpret_cast<uintptr_t>(view->values)) & 15u) == 0,
             "an 8-bit cache's numbers must be 16-byte aligned");
  CAPI_CHECK(rope_table != nullptr && (reinterpret_cast<uintptr_t>(rope_table) & 7u) == 0,
             "batch_norm_rope_write_kv8 needs an 8-byte aligned RoPE table");
  Heads8Args a;
  a.q_out = static_cast<elem_t*>(q_out);
  a.view = Kv8View::from_c(*view);
  a.q = static_cast<const elem_t*>(q);
  a.k = static_cast<const elem_t*>(k);
  a.v = static_cast<const elem_t*>(v);
  a.q_norm = static_cast<const elem_t*>(q_norm);
  a.k_norm = static_cast<const elem_t*>(k_norm);
  a.eps = eps;
  a.table = reinterpret_cast<const float2*>(rope_table);
  a.table_positions = table_positions;
  a.positions = positions;
  a.slots = slots;
  a.tokens = tokens;
  a.num_heads = num_heads;
  a.pool_slots = pool_pages * view->page_size;
  a.src_row_stride = src_row_stride;
  auto s = static_cast<hipStream_t>(stream);
  const bool aligned = on_bytes(q_out, 16) && on_bytes(q, 16) && on_bytes(k, 16) && on_bytes(v, 16) &&
                       on_bytes(q_norm, 16) && on_bytes(k_norm, 16) && on_bytes(rope_table, 16) && src_row_stride % 8 == 0;
  if (aligned && view->head_dim == 64) {
    launch_heads<64>(a, s);
  } else if (aligned && view->head_dim == 128) {
    launch_heads<128>(a, s);
  } else {
    const unsigned blocks = static_cast<unsigned>((tokens * heads + kHeadsWaves - 1) / kHeadsWaves);
    batch_kv8_heads_any_kernel<<<blocks, kHeadsThreads, 0, s>>>(a);
  }
  CAPI_LAUNCHED();
  return LCR_OK;
}
