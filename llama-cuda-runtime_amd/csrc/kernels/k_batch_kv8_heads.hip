// lcr_batch_norm_rope_write_kv8: per-head RMSNorm and rotation of a step's rows,
// queries to a buffer, keys and values appended to a cache of 8-bit numbers.
//
// A block of 16 positions of a head shares a scale, so the rows of a call that lie
// in one block are a wave's work together: the largest of their values decides
// whether the scale holds, and where it does not, the numbers held are rounded to
// the new one. The wave of the first of those rows does it; rows that are not the
// first of their block have none. A row knows by the 15 rows before it, and its
// block's others are among the 15 behind it.
#include <algorithm>
#include <cstdint>

#include "../capi_util.h"
#include "kv8.h"

namespace lcr {
namespace {

constexpr int kHeadsThreads = 256;
constexpr int kHeadsWaves = kHeadsThreads / 64;
constexpr int kMaxHeadDim = 256;

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
  const unsigned blocks = static_cast<unsigned>((tokens * heads + kHeadsWaves - 1) / kHeadsWaves);
  batch_kv8_heads_any_kernel<<<blocks, kHeadsThreads, 0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
