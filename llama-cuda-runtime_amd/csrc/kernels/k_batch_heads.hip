// lcr_batch_norm_rope_write_kv: per-head RMSNorm, rotation and the cache write
// of a step's rows in one pass over the q/k/v projection.
//
// A head is normed over its own head_dim elements and rotated in pairs
// (i, i + head_dim/2). head_dim / 16 lanes take a head, lane i the elements
// 8i .. 8i + 7 of both halves: a pair never leaves its lane, the mean square
// needs two to four lane exchanges, and every access is 16 bytes. Everything
// between the load and the store is fp32, with one rounding to the element
// type. The projection is read once and written once: bound by memory. 6779 rows
// of 32 + 8 + 8 heads of 64 (85 MB read and written) take 18.2 us, 4.7 TB/s, of a
// copy's 5.2; 8 rows 3.3 us, one chain of four reads.
#include <algorithm>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "../kv_cache.h"
#include "head_rotation.h"

namespace lcr {
namespace {

constexpr int kHeadsThreads = 256;
constexpr int kMaxHeadDimPairs = 256;  // head_dim up to 512

struct HeadsArgs {
  elem_t* q_out;
  KvCacheView view;
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

// Where head `slot of the row` comes from, goes to, and what it is normed with
// (nullptr: not normed). The heads of a row are its queries, keys and values.
struct HeadPlace {
  const elem_t* src;
  elem_t* dst;
  const elem_t* weight;
  bool rotate;
};

__device__ __forceinline__ HeadPlace place_head(const HeadsArgs& a, int row, int head, int cache_slot, int head_dim) {
  const size_t src_row = static_cast<size_t>(row) * static_cast<size_t>(a.src_row_stride);
  if (head < a.num_heads) {
    return HeadPlace{a.q + src_row + static_cast<size_t>(head) * head_dim,
                     a.q_out + (static_cast<size_t>(row) * a.num_heads + head) * head_dim, a.q_norm, true};
  }
  const int kv = a.view.num_kv_heads;
  const bool is_key = head < a.num_heads + kv;
  const int h = head - a.num_heads - (is_key ? 0 : kv);
  const int page = cache_slot / a.view.page_size;
  const int in_page = cache_slot - page * a.view.page_size;
  const size_t at = static_cast<size_t>(page) * static_cast<size_t>(a.view.page_stride) +
                    static_cast<size_t>(h) * static_cast<size_t>(a.view.head_stride) +
                    static_cast<size_t>(in_page) * static_cast<size_t>(head_dim);
  return HeadPlace{(is_key ? a.k : a.v) + src_row + static_cast<size_t>(h) * head_dim,
                   (is_key ? a.view.keys : a.view.values) + at, is_key ? a.k_norm : nullptr, is_key};
}

template <int kHeadDim>
__global__ __launch_bounds__(kHeadsThreads) void batch_heads_kernel(HeadsArgs a) {
  constexpr int kLanes = kHeadDim / 16;
  constexpr int kHalf = kHeadDim / 2;
  const int heads = a.num_heads + 2 * a.view.num_kv_heads;
  const long long unit = (static_cast<long long>(blockIdx.x) * kHeadsThreads + threadIdx.x) / kLanes;
  const int row = static_cast<int>(unit / heads);
  const int head = static_cast<int>(unit - static_cast<long long>(row) * heads);
  const int i = 8 * (static_cast<int>(threadIdx.x) % kLanes);
  if (row >= a.tokens) return;  // whole heads leave together
  const int cache_slot = a.slots[row];
  const int position = a.positions[row];
  if (cache_slot < 0 || cache_slot >= a.pool_slots || position < 0 || position >= a.table_positions) return;
  const HeadPlace h = place_head(a, row, head, cache_slot, kHeadDim);
  vec16 lo = load16(h.src + i), hi = load16(h.src + kHalf + i);
  if (h.rotate) {
    norm_rotate<kHeadDim>(lo, hi, h.weight, a.eps, a.table + static_cast<size_t>(position) * kHalf, i);
  }
  store16(h.dst + i, lo);
  store16(h.dst + kHalf + i, hi);
}

// Any even head_dim up to 512 and any alignment: a wave per head, four pairs a
// lane.
__global__ __launch_bounds__(kHeadsThreads) void batch_heads_generic_kernel(HeadsArgs a) {
  constexpr int kPairs = kMaxHeadDimPairs / 64;
  const int heads = a.num_heads + 2 * a.view.num_kv_heads;
  const long long unit = static_cast<long long>(blockIdx.x) * (kHeadsThreads / 64) + (threadIdx.x >> 6);
  const int row = static_cast<int>(unit / heads);
  const int head = static_cast<int>(unit - static_cast<long long>(row) * heads);
  if (row >= a.tokens) return;
  const int cache_slot = a.slots[row];
  const int position = a.positions[row];
  if (cache_slot < 0 || cache_slot >= a.pool_slots || position < 0 || position >= a.table_positions) return;
  const int head_dim = a.view.head_dim;
  const int half = head_dim / 2;
  const HeadPlace h = place_head(a, row, head, cache_slot, head_dim);
  elem_t lo[kPairs], hi[kPairs];
  float square = 0.0f;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const int i = lane_id() + 64 * j;
    lo[j] = hi[j] = elem_t{0};
    if (i < half) {
      lo[j] = h.src[i];
      hi[j] = h.src[half + i];
      const float x = elem_to_float(lo[j]), y = elem_to_float(hi[j]);
      square = __builtin_fmaf(x, x, __builtin_fmaf(y, y, square));
    }
  }
  const float scale = 1.0f / sqrtf(wave_sum(square) / static_cast<float>(head_dim) + a.eps);
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const int i = lane_id() + 64 * j;
    if (i >= half) continue;
    if (h.rotate) {
      float x = elem_to_float(lo[j]), y = elem_to_float(hi[j]);
      if (h.weight != nullptr) {
        x = x * scale * elem_to_float(h.weight[i]);
        y = y * scale * elem_to_float(h.weight[half + i]);
      }
      const float2 r = rope_rotate(x, y, a.table[static_cast<size_t>(position) * half + i]);
      lo[j] = float_to_elem(r.x);
      hi[j] = float_to_elem(r.y);
    }
    h.dst[i] = lo[j];
    h.dst[half + i] = hi[j];
  }
}

// Lanes that a head takes.
int head_lanes(const HeadsArgs& a, bool aligned) {
  const int d = a.view.head_dim;
  return aligned && (d == 64 || d == 128 || d == 256) ? d / 16 : 64;
}

template <int kHeadDim>
void launch_heads(const HeadsArgs& a, hipStream_t s) {
  const long long lanes = static_cast<long long>(a.tokens) * (a.num_heads + 2 * a.view.num_kv_heads) * (kHeadDim / 16);
  const unsigned blocks = static_cast<unsigned>((lanes + kHeadsThreads - 1) / kHeadsThreads);
  batch_heads_kernel<kHeadDim><<<blocks, kHeadsThreads, 0, s>>>(a);
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" int lcr_batch_norm_rope_write_kv(void* q_out, const lcr_kv_view* view, const void* q, const void* k,
                                            const void* v, const void* q_norm, const void* k_norm, float eps,
                                            const float* rope_table, int table_positions, const int32_t* positions,
                                            const int32_t* slots, int tokens, int num_heads, int pool_pages,
                                            int src_row_stride, void* stream) {
  CAPI_CHECK(view != nullptr, "batch_norm_rope_write_kv needs a cache view");
  CAPI_CHECK(tokens >= 0 && num_heads >= 0 && view->num_kv_heads >= 0,
             "batch_norm_rope_write_kv needs non-negative sizes");
  CAPI_CHECK(view->head_dim > 0 && view->head_dim % 2 == 0,
             "head_dim must be positive and even for RoPE, got " << view->head_dim);
  CAPI_CHECK(view->head_dim / 2 <= kMaxHeadDimPairs,
             "batch_norm_rope_write_kv supports head_dim up to " << 2 * kMaxHeadDimPairs);
  const long long heads = num_heads + 2ll * view->num_kv_heads;
  if (tokens == 0 || heads == 0) return LCR_OK;
  CAPI_CHECK(view->page_size > 0, "a paged cache view needs a positive page size");
  CAPI_CHECK(pool_pages >= 0 && table_positions >= 0, "batch_norm_rope_write_kv needs a non-negative pool and table");
  CAPI_CHECK(static_cast<long long>(pool_pages) * view->page_size <= INT32_MAX,
             "a pool of " << pool_pages << " pages of " << view->page_size << " positions has slots past 32 bits");
  CAPI_CHECK(view->page_stride >= 0 && view->head_stride >= 0, "batch_norm_rope_write_kv needs non-negative cache strides");
  const long long widest = static_cast<long long>(std::max(num_heads, view->num_kv_heads)) * view->head_dim;
  CAPI_CHECK(src_row_stride >= widest, "rows of " << widest << " elements cannot lie " << src_row_stride << " apart");
  CAPI_CHECK(tokens * heads <= (1ll << 32), "batch_norm_rope_write_kv takes up to 2^32 heads in all, got "
                                                << tokens * heads);
  CAPI_CHECK(positions != nullptr && slots != nullptr, "batch_norm_rope_write_kv needs positions and slots");
  CAPI_CHECK(num_heads == 0 || (q_out != nullptr && q != nullptr), "batch_norm_rope_write_kv needs its queries");
  CAPI_CHECK(view->num_kv_heads == 0 || (k != nullptr && v != nullptr && view->keys != nullptr && view->values != nullptr),
             "batch_norm_rope_write_kv needs its keys and values and a cache to write");
  CAPI_CHECK(rope_table != nullptr && (reinterpret_cast<uintptr_t>(rope_table) & 7u) == 0,
             "batch_norm_rope_write_kv needs an 8-byte aligned RoPE table");
  HeadsArgs a;
  a.q_out = static_cast<elem_t*>(q_out);
  a.view = KvCacheView::from_c(*view);
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
                       on_bytes(q_norm, 16) && on_bytes(k_norm, 16) && on_bytes(rope_table, 16) &&
                       on_bytes(view->keys, 16) && on_bytes(view->values, 16) && src_row_stride % 8 == 0 &&
                       view->page_stride % 8 == 0 && view->head_stride % 8 == 0;
  // A launch has fewer than 2^32 threads in all.
  CAPI_CHECK(tokens * heads * head_lanes(a, aligned) <= UINT32_MAX - kHeadsThreads,
             "batch_norm_rope_write_kv of " << tokens * heads << " heads needs more than 2^32 threads");
  if (aligned && view->head_dim == 64) {
    launch_heads<64>(a, s);
  } else if (aligned && view->head_dim == 128) {
    launch_heads<128>(a, s);
  } else if (aligned && view->head_dim == 256) {
    launch_heads<256>(a, s);
  } else {
    const unsigned blocks = static_cast<unsigned>((tokens * heads + 3) / 4);
    batch_heads_generic_kernel<<<blocks, kHeadsThreads, 0, s>>>(a);
  }
  CAPI_LAUNCHED();
  return LCR_OK;
}
