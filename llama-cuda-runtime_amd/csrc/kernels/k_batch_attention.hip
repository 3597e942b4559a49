// lcr_batch_attention: causal GQA attention of many sequences' rows over one
// paged cache.
#include <algorithm>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "../kv_cache.h"
#include "device_common.h"

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
  float scale;
};

// ---------------------------------------------------------------------------
// Any head_dim up to 256, any alignment: a wave per (row, query head).
// ---------------------------------------------------------------------------

constexpr int kGenericWaves = 4;
constexpr int kGenericThreads = 64 * kGenericWaves;
constexpr int kGenericMaxDim = 256;

// Lane L of a 64-key tile takes key L's whole dot product; the tile's weights
// go through LDS, and lane L then holds elements L, L + 64, ... of the output.
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
  const int head_dim = a.view.head_dim;
  const int kv = head / a.group;
  const long long position = static_cast<long long>(a.lengths[b]) - (a.row_starts[b + 1] - row);
  const long long held = static_cast<long long>(a.table_stride) * a.view.page_size;
  const int limit = in_sequence < a.max_new ? static_cast<int>(max(0ll, min(position + 1, held))) : 0;
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
    weights[wave][lane] = elem_to_float(float_to_elem(p));
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

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" size_t lcr_batch_attention_workspace_bytes(int batch, int tokens, int max_new, int num_heads,
                                                      int heads_per_kv, int head_dim) {
  if (batch <= 0 || tokens <= 0 || max_new <= 0 || num_heads <= 0 || heads_per_kv <= 0 || head_dim <= 0) return 0;
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
  CAPI_CHECK(view->page_stride >= 0 && view->head_stride >= 0, "batch attention needs non-negative cache strides");
  CAPI_CHECK(q_row_stride >= static_cast<long long>(num_heads) * view->head_dim,
             "query rows of " << num_heads << " heads cannot lie " << q_row_stride << " elements apart");
  CAPI_CHECK(static_cast<long long>(tokens) * num_heads <= INT32_MAX,
             "batch attention takes up to 2^31 - 1 query heads in all");
  CAPI_CHECK(out != nullptr && q != nullptr && view->keys != nullptr && view->values != nullptr &&
                 row_starts != nullptr && lengths != nullptr,
             "batch attention needs its arrays");
  CAPI_CHECK(workspace != nullptr || workspace_bytes == 0,
             "batch attention workspace of " << workspace_bytes << " bytes has no pointer");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch attention workspace must be 16-byte aligned");
  BatchAttnArgs a{static_cast<elem_t*>(out), static_cast<const elem_t*>(q), KvCacheView::from_c(*view), row_starts,
                  lengths, batch, tokens, max_new, num_heads, heads_per_kv, table_stride, pool_pages, q_row_stride, scale};
  auto s = static_cast<hipStream_t>(stream);
  const long long units = static_cast<long long>(tokens) * num_heads;
  batch_attention_generic_kernel<<<static_cast<unsigned>((units + kGenericWaves - 1) / kGenericWaves), kGenericThreads,
                                   0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
