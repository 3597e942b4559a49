// lcr_batch_map: page tables, row starts, positions and slots of a step, from
// the sequences' lengths.
//
// With need(b) = max(0, ceil((length + new) / page_size) - mapped), the rows
// and new pages of sequence b start at the sums of new and need over the
// sequences before it. Every block takes these two prefix sums over the whole
// batch itself (at most 4096 sequences, 48 KiB read) and keeps them in LDS,
// rather than waiting for another block or kernel to have done so; then the
// blocks share the rows, the new pages and the sequences, each finding its
// sequence by bisection. The work is a chain of dependent reads (lengths, scan,
// bisection, table entry), so it is bound by their latency and not by bytes: 3.6
// us for 8 sequences of one token, 5.2 for 256 with 4021 rows, 7.9 for 1024 with
// 46309 (0.4 MB, which a copy moves in 0.1).
#include <algorithm>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "device_common.h"

namespace lcr {
namespace {

constexpr int kMapThreads = 256;
constexpr int kMapWaves = kMapThreads / 64;

struct MapArgs {
  int32_t* row_starts;
  int32_t* positions;
  int32_t* slots;
  int32_t* lengths_out;
  int32_t* mapped_out;
  int32_t* counts;
  int32_t* page_tables;
  const int32_t* lengths;
  const int32_t* new_tokens;
  const int32_t* mapped;
  const int32_t* free_pages;
  const int32_t* free_count;
  int batch;
  int max_rows;
  int table_stride;
  int page_size;
  int pool_pages;
  int free_capacity;
};

// Inclusive sums over the wave of two counters.
__device__ __forceinline__ void wave_inclusive_scan2(long long& a, long long& b) {
  const int lane = lane_id();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long x = __shfl_up(a, o, 64);
    const long long y = __shfl_up(b, o, 64);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
}

// The last index in [0, count) whose start is <= value (starts ascending,
// starts[0] = 0 <= value): behind empty sequences the one that holds the row.
__device__ __forceinline__ int bisect(const int* starts, int count, int value) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= value) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

__global__ __launch_bounds__(kMapThreads) void batch_map_kernel(MapArgs a) {
  __shared__ int row_start[LCR_BATCH_MAX_SEQUENCES + 1];
  __shared__ int page_start[LCR_BATCH_MAX_SEQUENCES + 1];
  __shared__ long long wave_rows[kMapWaves], wave_pages[kMapWaves];
  __shared__ int wave_fail[kMapWaves];
  const int t = threadIdx.x;
  const int lane = lane_id();
  const int wave = t >> 6;
  const int per = (a.batch + kMapThreads - 1) / kMapThreads;
  const int first = t * per;
  const int free = min(max(a.free_count[0], 0), a.free_capacity);
  const long long capacity = static_cast<long long>(a.table_stride) * a.page_size;
  if (t == 0 && a.batch == 0) row_start[0] = page_start[0] = 0;  // read behind the barriers

  // Sums over this thread's sequences. They are kept in 64 bits: before the
  // first sequence that fails they fit 32, behind it they only have to stay
  // large.
  long long rows = 0, pages = 0;
  for (int k = 0; k < per; ++k) {
    const int b = first + k;
    if (b >= a.batch) break;
    const int n = a.new_tokens[b];
    const long long total = static_cast<long long>(a.lengths[b]) + n;
    rows += max(n, 0);
    pages += max((total + a.page_size - 1) / a.page_size - a.mapped[b], 0ll);
  }
  long long rows_to = rows, pages_to = pages;
  wave_inclusive_scan2(rows_to, pages_to);
  if (lane == 63) {
    wave_rows[wave] = rows_to;
    wave_pages[wave] = pages_to;
  }
  __syncthreads();
  rows_to -= rows;
  pages_to -= pages;
  for (int w = 0; w < wave; ++w) {
    rows_to += wave_rows[w];
    pages_to += wave_pages[w];
  }
  // The first sequence that cannot be placed; starts up to it.
  int fail = a.batch;
  for (int k = 0; k < per; ++k) {
    const int b = first + k;
    if (b >= a.batch) break;
    const int n = a.new_tokens[b];
    const int length = a.lengths[b];
    const int mapped = a.mapped[b];
    const long long total = static_cast<long long>(length) + n;
    row_start[b] = static_cast<int>(min(rows_to, static_cast<long long>(a.max_rows)));
    page_start[b] = static_cast<int>(min(pages_to, static_cast<long long>(free)));
    rows_to += max(n, 0);
    pages_to += max((total + a.page_size - 1) / a.page_size - mapped, 0ll);
    if (fail == a.batch && (n < 0 || length < 0 || mapped < 0 || total > capacity || rows_to > a.max_rows ||
                            pages_to > free)) {
      fail = b;
    }
    if (b == a.batch - 1) {
      row_start[a.batch] = static_cast<int>(min(rows_to, static_cast<long long>(a.max_rows)));
      page_start[a.batch] = static_cast<int>(min(pages_to, static_cast<long long>(free)));
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) fail = min(fail, __shfl_xor(fail, o, 64));
  if (lane == 0) wave_fail[wave] = fail;
  __syncthreads();
  int placed = wave_fail[0];
#pragma unroll
  for (int w = 1; w < kMapWaves; ++w) placed = min(placed, wave_fail[w]);
  const int all_rows = row_start[placed];
  const int all_pages = page_start[placed];

  const int step = static_cast<int>(gridDim.x) * kMapThreads;
  const int me = static_cast<int>(blockIdx.x) * kMapThreads + t;
  if (me == 0) {
    a.counts[0] = placed;
    a.counts[1] = free - all_pages;
  }
  for (int b = me; b <= a.batch; b += step) {
    a.row_starts[b] = b < placed ? row_start[b] : all_rows;
    if (b < a.batch) {
      const int n = b < placed ? a.new_tokens[b] : 0;
      const int taken = b < placed ? page_start[b + 1] - page_start[b] : 0;
      a.lengths_out[b] = a.lengths[b] + n;
      a.mapped_out[b] = a.mapped[b] + taken;
    }
  }
  // New page j is free_pages[free - 1 - j].
  for (long long i = me; i < all_pages; i += step) {
    const int j = static_cast<int>(i);
    const int b = bisect(page_start, placed, j);
    const int column = a.mapped[b] + j - page_start[b];
    a.page_tables[static_cast<size_t>(b) * a.table_stride + column] = a.free_pages[free - 1 - j];
  }
  for (long long r = me; r < a.max_rows; r += step) {
    const int row = static_cast<int>(r);
    int position = -1, slot = -1;
    if (row < all_rows) {
      const int b = bisect(row_start, placed, row);
      position = a.lengths[b] + row - row_start[b];
      const int column = position / a.page_size;
      const int mapped = a.mapped[b];
      // A page that this call maps is read from the free list, not from the
      // table that another block may not have written yet.
      const int page = column < mapped ? a.page_tables[static_cast<size_t>(b) * a.table_stride + column]
                                       : a.free_pages[free - 1 - (page_start[b] + column - mapped)];
      if (page >= 0 && page < a.pool_pages) slot = page * a.page_size + position % a.page_size;
    }
    a.positions[row] = position;
    a.slots[row] = slot;
  }
}

int launch_map(const MapArgs& a, void* stream) {
  // One row or sequence a thread up to 512 blocks.
  const int items = std::max(a.max_rows, a.batch + 1);
  const int blocks = std::min(512, (items - 1) / kMapThreads + 1);
  batch_map_kernel<<<blocks, kMapThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}

// Whether this process's HIP runtime knows the address.
bool known_address(const void* p) {
  hipPointerAttribute_t attributes{};
  const bool known = hipPointerGetAttributes(&attributes, p) == hipSuccess &&
                     attributes.type != hipMemoryTypeUnregistered;
  (void)hipGetLastError();  // an address that is not known leaves an error
  return known;
}

// A step of no sequences is a step: no rows, and the free count handed on. Its
// sequences' arrays are not read and may be NULL. Where only some of them are,
// the call may have been made of stand-ins for arrays, which are not followed.
int map_nothing(MapArgs a, void* stream) {
  const bool rows = a.max_rows == 0 || (a.positions != nullptr && a.slots != nullptr);
  if (a.row_starts == nullptr || a.counts == nullptr || a.free_count == nullptr || !rows) return LCR_OK;
  const int given = (a.lengths != nullptr) + (a.new_tokens != nullptr) + (a.mapped != nullptr);
  if (given != 0 && given != 3 && !known_address(a.counts)) return LCR_OK;
  a.free_capacity = std::max(a.free_capacity, 0);
  return launch_map(a, stream);
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" int lcr_batch_map(int32_t* row_starts, int32_t* positions, int32_t* slots, int32_t* lengths_out,
                             int32_t* mapped_out, int32_t* counts, int32_t* page_tables, const int32_t* lengths,
                             const int32_t* new_tokens, const int32_t* mapped, const int32_t* free_pages,
                             const int32_t* free_count, int batch, int max_rows, int table_stride, int page_size,
                             int pool_pages, int free_capacity, void* stream) {
  CAPI_CHECK(batch >= 0 && max_rows >= 0, "batch_map needs non-negative sizes");
  CAPI_CHECK(batch <= LCR_BATCH_MAX_SEQUENCES,
             "batch_map takes up to " << LCR_BATCH_MAX_SEQUENCES << " sequences, got " << batch);
  MapArgs a{row_starts, positions, slots,     lengths_out, mapped_out, counts,   page_tables, lengths,    new_tokens,
            mapped,     free_pages, free_count, batch,      max_rows,   table_stride, page_size, pool_pages, free_capacity};
  if (batch == 0) return map_nothing(a, stream);
  CAPI_CHECK(page_size > 0, "batch_map needs a positive page size, got " << page_size);
  CAPI_CHECK(table_stride > 0, "batch_map needs page tables of at least one page, got " << table_stride);
  CAPI_CHECK(pool_pages >= 0 && free_capacity >= 0, "batch_map needs non-negative page counts");
  CAPI_CHECK(static_cast<long long>(pool_pages) * page_size <= INT32_MAX,
             "a pool of " << pool_pages << " pages of " << page_size << " positions has slots past 32 bits");
  CAPI_CHECK(static_cast<long long>(table_stride) * page_size <= INT32_MAX,
             "tables of " << table_stride << " pages of " << page_size << " hold positions past 32 bits");
  CAPI_CHECK(row_starts != nullptr && lengths_out != nullptr && mapped_out != nullptr && counts != nullptr &&
                 page_tables != nullptr && lengths != nullptr && new_tokens != nullptr && mapped != nullptr &&
                 free_count != nullptr,
             "batch_map needs its arrays");
  CAPI_CHECK(max_rows == 0 || (positions != nullptr && slots != nullptr), "batch_map needs positions and slots");
  CAPI_CHECK(free_capacity == 0 || free_pages != nullptr, "a free list of " << free_capacity << " pages has no pointer");
  // Every block reads the inputs, so none may be written over by another.
  CAPI_CHECK(lengths_out != lengths && lengths_out != new_tokens && mapped_out != mapped && counts != free_count &&
                 counts + 1 != free_count,
             "batch_map writes its outputs beside its inputs, not over them");
  return launch_map(a, stream);
}
