// lcr_batch_logprobs: log probabilities of given tokens, with their rows'
// entropies and likeliest ids.
#include <algorithm>
#include <climits>
#include <cstdint>

#include "../../../include/lcr_batch.h"
#include "../capi_util.h"
#include "device_common.h"

namespace lcr {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

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
};

// A logit's order: by value, equal ones by ascending id.
__device__ __forceinline__ bool before(float a, int i, float b, int j) { return a > b || (a == b && i < j); }
__device__ __forceinline__ float clean(float l) { return l == l ? l : -__builtin_huge_valf(); }

__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobArgs a) {
  __shared__ float lds_value[kWaves];
  __shared__ int lds_id[kWaves];
  __shared__ double lds_sum[kWaves][3];
  const int row = blockIdx.x;
  const int token = a.token_ids != nullptr ? a.token_ids[row] : -1;
  if (a.token_ids != nullptr && token < 0) return;
  const float* logits = a.logits + static_cast<size_t>(row) * a.logits_stride;
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  // the first logit behind (value, id)
  auto next = [&](float value, int id) {
    float best = -__builtin_huge_valf();
    int at = INT_MAX;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const float l = clean(logits[i]);
      if (before(value, id, l, i) && before(l, i, best, at)) {
        best = l;
        at = i;
      }
    }
    for (int o = 1; o < 64; o <<= 1) {
      const float other = __shfl_xor(best, o, 64);
      const int j = __shfl_xor(at, o, 64);
      if (before(other, j, best, at)) {
        best = other;
        at = j;
      }
    }
    __syncthreads();
    if (lane_id() == 0) {
      lds_value[wave] = best;
      lds_id[wave] = at;
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
      if (before(lds_value[w], lds_id[w], best, at)) {
        best = lds_value[w];
        at = lds_id[w];
      }
    }
    return make_int2(__float_as_int(best), at);
  };
  const int2 first = next(__builtin_huge_valf(), -1);
  const float max = __int_as_float(first.x);
  const bool hot = !(fabsf(max) < __builtin_huge_valf());  // p is 1 at first.y
  const bool inside = token >= 0 && token < a.vocab;
  const float given = inside ? clean(logits[token]) : -__builtin_huge_valf();
  double sum = 0.0, weighted = 0.0, above = 0.0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float l = clean(logits[i]);
    if (l > given) above += 1.0;
    if (hot || l == -__builtin_huge_valf()) continue;
    const double z = static_cast<double>(l) - max;
    const double w = exp(z);
    sum += w;
    weighted += w * z;
  }
  for (int o = 1; o < 64; o <<= 1) {
    sum += __shfl_xor(sum, o, 64);
    weighted += __shfl_xor(weighted, o, 64);
    above += __shfl_xor(above, o, 64);
  }
  if (lane_id() == 0) {
    lds_sum[wave][0] = sum;
    lds_sum[wave][1] = weighted;
    lds_sum[wave][2] = above;
  }
  __syncthreads();
  sum = weighted = above = 0.0;
  for (int w = 0; w < kWaves; ++w) {
    sum += lds_sum[w][0];
    weighted += lds_sum[w][1];
    above += lds_sum[w][2];
  }
  const double log_sum = hot ? 0.0 : log(sum);
  auto logprob = [&](float l, int id) {
    if (hot) return id == first.y ? 0.0f : -__builtin_huge_valf();
    return static_cast<float>(static_cast<double>(l) - max - log_sum);
  };
  if (threadIdx.x == 0) {
    if (a.token_ids != nullptr && a.logprobs != nullptr) {
      a.logprobs[row] = inside ? logprob(given, token) : -__builtin_huge_valf();
    }
    if (a.token_ids != nullptr && a.ranks != nullptr) a.ranks[row] = inside ? static_cast<int>(above) : a.vocab;
    if (a.entropies != nullptr) a.entropies[row] = hot ? 0.0f : static_cast<float>(log_sum - weighted / sum);
  }
  int2 at = first;
  for (int k = 0; k < a.top; ++k) {
    const bool there = k < a.vocab;
    if (threadIdx.x == 0) {
      a.top_ids[static_cast<size_t>(row) * a.top + k] = there ? at.y : -1;
      a.top_logprobs[static_cast<size_t>(row) * a.top + k] =
          there ? logprob(__int_as_float(at.x), at.y) : -__builtin_huge_valf();
    }
    if (there) at = next(__int_as_float(at.x), at.y);
  }
}

}  // namespace
}  // namespace lcr

using namespace lcr;

extern "C" size_t lcr_batch_logprobs_workspace_bytes(int rows, int top, int vocab) { return 0; }

extern "C" int lcr_batch_logprobs(float* logprobs, int32_t* ranks, float* entropies, int32_t* top_ids,
                                  float* top_logprobs, const float* logits, const int32_t* token_ids, int rows, int top,
                                  int vocab, int logits_stride, void* workspace, size_t workspace_bytes, void* stream) {
  CAPI_CHECK(rows >= 0 && top >= 0, "batch_logprobs needs non-negative sizes");
  CAPI_CHECK(top <= LCR_BATCH_MAX_ALTERNATIVES,
             "batch_logprobs takes up to " << LCR_BATCH_MAX_ALTERNATIVES << " alternatives, got " << top);
  if (rows == 0) return LCR_OK;
  CAPI_CHECK(vocab > 0, "batch_logprobs needs a vocabulary, got " << vocab);
  CAPI_CHECK(logits_stride >= vocab, "rows of " << vocab << " logits cannot lie " << logits_stride << " apart");
  CAPI_CHECK(logits != nullptr, "batch_logprobs needs logits");
  CAPI_CHECK(top == 0 || (top_ids != nullptr && top_logprobs != nullptr),
             "batch_logprobs needs room for its alternatives");
  CAPI_CHECK(token_ids != nullptr || (logprobs == nullptr && ranks == nullptr),
             "batch_logprobs needs the tokens whose probabilities it writes");
  CAPI_CHECK(workspace != nullptr || workspace_bytes == 0,
             "batch_logprobs workspace of " << workspace_bytes << " bytes has no pointer");
  CAPI_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "batch_logprobs workspace must be 16-byte aligned");
  CAPI_CHECK(static_cast<long long>(rows) * kThreads <= UINT32_MAX,
             "batch_logprobs of " << rows << " rows needs more than 2^32 threads");
  const LogprobArgs a{logprobs, ranks, entropies, top_ids, top_logprobs, logits, token_ids, top, vocab, logits_stride};
  auto s = static_cast<hipStream_t>(stream);
  logprobs_kernel<<<static_cast<unsigned>(rows), kThreads, 0, s>>>(a);
  CAPI_LAUNCHED();
  return LCR_OK;
}
