// What the paged-cache kernels share (paged.hip, paged_attention.hip): the
// argument block made from a checked hk_paged_cache, and the launches.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>

#include "hk_internal.h"
#include "hk_paged.h"
#include "paged_plan.h"

namespace hk {

// The workspace's first words: tickets of the attention, zero between calls.
constexpr int kPagedTicketWords = 4096;

// One layer's pools where the call is for one layer.
struct PagedPool {
  char* k;
  char* v;
  const float* k_scale;  // [kv_heads], e4m3 only
  const float* v_scale;
  const int32_t* table;
  const int32_t* length;
  int64_t page_bytes;    // from page to page
  int kv_heads, page_shift, pages, seqs, width, elt;  // elt: bytes of an element
};

struct PagedBatch {
  const int32_t* seqs;
  const int32_t* first;
  int n, tokens;
};

struct PagedAttnArgs {
  PagedPool c;
  PagedBatch b;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int64_t q_stride, out_stride;
  int q_heads, group, window, max_new;
  PlanDivisor by_group;    // set by the launch
  int rows_min, rows_max;  // set by the launch: rows (tokens x group) of the entries it takes
  int ticket0, part0;      // set by the launch: its first ticket, and byte of partial results
  float scale;
  void* workspace;
};
int launch_paged_attention(const PagedAttnArgs& a, int head_dim, hipStream_t stream);

#ifdef __HIPCC__
// A launch, and its own error: hipGetLastError would also give one that an
// earlier HIP call of the caller's has left, and a fork that stopped for that
// between its two launches would leave pages that nobody has copied.
template <typename... P, typename... A>
int paged_launch(const char* what, void (*kernel)(P...), int groups, int threads, hipStream_t stream, const A&... args) {
  std::tuple<P...> given(args...);
  const hipError_t err = std::apply(
      [&](auto&... a) {
        void* at[] = {&a...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(groups), dim3(threads), at, 0, stream);
      },
      given);
  return err == hipSuccess ? 0 : hip_fail(err, what);
}

// Rows of entry b, within the batch's rows whatever `first` holds.
__device__ __forceinline__ int2 entry_rows(const PagedBatch& b, int entry) {
  const int f0 = min(max(b.first[entry], 0), b.tokens);
  return make_int2(f0, min(max(b.first[entry + 1], f0), b.tokens));
}

// The entry's sequence (-1: outside the cache) and its length.
__device__ __forceinline__ int2 entry_seq(const PagedPool& c, const PagedBatch& b, int entry) {
  const int s = b.seqs ? b.seqs[entry] : entry;
  if ((unsigned)s >= (unsigned)c.seqs) return make_int2(-1, 0);
  return make_int2(s, min(max(c.length[s], 0), c.width << c.page_shift));
}
#endif

}  // namespace hk
