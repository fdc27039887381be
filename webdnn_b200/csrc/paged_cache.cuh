// What the kernels over a paged 8-bit cache share: the checks of a pool's and a batch's description, and how a sequence's length,
// count and pages are read on the device.
#pragma once

#include "tape.cuh"

// New tokens of one sequence, or nothing (count 0) where the numbers do not fit the call.
struct CacheSpan {
  int length, count;
};
__device__ __forceinline__ CacheSpan cache_span(const int32_t* lengths, const int32_t* counts, int b, int tokens,
                                                int64_t capacity, int* status) {
  CacheSpan s;
  s.length = pdl_ld(lengths + b);
  s.count = counts ? pdl_ld(counts + b) : tokens;
  if (s.length < 0 || s.length > capacity || s.count < 0 || s.count > tokens || s.count > s.length) {
    status[WDC_STATUS_CACHE] = 1;
    s.length = s.count = 0;
  }
  return s;
}
// A page of the table, or -1.
__device__ __forceinline__ int cache_page(const int32_t* row, int64_t i, int64_t pages, int* status) {
  const int page = pdl_ld(row + i);
  if (page >= 0 && page < pages) return page;
  status[WDC_STATUS_CACHE] = 1;
  return -1;
}

static inline bool cache_aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The pool part of a description.  Pages are counted in 31 bits (a table's entry); everything behind is 64-bit.
static inline int cache_check_pool(wdc_context* ctx, const char* who, int64_t pages, int64_t kv_heads, int64_t page_tokens,
                                   int64_t head_size) {
  WDC_REQUIRE(ctx, pages > 0 && pages < (1ll << 31) && kv_heads > 0 && kv_heads <= 65535, "%s: bad pool", who);
  if ((page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128) ||
      (head_size != 32 && head_size != 64 && head_size != 128))
    return wdc_fail(ctx, WDC_ERR_UNSUPPORTED, "%s: pages of %lld tokens with heads of %lld (supported: 16, 32, 64, 128 tokens; "
                    "heads of 32, 64, 128)", who, (long long)page_tokens, (long long)head_size);
  return WDC_OK;
}
static inline int cache_check_batch(wdc_context* ctx, const char* who, int64_t batch, int64_t tokens, int64_t table_pages,
                                    int64_t page_tokens) {
  WDC_REQUIRE(ctx, batch >= 0 && batch < (1ll << 24) && tokens >= 0 && tokens < (1ll << 24) && table_pages >= 0 &&
              table_pages * page_tokens < (1ll << 31) - 256, "%s: bad batch", who);
  return WDC_OK;
}
static inline int cache_check_strides(wdc_context* ctx, const char* who, const int64_t* strides, int n) {
  for (int i = 0; i < n; i++)
    WDC_REQUIRE(ctx, strides[i] >= 0 && strides[i] % 4 == 0, "%s: strides must be non-negative multiples of 4", who);
  return WDC_OK;
}
#define CACHE_TRY(call)                 \
  do {                                  \
    const int s_ = (call);              \
    if (s_ != WDC_OK) return s_;        \
  } while (0)
