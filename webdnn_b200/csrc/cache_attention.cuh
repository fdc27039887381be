// What the kernels for attention over a paged 8-bit cache share.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include "paged_cache.cuh"

struct CacheAttArgs {
  const float* q;
  const int8_t* codes;
  const float* scales;
  const int32_t *page_table, *lengths, *counts;
  const int32_t* parents;          // of new tokens that are a tree, or null
  float* y;
  int* status;
  int64_t pages, table_pages;
  int64_t q_sb, q_sh, q_st, y_sb, y_sh, y_st;
  int batch, tokens, heads, kv_heads, group, page_shift;   // 2^page_shift tokens a page
  int row_tiles;
  int splits;                      // CTAs of a unit; 0: the tiles of all units are shared out
  float *part_rows, *part_stats;   // of every unit and split, or two of every CTA: O of a unit's rows; m, M and l
  int* part_plan;                  // first tile of each sequence in the order of all, their number, tiles of a CTA
  float scale_log2;                // scale * log2(e): the softmax runs on exp2
};

constexpr float WEIGHT_BITS = 14.f;        // weights are less than 2^15: both halves stay in float16's normal range
constexpr int QUERY_BITS = 13;             // a row's queries are scaled to less than 2^14

// New tokens that are a tree: token i sees what is before the new ones, its ancestors and itself, as a bit for each place from the last
// multiple of 32 on that is not behind the first new one.  At most TREE_MOST new tokens.
constexpr int TREE_MOST = 1024, TREE_WORDS = TREE_MOST / 32 + 1;
// The row of new token `token` (behind the count: all bits, nobody reads its row), of words up to that of place `end` - 1.
__device__ __forceinline__ void tree_row(uint32_t* words, const int32_t* parents, int token, int count, int before, int end, int* status) {
  const int first = before & ~31, n = min((end - first + 31) >> 5, TREE_WORDS);
  for (int w = 0; w < n; w++) words[w] = token >= count ? 0xffffffffu : w == 0 ? (1u << (before & 31)) - 1 : 0u;
  for (int i = token; i >= 0 && token < count;) {
    const int at = (before & 31) + i;
    words[at >> 5] |= 1u << (at & 31);
    const int parent = pdl_ld(parents + i);
    if (parent < -1 || parent >= i) status[WDC_STATUS_DRAFT] = 1;
    i = parent < i ? parent : -1;
  }
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Two halves of a pair: h = x in float16, l = what is missing.
__device__ __forceinline__ void split_halves(float x, float y, uint32_t& h, uint32_t& l) {
  const __half2 hi = __floats2half2_rn(x, y);
  const float2 back = __half22float2(hi);
  h = half2_bits(hi);
  l = half2_bits(__floats2half2_rn(x - back.x, y - back.y));
}
// Two bytes of a word of codes + 128 as float16: 0x6400 + byte is 1024 + byte.
template <int SELECT>
__device__ __forceinline__ uint32_t two_codes(uint32_t w) {
  const uint32_t u = __byte_perm(w, 0x64646464u, SELECT);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return half2_bits(v);
}

__device__ __forceinline__ float exp2_of(float x) {      // results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A key scale; one that is no number or infinite makes every score NaN, whatever the codes beside it are.
__device__ __forceinline__ float key_scale_of(float scale) { return fabsf(scale) < INFINITY ? scale : NAN; }
// A value scale as 2^e * f, 1 <= f < 2 (0: e = -infinity; no number: f is NaN).
__device__ __forceinline__ void exponent_of(float scale, float& e, float& f) {
  const bool small = scale < 1.2e-38f;                       // (below the normal range)
  const uint32_t bits = __float_as_uint(small ? scale * 16777216.f : scale);
  e = scale > 0.f && scale < INFINITY ? (float)((int)(bits >> 23) - (small ? 151 : 127)) : scale == 0.f ? -INFINITY : 0.f;
  f = scale < INFINITY ? __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) : NAN;
}

__device__ __forceinline__ float finite_or_0(float x) { return x == -INFINITY ? 0.f : x; }   // a reference to subtract
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127
// What a row of queries is scaled by, 2^(QUERY_BITS - exponent of its largest) with the sign of `scale`, and what its scores are to be
// scaled by for it, which is not negative.  No exponent below -100: smaller queries than that weigh nothing.
__device__ __forceinline__ float query_scale(float peak, float scale, float& row_scale) {
  const int e = max((int)(__float_as_uint(peak) >> 23) - 127, -100);
  row_scale = power_of_2(e - QUERY_BITS) * fabsf(scale);
  return copysignf(power_of_2(QUERY_BITS - e), scale);
}

// For many new tokens (cache_attention_tc.cu); WDC_ERR_UNSUPPORTED where the other kernel is to run.
int wdc_cache_attention_tc(wdc_context* ctx, CacheAttArgs a, int head_size);
// Joins a.splits equal parts of tiles of `tile_rows` rows, 8 or 128 (cache_attention.cu).
int wdc_cache_attention_join(wdc_context* ctx, const CacheAttArgs& a, int head_size, int tile_rows);
