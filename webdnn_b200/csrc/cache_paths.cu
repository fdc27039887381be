// The tokens of a tree that stand move to the front of their sequence's new ones (wdc_cache_keep_paths).  The reference has no such
// operator.
#include "paged_cache.cuh"

namespace {

struct KeepArgs {
  int8_t* codes;
  float* scales;
  const int32_t *page_table, *lengths, *counts, *path, *accepted;
  int* status;
  int64_t pages, table_pages;
  int layers, kv_heads, tokens, page_shift, lane_shift;   // 2^lane_shift lanes have 16 bytes each of a token's head
};
constexpr int WARPS = 4;

// |code|, the largest of a word's four.
__device__ __forceinline__ uint32_t abs_max4(uint32_t w, uint32_t most) { return __vmaxu4(__vabs4(w), most); }
__device__ __forceinline__ uint32_t largest_byte(uint32_t w) {
  w = __vmaxu4(w, w >> 16);
  return max(w & 255u, w >> 8 & 255u);
}
// Codes in units of `from` as codes in units of `to`, rint(code * from / to).  A page that stands for NaN has codes of 0.
__device__ __noinline__ uint32_t divided4(uint32_t w, float from, float to) {
  uint32_t out = 0;
  if (!(to > 0.f && to < INFINITY)) return 0;
#pragma unroll 1
  for (int j = 0; j < 32; j += 8) {
    const float r = rintf(__fdiv_rn(__fmul_rn((float)(int8_t)(w >> j), from), to));
    out |= (uint32_t)((int)fminf(fmaxf(r, -127.f), 127.f) & 255) << j;
  }
  return out;
}
// Without a division where it cannot matter: the product with 1 / to is within 3e-5 of the quotient (at most 127, three roundings of 2^-24), so
// where it is further than that from a half the nearest whole number is the same, and is read off the sum with 1.5 * 2^23.  (A code + 128
// as the last byte of 2^23 is a float32 number.)  inverse: 0 where 1 / to might leave the normal range, a code * from
// might (`from` is at most 127 `to` where the code is not 0), or `to` is no number.
__device__ __forceinline__ uint32_t again4(uint32_t w, float from, float to, float inverse) {
  const float magic = 12582912.f, zero = 8388736.f;
  const uint32_t biased = w ^ 0x80808080u;
  float r[4], off = 0.f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float t = __fmul_rn(__fmul_rn(__uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7650 + j)) - zero, from), inverse);
    r[j] = t + magic;
    off = fmaxf(off, fabsf(t - (r[j] - magic)));
  }
  if (off < 0.4999f && inverse > 0.f)
    return __byte_perm(__byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040), __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040), 0x5410);
  return divided4(w, from, to);
}
__device__ __forceinline__ float inverse_of(float to) { return to > 1e-30f && to < 1e30f ? __frcp_rn(to) : 0.f; }
__device__ __forceinline__ uint4 again16(uint4 v, float from, float to, float inverse) {
  return make_uint4(again4(v.x, from, to, inverse), again4(v.y, from, to, inverse), again4(v.z, from, to, inverse), again4(v.w, from, to, inverse));
}

// A warp per sequence, layer, side and head; 2^(5 - lane_shift) tokens at a time, of 32 that the lanes have looked up.  A path rises, so a
// token's old place is never before its new one: taken in order, with all of a step's loads before its stores, and page after page,
// nothing is overwritten before it is read.
// A page's new scale is known from a first pass over the tokens that come to it.  Bound: issue, of the codes that are rounded again (40
// sequences, up to nine tokens, 30 layers of 8 heads of 128: 15.3 us; with a division each 17.8, two steps' loads together 15.7, four 18.8),
// and the chain of dependent loads (path, page table, scales, codes) where they are few (2.7 us).
__global__ void __launch_bounds__(32 * WARPS) cache_keep_kernel(const KeepArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31, b = (int)blockIdx.y;
  const int64_t unit = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);          // layer, side, head
  if (unit >= (int64_t)a.layers * 2 * a.kv_heads) return;
  const CacheSpan span = cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages << a.page_shift, a.status);
  const int accepted = pdl_ld(a.accepted + b), start = span.length - span.count;
  const int32_t* path = pdl_after(a.path) + (int64_t)b * a.tokens;
  if (accepted < 0 || accepted > span.count) {
    a.status[WDC_STATUS_DRAFT] = 1;
    return;
  }
  int first = accepted;                            // the first token that is elsewhere
  bool rises = true;
  for (int i = lane; i < accepted; i += 32) {
    const int p = path[i], last = i ? path[i - 1] : -1;
    rises &= p > last && p < span.count;
    if (p != i) first = min(first, i);
  }
  if (!__all_sync(0xffffffffu, rises)) {
    if (lane == 0) a.status[WDC_STATUS_DRAFT] = 1;
    return;
  }
  first = __reduce_min_sync(0xffffffffu, first);
  const int kinds = 2 * a.kv_heads, layer = (int)(unit / kinds), kind = (int)(unit - (int64_t)layer * kinds);
  const int64_t block_bytes = (int64_t)16 << (a.page_shift + a.lane_shift);       // of a page, side and head
  int8_t* codes = pdl_after(a.codes) + (int64_t)layer * a.pages * kinds * block_bytes;
  float* scales = pdl_after(a.scales) + (int64_t)layer * a.pages * kinds;
  const int32_t* table = pdl_after(a.page_table) + (int64_t)b * a.table_pages;
  const int size = 1 << a.page_shift, lanes = 1 << a.lane_shift, together = 32 >> a.lane_shift;
  const int mine = lane >> a.lane_shift, piece = lane & (lanes - 1);
  const auto block_of = [&](int page) { return (int64_t)page * kinds + kind; };
  const auto page_at = [&](int64_t index) { return cache_page(table, index, a.pages, a.status); };
  const auto piece_of = [&](int page, int in_page) {
    return reinterpret_cast<uint4*>(codes) + (block_of(page) << (a.page_shift + a.lane_shift)) + ((in_page << a.lane_shift) + piece);
  };

  // What a lane knows of a token of the path: where it comes from, and the page and scale of that.
  int of = -1, at_in_page = 0;
  float by = 0.f;
  const auto look_up = [&](int i, int end, int page) {
    of = -1;
    if (i < end) {
      const int from = start + path[i];
      of = page_at(from >> a.page_shift);
      at_in_page = from & (size - 1);
      by = of >= 0 && of != page ? scales[block_of(of)] : 0.f;
    }
  };
  // The piece of token k + mine of those that the lanes know of, where it comes from (or -1) and the scale there.
  struct Source {
    uint4 v;
    int of;
    float by;
  };
  const auto source = [&](int k, int not_of) {
    const int token = (k + mine) & 31, at = __shfl_sync(0xffffffffu, at_in_page, token);
    Source s = {make_uint4(0, 0, 0, 0), __shfl_sync(0xffffffffu, of, token), __shfl_sync(0xffffffffu, by, token)};
    if (s.of == not_of) s.of = -1;
    if (s.of >= 0) s.v = *piece_of(s.of, at);
    return s;
  };

  for (int i0 = first; i0 < accepted;) {           // the kept tokens of one page: i0 .. i1 - 1
    const int index = (start + i0) >> a.page_shift, i1 = min(accepted, ((index + 1) << a.page_shift) - start);
    const int page = page_at(index);
    if (page < 0) {
      i0 = i1;
      continue;
    }
    const float before = scales[block_of(page)];
    float scale = before;
    uint32_t peak = 0;                             // of this lane, as bits: a NaN is above infinity
    for (int c = i0; c < i1; c += 32) {
      look_up(c + lane, i1, page);
      if (!__any_sync(0xffffffffu, of >= 0 && of != page)) continue;
      for (int k = 0; k < min(32, i1 - c); k += together) {
        const Source s = source(k, page);
        const uint32_t most = largest_byte(abs_max4(s.v.x, abs_max4(s.v.y, abs_max4(s.v.z, abs_max4(s.v.w, 0)))));
        // (a scale that is no number or infinite stands for NaN)
        if (s.of >= 0) peak = max(peak, __float_as_uint(fabsf(s.by) < INFINITY ? __fdiv_rn(__fmul_rn((float)most, s.by), 127.f) : NAN) & 0x7fffffffu);
      }
    }
    const float fresh = __uint_as_float(__reduce_max_sync(0xffffffffu, peak));
    if (!(fresh <= scale) && fabsf(scale) < INFINITY) scale = fresh;
    const bool grown = __float_as_uint(scale) != __float_as_uint(before);
    const float inverse = inverse_of(scale);
    if (grown) {
      // what the page holds already: older tokens, and the first of the new ones, which stay where they are
      const int old = start + i0 - (index << a.page_shift);
      for (int t = mine; t < old; t += together) {
        uint4* at = piece_of(page, t);
        *at = again16(*at, before, scale, inverse);
      }
    }
    for (int c = i0; c < i1; c += 32) {
      if (i1 - i0 > 32) look_up(c + lane, i1, page);
      for (int k = 0; k < min(32, i1 - c); k += together) {
        const Source s = source(k, -1);
        __syncwarp();
        const bool stays = s.of == page;
        if (s.of >= 0) *piece_of(page, (start + c + k + mine) & (size - 1)) = stays && !grown ? s.v : again16(s.v, stays ? before : s.by, scale, inverse);
        __syncwarp();
      }
    }
    if (grown && lane == 0) scales[block_of(page)] = scale;
    __syncwarp();
    i0 = i1;
  }
}

}  // namespace

extern "C" int wdc_cache_keep_paths(wdc_context* ctx, const wdc_cache_keep_desc* d, void* codes, float* scales, const int32_t* page_table,
                                    const int32_t* lengths, const int32_t* counts, const int32_t* path, const int32_t* accepted) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_cache_keep_paths: null context");
  WDC_NO_TAPE(ctx);   // (a second time it would move what has been moved)
  wdc_note_write(ctx, codes);
  wdc_note_write(ctx, scales);
  const char* who = "wdc_cache_keep_paths";
  WDC_REQUIRE(ctx, d, "%s: null argument", who);
  CACHE_TRY(cache_check_pool(ctx, who, d->pages, d->kv_heads, d->page_tokens, d->head_size));
  CACHE_TRY(cache_check_batch(ctx, who, d->batch, d->tokens, d->table_pages, d->page_tokens));
  WDC_REQUIRE(ctx, d->layers > 0 && d->layers < (1ll << 20), "%s: bad pool", who);
  if (d->batch == 0 || d->tokens == 0) return WDC_OK;
  WDC_REQUIRE(ctx, codes && scales && lengths && path && accepted && (page_table || d->table_pages == 0), "%s: null argument", who);
  WDC_REQUIRE(ctx, cache_aligned(codes, 16) && cache_aligned(scales, 4) && cache_aligned(page_table, 4) && cache_aligned(lengths, 4) &&
              cache_aligned(counts, 4) && cache_aligned(path, 4) && cache_aligned(accepted, 4), "%s: buffers are not aligned", who);
  KeepArgs a = {(int8_t*)codes, scales, page_table, lengths, counts, path, accepted, ctx->status_word, d->pages, d->table_pages,
                (int)d->layers, (int)d->kv_heads, (int)d->tokens, 4, 1};
  while (1 << a.page_shift < d->page_tokens) a.page_shift++;
  while (16 << a.lane_shift < d->head_size) a.lane_shift++;
  const int64_t ctas = ceil_div64(d->layers * 2 * d->kv_heads, WARPS);
  WDC_REQUIRE(ctx, ctas < (1ll << 31) && d->batch <= 65535, "%s: batch exceeds the grid", who);
  DeviceGuard g(ctx->device);
  wdc_launch_pdl(ctx, cache_keep_kernel, dim3((unsigned)ctas, (unsigned)d->batch), dim3(32 * WARPS), 0, a);
  return wdc_check_launch(ctx, "cache_keep_kernel");
}
