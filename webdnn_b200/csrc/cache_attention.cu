// Attention of new tokens over a paged cache in 8 bits:  y = softmax(scale * q k^T) v,  k = code * (scale of page and head).
// The reference has no such operator.
#include <math.h>

#include "paged_cache.cuh"

namespace {

constexpr int THREADS = 128;

struct CacheAttArgs {
  const float* q;
  const int8_t* codes;
  const float* scales;
  const int32_t *page_table, *lengths, *counts;
  float* y;
  int* status;
  int64_t pages, table_pages;
  int64_t q_sb, q_sh, q_st, y_sb, y_sh, y_st;
  int tokens, heads, kv_heads, group, page_tokens;
  float scale_log2;   // scale * log2(e): the softmax runs on exp2
};

// One CTA per (sequence, new token, query head); warp w takes tokens w, w + 4, ..., a lane DH / 32 channels, and the warps'
// maxima, sums and rows are joined at the end.
template <int DH>
__global__ void __launch_bounds__(THREADS) cache_attention_kernel(const CacheAttArgs a) {
  constexpr int C = DH / 32, WARPS = THREADS / 32;
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = (int)(blockIdx.x % (unsigned)a.heads), rest = (int)(blockIdx.x / (unsigned)a.heads);
  const int i = rest % a.tokens, b = rest / a.tokens;
  const CacheSpan span = cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages * a.page_tokens, a.status);
  const int last = i < span.count ? span.length - span.count + i : -1;   // the token itself
  const float* q = pdl_after(a.q) + b * a.q_sb + h * a.q_sh + i * a.q_st;
  float qc[C], o[C], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < C; c++) {
    qc[c] = last >= 0 ? pdl_ld(q + lane * C + c) * a.scale_log2 : 0.f;
    o[c] = 0.f;
  }
  for (int t = warp; t <= last; t += WARPS) {
    const int page = cache_page(a.page_table + (int64_t)b * a.table_pages, t / a.page_tokens, a.pages, a.status);
    if (page < 0) continue;
    const int64_t block = (int64_t)page * 2 * a.kv_heads + h / a.group;
    const int8_t* k = pdl_after(a.codes) + (block * a.page_tokens + t % a.page_tokens) * DH + lane * C;
    const int8_t* v = k + (int64_t)a.kv_heads * a.page_tokens * DH;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++) s = fmaf(qc[c], (float)k[c], s);
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= pdl_ld(a.scales + block);
    const float vs = pdl_ld(a.scales + block + a.kv_heads);
    const float top = fmaxf(m, s);
    const float keep = top == -INFINITY ? 1.f : exp2f(m - top), e = top == -INFINITY ? 0.f : exp2f(s - top);
    l = l * keep + e;
#pragma unroll
    for (int c = 0; c < C; c++) o[c] = o[c] * keep + e * vs * (float)v[c];
    m = s == s ? top : s;
  }
  __shared__ float ms[WARPS], ls[WARPS], os[WARPS][DH];
  if (lane == 0) {
    ms[warp] = m;
    ls[warp] = l;
  }
#pragma unroll
  for (int c = 0; c < C; c++) os[warp][lane * C + c] = o[c];
  __syncthreads();
  if ((int)threadIdx.x < DH) {
    float top = -INFINITY, total = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, ms[w]);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = ms[w] == -INFINITY ? 0.f : exp2f(ms[w] - top);
      total = fmaf(ls[w], f, total);
      sum = fmaf(os[w][threadIdx.x], f, sum);
    }
    a.y[b * a.y_sb + h * a.y_sh + i * a.y_st + threadIdx.x] = total == 0.f ? 0.f : sum / total;
  }
}

}  // namespace

extern "C" int wdc_cache_attention(wdc_context* ctx, const wdc_cache_attention_desc* d, const float* q, const void* codes,
                                   const float* scales, const int32_t* page_table, const int32_t* lengths,
                                   const int32_t* counts, float* y) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_cache_attention: null context");
  WDC_TAPE(ctx, wdc_cache_attention, tape_desc(d), q, codes, scales, page_table, lengths, counts, y);
  wdc_note_write(ctx, y);
  WDC_REQUIRE(ctx, d, "wdc_cache_attention: null argument");
  CACHE_TRY(cache_check_pool(ctx, "wdc_cache_attention", d->pages, d->kv_heads, d->page_tokens, d->head_size));
  CACHE_TRY(cache_check_batch(ctx, "wdc_cache_attention", d->batch, d->tokens, d->table_pages, d->page_tokens));
  WDC_REQUIRE(ctx, d->heads > 0 && d->heads <= 65535 && d->heads % d->kv_heads == 0,
              "wdc_cache_attention: %lld query heads for %lld key heads", (long long)d->heads, (long long)d->kv_heads);
  const int64_t strides[6] = {d->q_sb, d->q_sh, d->q_st, d->y_sb, d->y_sh, d->y_st};
  CACHE_TRY(cache_check_strides(ctx, "wdc_cache_attention", strides, 6));
  if (d->batch == 0 || d->tokens == 0) return WDC_OK;
  WDC_REQUIRE(ctx, q && codes && scales && lengths && y && (page_table || d->table_pages == 0),
              "wdc_cache_attention: null argument");
  WDC_REQUIRE(ctx, cache_aligned(q, 16) && cache_aligned(codes, 16) && cache_aligned(y, 16) && cache_aligned(scales, 4) &&
              cache_aligned(page_table, 4) && cache_aligned(lengths, 4) && cache_aligned(counts, 4),
              "wdc_cache_attention: buffers are not aligned");
  CacheAttArgs a = {q, (const int8_t*)codes, scales, page_table, lengths, counts, y, ctx->status_word, d->pages,
                    d->table_pages, d->q_sb, d->q_sh, d->q_st, d->y_sb, d->y_sh, d->y_st, (int)d->tokens, (int)d->heads,
                    (int)d->kv_heads, (int)(d->heads / d->kv_heads), (int)d->page_tokens, d->scale * 1.4426950408889634f};
  const int64_t ctas = d->batch * d->tokens * d->heads;
  WDC_REQUIRE(ctx, ctas < (1ll << 31), "wdc_cache_attention: batch exceeds the grid");
  DeviceGuard g(ctx->device);
  auto kernel = d->head_size == 32 ? cache_attention_kernel<32> : d->head_size == 64 ? cache_attention_kernel<64>
                                                                                      : cache_attention_kernel<128>;
  wdc_launch_pdl(ctx, kernel, dim3((unsigned)ctas), dim3(THREADS), 0, a);
  return wdc_check_launch(ctx, "cache_attention_kernel");
}
