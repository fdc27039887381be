// Log probabilities of given tokens under softmax(logits), the distribution's entropy and its best alternatives.  The
// reference has no such operator: its graphs end at Softmax (operators/cpu/operators/standard/softmax.ts:15-59).
#include <math.h>

#include "tape.cuh"

namespace {

constexpr int THREADS = 256, TOP_MOST = 32;

struct LogprobArgs {
  const float* logits;
  const int32_t* tokens;
  float *logprob, *entropy, *top_logprobs;
  int32_t* top_ids;
  int64_t row_stride;
  int vocab, top;
};

// A key that orders by value, NaN above everything and -0 as 0, then by the lower index.
__device__ __forceinline__ uint64_t order_key(float x, int index) {
  uint32_t bits = x == x ? __float_as_uint(x + 0.f) : 0x7fffffffu;
  bits = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return (uint64_t)bits << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t bits = (uint32_t)(key >> 32);
  return __uint_as_float(bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
}

// s = sum e^(x - m), t = sum (x - m) e^(x - m), without terms of x = -inf.
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
  if (a.m == -INFINITY) return b;
  if (b.m == -INFINITY) return a;
  const float m = fmaxf(a.m, b.m), fa = expf(a.m - m), fb = expf(b.m - m);
  Sums r;
  r.m = m;
  r.s = a.s * fa + b.s * fb;
  // (a difference whose exponential is 0 is cut off: times the sum it could be infinite, and 0 times that NaN)
  r.t = fa * fmaf(a.s, fmaxf(a.m - m, -200.f), a.t) + fb * fmaf(b.s, fmaxf(b.m - m, -200.f), b.t);
  return r;
}

__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const LogprobArgs a) {
  pdl_wait();
  __shared__ Sums parts[THREADS / 32];
  __shared__ uint64_t best[THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const float* x = pdl_after(a.logits) + row * a.row_stride;
  Sums sums = {-INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
    const float v = pdl_ld(x + i);
    if (v != -INFINITY) sums = joined(sums, {v, 1.f + (v - v), v - v});   // (v - v: NaN for infinity and NaN)
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1)
    sums = joined(sums, {__shfl_xor_sync(0xffffffffu, sums.m, w), __shfl_xor_sync(0xffffffffu, sums.s, w),
                         __shfl_xor_sync(0xffffffffu, sums.t, w)});
  if (lane == 0) parts[warp] = sums;
  __syncthreads();
  sums = parts[0];
  for (int w = 1; w < THREADS / 32; w++) sums = joined(sums, parts[w]);
  const float log_s = logf(sums.s);
  const bool none = sums.m == -INFINITY;
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int token = pdl_ld(a.tokens + row);
      a.logprob[row] = none || token < 0 || token >= a.vocab ? NAN : x[token] - sums.m - log_s;
    }
    if (a.entropy) a.entropy[row] = none ? NAN : log_s - sums.t / sums.s;
  }
  uint64_t below = ~0ull;
  for (int k = 0; k < a.top; k++) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
      const uint64_t key = order_key(pdl_ld(x + i), i);
      if (key < below && key > mine) mine = key;
    }
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, w));
    __syncthreads();
    if (lane == 0) best[warp] = mine;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; w++) mine = max(mine, best[w]);
    below = mine;
    if (threadIdx.x == 0) {
      a.top_ids[row * a.top + k] = (int32_t)~(uint32_t)mine;
      a.top_logprobs[row * a.top + k] = none ? NAN : key_value(mine) - sums.m - log_s;
    }
  }
}

}  // namespace

extern "C" int wdc_token_logprobs(wdc_context* ctx, const wdc_logprobs_desc* d, const float* logits, const int32_t* tokens,
                                  float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_token_logprobs: null context");
  WDC_TAPE(ctx, wdc_token_logprobs, tape_desc(d), logits, tokens, logprob, entropy, top_ids, top_logprobs);
  wdc_note_write(ctx, logprob);
  wdc_note_write(ctx, entropy);
  wdc_note_write(ctx, top_ids);
  wdc_note_write(ctx, top_logprobs);
  WDC_REQUIRE(ctx, d, "wdc_token_logprobs: null argument");
  WDC_REQUIRE(ctx, d->rows >= 0 && d->rows < (1ll << 31) && d->vocab > 0 && d->vocab < (1ll << 31) - 4096 && d->row_stride >= 0,
              "wdc_token_logprobs: bad shape");
  WDC_REQUIRE(ctx, d->top >= 0 && d->top <= TOP_MOST && d->top <= d->vocab, "wdc_token_logprobs: top %lld of %lld (0 to %d)",
              (long long)d->top, (long long)d->vocab, TOP_MOST);
  if (d->rows == 0) return WDC_OK;
  WDC_REQUIRE(ctx, logits && (tokens || !logprob) && !top_ids == !top_logprobs, "wdc_token_logprobs: null argument");
  DeviceGuard g(ctx->device);
  LogprobArgs a = {logits, tokens, logprob, entropy, top_logprobs, top_ids, d->row_stride, (int)d->vocab,
                   top_ids ? (int)d->top : 0};
  wdc_launch_pdl(ctx, token_logprobs_kernel, dim3((unsigned)d->rows), dim3(THREADS), 0, a);
  return wdc_check_launch(ctx, "token_logprobs_kernel");
}
