// Heads normalised and rotated by their positions (wdc_rotate_heads): ONNX's RotaryEmbedding, with the norm of each head that comes
// before it in many decoders.  The reference has no such operator.
#include <math.h>

#include "head_rotation.cuh"

namespace {

constexpr int THREADS = 64;

struct RotateArgs {
  const float *x, *weight;
  float* y;
  int* status;
  HeadRotation rotation;
  int64_t x_st, x_sh, y_st, y_sh;
  int heads, head_size;
  uint32_t chunks, items;            // chunks of EACH heads a row, and in all
};

// A group of LANES lanes takes EACH heads of a row, SLOTS slots a lane.  y may be x: no two groups have a head.
//
// Bound: the latency of loads (9001 rows of 24 heads of 80, 139 MB: 26.5 us, 5.2 TB/s, at 43% of what DRAM could and 35% of the issue slots: 128
// registers a thread leave 3.6 warps a scheduler, which wait; of 16 heads of 128 25.1, 5.9 TB/s); the launch for few (1.7 us).
// A CTA is a chain of loads, sums and stores, so small ones, which end at different times, leave fewer gaps (us of these three and of
// 500 rows of 8 heads of 128, by threads a CTA: 256 29.9, 26.1, 1.85, 2.09; 128 27.7, 25.2, 1.57, 2.06; 64 27.0, 25.1, 1.56, 2.06; 32 26.7, 25.0,
// 1.64, 2.35).  CTAS: of 256 threads an SM, that many registers.
template <int LANES, int SLOTS, int EACH, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS * 256 / THREADS) rotate_heads_kernel(const RotateArgs a) {
  pdl_wait();
  const uint32_t item = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
  const bool there = item < a.items;
  const uint32_t at = there ? item / a.chunks : 0;
  const int head0 = there ? (int)(item - at * a.chunks) * EACH : 0, heads = there ? min(EACH, a.heads - head0) : 0;
  const int64_t row = at, position = a.rotation.half && a.rotation.positions ? (int64_t)pdl_ld(a.rotation.positions + row) : row;
  rotate_heads_of<SLOTS, EACH>(a.rotation, pdl_after(a.x) + row * a.x_st + head0 * a.x_sh, a.x_sh, a.y + row * a.y_st + head0 * a.y_sh, a.y_sh, heads, 0,
                               threadIdx.x % LANES, LANES, a.head_size >> 2, a.weight, position, a.status);
}

template <int LANES, int SLOTS, int MOST, int CTAS>
int launch(wdc_context* ctx, RotateArgs& a, int64_t rows) {
  constexpr int GROUPS = THREADS / LANES;
  // several heads a group where that still gives every SM work
  const bool many = rows * a.heads >= 2 * MOST * GROUPS * (int64_t)ctx->sm_count;
  const int each = many ? MOST : 1;
  a.chunks = (uint32_t)((a.heads + each - 1) / each);
  WDC_REQUIRE(ctx, rows * a.chunks < (1ll << 32) - THREADS, "wdc_rotate_heads: rows exceed the grid");
  a.items = (uint32_t)(rows * a.chunks);
  const int64_t ctas = ceil_div64(a.items, GROUPS);
  wdc_launch_pdl(ctx, many ? rotate_heads_kernel<LANES, SLOTS, MOST, CTAS> : rotate_heads_kernel<LANES, SLOTS, 1, CTAS>, dim3((unsigned)ctas), dim3(THREADS),
                 0, a);
  return wdc_check_launch(ctx, "rotate_heads_kernel");
}

}  // namespace

extern "C" int wdc_rotate_heads(wdc_context* ctx, const wdc_rotate_desc* d, const float* x, const float* weight, const float* cos,
                                const float* sin, const int32_t* positions, float* y) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_rotate_heads: null context");
  WDC_TAPE(ctx, wdc_rotate_heads, tape_desc(d), x, weight, cos, sin, positions, y);
  wdc_note_write(ctx, y);
  WDC_REQUIRE(ctx, d, "wdc_rotate_heads: null argument");
  WDC_REQUIRE(ctx, d->rows >= 0 && d->rows < (1ll << 31) && d->heads >= 0 && d->heads <= 65535 && d->head_size > 0, "wdc_rotate_heads: bad shape");
  if (d->head_size % 4 || d->head_size > 256)
    return wdc_fail(ctx, WDC_ERR_UNSUPPORTED, "wdc_rotate_heads: heads of %lld (multiples of 4 up to 256)", (long long)d->head_size);
  const int64_t strides[4] = {d->x_st, d->x_sh, d->y_st, d->y_sh};
  CACHE_TRY(cache_check_strides(ctx, "wdc_rotate_heads", strides, 4));
  RotateArgs a = {x, weight, y, ctx->status_word, {}, d->x_st, d->x_sh, d->y_st, d->y_sh, (int)d->heads, (int)d->head_size, 0, 0};
  if (d->rows == 0 || d->heads == 0) return WDC_OK;
  CACHE_TRY(rotation_check(ctx, "wdc_rotate_heads", a.rotation, d->head_size, d->rotary, d->places, cos, sin, positions, d->epsilon, d->interleaved));
  WDC_REQUIRE(ctx, x && y, "wdc_rotate_heads: null argument");
  WDC_REQUIRE(ctx, cache_aligned(x, 16) && cache_aligned(y, 16) && cache_aligned(weight, 16), "wdc_rotate_heads: buffers are not aligned");
  // (groups write in no order: what others are still to read would be gone)
  const HeadRows from = {x, {1, d->rows, d->heads}, {0, d->x_st, d->x_sh}, d->head_size}, to = {y, {1, d->rows, d->heads}, {0, d->y_st, d->y_sh}, d->head_size};
  WDC_REQUIRE(ctx, from.same(to) || !heads_overlap(from, to), "wdc_rotate_heads: y overlaps x and is not x");
  DeviceGuard g(ctx->device);
  const int slots = (a.head_size / 4 + 1) / 2;
  // Lanes, slots and heads a group by what was measured with CTAs of 256 threads, us of 173 million numbers (floor 22): heads of 32 26.2 (two
  // slots a lane 34.1), of 64 25.7 (two slots 26.5, two heads 27.1), of 128 25.8 (one slot 25.7, one head 27.5), of 80 29.2 (8 lanes of two
  // slots 31.0, 16 of one 31.4, 2 of five 42).
  return slots <= 4    ? launch<4, 1, 4, 3>(ctx, a, d->rows)
         : slots <= 8  ? launch<8, 1, 4, 3>(ctx, a, d->rows)
         : slots <= 12 ? launch<4, 3, 2, 2>(ctx, a, d->rows)
         : slots <= 16 ? launch<8, 2, 2, 3>(ctx, a, d->rows)
         : slots <= 24 ? launch<8, 3, 2, 2>(ctx, a, d->rows)
                       : launch<16, 2, 2, 3>(ctx, a, d->rows);
}
