// Heads normalised and rotated by their positions (wdc_rotate_heads): ONNX's RotaryEmbedding, with the norm of each head that comes
// before it in many decoders.  The reference has no such operator.
#include <math.h>

#include "head_rotation.cuh"

namespace {

constexpr int THREADS = 256;

struct RotateArgs {
  const float *x, *weight;
  float* y;
  int* status;
  HeadRotation rotation;
  int64_t rows, x_st, x_sh, y_st, y_sh;
  int heads, head_size, chunks;      // chunks of EACH heads a row
};

// A group of LANES lanes takes EACH heads of a row, QUADS float4 a lane, all of them loaded before the first is used.  Nothing of a
// head is written before all of it has been read: y may be x.
template <int LANES, int QUADS, int EACH>
__global__ void __launch_bounds__(THREADS) rotate_heads_kernel(const RotateArgs a) {
  pdl_wait();
  constexpr int GROUPS = THREADS / LANES;
  const int lane = threadIdx.x % LANES, quads = a.head_size >> 2;
  const int64_t item = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
  const bool there = item < a.rows * a.chunks;
  const int64_t row = there ? item / a.chunks : 0;
  const int head0 = there ? (int)(item - row * a.chunks) * EACH : 0;
  const int heads = there ? min(EACH, a.heads - head0) : 0;
  const float* x = pdl_after(a.x) + row * a.x_st + head0 * a.x_sh;
  float4 v[EACH][QUADS];
#pragma unroll
  for (int e = 0; e < EACH; e++)
#pragma unroll
    for (int k = 0; k < QUADS; k++) {
      const int quad = lane + k * LANES;
      v[e][k] = e < heads && quad < quads ? pdl_ld(reinterpret_cast<const float4*>(x + e * a.x_sh) + quad) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  QuadAngles angles[QUADS];
  float4 weight[QUADS];
  const int64_t position = a.rotation.half == 0 ? 0 : a.rotation.positions ? (int64_t)pdl_ld(a.rotation.positions + row) : row;
  const int64_t place = a.rotation.half == 0 ? 0 : rotation_place(a.rotation, position, a.status);
#pragma unroll
  for (int k = 0; k < QUADS; k++) {
    const int quad = lane + k * LANES;
    angles[k] = rotation_angles(a.rotation, place, quad);
    weight[k] = a.weight && quad < quads ? pdl_ld(reinterpret_cast<const float4*>(a.weight) + quad) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float* y = a.y + row * a.y_st + head0 * a.y_sh;
#pragma unroll
  for (int e = 0; e < EACH; e++) {
    if (QUADS == 1) {
      const float4 out = rotated_head(a.rotation, v[e][0], lane, LANES, a.head_size, a.weight != nullptr, weight[0], angles[0]);
      if (e < heads && lane < quads) *(reinterpret_cast<float4*>(y + e * a.y_sh) + lane) = out;
    } else {
      Quad64 n[QUADS];
      double sum = 0.0;
#pragma unroll
      for (int k = 0; k < QUADS; k++) sum += square_sum(v[e][k]);
      const double by = a.weight ? rsqrt(group_sum(sum, LANES) / a.head_size + a.rotation.epsilon) : 1.0;
#pragma unroll
      for (int k = 0; k < QUADS; k++)
        n[k] = a.weight ? scaled(v[e][k], by, weight[k]) : Quad64{v[e][k].x, v[e][k].y, v[e][k].z, v[e][k].w};
#pragma unroll
      for (int k = 0; k < QUADS; k++) {
        const int quad = lane + k * LANES;
        const bool turns = quad * 2 < a.rotation.half;
        float4 out;
        if (a.rotation.interleaved) {
          out = turns ? rotated_neighbours(n[k], angles[k]) : rounded(n[k]);
        } else {
          // the other channels are in any lane, in any of its float4
          const int other = other_quad(a.rotation, quad);
          Quad64 o = from_lane(n[0], other % LANES);
#pragma unroll
          for (int m = 1; m < QUADS; m++) {
            const Quad64 p = from_lane(n[m], other % LANES);
            if (other / LANES == m) o = p;
          }
          out = turns ? rotated_halves(n[k], o, angles[k], quad * 4 >= a.rotation.half) : rounded(n[k]);
        }
        if (e < heads && quad < quads) *(reinterpret_cast<float4*>(y + e * a.y_sh) + quad) = out;
      }
    }
  }
}

template <int LANES, int QUADS>
int launch(wdc_context* ctx, RotateArgs& a) {
  constexpr int GROUPS = THREADS / LANES;
  // four heads a group where that still gives every SM work
  const bool many = a.rows * a.heads >= 4 * GROUPS * (int64_t)ctx->sm_count;
  a.chunks = many ? (a.heads + 3) / 4 : a.heads;
  const int64_t ctas = ceil_div64(a.rows * a.chunks, GROUPS);
  WDC_REQUIRE(ctx, ctas < (1ll << 31), "wdc_rotate_heads: rows exceed the grid");
  wdc_launch_pdl(ctx, many ? rotate_heads_kernel<LANES, QUADS, 4> : rotate_heads_kernel<LANES, QUADS, 1>, dim3((unsigned)ctas), dim3(THREADS),
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
  RotateArgs a = {x, weight, y, ctx->status_word, {}, d->rows, d->x_st, d->x_sh, d->y_st, d->y_sh, (int)d->heads, (int)d->head_size, 0};
  if (d->rows == 0 || d->heads == 0) return WDC_OK;
  CACHE_TRY(rotation_check(ctx, "wdc_rotate_heads", a.rotation, d->head_size, d->rotary, d->places, cos, sin, positions, d->epsilon, d->interleaved));
  WDC_REQUIRE(ctx, x && y, "wdc_rotate_heads: null argument");
  WDC_REQUIRE(ctx, cache_aligned(x, 16) && cache_aligned(y, 16) && cache_aligned(weight, 16), "wdc_rotate_heads: buffers are not aligned");
  DeviceGuard g(ctx->device);
  const int quads = a.head_size / 4;
  return quads <= 8 ? launch<8, 1>(ctx, a) : quads <= 16 ? launch<16, 1>(ctx, a) : quads <= 32 ? launch<32, 1>(ctx, a) : launch<32, 2>(ctx, a);
}
