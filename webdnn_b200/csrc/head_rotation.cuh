// The norm of a head and its rotation by a position, as wdc_rotate_heads and wdc_cache_append_rotary share them.
//
//   n = x * w / sqrt(mean(x^2) + epsilon)                     (or n = x)
//   y1 = n1 cos - n2 sin,   y2 = n2 cos + n1 sin              for the pairs (n1, n2) of the first 2 * half channels
//
// A group of lanes (8, 16 or 32, enough for one float4 each) holds a head.  Everything between the float32 numbers that are read and
// the one that is written is in 64 bits, so that a result is the definition's, rounded once: the code of a key in a cache depends on its
// last bit, and is then the same wherever the head was rotated.
#pragma once

#include "paged_cache.cuh"

struct HeadRotation {
  const float *cos, *sin;          // [places][half]
  const int32_t* positions;        // null: a row's own number
  int64_t places;
  double epsilon;
  int half, interleaved;           // half: pairs, a multiple of 4
};

// The row of the tables that a position names; the nearest one where there is none.
__device__ __forceinline__ int64_t rotation_place(const HeadRotation& r, int64_t position, int* status) {
  if (position >= 0 && position < r.places) return position;
  status[WDC_STATUS_DRAFT] = 1;
  return position < 0 ? 0 : r.places - 1;
}
// Cosines and sines of float4 number `quad` of a head: of its four channels, or (x, y) of its two pairs.
struct QuadAngles {
  float4 cos, sin;
};
__device__ __forceinline__ QuadAngles rotation_angles(const HeadRotation& r, int64_t place, int quad) {
  QuadAngles a = {};
  if (quad * 2 >= r.half) return a;
  if (r.interleaved) {
    const int64_t at = place * r.half + quad * 2;
    const float2 c = *reinterpret_cast<const float2*>(pdl_after(r.cos) + at), s = *reinterpret_cast<const float2*>(pdl_after(r.sin) + at);
    a.cos.x = c.x; a.cos.y = c.y;
    a.sin.x = s.x; a.sin.y = s.y;
  } else {
    const int64_t at = place * r.half + (quad * 4 >= r.half ? quad * 4 - r.half : quad * 4);
    a.cos = pdl_ld(reinterpret_cast<const float4*>(r.cos + at));
    a.sin = pdl_ld(reinterpret_cast<const float4*>(r.sin + at));
  }
  return a;
}
__device__ __forceinline__ double square_sum(float4 x) {
  const double a = x.x, b = x.y, c = x.z, d = x.w;
  return fma(a, a, fma(b, b, fma(c, c, d * d)));
}
// Of a group of `lanes`, a power of two.
__device__ __forceinline__ double group_sum(double x, int lanes) {
  for (int w = lanes / 2; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
struct Quad64 {
  double x, y, z, w;
};
__device__ __forceinline__ Quad64 scaled(float4 x, double by, float4 weight) {
  return {x.x * by * weight.x, x.y * by * weight.y, x.z * by * weight.z, x.w * by * weight.w};
}
__device__ __forceinline__ float4 rounded(Quad64 n) { return make_float4((float)n.x, (float)n.y, (float)n.z, (float)n.w); }
// Pairs of neighbours; pairs of channels `half` apart, whose other channels `o` another lane has.
__device__ __forceinline__ float4 rotated_neighbours(Quad64 n, QuadAngles a) {
  const double c0 = a.cos.x, s0 = a.sin.x, c1 = a.cos.y, s1 = a.sin.y;
  return rounded({n.x * c0 - n.y * s0, n.y * c0 + n.x * s0, n.z * c1 - n.w * s1, n.w * c1 + n.z * s1});
}
__device__ __forceinline__ float4 rotated_halves(Quad64 n, Quad64 o, QuadAngles a, bool upper) {
  const double sign = upper ? 1.0 : -1.0;
  return rounded({n.x * a.cos.x + sign * a.sin.x * o.x, n.y * a.cos.y + sign * a.sin.y * o.y, n.z * a.cos.z + sign * a.sin.z * o.z,
                  n.w * a.cos.w + sign * a.sin.w * o.w});
}
__device__ __forceinline__ Quad64 from_lane(Quad64 n, int lane) {
  return {__shfl_sync(0xffffffffu, n.x, lane), __shfl_sync(0xffffffffu, n.y, lane), __shfl_sync(0xffffffffu, n.z, lane),
          __shfl_sync(0xffffffffu, n.w, lane)};
}
// The lane, or number, of the float4 that holds the other channels of float4 `quad`'s pairs.
__device__ __forceinline__ int other_quad(const HeadRotation& r, int quad) {
  const int h = r.half >> 2;
  return quad < h ? quad + h : quad < 2 * h ? quad - h : quad;
}
// One float4 a lane.  All lanes of the warp; lanes without a part of a head hold zeros.  normed: `weight` counts.
__device__ __forceinline__ float4 rotated_head(const HeadRotation& r, float4 x, int quad, int lanes, int head_size, bool normed, float4 weight,
                                               QuadAngles a) {
  Quad64 n = {x.x, x.y, x.z, x.w};
  if (normed) n = scaled(x, rsqrt(group_sum(square_sum(x), lanes) / head_size + r.epsilon), weight);
  if (r.half == 0) return rounded(n);
  const bool turns = quad * 2 < r.half;
  if (r.interleaved) return turns ? rotated_neighbours(n, a) : rounded(n);
  const Quad64 o = from_lane(n, (int)(threadIdx.x & 31) - quad + other_quad(r, quad));
  return turns ? rotated_halves(n, o, a, quad * 4 >= r.half) : rounded(n);
}

static inline int rotation_check(wdc_context* ctx, const char* who, HeadRotation& r, int64_t head_size, int64_t rotary, int64_t places,
                                 const float* cos, const float* sin, const int32_t* positions, float epsilon, int interleaved) {
  WDC_REQUIRE(ctx, rotary >= 0 && rotary <= head_size && places >= 0 && places < (1ll << 31), "%s: bad rotation", who);
  if (rotary % 8) return wdc_fail(ctx, WDC_ERR_UNSUPPORTED, "%s: %lld rotated channels (multiples of 8)", who, (long long)rotary);
  WDC_REQUIRE(ctx, epsilon >= 0.f && epsilon < INFINITY, "%s: bad epsilon", who);
  if (rotary) {
    WDC_REQUIRE(ctx, places > 0 && cos && sin, "%s: a rotation has tables", who);
    WDC_REQUIRE(ctx, cache_aligned(cos, 16) && cache_aligned(sin, 16) && cache_aligned(positions, 4), "%s: buffers are not aligned", who);
  }
  r = {cos, sin, positions, places, (double)epsilon, (int)(rotary / 2), interleaved != 0};
  return WDC_OK;
}
