// The norm of a head and its rotation by a position, as wdc_rotate_heads and wdc_cache_append_rotary share them.
//
//   n = x * w / sqrt(mean(x^2) + epsilon)                     (or n = x)
//   y1 = n1 cos - n2 sin,   y2 = n2 cos + n1 sin              for the pairs (n1, n2) of the first 2 * half channels
//
// A head's float4 are taken two at a time, so that the channels of a pair are in one thread: slot p has float4 p and p + half / 4 while
// there are pairs that far apart, float4 2 p and 2 p + 1 of what is left (or with `interleaved`); in either case its cosines are those
// from number 4 p on.  A group of lanes has a head's slots, and the norm alone is an exchange between lanes.
//
// T is what lies between the float32 numbers that are read and the ones that are written.  Heads that stay float32 are computed in that:
// |error| <= 2^-20 (|n1| + |n2|) (a sum of at most 256 squares in at most 13 additions one after the other, so that its root is 7 x
// 2^-24 off, 3 x for rsqrtf, and two products and a rotation), with 64 bits for heads whose squares leave the range.  The keys of a cache
// are computed in 64 bits and rounded once: their codes hang on the last bit.  (In 64 bits everywhere, 9001 x 24 heads of 80 took 48 us, as
// long as the conversions do, of which an SM makes 16 a cycle and a head needs three a number.)
#pragma once

#include "paged_cache.cuh"

struct HeadRotation {
  const float *cos, *sin;          // [places][half]
  const int32_t* positions;        // null: a row's own number
  int64_t places;
  double epsilon, share;           // share: 1 / head_size
  int half, interleaved;           // half: pairs, a multiple of 4
};

// The row of the tables that a position names; the nearest one where there is none.
__device__ __forceinline__ int64_t rotation_place(const HeadRotation& r, int64_t position, int* status) {
  if (position >= 0 && position < r.places) return position;
  status[WDC_STATUS_DRAFT] = 1;
  return position < 0 ? 0 : r.places - 1;
}
template <class T>
struct Quad {
  T x, y, z, w;
};
// (volatile: a number is converted once and not again at each use)
__device__ __forceinline__ void widen(float x, double& y) { asm volatile("cvt.f64.f32 %0, %1;" : "=d"(y) : "f"(x)); }
__device__ __forceinline__ void widen(float x, float& y) { y = x; }
template <class T>
__device__ __forceinline__ Quad<T> quad_of(float4 x) {
  Quad<T> q;
  widen(x.x, q.x);
  widen(x.y, q.y);
  widen(x.z, q.z);
  widen(x.w, q.w);
  return q;
}
template <class T>
__device__ __forceinline__ float4 rounded(Quad<T> n) { return make_float4((float)n.x, (float)n.y, (float)n.z, (float)n.w); }
template <class T>
__device__ __forceinline__ T square_sum(Quad<T> x) { return x.x * x.x + x.y * x.y + (x.z * x.z + x.w * x.w); }
template <class T>
__device__ __forceinline__ Quad<T> scaled(Quad<T> x, T by, Quad<T> weight) {
  return {x.x * by * weight.x, x.y * by * weight.y, x.z * by * weight.z, x.w * by * weight.w};
}

// The two float4 of slot p of a head, and whether they are rotated.
struct Slot {
  int a, b;
  bool turns;
  __device__ __forceinline__ Slot(const HeadRotation& r, int p) {
    const int h = r.half >> 2;
    turns = p < h;
    a = turns && !r.interleaved ? p : 2 * p;
    b = turns && !r.interleaved ? p + h : 2 * p + 1;
  }
};
template <class T>
struct Angles {
  Quad<T> cos, sin;
};
template <class T>
__device__ __forceinline__ Angles<T> rotation_angles(const HeadRotation& r, int64_t place, int p) {
  if (4 * p >= r.half) return {};
  const int64_t at = place * r.half + 4 * p;
  return {quad_of<T>(pdl_ld(reinterpret_cast<const float4*>(r.cos + at))), quad_of<T>(pdl_ld(reinterpret_cast<const float4*>(r.sin + at)))};
}
template <class T>
__device__ __forceinline__ void rotate_slot(const HeadRotation& r, Quad<T>& a, Quad<T>& b, const Angles<T>& t) {
  const Quad<T> x = a, y = b, c = t.cos, s = t.sin;
  if (r.interleaved) {
    a = {x.x * c.x - x.y * s.x, x.y * c.x + x.x * s.x, x.z * c.y - x.w * s.y, x.w * c.y + x.z * s.y};
    b = {y.x * c.z - y.y * s.z, y.y * c.z + y.x * s.z, y.z * c.w - y.w * s.w, y.w * c.w + y.z * s.w};
  } else {
    a = {x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y, x.z * c.z - y.z * s.z, x.w * c.w - y.w * s.w};
    b = {y.x * c.x + x.x * s.x, y.y * c.y + x.y * s.y, y.z * c.z + x.z * s.z, y.w * c.w + x.w * s.w};
  }
}
template <class T>
__device__ __forceinline__ T group_sum(T x, int lanes) {
  for (int w = lanes / 2; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
// Normalises a head, of which a lane has SLOTS slots and a group of `lanes`, a power of two, all of them.  All lanes of the warp.
template <int SLOTS>
__device__ __forceinline__ void normalise(const HeadRotation& r, Quad<double> (&a)[SLOTS], Quad<double> (&b)[SLOTS], int lanes,
                                          const Quad<double> (&wa)[SLOTS], const Quad<double> (&wb)[SLOTS]) {
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < SLOTS; k++) sum += square_sum(a[k]) + square_sum(b[k]);
  const double by = rsqrt(fma(group_sum(sum, lanes), r.share, r.epsilon));
#pragma unroll
  for (int k = 0; k < SLOTS; k++) {
    a[k] = scaled(a[k], by, wa[k]);
    b[k] = scaled(b[k], by, wb[k]);
  }
}
// (squares that are not normal numbers count, or may be missing: every number by itself in 64 bits)
template <int SLOTS>
__device__ __noinline__ void normalise_far(double share, double epsilon, float4 (&a)[SLOTS], float4 (&b)[SLOTS], int lanes, const float4 (&wa)[SLOTS],
                                           const float4 (&wb)[SLOTS]) {
  double sum = 0.0;
  for (int k = 0; k < SLOTS; k++) sum += square_sum(quad_of<double>(a[k])) + square_sum(quad_of<double>(b[k]));
  const double by = rsqrt(fma(group_sum(sum, lanes), share, epsilon));
  for (int k = 0; k < SLOTS; k++) {
    a[k] = rounded(scaled(quad_of<double>(a[k]), by, quad_of<double>(wa[k])));
    b[k] = rounded(scaled(quad_of<double>(b[k]), by, quad_of<double>(wb[k])));
  }
}
template <int SLOTS>
__device__ __forceinline__ void normalise(const HeadRotation& r, Quad<float> (&a)[SLOTS], Quad<float> (&b)[SLOTS], int lanes,
                                          const Quad<float> (&wa)[SLOTS], const Quad<float> (&wb)[SLOTS]) {
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < SLOTS; k++) sum += square_sum(a[k]) + square_sum(b[k]);
  const float mean = fmaf(group_sum(sum, lanes), (float)r.share, (float)r.epsilon);
  const bool far = !(mean > 1e-24f && mean < 1e30f);
  if (__any_sync(0xffffffffu, far)) {
    float4 x[SLOTS], y[SLOTS], u[SLOTS], v[SLOTS];
#pragma unroll
    for (int k = 0; k < SLOTS; k++) {
      x[k] = rounded(a[k]); y[k] = rounded(b[k]); u[k] = rounded(wa[k]); v[k] = rounded(wb[k]);
    }
    normalise_far(r.share, r.epsilon, x, y, lanes, u, v);
#pragma unroll
    for (int k = 0; k < SLOTS; k++)
      if (far) {
        a[k] = quad_of<float>(x[k]);
        b[k] = quad_of<float>(y[k]);
      }
  }
  if (far) return;
  const float by = rsqrtf(mean);
#pragma unroll
  for (int k = 0; k < SLOTS; k++) {
    a[k] = scaled(a[k], by, wa[k]);
    b[k] = scaled(b[k], by, wb[k]);
  }
}

// EACH heads of a row, x_sh and y_sh apart, by a group of `lanes`: the first `heads` are normalised and rotated, and of the others the
// first `cleared` become zero.  All loads are on their way before the first is used, and nothing of a head is written before all of it has
// been read.  All lanes of the warp.
template <int SLOTS, int EACH>
__device__ __forceinline__ void rotate_heads_of(const HeadRotation& r, const float* x, int64_t x_sh, float* y, int64_t y_sh, int heads, int cleared, int lane,
                                                int lanes, int quads, const float* weights, int64_t position, int* status) {
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 va[EACH][SLOTS], vb[EACH][SLOTS];
#pragma unroll
  for (int e = 0; e < EACH; e++) {
    const float4* head = reinterpret_cast<const float4*>(x + e * x_sh);
#pragma unroll
    for (int k = 0; k < SLOTS; k++) {
      const Slot slot(r, lane + k * lanes);
      va[e][k] = e < heads && slot.a < quads ? pdl_ld(head + slot.a) : zero;
      vb[e][k] = e < heads && slot.b < quads ? pdl_ld(head + slot.b) : zero;
    }
  }
  const int64_t place = r.half == 0 || heads == 0 ? 0 : rotation_place(r, position, status);
  const float4* weight = reinterpret_cast<const float4*>(weights);
  Quad<float> wa[SLOTS], wb[SLOTS];
  Angles<float> angles[SLOTS];
#pragma unroll
  for (int k = 0; k < SLOTS; k++) {
    const Slot slot(r, lane + k * lanes);
    wa[k] = quad_of<float>(weight && slot.a < quads ? pdl_ld(weight + slot.a) : zero);
    wb[k] = quad_of<float>(weight && slot.b < quads ? pdl_ld(weight + slot.b) : zero);
    angles[k] = rotation_angles<float>(r, place, lane + k * lanes);
  }
#pragma unroll
  for (int e = 0; e < EACH; e++) {
    Quad<float> na[SLOTS], nb[SLOTS];
#pragma unroll
    for (int k = 0; k < SLOTS; k++) {
      na[k] = quad_of<float>(va[e][k]);
      nb[k] = quad_of<float>(vb[e][k]);
    }
    if (weight) normalise(r, na, nb, lanes, wa, wb);
    float4* head = reinterpret_cast<float4*>(y + e * y_sh);
#pragma unroll
    for (int k = 0; k < SLOTS; k++) {
      const Slot slot(r, lane + k * lanes);
      if (slot.turns) rotate_slot(r, na[k], nb[k], angles[k]);
      if (e < heads && slot.a < quads) head[slot.a] = rounded(na[k]);
      if (e < heads && slot.b < quads) head[slot.b] = rounded(nb[k]);
      if (e >= heads && e < cleared && slot.a < quads) head[slot.a] = zero;
      if (e >= heads && e < cleared && slot.b < quads) head[slot.b] = zero;
    }
  }
}

// Heads in memory: `size` floats at every batch * stride[0] + row * stride[1] + head * stride[2].
struct HeadRows {
  const float* at;
  int64_t count[3], stride[3], size;
  bool any() const { return at && count[0] > 0 && count[1] > 0 && count[2] > 0; }
  // Floats from the first to behind the last, of the strides that are no multiple of `pitch` (0: of all).
  int64_t span(int64_t pitch) const {
    int64_t n = size;
    for (int i = 0; i < 3; i++)
      if (count[i] > 1 && (pitch == 0 || stride[i] % pitch)) n += (count[i] - 1) * stride[i];
    return n;
  }
  bool same(const HeadRows& o) const {
    bool same = at == o.at;
    for (int i = 0; i < 3; i++) same = same && (count[i] <= 1 || stride[i] == o.stride[i]);
    return same;
  }
};
// Whether heads that are written may be some of those that are read.  (Columns of one buffer, both in rows as wide as that, lie
// beside one another.)
static inline bool heads_overlap(const HeadRows& x, const HeadRows& y) {
  if (!x.any() || !y.any()) return false;
  const uintptr_t from_x = reinterpret_cast<uintptr_t>(x.at), from_y = reinterpret_cast<uintptr_t>(y.at);
  if (from_x + 4 * x.span(0) <= from_y || from_y + 4 * y.span(0) <= from_x) return false;
  const int64_t apart = from_y > from_x ? (int64_t)(from_y - from_x) / 4 : -((int64_t)(from_x - from_y) / 4);
  for (const int64_t pitch : {x.stride[0], x.stride[1], x.stride[2], y.stride[0], y.stride[1], y.stride[2]}) {
    if (pitch == 0) continue;
    const int64_t behind = (apart % pitch + pitch) % pitch, x_wide = x.span(pitch), y_wide = y.span(pitch);
    if (x_wide <= behind && y_wide <= pitch - behind) return false;
  }
  return true;
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
  r = {cos, sin, positions, places, (double)epsilon, 1.0 / (double)head_size, (int)(rotary / 2), interleaved != 0};
  return WDC_OK;
}
