// Which drafted tokens of a tree stand, and the token that follows them (wdc_verify_drafts).  The reference has no such operator: its
// graphs end at Softmax (operators/cpu/operators/standard/softmax.ts:15-59).
//
// The walk from token to token is serial, and only the rows of logits that it comes by are needed.  A cluster of CTAs takes a
// sequence: each warp of it has a range of the vocabulary, whose maximum and sum of exponentials it finds; the first CTA (the leader)
// joins them, tests or draws, and tells the others what to do next.
//
// A drawn token is the one in whose range of the running sum a number falls, and with 100000 tokens there are borders everywhere: sums that
// are 2^-22 of the whole off would name another token in several of a hundred draws.  In 64 bits a weight takes 25 instructions, four
// times as many as in 32.  So a walk is made in 32 bits, together with a bound of what that leaves out; a test or a draw that is nearer
// to a border than the bound stops it, and a second kernel, in 64 bits, goes on from the token that it stands at.
//
// In 32 bits the weights stay in shared memory, where a rejection makes p into max(p - q, 0).  The bound E is one of the sum of all weights'
// errors (so of any running sum's, too):
//   a weight 2^t, t = (x - top) c:  2^-22 of it for the exponential, 3 * 2^-24 |t| ln 2 for t's three roundings, and the sum of four
//   weights in 32 bits two more of 2^-24; so E = 1.6 * 2^-22 S + 2.2 * 2^-24 sum w |t|, S = sum w.  The last sum is that of -w log2 w,
//   which is concave: over n weights it is at most S log2(n / S);
//   a rejection, p / S - q with q of sum 1:  E' = 2 E / S + Eq + 8 * 2^-24  (S is off by E itself; four roundings, and the sum's two).
// In 64 bits the exponential is 2^(n / 16) from a table times a polynomial in what is left, 11 operations in all, within 2^-42.
//
// Bound: what is serial, the chain of a pass (logits to shared memory, weights, sums, two barriers of the cluster, the leader's decision),
// 12000 to 20000 cycles of which memory has a tenth; 28% of the issue slots are used.  One sequence of 5 new tokens, 32000 in the
// vocabulary, drafts with their logits: 20.6 us; 16 of 25, 100003, without them: 48.6; 64 of 9, 50001, with them: 112, of which the 64-bit kernel
// has 45 for four walks (64 bits alone: 28.7, 62 and 144).  What 64 bits do alone: temperature 0 (16 of 25, 100003: 58), and drafts with their
// logits above about 108000 tokens, whose rows have no room in shared memory (one sequence of 5: 25 us of 100000, 77 of 128256).
#include <limits.h>
#include <math.h>

#include "paged_cache.cuh"

namespace {

constexpr int WARPS = 16, THREADS = 32 * WARPS, PARTS_MOST = 8, RANGES_MOST = WARPS * PARTS_MOST;
constexpr int TOKENS_MOST = 1024;
constexpr int PART_LEAST = 1024;                   // logits of a CTA, where a row is cut into several
constexpr int SLICE_BYTES = 106 * 1024;            // shared memory for a CTA's logits and what it has of tokens, two CTAs an SM

struct VerifyArgs {
  const float *logits, *draft, *uniforms;
  const int32_t *tokens, *parents, *counts;
  int32_t *path, *accepted, *next;
  int* status;
  int64_t logits_sb, logits_st, draft_sb, draft_st;
  int n_tokens, vocab, parts;
  int goes_on;
  int chunk, chunks;                               // float4 of a warp's range that are in shared memory at a time, and how many times
  double scale, draft_scale;                       // 16 log2(e) / temperature; 0: temperature 0
};

// What a range of a row has, or all of a CTA's, or the row: the largest logit, the sum of 2^((x - top) scale / 16), or where the first of
// the largest is; whether there is a NaN or +inf.
struct Range {
  double sum, off;                                 // off: E
  float top;
  int first, bad, unused;
};
__device__ __forceinline__ Range nothing() { return {0.0, 0.0, -INFINITY, 0x7fffffff, 0, 0}; }
enum Todo { STOP = 0, ROW = 1, RESIDUAL = 2 };
struct Command {
  int todo, token;                                 // the token that the walk stands at
  int with_draft;                                  // ROW: whether the draft's row is wanted; RESIDUAL: rejections, this one included
  int first, draft_first;
  float top, draft_top;
  int guess;                                       // the token that the walk may come to next, or -1
  double draft_inverse, step;                      // 1 / sum of the draft's weights, of those before the last rejection
};
struct Shared {
  double table[16];
  // as many as there are tokens, behind the logits
  double* steps;                                   // 1 / the sums that a rejection divided by
  float* uniforms;                                 // of the leader
  int *tokens, *parents, *path;
  Command command;
  Range mine[2][WARPS];                            // of this CTA's ranges: target and draft
  float tops[2][WARPS];                            // their largest logits
  // of the leader
  Range parts[2][PARTS_MOST];
  double run[RANGES_MOST], fresh[RANGES_MOST];     // sums of all ranges, relative to their CTA's largest; after the last rejection
  double part_factors[PARTS_MOST];                 // what relates that to the row's
  double warp_sums[WARPS];
  float all_tops[2][RANGES_MOST];                  // the largest logits of all ranges
  double draw_error;                               // E, for a draw
  int draw;                                        // which uniform a token is to be drawn with, or -1
  uint32_t found, last;
};
constexpr int TOKEN_BYTES = 24;

__device__ __forceinline__ uint32_t cluster_at(const void* p, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void cluster_put(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
template <class T>
__device__ __forceinline__ void cluster_put(T* to, int rank, const T& value) {
  static_assert(sizeof(T) % 4 == 0, "words");
  const uint32_t at = cluster_at(to, rank);
  uint32_t w[sizeof(T) / 4];
  memcpy(w, &value, sizeof(T));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); i++) cluster_put(at + 4 * i, w[i]);
}
// All threads of the cluster wait for one another.  What a CTA has written by then is seen by the others: its warp 0, behind a barrier of the
// CTA's, says so for all.
__device__ __forceinline__ void cluster_sync() {
  if (threadIdx.x < 32) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  else asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// 2^(d scale / 16), d = x - top <= 0, within 2^-42 of it; 0 where that is below 2^-1000 (d is -inf or NaN).  n is the nearest whole
// number to d scale, which adding 1.5 * 2^52 leaves in the last bits; 2^(g / 16), |g| <= 1/2, by five terms of its series.  N of
// them side by side, step by step: one waits for 14 operations in a row.
template <int N>
__device__ __forceinline__ void powers(const float (&x)[N], float top, double scale, const double* table, double (&out)[N]) {
  const double magic = 6755399441055744.0, u = 0.043321698784996582, high = top;           // ln(2) / 16
  const float near_scale = (float)scale;
  double d[N], shifted[N], g[N], p[N], t[N];
#pragma unroll
  for (int i = 0; i < N; i++) d[i] = (double)x[i] - high;
#pragma unroll
  for (int i = 0; i < N; i++) shifted[i] = fma(d[i], scale, magic);
#pragma unroll
  for (int i = 0; i < N; i++) t[i] = table[__double2loint(shifted[i]) & 15];
#pragma unroll
  for (int i = 0; i < N; i++) g[i] = fma(d[i], scale, magic - shifted[i]);
#pragma unroll
  for (int i = 0; i < N; i++) p[i] = fma(u * u * u * u * u / 120, g[i], u * u * u * u / 24);
#pragma unroll
  for (int i = 0; i < N; i++) p[i] = fma(p[i], g[i], u * u * u / 6);
#pragma unroll
  for (int i = 0; i < N; i++) p[i] = fma(p[i], g[i], u * u / 2);
#pragma unroll
  for (int i = 0; i < N; i++) p[i] = fma(p[i], g[i], u) * g[i];
#pragma unroll
  for (int i = 0; i < N; i++) p[i] = fma(t[i], p[i], t[i]);
#pragma unroll
  for (int i = 0; i < N; i++) {
    const double y = __hiloint2double(__double2hiint(p[i]) + ((__double2loint(shifted[i]) >> 4) << 20), __double2loint(p[i]));
    out[i] = (x[i] - top) * near_scale > -16000.f ? y : 0.0;
  }
}
__device__ __forceinline__ double power(float x, float top, double scale, const double* table) {
  const float one[1] = {x};
  double out[1];
  powers(one, top, scale, table, out);
  return out[0];
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
template <int LANES>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
  for (int w = 1; w < LANES; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
  return x;
}
template <int LANES>
__device__ __forceinline__ int group_min(int x) {
#pragma unroll
  for (int w = 1; w < LANES; w <<= 1) x = min(x, __shfl_xor_sync(0xffffffffu, x, w));
  return x;
}

// How a row is cut: float4 number j has logits 4 j - before .. + 3 (`before`: how far the row is behind a 16-byte boundary), and a
// warp has `each` float4 of them.
struct Cut {
  int before, quads, each;
  __device__ __forceinline__ Cut(const float* row, int vocab, int ranges_shift) {
    before = (int)(reinterpret_cast<uintptr_t>(row) >> 2 & 3);
    quads = (vocab + before + 3) >> 2;
    each = (quads + (1 << ranges_shift) - 1) >> ranges_shift;
  }
  __device__ __forceinline__ int first(int range) const { return min(range * each, quads); }
  __device__ __forceinline__ int logit(int quad) const { return max(4 * quad - before, 0); }
};

// `quads` float4 of a row, from logit i0 on, to shared memory, by asynchronous copies of a warp; -inf where the row has none, which is in the
// first and the last.  whole: as they are in memory.
__device__ __forceinline__ void fetch_quads(float4* to, const float* row, int vocab, int i0, int quads, bool whole) {
  const int lane = threadIdx.x & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(to);
  const bool cut_off = quads > 0 && (i0 < 0 || i0 + 4 * quads > vocab);
  if (whole) {
    const int end = i0 + 4 * quads > vocab ? quads - 1 : quads;
    int j = i0 < 0 && lane == 0 ? 32 : lane;       // (the first float4 is cut off)
    const float* from = row + i0 + 4 * j;
    uint32_t at = base + 16 * j;
#pragma unroll 4
    for (; j < end; j += 32, from += 128, at += 512) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    if (!cut_off) return;
  }
  // number by number: all of them, or the first and the last float4
#pragma unroll 1
  for (int k = lane; k < 4 * quads; k += 32) {
    if (whole && k >= 4 && k < 4 * quads - 4) continue;
    const int i = i0 + k;
    if (i >= 0 && i < vocab) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(base + 4 * k), "l"(row + i) : "memory");
    else reinterpret_cast<float*>(to)[k] = -INFINITY;
  }
}

// What a warp's range has: its float4, `quads` from logit i0 on, which are in `mine`, or are brought there a chunk at a time where they
// are several chunks.  (A function of its own, which has the registers to itself.)
__device__ __noinline__ Range row_range(float4* mine, const float* row, int vocab, int i0, int quads, int chunk, int chunks, bool whole, double scale,
                                        const double* table) {
  const int lane = threadIdx.x & 31;
  Range r = nothing();
#pragma unroll 1
  for (; quads > 0; quads -= chunk, i0 += 4 * chunk) {
    const int n = min(quads, chunk);
    if (chunks > 1) {
      __syncwarp();
      fetch_quads(mine, row, vocab, i0, n, whole);
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
    float its_top = -INFINITY;
    int bad = 0;
#pragma unroll 2
    for (int j = lane; j < n; j += 32) {
      const float4 v = mine[j];
      const float most = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
      if (most > its_top) {
        its_top = most;
        if (scale == 0.0 && most > r.top) r.first = i0 + 4 * j + (v.x == most ? 0 : v.y == most ? 1 : v.z == most ? 2 : 3);
      }
      bad |= !(v.x < INFINITY) | !(v.y < INFINITY) | !(v.z < INFINITY) | !(v.w < INFINITY);
    }
    r.bad |= bad;
    if (scale == 0.0) {                            // (lanes have their own largest, and the first of it)
      r.top = fmaxf(r.top, its_top);
      continue;
    }
    const float top = fmaxf(r.top, group_max<32>(its_top));
    if (top > r.top) {
      r.sum *= power(r.top, top, scale, table);
      r.top = top;
    }
#pragma unroll 1
    for (int j = lane; j < n; j += 32) {
      const float4 v = mine[j];
      const float x[4] = {v.x, v.y, v.z, v.w};
      double w[4];
      powers(x, r.top, scale, table, w);
      r.sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
  }
  r.bad = __any_sync(0xffffffffu, r.bad);
  if (scale == 0.0) {
    const float top = group_max<32>(r.top);
    r.first = __reduce_min_sync(0xffffffffu, r.top == top ? r.first : 0x7fffffff);
    r.top = top;
  } else {
    r.sum = warp_sum(r.sum);
  }
  return r;
}

// The weight of tokens under the target's distribution after `n` rejections, not normalised.
struct Weights {
  const Command& c;
  const double *table, *steps;
  double scale, draft_scale;
  int n;
  template <int N>
  __device__ __forceinline__ void drafted(int i, int step, const float (&y)[N], double (&q)[N]) const {
    if (draft_scale != 0.0) powers(y, c.draft_top, draft_scale, table, q);
#pragma unroll
    for (int e = 0; e < N; e++) q[e] = draft_scale == 0.0 ? (double)(i + e * step == c.draft_first) : q[e] * c.draft_inverse;
  }
  // of N tokens i, i + step, .. with logits x and y
  template <int N>
  __device__ __forceinline__ void of(int i, int step, const float (&x)[N], const float (&y)[N], double (&p)[N]) const {
    if (scale != 0.0) powers(x, c.top, scale, table, p);
#pragma unroll
    for (int e = 0; e < N; e++)
      if (scale == 0.0) p[e] = (double)(i + e * step == c.first);
    if (n == 0) return;
    double q[N];
    drafted(i, step, y, q);
    // (both rounded before the difference: where the distributions are equal it is 0, and not what rounding q left out)
#pragma unroll 1
    for (int k = 0; k < n; k++) {
      const double by = steps[k];
#pragma unroll
      for (int e = 0; e < N; e++) p[e] = fmax(__dsub_rn(__dmul_rn(p[e], by), q[e]), 0.0);
    }
  }
  // For a draw: of tokens from, from + 1, .. < hi of a range; 0 behind it.
  __device__ __forceinline__ const Weights& in(int, const Cut&) const { return *this; }
  template <int N>
  __device__ __forceinline__ void take(const float* row, const float* draft, int from, int hi, double (&p)[N]) const {
    float x[N], y[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
      x[e] = from + e < hi ? pdl_ld(row + from + e) : -INFINITY;
      y[e] = from + e < hi && n ? pdl_ld(draft + from + e) : -INFINITY;
    }
    of(from, 1, x, y, p);
#pragma unroll
    for (int e = 0; e < N; e++) p[e] = from + e < hi ? p[e] : 0.0;
  }
};

// The sum of a warp's range after `n` rejections; its float4 of both sides are in shared memory, `apart` float4 from one another, or are
// brought there again where they are several chunks.
__device__ __noinline__ double residual(float4* mine, int apart, const float* row, const float* draft, int vocab, int i0, int quads, int chunk, int chunks,
                                        bool same, const Weights& weights) {
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
#pragma unroll 1
  for (; quads > 0; quads -= chunk, i0 += 4 * chunk) {
    const int n = min(quads, chunk);
    if (chunks > 1) {
      __syncwarp();
      fetch_quads(mine, row, vocab, i0, n, true);
      fetch_quads(mine + apart, draft, vocab, i0, n, same);
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
#pragma unroll 1
    for (int j = lane; j < n; j += 32) {
      const float4 v = mine[j], u = mine[apart + j];
      const float x[4] = {v.x, v.y, v.z, v.w}, y[4] = {u.x, u.y, u.z, u.w};
      double w[4];
      weights.of(i0 + 4 * j, 1, x, y, w);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
  }
  return warp_sum(sum);
}

// ------------------------------------------------------------------------------------------- in 32 bits
__device__ __forceinline__ float exp2_of(float x) {      // results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (top: not -inf)
__device__ __forceinline__ float near_weight(float x, float top, float c) { return exp2_of((x - top) * c); }
// A warp's logits in shared memory become weights relative to the largest of them, both sides together (SIDES), so that one's exchanges
// between lanes hide the other's.  (A NaN or +inf makes the sum NaN.)
template <int SIDES>
__device__ __noinline__ void near_ranges(Shared& sh, float4* mine, int apart, int quads, double scale, double draft_scale) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float top[SIDES], ref[SIDES];
  const float c[2] = {(float)(scale / 16), (float)(draft_scale / 16)};
#pragma unroll
  for (int side = 0; side < SIDES; side++) top[side] = -INFINITY;
#pragma unroll 2
  for (int j = lane; j < quads; j += 32) {
#pragma unroll
    for (int side = 0; side < SIDES; side++) {
      const float4 v = mine[side * apart + j];
      top[side] = fmaxf(top[side], fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1)
#pragma unroll
    for (int side = 0; side < SIDES; side++) top[side] = fmaxf(top[side], __shfl_xor_sync(0xffffffffu, top[side], w));
  double sum[SIDES];
#pragma unroll
  for (int side = 0; side < SIDES; side++) {
    ref[side] = top[side] == -INFINITY ? 0.f : top[side];
    sum[side] = 0.0;
  }
#pragma unroll 2
  for (int j = lane; j < quads; j += 32) {
#pragma unroll
    for (int side = 0; side < SIDES; side++) {
      const float4 x = mine[side * apart + j];
      const float4 w = make_float4(near_weight(x.x, ref[side], c[side]), near_weight(x.y, ref[side], c[side]), near_weight(x.z, ref[side], c[side]),
                                   near_weight(x.w, ref[side], c[side]));
      mine[side * apart + j] = w;
      sum[side] += (double)((w.x + w.y) + (w.z + w.w));
    }
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1)
#pragma unroll
    for (int side = 0; side < SIDES; side++) sum[side] += __shfl_xor_sync(0xffffffffu, sum[side], w);
  if (lane == 0) {
#pragma unroll
    for (int side = 0; side < SIDES; side++) {
      sh.mine[side][warp] = {sum[side], 0.0, top[side], 0x7fffffff, sum[side] != sum[side], 0};
      sh.tops[side][warp] = top[side];
    }
  }
}
// p, number by number, becomes max(p f - q g, 0); returns the sum.
__device__ __noinline__ double near_residual(float4* mine, int apart, int quads, float f, float g) {
  double sum = 0.0;
#pragma unroll 2
  for (int j = (int)(threadIdx.x & 31); j < quads; j += 32) {
    float4 p = mine[j];
    const float4 q = mine[apart + j];
    p = make_float4(fmaxf(fmaf(p.x, f, -(q.x * g)), 0.f), fmaxf(fmaf(p.y, f, -(q.y * g)), 0.f), fmaxf(fmaf(p.z, f, -(q.z * g)), 0.f),
                    fmaxf(fmaf(p.w, f, -(q.w * g)), 0.f));
    mine[j] = p;
    sum += (double)((p.x + p.y) + (p.z + p.w));
  }
  return warp_sum(sum);
}
// The weights of a range: from the logits once more, as they are in its warp's shared memory, for a test; or those themselves.
struct NearWeights {
  const Shared& sh;
  const float4* slices;
  int chunk;
  double scale, draft_scale;
  int n;
  struct InRange {
    float top, draft_top, c, draft_c;
    double factor, draft_factor;
    const double* steps;
    int n;
    template <int N>
    __device__ __forceinline__ void of(int, int, const float (&x)[N], const float (&y)[N], double (&p)[N]) const {
#pragma unroll
      for (int e = 0; e < N; e++) {
        float w = near_weight(x[e], top, c);
        if (n == 0) {
          p[e] = (double)w * factor;
          continue;
        }
        const float q = near_weight(y[e], draft_top, draft_c), g = (float)draft_factor;
#pragma unroll 1
        for (int k = 0; k < n; k++) w = fmaxf(fmaf(w, (float)(k ? steps[k] : steps[k] * factor), -(q * g)), 0.f);
        p[e] = (double)w;
      }
    }
    __device__ __forceinline__ double drafted(float y) const { return (double)near_weight(y, draft_top, draft_c) * draft_factor; }
  };
  // For a draw, in the shared memory of the CTA that has the range.
  struct Taken {
    uint32_t at;
    int i0;
    double factor;
    template <int N>
    __device__ __forceinline__ void take(const float*, const float*, int from, int hi, double (&p)[N]) const {
      float w[N];
#pragma unroll
      for (int e = 0; e < N; e++) {
        w[e] = 0.f;
        if (from + e < hi) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w[e]) : "r"(at + 4 * (from + e - i0)) : "memory");
      }
#pragma unroll
      for (int e = 0; e < N; e++) p[e] = (double)w[e] * factor;
    }
  };
  __device__ __forceinline__ Taken in(int range, const Cut& cut) const {
    return {cluster_at(slices + range % WARPS * chunk, range / WARPS), 4 * cut.first(range) - cut.before,
            n ? 1.0 : power(sh.all_tops[0][range], sh.command.top, scale, sh.table)};
  }
  __device__ __forceinline__ InRange in(int range) const {
    const Command& c = sh.command;
    InRange r = {sh.all_tops[0][range], sh.all_tops[1][range], (float)(scale / 16), (float)(draft_scale / 16), 0.0, 0.0, sh.steps, n};
    r.factor = power(r.top, c.top, scale, sh.table);
    r.draft_factor = power(r.draft_top, c.draft_top, draft_scale, sh.table) * c.draft_inverse;
    if (r.top == -INFINITY) r.top = 0.f;
    if (r.draft_top == -INFINITY) r.draft_top = 0.f;
    return r;
  }
};

// ------------------------------------------------------------------------------------------- both
constexpr int NEAR = -2;                           // a draw that is too near to a border
constexpr int32_t UNDECIDED = INT_MIN;           // `next` of a walk that the second kernel goes on with

// Sums of the lanes up to this one.
__device__ __forceinline__ double warp_scan(double x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, x, w);
    if (lane >= w) x += other;
  }
  return x;
}
// The first token whose running sum passes u times all of it, or -1 where nothing weighs anything; the ranges' sums are in `run`, and off by
// up to `error` in all (0: in 64 bits).  All threads of the leader: every warp finds the range, then each has neighbours of it.
// sh.found and sh.last are 0 before.
template <class W>
__device__ __noinline__ int drawn(Shared& sh, const W& every, const float* row, const float* draft, const Cut& cut, int vocab, int ranges, float uniform,
                                  double error) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const double u = (double)fminf(fmaxf(uniform, 0.f), 0.999999940395355f);      // (NaN: 0)
  constexpr int PER = RANGES_MOST / 32, N = 2;     // ranges of a lane, all of one CTA; tokens of a thread
  double mine[PER], sum = 0.0;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int r = lane * PER + k;
    mine[k] = r < ranges ? sh.run[r] * (every.n ? 1.0 : sh.part_factors[r / WARPS]) : 0.0;
    sum += mine[k];
  }
  double up = warp_scan(sum), before = up - sum;
  const double goal = u * __shfl_sync(0xffffffffu, up, 31);
  int range = -1;
  double base = 0.0;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    if (range < 0 && before + mine[k] > goal && mine[k] > 0.0) {
      range = lane * PER + k;
      base = before;
    }
    before += mine[k];
  }
  const unsigned have = __ballot_sync(0xffffffffu, range >= 0);
  if (!have) return error > 0.0 ? NEAR : -1;
  const int who = __ffs((int)have) - 1;
  range = __shfl_sync(0xffffffffu, range, who);
  base = __shfl_sync(0xffffffffu, base, who);
  const auto weights = every.in(range, cut);
  const int lo = cut.logit(cut.first(range)), hi = min(cut.logit(cut.first(range + 1)), vocab);
#pragma unroll 1
  for (int i0 = lo; i0 < hi; i0 += THREADS * N) {
    const int from = i0 + (int)threadIdx.x * N;
    double w[N];
    weights.take(row, draft, from, hi, w);
    const double scan = warp_scan(w[0] + w[1]);
    if (lane == 31) sh.warp_sums[warp] = scan;
    __syncthreads();
    double running = base + (scan - (w[0] + w[1]));
#pragma unroll 1
    for (int k = 0; k < WARPS; k++) {
      const double of_warp = sh.warp_sums[k];
      if (k < warp) running += of_warp;
      base += of_warp;
    }
    // the token that passes, the first the largest number; where roundings keep all from it, the last that weighs anything
    uint32_t passes = 0, last = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
      if (w[e] > 0.0) {
        last = (uint32_t)(from + e) + 1;
        if (!passes && running + w[e] > goal)
          passes = 2u * (uint32_t)((1 << 30) - (from + e)) + (error > 0.0 && (running + error > goal || running + w[e] < goal + error));
      }
      running += w[e];
    }
    passes = __reduce_max_sync(0xffffffffu, passes);
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0 && passes) atomicMax(&sh.found, passes);
    if (lane == 0 && last) atomicMax(&sh.last, last);
    __syncthreads();
    if (sh.found) break;
  }
  const uint32_t found = sh.found;
  if (!found) return error > 0.0 ? NEAR : (int)sh.last - 1;
  return found & 1 ? NEAR : (1 << 30) - (int)(found >> 1);
}

// The next child of new token `of` behind new token `after`, which has token `want` where `only` is set, or -1.  Every warp finds it.
__device__ __forceinline__ int child_of(const Shared& sh, int of, int after, int count, bool only = false, int want = 0) {
  for (int i0 = after + 1; i0 < count; i0 += 32) {
    const int i = i0 + (int)(threadIdx.x & 31);
    const unsigned is = __ballot_sync(0xffffffffu, i < count && sh.parents[i] == of && (!only || sh.tokens[i] == want));
    if (is) return i0 + __ffs((int)is) - 1;
  }
  return -1;
}

// A CTA's ranges, of `most` logits each, both sides at once, to the leader.  Warp 0.
__device__ __forceinline__ void to_leader(Shared& sh, const VerifyArgs& a, int rank, bool row, bool with_draft, int most) {
  const int lane = threadIdx.x & 31, side = lane / WARPS, r = lane % WARPS;
  Range its = nothing();
  if (side == 0 || with_draft) its = sh.mine[side][r];
  const double scale = side ? a.draft_scale : a.scale;
  // (the sides' scales may differ: exchanges between lanes are outside of what depends on them)
  const float top = group_max<WARPS>(its.top);
  const int first = group_min<WARPS>(its.top == top ? its.first : 0x7fffffff);
  if (row && scale == 0.0) its.sum = its.first == first && its.top > -INFINITY ? 1.0 : 0.0;
  else if (row) {
    const double f = power(its.top, top, scale, sh.table);
    // (E, where it is wanted; the logarithm is 2^-20 off, which the slack of 1.6 holds)
    if (its.sum > 0.0) its.off = its.sum * f * (1.6 / (1 << 22) + 2.2 / (1 << 24) * (double)fmaxf(__log2f((float)most / (float)its.sum), 0.f));
    its.sum *= f;
    cluster_put(&sh.all_tops[side][rank * WARPS + r], 0, its.top);
  }
  its.first = first;
  its.top = top;
  if (side == 0) cluster_put((row ? sh.run : sh.fresh) + rank * WARPS + r, 0, its.sum);
#pragma unroll
  for (int w = 1; w < WARPS; w <<= 1) {
    its.sum += __shfl_xor_sync(0xffffffffu, its.sum, w);
    its.off += __shfl_xor_sync(0xffffffffu, its.off, w);
    its.bad |= __shfl_xor_sync(0xffffffffu, its.bad, w);
  }
  if (r == 0) cluster_put(&sh.parts[side][rank], 0, its);
}

// Warp 0 of the leader: where the walk stands, and what the last pass has to say about it.
struct Walk {
  int at = 0, length = 1, child = 0, rejections = 0, next = -1;
  double total = 0.0, error = 0.0, draft_error = 0.0;
};

// FAST: in 32 bits.  Else, where a.goes_on, the walks that the other left undecided; all of them otherwise.
template <bool FAST>
__global__ void __launch_bounds__(THREADS, FAST ? 2 : 1) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
  extern __shared__ float4 slices[];               // logits: each warp's of the target, then of the draft
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x % (unsigned)a.parts), b = (int)(blockIdx.x / (unsigned)a.parts), ranges = a.parts * WARPS;
  const int ranges_shift = 31 - __clz(ranges);     // (a power of two)
  if (threadIdx.x < 16) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 16);
  if (threadIdx.x == 0) {
    sh.steps = reinterpret_cast<double*>(slices + (a.draft ? 2 : 1) * WARPS * a.chunk);
    sh.uniforms = reinterpret_cast<float*>(sh.steps + a.n_tokens);
    sh.tokens = reinterpret_cast<int*>(sh.uniforms + a.n_tokens);
    sh.parents = sh.tokens + a.n_tokens;
    sh.path = sh.parents + a.n_tokens;
  }
  __syncthreads();
  pdl_wait();
  Walk walk;
  if (!FAST && a.goes_on) {
    if (pdl_ld(a.next + b) != UNDECIDED) return;   // (all CTAs of the cluster)
    walk.length = pdl_ld(a.accepted + b);
    walk.at = pdl_ld(a.path + (int64_t)b * a.n_tokens + walk.length - 1);
  }
  int count = a.counts ? pdl_ld(a.counts + b) : a.n_tokens;
  if (count < 0 || count > a.n_tokens) {
    if (threadIdx.x == 0) a.status[WDC_STATUS_DRAFT] = 1;
    count = 0;
  }
  if (rank == 0 && walk.length > 1)
    for (int i = threadIdx.x; i < walk.length; i += THREADS) sh.path[i] = pdl_ld(a.path + (int64_t)b * a.n_tokens + i);
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const int64_t at = (int64_t)b * a.n_tokens + i;
    int parent = a.parents ? pdl_ld(a.parents + at) : i - 1;
    if (parent < -1 || parent >= i) {
      a.status[WDC_STATUS_DRAFT] = 1;
      parent = -1;
    }
    sh.parents[i] = parent;                        // (of every CTA: all of them know the first command)
    if (rank == 0) {
      sh.tokens[i] = pdl_ld(a.tokens + at);
      sh.uniforms[i] = a.uniforms ? pdl_ld(a.uniforms + at) : 0.f;
    }
  }
  __syncthreads();
  if (warp == 0) {
    Command c = {};
    c.todo = ROW;
    c.token = walk.at;
    c.guess = child_of(sh, walk.at, walk.at, count);
    c.with_draft = a.draft && c.guess >= 0;        // (the draft's row behind a token without children has no say)
    if (lane == 0) {
      sh.command = c;
      if (walk.length == 1 && a.n_tokens > 0) sh.path[0] = 0;
    }
  }
  cluster_sync();                                  // all CTAs of the cluster have begun

  float4* const mine = slices + warp * a.chunk;
  const int apart = WARPS * a.chunk;
#pragma unroll 1
  for (;;) {
    const int todo = sh.command.todo, standing = sh.command.token, with_draft = sh.command.with_draft;
    if (todo == STOP) break;
    const float* row = a.logits + b * a.logits_sb + standing * a.logits_st;
    const float* draft = a.draft ? a.draft + b * a.draft_sb + standing * a.draft_st : nullptr;
    const Cut cut(row, a.vocab, ranges_shift);
    const int first = cut.first(rank * WARPS + warp), quads = cut.first(rank * WARPS + warp + 1) - first, i0 = 4 * first - cut.before;
    const bool same = (reinterpret_cast<uintptr_t>(row) >> 2 & 3) == (reinterpret_cast<uintptr_t>(draft) >> 2 & 3);
    // The leader's next draft to test, and what the logits have for it: known before the pass, so that nothing waits for it behind it.
    float target_logit[1] = {0.f}, draft_logit[1] = {0.f};
    if (rank == 0 && warp == 0 && a.draft && count > 0) {
      walk.child = child_of(sh, standing, todo == ROW ? standing : walk.child, count);
      const int token = walk.child < 0 ? -1 : sh.tokens[walk.child];
      if (token >= 0 && token < a.vocab) {
        target_logit[0] = pdl_ld(row + token);
        draft_logit[0] = pdl_ld(draft + token);
      }
    }
    if (count == 0) {
    } else if (todo == ROW) {
      if (a.chunks == 1) {
#pragma unroll 1
        for (int side = 0; side <= (with_draft != 0); side++) fetch_quads(mine + side * apart, side ? draft : row, a.vocab, i0, quads, side == 0 || same);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
      }
      if constexpr (FAST) {
        if (with_draft) near_ranges<2>(sh, mine, apart, quads, a.scale, a.draft_scale);
        else near_ranges<1>(sh, mine, apart, quads, a.scale, a.draft_scale);
      } else {
#pragma unroll 1
        for (int side = 0; side <= (with_draft != 0); side++) {
          const Range r = row_range(mine + side * apart, side ? draft : row, a.vocab, i0, quads, a.chunk, a.chunks, side == 0 || same,
                                    side ? a.draft_scale : a.scale, sh.table);
          if (lane == 0) sh.mine[side][warp] = r;
        }
      }
    } else {
      // the rejection that has just been: its step is the last
      if (threadIdx.x == 0) sh.steps[with_draft - 1] = sh.command.step;
      __syncthreads();
      double sum;
      if constexpr (FAST) {
        // (the first time p is still relative to the range's largest)
        const Command& c = sh.command;
        const double f = with_draft > 1 ? c.step : c.step * power(sh.tops[0][warp], c.top, a.scale, sh.table);
        const double g = power(sh.tops[1][warp], c.draft_top, a.draft_scale, sh.table) * c.draft_inverse;
        sum = near_residual(mine, apart, quads, (float)f, (float)g);
      } else {
        const Weights weights = {sh.command, sh.table, sh.steps, a.scale, a.draft_scale, with_draft};
        sum = residual(mine, apart, row, draft, a.vocab, i0, quads, a.chunk, a.chunks, same, weights);
      }
      if (lane == 0) sh.mine[0][warp] = {sum, 0.0, 0.f, 0, 0, 0};
    }
    if (todo == ROW && sh.command.guess >= 0 && quads > 0) {
      // while the leader decides, the rows of the first child on their way to L2, a line a lane
      const int64_t from = 4 * (int64_t)first - cut.before, to = from + 4 * quads < a.vocab ? from + 4 * quads : a.vocab;
      for (int64_t i = (from > 0 ? from : 0) + lane * 32; i < to; i += 32 * 32) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(a.logits + b * a.logits_sb + sh.command.guess * a.logits_st + i));
        if (a.draft) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.draft + b * a.draft_sb + sh.command.guess * a.draft_st + i));
      }
    }
    __syncthreads();
    if (warp == 0 && count > 0) to_leader(sh, a, rank, todo == ROW, todo == ROW && with_draft, 4 * cut.each);
    cluster_sync();
    if (rank == 0) {
      Command c = {};                              // (of warp 0, which decides; all threads draw)
      bool test = false, near = false;             // near: a decision that 32 bits do not make
      if (warp == 0) {
        c = sh.command;
        c.todo = STOP;
        int draw = -1;
        if (count > 0) {
          // the CTAs' parts, both sides at once
          const int side = lane / PARTS_MOST & 1, part = lane % PARTS_MOST;
          const bool there = lane < 2 * PARTS_MOST && part < a.parts && (side == 0 || (todo == ROW && with_draft));
          Range its = nothing();
          if (there) its = sh.parts[side][part];
          const double scale = side ? a.draft_scale : a.scale;
          const float top = group_max<PARTS_MOST>(its.top);
          const int first_of_all = group_min<PARTS_MOST>(its.top == top ? its.first : 0x7fffffff);
          double f = 1.0;
          if (todo == ROW) {
            f = scale == 0.0 ? (double)(its.first == first_of_all && its.top > -INFINITY) : power(its.top, top, scale, sh.table);
            if (there && side == 0) sh.part_factors[part] = f;
          }
          its.sum *= f;
          its.off *= f;
#pragma unroll
          for (int w = 1; w < PARTS_MOST; w <<= 1) {
            its.sum += __shfl_xor_sync(0xffffffffu, its.sum, w);
            if (FAST) its.off += __shfl_xor_sync(0xffffffffu, its.off, w);
            its.bad |= __shfl_xor_sync(0xffffffffu, its.bad, w);
          }
          const double total = __shfl_sync(0xffffffffu, its.sum, 0), draft_total = __shfl_sync(0xffffffffu, its.sum, PARTS_MOST);
          if (todo == ROW) {
            const bool none = __any_sync(0xffffffffu, lane < (with_draft ? 2 : 1) * PARTS_MOST && (its.bad || top == -INFINITY));
            c.first = __shfl_sync(0xffffffffu, first_of_all, 0);
            c.top = __shfl_sync(0xffffffffu, top, 0);
            c.draft_first = __shfl_sync(0xffffffffu, first_of_all, PARTS_MOST);
            c.draft_top = __shfl_sync(0xffffffffu, top, PARTS_MOST);
            c.draft_inverse = with_draft ? 1.0 / draft_total : 1.0;
            walk.total = total;
            if (FAST) {
              walk.error = __shfl_sync(0xffffffffu, its.off, 0);
              walk.draft_error = 2 * __shfl_sync(0xffffffffu, its.off, PARTS_MOST) * c.draft_inverse + 4.0 / (1 << 24);
            }
            walk.rejections = 0;
            test = !none && a.draft;
            if (!none && !a.draft) draw = standing;
          } else {
            if (FAST) {
              walk.error = 2 * walk.error / walk.total + walk.draft_error + 8.0 / (1 << 24);
              near = !(total > 4 * walk.error);
            }
            if (total > 0.0) {
              for (int r = lane; r < ranges; r += 32) sh.run[r] = sh.fresh[r];
              walk.total = total;
              walk.rejections = with_draft;
            }
            test = !near;
          }
          if (test && walk.child < 0) draw = 0;
        }
        __syncwarp();
        if (lane == 0) {
          sh.command = c;                          // (for the weights below; told to the others at the end)
          sh.command.with_draft = walk.rejections;
          sh.draw = draw;
          sh.draw_error = walk.error;
          sh.found = sh.last = 0;
        }
        __syncwarp();
      }
      __syncthreads();
      if (sh.draw >= 0) {
        int token;
        if constexpr (FAST) {
          const NearWeights weights = {sh, slices, a.chunk, a.scale, a.draft_scale, sh.command.with_draft};
          token = drawn(sh, weights, row, draft, cut, a.vocab, ranges, sh.uniforms[sh.draw], sh.draw_error);
        } else {
          const Weights weights = {sh.command, sh.table, sh.steps, a.scale, a.draft_scale, sh.command.with_draft};
          token = drawn(sh, weights, row, draft, cut, a.vocab, ranges, sh.uniforms[sh.draw], 0.0);
        }
        if (warp == 0) {
          near = token == NEAR;
          walk.child = token < 0 || a.draft ? -1 : child_of(sh, standing, standing, count, true, token);
          if (near) {
          } else if (walk.child < 0) {
            walk.next = token;
          } else {
            walk.at = walk.child;
            c.todo = ROW;
          }
        }
      } else if (test) {
        const int token = sh.tokens[walk.child];
        const double u = (double)fminf(fmaxf(sh.uniforms[walk.child], 0.f), 0.999999940395355f);
        bool stands = false;
        if (token >= 0 && token < a.vocab) {
          double p[1], q[1];
          if constexpr (FAST) {
            const NearWeights weights = {sh, slices, a.chunk, a.scale, a.draft_scale, walk.rejections};
            const auto its = weights.in((token + cut.before) / 4 / cut.each);
            its.of(token, 1, target_logit, draft_logit, p);
            q[0] = its.drafted(draft_logit[0]);
            near = fabs(u * q[0] * walk.total - p[0]) <= 2 * walk.error + walk.total * walk.draft_error;
          } else {
            const Weights weights = {sh.command, sh.table, sh.steps, a.scale, a.draft_scale, walk.rejections};
            weights.of(token, 1, target_logit, draft_logit, p);
            weights.drafted(token, 1, draft_logit, q);
          }
          stands = u * q[0] * walk.total < p[0];
        }
        if (near) {
        } else if (stands) {
          walk.at = walk.child;
          c.todo = ROW;
        } else {
          c.todo = RESIDUAL;
          c.with_draft = walk.rejections + 1;
          c.step = 1.0 / walk.total;
        }
      }
      if (warp == 0) {
        if (near) walk.next = UNDECIDED;           // (and STOP)
        if (c.todo == ROW) {
          c.token = walk.at;
          c.guess = child_of(sh, walk.at, walk.at, count);
          c.with_draft = a.draft && c.guess >= 0;
          if (lane == 0) sh.path[walk.length] = walk.at;
          walk.length++;
        }
        __syncwarp();
        if (lane < a.parts) cluster_put(&sh.command, lane, c);
      }
    }
    cluster_sync();
  }
  if (rank != 0 || warp != 0) return;
  __syncwarp();
  for (int i = lane; i < a.n_tokens; i += 32) a.path[(int64_t)b * a.n_tokens + i] = count > 0 && i < walk.length ? sh.path[i] : -1;
  if (lane == 0) {
    a.accepted[b] = count > 0 ? walk.length : 0;
    a.next[b] = walk.next;
  }
}

}  // namespace

extern "C" int wdc_verify_drafts(wdc_context* ctx, const wdc_verify_desc* d, const float* logits, const float* draft_logits,
                                 const int32_t* tokens, const int32_t* parents, const int32_t* counts, const float* uniforms,
                                 int32_t* path, int32_t* accepted, int32_t* next) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_verify_drafts: null context");
  WDC_TAPE(ctx, wdc_verify_drafts, tape_desc(d), logits, draft_logits, tokens, parents, counts, uniforms, path, accepted, next);
  wdc_note_write(ctx, path);
  wdc_note_write(ctx, accepted);
  wdc_note_write(ctx, next);
  const char* who = "wdc_verify_drafts";
  WDC_REQUIRE(ctx, d, "%s: null argument", who);
  WDC_REQUIRE(ctx, d->batch >= 0 && d->tokens >= 0 && d->vocab > 0 && d->logits_sb >= 0 && d->logits_st >= 0 && d->draft_sb >= 0 &&
              d->draft_st >= 0, "%s: bad shape", who);
  if (d->batch > 65535 || d->tokens > TOKENS_MOST || d->vocab >= 1ll << 30)
    return wdc_fail(ctx, WDC_ERR_UNSUPPORTED, "%s: %lld sequences of %lld tokens of %lld (up to 65535, %d, 2^30 - 1)", who, (long long)d->batch,
                    (long long)d->tokens, (long long)d->vocab, TOKENS_MOST);
  for (const float t : {d->temperature, d->draft_temperature})
    WDC_REQUIRE(ctx, t == 0.f || (t >= 1e-6f && t <= 1e6f), "%s: a temperature is 0, or 1e-6 to 1e6", who);
  if (d->batch == 0) return WDC_OK;
  WDC_REQUIRE(ctx, accepted && next && (d->tokens == 0 || (logits && tokens && path && (uniforms || (d->temperature == 0.f && !draft_logits)))),
              "%s: null argument", who);
  for (const void* p : {(const void*)logits, (const void*)draft_logits, (const void*)tokens, (const void*)parents, (const void*)counts,
                        (const void*)uniforms, (const void*)path, (const void*)accepted, (const void*)next})
    WDC_REQUIRE(ctx, (reinterpret_cast<uintptr_t>(p) & 3u) == 0, "%s: buffers are not aligned", who);
  // (the second kernel reads what the first has read, after that has written its results)
  const int64_t per_row = d->batch * d->tokens, row_end = d->tokens ? d->vocab : 0;
  const auto extent = [&](int64_t sb, int64_t st) { return row_end ? (d->batch - 1) * sb + (d->tokens - 1) * st + row_end : 0; };
  struct Words {
    const void* at;
    int64_t n;
  };
  const Words used[9] = {{path, per_row}, {accepted, d->batch}, {next, d->batch}, {tokens, per_row}, {parents, per_row}, {counts, d->batch}, {uniforms, per_row},
                         {logits, extent(d->logits_sb, d->logits_st)}, {draft_logits, extent(d->draft_sb, d->draft_st)}};
  for (int i = 0; i < 3; i++)
    for (int j = i + 1; j < 9; j++) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(used[i].at), y = reinterpret_cast<uintptr_t>(used[j].at);
      WDC_REQUIRE(ctx, !x || !y || x + 4 * used[i].n <= y || y + 4 * used[j].n <= x, "%s: a result overlaps another buffer", who);
    }
  VerifyArgs a = {logits, draft_logits, uniforms, tokens, parents, counts, path, accepted, next, ctx->status_word,
                  d->logits_sb, d->logits_st, d->draft_sb, d->draft_st, (int)d->tokens, (int)d->vocab, 1, 0, 1, 1, 0.0, 0.0};
  const double to16 = 16 * 1.4426950408889634;     // 16 log2(e)
  if (d->temperature > 0.f) a.scale = to16 / d->temperature;
  if (d->draft_temperature > 0.f) a.draft_scale = to16 / d->draft_temperature;
  // CTAs of a sequence: as many as fill the SMs once, of enough logits each.  Measured, us of 1 / 2 / 4 / 8, drafts with their logits: one sequence, 4000
  // in the vocabulary, 20.2 / 18.8 / 18.5 / 18.6, 16000 34.5 / 34.6 / 30.7 / 28.1; 64 of 12000 88 / 74 / 78 / 97; 200 of 12000 75 / 76 / 110 / 176.
  while (a.parts < PARTS_MOST && 2 * d->batch * a.parts <= ctx->sm_count && d->vocab / (2 * a.parts) >= PART_LEAST) a.parts *= 2;
  // Shared memory for the logits of a warp's range, by more CTAs if need be; or for as many of them as there is room for.
  const int sides = draft_logits ? 2 : 1;
  const int64_t most = (SLICE_BYTES - TOKEN_BYTES * d->tokens) / (16 * WARPS * sides);
  const auto each = [&]() { return ceil_div64((d->vocab + 6) / 4, a.parts * WARPS); };
  const int parts = a.parts;
  while (a.parts < PARTS_MOST && each() > most) a.parts *= 2;
  if (each() > most) a.parts = parts;
  a.chunk = (int)(each() < most ? each() : most);
  a.chunks = (int)ceil_div64(each(), a.chunk);
  DeviceGuard g(ctx->device);
  static bool opted_in[64] = {};     // per device: more than 48 KB of dynamic shared memory needs the attribute
  WDC_REQUIRE(ctx, ctx->device >= 0 && ctx->device < 64, "%s: device index out of range", who);
  if (!opted_in[ctx->device]) {
    WDC_CUDA(ctx, cudaFuncSetAttribute(verify_drafts_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SLICE_BYTES));
    WDC_CUDA(ctx, cudaFuncSetAttribute(verify_drafts_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SLICE_BYTES));
    opted_in[ctx->device] = true;
  }
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS);
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
  cfg.numAttrs++;
  if (ctx->opt_pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs++;
  }
  const auto shape = [&]() {
    cfg.gridDim = dim3((unsigned)(d->batch * a.parts));
    cfg.dynamicSmemBytes = (size_t)(16 * WARPS * sides) * a.chunk + TOKEN_BYTES * d->tokens;
    attr[0].val.clusterDim.x = (unsigned)a.parts;
  };
  shape();
  // In 32 bits first, where all of a row's weights have room and there is something to weigh; then what that left undecided.
  if (a.chunks == 1 && d->temperature > 0.f && (!draft_logits || d->draft_temperature > 0.f)) {
    WDC_CUDA(ctx, cudaLaunchKernelEx(&cfg, verify_drafts_kernel<true>, a));
    CACHE_TRY(wdc_check_launch(ctx, "verify_drafts_kernel"));
    // (few walks have anything left to do, so that each may have many CTAs; the others pay for CTAs that begin, one an SM, and leave: of
    // 50001 tokens 3 us for one sequence, 4 for 16, 6 for 64)
    a.goes_on = 1;
    while (a.parts < PARTS_MOST && d->vocab / (2 * a.parts) >= PART_LEAST) a.parts *= 2;
    a.chunk = (int)each();
    shape();
  }
  WDC_CUDA(ctx, cudaLaunchKernelEx(&cfg, verify_drafts_kernel<false>, a));
  return wdc_check_launch(ctx, "verify_drafts_kernel");
}
