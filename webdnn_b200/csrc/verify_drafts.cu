// Which drafted tokens of a tree stand, and the token that follows them (wdc_verify_drafts).  The reference has no such operator: its
// graphs end at Softmax (operators/cpu/operators/standard/softmax.ts:15-59).
//
// The walk from token to token is serial, and only the rows of logits that it comes by are needed.  A cluster of CTAs takes a
// sequence: each warp of it has a range of the vocabulary, whose maximum and sum of exponentials it finds in one pass; the first CTA
// (the leader) joins them, tests or draws, and tells the others what to do next.
//
// A drawn token is the one in whose range of the running sum a number falls, and with 100000 tokens there are borders everywhere: sums that
// are 2^-22 of the whole off would name another token in several of a hundred draws.  So weights and sums are in 64 bits.  Their
// exponential is 2^(n / 16) from a table times a polynomial in what is left, 11 operations in all.  At an SM's 64 lanes that is 0.17
// cycles a logit, what reading it takes (0.17 at 24 bytes a cycle and SM).
#include <math.h>

#include "paged_cache.cuh"

namespace {

constexpr int WARPS = 16, THREADS = 32 * WARPS, PARTS_MOST = 8, RANGES_MOST = WARPS * PARTS_MOST;
constexpr int EACH = 4;                            // float4 a lane that are on their way
constexpr int TOKENS_MOST = 1024;
constexpr int PART_LEAST = 2048;                   // logits of a CTA, where a row is cut into several

struct VerifyArgs {
  const float *logits, *draft, *uniforms;
  const int32_t *tokens, *parents, *counts;
  int32_t *path, *accepted, *next;
  int* status;
  int64_t logits_sb, logits_st, draft_sb, draft_st;
  int n_tokens, vocab, parts;
  double scale, draft_scale;                       // 16 log2(e) / temperature; 0: temperature 0
};

// What a range of a row (or all of it) has: the largest logit, the sum of 2^((x - top) scale / 16), or where the first of the largest
// is; whether there is a NaN or +inf.
struct Range {
  double sum;
  float top;
  int first, bad;
};
enum Todo { STOP = 0, ROW = 1, RESIDUAL = 2 };
struct Command {
  int todo, token;                                 // the token that the walk stands at
  int with_draft, first, draft_first;
  float top, draft_top;
  double draft_inverse, step;                      // 1 / sum of the draft's weights, of those before the last rejection
};
struct Shared {
  double table[16];
  double steps[TOKENS_MOST];                       // 1 / the sums that a rejection divided by
  Command command;
  // of the leader
  Range ranges[2][RANGES_MOST];                    // target and draft
  double run[RANGES_MOST], fresh[RANGES_MOST];     // sums of the ranges, all relative to one maximum; after the last rejection
  double warp_sums[WARPS];
  float uniforms[TOKENS_MOST];
  int tokens[TOKENS_MOST], parents[TOKENS_MOST], path[TOKENS_MOST];
  int found, child;
};

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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// 2^(d scale / 16) for d <= 0, within 2^-42 of it; 0 where that is below 2^-1000 (d is -inf or NaN).  n is the nearest whole number
// to d scale, which adding 1.5 * 2^52 leaves in the last bits; 2^(g / 16), |g| <= 1/2, by five terms of its series.
__device__ __forceinline__ double power(float x, float top, double scale, const double* table) {
  const double magic = 6755399441055744.0, u = 0.043321698784996582;           // ln(2) / 16
  const double d = (double)x - (double)top, shifted = fma(d, scale, magic), g = fma(d, scale, magic - shifted);
  const int n = __double2loint(shifted);
  double p = u * u * u * u * u / 120;
  p = fma(p, g, u * u * u * u / 24);
  p = fma(p, g, u * u * u / 6);
  p = fma(p, g, u * u / 2);
  p = fma(p, g, u);
  const double t = table[n & 15], y = fma(t, p * g, t);
  const double out = __hiloint2double(__double2hiint(y) + ((n >> 4) << 20), __double2loint(y));
  return (x - top) * (float)scale > -16000.f ? out : 0.0;
}

__device__ __forceinline__ Range joined(Range a, const Range& b, double scale, const double* table) {
  const float top = fmaxf(a.top, b.top);
  if (scale == 0.0) {
    if (b.top > a.top || (b.top == a.top && b.first < a.first)) a.first = b.first;
  } else {
    a.sum = a.sum * (a.top < top ? power(a.top, top, scale, table) : 1.0) + b.sum * (b.top < top ? power(b.top, top, scale, table) : 1.0);
  }
  a.top = top;
  a.bad |= b.bad;
  return a;
}
__device__ __forceinline__ Range warp_joined(Range a, double scale, const double* table) {
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    Range b;
    b.sum = __shfl_xor_sync(0xffffffffu, a.sum, w);
    b.top = __shfl_xor_sync(0xffffffffu, a.top, w);
    b.first = __shfl_xor_sync(0xffffffffu, a.first, w);
    b.bad = __shfl_xor_sync(0xffffffffu, a.bad, w);
    a = joined(a, b, scale, table);
  }
  return a;
}

// How a row is cut: float4 number j has logits 4 j - before .. + 3 (`before`: how far the row is behind a 16-byte boundary), and a
// warp has `each` float4 of them.
struct Cut {
  int before, quads, each;
  __device__ Cut(const float* row, int vocab, int ranges) {
    before = (int)(reinterpret_cast<uintptr_t>(row) >> 2 & 3);
    quads = (int)(((int64_t)vocab + before + 3) / 4);
    each = (quads + ranges - 1) / ranges;
  }
  __device__ int first(int range) const { return (int)min((int64_t)range * each, (int64_t)quads); }
  __device__ int logit(int quad) const { return max(4 * quad - before, 0); }
};

__device__ Range row_range(const float* row, int vocab, int range, int ranges, double scale, const double* table) {
  const Cut cut(row, vocab, ranges);
  const int lane = threadIdx.x & 31, end = cut.first(range + 1);
  Range r = {0.0, -INFINITY, 0x7fffffff, 0};
  for (int j0 = cut.first(range) + lane; j0 < end; j0 += 32 * EACH) {
    float x[EACH][4];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const int j = j0 + e * 32, i = 4 * j - cut.before;
      if (j < end && i >= 0 && i + 3 < vocab) {
        const float4 v = pdl_ld(reinterpret_cast<const float4*>(row + i));
        x[e][0] = v.x; x[e][1] = v.y; x[e][2] = v.z; x[e][3] = v.w;
      } else {
#pragma unroll
        for (int c = 0; c < 4; c++) x[e][c] = j < end && i + c >= 0 && i + c < vocab ? pdl_ld(row + i + c) : -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const float top = fmaxf(fmaxf(x[e][0], x[e][1]), fmaxf(x[e][2], x[e][3]));
#pragma unroll
      for (int c = 0; c < 4; c++) r.bad |= !(x[e][c] < INFINITY);
      if (top > r.top) {
        if (scale == 0.0)
          r.first = 4 * (j0 + e * 32) - cut.before + (x[e][0] == top ? 0 : x[e][1] == top ? 1 : x[e][2] == top ? 2 : 3);
        else
          r.sum *= power(r.top, top, scale, table);
        r.top = top;
      }
      if (scale != 0.0) {
#pragma unroll
        for (int c = 0; c < 4; c++) r.sum += power(x[e][c], r.top, scale, table);
      }
    }
  }
  return warp_joined(r, scale, table);
}

// The weight of one token under the target's distribution after `n` rejections, not normalised.
struct Weights {
  const float *row, *draft;
  double scale, draft_scale;
  const Shared* sh;
  int n;
  __device__ double draft_at(int i) const {
    const Command& c = sh->command;
    return draft_scale == 0.0 ? (double)(i == c.draft_first) : power(pdl_ld(draft + i), c.draft_top, draft_scale, sh->table) * c.draft_inverse;
  }
  __device__ double at(int i) const {
    const Command& c = sh->command;
    double p = scale == 0.0 ? (double)(i == c.first) : power(pdl_ld(row + i), c.top, scale, sh->table);
    if (n) {
      const double q = draft_at(i);
      for (int k = 0; k < n; k++) p = fmax(fma(p, sh->steps[k], -q), 0.0);
    }
    return p;
  }
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}

// The first token whose running sum passes u times all of it; the ranges' sums are in `run`.  All threads of the leader.
__device__ int drawn(Shared& sh, const Weights& weights, const Cut& cut, int vocab, int ranges, float uniform) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const double u = (double)fminf(fmaxf(uniform, 0.f), 0.999999940395355f);      // (NaN: 0)
  if (threadIdx.x == 0) sh.found = -1;
  // every warp finds the range: lane l has ranges l * per .. of it
  constexpr int PER = RANGES_MOST / 32;
  double mine[PER], sum = 0.0;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    mine[k] = lane * PER + k < ranges ? sh.run[lane * PER + k] : 0.0;
    sum += mine[k];
  }
  double up = sum;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, up, w);
    if (lane >= w) up += other;
  }
  const double goal = u * __shfl_sync(0xffffffffu, up, 31);
  double before = __shfl_up_sync(0xffffffffu, up, 1);
  if (lane == 0) before = 0.0;
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
  const int who = have ? __ffs((int)have) - 1 : 0;
  range = __shfl_sync(0xffffffffu, range, who);
  base = __shfl_sync(0xffffffffu, base, who);
  __syncthreads();
  if (range < 0) return -1;                        // (nothing weighs anything)
  // its tokens, a few neighbours each thread
  const int lo = cut.logit(cut.first(range)), hi = min(cut.logit(cut.first(range + 1)), vocab);
  const int per = (hi - lo + THREADS - 1) / THREADS, from = lo + (int)threadIdx.x * per, to = min(from + per, hi);
  double own = 0.0;
  for (int i = from; i < to; i++) own += weights.at(i);
  double scan = own;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, scan, w);
    if (lane >= w) scan += other;
  }
  if (lane == 31) sh.warp_sums[warp] = scan;
  __syncthreads();
  double running = base;
  for (int w = 0; w < warp; w++) running += sh.warp_sums[w];
  const double shifted = __shfl_up_sync(0xffffffffu, scan, 1);
  running += lane ? shifted : 0.0;
  // the token that passes; where roundings of 2^-53 keep all from it, the last that weighs anything
  int token = -1, last = -1;
  for (int i = from; i < to; i++) {
    const double w = weights.at(i);
    running += w;
    if (w > 0.0) {
      last = i;
      if (token < 0 && running > goal) token = i;
    }
  }
  const unsigned passes = __ballot_sync(0xffffffffu, token >= 0);
  // (found: tokens that pass count down from 2^30, so that the first is the largest, and are above all that do not)
  if (passes && lane == __ffs((int)passes) - 1) atomicMax(&sh.found, (1 << 30) + ((1 << 30) - 1 - token));
  else if (!passes) {
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0 && last >= 0) atomicMax(&sh.found, last);
  }
  __syncthreads();
  const int found = sh.found;
  __syncthreads();
  return found >= 1 << 30 ? (1 << 30) - 1 - (found - (1 << 30)) : found;
}

// The next child of new token `of` behind new token `after`, which has token `want` where `only` is set, or -1.  All threads of the
// leader.
__device__ int child_of(Shared& sh, int of, int after, int count, bool only = false, int want = 0) {
  __syncthreads();
  if (threadIdx.x == 0) sh.child = 0x7fffffff;
  __syncthreads();
  for (int i = after + 1 + (int)threadIdx.x; i < count; i += THREADS)
    if (sh.parents[i] == of && (!only || sh.tokens[i] == want)) {
      atomicMin(&sh.child, i);
      break;
    }
  __syncthreads();
  const int child = sh.child;
  return child == 0x7fffffff ? -1 : child;
}

__global__ void __launch_bounds__(THREADS, 2) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x % (unsigned)a.parts), b = (int)(blockIdx.x / (unsigned)a.parts), ranges = a.parts * WARPS;
  if (threadIdx.x < 16) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 16);
  pdl_wait();
  int count = a.counts ? pdl_ld(a.counts + b) : a.n_tokens;
  if (count < 0 || count > a.n_tokens) {
    if (threadIdx.x == 0) a.status[WDC_STATUS_DRAFT] = 1;
    count = 0;
  }
  if (threadIdx.x == 0) {
    Command c = {};
    c.todo = ROW;
    c.with_draft = a.draft && count > 1;
    sh.command = c;
  }
  if (rank == 0) {
    for (int i = threadIdx.x; i < count; i += THREADS) {
      const int64_t at = (int64_t)b * a.n_tokens + i;
      int parent = a.parents ? pdl_ld(a.parents + at) : i - 1;
      if (parent < -1 || parent >= i) {
        a.status[WDC_STATUS_DRAFT] = 1;
        parent = -1;
      }
      sh.parents[i] = parent;
      sh.tokens[i] = pdl_ld(a.tokens + at);
      sh.uniforms[i] = a.uniforms ? pdl_ld(a.uniforms + at) : 0.f;
    }
  }
  cluster_sync();                                  // all CTAs of the cluster have begun

  // of the leader
  int at = 0, length = 1, child = 0, rejections = 0, next = -1;
  double total = 0.0;
  if (rank == 0 && threadIdx.x == 0) sh.path[0] = 0;
  for (;;) {
    const Command now = sh.command;
    if (now.todo == STOP) break;
    const float* row = a.logits + b * a.logits_sb + now.token * a.logits_st;
    const float* draft = a.draft ? a.draft + b * a.draft_sb + now.token * a.draft_st : nullptr;
    const int range = rank * WARPS + warp;
    if (now.todo == ROW) {
      if (count > 0) {
        const Range r = row_range(row, a.vocab, range, ranges, a.scale, sh.table);
        if (lane == 0) cluster_put(&sh.ranges[0][range], 0, r);
        if (now.with_draft) {
          const Range q = row_range(draft, a.vocab, range, ranges, a.draft_scale, sh.table);
          if (lane == 0) cluster_put(&sh.ranges[1][range], 0, q);
        }
      }
    } else {
      // the rejection that has just been: its step is the last
      if (threadIdx.x == 0) sh.steps[now.with_draft - 1] = now.step;
      __syncthreads();
      const Weights weights = {row, draft, a.scale, a.draft_scale, &sh, now.with_draft};
      const Cut cut(row, a.vocab, ranges);
      const int hi = min(cut.logit(cut.first(range + 1)), a.vocab);
      double sum = 0.0;
#pragma unroll 4
      for (int i = cut.logit(cut.first(range)) + lane; i < hi; i += 32) sum += weights.at(i);
      sum = warp_sum(sum);
      if (lane == 0) cluster_put(&sh.fresh[range], 0, sum);
    }
    cluster_sync();
    if (rank == 0) {
      Command c = now;
      c.todo = STOP;
      const Cut cut(row, a.vocab, ranges);
      bool test = false;                           // whether drafts of `at` are to be tried
      if (now.todo == ROW && count > 0) {
        // every warp joins the ranges
        Range p = {0.0, -INFINITY, 0x7fffffff, 0}, q = p;
        for (int r = lane; r < ranges; r += 32) {
          p = joined(p, sh.ranges[0][r], a.scale, sh.table);
          if (now.with_draft) q = joined(q, sh.ranges[1][r], a.draft_scale, sh.table);
        }
        p = warp_joined(p, a.scale, sh.table);
        q = warp_joined(q, a.draft_scale, sh.table);
        const bool none = p.bad || p.top == -INFINITY || (now.with_draft && (q.bad || q.top == -INFINITY));
        __syncthreads();
        for (int r = threadIdx.x; r < ranges; r += THREADS) {
          const Range mine = sh.ranges[0][r];
          sh.run[r] = a.scale == 0.0 ? (mine.top == p.top && mine.first == p.first ? 1.0 : 0.0) : mine.top == -INFINITY ? 0.0
                                     : mine.sum * (mine.top < p.top ? power(mine.top, p.top, a.scale, sh.table) : 1.0);
        }
        total = a.scale == 0.0 ? 1.0 : p.sum;
        c.first = p.first; c.top = p.top;
        c.draft_first = q.first; c.draft_top = q.top;
        c.draft_inverse = a.draft_scale == 0.0 ? 1.0 : 1.0 / q.sum;
        c.with_draft = rejections = 0;
        __syncthreads();
        if (threadIdx.x == 0) sh.command = c;      // (for the weights below; told to the others at the end)
        __syncthreads();
        if (!none && a.draft) {
          child = child_of(sh, at, at, count);
          test = true;
        } else if (!none) {
          const Weights weights = {row, draft, a.scale, a.draft_scale, &sh, 0};
          const int token = a.scale == 0.0 ? p.first : drawn(sh, weights, cut, a.vocab, ranges, sh.uniforms[at]);
          child = child_of(sh, at, at, count, true, token);
          if (child < 0) {
            next = token;
          } else {
            at = child;
            c.todo = ROW;
          }
        }
      } else if (now.todo == RESIDUAL) {
        double sum = 0.0;
        for (int r = lane; r < ranges; r += 32) sum += sh.fresh[r];
        sum = warp_sum(sum);
        __syncthreads();
        if (sum > 0.0) {
          for (int r = threadIdx.x; r < ranges; r += THREADS) sh.run[r] = sh.fresh[r];
          total = sum;
          rejections = now.with_draft;
        }
        child = child_of(sh, at, child, count);
        test = true;
      }
      if (test) {
        const Weights weights = {row, draft, a.scale, a.draft_scale, &sh, rejections};
        if (child < 0) {
          next = drawn(sh, weights, cut, a.vocab, ranges, sh.uniforms[0]);
        } else {
          const int token = sh.tokens[child];
          const bool there = token >= 0 && token < a.vocab;
          const double u = (double)fminf(fmaxf(sh.uniforms[child], 0.f), 0.999999940395355f);
          if (there && u * weights.draft_at(token) * total < weights.at(token)) {
            at = child;
            c.todo = ROW;
          } else {
            c.todo = RESIDUAL;
            c.with_draft = rejections + 1;
            c.step = 1.0 / total;
          }
        }
      }
      if (c.todo == ROW) {
        c.token = at;
        if (threadIdx.x == 0) sh.path[length] = at;
        length++;
        c.with_draft = a.draft && child_of(sh, at, at, count) >= 0;
      }
      __syncthreads();
      if (threadIdx.x < a.parts) cluster_put(&sh.command, (int)threadIdx.x, c);
    }
    cluster_sync();
  }
  if (rank != 0) return;
  for (int i = threadIdx.x; i < a.n_tokens; i += THREADS)
    a.path[(int64_t)b * a.n_tokens + i] = count > 0 && i < length ? sh.path[i] : -1;
  if (threadIdx.x == 0) {
    a.accepted[b] = count > 0 ? length : 0;
    a.next[b] = next;
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
  VerifyArgs a = {logits, draft_logits, uniforms, tokens, parents, counts, path, accepted, next, ctx->status_word,
                  d->logits_sb, d->logits_st, d->draft_sb, d->draft_st, (int)d->tokens, (int)d->vocab, 1, 0.0, 0.0};
  const double to16 = 16 * 1.4426950408889634;     // 16 log2(e)
  if (d->temperature > 0.f) a.scale = to16 / d->temperature;
  if (d->draft_temperature > 0.f) a.draft_scale = to16 / d->draft_temperature;
  while (a.parts < PARTS_MOST && d->batch * a.parts < ctx->sm_count && d->vocab / (2 * a.parts) >= PART_LEAST) a.parts *= 2;
  DeviceGuard g(ctx->device);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d->batch * a.parts));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.x = (unsigned)a.parts;
  attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
  cfg.numAttrs++;
  if (ctx->opt_pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs++;
  }
  WDC_CUDA(ctx, cudaLaunchKernelEx(&cfg, verify_drafts_kernel, a));
  return wdc_check_launch(ctx, "verify_drafts_kernel");
}
