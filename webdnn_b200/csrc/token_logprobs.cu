// Log probabilities of given tokens under softmax(logits), the distribution's entropy and its best alternatives.  The
// reference has no such operator: its graphs end at Softmax (operators/cpu/operators/standard/softmax.ts:15-59).
#include <math.h>

#include "tape.cuh"

namespace {

constexpr int EACH = 4;                                        // float4 a thread and round
constexpr int WARPS_MOST = 8, SM_WARPS = 24;                   // of a CTA; of an SM (80 registers a thread)
constexpr int TOP_MOST = 32, PARTS_MOST = 8;
// Which best are wanted: none, some, or many of a row of few rounds.  In the first round then most threads have candidates, and the
// kernel looks at all of them at once (3 x 384 with 32: 5.8 against 8.4 us); its code is too long for the other kernel to have it as
// well (3000 x 50001 with 1: 116 against 106).
enum { NONE = 0, SOME = 1, MANY = 2 };
constexpr int MANY_TOP = 9, MANY_ROUNDS = 2;
constexpr int PART_LEAST = 4096;                               // logits of a part, where a row is cut into several

struct LogprobArgs {
  const float* logits;
  const int32_t* tokens;
  float *logprob, *entropy, *top_logprobs;
  int32_t* top_ids;
  int64_t row_stride;
  int vocab, top, parts;
};

// A key that orders by value, NaN above everything and -0 as 0, then by the lower index.  No key is 0 or ~0, which stand below and
// above all of them.
__device__ __forceinline__ uint64_t order_key(float x, int index) {
  uint32_t bits = x == x ? __float_as_uint(x + 0.f) : 0x7fc00000u;
  bits = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return (uint64_t)bits << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t bits = (uint32_t)(key >> 32);
  return __uint_as_float(bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
}
__device__ __forceinline__ float exp_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

// s + c = sum e^(x - m), t = sum (x - m) e^(x - m).  c has what the additions to s rounded off: a sum is often 1 and many terms too
// small for it.  A difference below -200, whose exponential is 0, counts as -200 in t: it may be infinite, and infinity times 0 is
// NaN.  A NaN or +inf makes s NaN.
struct Sums {
  float m, s, c, t;
};
__device__ __forceinline__ void raise_to(Sums& a, float m) {
  if (m > a.m) {
    const float d = a.m - m, f = exp_of(d);
    a.t = f * fmaf(a.s, fmaxf(d, -200.f), a.t);
    a.s *= f;
    a.c *= f;
    a.m = m;
  }
}
__device__ __forceinline__ void add_to(Sums& a, float s, float c, float t) {
  const float sum = a.s + s, of_s = sum - a.s;
  a.c += c + ((a.s - (sum - of_s)) + (s - of_s));
  a.s = sum;
  a.t += t;
}
__device__ __forceinline__ void add(Sums& a, Sums b) {
  raise_to(a, b.m);
  raise_to(b, a.m);
  add_to(a, b.s, b.c, b.t);
}
// Four logits: their exponentials' sum, and that of their products.
__device__ __forceinline__ float2 four_terms(float4 x, float ref) {
  const float4 d = make_float4(x.x - ref, x.y - ref, x.z - ref, x.w - ref);
  const float4 e = make_float4(exp_of(d.x), exp_of(d.y), exp_of(d.z), exp_of(d.w));
  return make_float2((e.x + e.y) + (e.z + e.w), fmaf(fmaxf(d.x, -200.f), e.x, fmaxf(d.y, -200.f) * e.y) +
                                                    fmaf(fmaxf(d.z, -200.f), e.z, fmaxf(d.w, -200.f) * e.w));
}

// Keys of a warp, one a lane: sorted, largest in lane 0; and the 32 largest of two sorted lists, `b` given backwards.
__device__ __forceinline__ uint64_t exchange(uint64_t key, int with, bool larger) {
  const uint64_t other = __shfl_xor_sync(0xffffffffu, key, with);
  return (key > other) == larger ? key : other;
}
__device__ __forceinline__ uint64_t warp_sorted(uint64_t key) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int w = size / 2; w > 0; w /= 2) key = exchange(key, w, !(lane & w) == !(lane & size));
  return key;
}
__device__ __forceinline__ uint64_t warp_joined(uint64_t a, uint64_t b_backwards) {
  const int lane = threadIdx.x & 31;
  uint64_t key = a > b_backwards ? a : b_backwards;
#pragma unroll
  for (int w = 16; w > 0; w /= 2) key = exchange(key, w, !(lane & w));
  return key;
}

template <int WARPS, int KEPT, bool kCluster>
struct Shared {
  uint64_t kept[WARPS][KEPT];          // a warp's candidates, in no order
  float4 looked_at[WARPS][2][EACH];    // a round of the two threads that a warp looks at
  uint64_t lists[WARPS][32];
  uint64_t part_lists[kCluster ? PARTS_MOST : 1][32];   // of the parts of a row, in the first CTA of its cluster
  Sums part_sums[kCluster ? PARTS_MOST : 1];
  Sums sums[WARPS];
  uint64_t best[WARPS];
  unsigned long long floor_key;
};

// The 32 largest of `count` sorted lists in shared memory, to list 0.  All threads; a barrier at both ends.
__device__ __forceinline__ void join_lists(uint64_t (*lists)[32], int count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  for (int step = count / 2; step > 0; step /= 2) {
    if (warp < step) lists[warp][lane] = warp_joined(lists[warp][lane], lists[warp + step][31 - lane]);
    __syncthreads();
  }
}
// The 32 largest of a warp's candidates, sorted.
__device__ __forceinline__ uint64_t warp_best(const uint64_t* kept, int have) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  uint64_t key = warp_sorted(lane < have ? kept[lane] : 0);
  for (int at = 32; at < have; at += 32) {
    const uint64_t more = warp_sorted(at + lane < have ? kept[at + lane] : 0);
    key = warp_joined(key, __shfl_sync(0xffffffffu, more, 31 - lane));
  }
  return key;
}

__device__ __forceinline__ uint32_t cluster_at(const void* p, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// One CTA per row, of as few warps as still fill the GPU with the rows there are (one where rows are many: then nothing waits for
// another warp); where rows are fewer than that with eight warps, a cluster of `parts` CTAs, each on a range of the row.  A round is EACH
// float4 a thread, and the next round's are on their way.
//
// Bound: memory where rows are many (3000 x 50001: 105 to 115 us by machine and inputs, 5.2 to 5.7 TB/s, 80 to 87% of a copy's rate);
// launch, first round and joins where they are few (1 x 32000: 6.9 us, 36 x 100003: 12.7 us).
//
// Candidates for the best `top`: the floor is a key that `top` logits of the range are known to be above.  After the first round it
// is just below the `top`-th largest of the threads' largest keys; from then on every warp keeps what is above it in a list of its
// own, without a barrier.  A list that might overflow is cut to its `top` largest, which raises the floor for all.
template <int WARPS, int kTop, bool kCluster>
__global__ void __launch_bounds__(32 * WARPS, SM_WARPS / WARPS) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int THREADS = 32 * WARPS;
  constexpr int KEPT = kTop == MANY ? 192 : 128;   // keys that a warp's list of candidates holds
  __shared__ Shared<WARPS, KEPT, kCluster> sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kCluster ? (int)(blockIdx.x % (unsigned)a.parts) : 0;
  const int64_t row = kCluster ? blockIdx.x / (unsigned)a.parts : blockIdx.x;
  if (kCluster) cluster_arrive();   // this CTA has begun: the others may write to its shared memory (waited for below)
  if (kTop && threadIdx.x == 0) sh.floor_key = 0;
  pdl_wait();
  const float* x = pdl_after(a.logits) + row * a.row_stride;
  // float4 from the first 16-byte boundary on; what is before and behind them goes by single floats, to the first part
  const int before = min((int)(-(intptr_t)x >> 2 & 3), a.vocab), quads = (a.vocab - before) / 4;
  const int begin = kCluster ? (int)((int64_t)rank * quads / a.parts) : 0;
  const int end = kCluster ? (int)((int64_t)(rank + 1) * quads / a.parts) : quads;
  const float4* x4 = reinterpret_cast<const float4*>(x + before);

  // the given token's logit, asked for early and behind the first round's: two loads that nothing waits for until the end
  const bool asks = a.logprob && rank == 0 && warp == 0;
  const int token = asks ? pdl_ld(a.tokens + row) : -1;
  float chosen = NAN;
  const auto ask = [&]() {
    if (token >= 0 && token < a.vocab) chosen = pdl_ld(x + token);
  };

  Sums sums = {-INFINITY, 0.f, 0.f, 0.f};
  uint64_t floor_key = 0;
  uint64_t* kept = sh.kept[warp];
  int have = 0;                                    // candidates of this warp
  if (rank == 0 && warp == 0) {
    const int singles = a.vocab - quads * 4;       // up to six
    if (lane < singles) {
      const int i = lane < before ? lane : quads * 4 + lane;
      const float v = pdl_ld(x + i);
      raise_to(sums, v);
      const float2 terms = four_terms(make_float4(v, -INFINITY, -INFINITY, -INFINITY), sums.m == -INFINITY ? 0.f : sums.m);
      add_to(sums, terms.x, 0.f, terms.y);
      if (kTop) kept[lane] = order_key(v, i);
    }
    have = singles;
  }
  constexpr int ROUND = THREADS * EACH;
  const auto load = [&](float4 (&f)[EACH], int base) {
    if (base + ROUND <= end) {
#pragma unroll
      for (int j = 0; j < EACH; j++) f[j] = pdl_ld(x4 + base + j * THREADS + (int)threadIdx.x);
    } else {
#pragma unroll
      for (int j = 0; j < EACH; j++) {
        const int at = base + j * THREADS + (int)threadIdx.x;
        f[j] = at < end ? pdl_ld(x4 + at) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
    }
  };
  // adds a round to the sums; the largest of each float4
  const auto sum_up = [&](const float4 (&f)[EACH], float (&peaks)[EACH]) {
#pragma unroll
    for (int j = 0; j < EACH; j++) peaks[j] = fmaxf(fmaxf(f[j].x, f[j].y), fmaxf(f[j].z, f[j].w));
    const float peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
    raise_to(sums, peak);
    const float ref = sums.m == -INFINITY ? 0.f : sums.m;
    float2 terms[EACH];
#pragma unroll
    for (int j = 0; j < EACH; j++) terms[j] = four_terms(f[j], ref);
    add_to(sums, (terms[0].x + terms[1].x) + (terms[2].x + terms[3].x), 0.f, (terms[0].y + terms[1].y) + (terms[2].y + terms[3].y));
    return peak;
  };
  // cuts the list to its `top` largest, where there are more
  const auto cut = [&]() {
    const uint64_t key = warp_best(kept, have), least = __shfl_sync(0xffffffffu, key, a.top - 1) - 1;
    __syncwarp();
    kept[lane] = key;
    have = a.top;
    if (least > floor_key) {
      floor_key = least;
      if (lane == 0) atomicMax(&sh.floor_key, least);
    }
    __syncwarp();
  };
  // keeps what a round has above the floor: the first one, of which many threads have some
  const auto keep_first = [&](const float4 (&f)[EACH]) {
#pragma unroll
    for (int j = 0; j < EACH; j++) {
      const int at = begin + j * THREADS + (int)threadIdx.x;
      const float v[4] = {f[j].x, f[j].y, f[j].z, f[j].w};
      if (!__any_sync(0xffffffffu, at < end)) break;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const uint64_t key = order_key(v[c], before + 4 * at + c);
        const bool above = at < end && key > floor_key && v[c] == v[c];
        const unsigned who = __ballot_sync(0xffffffffu, above);
        if (above) kept[have + __popc(who & ((1u << lane) - 1))] = key;
        have += __popc(who);
      }
      if (have > KEPT - 128) cut();                // (64 or more)
    }
  };
  // and the others
  const auto keep = [&](const float4 (&f)[EACH], float peak, int base) {
    const uint64_t raised = *(volatile unsigned long long*)&sh.floor_key;
    floor_key = raised > floor_key ? raised : floor_key;
    const float floor_value = floor_key ? key_value(floor_key) : -INFINITY;
    // two threads at a time, their 16 logits by as many lanes each: there are few such threads after the first rounds
    static_assert(EACH == 4, "16 lanes a thread");
    unsigned who = __ballot_sync(0xffffffffu, peak >= floor_value);
    while (who) {
      const int first = __ffs((int)who) - 1;
      who &= who - 1;
      const int second = __ffs((int)who) - 1;      // (-1: there is no second)
      who &= who - 1;
      if (have > KEPT - 32) cut();
      if (lane == first || lane == second) {
#pragma unroll
        for (int j = 0; j < EACH; j++) sh.looked_at[warp][lane == second][j] = f[j];
      }
      __syncwarp();
      const int of = lane < 16 ? first : second, at = base + lane % 16 / 4 * THREADS + warp * 32 + of;
      const float v = reinterpret_cast<const float*>(sh.looked_at[warp])[lane];
      const uint64_t key = order_key(v, before + 4 * at + lane % 4);
      const bool above = of >= 0 && at < end && key > floor_key && v == v;
      const unsigned new_ones = __ballot_sync(0xffffffffu, above);
      if (above) kept[have + __popc(new_ones & ((1u << lane) - 1))] = key;
      have += __popc(new_ones);
      __syncwarp();
    }
  };
  // (two buffers in turn, so that nothing is moved from one to the other)
  float4 even[EACH], odd[EACH];
  float peaks[EACH], peak;
  if (begin < end) {
    load(even, begin);
    load(odd, begin + ROUND);
    ask();
    peak = sum_up(even, peaks);
    if (kTop) {
      // the floor: below the `top`-th largest of the threads' largest keys
      uint64_t mine = 0;
#pragma unroll
      for (int j = 0; j < EACH; j++) {
        const int at = begin + j * THREADS + (int)threadIdx.x;
        if (at >= end) break;
        // the largest of the four, and the first of those
        const uint64_t key = order_key(peaks[j], before + 4 * at + (even[j].x == peaks[j] ? 0 : even[j].y == peaks[j] ? 1 : even[j].z == peaks[j] ? 2 : 3));
        mine = key > mine ? key : mine;
      }
      sh.lists[warp][lane] = warp_sorted(mine);
      join_lists(sh.lists, WARPS);
      floor_key = sh.lists[0][a.top - 1];
      if (floor_key) floor_key--;                  // (fewer than `top` threads have any)
      __syncthreads();                             // (the lists are used again)
      if (kTop == MANY) keep_first(even);
      else keep(even, peak, begin);
    }
    for (int base = begin + ROUND; base < end; base += 2 * ROUND) {
      load(even, base + ROUND);
      peak = sum_up(odd, peaks);
      if (kTop) keep(odd, peak, base);
      if (base + ROUND >= end) break;
      load(odd, base + 2 * ROUND);
      peak = sum_up(even, peaks);
      if (kTop) keep(even, peak, base + ROUND);
    }
  } else {
    ask();
  }

#pragma unroll
  for (int w = 1; w < 32; w <<= 1)
    add(sums, {__shfl_xor_sync(0xffffffffu, sums.m, w), __shfl_xor_sync(0xffffffffu, sums.s, w),
               __shfl_xor_sync(0xffffffffu, sums.c, w), __shfl_xor_sync(0xffffffffu, sums.t, w)});
  if (lane == 0) sh.sums[warp] = sums;
  if (kTop) {
    sh.lists[warp][lane] = warp_best(kept, have);
    join_lists(sh.lists, WARPS);
  } else {
    __syncthreads();
  }
  sums = sh.sums[0];
#pragma unroll
  for (int w = 1; w < WARPS; w++) add(sums, sh.sums[w]);
  if (kCluster) {
    cluster_wait();
    if (warp == 0) {
      if (kTop)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_at(&sh.part_lists[rank][lane], 0)), "l"(sh.lists[0][lane]) : "memory");
      if (lane < 4)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_at(&sh.part_sums[rank].m + lane, 0)),
                     "f"(lane == 0 ? sums.m : lane == 1 ? sums.s : lane == 2 ? sums.c : sums.t) : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    for (int r = 1; r < a.parts; r++) add(sums, sh.part_sums[r]);
    if (kTop) join_lists(sh.part_lists, a.parts);
  }
  const bool none = sums.m == -INFINITY;
  // log(s + c): a sum just above 1 by its small part
  const float above = (sums.s - 1.f) + sums.c, log_s = none ? NAN : above < 0.5f ? log1pf(above) : logf(sums.s + sums.c);
  if (threadIdx.x == 0) {
    if (a.logprob) a.logprob[row] = chosen - sums.m - log_s;
    if (a.entropy) a.entropy[row] = log_s - sums.t / sums.s;
  }
  if (!kTop) return;
  if (sums.s == sums.s) {
    if (warp == 0 && lane < a.top) {
      const uint64_t best = kCluster ? sh.part_lists[0][lane] : sh.lists[0][lane];
      a.top_ids[row * a.top + lane] = (int32_t)~(uint32_t)best;
      a.top_logprobs[row * a.top + lane] = key_value(best) - sums.m - log_s;
    }
    return;
  }
  // a NaN, which no maximum above shows: the next largest key of the whole row, `top` times
  uint64_t below = ~0ull;
  for (int k = 0; k < a.top; k++) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
      const uint64_t key = order_key(pdl_ld(x + i), i);
      if (key < below && key > mine) mine = key;
    }
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, mine, w);
      mine = mine > other ? mine : other;
    }
    __syncthreads();
    if (lane == 0) sh.best[warp] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) mine = mine > sh.best[w] ? mine : sh.best[w];
    below = mine;
    if (threadIdx.x == 0) {
      a.top_ids[row * a.top + k] = (int32_t)~(uint32_t)mine;
      a.top_logprobs[row * a.top + k] = NAN;
    }
  }
}

template <int WARPS, bool kCluster>
cudaError_t launch(wdc_context* ctx, const LogprobArgs& a, int64_t rows) {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * a.parts));
  cfg.blockDim = dim3(32 * WARPS);
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  if (kCluster) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)a.parts;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  if (ctx->opt_pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs++;
  }
  if (!a.top) return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<WARPS, NONE, kCluster>, a);
  if (a.top >= MANY_TOP && a.vocab <= MANY_ROUNDS * a.parts * WARPS * 32 * EACH * 4)
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<WARPS, MANY, kCluster>, a);
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<WARPS, SOME, kCluster>, a);
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
  for (const void* p : {(const void*)logits, (const void*)tokens, (const void*)logprob, (const void*)entropy,
                        (const void*)top_ids, (const void*)top_logprobs})
    WDC_REQUIRE(ctx, (reinterpret_cast<uintptr_t>(p) & 3u) == 0, "wdc_token_logprobs: buffers are not aligned");
  DeviceGuard g(ctx->device);
  LogprobArgs a = {logits, tokens, logprob, entropy, top_logprobs, top_ids, d->row_stride, (int)d->vocab,
                   top_ids ? (int)d->top : 0, 1};
  int warps = 1;
  while (warps < WARPS_MOST && d->rows * 2 * warps <= (int64_t)SM_WARPS * ctx->sm_count && d->vocab >= 2 * warps * 32 * EACH * 4) warps *= 2;
  if (warps == WARPS_MOST)
    while (a.parts < PARTS_MOST && d->rows * a.parts < 2 * ctx->sm_count && d->vocab / (2 * a.parts) >= PART_LEAST) a.parts *= 2;
  WDC_REQUIRE(ctx, d->rows * a.parts < (1ll << 31), "wdc_token_logprobs: rows exceed the grid");
  const cudaError_t e = a.parts > 1  ? launch<8, true>(ctx, a, d->rows)
                        : warps == 8 ? launch<8, false>(ctx, a, d->rows)
                        : warps == 4 ? launch<4, false>(ctx, a, d->rows)
                        : warps == 2 ? launch<2, false>(ctx, a, d->rows) : launch<1, false>(ctx, a, d->rows);
  WDC_CUDA(ctx, e);
  return wdc_check_launch(ctx, "token_logprobs_kernel");
}
