// Attention of new tokens over a paged cache in 8 bits:  y = softmax(scale * q k^T) v,  k = code * (scale of page and head).
// The reference has no such operator.
#include <cuda_fp16.h>
#include <math.h>

#include "cache_attention.cuh"

namespace {

// A unit of work is eight rows of one sequence and key head, row = new token * group + query head of the group, and the tiles of 32
// tokens of that sequence.  The warps of a CTA take tiles in turn, each through a ring of its own in shared memory that asynchronous
// copies fill two or three tiles ahead, so that no warp waits for another before the end.
//
// Where units are fewer than the GPU holds CTAs, each is cut into parts, which leave their results (rows, m, M, l) in memory for a
// second kernel to join.  Either `splits` equal parts, a CTA each; or, where sequences are few and long, so that their
// lengths decide how long the longest part takes, the tiles of all units, in the order sequence, head and rows, tile, are cut into
// one range for each CTA that the GPU holds, all of the same length (shared out).  The beginning of a unit (queries, first
// copies, joining the warps) counts as BEGIN tiles there, and a CTA has at most two such parts: of the unit that began before its
// range and of the one that ends behind it.
//
// Both products run on mma.m16n8k16 with float16 operands and 32-bit sums.  A code (-127 .. 127) is exact in float16; a
// query is split into a high and a low half, 22 bits together, and so is a weight.  The halves are the two halves of the
// instruction's 16 rows: eight rows with both halves are one instruction, and their sums meet in one thread's registers.
// (Codes + 128 would be exact as well, and two instructions a word less.  But the scores' sums would be of that size, and cancel
// when the 128 is taken off: with codes of about 3 two scores' difference was up to 9 x 2^-21 of sum |q k| off, 26 x with queries of a
// mean of 5, against 1 x.)
//
// Weights carry the value scale of their page.  With s the scores (base 2) and lv = log2(value scale) of a group of 16 tokens,
//   m = max s,  l = sum 2^(s - m);      M = max (s + [lv]),  O = sum 2^(s + lv - M) code,      y = O 2^(M - m) / l,
// so that what is split into halves is relative to the largest term of O, whatever the pages' scales are.  ([lv] is the scale's
// binary exponent: the maxima need no logarithm, and the weights take the scale itself.)  M need not be that maximum, only no
// less: it starts HEADROOM above what the first tile has, and rises only when a term would pass it, so that O is rarely scaled
// again.  A tile's tokens of one page are a group: 32 of them, or 16 where pages hold no more (GROUPS).
//
// Bound: 380 cycles of an SM a tile of heads of 128 (8 KB; 6.0 TB/s over all), of which issue takes 190 (about 760 instructions, of
// which 225 and 230 are the widening of keys and values and the products with them) and the ALUs, shared memory and tensor core half
// each; 16 warps an SM need as long.  Around that, beginnings and ends of units.  Measured: 48 sequences of 1 to 4100 tokens, 32 query and
// 8 key heads of 128, 52.7 us (3.9 TB/s); 3 of 12000 to 40001, 16 heads, 71.5 us (4.5 TB/s); one of 700, 16 and 4 heads of 64, 6.4 us.
constexpr int WARPS = 4, THREADS = 32 * WARPS, TILE = 32, ROWS = 8;
constexpr int PLAN_MOST = 512;             // sequences whose tiles are shared out
constexpr int BEGIN = 8;
constexpr float HEADROOM = 3.f;
// Tiles whose weighted values the tensor core adds up before the sum goes to one of the thread's own.  It rounds towards zero, 2^-25
// of the sum at each of two additions a tile: 44 in a row were 1.3e-6 short, 1000 would be 3e-5.  (Folding costs 4% of 3 x 40001.)
constexpr int FOLD = 16;

template <int DH>
struct Layout {
  static constexpr int CTAS = DH == 128 ? 3 : 4;                     // per SM: what registers and shared memory have room for
  static constexpr int STAGES = DH == 128 ? 2 : 3;
  static constexpr int SCALES = 2 * TILE * DH;                       // behind a stage's keys and values: its groups' scales, and
  static constexpr int THERE = SCALES + 16;                          // which of its groups are there
  static constexpr int STAGE = SCALES + 128, RING = STAGES * STAGE;  // (128-byte lines, for value_at)
  static constexpr int STRIDE = DH + 4, STATS = ROWS * STRIDE;       // floats: a row when the warps join; behind them m, M, l
  static constexpr int PART = STATS + 3 * ROWS;
  static constexpr int SMEM = WARPS * (RING > PART * 4 ? RING : PART * 4);
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int TO, int FROM>
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(to), "l"(from), "n"(TO), "n"(FROM) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Where the 16-byte chunk `c` of token `t` lies in a tile of keys or values: as in memory, chunks of a 128-byte line exchanged
// so that the eight (16-byte loads), sixteen (8) or 32 (4) threads that load at a time meet different banks.
template <int DH>
__device__ __forceinline__ int key_at(int t, int c) {
  const int x = t * (DH / 16) + c;
  return (DH == 128 ? x ^ (t & 1) << 2 : x) * 16;
}
template <int DH>
__device__ __forceinline__ int value_at(int t, int c) {
  const int x = t * (DH / 16) + c;
  return (DH == 32 ? x ^ (t >> 2 & 1) << 1 : x ^ (t >> 1 & 3) << 1) * 16;
}
template <int BYTES>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[BYTES / 4]) {
  if (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[BYTES > 4] = v.y; w[BYTES / 8] = v.z; w[BYTES / 4 - 1] = v.w;
  } else if (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[BYTES / 4 - 1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int i = 0; i < BYTES / 4; i++) w[i] ^= 0x80808080u;
}

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// Asynchronous copies of 16 tokens' keys and values by a warp.  `k` and `v` are at this lane's 16 bytes; MORE: how far behind.
template <int DH, int TO, int MORE>
__device__ __forceinline__ void copy_half(uint32_t to_k, uint32_t to_v, const int8_t* k, const int8_t* v) {
  copy16<TO, MORE>(to_k, k);
  copy16<TO, MORE>(to_v, v);
  if (DH >= 64) {
    // (128: eight rows of a line's exchange pattern are two copies, so that every other copy's is the other half's)
    copy16<TO + (DH >= 64 ? 512 : 0), MORE + (DH >= 64 ? 512 : 0)>(to_k, k);
    copy16<TO + (DH >= 64 ? 512 : 0), MORE + (DH >= 64 ? 512 : 0)>(DH == 128 ? to_v ^ 64 : to_v, v);
  }
  if (DH == 128) {
    copy16<TO + 1024, MORE + 1024>(to_k, k);
    copy16<TO + 1024, MORE + 1024>(to_v, v);
    copy16<TO + 1536, MORE + 1536>(to_k, k);
    copy16<TO + 1536, MORE + 1536>(to_v ^ 64, v);
  }
}

template <int DH, int GROUPS>
__global__ void __launch_bounds__(THREADS, Layout<DH>::CTAS) cache_attention_kernel(const CacheAttArgs a) {
  constexpr int STEPS = DH / 16;                  // of the score product's sum; also columns of O a thread and key row
  constexpr int KB = DH == 32 ? 8 : 16;           // bytes of a key a thread loads at a time
  constexpr int VB = DH / 8;                      // bytes of a value row a thread loads
  using L = Layout<DH>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int plan[PLAN_MOST + 1], plan_sums[WARPS];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int units = a.kv_heads * a.row_tiles;     // of a sequence
  int pos = 0, stop = 0, b = 0, segment = 0;
  if (!a.splits) {
    // the sequences' tiles, all units together, and where each begins
    constexpr int EACH = PLAN_MOST / THREADS;
    int mine[EACH], sum = 0;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int s = (int)threadIdx.x * EACH + k;
      mine[k] = sum;
      if (s < a.batch) {
        const CacheSpan span = cache_span(a.lengths, a.counts, s, a.tokens, a.table_pages << a.page_shift, a.status);
        sum += span.count ? ((span.length + TILE - 1) / TILE + BEGIN) * units : 0;
      }
    }
    int up = sum;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, up, w);
      if (lane >= w) up += other;
    }
    if (lane == 31) plan_sums[warp] = up;
    __syncthreads();
    up -= sum;
    for (int w = 0; w < warp; w++) up += plan_sums[w];
#pragma unroll
    for (int k = 0; k < EACH; k++)
      if ((int)threadIdx.x * EACH + k <= a.batch) plan[threadIdx.x * EACH + k] = up + mine[k];
    if (threadIdx.x == THREADS - 1 && a.batch == PLAN_MOST) plan[PLAN_MOST] = up + sum;
    __syncthreads();
    const int total = plan[a.batch];
    const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, WARPS);
    if (blockIdx.x == 0) {
      for (int s = threadIdx.x; s <= a.batch; s += THREADS) a.part_plan[s] = plan[s];
      if (threadIdx.x == 0) a.part_plan[a.batch + 1] = share;
    }
    pos = (int)min((int64_t)blockIdx.x * share, (int64_t)total);
    stop = min(pos + share, total);
    if (pos == stop) return;
    int past = a.batch;                            // the sequence that holds tile `pos`: plan[b] <= pos < plan[b + 1]
    b = 0;
    while (past - b > 1) {
      const int middle = (b + past) / 2;
      if (plan[middle] <= pos) b = middle;
      else past = middle;
    }
  }
next_segment:
  int unit = 0, first = 0, end = 0;
  bool complete = a.splits == 1, began_here = true;
  if (a.splits) {
    unit = (int)(blockIdx.x / (unsigned)a.splits);
    b = unit / units;
    unit -= b * units;
  } else {
    while (plan[b + 1] <= pos) b++;
    const int size = (plan[b + 1] - plan[b]) / units;                // BEGIN, then the unit's tiles
    unit = (pos - plan[b]) / size;
    const int from = plan[b] + unit * size;
    began_here = segment > 0 || pos == from;
    first = max(pos - from - BEGIN, 0);
    end = min(size, stop - from) - BEGIN;
    pos = from + BEGIN + end;
    if (end <= 0) return;                                            // (its tiles are the next CTA's)
    complete = first == 0 && end == size - BEGIN;
  }
  const int tile = unit % a.row_tiles, kvh = unit / a.row_tiles;
  const CacheSpan span = cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages << a.page_shift, a.status);
  const int row = tile * ROWS + g, token = row / a.group, head = kvh * a.group + row % a.group;   // this thread's row
  const int before = span.length - span.count;
  // the last token that this row sees (rows of padding see all: nobody reads theirs), and those of the tile's first and last row
  const int first_token = tile * ROWS / a.group, top_token = min((tile * ROWS + ROWS - 1) / a.group, span.count - 1);
  const int last = token < span.count ? before + token : 0x7fffffff;
  const int seen_by_all = before + first_token + 1;
  const int seen = first_token < span.count ? before + top_token + 1 : 0;
  {
    const int tiles = (seen + TILE - 1) / TILE, part = (int)(blockIdx.x % (unsigned)max(a.splits, 1));
    if (a.splits) first = (int)((int64_t)part * tiles / a.splits);
    end = a.splits ? (int)((int64_t)(part + 1) * tiles / a.splits) : min(end, tiles);
  }
  const int32_t* table = a.page_table + (int64_t)b * a.table_pages;
  unsigned char* ring = smem + warp * L::RING;

  // a lane's place in a group of 16 tokens, in memory and in a stage
  const uint32_t page_bytes = (uint32_t)(2 * a.kv_heads * DH) << a.page_shift, side_bytes = page_bytes / 2;
  const int8_t* codes = a.codes + (int64_t)kvh * (DH << a.page_shift) + lane * 16;
  const uint32_t to_k = smem_u32(ring + key_at<DH>(lane / (DH / 16), lane % (DH / 16)));
  const uint32_t to_v = smem_u32(ring + TILE * DH + value_at<DH>(lane / (DH / 16), lane % (DH / 16)));
  const float* scales = a.scales + kvh + (lane & 1) * a.kv_heads;
  const uint32_t to_scale = smem_u32(ring + L::SCALES + (lane & 1) * 4);

  // the pages of a tile's groups (-1: nothing is there), and their copies to a stage
  constexpr int SIZE = TILE / GROUPS;
  const auto pages_of = [&](int i, int (&page)[GROUPS]) {
#pragma unroll
    for (int group = 0; group < GROUPS; group++) {
      const int t0 = i * TILE + group * SIZE;
      page[group] = i < end && t0 < seen ? cache_page(table, t0 >> a.page_shift, a.pages, a.status) : -1;
    }
  };
  const auto fetch = [&](int i, const int (&page)[GROUPS], uint32_t stage_at) {
    int there = 0;
#pragma unroll
    for (int group = 0; group < GROUPS; group++) {
      if (page[group] < 0) continue;
      there |= 1 << group;
      // (a group of 16 is a page of 16, from its first token on)
      const uint32_t in_page = GROUPS == 2 ? 0 : (uint32_t)(i * TILE) & ((1u << a.page_shift) - 1);
      const int8_t* k = codes + ((uint64_t)(uint32_t)page[group] * page_bytes + in_page * DH);
      if (GROUPS == 1 || group == 0) copy_half<DH, 0, 0>(to_k + stage_at, to_v + stage_at, k, k + side_bytes);
      if (GROUPS == 1) copy_half<DH, 16 * DH, 16 * DH>(to_k + stage_at, to_v + stage_at, k, k + side_bytes);
      else if (group == 1) copy_half<DH, 16 * DH, 0>(to_k + stage_at, to_v + stage_at, k, k + side_bytes);
      if (lane < 2) copy4(to_scale + stage_at + group * 8, scales + (uint64_t)(uint32_t)page[group] * (uint32_t)(2 * a.kv_heads));
    }
    copies_commit();
    if (lane == 0) *reinterpret_cast<int*>(ring + stage_at + L::THERE) = there;
  };
  int next = first + warp, page[GROUPS];
#pragma unroll
  for (int s = 0; s < L::STAGES; s++, next += WARPS) {
    pages_of(next, page);
    fetch(next, page, s * L::STAGE);
  }
  pages_of(next, page);

  // this row's queries, scaled by a power of two, in halves: step j of the sum covers channels at(j) .. + 3 of thread t
  uint32_t q[STEPS][4];
  float row_scale;
  {
    const float* qp = pdl_after(a.q) + b * a.q_sb + head * a.q_sh + token * a.q_st;
    float4 x[STEPS];
    float peak = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
      const int at = DH == 32 ? t * 8 + j * 4 : (j / 4) * 64 + t * 16 + (j % 4) * 4;
      x[j] = token < span.count ? pdl_ld(reinterpret_cast<const float4*>(qp + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
      peak = fmaxf(fmaxf(fmaxf(peak, fabsf(x[j].x)), fmaxf(fabsf(x[j].y), fabsf(x[j].z))), fabsf(x[j].w));
    }
    peak = quad_max(peak);
    const float up = query_scale(peak, a.scale_log2, row_scale);
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
      split_halves(x[j].x * up, x[j].y * up, q[j][0], q[j][1]);
      split_halves(x[j].z * up, x[j].w * up, q[j][2], q[j][3]);
    }
  }

  float o[DH / 8][4], m = -INFINITY, big = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < DH / 8; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) o[d][i] = 0.f;

  // sums of FOLD tiles and more, in local memory: channels of this thread's two columns, relative to 2^total_big
  float total_room[DH / 4], total_big = -INFINITY;
  volatile float* total = total_room;
  int added = 0;
  uint32_t stage_at = 0;
  for (int i = first + warp; i < end; i += WARPS) {
    if (added == FOLD) {
      const float keep = exp2_of(total_big - finite_or_0(big));
      const bool some = total_big > -INFINITY;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float before[DH / 8];
#pragma unroll
        for (int d = 0; d < DH / 8; d++) before[d] = total[k * (DH / 8) + d];      // (all loads before the first store)
#pragma unroll
        for (int d = 0; d < DH / 8; d++) {
          const float sum = o[d][k] + o[d][k + 2];
          total[k * (DH / 8) + d] = some ? fmaf(before[d], keep, sum) : sum;
          o[d][k] = o[d][k + 2] = 0.f;
        }
      }
      total_big = fmaxf(big, -1e30f);
      added = 0;
    }
    added++;
    copies_wait<L::STAGES - 1>();
    __syncwarp();
    const unsigned char* tile_at = ring + stage_at;
    float key_scale[GROUPS], value_scale[GROUPS];
#pragma unroll
    for (int group = 0; group < GROUPS; group++) {
      const float2 sc = *reinterpret_cast<const float2*>(tile_at + L::SCALES + group * 8);
      key_scale[group] = key_scale_of(sc.x);
      value_scale[group] = sc.y;
    }
    const int there = *reinterpret_cast<const int*>(tile_at + L::THERE);
    constexpr int PER = 4 / GROUPS;                // sets of eight tokens a group
    float s[4][2];
#pragma unroll
    for (int n = 0; n < 4; n++) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < STEPS; j += KB / 4) {
        uint32_t w[KB / 4];
        load_words<KB>(tile_at + (DH == 32 ? key_at<DH>(n * 8 + g, t >> 1) + (t & 1) * 8 : key_at<DH>(n * 8 + g, j + t)), w);
#pragma unroll
        for (int k = 0; k < KB / 4; k++) mma(c, q[j + k], two_codes<0x4140>(w[k]), two_codes<0x4342>(w[k]));
      }
      const float by = row_scale * key_scale[n / PER];
      s[n][0] = (c[0] + c[2]) * by;
      s[n][1] = (c[1] + c[3]) * by;
    }
    // what this row does not see
    const bool whole = (i + 1) * TILE <= seen_by_all && there == (1 << GROUPS) - 1;
    if (!whole) {
      const int t0 = i * TILE + 2 * t;
#pragma unroll
      for (int n = 0; n < 4; n++)
#pragma unroll
        for (int k = 0; k < 2; k++)
          if (t0 + n * 8 + k > last || !(there >> (n / PER) & 1)) s[n][k] = -INFINITY;
    }
    float e[GROUPS], f[GROUPS], m_new = m, big_new = -INFINITY;
#pragma unroll
    for (int group = 0; group < GROUPS; group++) {
      float top = -INFINITY;
#pragma unroll
      for (int n = group * PER; n < (group + 1) * PER; n++) top = fmaxf(top, fmaxf(s[n][0], s[n][1]));
      top = quad_max(top);
      exponent_of(value_scale[group], e[group], f[group]);
      m_new = fmaxf(m_new, top);
      big_new = fmaxf(big_new, top + e[group]);
    }
    if (__any_sync(0xffffffffu, big_new > big)) {
      big_new = big_new > big ? big_new + HEADROOM : big;
      const float keep = exp2_of(big - finite_or_0(big_new));
#pragma unroll
      for (int d = 0; d < DH / 8; d++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[d][k] *= keep;
      big = big_new;
    }
    const float m_ref = finite_or_0(m_new), big_ref = finite_or_0(big);
    l *= exp2_of(m - m_ref);
    m = m_new;
#pragma unroll
    for (int group = 0; group < GROUPS; group++) f[group] *= exp2_of(fminf(m_ref + e[group] - big_ref + WEIGHT_BITS, 126.f));
    float w[4][2];
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const float p = exp2_of(s[n][k] - m_ref);
        l += p;
        w[n][k] = p * f[n / PER];
      }
    if (!whole) {                                  // (a scale that is no number is for the rows that see it)
#pragma unroll
      for (int n = 0; n < 4; n++)
#pragma unroll
        for (int k = 0; k < 2; k++)
          if (s[n][k] == -INFINITY) w[n][k] = 0.f;
    }
    uint32_t p[2][4];
#pragma unroll
    for (int n = 0; n < 4; n++) split_halves(w[n][0], w[n][1], p[n >> 1][(n & 1) * 2], p[n >> 1][(n & 1) * 2 + 1]);
    const unsigned char* values = tile_at + TILE * DH;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      uint32_t v[4][VB / 4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int key = half * 16 + 2 * t + (r & 1) + (r >> 1) * 8;
        load_words<VB>(values + value_at<DH>(key, g * VB / 16) + g * VB % 16, v[r]);
      }
#pragma unroll
      for (int w = 0; w < VB / 4; w++) {
        const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
        const uint32_t b0 = __byte_perm(v[2][w], v[3][w], 0x5140), b1 = __byte_perm(v[2][w], v[3][w], 0x7362);
        mma(o[w * 4 + 0], p[half], two_codes<0x4140>(a0), two_codes<0x4140>(b0));
        mma(o[w * 4 + 1], p[half], two_codes<0x4342>(a0), two_codes<0x4342>(b0));
        mma(o[w * 4 + 2], p[half], two_codes<0x4140>(a1), two_codes<0x4140>(b1));
        mma(o[w * 4 + 3], p[half], two_codes<0x4342>(a1), two_codes<0x4342>(b1));
      }
    }
    __syncwarp();
    fetch(next, page, stage_at);
    next += WARPS;
    pages_of(next, page);
    stage_at = stage_at == (L::STAGES - 1) * L::STAGE ? 0 : stage_at + L::STAGE;
  }

  // the warps' results: channel c of row g is in thread c / (2 * DH / 8), its two halves beside one another
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  copies_wait<0>();
  __syncthreads();
  float* parts = reinterpret_cast<float*>(smem);
  {
    float* mine = parts + warp * L::PART;
    const float keep = exp2_of(total_big - finite_or_0(big));
    if (total_big > -INFINITY) {
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int d = 0; d < DH / 8; d++) o[d][k] = fmaf(total[k * (DH / 8) + d], keep, o[d][k]);
    }
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int d = 0; d < DH / 8; d += 4)
        *reinterpret_cast<float4*>(mine + g * L::STRIDE + (2 * t + k) * (DH / 8) + d) =
            make_float4(o[d][k] + o[d][k + 2], o[d + 1][k] + o[d + 1][k + 2], o[d + 2][k] + o[d + 2][k + 2], o[d + 3][k] + o[d + 3][k + 2]);
    if (t == 0) {
      float* stats = mine + L::STATS;
      stats[g] = m;
      stats[ROWS + g] = big;
      stats[2 * ROWS + g] = l;
    }
  }
  __syncthreads();
  constexpr int PER = THREADS / ROWS;             // threads a row, DH / PER channels each
  const int r = threadIdx.x / PER, c0 = threadIdx.x % PER * (DH / PER);
  float mw[WARPS], bw[WARPS], lw[WARPS], m_all = -INFINITY, big_all = -INFINITY, l_all = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    const float* stats = parts + w * L::PART + L::STATS;
    mw[w] = stats[r];
    bw[w] = stats[ROWS + r];
    lw[w] = stats[2 * ROWS + r];
    m_all = fmaxf(m_all, mw[w]);
    big_all = fmaxf(big_all, bw[w]);
  }
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    l_all = fmaf(lw[w], exp2f(mw[w] - finite_or_0(m_all)), l_all);
    bw[w] = exp2f(bw[w] - finite_or_0(big_all));
  }
  float out[DH / PER];
#pragma unroll
  for (int c = 0; c < DH / PER; c++) {
    out[c] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) out[c] = fmaf(parts[w * L::PART + r * L::STRIDE + c0 + c], bw[w], out[c]);
  }
  const int out_row = tile * ROWS + r;
  if (out_row < a.tokens * a.group) {
    if (complete) {
      const float by = l_all == 0.f || out_row / a.group >= span.count ? 0.f : exp2f(big_all - finite_or_0(m_all) - WEIGHT_BITS) / l_all;
      float* y = a.y + b * a.y_sb + (kvh * a.group + out_row % a.group) * a.y_sh + out_row / a.group * a.y_st + c0;
#pragma unroll
      for (int c = 0; c < DH / PER; c++) y[c] = out[c] * by;
    } else {
      const int64_t at = (a.splits ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 2 + began_here) * ROWS + r;
      float* to = a.part_rows + at * DH + c0;
#pragma unroll
      for (int c = 0; c < DH / PER; c++) to[c] = out[c];
      if (c0 == 0) {
        a.part_stats[at * 3] = m_all;
        a.part_stats[at * 3 + 1] = big_all;
        a.part_stats[at * 3 + 2] = l_all;
      }
    }
  }
  if (pos < stop) {
    segment++;
    __syncthreads();                               // the joined rows have been read: the rings are free
    goto next_segment;
  }
}

// Joins the parts of a row, one CTA each, where its unit was cut: warp w takes parts w, w + 4, ...  Rows of empty sequences are
// its business too.
template <int DH>
__global__ void __launch_bounds__(THREADS) cache_attention_join_kernel(const CacheAttArgs a) {
  pdl_wait();
  constexpr int C = DH / 32;
  __shared__ float sums[WARPS][DH + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = (int)(blockIdx.x % (unsigned)(a.tokens * a.group)), bh = (int)(blockIdx.x / (unsigned)(a.tokens * a.group));
  const int kvh = bh % a.kv_heads, b = bh / a.kv_heads, token = row / a.group, units = a.kv_heads * a.row_tiles;
  int64_t begin = 0;                               // the place of part 0; that of a shared-out unit: of its first CTA
  int parts = a.splits, share = 0, cta = 0, from = 0;
  if (a.splits) {
    begin = ((int64_t)bh * a.row_tiles + row / ROWS) * a.splits;
  } else {
    const int* plan = pdl_after(a.part_plan);
    const int size = (plan[b + 1] - plan[b]) / units;
    share = plan[a.batch + 1];
    from = plan[b] + (kvh * a.row_tiles + row / ROWS) * size;             // the unit's beginning
    cta = (from + BEGIN) / share;
    parts = size ? (from + size - 1) / share - cta + 1 : 0;
    if (parts == 1) return;
  }
  const auto place = [&](int p) {
    return (share ? (int64_t)(cta + p) * 2 + (from >= (int64_t)(cta + p) * share) : begin + p) * ROWS + row % ROWS;
  };
  const float* stats = pdl_after(a.part_stats);
  const float* rows = pdl_after(a.part_rows) + lane * C;
  const int count = a.counts ? pdl_ld(a.counts + b) : a.tokens;
  float m = -INFINITY, big = -INFINITY, l = 0.f, o[C];
  for (int p = lane; p < parts; p += 32) {
    m = fmaxf(m, stats[place(p) * 3]);
    big = fmaxf(big, stats[place(p) * 3 + 1]);
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, w));
  }
#pragma unroll
  for (int c = 0; c < C; c++) o[c] = 0.f;
#pragma unroll 4
  for (int p = warp; p < parts; p += WARPS) {
    const float* st = stats + place(p) * 3;
    l = fmaf(st[2], exp2f(st[0] - finite_or_0(m)), l);
    const float f = exp2f(st[1] - finite_or_0(big));
#pragma unroll
    for (int c = 0; c < C; c++) o[c] = fmaf(rows[place(p) * DH + c], f, o[c]);
  }
#pragma unroll
  for (int c = 0; c < C; c++) sums[warp][lane * C + c] = o[c];
  if (lane == 0) sums[warp][DH] = l;
  __syncthreads();
  if ((int)threadIdx.x >= DH) return;
  float total = 0.f, sum = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    total += sums[w][DH];
    sum += sums[w][threadIdx.x];
  }
  // (a count out of range leaves l at 0)
  const float by = total == 0.f || token >= count ? 0.f : exp2f(big - finite_or_0(m) - WEIGHT_BITS) / total;
  a.y[b * a.y_sb + (kvh * a.group + row % a.group) * a.y_sh + token * a.y_st + threadIdx.x] = sum * by;
}

template <int DH, int GROUPS>
int launch(wdc_context* ctx, CacheAttArgs& a) {
  static bool opted_in[64] = {};     // per device: more than 48 KB of dynamic shared memory needs the attribute
  WDC_REQUIRE(ctx, ctx->device >= 0 && ctx->device < 64, "wdc_cache_attention: device index out of range");
  if (!opted_in[ctx->device]) {
    WDC_CUDA(ctx, cudaFuncSetAttribute(cache_attention_kernel<DH, GROUPS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Layout<DH>::SMEM));
    opted_in[ctx->device] = true;
  }
  const int64_t units = (int64_t)a.batch * a.kv_heads * a.row_tiles, slots = Layout<DH>::CTAS * ctx->sm_count;
  const int64_t tiles = ceil_div64(a.table_pages << a.page_shift, TILE);
  // As many parts as make one wave of CTAs (two, where that would leave a third of it empty or more); shared out where a CTA has 32
  // tiles and more, as far as the table's width tells.  Measured, us with equal parts / shared out, heads of 128 (units, tiles a CTA): 3
  // sequences of 12000 to 40001 tokens and 16 key heads (48, 142) 84.2 / 70.7; 16 of 1959 to 2979 and 16 (256, 57) 53.8 / 44.3; of 1 to 4100
  // and 8 key heads, 32 sequences (256, 78) 46.0 / 40.4, 64 (512, 157) 78.6 / 66.6; 20 of 100 to 1500 and 8, two row tiles (320, 27) 17.0 /
  // 20.2; 16 of 2243 to 11554 and 2, heads of 32 (32, 20) 13.5 / 16.3.  Two and more equal parts or whole units for each place can be the
  // better ones when uneven units happen to fill their waves: 48 of 1 to 4100 (384, 118) 49.7 / 52.6, 96 (768, 235) 81.1 / 92.5; but 48 of
  // 3000 to 4100 (384, 118) 79.3 / 77.5.  The host does not know the lengths that decide it.
  a.splits = (int)(2 * units <= slots ? slots / units : units < slots ? 2 : 1);
  if (a.splits > ceil_div64(tiles, WARPS)) a.splits = (int)ceil_div64(tiles, WARPS);
  if (a.splits < 1) a.splits = 1;
  if (a.batch <= PLAN_MOST && units < 2 * slots && units * tiles >= 32 * slots &&
      units * (tiles + BEGIN) < (1ll << 31) - slots * WARPS)
    a.splits = 0;
  const int64_t ctas = a.splits ? units * a.splits : slots, parts = a.splits == 1 ? 0 : a.splits ? ctas : 2 * ctas;
  float* scratch = nullptr;
  if (parts) {
    CACHE_TRY(wdc_alloc(ctx, (parts * ROWS * (DH + 3) + a.batch + 2) * 4, (void**)&scratch));
    a.part_rows = scratch;
    a.part_stats = scratch + parts * ROWS * DH;
    a.part_plan = (int*)(a.part_stats + parts * ROWS * 3);
  }
  WDC_REQUIRE(ctx, ctas < (1ll << 31), "wdc_cache_attention: batch exceeds the grid");
  wdc_launch_pdl(ctx, cache_attention_kernel<DH, GROUPS>, dim3((unsigned)ctas), dim3(THREADS), Layout<DH>::SMEM, a);
  int s = wdc_check_launch(ctx, "cache_attention_kernel");
  if (s == WDC_OK && parts) {
    wdc_launch_pdl(ctx, cache_attention_join_kernel<DH>, dim3((unsigned)((int64_t)a.batch * a.heads * a.tokens)), dim3(THREADS), 0, a);
    s = wdc_check_launch(ctx, "cache_attention_join_kernel");
  }
  if (scratch) wdc_free(ctx, scratch);   // stream-ordered: reused only by work queued after the kernels
  return s;
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
  CacheAttArgs a = {};
  a.q = q; a.codes = (const int8_t*)codes; a.scales = scales;
  a.page_table = page_table; a.lengths = lengths; a.counts = counts;
  a.y = y; a.status = ctx->status_word;
  a.pages = d->pages; a.table_pages = d->table_pages;
  a.q_sb = d->q_sb; a.q_sh = d->q_sh; a.q_st = d->q_st;
  a.y_sb = d->y_sb; a.y_sh = d->y_sh; a.y_st = d->y_st;
  a.batch = (int)d->batch; a.tokens = (int)d->tokens; a.heads = (int)d->heads; a.kv_heads = (int)d->kv_heads;
  a.group = (int)(d->heads / d->kv_heads); a.page_shift = 4;
  while (1 << a.page_shift < d->page_tokens) a.page_shift++;
  WDC_REQUIRE(ctx, d->tokens * a.group < (1ll << 31) - ROWS && d->batch * d->heads * d->tokens < (1ll << 31),
              "wdc_cache_attention: batch exceeds the grid");
  a.row_tiles = (int)ceil_div64(d->tokens * a.group, ROWS);
  a.scale_log2 = d->scale * 1.4426950408889634f;
  DeviceGuard g(ctx->device);
  {
    const int s = wdc_cache_attention_tc(ctx, a, (int)d->head_size);
    if (s != WDC_ERR_UNSUPPORTED) return s;
  }
  const bool small = d->page_tokens < TILE;
  if (d->head_size == 32) return small ? launch<32, 2>(ctx, a) : launch<32, 1>(ctx, a);
  if (d->head_size == 64) return small ? launch<64, 2>(ctx, a) : launch<64, 1>(ctx, a);
  return small ? launch<128, 2>(ctx, a) : launch<128, 1>(ctx, a);
}
