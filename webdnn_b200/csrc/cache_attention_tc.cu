// Attention over a paged 8-bit cache for many new tokens (prompts) on the 5th-generation tensor cores (tcgen05, sm_100a).  The
// mathematics is that of cache_attention.cu: codes are exact in float16, queries and weights are float16 halves, 22 bits together,
// and weights carry the value scale of their page relative to the largest term of the sum.
//
// One CTA owns 128 rows of one sequence and key head, row = new token * group + query head of the group, and walks the tokens that
// they see in chunks of 64:
//   S  = Q K_chunk^T     two tcgen05.mma.kind::f16 products, M = 128, N = 64, K = head size: low half, high half.  Q is the A
//                        operand in TENSOR MEMORY (from shared memory each chunk would read all of it again: 768 cycles of the
//                        ports at 128 bytes), K_chunk the B operand in shared memory
//   P  = weights         by the row threads, in halves to tensor memory, as the next A operand
//   Oc = P V_chunk       two products, M = 128, N = head size, K = 64; V_chunk^T the B operand in shared memory
//   O  = O * keep + Oc   in the row threads' registers, rounded to nearest
// Warps 0-7 are row threads, two of a row (= TMEM lane): each has half of the chunk's scores and half of O's channels, and they
// exchange their maxima through shared memory.  Warps 8-11 bring values in and 12-14 keys, widening the codes to float16 in the tensor
// core's K-major layout with 128-byte swizzle (values transposed on the way), three chunks deep; warp 15 issues the products.  S and P
// have two buffers: while a chunk's rows are turned into weights, the tensor core works on the last chunk's values and the next
// one's scores.
//
// Bound: the chain of a row's weights (scores out of tensor memory, the maximum with the other thread, exponentials, halves), about 2600
// cycles a chunk, of which the tensor pipe needs 1000; 51% of the issue slots are used.  A tile's beginning and end are 10 us.  Measured:
// prompts of up to 900 tokens, three sequences of 450 to 1800, 16 query and 4 key heads of 128: 66 us (234 TFLOP/s).
// Every mbarrier wait is bounded (2 s): on expiry the CTA records a status code, raises its abort flag, frees its TMEM and returns.
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include "cache_attention.cuh"

namespace {

constexpr int BQ = 128, BK = 64, STAGES = 3;
constexpr int ROW_THREADS = 256, VALUE_THREADS = 128, KEY_THREADS = 96, ISSUER = 15, THREADS = 512;
// 128 registers a thread at launch; four groups of four warps: 2 * 160 + 2 * 96 = 4 * 128
constexpr int ROW_REGISTERS = 160, OTHER_REGISTERS = 96;
constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;

struct Shared {
  unsigned long long kv_full[STAGES], kv_empty[STAGES], s_full[2], q_ready, p_ready, o_full;
  float key_scale[STAGES][4], exponent[STAGES][4], fraction[STAGES][4];   // of a chunk's groups of 16 tokens (values: 2^e * f)
  int there[STAGES];                                                      // which of the groups are there
  float2 tops[2][2][BQ];                                                  // maxima of a row's halves, of two chunks
  float row_scale[BQ], sums[BQ];
  int row_stop[2];                                                        // of two chunks: a row thread's wait has expired
  int4 work;                                                              // sequence, tile, length, count
  unsigned int tmem_base;
  volatile int abort_flag;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(unsigned long long* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long global_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Bounded wait.  Returns false if the wait was abandoned (time limit or CTA-wide abort).
__device__ __forceinline__ bool mbar_wait_slow(unsigned long long* bar, uint32_t parity, Shared* sh, int* status, int code) {
  const unsigned long long t0 = global_ns();
  for (;;) {
    for (int i = 0; i < 1024; i++)
      if (mbar_try_wait(bar, parity)) return true;
    if (sh->abort_flag) return false;
    if (global_ns() - t0 > WAIT_LIMIT_NS) {
      sh->abort_flag = 1;
      atomicCAS(status, 0, code);
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, uint32_t parity, Shared* sh, int* status, int code) {
  for (int i = 0; i < 64; i++)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, sh, status, code);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "elect.sync _|P, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(pred));
  return pred != 0;
}
// shared-memory matrix descriptor: K-major, 128-byte swizzle, rows of 128 bytes, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t make_smem_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// instruction descriptor: D = f32, A = B = f16, both K-major, dense, M = 128, N = n
__device__ __forceinline__ uint32_t make_idesc(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
}
__device__ __forceinline__ void umma_one(uint32_t tmem_c, uint32_t tmem_a, uint32_t desc_lo, uint32_t desc_top, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 d;\n\t"
      "mov.b64 d, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], d, %4, p;\n\t}" ::"r"(tmem_c),
      "r"(tmem_a), "r"(desc_lo), "r"(desc_top), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit_one(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void store16(unsigned char* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *reinterpret_cast<uint4*>(p) = make_uint4(a, b, c, d);
}

template <int DH>
struct Tile {
  static constexpr int K_BLOCK = BK * 128;                 // 64 tokens x 64 channels
  static constexpr int KEYS = 0, VALUES = DH / 64 * K_BLOCK, STAGE = 2 * VALUES;
  static constexpr int Q = STAGES * STAGE, Q_STRIDE = 4 * DH + 16;   // queries on their way: a row's high halves, then the low ones
  static constexpr int OUT_STRIDE = DH + 4;                // floats of a row of the result, over all of this at the end
  static constexpr int SMEM = Q + BQ * Q_STRIDE + 1024;
  // tensor-memory columns; S and P of two chunks
  static constexpr int Q_HI = 0, Q_LO = DH / 2, S = DH, P = S + 2 * BK, O = P + 2 * BK, COLS = 512;
  static_assert(BQ * OUT_STRIDE * 4 <= SMEM - 1024, "the result's place");
};

// The rows of a tile that a warp of the row threads reads or writes whole, and a lane's four channels of them.
template <int DH>
struct WholeRows {
  static constexpr int LANES = DH / 4, TOGETHER = 32 / LANES, PASSES = BQ / (ROW_THREADS / 32) / TOGETHER;
  int group, row, token, head, channel;
  __device__ WholeRows(const CacheAttArgs& a, int tile, int warp, int lane) : group(a.group) {
    row = warp * PASSES * TOGETHER + lane / LANES;
    token = (tile * BQ + row) / group;
    head = tile * BQ + row - token * group;
    channel = lane % LANES * 4;
  }
  __device__ void next() {
    row += TOGETHER;
    head += TOGETHER;
    while (head >= group) {
      head -= group;
      token++;
    }
  }
};

// The tile (sequence, tile, length, count), of all sequences', that is number `place` when those with the most chunks come first, so
// that the last CTAs to begin are short; the sequences' last tiles come first otherwise.  Each lane counts the tiles of another number
// of chunks and more.  It costs a CTA 1 us, and is done where more than one wave of CTAs and tiles of 16 chunks and more make it worth
// that, and sequences are at most ORDERED.  Measured, us without / with: three prompts of 900, 750 and 450 tokens behind 900, 375
// and 0, heads of 128 80.6 / 65.9 and of 64 60.1 / 50.7; four of 1000 to 500 behind none 123.5 / 125.4; six of 153 to 83 18.3 / 21.2.
// With more sequences the waves are many, and less is gained than taking a tile costs: up to 900 new tokens of 100 to 1000, 12 sequences
// 139.5 / 151.8 and 24 269 / 324; 300 of 100 to 2000, 12 sequences 113.2 / 104.2 and 24 201 / 216.
constexpr int ORDERED = 8;
__device__ __forceinline__ int4 take_tile(const CacheAttArgs& a, int place, int lane) {
  const int64_t capacity = a.table_pages << a.page_shift;
  CacheSpan span = {0, 0};                         // of sequence `lane`
  if (lane < a.batch) span = cache_span(a.lengths, a.counts, lane, a.tokens, capacity, a.status);
  const int tiles = span.count ? (span.count * a.group - 1) / BQ + 1 : 0;
  // tiles of a sequence that have `least` chunks and more; they are its last ones (0: and those without tokens)
  const auto count = [&](int least, int length, int count, int tiles) {
    if (least == 0) return a.row_tiles;
    const int token = (least - 1) * BK - (length - count);                       // that a tile's last row has to be at least
    return token <= 0 ? tiles : token >= count ? 0 : tiles - token * a.group / BQ;
  };
  int least = 0, width = __reduce_max_sync(0xffffffffu, span.count ? (span.length + BK - 1) / BK : 0) + 1;
  while (width > 1) {
    const int step = (width + 31) / 32, mine = least + min(lane * step, width);
    int sum = 0;
#pragma unroll 4
    for (int s = 0; s < a.batch; s++)
      sum += count(mine, __shfl_sync(0xffffffffu, span.length, s), __shfl_sync(0xffffffffu, span.count, s), __shfl_sync(0xffffffffu, tiles, s));
    least += (31 - __clz(__ballot_sync(0xffffffffu, lane * step < width && (sum > place || lane == 0)))) * step;
    width = step;
  }
  int above = 0, n = 0;
  if (lane < a.batch) {
    above = count(least + 1, span.length, span.count, tiles);
    n = count(least, span.length, span.count, tiles) - above;
  }
  int from = __reduce_add_sync(0xffffffffu, above) - n, up = n;
#pragma unroll
  for (int w = 1; w < ORDERED; w <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, up, w);
    if (lane >= w) up += other;
  }
  from += up;                                      // places before this lane's tiles of `least` chunks
  const int b = __ffs(__ballot_sync(0xffffffffu, place >= from && place < from + n)) - 1;
  const int tile = (least ? tiles - n - above : tiles) + place - from;
  return make_int4(b, __shfl_sync(0xffffffffu, tile, b), __shfl_sync(0xffffffffu, span.length, b), __shfl_sync(0xffffffffu, span.count, b));
}

template <int DH, bool IN_ORDER>
__global__ void __launch_bounds__(THREADS, 1) cache_attention_tc_kernel(const CacheAttArgs a) {
  using T = Tile<DH>;
  using Rows = WholeRows<DH>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Shared sh;
  unsigned char* stages = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&sh.kv_full[s], (VALUE_THREADS + KEY_THREADS) / 32);
      mbar_init(&sh.kv_empty[s], 1);
    }
    mbar_init(&sh.s_full[0], 1);
    mbar_init(&sh.s_full[1], 1);
    mbar_init(&sh.q_ready, ROW_THREADS / 32);
    mbar_init(&sh.p_ready, ROW_THREADS / 32);
    mbar_init(&sh.o_full, 1);
    sh.abort_flag = sh.row_stop[0] = sh.row_stop[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(T::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (IN_ORDER) {
    pdl_wait();
    if (warp == 1) {
      const int4 work = take_tile(a, (int)(blockIdx.x / (unsigned)a.kv_heads), lane);
      if (lane == 0) sh.work = work;
    }
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem_base = sh.tmem_base;
  if (!IN_ORDER) pdl_wait();

  const int bh = (int)(blockIdx.x % (unsigned)(a.batch * a.kv_heads));
  const int tile = IN_ORDER ? sh.work.y : a.row_tiles - 1 - (int)(blockIdx.x / (unsigned)(a.batch * a.kv_heads));
  const int kvh = bh % a.kv_heads, b = IN_ORDER ? sh.work.x : bh / a.kv_heads;
  const CacheSpan span = IN_ORDER ? CacheSpan{sh.work.z, sh.work.w}
                                  : cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages << a.page_shift, a.status);
  const int before = span.length - span.count;
  const int first_token = tile * BQ / a.group, top_token = min((tile * BQ + BQ - 1) / a.group, span.count - 1);
  const int seen = first_token < span.count ? before + top_token + 1 : 0;
  const int seen_by_all = before + first_token + 1;
  const int chunks = (seen + BK - 1) / BK;

  bool ok = true;
  if (warp < ROW_THREADS / 32) {
    // ============================================================================ row threads
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(ROW_REGISTERS));
    constexpr int HALF = DH / 2;                   // channels of O (and of Q, to be stored) a thread
    const uint32_t lane_base = tmem_base + ((uint32_t)(warp % 4 * 32) << 16);
    const int in_tile = (int)threadIdx.x % BQ, half = (int)threadIdx.x / BQ;
    const int token = (tile * BQ + in_tile) / a.group;
    const int last = token < span.count ? before + token : 0x7fffffff;
    {
      // The tile's queries, whole rows by a warp: scaled by a power of two, in halves, through shared memory to tensor memory.  (A
      // loop that is short in code: what runs once waits for its instructions, about as long as they are.)
      Rows rows(a, tile, warp, lane);
#pragma unroll 1
      for (int i = 0; i < Rows::PASSES; i += 4) {
        float4 x[4];
        int r[4];
#pragma unroll
        for (int k = 0; k < 4; k++, rows.next()) {
          r[k] = rows.row;
          x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (rows.token < span.count)
            x[k] = pdl_ld(reinterpret_cast<const float4*>(pdl_after(a.q) + b * a.q_sb + (kvh * a.group + rows.head) * a.q_sh + rows.token * a.q_st + rows.channel));
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float peak = fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
#pragma unroll
          for (int w = 1; w < Rows::LANES; w <<= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, w));
          float row_scale;
          const float up = query_scale(peak, a.scale_log2, row_scale);
          if (rows.channel == 0) sh.row_scale[r[k]] = row_scale;
          uint2 hi, lo;
          split_halves(x[k].x * up, x[k].y * up, hi.x, lo.x);
          split_halves(x[k].z * up, x[k].w * up, hi.y, lo.y);
          unsigned char* to = stages + T::Q + r[k] * T::Q_STRIDE + rows.channel * 2;
          *reinterpret_cast<uint2*>(to) = hi;
          *reinterpret_cast<uint2*>(to + 2 * DH) = lo;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(ROW_THREADS) : "memory");
      // (16 bytes are eight channels, four columns)
      const unsigned char* from = stages + T::Q + in_tile * T::Q_STRIDE + half * DH;
#pragma unroll
      for (int i = 0; i < DH / 16; i += 2) {
#pragma unroll
        for (int part = 0; part < 2; part++) {
          const uint4 x = *reinterpret_cast<const uint4*>(from + part * 2 * DH + i * 16);
          const uint4 y = *reinterpret_cast<const uint4*>(from + part * 2 * DH + i * 16 + 16);
          const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          tmem_st8(lane_base + (uint32_t)((part ? T::Q_LO : T::Q_HI) + half * (DH / 4) + i * 4), w);
        }
      }
      tmem_stored();
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_ready);
    }
    const float row_scale = sh.row_scale[in_tile];
    float o[HALF], m = -INFINITY, big = -INFINITY, l = 0.f, keep = 0.f;
#pragma unroll
    for (int c = 0; c < HALF; c++) o[c] = 0.f;
    const auto add_values = [&](int chunk) {       // O of a chunk, whose weights were relative to `big` of that time
      if (!__all_sync(0xffffffffu, mbar_wait(&sh.o_full, (uint32_t)(chunk & 1), &sh, a.status, 82))) return false;
      after_sync();
#pragma unroll
      for (int c0 = 0; c0 < HALF; c0 += 32) {
        float oc[32];
        tmem_ld16(lane_base + (uint32_t)(T::O + half * HALF + c0), oc);
        tmem_ld16(lane_base + (uint32_t)(T::O + half * HALF + c0 + 16), oc + 16);
        tmem_loaded();
#pragma unroll
        for (int c = 0; c < 32; c++) o[c0 + c] = fmaf(o[c0 + c], keep, oc[c]);
      }
      before_sync();
      return true;
    };
    for (int j = 0; j < chunks; j++) {
      const int st = j % STAGES;
      ok = ok && mbar_wait(&sh.kv_full[st], (uint32_t)(j / STAGES & 1), &sh, a.status, 80) &&
           mbar_wait(&sh.s_full[j & 1], (uint32_t)(j >> 1 & 1), &sh, a.status, 81);
      // (on expiry all row threads leave together, behind the barrier below)
      if (!ok) sh.row_stop[j & 1] = 1;
      __syncwarp();
      after_sync();
      float s[32];
      tmem_ld16(lane_base + (uint32_t)(T::S + (j & 1) * BK + half * 32), s);
      tmem_ld16(lane_base + (uint32_t)(T::S + (j & 1) * BK + half * 32 + 16), s + 16);
      tmem_loaded();
      const int there = sh.there[st] >> (half * 2), t0 = j * BK + half * 32;
      const bool whole = (j + 1) * BK <= seen_by_all && sh.there[st] == 15;
      float by[2], e[2], f[2], top_s = -INFINITY, top_big = -INFINITY;
#pragma unroll
      for (int g = 0; g < 2; g++) {
        by[g] = row_scale * sh.key_scale[st][half * 2 + g];                    // (not negative)
        e[g] = sh.exponent[st][half * 2 + g];
        f[g] = sh.fraction[st][half * 2 + g];
        if (!whole) {
#pragma unroll
          for (int c = g * 16; c < g * 16 + 16; c++)
            if (t0 + c > last || !(there >> g & 1)) s[c] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int c = g * 16; c < g * 16 + 16; c++) top = fmaxf(top, s[c]);
        top = top == -INFINITY ? top : top * by[g];
        top_s = fmaxf(top_s, top);
        top_big = fmaxf(top_big, top + e[g]);
      }
      sh.tops[j & 1][half][in_tile] = make_float2(top_s, top_big);
      asm volatile("bar.sync 1, %0;" ::"n"(ROW_THREADS) : "memory");
      if (((volatile int*)sh.row_stop)[j & 1]) {
        ok = false;
        break;
      }
      const float2 other = sh.tops[j & 1][half ^ 1][in_tile];
      const float m_new = fmaxf(m, fmaxf(top_s, other.x)), big_new = fmaxf(big, fmaxf(top_big, other.y));
      const float m_ref = finite_or_0(m_new), big_ref = finite_or_0(big_new);
      l *= exp2_of(m - m_ref);
      const float keep_new = exp2_of(big - big_ref);
      m = m_new;
      big = big_new;
      const uint32_t to = lane_base + (uint32_t)(T::P + (j & 1) * BK + half * 16);   // (chunk j - 2's values are done: o_full)
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const float weigh = f[g] * exp2_of(fminf(m_ref + e[g] - big_ref + WEIGHT_BITS, 126.f));
        float sum = 0.f;
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const float s0 = s[g * 16 + c], s1 = s[g * 16 + c + 1];
          float p0 = exp2_of(fmaf(s0, by[g], -m_ref)), p1 = exp2_of(fmaf(s1, by[g], -m_ref));
          float w0 = p0 * weigh, w1 = p1 * weigh;
          if (!whole) {                            // (nothing of what the row does not see, not even a scale that is no number)
            if (s0 == -INFINITY) p0 = w0 = 0.f;
            if (s1 == -INFINITY) p1 = w1 = 0.f;
          }
          sum += p0 + p1;
          split_halves(w0, w1, hi[c / 2], lo[c / 2]);
        }
        l += sum;
        tmem_st8(to + (uint32_t)(g * 8), hi);
        tmem_st8(to + (uint32_t)(BK / 2 + g * 8), lo);
      }
      if (j > 0) ok = add_values(j - 1);
      keep = keep_new;
      tmem_stored();
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_ready);
    }
    if (ok && chunks > 0) ok = add_values(chunks - 1);
    // the halves' sums
    if (half) sh.sums[in_tile] = l;
    asm volatile("bar.sync 1, %0;" ::"n"(ROW_THREADS) : "memory");
    if (!half) {
      l += sh.sums[in_tile];
      sh.tops[0][0][in_tile].x = l;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(ROW_THREADS) : "memory");
    l = sh.tops[0][0][in_tile].x;
    // The result through shared memory, so that rows are written whole: every product that reads it has completed.  (Not ok: it may
    // have not, and nothing is written.)
    const float by = l == 0.f ? 0.f : exp2f(big - finite_or_0(m) - WEIGHT_BITS) / l;
    float* out = reinterpret_cast<float*>(stages);
    if (ok && token < span.count) {
#pragma unroll
      for (int c = 0; c < HALF; c += 4)
        *reinterpret_cast<float4*>(out + in_tile * T::OUT_STRIDE + half * HALF + c) = make_float4(o[c] * by, o[c + 1] * by, o[c + 2] * by, o[c + 3] * by);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(ROW_THREADS) : "memory");
    Rows rows(a, tile, warp, lane);
#pragma unroll 1
    for (int i = 0; i < Rows::PASSES; i++, rows.next()) {
      if (!ok || rows.token >= a.tokens) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);                              // (padding)
      if (rows.token < span.count) x = *reinterpret_cast<const float4*>(out + rows.row * T::OUT_STRIDE + rows.channel);
      *reinterpret_cast<float4*>(a.y + b * a.y_sb + (kvh * a.group + rows.head) * a.y_sh + rows.token * a.y_st + rows.channel) = x;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGISTERS));
    const int32_t* table = a.page_table + (int64_t)b * a.table_pages;
    const int64_t block_bytes = (int64_t)DH << a.page_shift, side_bytes = block_bytes * a.kv_heads;
    const int8_t* mine = pdl_after(a.codes) + kvh * block_bytes;
    // Lane g of a warp has the page of a chunk's group g (-1: not there).  A table entry is read two chunks before its codes are
    // fetched, and looked at a chunk later: nothing waits for it.
    const auto entry_of = [&](int j) {
      const int t0 = j * BK + lane * 16;
      return lane < 4 && t0 < seen ? pdl_ld(table + (t0 >> a.page_shift)) : -1;
    };
    const auto page_of = [&](int entry, int j) {
      if (entry >= 0 && entry < a.pages) return entry;
      if (lane < 4 && j * BK + lane * 16 < seen) a.status[WDC_STATUS_CACHE] = 1;
      return -1;
    };
    const auto codes_at = [&](int pages, int j, int in_chunk) -> const int8_t* {        // a token's keys, or null
      const int page = __shfl_sync(0xffffffffu, pages, in_chunk / 16), token = j * BK + in_chunk;
      return page < 0 ? nullptr : mine + (int64_t)page * 2 * side_bytes + (token & ((1 << a.page_shift) - 1)) * DH;
    };
    const auto stage_free = [&](int j) { return mbar_wait(&sh.kv_empty[j % STAGES], (uint32_t)(j / STAGES & 1) ^ 1, &sh, a.status, 83); };
    const auto filled = [&](int st) {                // this warp's part of a stage
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");             // (the tensor core reads what was stored)
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.kv_full[st]);
    };
    const uint32_t flip = 0x80808080u;
    if (warp < (ROW_THREADS + VALUE_THREADS) / 32) {
      // ========================================================================== values: 8 tokens by 8 (or 4) channels a thread
      // row = channel, 128 bytes of 64 tokens, 16-byte pieces exchanged by the row's last three bits
      const int id = (int)threadIdx.x - ROW_THREADS, octet = id & 7, column = id >> 3;
      constexpr int VN = DH / 16, WORDS = VN / 4;
      uint32_t w[8][WORDS];
      const auto load = [&](const int8_t* from) {
#pragma unroll
        for (int r = 0; r < 8; r++)
#pragma unroll
          for (int i = 0; i < WORDS; i++)
            w[r][i] = from ? pdl_ld(reinterpret_cast<const uint32_t*>(from + side_bytes + r * DH + column * VN) + i) : 0u;
      };
      int pages = page_of(entry_of(0), 0), next_entry = entry_of(1);
      float key_scale = 0.f, value_scale = 0.f;      // of group `id` of the chunk, for the first four threads
      const auto load_scales = [&]() {
        key_scale = value_scale = 0.f;
        if (id < 4 && pages >= 0) {
          const float* scales = pdl_after(a.scales) + (int64_t)pages * 2 * a.kv_heads + kvh;
          key_scale = pdl_ld(scales);
          value_scale = pdl_ld(scales + a.kv_heads);
        }
      };
      load_scales();
      load(codes_at(pages, 0, octet * 8));
      for (int j = 0; j < chunks; j++) {
        const int st = j % STAGES;
        ok = stage_free(j);
        if (!ok) break;
        const bool there_now = pages >= 0;
        pages = page_of(next_entry, j + 1);
        next_entry = entry_of(j + 2);
        unsigned char* to = stages + st * T::STAGE + T::VALUES;
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
          uint32_t out[4][4];                                                  // [channel][pair of tokens]
#pragma unroll
          for (int r = 0; r < 8; r += 2) {
            const uint32_t x = w[r][i] ^ flip, y = w[r + 1][i] ^ flip;
            const uint32_t lo = __byte_perm(x, y, 0x5140), hi = __byte_perm(x, y, 0x7362);
            out[0][r / 2] = two_codes<0x4140>(lo);
            out[1][r / 2] = two_codes<0x4342>(lo);
            out[2][r / 2] = two_codes<0x4140>(hi);
            out[3][r / 2] = two_codes<0x4342>(hi);
          }
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int channel = column * VN + i * 4 + c;
            store16(to + channel * 128 + (octet ^ (channel & 7)) * 16, out[c][0], out[c][1], out[c][2], out[c][3]);
          }
        }
        load(codes_at(pages, j + 1, octet * 8));
        if (id < 4) {
          exponent_of(value_scale, sh.exponent[st][id], sh.fraction[st][id]);
          sh.key_scale[st][id] = key_scale_of(key_scale);
          const unsigned there = __ballot_sync(15u, there_now);
          if (id == 0) sh.there[st] = (int)there;
        }
        load_scales();
        filled(st);
      }
    } else if (warp < ISSUER) {
      // ========================================================================== keys: pieces of 16 bytes `part` and `part` + 4 of a
      // token (four threads read 64 bytes of a row), two or three tokens a thread.  row = token, 128 bytes of 64 channels
      const int id = (int)threadIdx.x - ROW_THREADS - VALUE_THREADS, part = id & 3, key0 = id >> 2;
      constexpr int EACH = 3, STEP = KEY_THREADS / 4, PIECES = DH / 64;
      uint4 w[EACH][PIECES];
      const auto load = [&](int n, int pages, int j) {
        const int key = key0 + n * STEP;
        const int8_t* from = codes_at(pages, j, key % BK);
#pragma unroll
        for (int i = 0; i < PIECES; i++)
          w[n][i] = from && key < BK ? pdl_ld(reinterpret_cast<const uint4*>(from) + i * 4 + part) : make_uint4(0, 0, 0, 0);
      };
      int pages = page_of(entry_of(0), 0), next_entry = entry_of(1);
#pragma unroll
      for (int n = 0; n < EACH; n++) load(n, pages, 0);
      for (int j = 0; j < chunks; j++) {
        const int st = j % STAGES;
        ok = stage_free(j);
        if (!ok) break;
        pages = page_of(next_entry, j + 1);
        next_entry = entry_of(j + 2);
#pragma unroll
        for (int n = 0; n < EACH; n++) {
          const int key = key0 + n * STEP;
          if (key < BK) {
#pragma unroll
            for (int i = 0; i < PIECES; i++) {       // (codes 16 (4 i + part) .. : block i, pieces 2 part and 2 part + 1)
              unsigned char* to = stages + st * T::STAGE + T::KEYS + i * T::K_BLOCK + key * 128;
              const uint32_t x = w[n][i].x ^ flip, y = w[n][i].y ^ flip, z = w[n][i].z ^ flip, u = w[n][i].w ^ flip;
              store16(to + ((2 * part) ^ (key & 7)) * 16, two_codes<0x4140>(x), two_codes<0x4342>(x), two_codes<0x4140>(y), two_codes<0x4342>(y));
              store16(to + ((2 * part + 1) ^ (key & 7)) * 16, two_codes<0x4140>(z), two_codes<0x4342>(z), two_codes<0x4140>(u), two_codes<0x4342>(u));
            }
          }
          load(n, pages, j + 1);
        }
        filled(st);
      }
    } else if (elect_one()) {
      // ========================================================================== the products
      const uint32_t idesc_s = make_idesc(BK), idesc_o = make_idesc(DH);
      const auto scores = [&](int j) {
        const int st = j % STAGES;
        if (!mbar_wait(&sh.kv_full[st], (uint32_t)(j / STAGES & 1), &sh, a.status, 84)) return false;
        after_sync();
        const uint64_t desc = make_smem_desc(smem_u32(stages + st * T::STAGE + T::KEYS));
        const uint32_t lo0 = (uint32_t)desc, top = (uint32_t)(desc >> 32), to = tmem_base + T::S + (uint32_t)(j & 1) * BK;
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
          for (int k = 0; k < DH / 16; k++)
            umma_one(to, tmem_base + (uint32_t)((half ? T::Q_HI : T::Q_LO) + k * 8), lo0 + (uint32_t)((k / 4 * T::K_BLOCK + k % 4 * 32) >> 4),
                     top, idesc_s, half | k ? 1u : 0u);
        umma_commit_one(&sh.s_full[j & 1]);
        return true;
      };
      ok = mbar_wait(&sh.q_ready, 0, &sh, a.status, 85);
      after_sync();
      if (ok && chunks > 0) ok = scores(0);
      for (int j = 0; j < chunks && ok; j++) {
        // (the scores that were in the next buffer are weights already: p_ready of chunk j - 1)
        if (j + 1 < chunks) ok = scores(j + 1);
        ok = ok && mbar_wait(&sh.p_ready, (uint32_t)(j & 1), &sh, a.status, 86);
        if (!ok) break;
        after_sync();
        const int st = j % STAGES;
        const uint64_t desc = make_smem_desc(smem_u32(stages + st * T::STAGE + T::VALUES));
        const uint32_t lo0 = (uint32_t)desc, top = (uint32_t)(desc >> 32);
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
          for (int k = 0; k < BK / 16; k++)
            umma_one(tmem_base + T::O, tmem_base + (uint32_t)(T::P + (j & 1) * BK + (half ? 0 : BK / 2) + k * 8), lo0 + (uint32_t)(k * 2), top,
                     idesc_o, half | k ? 1u : 0u);
        umma_commit_one(&sh.kv_empty[st]);
        umma_commit_one(&sh.o_full);
      }
    }
  }
  before_sync();
  __syncthreads();
  if (warp == ISSUER) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(T::COLS));
  }
}

template <int DH, bool IN_ORDER>
int launch(wdc_context* ctx, const CacheAttArgs& a, int64_t ctas) {
  static bool opted_in[64] = {};     // per device: more than 48 KB of dynamic shared memory needs the attribute
  WDC_REQUIRE(ctx, ctx->device >= 0 && ctx->device < 64, "wdc_cache_attention: device index out of range");
  if (!opted_in[ctx->device]) {
    WDC_CUDA(ctx, cudaFuncSetAttribute(cache_attention_tc_kernel<DH, IN_ORDER>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<DH>::SMEM));
    opted_in[ctx->device] = true;
  }
  wdc_launch_pdl(ctx, cache_attention_tc_kernel<DH, IN_ORDER>, dim3((unsigned)ctas), dim3(THREADS), Tile<DH>::SMEM, a);
  ctx->n_tc_launch++;
  return wdc_check_launch(ctx, "cache_attention_tc_kernel");
}

}  // namespace

// WDC_ERR_UNSUPPORTED (nothing written): the caller runs the kernel for few rows, which is as fast at 64 rows of a key head, and at a tile
// of 128 for every fourth SM.  Measured, us here / by the other kernel, heads of 128: 8 sequences and 8 key heads of 500 tokens, 48 rows
// 20.5 / 24.8, 64 rows 20.6 / 18.1, 96 rows 21.0 / 39.6; of 4000 tokens 99.2 / 83.2, 99.2 / 105.7 and 99.6 / 151; 19 sequences 192 / 155,
// 193 / 193 and 193 / 274.  One sequence, tiles of all its key heads: of 600 tokens 32 tiles 23.8 / 26.4, 40 tiles 23.9 / 38.5; of 4000 98.3 /
// 103 and 98.3 / 126; of 20000 455 / 427 and 452 / 531.
int wdc_cache_attention_tc(wdc_context* ctx, CacheAttArgs a, int head_size) {
  if (head_size != 64 && head_size != 128) return WDC_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)a.tokens * a.group;
  a.row_tiles = (int)ceil_div64(rows, BQ);
  const int64_t ctas = (int64_t)a.batch * a.kv_heads * a.row_tiles;
  if (rows < BQ / 2 || rows > INT_MAX - BQ || 4 * ctas < ctx->sm_count || ctas >= (1ll << 31)) return WDC_ERR_UNSUPPORTED;
  const bool in_order = a.batch > 1 && a.batch <= ORDERED && ctas > ctx->sm_count && a.table_pages << a.page_shift >= 16 * BK;
  if (head_size == 64) return in_order ? launch<64, true>(ctx, a, ctas) : launch<64, false>(ctx, a, ctas);
  return in_order ? launch<128, true>(ctx, a, ctas) : launch<128, false>(ctx, a, ctas);
}
