// Attention over a paged 8-bit cache for many new tokens (prompts) on the 5th-generation tensor cores (tcgen05, sm_100a).  The
// mathematics is that of cache_attention.cu: codes are exact in float16, queries and weights are float16 halves, 22 bits together,
// and weights carry the value scale of their page relative to the largest term of the sum.
//
// One CTA owns 128 rows of one sequence and key head, row = new token * group + query head of the group, and walks the tokens that
// they see in chunks of 64:
//   S  = Q K_chunk^T     two tcgen05.mma.kind::f16 products, M = 128, N = 64, K = head size: low half, high half.  Q is the A
//                        operand in TENSOR MEMORY, K_chunk the B operand in shared memory
//   P  = weights         by the 128 row threads (thread r = row r = TMEM lane r), in halves back to tensor memory
//   Oc = P V_chunk       two products, M = 128, N = head size, K = 64; V_chunk^T the B operand in shared memory
//   O  = O * keep + Oc   in the row threads' registers, rounded to nearest
// Warps 0-3 are row threads, 4-7 bring keys and values in and widen the codes to float16 in the tensor core's K-major layout with
// 128-byte swizzle (values transposed on the way), three chunks deep; warp 7 issues the products too.  S has two buffers: while a
// chunk's rows are turned into weights, the tensor core works on the last chunk's values and the next one's scores.
//
// Bound: the row threads, about 18 instructions a score, against 16 cycles of the tensor pipe for four of them; measured below.
// Every mbarrier wait is bounded (2 s): on expiry the CTA records a status code, raises its abort flag, frees its TMEM and returns.
#include <cuda_fp16.h>
#include <math.h>

#include "cache_attention.cuh"

namespace {

constexpr int BQ = 128, BK = 64, STAGES = 3, THREADS = 256;   // (a ninth warp would leave each 168 registers)
constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;

struct Shared {
  unsigned long long kv_full[STAGES], kv_empty[STAGES], s_full[2], q_ready, p_ready, o_full;
  float key_scale[STAGES][4], exponent[STAGES][4], fraction[STAGES][4];   // of a chunk's groups of 16 tokens (values: 2^e * f)
  int there[STAGES];                                                      // which of the groups are there
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
__device__ __noinline__ bool mbar_wait_slow(unsigned long long* bar, uint32_t parity, Shared* sh, int* status, int code) {
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
  static constexpr int SMEM = STAGES * STAGE + 1024;
  // tensor-memory columns
  static constexpr int Q_HI = 0, Q_LO = DH / 2, S = DH, P_HI = S + 2 * BK, P_LO = P_HI + BK / 2, O = P_LO + BK / 2, COLS = 512;
};

template <int DH>
__global__ void __launch_bounds__(THREADS, 1) cache_attention_tc_kernel(const CacheAttArgs a) {
  using T = Tile<DH>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Shared sh;
  unsigned char* stages = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&sh.kv_full[s], 4);
      mbar_init(&sh.kv_empty[s], 1);
    }
    mbar_init(&sh.s_full[0], 1);
    mbar_init(&sh.s_full[1], 1);
    mbar_init(&sh.q_ready, 4);
    mbar_init(&sh.p_ready, 4);
    mbar_init(&sh.o_full, 1);
    sh.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 7) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(T::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem_base = sh.tmem_base;
  pdl_wait();

  // tiles that see the most tokens begin first
  const int bh = (int)(blockIdx.x % (unsigned)(a.batch * a.kv_heads)), tile = a.row_tiles - 1 - (int)(blockIdx.x / (unsigned)(a.batch * a.kv_heads));
  const int kvh = bh % a.kv_heads, b = bh / a.kv_heads;
  const CacheSpan span = cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages << a.page_shift, a.status);
  const int before = span.length - span.count;
  const int first_token = tile * BQ / a.group, top_token = min((tile * BQ + BQ - 1) / a.group, span.count - 1);
  const int seen = first_token < span.count ? before + top_token + 1 : 0;
  const int seen_by_all = before + first_token + 1;
  const int chunks = (seen + BK - 1) / BK;

  bool ok = true;
  if (warp < 4) {
    // ============================================================================ row threads
    const uint32_t lane_base = tmem_base + ((uint32_t)(warp * 32) << 16);
    const int row = tile * BQ + (int)threadIdx.x, token = row / a.group, head = kvh * a.group + row % a.group;
    const int last = token < span.count ? before + token : 0x7fffffff;
    float row_scale;
    {
      const float* qp = pdl_after(a.q) + b * a.q_sb + head * a.q_sh + token * a.q_st;
      float peak = 0.f;
      if (token < span.count) {
#pragma unroll 8
        for (int c = 0; c < DH; c += 4) {
          const float4 x = pdl_ld(reinterpret_cast<const float4*>(qp + c));
          peak = fmaxf(fmaxf(fmaxf(peak, fabsf(x.x)), fmaxf(fabsf(x.y), fabsf(x.z))), fabsf(x.w));
        }
      }
      const float up = query_scale(peak, a.scale_log2, row_scale);
#pragma unroll
      for (int c0 = 0; c0 < DH; c0 += 16) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (token < span.count) x = pdl_ld(reinterpret_cast<const float4*>(qp + c0 + c));
          split_halves(x.x * up, x.y * up, hi[c / 2], lo[c / 2]);
          split_halves(x.z * up, x.w * up, hi[c / 2 + 1], lo[c / 2 + 1]);
        }
        tmem_st8(lane_base + (uint32_t)(T::Q_HI + c0 / 2), hi);
        tmem_st8(lane_base + (uint32_t)(T::Q_LO + c0 / 2), lo);
      }
      tmem_stored();
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_ready);
    }
    float o[DH], m = -INFINITY, big = -INFINITY, l = 0.f, keep = 0.f;
#pragma unroll
    for (int c = 0; c < DH; c++) o[c] = 0.f;
    const auto add_values = [&](int chunk) {       // O of a chunk, whose weights were relative to `big` of that time
      if (!mbar_wait(&sh.o_full, (uint32_t)(chunk & 1), &sh, a.status, 82)) return false;
      after_sync();
#pragma unroll
      for (int c0 = 0; c0 < DH; c0 += 32) {
        float oc[32];
        tmem_ld16(lane_base + (uint32_t)(T::O + c0), oc);
        tmem_ld16(lane_base + (uint32_t)(T::O + c0 + 16), oc + 16);
        tmem_loaded();
#pragma unroll
        for (int c = 0; c < 32; c++) o[c0 + c] = fmaf(o[c0 + c], keep, oc[c]);
      }
      before_sync();
      return true;
    };
    for (int j = 0; j < chunks; j++) {
      const int st = j % STAGES;
      ok = mbar_wait(&sh.kv_full[st], (uint32_t)(j / STAGES & 1), &sh, a.status, 80) &&
           mbar_wait(&sh.s_full[j & 1], (uint32_t)(j >> 1 & 1), &sh, a.status, 81);
      if (!ok) break;
      after_sync();
      float s[BK];
#pragma unroll
      for (int c0 = 0; c0 < BK; c0 += 16) tmem_ld16(lane_base + (uint32_t)(T::S + (j & 1) * BK + c0), s + c0);
      tmem_loaded();
      float e[4], f[4], m_new = m, big_new = big;
      const int there = sh.there[st];
      const bool whole = (j + 1) * BK <= seen_by_all && there == 15;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const float by = row_scale * sh.key_scale[st][g];
        e[g] = sh.exponent[st][g];
        f[g] = sh.fraction[st][g];
#pragma unroll
        for (int c = g * 16; c < g * 16 + 16; c++) s[c] *= by;
      }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < BK; c++)
          if (j * BK + c > last || !(there >> (c / 16) & 1)) s[c] = -INFINITY;
      }
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float top = s[g * 16];
#pragma unroll
        for (int c = 1; c < 16; c++) top = fmaxf(top, s[g * 16 + c]);
        m_new = fmaxf(m_new, top);
        big_new = fmaxf(big_new, top + e[g]);
      }
      const float m_ref = finite_or_0(m_new), big_ref = finite_or_0(big_new);
      l *= exp2_of(m - m_ref);
      const float keep_new = exp2_of(big - big_ref);
      m = m_new;
      big = big_new;
      uint32_t hi[BK / 2], lo[BK / 2];
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const float by = f[g] * exp2_of(fminf(m_ref + e[g] - big_ref + WEIGHT_BITS, 126.f));
        float sum = 0.f;
#pragma unroll
        for (int c = g * 16; c < g * 16 + 16; c += 2) {
          const float p0 = exp2_of(s[c] - m_ref), p1 = exp2_of(s[c + 1] - m_ref);
          sum += p0 + p1;
          float w0 = p0 * by, w1 = p1 * by;
          if (!whole) {                            // (a scale that is no number is for the rows that see it)
            w0 = s[c] == -INFINITY ? 0.f : w0;
            w1 = s[c + 1] == -INFINITY ? 0.f : w1;
          }
          split_halves(w0, w1, hi[c / 2], lo[c / 2]);
        }
        l += sum;
      }
      if (j > 0) {
        ok = add_values(j - 1);
        if (!ok) break;
      }
      keep = keep_new;
#pragma unroll
      for (int c = 0; c < BK / 2; c += 8) {
        tmem_st8(lane_base + (uint32_t)(T::P_HI + c), hi + c);
        tmem_st8(lane_base + (uint32_t)(T::P_LO + c), lo + c);
      }
      tmem_stored();
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_ready);
    }
    if (ok && chunks > 0) ok = add_values(chunks - 1);
    if (ok && row < a.tokens * a.group) {
      const float by = l == 0.f || token >= span.count ? 0.f : exp2f(big - finite_or_0(m) - WEIGHT_BITS) / l;
      const bool some = by != 0.f || token < span.count;     // (padding: 0, whatever the sums are)
      float* y = a.y + b * a.y_sb + head * a.y_sh + token * a.y_st;
#pragma unroll
      for (int c = 0; c < DH; c += 4)
        *reinterpret_cast<float4*>(y + c) = some ? make_float4(o[c] * by, o[c + 1] * by, o[c + 2] * by, o[c + 3] * by)
                                                 : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    // ============================================================================ keys and values
    const int id = (int)threadIdx.x - 128;
    const int32_t* table = a.page_table + (int64_t)b * a.table_pages;
    const int64_t block_bytes = (int64_t)DH << a.page_shift, side_bytes = block_bytes * a.kv_heads;
    // keys: a thread takes half a head of one token (or all of it in two threads' stead); values: 8 tokens, 8 channels
    const int key = id & 63, part = id >> 6, octet = id & 7, column = id >> 3;
    constexpr int KW = DH / 8, VN = DH == 128 ? 8 : 4;               // words of a key half; channels of a value octet
    const auto at = [&](int token) -> const int8_t* {                // a token's keys, or null
      if (token >= seen) return nullptr;
      const int page = cache_page(table, token >> a.page_shift, a.pages, a.status);
      if (page < 0) return nullptr;
      return a.codes + ((int64_t)page * 2 * a.kv_heads + kvh) * block_bytes + (token & ((1 << a.page_shift) - 1)) * DH;
    };
    uint32_t kw[KW], vw[8][VN / 4];
    const auto load = [&](int j) {
      const int8_t* k = j < chunks ? at(j * BK + key) : nullptr;
      const int8_t* v = j < chunks ? at(j * BK + octet * 8) : nullptr;
#pragma unroll
      for (int i = 0; i < KW; i += 4) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (k) x = pdl_ld(reinterpret_cast<const uint4*>(pdl_after(k) + part * (DH / 2) + i * 4));
        kw[i] = x.x; kw[i + 1] = x.y; kw[i + 2] = x.z; kw[i + 3] = x.w;
      }
#pragma unroll
      for (int r = 0; r < 8; r++)
#pragma unroll
        for (int i = 0; i < VN / 4; i++)
          vw[r][i] = v ? pdl_ld(reinterpret_cast<const uint32_t*>(pdl_after(v) + side_bytes + r * DH + column * VN) + i) : 0u;
    };
    const auto convert = [&](int j) {
      const int st = j % STAGES;
      if (!mbar_wait(&sh.kv_empty[st], (uint32_t)(j / STAGES & 1) ^ 1, &sh, a.status, 83)) return false;
      unsigned char* stage = stages + st * T::STAGE;
      // keys: row = token, 128 bytes of 64 channels, 16-byte pieces exchanged by the row's last three bits
      uint32_t w[KW][2];
#pragma unroll
      for (int i = 0; i < KW; i++) {
        const uint32_t u = kw[i] ^ 0x80808080u;
        w[i][0] = two_codes<0x4140>(u);
        w[i][1] = two_codes<0x4342>(u);
      }
#pragma unroll
      for (int i = 0; i < KW; i += 2) {
        const int channel = part * (DH / 2) + i * 4;                 // of the piece's eight
        store16(stage + T::KEYS + channel / 64 * T::K_BLOCK + key * 128 + ((channel % 64 / 8) ^ (key & 7)) * 16, w[i][0], w[i][1],
                w[i + 1][0], w[i + 1][1]);
      }
      // values: row = channel, 128 bytes of 64 tokens
#pragma unroll
      for (int i = 0; i < VN / 4; i++) {
        uint32_t out[4][4];                                          // [channel][pair of tokens]
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          const uint32_t x = vw[r][i] ^ 0x80808080u, y = vw[r + 1][i] ^ 0x80808080u;
          const uint32_t lo = __byte_perm(x, y, 0x5140), hi = __byte_perm(x, y, 0x7362);
          out[0][r / 2] = two_codes<0x4140>(lo);
          out[1][r / 2] = two_codes<0x4342>(lo);
          out[2][r / 2] = two_codes<0x4140>(hi);
          out[3][r / 2] = two_codes<0x4342>(hi);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int channel = column * VN + i * 4 + c;
          store16(stage + T::VALUES + channel * 128 + (octet ^ (channel & 7)) * 16, out[c][0], out[c][1], out[c][2], out[c][3]);
        }
      }
      if (id < 4) {
        const int t0 = j * BK + id * 16;
        const int page = t0 < seen ? cache_page(table, t0 >> a.page_shift, a.pages, a.status) : -1;
        const float* scales = pdl_after(a.scales) + (int64_t)max(page, 0) * 2 * a.kv_heads + kvh;
        float e, f;
        exponent_of(page >= 0 ? pdl_ld(scales + a.kv_heads) : 0.f, e, f);
        sh.key_scale[st][id] = page >= 0 ? pdl_ld(scales) : 0.f;
        sh.exponent[st][id] = e;
        sh.fraction[st][id] = f;
        const unsigned there = __ballot_sync(15u, page >= 0);
        if (id == 0) sh.there[st] = (int)there;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor core reads what was stored here
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.kv_full[st]);
      load(j + 1);
      return true;
    };
    load(0);
    if (warp < 7) {
      for (int j = 0; j < chunks && ok; j++) ok = convert(j);
    } else {
      // ========================================================================== the products
      const uint32_t idesc_s = make_idesc(BK), idesc_o = make_idesc(DH);
      const auto scores = [&](int j) {
        const int st = j % STAGES;
        if (!mbar_wait(&sh.kv_full[st], (uint32_t)(j / STAGES & 1), &sh, a.status, 84)) return false;
        after_sync();
        const uint64_t desc = make_smem_desc(smem_u32(stages + st * T::STAGE + T::KEYS));
        const uint32_t lo0 = (uint32_t)desc, top = (uint32_t)(desc >> 32), to = tmem_base + T::S + (uint32_t)(j & 1) * BK;
        if (elect_one()) {
#pragma unroll
          for (int half = 0; half < 2; half++)
#pragma unroll
            for (int k = 0; k < DH / 16; k++)
              umma_one(to, tmem_base + (half ? T::Q_HI : T::Q_LO) + (uint32_t)(k * 8),
                       lo0 + (uint32_t)((k / 4 * T::K_BLOCK + k % 4 * 32) >> 4), top, idesc_s, half | k ? 1u : 0u);
          umma_commit_one(&sh.s_full[j & 1]);
        }
        __syncwarp();
        return true;
      };
      if (chunks > 0) ok = convert(0);
      if (ok && chunks > 1) ok = convert(1);
      ok = ok && mbar_wait(&sh.q_ready, 0, &sh, a.status, 85);
      after_sync();
      if (ok && chunks > 0) ok = scores(0);
      if (ok && chunks > 1) ok = scores(1);
      for (int j = 0; j < chunks && ok; j++) {
        if (j + 2 < chunks) ok = convert(j + 2);
        ok = ok && mbar_wait(&sh.p_ready, (uint32_t)(j & 1), &sh, a.status, 86);
        if (!ok) break;
        after_sync();
        const int st = j % STAGES;
        const uint64_t desc = make_smem_desc(smem_u32(stages + st * T::STAGE + T::VALUES));
        const uint32_t lo0 = (uint32_t)desc, top = (uint32_t)(desc >> 32);
        if (elect_one()) {
#pragma unroll
          for (int half = 0; half < 2; half++)
#pragma unroll
            for (int k = 0; k < BK / 16; k++)
              umma_one(tmem_base + T::O, tmem_base + (half ? T::P_HI : T::P_LO) + (uint32_t)(k * 8), lo0 + (uint32_t)(k * 2), top,
                       idesc_o, half | k ? 1u : 0u);
          umma_commit_one(&sh.kv_empty[st]);
          umma_commit_one(&sh.o_full);
        }
        __syncwarp();
        // (chunk j's scores are weights: their buffer is free)
        if (j + 2 < chunks) ok = scores(j + 2);
      }
    }
  }
  before_sync();
  __syncthreads();
  if (warp == 7) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(T::COLS));
  }
}

template <int DH>
int launch(wdc_context* ctx, const CacheAttArgs& a, int64_t ctas) {
  static bool opted_in[64] = {};     // per device: more than 48 KB of dynamic shared memory needs the attribute
  WDC_REQUIRE(ctx, ctx->device >= 0 && ctx->device < 64, "wdc_cache_attention: device index out of range");
  if (!opted_in[ctx->device]) {
    WDC_CUDA(ctx, cudaFuncSetAttribute(cache_attention_tc_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<DH>::SMEM));
    opted_in[ctx->device] = true;
  }
  wdc_launch_pdl(ctx, cache_attention_tc_kernel<DH>, dim3((unsigned)ctas), dim3(THREADS), Tile<DH>::SMEM, a);
  ctx->n_tc_launch++;
  return wdc_check_launch(ctx, "cache_attention_tc_kernel");
}

}  // namespace

// WDC_ERR_UNSUPPORTED (nothing written): the caller runs the kernel for few rows.
int wdc_cache_attention_tc(wdc_context* ctx, CacheAttArgs a, int head_size) {
  if (head_size != 64 && head_size != 128) return WDC_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)a.tokens * a.group;
  a.row_tiles = (int)ceil_div64(rows, BQ);
  const int64_t ctas = (int64_t)a.batch * a.kv_heads * a.row_tiles;
  if (rows < BQ / 2 || 4 * ctas < ctx->sm_count || ctas >= (1ll << 31)) return WDC_ERR_UNSUPPORTED;
  return head_size == 64 ? launch<64>(ctx, a, ctas) : launch<128>(ctx, a, ctas);
}
