// Writing to a paged cache in 8 bits: the new tokens' keys and values (wdc_cache_append), with the keys' norms and rotations on the way
// (wdc_cache_append_rotary), and copies of pages (wdc_cache_copy_pages).  None has a counterpart in the reference.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "head_rotation.cuh"

namespace {


struct AppendArgs {
  const float *k, *v;
  int8_t* codes;
  float* scales;
  const int32_t *page_table, *lengths, *counts;
  int* status;
  int64_t pages, table_pages;
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int tokens, kv_heads, page_shift, quad_shift;   // 2^page_shift tokens a page, 2^quad_shift float4 a head
};
struct RotaryAppendArgs : AppendArgs {
  HeadRotation rotation;
  const float *q, *q_weight, *k_weight;
  float* y;
  int64_t q_sb, q_sh, q_st, y_sb, y_sh, y_st;
  int heads, chunks;               // of q, and groups that take a row of them
};

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ int quantise(float x, float scale) {
  const float r = rintf(__fdiv_rn(x, scale));
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)(d & 255) << 24;
}
// Four codes rint(x / scale) without a division where it cannot matter: x * (1 / scale) is within 3e-5 of the rounded quotient
// (|x / scale| <= 127, three roundings of 2^-24), so where it is further than that from a half the nearest whole number is
// the same, and is read off the sum with 1.5 * 2^23, whose last bits are that number.  About one quadruple in 1200 divides.
// inverse: 0 where 1 / scale might leave the normal range.
__device__ __forceinline__ uint32_t quantise4(float4 x, float scale, float inverse) {
  const float magic = 12582912.f;
  const float4 t = make_float4(x.x * inverse, x.y * inverse, x.z * inverse, x.w * inverse);
  const float4 r = make_float4(t.x + magic, t.y + magic, t.z + magic, t.w + magic);
  const float off = fmaxf(fmaxf(fabsf(t.x - (r.x - magic)), fabsf(t.y - (r.y - magic))),
                          fmaxf(fabsf(t.z - (r.z - magic)), fabsf(t.w - (r.w - magic))));
  if (off < 0.4999f && inverse > 0.f)
    return __byte_perm(__byte_perm(__float_as_uint(r.x), __float_as_uint(r.y), 0x0040),
                       __byte_perm(__float_as_uint(r.z), __float_as_uint(r.w), 0x0040), 0x5410);
  return pack4(quantise(x.x, scale), quantise(x.y, scale), quantise(x.z, scale), quantise(x.w, scale));
}

// Normalises and rotates the keys that a thread holds, in 64 bits: f[j] and f[j + 1] are the two float4 of a slot of a head.  Slot number
// i = threadIdx.x + j / 2 * APPEND_THREADS of `n` is slot i % 2^(quad_shift - 1) of the head of new token row0 + (i >> (quad_shift - 1)),
// whose place in its sequence is `start` further on.
template <int APPEND_THREADS, int HELD>
__device__ __forceinline__ void rotate_keys(const RotaryAppendArgs& a, float4 (&f)[HELD], int n, int row0, int start, int b) {
  const HeadRotation& r = a.rotation;
  const int shift = a.quad_shift - 1, p = threadIdx.x & ((1 << shift) - 1);
  const Slot slot(r, p);
  int64_t position[HELD / 2];
#pragma unroll
  for (int j = 0; j < HELD / 2; j++) {
    const int i = threadIdx.x + j * APPEND_THREADS, row = row0 + (i >> shift);
    position[j] = i >= n || r.half == 0 ? 0 : r.positions ? (int64_t)pdl_ld(r.positions + (int64_t)b * a.tokens + row) : start + row;
  }
  Quad<double> wa[1] = {}, wb[1] = {};
  if (a.k_weight) {
    wa[0] = quad_of<double>(pdl_ld(reinterpret_cast<const float4*>(a.k_weight) + slot.a));
    wb[0] = quad_of<double>(pdl_ld(reinterpret_cast<const float4*>(a.k_weight) + slot.b));
  }
#pragma unroll
  for (int j = 0; j < HELD / 2; j++) {
    if (j * APPEND_THREADS >= n) break;            // (nobody has any)
    Quad<double> na[1] = {quad_of<double>(f[2 * j])}, nb[1] = {quad_of<double>(f[2 * j + 1])};
    if (a.k_weight) normalise(r, na, nb, 1 << shift, wa, wb);
    if (slot.turns) rotate_slot(r, na[0], nb[0], rotation_angles<double>(r, rotation_place(r, position[j], a.status), p));
    f[2 * j] = rounded(na[0]);
    f[2 * j + 1] = rounded(nb[0]);
  }
}

// Queries: a group of 2^(quad_shift - 1) lanes takes EACH heads of a row, of the call's rows with number slot * 2^page_shift and up; rows
// of padding become zero.
template <int EACH>
__device__ __forceinline__ void append_queries(const RotaryAppendArgs& a, int part, int slot, int b) {
  const int shift = a.quad_shift - 1, lanes = 1 << shift;
  const int row0 = slot << a.page_shift, rows = min(a.tokens - row0, 1 << a.page_shift);
  const int item = (part * (int)blockDim.x + (int)threadIdx.x) >> shift, in_slot = item / a.chunks;
  const bool there = in_slot < rows;
  if (!__any_sync(0xffffffffu, there)) return;
  const CacheSpan span = cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages << a.page_shift, a.status);
  const int row = there ? row0 + in_slot : row0, head0 = there ? (item - in_slot * a.chunks) * EACH : 0;
  const int heads = there ? min(EACH, a.heads - head0) : 0;
  const bool padding = row >= span.count;
  const HeadRotation& r = a.rotation;
  const int64_t position = padding || r.half == 0 ? 0 : r.positions ? (int64_t)pdl_ld(r.positions + (int64_t)b * a.tokens + row)
                                                                    : span.length - span.count + row;
  rotate_heads_of<1, EACH>(r, pdl_after(a.q) + b * a.q_sb + row * a.q_st + head0 * a.q_sh, a.q_sh, a.y + b * a.y_sb + row * a.y_st + head0 * a.y_sh, a.y_sh,
                           padding ? 0 : heads, heads, threadIdx.x & (lanes - 1), lanes, 2 * lanes, a.q_weight, position, a.status);
}

// One CTA per (sequence, touched page, head, keys or values): max |x| of the page's new tokens, the page's scale, the codes.
// Absolute values are compared as bits, in which a NaN is above infinity: either one becomes the scale.  The new numbers are read
// once and wait in registers for their scale, HELD float4 a thread (a whole page).  Bound: for prompts the length of a CTA's
// dependent loads (9131 tokens of 8 heads of 128: 18.6 us, 4.9 TB/s), as for single tokens (64 x 1: 2.2 us).
//
// With rotations a thread has float4 in twos, the slots of a head, whose channels are rotated together; and further CTAs take the
// queries of as many tokens as a page has.  Bound: the CTAs' chains and their instructions (five prompts of up to 2001 tokens, 24 query, 8
// key heads of 64: 33.2 us, 4.0 TB/s; 64 new tokens, 32 query, 8 key heads of 128: 3.9), so that 1024 threads an SM are worth the
// registers that they leave in local memory, 252 bytes of stores and 292 of loads a thread that holds 8 float4 (33.2 against 34.6 of 768 and
// 42.8 of 512; heads of 128 in pages of 64 42.3, 44.1, 55.0).  Without rotations there are none.
template <int APPEND_THREADS, int HELD, class Args>
__global__ void __launch_bounds__(APPEND_THREADS, std::is_same<Args, RotaryAppendArgs>::value ? 1024 / APPEND_THREADS : 0) cache_append_kernel(const Args a) {
  constexpr bool ROTARY = std::is_same<Args, RotaryAppendArgs>::value;
  pdl_wait();
  const int part = (int)blockIdx.x, slot = (int)blockIdx.y, b = (int)blockIdx.z;
  if constexpr (ROTARY) {
    if (part >= 2 * a.kv_heads) {
      append_queries<HELD / 2>(a, part - 2 * a.kv_heads, slot, b);
      return;
    }
  }
  const int is_v = part >= a.kv_heads, head = part - is_v * a.kv_heads;
  const CacheSpan span = cache_span(a.lengths, a.counts, b, a.tokens, a.table_pages << a.page_shift, a.status);
  if (span.count == 0) return;
  const int start = span.length - span.count, index = (start >> a.page_shift) + slot;
  const int first = index << a.page_shift;                       // the page's first token
  if (first >= span.length) return;
  const int page = pdl_ld(a.page_table + (int64_t)b * a.table_pages + index);   // (looked at when the new numbers are on their way)
  const int lo = max(start, first), hi = min(span.length, first + (1 << a.page_shift));
  const float* x = is_v ? pdl_after(a.v) + b * a.v_sb + head * a.v_sh + (lo - start) * a.v_st
                        : pdl_after(a.k) + b * a.k_sb + head * a.k_sh + (lo - start) * a.k_st;
  const int64_t row = is_v ? a.v_st : a.k_st;
  const int n = (hi - lo) << a.quad_shift, quad = (1 << a.quad_shift) - 1;      // float4 of the new tokens
  __shared__ uint32_t peaks[APPEND_THREADS / 32];
  uint32_t peak = 0;
  // where float4 number j of this thread is: which of the new tokens' float4, at or behind n: none
  const auto held = [&](int j) {
    const int i = threadIdx.x + (ROTARY ? j / 2 : j) * APPEND_THREADS;
    if constexpr (ROTARY) {
      const Slot slot(a.rotation, i & (quad >> 1));
      return (i >> (a.quad_shift - 1) << a.quad_shift) + (j & 1 ? slot.b : slot.a);
    }
    return i;
  };
  float4 f[HELD];
#pragma unroll
  for (int j = 0; j < HELD; j++) {
    const int i = held(j);
    f[j] = i < n ? pdl_ld(reinterpret_cast<const float4*>(x + (i >> a.quad_shift) * row) + (i & quad)) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (page < 0 || page >= a.pages) {
    a.status[WDC_STATUS_CACHE] = 1;
    return;
  }
  if constexpr (ROTARY) {
    if (!is_v && (a.k_weight || a.rotation.half)) rotate_keys<APPEND_THREADS, HELD>(a, f, n >> 1, lo - start, start, b);
  }
  const int64_t block = ((int64_t)page * 2 + is_v) * a.kv_heads + head;
  uint32_t* codes = reinterpret_cast<uint32_t*>(a.codes) + (block << (a.page_shift + a.quad_shift));
  const float before = lo > first ? pdl_ld(a.scales + block) : 0.f;
#pragma unroll
  for (int j = 0; j < HELD; j++)
    peak = max(max(max(peak, abs_bits(f[j].x)), max(abs_bits(f[j].y), abs_bits(f[j].z))), abs_bits(f[j].w));
  peak = __reduce_max_sync(0xffffffffu, peak);
  if ((threadIdx.x & 31) == 0) peaks[threadIdx.x >> 5] = peak;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < APPEND_THREADS / 32; i++) peak = max(peak, peaks[i]);
  const float fresh = __fdiv_rn(__uint_as_float(peak), 127.f);
  const float scale = lo > first && !(fresh > before) && fresh == fresh ? before : fresh;
  const bool usable = scale > 0.f && scale < INFINITY;            // (all zero, or it stands for NaN: codes of 0)
  const float inverse = scale > 1e-30f ? __frcp_rn(scale) : 0.f;

  if (lo > first && scale > before) {
    const int old = (lo - first) << a.quad_shift;
    for (int i = threadIdx.x; i < old; i += APPEND_THREADS) {
      const uint32_t w = pdl_ld(codes + i);
      int c[4];
#pragma unroll
      for (int j = 0; j < 4; j++) c[j] = usable ? quantise(__fmul_rn((float)(int8_t)(w >> (8 * j)), before), scale) : 0;
      codes[i] = pack4(c[0], c[1], c[2], c[3]);
    }
  }
  uint32_t* to = codes + ((lo - first) << a.quad_shift);
#pragma unroll
  for (int j = 0; j < HELD; j++) {
    const int i = held(j);
    if (i < n) to[i] = usable ? quantise4(f[j], scale, inverse) : 0u;
  }
  if (threadIdx.x == 0) a.scales[block] = scale;
}

// ------------------------------------------------------------------------------------------- copies
// Bound: memory (150 pages of 24 layers, 944 MB read and written: 143.5 us, 6.6 TB/s); the launch for a few (1.7 us).
constexpr int COPY_THREADS = 256, COPY_EACH = 4, COPY_PIECE = COPY_THREADS * COPY_EACH;   // uint4 a CTA
constexpr int COPY_PAIRS = 480;            // that fit a launch's arguments (4 KB)

struct CopyArgs {
  uint4* codes;
  float* scales;
  int64_t page_units, layer_units;         // uint4 of a page, and of a layer
  int64_t layer_scales;
  int page_scales, pieces, n;
  int32_t from[COPY_PAIRS], to[COPY_PAIRS];
};

__global__ void __launch_bounds__(COPY_THREADS) cache_copy_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  const int64_t at = blockIdx.x;
  const int piece = (int)(at % a.pieces), pair = (int)(at / a.pieces % a.n);
  const int64_t layer = at / a.pieces / a.n;
  const uint4* from = pdl_after(a.codes) + layer * a.layer_units + a.from[pair] * a.page_units;
  uint4* to = a.codes + layer * a.layer_units + a.to[pair] * a.page_units;
  uint4 v[COPY_EACH];
  int64_t i = (int64_t)piece * COPY_PIECE + threadIdx.x;
#pragma unroll
  for (int j = 0; j < COPY_EACH; j++)
    if (i + j * COPY_THREADS < a.page_units) v[j] = pdl_ld(from + i + j * COPY_THREADS);
#pragma unroll
  for (int j = 0; j < COPY_EACH; j++)
    if (i + j * COPY_THREADS < a.page_units) to[i + j * COPY_THREADS] = v[j];
  if (piece == 0) {
    const float* s = pdl_after(a.scales) + layer * a.layer_scales + (int64_t)a.from[pair] * a.page_scales;
    float* t = a.scales + layer * a.layer_scales + (int64_t)a.to[pair] * a.page_scales;
    for (int k = threadIdx.x; k < a.page_scales; k += COPY_THREADS) t[k] = pdl_ld(s + k);
  }
}

}  // namespace

// What both kinds of append check and fill in; *slots: pages that a sequence may touch.
static int append_args(wdc_context* ctx, const char* who, const wdc_cache_append_desc* d, AppendArgs& a, const float* k, const float* v, void* codes,
                       float* scales, const int32_t* page_table, const int32_t* lengths, const int32_t* counts, int64_t* slots) {
  CACHE_TRY(cache_check_pool(ctx, who, d->pages, d->kv_heads, d->page_tokens, d->head_size));
  CACHE_TRY(cache_check_batch(ctx, who, d->batch, d->tokens, d->table_pages, d->page_tokens));
  const int64_t strides[6] = {d->k_sb, d->k_sh, d->k_st, d->v_sb, d->v_sh, d->v_st};
  CACHE_TRY(cache_check_strides(ctx, who, strides, 6));
  *slots = 0;
  if (d->batch == 0 || d->tokens == 0) return WDC_OK;
  WDC_REQUIRE(ctx, k && v && codes && scales && lengths && (page_table || d->table_pages == 0), "%s: null argument", who);
  WDC_REQUIRE(ctx, cache_aligned(k, 16) && cache_aligned(v, 16) && cache_aligned(codes, 16) && cache_aligned(scales, 4) &&
              cache_aligned(page_table, 4) && cache_aligned(lengths, 4) && cache_aligned(counts, 4),
              "%s: buffers are not aligned", who);
  a = {k, v, (int8_t*)codes, scales, page_table, lengths, counts, ctx->status_word, d->pages, d->table_pages,
       d->k_sb, d->k_sh, d->k_st, d->v_sb, d->v_sh, d->v_st, (int)d->tokens, (int)d->kv_heads, 4, 3};
  while (1 << a.page_shift < d->page_tokens) a.page_shift++;
  while (4 << a.quad_shift < d->head_size) a.quad_shift++;
  *slots = (d->tokens + d->page_tokens - 2) / d->page_tokens + 1;
  WDC_REQUIRE(ctx, *slots <= 65535 && d->batch <= 65535, "%s: batch exceeds the grid", who);
  return WDC_OK;
}

template <class Args>
static int append_launch(wdc_context* ctx, const wdc_cache_append_desc* d, const Args& args, int64_t slots) {
  // float4 of a page's new tokens a thread: of all its tokens, or of as many as the call can bring
  const int64_t most = (d->tokens < d->page_tokens ? d->tokens : d->page_tokens) * d->head_size / 4;
  DeviceGuard g(ctx->device);
  const auto launch = [&](auto kernel, int threads, int held) {
    Args a = args;
    int64_t parts = 2 * d->kv_heads;
    if constexpr (std::is_same<Args, RotaryAppendArgs>::value) {
      a.chunks = (a.heads + held / 2 - 1) / (held / 2);
      parts += ceil_div64((d->tokens < d->page_tokens ? d->tokens : d->page_tokens) * a.chunks << (a.quad_shift - 1), threads);
    }
    wdc_launch_pdl(ctx, kernel, dim3((unsigned)parts, (unsigned)slots, (unsigned)d->batch), dim3((unsigned)threads), 0, a);
  };
  // (few threads with many loads each on their way, where a page has them: 1024 by 128 threads 16.7 us, by 256 22.0, by 64 18.1; 4096 by
  // 512 19.9, by 256 21.4; 256 by 64 11.5, by 128 12.0)
  constexpr bool ROTARY = std::is_same<Args, RotaryAppendArgs>::value;
  if (most <= 64) launch(cache_append_kernel<ROTARY ? 32 : 64, ROTARY ? 2 : 1, Args>, ROTARY ? 32 : 64, ROTARY ? 2 : 1);
  else if (most <= 256) launch(cache_append_kernel<64, 4, Args>, 64, 4);
  else if (most <= 1024) launch(cache_append_kernel<128, 8, Args>, 128, 8);
  else if (most <= 2048) launch(cache_append_kernel<256, 8, Args>, 256, 8);
  else launch(cache_append_kernel<512, 8, Args>, 512, 8);
  return wdc_check_launch(ctx, "cache_append_kernel");
}

extern "C" int wdc_cache_append(wdc_context* ctx, const wdc_cache_append_desc* d, const float* k, const float* v, void* codes,
                                float* scales, const int32_t* page_table, const int32_t* lengths, const int32_t* counts) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_cache_append: null context");
  WDC_TAPE(ctx, wdc_cache_append, tape_desc(d), k, v, codes, scales, page_table, lengths, counts);
  wdc_note_write(ctx, codes);
  wdc_note_write(ctx, scales);
  WDC_REQUIRE(ctx, d, "wdc_cache_append: null argument");
  AppendArgs a;
  int64_t slots = 0;
  CACHE_TRY(append_args(ctx, "wdc_cache_append", d, a, k, v, codes, scales, page_table, lengths, counts, &slots));
  return slots ? append_launch(ctx, d, a, slots) : WDC_OK;
}

extern "C" int wdc_cache_append_rotary(wdc_context* ctx, const wdc_cache_append_rotary_desc* d, const float* q, const float* k,
                                       const float* v, const float* q_weight, const float* k_weight, const float* cos,
                                       const float* sin, const int32_t* positions, void* codes, float* scales,
                                       const int32_t* page_table, const int32_t* lengths, const int32_t* counts, float* q_out) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_cache_append_rotary: null context");
  WDC_TAPE(ctx, wdc_cache_append_rotary, tape_desc(d), q, k, v, q_weight, k_weight, cos, sin, positions, codes, scales, page_table,
           lengths, counts, q_out);
  wdc_note_write(ctx, codes);
  wdc_note_write(ctx, scales);
  wdc_note_write(ctx, q_out);
  const char* who = "wdc_cache_append_rotary";
  WDC_REQUIRE(ctx, d, "%s: null argument", who);
  RotaryAppendArgs a = {};
  int64_t slots = 0;
  CACHE_TRY(append_args(ctx, who, &d->append, a, k, v, codes, scales, page_table, lengths, counts, &slots));
  CACHE_TRY(rotation_check(ctx, who, a.rotation, d->append.head_size, d->rotary, d->places, cos, sin, positions, d->epsilon, d->interleaved));
  const int64_t strides[6] = {d->q_sb, d->q_sh, d->q_st, d->y_sb, d->y_sh, d->y_st};
  CACHE_TRY(cache_check_strides(ctx, who, strides, 6));
  WDC_REQUIRE(ctx, d->heads >= 0 && d->heads <= 65535 && !q == !q_out && (q || d->heads == 0 || !slots), "%s: bad queries", who);
  WDC_REQUIRE(ctx, cache_aligned(q, 16) && cache_aligned(q_out, 16) && cache_aligned(q_weight, 16) && cache_aligned(k_weight, 16),
              "%s: buffers are not aligned", who);
  // (other heads are still to be read when the first are written)
  const wdc_cache_append_desc& n = d->append;
  const auto rows = [&](const float* at, int64_t heads, int64_t sb, int64_t st, int64_t sh) {
    return HeadRows{at, {n.batch, n.tokens, heads}, {sb, st, sh}, n.head_size};
  };
  const HeadRows from = rows(q, d->heads, d->q_sb, d->q_st, d->q_sh), to = rows(q_out, d->heads, d->y_sb, d->y_st, d->y_sh);
  WDC_REQUIRE(ctx, (from.same(to) || !heads_overlap(from, to)) && !heads_overlap(rows(k, n.kv_heads, n.k_sb, n.k_st, n.k_sh), to) &&
              !heads_overlap(rows(v, n.kv_heads, n.v_sb, n.v_st, n.v_sh), to), "%s: q_out overlaps k or v, or q and is not q", who);
  a.q = q; a.y = q_out; a.q_weight = q_weight; a.k_weight = k_weight;
  a.q_sb = d->q_sb; a.q_sh = d->q_sh; a.q_st = d->q_st;
  a.y_sb = d->y_sb; a.y_sh = d->y_sh; a.y_st = d->y_st;
  a.heads = q ? (int)d->heads : 0;
  return slots ? append_launch(ctx, &d->append, a, slots) : WDC_OK;
}

extern "C" int wdc_cache_copy_pages(wdc_context* ctx, const wdc_cache_pages_desc* d, void* codes, float* scales, int64_t n,
                                    const int32_t* from, const int32_t* to) {
  if (!ctx) return wdc_fail(ctx, WDC_ERR_INVALID, "wdc_cache_copy_pages: null context");
  WDC_NO_TAPE(ctx);   // (which pages are copied is the host's decision of the moment)
  wdc_note_write(ctx, codes);
  wdc_note_write(ctx, scales);
  WDC_REQUIRE(ctx, d && n >= 0, "wdc_cache_copy_pages: bad argument");
  CACHE_TRY(cache_check_pool(ctx, "wdc_cache_copy_pages", d->pages, d->kv_heads, d->page_tokens, d->head_size));
  WDC_REQUIRE(ctx, d->layers > 0 && d->layers < (1ll << 20), "wdc_cache_copy_pages: bad pool");
  if (n == 0) return WDC_OK;
  WDC_REQUIRE(ctx, codes && scales && from && to, "wdc_cache_copy_pages: null argument");
  WDC_REQUIRE(ctx, cache_aligned(codes, 16) && cache_aligned(scales, 4), "wdc_cache_copy_pages: buffers are not aligned");
  WDC_REQUIRE(ctx, n <= d->pages, "wdc_cache_copy_pages: more copies than pages");
  try {
    std::vector<int32_t> written(to, to + n);
    std::sort(written.begin(), written.end());
    WDC_REQUIRE(ctx, written.front() >= 0 && written.back() < d->pages, "wdc_cache_copy_pages: a page outside 0 .. %lld",
                (long long)d->pages - 1);
    WDC_REQUIRE(ctx, std::adjacent_find(written.begin(), written.end()) == written.end(),
                "wdc_cache_copy_pages: a page is written twice");
    for (int64_t i = 0; i < n; i++) {
      WDC_REQUIRE(ctx, from[i] >= 0 && from[i] < d->pages, "wdc_cache_copy_pages: page %d of 0 .. %lld", from[i],
                  (long long)d->pages - 1);
      WDC_REQUIRE(ctx, !std::binary_search(written.begin(), written.end(), from[i]),
                  "wdc_cache_copy_pages: page %d is read and written", from[i]);
    }
  } catch (const std::bad_alloc&) {
    return wdc_fail(ctx, WDC_ERR_OOM, "wdc_cache_copy_pages: no host memory");
  }
  CopyArgs a;
  a.codes = (uint4*)codes;
  a.scales = scales;
  a.page_units = 2 * d->kv_heads * d->page_tokens * d->head_size / 16;
  a.layer_units = a.page_units * d->pages;
  a.page_scales = (int)(2 * d->kv_heads);
  a.layer_scales = d->pages * a.page_scales;
  a.pieces = (int)ceil_div64(a.page_units, COPY_PIECE);
  WDC_REQUIRE(ctx, d->layers * (n < COPY_PAIRS ? n : COPY_PAIRS) * a.pieces < (1ll << 31),
              "wdc_cache_copy_pages: copies exceed the grid");
  DeviceGuard g(ctx->device);
  for (int64_t i = 0; i < n; i += COPY_PAIRS) {
    a.n = (int)(n - i < COPY_PAIRS ? n - i : COPY_PAIRS);
    for (int j = 0; j < a.n; j++) {
      a.from[j] = from[i + j];
      a.to[j] = to[i + j];
    }
    const int64_t ctas = d->layers * a.n * a.pieces;
    wdc_launch_pdl(ctx, cache_copy_kernel, dim3((unsigned)ctas), dim3(COPY_THREADS), 0, a);
    CACHE_TRY(wdc_check_launch(ctx, "cache_copy_kernel"));
  }
  return WDC_OK;
}
