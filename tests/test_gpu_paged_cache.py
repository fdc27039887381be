"""The paged 8-bit cache on the GPU: appending, attention, copies of pages, against the definitions in 64 bits (and, for what is
rounded to 8 bits, in the 32-bit steps that the definition names).

Tolerance of the attention, from the formula: a score is a sum of head_size products of float32 numbers with whole numbers, so
it is off by at most 2^-21 of the sum of their magnitudes (rounding of the queries to 22 bits, of the products' sum and of
the scale); a weight's relative error is twice that of its score and its sum's together, and the weighted sum adds a few roundings of its
own: |error| <= max |v| * 2^-21 * (8 + 2 * max sum |q k| * scale).
"""
from ctypes import byref, c_void_p

import numpy as np
import pytest

from webdnn_b200.backend import CPUTensor
from webdnn_b200.lib import CacheAppendDesc, CacheAttentionDesc, CachePagesDesc, CudaBackendError
from webdnn_b200.paged_cache import PagedCache

pytestmark = pytest.mark.gpu
f32 = np.float32


def dev(ctx, a):
    return ctx.move_tensor(CPUTensor.from_array(np.ascontiguousarray(a)))


def pool_codes(cache):
    return cache.codes.get_data().view(np.int8).reshape(cache.layers, cache.pages, 2, cache.kv_heads, cache.page_tokens,
                                                        cache.head_size)


def pool_scales(cache):
    return cache.scales.get_data().reshape(cache.layers, cache.pages, 2, cache.kv_heads)


def set_pool(cache, codes, scales):
    cache.codes.set_data(np.ascontiguousarray(codes).view(np.int32))
    cache.scales.set_data(scales)


def random_pool(rng, cache):
    shape = (cache.layers, cache.pages, 2, cache.kv_heads, cache.page_tokens, cache.head_size)
    codes = rng.integers(-127, 128, shape).astype(np.int8)
    scales = (np.exp(rng.standard_normal(shape[:4]) * 0.5) / 60).astype(f32)
    set_pool(cache, codes, scales)
    return codes, scales


def reference_append(codes, scales, k, v, table, lengths, counts, size):
    """One layer's codes [pages, 2, heads, size, c] and scales [pages, 2, heads], in place.  k, v [batch, tokens, heads, c]."""
    for b, (length, count) in enumerate(zip(lengths, counts)):
        start = length - count
        for i in range(start // size, -(-length // size)) if count else ():
            page, lo, hi = table[b][i], max(start, i * size), min(length, (i + 1) * size)
            old = lo - i * size
            for side, x in enumerate((k, v)):
                new = x[b, lo - start:hi - start].transpose(1, 0, 2)              # [heads, n, c]
                fresh = (np.abs(new).max((1, 2)) / f32(127)).astype(f32)
                before = scales[page, side].copy()
                scale = np.maximum(before, fresh) if old else fresh
                by = np.where(scale > 0, scale, f32(1))[:, None, None]
                if old:
                    again = np.rint(codes[page, side, :, :old].astype(f32) * before[:, None, None] / by)
                    codes[page, side, :, :old] = np.where((scale > before)[:, None, None], np.clip(again, -127, 127),
                                                          codes[page, side, :, :old])
                codes[page, side, :, old:old + hi - lo] = np.clip(np.rint(new / by), -127, 127)
                scales[page, side] = scale


def reference_attention(q, codes, scales, table, lengths, counts, size, scale):
    """(y [batch, tokens, heads, c] in 64 bits, tolerance).  q [batch, tokens, heads, c]; codes and scales of one layer."""
    batch, tokens, heads, c = q.shape
    kv_heads = codes.shape[2]
    y, worst, top = np.zeros(q.shape), 0.0, 0.0
    for b, (length, count) in enumerate(zip(lengths, counts)):
        if not count:
            continue
        pages = np.asarray(table[b][:-(-length // size)])
        full = codes[pages].astype(np.float64) * scales[pages].astype(np.float64)[..., None, None]
        k, v = (full[:, i].transpose(1, 0, 2, 3).reshape(kv_heads, -1, c)[:, :length] for i in (0, 1))
        seen = np.tril(np.ones((count, length), bool), length - count)
        for h in range(heads):
            g = h // (heads // kv_heads)
            qh = q[b, :count, h].astype(np.float64)
            s = np.where(seen, qh @ k[g].T * scale, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            y[b, :count, h] = p @ v[g] / p.sum(1, keepdims=True)
            worst = max(worst, (np.abs(qh) @ np.abs(k[g]).T * abs(scale)).max())
            top = max(top, np.abs(v[g]).max())
    return y, top * 2.0 ** -21 * (8 + 2 * worst)


def tables(rng, cache, lengths, spare=2):
    need = [-(-n // cache.page_tokens) for n in lengths]
    assert sum(need) <= cache.pages
    order = rng.permutation(cache.pages)
    table = np.full((len(lengths), max(need) + spare), -1, np.int32)
    at = 0
    for row, n in zip(table, need):
        row[:n] = order[at:at + n]
        at += n
    return table


def run_append(ctx, cache, k, v, table, lengths, counts, layer=0):
    b, t = k.shape[:2]
    ts = [dev(ctx, a) for a in (k.reshape(b, t, -1), v.reshape(b, t, -1), np.asarray(table, np.int32),
                                np.asarray(lengths, np.int32))]
    n = dev(ctx, np.asarray(counts, np.int32)) if counts is not None else None
    cache.append(layer, *ts, n)
    for x in ts + ([n] if n else []):
        x.dispose()


def run_attention(ctx, cache, q, table, lengths, counts, layer=0, scale=None):
    b, t = q.shape[:2]
    ts = [dev(ctx, a) for a in (q.reshape(b, t, -1), np.asarray(table, np.int32), np.asarray(lengths, np.int32))]
    n = dev(ctx, np.asarray(counts, np.int32)) if counts is not None else None
    y = cache.attention(layer, *ts, n, scale=scale)
    got = y.get_data().reshape(q.shape)
    ctx.sync()
    for x in ts + [y] + ([n] if n else []):
        x.dispose()
    return got


# -------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("size,c,heads,lengths,counts", [
    (16, 32, 1, [1], [1]), (16, 64, 3, [17, 1, 16, 40], [1, 1, 1, 1]), (32, 128, 2, [33, 64, 100], [33, 31, 1]),
    (64, 64, 5, [200, 65, 3, 129], [200, 1, 0, 66]), (128, 128, 2, [300, 128, 129], [173, 128, 2]),
    (16, 128, 1, [50] * 9, [3] * 9), (64, 32, 2, [64, 63], [1, 63])])
def test_append(cuda_context, size, c, heads, lengths, counts):
    rng = np.random.default_rng(size + c + heads)
    cache = PagedCache(cuda_context, 2, sum(-(-n // size) for n in lengths) + 3, heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    shape = (len(lengths), max(counts), heads, c)
    k, v = (rng.standard_normal(shape).astype(f32) * 2 for _ in range(2))
    run_append(cuda_context, cache, k, v, table, lengths, counts, layer=1)
    reference_append(codes[1], scales[1], k, v, table, lengths, counts, size)
    assert np.array_equal(pool_scales(cache), scales)
    assert np.array_equal(pool_codes(cache), codes)
    run_append(cuda_context, cache, k, v, table, lengths, counts, layer=1)      # the same again changes nothing
    assert np.array_equal(pool_codes(cache), codes) and np.array_equal(pool_scales(cache), scales)
    cache.dispose()


@pytest.mark.parametrize("size,c,heads,lengths,counts", [
    (64, 128, 3, [130, 64, 190], [130, 1, 77]), (128, 64, 2, [128, 300], [127, 129]), (128, 32, 2, [255, 40, 129], [35, 40, 33])])
def test_append_with_many_numbers_a_thread(cuda_context, size, c, heads, lengths, counts):
    test_append(cuda_context, size, c, heads, lengths, counts)


def test_append_token_by_token_keeps_the_scale_growing(cuda_context):
    """A page filled one token at a time, each larger than those before it: every step rounds the older codes again."""
    rng = np.random.default_rng(3)
    cache = PagedCache(cuda_context, 1, 4, 2, 64, 16)
    codes, scales = random_pool(rng, cache)
    table = [[2, 0, -1]]
    for n in range(1, 25):
        k, v = (rng.standard_normal((1, 1, 2, 64)).astype(f32) * 1.3 ** n for _ in range(2))
        run_append(cuda_context, cache, k, v, table, [n], None)
        reference_append(codes[0], scales[0], k, v, table, [n], [1], 16)
        assert np.array_equal(pool_codes(cache), codes) and np.array_equal(pool_scales(cache), scales)
    cache.dispose()


def test_append_of_zeros_and_of_tiny_numbers(cuda_context):
    cache = PagedCache(cuda_context, 1, 3, 1, 32, 16)
    rng = np.random.default_rng(4)
    codes, scales = random_pool(rng, cache)
    k = np.zeros((3, 2, 1, 32), f32)
    v = np.zeros_like(k)
    v[1] = 1e-42                          # a scale that is itself below the normal range
    v[2, 1] = 5e-36
    table, lengths = [[0], [1], [2]], [2, 2, 2]
    run_append(cuda_context, cache, k, v, table, lengths, None)
    reference_append(codes[0], scales[0], k, v, table, lengths, [2] * 3, 16)
    assert np.array_equal(pool_codes(cache), codes) and np.array_equal(pool_scales(cache), scales)
    cache.dispose()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_number_that_is_not_finite_makes_its_page_and_head_nan(cuda_context, bad):
    rng = np.random.default_rng(5)
    cache = PagedCache(cuda_context, 1, 3, 2, 32, 16)
    set_pool(cache, np.zeros((1, 3, 2, 2, 16, 32), np.int8), np.zeros((1, 3, 2, 2), f32))
    k, v = (rng.standard_normal((1, 20, 2, 32)).astype(f32) for _ in range(2))
    v[0, 3, 1, 7] = bad
    table = [[1, 2]]
    run_append(cuda_context, cache, k, v, table, [20], None)
    scales = pool_scales(cache)[0]
    assert not np.isfinite(scales[1, 1, 1]) and np.isfinite(np.delete(scales.reshape(-1), 1 * 4 + 3)).all()
    q = rng.standard_normal((1, 20, 2, 32)).astype(f32)
    y = run_attention(cuda_context, cache, q, table, [20], None)
    assert np.isnan(y[0, :, 1]).all() and np.isfinite(y[0, :, 0]).all()
    k, v = (rng.standard_normal((1, 1, 2, 32)).astype(f32) for _ in range(2))     # a page's first token ends it
    run_append(cuda_context, cache, k, v, table, [1], None)
    assert np.isfinite(run_attention(cuda_context, cache, q[:, :1], table, [1], None)).all()
    cache.dispose()


def test_operands_may_be_columns_of_wider_tensors(cuda_context):
    """Queries, keys and values side by side in one tensor, as a merged projection leaves them."""
    rng = np.random.default_rng(6)
    b, t, heads, kv, c = 2, 5, 4, 2, 32
    cache = PagedCache(cuda_context, 1, 8, kv, c, 16)
    codes, scales = random_pool(rng, cache)
    qkv = rng.standard_normal((b, t, (heads + 2 * kv) * c + 8)).astype(f32)
    q, k, v = qkv[..., :heads * c], qkv[..., heads * c + 4:(heads + kv) * c + 4], qkv[..., (heads + kv) * c + 4:-4]
    lengths, counts = [21, 4], [5, 4]
    table = tables(rng, cache, lengths)
    ts = [dev(cuda_context, a) for a in (qkv, table, np.array(lengths, np.int32), np.array(counts, np.int32))]
    cache.append(0, ts[0], ts[0], *ts[1:], k_column=heads * c + 4, v_column=(heads + kv) * c + 4)
    y = cache.attention(0, *ts, heads=heads).get_data().reshape(b, t, heads, c)
    split = lambda x: x.reshape(b, t, -1, c)  # noqa: E731
    reference_append(codes[0], scales[0], split(k), split(v), table, lengths, counts, 16)
    assert np.array_equal(pool_codes(cache), codes)
    want, tol = reference_attention(split(q), codes[0], scales[0], table, lengths, counts, 16, c ** -0.5)
    assert np.abs(y - want).max() <= tol
    cache.dispose()


# ----------------------------------------------------------------------------------------------- attention
ATTENTION = [
    # size, c, heads, kv_heads, lengths, counts
    (16, 32, 1, 1, [1], [1]), (16, 64, 4, 4, [15, 16, 17, 31, 32, 33], [1] * 6), (32, 128, 8, 1, [100, 1, 7], [1, 1, 1]),
    (64, 128, 24, 2, [65, 500], [1, 1]), (128, 64, 6, 2, [1000, 129, 127], [1, 1, 1]), (16, 32, 9, 3, [77, 300], [4, 2]),
    (32, 64, 10, 2, [90, 33, 6, 1], [7, 5, 6, 1]), (64, 128, 4, 4, [130, 64, 63], [130, 64, 3]),
    (16, 128, 3, 1, [260], [250]), (64, 32, 40, 1, [100, 3], [1, 3]), (128, 128, 16, 2, [700, 400], [33, 12]),
    (64, 64, 2, 2, [3000], [1]), (16, 64, 8, 2, [2500, 9], [1, 1]), (32, 128, 4, 2, [333, 222, 111], [200, 222, 64]),
    (64, 128, 8, 8, [5000], [2]), (32, 32, 12, 4, [640, 64], [64, 64]),
]


@pytest.mark.parametrize("size,c,heads,kv_heads,lengths,counts", ATTENTION)
def test_attention(cuda_context, size, c, heads, kv_heads, lengths, counts):
    rng = np.random.default_rng(size + c + heads + len(lengths))
    cache = PagedCache(cuda_context, 1, sum(-(-n // size) for n in lengths) + 1, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    q = rng.standard_normal((len(lengths), max(counts), heads, c)).astype(f32)
    got = run_attention(cuda_context, cache, q, table, lengths, counts)
    want, tol = reference_attention(q, codes[0], scales[0], table, lengths, counts, size, c ** -0.5)
    assert np.abs(got - want).max() <= tol
    for b, n in enumerate(counts):
        assert not got[b, n:].any()                   # padding
    cache.dispose()


PROMPTS = [
    # enough rows of new tokens for the tensor-core kernel: 37 tiles of 128 rows
    (64, 128, 16, 8, [300, 500], [290, 300]), (16, 64, 8, 8, [200, 150, 131], [200, 100, 131]),
    (128, 128, 12, 4, [900], [700]), (32, 64, 30, 10, [150, 151], [90, 33]), (16, 128, 10, 10, [64, 65, 300, 63], [64, 1, 129, 63]),
    (64, 64, 64, 2, [80, 1000], [80, 77]), (32, 128, 5, 5, [1000, 999], [513, 512]), (64, 128, 20, 20, [2000, 70], [100, 70]),
]


@pytest.mark.parametrize("size,c,heads,kv_heads,lengths,counts", PROMPTS)
def test_attention_of_prompts(cuda_context, size, c, heads, kv_heads, lengths, counts):
    rng = np.random.default_rng(size + c + heads + len(lengths))
    ctx = cuda_context
    cache = PagedCache(ctx, 1, sum(-(-n // size) for n in lengths) + 1, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    q = rng.standard_normal((len(lengths), max(counts), heads, c)).astype(f32)
    before = ctx.stats()["tensor_core_launches"]
    got = run_attention(ctx, cache, q, table, lengths, counts)
    assert ctx.stats()["tensor_core_launches"] == before + 1
    want, tol = reference_attention(q, codes[0], scales[0], table, lengths, counts, size, c ** -0.5)
    assert np.abs(got - want).max() <= tol
    for b, n in enumerate(counts):
        assert not got[b, n:].any()                   # padding
    cache.dispose()


@pytest.mark.parametrize("batch,c,group", [(50, 64, 2), (8, 128, 7), (5, 64, 12), (70, 64, 1)])
def test_prompts_of_many_uneven_sequences(cuda_context, batch, c, group):
    """More tiles than SMs, of sequences whose order says nothing about their lengths; some are empty, some have nothing new."""
    rng = np.random.default_rng(batch)
    ctx, size, kv_heads = cuda_context, 32, 4
    lengths = [int(n) for n in rng.integers(1, 260, batch)]
    counts = [int(min(n, m)) for n, m in zip(lengths, rng.integers(0, 151, batch))]
    lengths[2] = counts[2] = counts[1] = 0
    lengths[batch - 2], counts[batch - 2] = 1100, 150
    cache = PagedCache(ctx, 1, sum(-(-n // size) for n in lengths) + 1, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    q = rng.standard_normal((batch, 150, group * kv_heads, c)).astype(f32)
    before = ctx.stats()["tensor_core_launches"]
    got = run_attention(ctx, cache, q, table, lengths, counts)
    assert ctx.stats()["tensor_core_launches"] == before + 1
    want, tol = reference_attention(q, codes[0], scales[0], table, lengths, counts, size, c ** -0.5)
    assert np.abs(got - want).max() <= tol
    for b, n in enumerate(counts):
        assert not got[b, n:].any()
    cache.dispose()


def test_prompts_with_sharp_scores_missing_pages_and_scales_that_are_no_numbers(cuda_context):
    rng = np.random.default_rng(20)
    ctx, size, c, heads = cuda_context, 16, 64, 20
    cache = PagedCache(ctx, 1, 41, heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, [300, 320])
    scales[0, table[0, :19], 0] *= np.linspace(0.2, 8, 19, dtype=f32)[:, None]
    scales[0, table[0, 18], 1] = 0
    scales[0, table[1, 12], 1, 3] = np.nan            # tokens 192 .. of the second sequence, one head's values
    scales[0, table[1, 5], 0, 4] = np.inf             # tokens 80 ..: another's keys
    set_pool(cache, codes, scales)
    lengths, counts = [300, 320], [170, 310]
    q = (rng.standard_normal((2, 310, heads, c)) * np.where(np.arange(heads) % 3 == 0, 20, 1)[:, None]).astype(f32)
    got = run_attention(ctx, cache, q, table, lengths, counts, scale=0.3)
    first = np.arange(310) + 10
    assert np.isnan(got[1, first >= 192, 3]).all() and np.isfinite(got[1, first < 192, 3]).all()
    assert np.isnan(got[1, first >= 80, 4]).all() and np.isfinite(got[1, first < 80, 4]).all()
    scales[0, table[1, 12], 1, 3] = scales[0, table[1, 5], 0, 4] = 0
    want, tol = reference_attention(q, codes[0], scales[0], table, lengths, counts, size, float(f32(0.3)))
    fine = np.isfinite(got)
    assert np.abs(got - want)[fine].max() <= tol and fine.mean() > 0.9
    # a page out of range: its tokens are left out
    set_pool(cache, codes, scales)
    holes = table.copy()
    holes[0, 3] = 41
    ts = [dev(ctx, a) for a in (q.reshape(2, 310, -1), holes, np.array(lengths, np.int32), np.array(counts, np.int32))]
    y = cache.attention(0, *ts, scale=0.3)
    with pytest.raises(CudaBackendError, match="out of range"):
        ctx.sync()
    got = y.get_data().reshape(q.shape)
    shorter = table.copy()
    shorter[0, 3:19] = table[0, 4:20]
    k_lengths = [300 - size, 320]
    want0, tol0 = reference_attention(q[:1], codes[0], scales[0], shorter[:1], k_lengths[:1], counts[:1], size, float(f32(0.3)))
    assert np.abs(got[0] - want0[0]).max() <= tol0
    for t in ts + [y]:
        t.dispose()
    cache.dispose()


@pytest.mark.parametrize("tokens", [1, 70])
def test_sharp_and_tiny_scores(cuda_context, tokens):
    """Scores spread over hundreds of units, the largest at the end, and queries of very different magnitudes."""
    rng = np.random.default_rng(8)
    cache = PagedCache(cuda_context, 1, 24, 2, 64, 16)
    codes, scales = random_pool(rng, cache)
    lengths, counts = [300, 71], [tokens, tokens]
    table = tables(rng, cache, lengths)
    scales[0, table[0, :19], 0] *= np.linspace(0.2, 8, 19, dtype=f32)[:, None]
    set_pool(cache, codes, scales)
    q = rng.standard_normal((2, tokens, 4, 64)).astype(f32) * np.array([30, 1, 1e-6, 1e-30], f32)[:, None]
    got = run_attention(cuda_context, cache, q, table, lengths, counts, scale=0.7)
    want, tol = reference_attention(q, codes[0], scales[0], table, lengths, counts, 16, float(f32(0.7)))
    assert np.abs(got - want).max() <= tol
    small, tol = reference_attention(q[:, :, 1:3], codes[0], scales[0], table, lengths, counts, 16, float(f32(0.7)))
    cache.dispose()


@pytest.mark.parametrize("tokens", [2, 130])
@pytest.mark.parametrize("scale", [-0.4, 0.0])
def test_scales_that_are_negative_or_zero(cuda_context, scale, tokens):
    rng = np.random.default_rng(21)
    cache = PagedCache(cuda_context, 1, 30, 20, 64, 32)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, [300, 140])
    q = rng.standard_normal((2, tokens, 20, 64)).astype(f32)
    got = run_attention(cuda_context, cache, q, table, [300, 140], [tokens] * 2, scale=scale)
    want, tol = reference_attention(q, codes[0], scales[0], table, [300, 140], [tokens] * 2, 32, float(f32(scale)))
    assert np.abs(got - want).max() <= tol
    cache.dispose()


def test_value_scales_that_differ_by_orders_of_magnitude(cuda_context):
    """The page with the large scale gets a small weight, so that both matter: errors are relative to what is in the sum."""
    rng = np.random.default_rng(9)
    c, size = 64, 16
    cache = PagedCache(cuda_context, 1, 6, 1, c, size)
    codes, scales = random_pool(rng, cache)
    codes[0, 1, 0] = -codes[0, 0, 0]
    scales[0, :, 1] = np.array([1e-9, 1e9, 1, 1e-20, 0, 1e20], f32)[:, None]
    set_pool(cache, codes, scales)
    q = rng.standard_normal((1, 1, 1, c)).astype(f32)
    for table, length in (([[0, 1]], 32), ([[1, 0]], 32), ([[3, 5, 4]], 48), ([[4]], 16), ([[4, 3]], 20), ([[5, 3, 0]], 48)):
        got = run_attention(cuda_context, cache, q, table, [length], [1])
        want, _ = reference_attention(q, codes[0], scales[0], table, [length], [1], size, c ** -0.5)
        worst = (np.abs(q[0, 0, 0].astype(np.float64)) @ np.abs(codes[0, table[0], 0, 0].reshape(-1, c).T *
                 scales[0, table[0], 0].repeat(size).astype(np.float64))).max() * c ** -0.5
        # the sum of weight * |v| is what the roundings are relative to
        pages = np.asarray(table[0])
        k = (codes[0, pages, 0, 0] * scales[0, pages, 0].astype(np.float64)[..., None]).reshape(-1, c)[:length]
        v = np.abs(codes[0, pages, 1, 0] * scales[0, pages, 1].astype(np.float64)[..., None]).reshape(-1, c)[:length]
        s = k @ q[0, 0, 0].astype(np.float64) * c ** -0.5
        p = np.exp(s - s.max())
        # each weight is split into 22 bits below the largest term
        bound = 2.0 ** -21 * (8 + 2 * worst) * ((p[:, None] * v).sum(0) + length * (p * v.max(1)).max()) / p.sum()
        assert (np.abs(got[0, 0, 0] - want[0, 0, 0]) <= bound).all(), (table, np.abs(got - want).max())
    cache.dispose()


def test_empty_sequences_and_what_is_out_of_range(cuda_context):
    """An empty sequence gives zeros; numbers out of range leave their part out and are reported once."""
    rng = np.random.default_rng(10)
    ctx, size, c = cuda_context, 16, 32
    cache = PagedCache(ctx, 1, 8, 1, c, size)
    codes, scales = random_pool(rng, cache)
    table = np.array([[0, 1, -1], [2, 3, 4], [5, 6, 7], [1, 2, 3], [-1, 99, 5], [6, 8, 7]], np.int32)
    q = rng.standard_normal((6, 2, 2, c)).astype(f32)
    lengths, counts = [0, 49, 5, -1, 40, 40], [0, 1, 6, 1, 2, 3]
    y = ctx.empty_tensor([6, 2, 2 * c])
    ts = [dev(ctx, a) for a in (q.reshape(6, 2, -1), table, np.array(lengths, np.int32), np.array(counts, np.int32))]
    cache.attention(0, *ts, out=y)
    with pytest.raises(CudaBackendError, match="out of range") as e:
        ctx.sync()
    assert e.value.status == 1
    ctx.sync()                                        # once
    got = y.get_data().reshape(q.shape)
    assert not got[[0, 1, 2, 3, 5]].any()             # empty, too long, count above length, negative, count above the call's
    only = codes[:, [5]], scales[:, [5]]              # of the fifth, only the third page is there
    k = only[0][0, 0, 0, 0].astype(np.float64) * only[1][0, 0, 0, 0]
    v = only[0][0, 0, 1, 0].astype(np.float64) * only[1][0, 0, 1, 0]
    for i, last in enumerate((38, 39)):
        for h in range(2):
            s = k[:last - 32 + 1] @ q[4, i, h].astype(np.float64) * c ** -0.5
            p = np.exp(s - s.max())
            np.testing.assert_allclose(got[4, i, h], p @ v[:last - 32 + 1] / p.sum(), atol=1e-5 * np.abs(v).max())
    kv = [dev(ctx, rng.standard_normal((6, 2, c)).astype(f32)) for _ in range(2)]
    before = pool_codes(cache).copy()
    lengths[4] = 20
    bad = dev(ctx, np.array(lengths, np.int32))
    cache.append(0, *kv, ts[1], bad, ts[3])
    with pytest.raises(CudaBackendError, match="out of range"):
        ctx.sync()
    assert np.array_equal(pool_codes(cache), before) and np.array_equal(pool_scales(cache), scales)
    for t in ts + kv + [bad, y]:
        t.dispose()
    cache.dispose()


def test_no_tokens_and_no_sequences(cuda_context):
    cache = PagedCache(cuda_context, 1, 2, 1, 32, 16)
    for b, t in ((0, 1), (1, 0)):
        ts = [dev(cuda_context, np.zeros((b, t, 32), f32)), dev(cuda_context, np.zeros((b, 1), np.int32)),
              dev(cuda_context, np.zeros(b, np.int32))]
        cache.append(0, ts[0], ts[0], *ts[1:])
        assert cache.attention(0, *ts).dims == [b, t, 32]
    cuda_context.sync()
    cache.dispose()


def test_results_do_not_depend_on_the_run(cuda_context):
    rng = np.random.default_rng(11)
    cache = PagedCache(cuda_context, 1, 200, 4, 128, 32)
    random_pool(rng, cache)
    lengths = [3000, 1, 800, 77]
    table = tables(rng, cache, lengths)
    q = rng.standard_normal((4, 1, 16, 128)).astype(f32)
    first = run_attention(cuda_context, cache, q, table, lengths, None)
    for _ in range(5):
        assert np.array_equal(run_attention(cuda_context, cache, q, table, lengths, None), first)
    # nor on what stands beside a sequence in the batch or how wide the table is
    for b in (0, 2):
        alone = run_attention(cuda_context, cache, q[b:b + 1], table[b:b + 1, :-(-lengths[b] // 32)], lengths[b:b + 1], None)
        want = first[b]
        assert np.abs(alone[0] - want).max() <= 1e-5 * np.abs(want).max()
    cache.dispose()


def test_an_offset_beyond_31_bits(cuda_context):
    """Pages behind the first 2 GB of a pool."""
    rng = np.random.default_rng(12)
    ctx, size, c, heads = cuda_context, 128, 128, 16
    page = 2 * heads * size * c
    cache = PagedCache(ctx, 1, (5 << 30) // page, heads, c, size)
    n = cache.pages
    assert n * page > 1 << 32
    table, lengths = [[n - 1, n // 2 + 3]], [150]
    k, v = (rng.standard_normal((1, 150, heads, c)).astype(f32) for _ in range(2))
    run_append(ctx, cache, k, v, table, lengths, None)
    codes, scales = np.zeros((2, 2, heads, size, c), np.int8), np.zeros((2, 2, heads), f32)
    reference_append(codes, scales, k, v, [[0, 1]], lengths, [150], size)
    q = rng.standard_normal((1, 1, heads, c)).astype(f32)
    want, tol = reference_attention(q, codes, scales, [[0, 1]], lengths, [1], size, c ** -0.5)
    assert np.abs(run_attention(ctx, cache, q, table, lengths, [1]) - want).max() <= tol
    cache.copy_pages([n - 1, n // 2 + 3], [1, n - 2])
    got = run_attention(ctx, cache, q, [[1, n - 2]], lengths, [1])
    assert np.abs(got - want).max() <= tol
    cache.dispose()


# ----------------------------------------------------------------------------------------------- copies, bookkeeping
@pytest.mark.parametrize("layers,size,c,heads,n", [(1, 16, 32, 1, 1), (3, 32, 64, 5, 7), (2, 16, 32, 3, 600), (5, 128, 128, 8, 2)])
def test_copies_of_pages(cuda_context, layers, size, c, heads, n):
    rng = np.random.default_rng(n)
    cache = PagedCache(cuda_context, layers, 2 * n + 5, heads, c, size)
    codes, scales = random_pool(rng, cache)
    order = rng.permutation(cache.pages)
    sources, targets = order[:n], order[n:2 * n]
    sources[n // 2] = sources[0]                     # one page may go to several
    cache.copy_pages(sources, targets)
    codes[:, targets], scales[:, targets] = codes[:, sources], scales[:, sources]
    assert np.array_equal(pool_codes(cache), codes) and np.array_equal(pool_scales(cache), scales)
    cache.copy_pages([], [])
    cache.dispose()


def test_fork_release_and_compaction_keep_every_sequence(cuda_context):
    """Sequences that grow, fork, end and move give what each would give in a cache of its own."""
    rng = np.random.default_rng(13)
    ctx, heads, c = cuda_context, 2, 32
    cache = PagedCache(ctx, 1, 60, heads, c, 16)
    texts = {}

    def grow(which):
        cache.extend({s: n for s, n in which.items()})
        width = max(which.values())
        k, v = (rng.standard_normal((len(which), width, heads, c)).astype(f32) for _ in range(2))
        table, lengths, counts = (t.numpy() for t in cache.batch(list(which), list(which.values())))
        run_append(ctx, cache, k, v, table, lengths, counts)
        for i, (s, n) in enumerate(which.items()):
            texts[s] = texts.get(s, []) + [(k[i:i + 1, :n], v[i:i + 1, :n])]

    def check():
        for s, parts in texts.items():
            own_codes, own_scales = np.zeros((9, 2, heads, 16, c), np.int8), np.zeros((9, 2, heads), f32)
            length = 0
            for k, v in parts:
                length += k.shape[1]
                reference_append(own_codes, own_scales, k, v, [range(9)], [length], [k.shape[1]], 16)
            pages = cache.sequence_pages(s)
            assert cache.length(s) == length and len(pages) == -(-length // 16)
            got_codes, got_scales = pool_codes(cache)[0][pages], pool_scales(cache)[0][pages]
            assert np.array_equal(got_scales, own_scales[:len(pages)])
            for t in range(length):
                assert np.array_equal(got_codes[t // 16, :, :, t % 16], own_codes[t // 16, :, :, t % 16])

    a, b = cache.add_sequence(), cache.add_sequence()
    grow({a: 37, b: 16})
    f = [cache.fork(a) for _ in range(3)] + [cache.fork(b)]
    for s in f:
        texts[s] = list(texts[b if s == f[3] else a])
    grow({f[0]: 1, a: 2, f[3]: 5})
    check()
    grow({f[1]: 20, b: 1, f[2]: 1, f[0]: 30})
    check()
    for s in (a, f[1]):
        cache.release(s)
        del texts[s]
    used = cache.used_pages
    assert cache.compact() > 0
    assert max(max(cache.sequence_pages(s)) for s in texts) == used - 1 and cache.used_pages == used
    check()
    cache.truncate(f[0], 48)
    texts[f[0]] = None
    del texts[f[0]]
    grow({f[2]: 3, b: 40})
    check()
    cache.dispose()


# ----------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_library(cuda_context):
    ctx = cuda_context
    cache = PagedCache(ctx, 1, 4, 2, 32, 16)
    x, i = ctx.empty_tensor([1024]), ctx.empty_tensor([64], "int32")
    ctx._call("wdc_fill_u32", c_void_p(i.ptr), 0, 64)
    at = lambda t, off=0: c_void_p(t.ptr + off)  # noqa: E731
    good_append = dict(pages=4, kv_heads=2, page_tokens=16, head_size=32, batch=1, tokens=1, table_pages=1, k_sb=64, k_sh=32,
                       k_st=64, v_sb=64, v_sh=32, v_st=64)
    good_att = dict(pages=4, kv_heads=2, page_tokens=16, head_size=32, batch=1, tokens=1, table_pages=1, heads=4, q_sb=128,
                    q_sh=32, q_st=128, y_sb=128, y_sh=32, y_st=128, scale=1.0)
    good_pages = dict(layers=1, pages=4, kv_heads=2, page_tokens=16, head_size=32)
    pool = [at(cache.codes), at(cache.scales)]

    def append(off=0, skip=None, **change):
        ptrs = [at(x, off), at(x), *pool, at(i), at(i), None]
        if skip is not None:
            ptrs[skip] = None
        ctx._call("wdc_cache_append", byref(CacheAppendDesc(**{**good_append, **change})), *ptrs)

    def attention(off=0, skip=None, **change):
        ptrs = [at(x, off), *pool, at(i), at(i), None, at(x)]
        if skip is not None:
            ptrs[skip] = None
        ctx._call("wdc_cache_attention", byref(CacheAttentionDesc(**{**good_att, **change})), *ptrs)

    def copy(frm, to, **change):
        a, b = (np.array(v, np.int32) for v in (frm, to))
        ctx._call("wdc_cache_copy_pages", byref(CachePagesDesc(**{**good_pages, **change})), *pool, len(frm),
                  a.ctypes.data_as(c_void_p), b.ctypes.data_as(c_void_p))

    def refused(status, f, *args, **kw):
        with pytest.raises(CudaBackendError) as e:
            f(*args, **kw)
        assert e.value.status == status, e.value

    for f in (append, attention):
        for change in (dict(page_tokens=24), dict(head_size=48), dict(head_size=256), dict(page_tokens=0)):
            refused(4, f, **change)
        for change in (dict(pages=0), dict(kv_heads=0), dict(batch=-1), dict(tokens=-1), dict(table_pages=-1),
                       dict(pages=1 << 31), dict(table_pages=1 << 40), dict(off=4)):
            refused(1, f, **change)
        for skip in range(5):
            refused(1, f, skip=skip)
    refused(1, append, k_st=6)
    refused(1, append, v_sh=-4)
    refused(1, attention, heads=3)
    refused(1, attention, heads=0)
    refused(1, attention, y_st=2)
    refused(1, attention, skip=6)
    refused(1, copy, [0], [4])
    refused(1, copy, [-1], [1])
    refused(1, copy, [0, 1], [2, 2])
    refused(1, copy, [0, 1], [1, 2])
    refused(1, copy, [3], [3])
    refused(1, copy, [0], [1], layers=0)
    refused(4, copy, [0], [1], head_size=40)
    with pytest.raises(CudaBackendError):
        ctx._call("wdc_cache_append", None, *[None] * 7)
    ctx.sync()
    for t in (x, i):
        t.dispose()
    cache.dispose()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("size,c", [(16, 32), (64, 64), (32, 128)])
def test_a_key_that_is_not_finite_makes_every_row_that_sees_its_page_nan(cuda_context, size, c, bad):
    rng = np.random.default_rng(c)
    heads, length = 8, 3 * size
    cache = PagedCache(cuda_context, 1, 4, 2, c, size)
    set_pool(cache, np.zeros(pool_codes(cache).shape, np.int8), np.zeros((1, 4, 2, 2), f32))
    k, v = (rng.standard_normal((1, length, 2, c)).astype(f32) for _ in range(2))
    k[0, size + 3, 1, 7] = bad
    table = [[2, 0, 3]]
    run_append(cuda_context, cache, k, v, table, [length], None)
    q = rng.standard_normal((1, length, heads, c)).astype(f32)
    y = run_attention(cuda_context, cache, q, table, [length], None)
    assert np.isfinite(y[0, :, :4]).all() and np.isfinite(y[0, :size]).all()
    assert np.isnan(y[0, size:, 4:]).all()
    cache.dispose()


@pytest.mark.parametrize("tokens", [5, 150])
def test_key_scales_that_are_no_numbers(cuda_context, tokens):
    """Whatever the codes beside such a scale are, and however few of them a row sees."""
    rng = np.random.default_rng(23)
    size, c, heads = 64, 64, 20
    cache = PagedCache(cuda_context, 1, 4, heads, c, size)
    codes, scales = random_pool(rng, cache)
    scales[0, 1, 0, ::2] = np.inf
    scales[0, 2, 0, 1::4] = np.nan
    set_pool(cache, codes, scales)
    table, lengths = [[1, 0, 0], [2, 3, 3]], [tokens, tokens]
    q = rng.standard_normal((2, tokens, heads, c)).astype(f32)
    before = cuda_context.stats()["tensor_core_launches"]
    y = run_attention(cuda_context, cache, q, table, lengths, None)
    assert cuda_context.stats()["tensor_core_launches"] == before + (tokens == 150)
    nan = np.zeros((2, heads), bool)
    nan[0, ::2] = nan[1, 1::4] = True
    assert (np.isnan(y) == nan[:, None, :, None]).all()
    cache.dispose()


@pytest.mark.parametrize("mean", [0.0, 5.0])
@pytest.mark.parametrize("size,c,heads,kv_heads,tokens", [(16, 32, 6, 2, 1), (32, 64, 4, 4, 3), (64, 128, 16, 2, 1), (16, 128, 24, 3, 2),
                                                          (32, 128, 48, 8, 70)])
def test_small_codes_and_queries_of_one_sign(cuda_context, size, c, heads, kv_heads, tokens, mean):
    """One key channel that is far larger than the others sets a page's scale, so that the codes of all others are small; and queries
    whose channels do not cancel: a score's error is relative to sum |q k|, which is then far below 127 times the sum of the queries."""
    rng = np.random.default_rng(size + c + heads)
    lengths = [max(tokens, n) for n in (2, 3, 33, 5, 90, 2, 4)]
    counts = [tokens] * len(lengths)
    cache = PagedCache(cuda_context, 1, sum(-(-n // size) for n in lengths), kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    codes[:, :, 0] = np.rint(rng.standard_normal(codes[:, :, 0].shape) * 3)
    codes[:, :, 0, :, size - 1, 9] = 127
    scales[:, :, 0] = 0.1
    set_pool(cache, codes, scales)
    table = tables(rng, cache, lengths)
    q = (rng.standard_normal((len(lengths), tokens, heads, c)) + mean).astype(f32)
    got = run_attention(cuda_context, cache, q, table, lengths, counts)
    for b, n in enumerate(lengths):                  # each with the tolerance of its own scores
        for h in range(heads):
            of = slice(h * kv_heads // heads, h * kv_heads // heads + 1)
            want, tol = reference_attention(q[b:b + 1, :, h:h + 1], codes[0][:, :, of], scales[0][:, :, of], table[b:b + 1], [n], [tokens],
                                            size, c ** -0.5)
            assert np.abs(got[b:b + 1, :, h:h + 1] - want).max() <= tol
    cache.dispose()


@pytest.mark.parametrize("tokens", [1, 70])
def test_sharp_and_tiny_scores_head_by_head(cuda_context, tokens):
    """Queries of very different magnitudes beside one another, each head within the tolerance of its own scores."""
    rng = np.random.default_rng(8)
    magnitudes = np.array([30, 1, 1e-6, 1e-30, 1e-37], f32)
    cache = PagedCache(cuda_context, 1, 24, 10, 64, 16)
    codes, scales = random_pool(rng, cache)
    lengths, counts = [300, 71], [tokens, tokens]
    table = tables(rng, cache, lengths)
    scales[0, table[0, :19], 0] *= np.linspace(0.2, 8, 19, dtype=f32)[:, None]
    set_pool(cache, codes, scales)
    q = rng.standard_normal((2, tokens, 20, 64)).astype(f32) * np.repeat(magnitudes, 4)[:, None]
    got = run_attention(cuda_context, cache, q, table, lengths, counts, scale=0.7)
    for h in range(20):
        of = slice(h // 2, h // 2 + 1)
        want, tol = reference_attention(q[:, :, h:h + 1], codes[0][:, :, of], scales[0][:, :, of], table, lengths, counts, 16, float(f32(0.7)))
        assert np.abs(got[:, :, h:h + 1] - want).max() <= tol
    cache.dispose()


def short_sequences_of_a_wide_table(ctx, batch, c, heads, kv_heads, size, tokens, wide, lengths, counts, seed):
    """Compares them with the reference; numbers of the sequences in `counts` that do not fit the call give rows of zeros."""
    rng = np.random.default_rng(seed)
    fits = [0 <= n <= m and n <= tokens and m <= wide * size for n, m in zip(counts, lengths)]
    held = [m if f else 0 for m, f in zip(lengths, fits)]
    cache = PagedCache(ctx, 1, sum(-(-m // size) for m in held) + 1, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, held)
    table = np.concatenate([table, np.full((batch, wide - table.shape[1]), -1, np.int32)], 1)
    q = rng.standard_normal((batch, tokens, heads, c)).astype(f32)
    ts = [dev(ctx, a) for a in (q.reshape(batch, tokens, -1), table, np.array(lengths, np.int32), np.array(counts, np.int32))]
    y = cache.attention(0, *ts)
    if all(fits):
        ctx.sync()
    else:
        with pytest.raises(CudaBackendError, match="out of range"):
            ctx.sync()
    got = y.get_data().reshape(q.shape)
    want, tol = reference_attention(q, codes[0], scales[0], table, held, [n if f else 0 for n, f in zip(counts, fits)], size, c ** -0.5)
    assert np.abs(got - want).max() <= tol
    for b, (n, f) in enumerate(zip(counts, fits)):
        assert not got[b, n if f else 0:].any()
    for t in ts + [y]:
        t.dispose()
    cache.dispose()


# (Such a call's tiles are shared out between three or four CTAs an SM where the table has room for 32 and more of them a CTA.)
@pytest.mark.parametrize("batch,c,heads,kv_heads,size,tokens,wide", [
    (1, 128, 2, 1, 128, 1, 3600), (3, 64, 8, 2, 64, 9, 400), (5, 64, 4, 2, 32, 1, 2000), (20, 32, 6, 2, 16, 3, 1000),
    (37, 128, 8, 4, 64, 2, 100), (200, 128, 4, 4, 128, 1, 40), (512, 64, 1, 1, 64, 1, 24), (511, 32, 4, 1, 32, 2, 40),
    (512, 128, 3, 1, 16, 2, 80), (2, 128, 24, 2, 32, 30, 700)])
def test_tiles_that_are_shared_out(cuda_context, batch, c, heads, kv_heads, size, tokens, wide):
    """Sequences of any length, some empty, some without new tokens."""
    rng = np.random.default_rng(batch + c)
    longest = min(wide * size, 40_000 // batch + 2 * tokens)
    lengths = [int(n) for n in rng.integers(1, longest + 1, batch)]
    counts = [int(rng.integers(0, min(n, tokens) + 1)) for n in lengths]
    lengths[0], counts[0] = longest, tokens
    if batch > 2:
        lengths[1] = counts[1] = counts[2] = 0
    short_sequences_of_a_wide_table(cuda_context, batch, c, heads, kv_heads, size, tokens, wide, lengths, counts, batch)


def test_tiles_that_are_shared_out_beside_numbers_out_of_range(cuda_context):
    lengths = [500, -1, 90, 3000 * 32 + 1, 70, 5, 41, 1000]
    counts = [2, 1, 3, 1, -1, 6, 2, 1]
    short_sequences_of_a_wide_table(cuda_context, 8, 64, 8, 2, 32, 2, 3000, lengths, counts, 1)


@pytest.mark.parametrize("batch,length", [(444, 250), (222, 768), (222, 250), (148, 500), (111, 500), (300, 1), (148, 32)])
def test_units_that_end_where_a_ctas_tiles_end(cuda_context, batch, length):
    """Equal units, of which whole ones, halves, thirds or quarters are a CTA's (or only a beginning, without a tile)."""
    short_sequences_of_a_wide_table(cuda_context, batch, 128, 2, 1, 128, 1, 140, [length] * batch, [1] * batch, batch)


@pytest.mark.parametrize("size,c,heads,kv_heads,tokens", [(16, 64, 8, 2, 1), (64, 128, 4, 4, 2), (32, 32, 9, 3, 12)])
def test_parts_without_a_tile(cuda_context, size, c, heads, kv_heads, tokens):
    """Sequences that are much shorter than the table has room for, cut into equal parts of which most have nothing."""
    lengths, counts = [1, 90, 0, 40, 700], [1, min(tokens, 9), 0, tokens, tokens]
    short_sequences_of_a_wide_table(cuda_context, 5, c, heads, kv_heads, size, tokens, 4096 // size, lengths, counts, c)
