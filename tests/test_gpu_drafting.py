"""The operators of a decoder that drafts on the GPU, against their definitions in 64 bits.

Tolerances, from the arithmetic that the operators promise:
* heads: a mean of at most 256 squares, 13 additions one after the other and a product, is (14 + 1) * 2^-24 off, its root half of that;
  rsqrtf 3 * 2^-24, two products with it and the weight 2, a rotation's products and sum 2 more: less than 15 * 2^-24 of |n1| + |n2|,
  which is less than 2^-20 of it;
* rotated keys are computed in 64 bits and rounded once, so codes of rotated keys and kept paths are whole numbers, verdicts are decisions: equal;
* attention of a tree: as that of a text (test_gpu_paged_cache).
"""
from ctypes import byref

import numpy as np
import pytest

from test_gpu_paged_cache import dev, pool_codes, pool_scales, random_pool, reference_append, run_attention, set_pool, tables
from webdnn_b200 import lib
from webdnn_b200.lib import CudaBackendError
from webdnn_b200.paged_cache import PagedCache

pytestmark = pytest.mark.gpu
f32 = np.float32


def tables_of(places, pairs, base=10000.0):
    angle = np.arange(places)[:, None] * base ** (-np.arange(pairs) / max(pairs, 1))
    return np.cos(angle).astype(f32), np.sin(angle).astype(f32)


def rotated(x, weight, cos, sin, epsilon, interleaved):
    """x [..., heads, c]; cos, sin [..., pairs] of the rows; in 64 bits."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(f32(epsilon))) * weight.astype(np.float64)
    y, pairs = x.copy(), cos.shape[-1]
    c, s = cos.astype(np.float64)[..., None, :], sin.astype(np.float64)[..., None, :]
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def assert_heads(got, x, weight, cos, sin, epsilon, interleaved):
    """``got`` is rotated(...), within 2^-20 of the magnitudes that a number is the sum of."""
    want = rotated(x, weight, cos, sin, epsilon, interleaved)
    parts = rotated(np.abs(x), None if weight is None else np.abs(weight), np.abs(cos), -np.abs(sin), epsilon, interleaved)
    other = rotated(np.abs(x), None if weight is None else np.abs(weight), np.abs(cos), np.abs(sin), epsilon, interleaved)
    room = 2.0 ** -20 * np.maximum(np.abs(parts), np.abs(other)) + 2.0 ** -148
    assert (np.abs(got.astype(np.float64) - want) <= room).all()


def dispose(*tensors):
    for t in tensors:
        if t is not None:
            t.dispose()


# -------------------------------------------------------------------------------------------------- heads
@pytest.mark.parametrize("rows,heads,c,pairs,interleaved,norm", [
    (1, 1, 32, 16, False, True), (1, 40, 128, 64, False, True), (7, 3, 64, 32, True, True), (5, 2, 80, 16, False, True),
    (33, 5, 96, 48, True, False), (3, 4, 128, 32, False, False), (2, 3, 256, 128, False, True), (9, 2, 200, 100, True, True),
    (4, 3, 132, 64, False, True), (6, 2, 256, 36, False, True), (11, 3, 8, 4, False, True), (5, 2, 4, 0, False, True),
    (3, 1, 36, 16, False, True), (2000, 7, 64, 32, False, True), (1300, 9, 20, 8, True, True), (900, 5, 144, 72, False, True),
    (4, 2, 64, 0, False, False), (8, 1, 128, 4, False, False), (700, 11, 128, 64, True, True)])
def test_heads(cuda_context, rows, heads, c, pairs, interleaved, norm):
    ctx, rng = cuda_context, np.random.default_rng(rows + heads + c)
    wide, column = heads * c + 12, 8
    x = rng.standard_normal((rows, wide)).astype(f32) * np.exp(rng.standard_normal((rows, 1)) * 3).astype(f32)
    weight = (1 + rng.standard_normal(c) * 0.3).astype(f32) if norm else None
    places = rows + 50
    cos, sin = tables_of(places, pairs)
    positions = rng.integers(0, places, rows).astype(np.int32)
    ts = [dev(ctx, a) if a is not None else None for a in (x, weight, cos if pairs else None, sin if pairs else None, positions if pairs else None)]
    y = ctx.rotate_heads(ts[0], heads, c, cos=ts[2], sin=ts[3], positions=ts[4], weight=ts[1], epsilon=1e-5, interleaved=interleaved, column=column)
    got = y.get_data().reshape(rows, heads, c)
    assert_heads(got, x[:, column:column + heads * c].reshape(rows, heads, c), weight, cos[positions], sin[positions], 1e-5, interleaved)
    ctx.sync()
    dispose(y, *ts)


def test_heads_in_place_and_rows_numbered(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(1)
    for c, pairs in ((64, 32), (256, 128), (40, 20)):
        x = rng.standard_normal((2, 50, 3 * c)).astype(f32)
        cos, sin = tables_of(100, pairs)
        t, tc, ts, w = dev(ctx, x), dev(ctx, cos), dev(ctx, sin), dev(ctx, np.ones(c, f32))
        y = ctx.rotate_heads(t, 3, c, cos=tc, sin=ts, weight=w, epsilon=0.0, out=t)
        assert y is t and y.dims == [2, 50, 3 * c]
        assert_heads(y.get_data().reshape(100, 3, c), x.reshape(100, 3, c), np.ones(c, f32), cos, sin, 0.0, False)
        dispose(t, tc, ts, w)


def test_heads_of_any_magnitude(cuda_context):
    """Squares of large or tiny numbers neither overflow nor vanish; a head of zeros stays zero; a NaN is its head's alone."""
    ctx = cuda_context
    x = np.ones((5, 2, 32), f32)
    x[0] *= f32(3e38)
    x[1] *= f32(1e-38)
    x[2] = 0
    x[3, 1, 5] = np.nan
    t, w = dev(ctx, x.reshape(5, 64)), dev(ctx, np.full(32, 2, f32))
    y = ctx.rotate_heads(t, 2, 32, weight=w, epsilon=1e-6)
    got = y.get_data().reshape(x.shape)
    assert np.allclose(got[0], 2, rtol=2.0 ** -22) and np.array_equal(got[2], np.zeros((2, 32), f32))
    assert_heads(got[1], x[1], np.full(32, 2, f32), np.zeros(0), np.zeros(0), 1e-6, False)
    y.dispose()
    y = ctx.rotate_heads(t, 2, 32, weight=w, epsilon=0.0)
    assert np.allclose(y.get_data().reshape(x.shape)[:2], 2, rtol=2.0 ** -20)
    assert np.isnan(got[3, 1]).all() and not np.isnan(got[3, 0]).any() and not np.isnan(got[4]).any()
    dispose(t, w, y)


def test_positions_out_of_range_count_as_the_nearest_and_are_reported(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(2)
    x = rng.standard_normal((3, 64)).astype(f32)
    cos, sin = tables_of(10, 32)
    t, tc, ts, p = dev(ctx, x), dev(ctx, cos), dev(ctx, sin), dev(ctx, np.array([-1, 10, 3], np.int32))
    y = ctx.rotate_heads(t, 1, 64, cos=tc, sin=ts, positions=p)
    with pytest.raises(CudaBackendError, match="position"):
        ctx.sync()
    ctx.sync()
    at = [0, 9, 3]
    assert_heads(y.get_data().reshape(3, 1, 64), x.reshape(3, 1, 64), None, cos[at], sin[at], 0, False)
    dispose(t, tc, ts, p, y)


# -------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("size,c,heads,kv_heads,lengths,counts,pairs,interleaved,norm", [
    (16, 32, 1, 1, [1], [1], 16, False, True), (16, 64, 12, 3, [17, 1, 16, 40], [1, 1, 1, 1], 32, False, True),
    (32, 128, 8, 2, [33, 64, 100], [33, 31, 1], 64, True, True), (64, 64, 5, 5, [200, 65, 3, 129], [200, 1, 0, 66], 16, False, True),
    (128, 128, 6, 2, [300, 128, 129], [173, 128, 2], 32, False, False), (16, 128, 7, 1, [50] * 9, [3] * 9, 64, True, False),
    (64, 32, 0, 2, [64, 63], [1, 63], 8, False, True), (32, 64, 3, 3, [70, 40], [20, 40], 0, False, True),
    (128, 64, 33, 1, [128, 200], [5, 5], 32, False, True)])
def test_append_of_rotated_keys(cuda_context, size, c, heads, kv_heads, lengths, counts, pairs, interleaved, norm):
    ctx, rng = cuda_context, np.random.default_rng(size + c + heads)
    cache = PagedCache(ctx, 2, sum(-(-n // size) for n in lengths) + 3, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    batch, tokens = len(lengths), max(counts)
    k, v = (rng.standard_normal((batch, tokens, kv_heads, c)).astype(f32) * 2 for _ in range(2))
    q = rng.standard_normal((batch, tokens, heads, c)).astype(f32) if heads else None
    qw, kw = ((1 + rng.standard_normal(c) * 0.2).astype(f32) for _ in range(2))
    cos, sin = tables_of(max(lengths) + 5, pairs)
    positions = np.minimum((np.array(lengths) - counts)[:, None] + np.arange(tokens), max(lengths)).astype(np.int32)
    place = lambda a, pad: np.pad(a.reshape(batch, tokens, -1), [(0, 0), (0, 0), pad])  # noqa: E731
    up = [dev(ctx, a) if a is not None else None for a in (
        place(k, (4, 0)), place(v, (0, 8)), table, np.asarray(lengths, np.int32), np.asarray(counts, np.int32), cos if pairs else None,
        sin if pairs else None, positions if pairs else None, place(q, (8, 4)) if heads else None, qw if norm and heads else None, kw if norm else None)]
    for _ in range(2):                                # (the same call again changes nothing)
        y = cache.append_rotary(1, *up[:5], cos=up[5], sin=up[6], positions=up[7], q=up[8], heads=heads or None, q_weight=up[9], k_weight=up[10],
                                epsilon=1e-6, interleaved=interleaved, k_column=4, q_column=8 if heads else 0)
        if heads:
            there = np.arange(tokens) < np.array(counts)[:, None]
            got = y.get_data().reshape(q.shape)
            assert not got[~there].any()
            assert_heads(got[there], q[there], qw if norm else None, cos[positions][there], sin[positions][there], 1e-6, interleaved)
            y.dispose()
        else:
            assert y is None
        turned = rotated(k, kw if norm else None, cos[positions], sin[positions], 1e-6, interleaved).astype(f32)
        reference_append(codes[1], scales[1], turned, v, table, lengths, counts, size)
        assert np.array_equal(pool_scales(cache), scales)
        assert np.array_equal(pool_codes(cache), codes)
    ctx.sync()
    dispose(*up)
    cache.dispose()


def test_append_without_positions_takes_the_places(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(5)
    lengths, counts = [40, 7, 90], [8, 7, 3]
    cos, sin = tables_of(100, 32)
    up = [dev(ctx, a) for a in (rng.standard_normal((3, 8, 64)).astype(f32), rng.standard_normal((3, 8, 64)).astype(f32))]
    where = [dev(ctx, np.array(a, np.int32)) for a in (lengths, counts)]
    tc, ts = dev(ctx, cos), dev(ctx, sin)
    places = dev(ctx, ((np.array(lengths) - counts)[:, None] + np.arange(8)).astype(np.int32))
    pools = []
    for positions in (None, places):
        cache = PagedCache(ctx, 1, 20, 1, 64, 16)
        set_pool(cache, np.zeros((1, 20, 2, 1, 16, 64), np.int8), np.zeros((1, 20, 2, 1), f32))
        t = dev(ctx, tables(np.random.default_rng(9), cache, lengths))
        q = cache.append_rotary(0, *up, t, *where, cos=tc, sin=ts, positions=positions, q=up[0])
        pools.append((pool_codes(cache), pool_scales(cache), q.get_data()))
        dispose(t, q)
        cache.dispose()
    assert all(np.array_equal(a, b) for a, b in zip(*pools))
    # without tables, weights and queries it is the plain append
    cache, other = PagedCache(ctx, 1, 20, 1, 64, 16), PagedCache(ctx, 1, 20, 1, 64, 16)
    t = dev(ctx, tables(np.random.default_rng(9), cache, lengths))
    for p in (cache, other):
        set_pool(p, np.zeros((1, 20, 2, 1, 16, 64), np.int8), np.zeros((1, 20, 2, 1), f32))
    cache.append_rotary(0, *up, t, *where)
    other.append(0, *up, t, *where)
    assert np.array_equal(pool_codes(cache), pool_codes(other)) and np.array_equal(pool_scales(cache), pool_scales(other))
    ctx.sync()
    dispose(t, tc, ts, places, *up, *where)
    cache.dispose()
    other.dispose()


# -------------------------------------------------------------------------------------------------- trees
def random_tree(rng, tokens, kind):
    if kind == "chain":
        return np.arange(-1, tokens - 1)
    if kind == "star":
        return np.where(np.arange(tokens) == 0, -1, 0)
    if kind == "apart":
        return np.full(tokens, -1)
    return np.array([-1] + [int(rng.integers(max(-1, i - 12), i)) for i in range(1, tokens)])


def reference_tree(q, codes, scales, table, lengths, counts, size, scale, parents):
    batch, tokens, heads, c = q.shape
    kv_heads = codes.shape[2]
    y, worst, top = np.zeros(q.shape), 0.0, 0.0
    for b, (length, count) in enumerate(zip(lengths, counts)):
        if not count:
            continue
        pages = np.asarray(table[b][:-(-length // size)])
        full = codes[pages].astype(np.float64) * scales[pages].astype(np.float64)[..., None, None]
        k, v = (full[:, i].transpose(1, 0, 2, 3).reshape(kv_heads, -1, c)[:, :length] for i in (0, 1))
        seen = np.zeros((count, length), bool)
        seen[:, :length - count] = True
        for i in range(count):
            j = i
            while j >= 0:
                seen[i, length - count + j] = True
                j = parents[b][j]
        for h in range(heads):
            g = h // (heads // kv_heads)
            qh = q[b, :count, h].astype(np.float64)
            s = np.where(seen, qh @ k[g].T * scale, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            y[b, :count, h] = p @ v[g] / p.sum(1, keepdims=True)
            worst = max(worst, (np.abs(qh) @ np.abs(k[g]).T * abs(scale)).max())
            top = max(top, np.abs(v[g]).max())
    return y, top * 2.0 ** -21 * (8 + 2 * worst)


def run_tree(ctx, cache, q, table, lengths, counts, parents, layer=0):
    b, t = q.shape[:2]
    ts = [dev(ctx, a) for a in (q.reshape(b, t, -1), np.asarray(table, np.int32), np.asarray(lengths, np.int32), np.asarray(counts, np.int32))]
    p = dev(ctx, np.asarray(parents, np.int32))
    y = cache.attention(layer, *ts, parents=p)
    got = y.get_data().reshape(q.shape)
    dispose(y, p, *ts)
    return got


@pytest.mark.parametrize("size,c,heads,kv_heads,lengths,counts,kind", [
    (16, 32, 2, 1, [5], [5], "any"), (16, 64, 4, 2, [40, 33, 1], [9, 7, 1], "any"), (32, 128, 4, 1, [100, 64, 95], [13, 13, 5], "any"),
    (64, 64, 6, 6, [300, 10, 0, 129], [40, 10, 0, 33], "any"), (128, 128, 8, 2, [700, 333], [31, 32], "star"), (16, 32, 8, 1, [64, 70], [33, 20], "apart"),
    (64, 128, 2, 2, [900], [64], "any"), (16, 64, 1, 1, [2000], [1], "any"), (32, 32, 3, 1, [1100], [1024], "any"), (64, 64, 1, 1, [700, 650], [600, 333], "any"),
    (64, 128, 32, 8, [500, 350, 400, 128], [25, 30, 16, 32], "any"), (64, 64, 16, 4, [200 + 13 * i for i in range(10)], [64 - i for i in range(10)], "any"),
    (128, 128, 16, 8, [2100, 1999, 1500, 64, 32], [64, 63, 33, 32, 31], "any"), (16, 128, 40, 5, [1030 + i for i in range(8)], [33] * 8, "star"),
    (32, 64, 24, 8, [1500 - 70 * i for i in range(20)], [5] * 20, "any"), (64, 128, 4, 4, [3000 + 500 * i for i in range(16)], [7] * 16, "any")])
def test_attention_of_a_tree(cuda_context, size, c, heads, kv_heads, lengths, counts, kind):
    rng = np.random.default_rng(size + c + len(lengths) + sum(counts))
    cache = PagedCache(cuda_context, 1, sum(-(-n // size) for n in lengths) + 3, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    q = rng.standard_normal((len(lengths), max(counts), heads, c)).astype(f32)
    parents = np.stack([random_tree(rng, max(counts), kind) for _ in lengths])
    got = run_tree(cuda_context, cache, q, table, lengths, counts, parents)
    cuda_context.sync()
    want, room = reference_tree(q, codes[0], scales[0], table, lengths, counts, size, c ** -0.5, parents)
    assert np.abs(got - want).max() <= room
    for b, n in enumerate(counts):
        assert not got[b, n:].any()
    # a chain is a text, whichever way its tokens are cut into parts: both are within `room` of it
    chain = np.tile(random_tree(rng, max(counts), "chain"), (len(lengths), 1))
    text = run_attention(cuda_context, cache, q, table, lengths, counts)
    assert np.abs(run_tree(cuda_context, cache, q, table, lengths, counts, chain) - text).max() <= 2 * room
    cache.dispose()


@pytest.mark.parametrize("tokens,heads", [(6, 2), (40, 8)])
def test_what_a_token_does_not_see_is_not_there(cuda_context, tokens, heads):
    """Another branch's values may be NaN, and a page of NaN behind the context is the business of the rows that see it."""
    ctx, rng = cuda_context, np.random.default_rng(tokens)
    cache = PagedCache(ctx, 1, 40, 1 if tokens < 40 else 8, 64, 16)
    codes, scales = random_pool(rng, cache)
    length, batch = 32 + tokens, 1 if tokens < 40 else 8
    table = tables(rng, cache, [length] * batch) if batch == 1 else np.tile(tables(rng, cache, [length]), (batch, 1))
    h = heads if batch == 1 else 16
    q = rng.standard_normal((batch, tokens, h, 64)).astype(f32)
    # every token continues the text directly; the first 16 are in a page whose scales are NaN
    parents = np.tile(np.full(tokens, -1), (batch, 1))
    scales[0, table[0][2]] = np.nan
    set_pool(cache, codes, scales)
    got = run_tree(ctx, cache, q, table, [length] * batch, [tokens] * batch, parents)
    assert np.isnan(got[:, :min(16, tokens)]).all()
    clean = scales.copy()
    clean[0, table[0][2]] = 1
    want, room = reference_tree(q, codes[0], clean[0], table, [length] * batch, [tokens] * batch, 16, 64 ** -0.5, parents)
    assert tokens <= 16 or np.abs(got[:, 16:] - want[:, 16:]).max() <= room
    cache.dispose()


@pytest.mark.parametrize("heads,kv_heads,c,lengths,counts", [
    (2, 1, 64, [30, 20, 9], [6, 1, 3]), (4, 1, 64, [3000], [3]), (16, 8, 128, [2100, 1999, 1500, 64], [64, 33, 1, 40]), (1, 1, 32, [400, 70], [60, 3])])
def test_rows_behind_the_new_tokens_are_zero_whatever_the_cache_holds(cuda_context, heads, kv_heads, c, lengths, counts):
    """Pages that stand for NaN, or whose values are infinite, are the business of the rows that are there."""
    ctx, rng = cuda_context, np.random.default_rng(c + len(lengths))
    cache = PagedCache(ctx, 1, sum(-(-n // 16) for n in lengths) + 3, kv_heads, c, 16)
    codes, scales = random_pool(rng, cache)
    table, tokens = tables(rng, cache, lengths), max(counts) + 4
    q = rng.standard_normal((len(lengths), tokens, heads, c)).astype(f32)
    parents = np.stack([random_tree(rng, tokens, "any") for _ in lengths])
    for value in (np.nan, np.inf):
        set_pool(cache, codes, np.full_like(scales, value))
        for got in (run_attention(ctx, cache, q, table, lengths, counts), run_tree(ctx, cache, q, table, lengths, counts, parents)):
            for b, n in enumerate(counts):
                assert np.isnan(got[b, :n]).all() and np.array_equal(got[b, n:], np.zeros_like(got[b, n:]))
    ctx.sync()
    cache.dispose()


def test_bad_parents_count_as_none_and_are_reported(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(4)
    cache = PagedCache(ctx, 1, 12, 2, 64, 16)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, [60])
    q = rng.standard_normal((1, 6, 4, 64)).astype(f32)
    parents = np.array([[0, -7, 2, 1 << 30, 9, 3]])
    got = run_tree_reporting(ctx, cache, q, table, [60], [6], parents)
    want, room = reference_tree(q, codes[0], scales[0], table, [60], [6], 16, 0.125, np.array([[-1, -1, -1, -1, -1, 3]]))
    assert np.abs(got - want).max() <= room
    cache.dispose()


def run_tree_reporting(ctx, cache, q, table, lengths, counts, parents):
    b, t = q.shape[:2]
    ts = [dev(ctx, a) for a in (q.reshape(b, t, -1), np.asarray(table, np.int32), np.asarray(lengths, np.int32), np.asarray(counts, np.int32))]
    p = dev(ctx, np.asarray(parents, np.int32))
    y = cache.attention(0, *ts, parents=p)
    with pytest.raises(CudaBackendError, match="parent"):
        ctx.sync()
    ctx.sync()
    got = y.get_data().reshape(q.shape)
    dispose(y, p, *ts)
    return got


# -------------------------------------------------------------------------------------------------- verdicts
def chances(x, temperature):
    x = x.astype(np.float64)
    if temperature == 0:
        p = np.zeros_like(x)
        p[int(x.argmax())] = 1
        return p
    e = np.exp((x - x.max()) / np.float64(f32(temperature)))
    return e / e.sum()


def taken_from(p, u):
    run = np.cumsum(p)
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24)
    return min(int(np.searchsorted(run, u * run[-1], side="right")), len(p) - 1)


def exists(x):
    return not (np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all())


def reference_verdict(logits, tokens, parents, count, uniforms, draft, temperature, draft_temperature):
    """(path, next) of one sequence."""
    if count == 0:
        return [], -1
    path = [0]
    while True:
        at = path[-1]
        children = [i for i in range(1, count) if parents[i] == at]
        if not exists(logits[at]):
            return path, -1
        p, found = chances(logits[at], temperature), None
        if draft is not None:
            if children and not exists(draft[at]):
                return path, -1
            for i in children:
                q = chances(draft[at], draft_temperature)
                there = 0 <= tokens[i] < len(p)
                if there and float(uniforms[i]) * q[tokens[i]] < p[tokens[i]]:
                    found = i
                    break
                left = np.maximum(p - q, 0)
                p = left / left.sum() if left.sum() > 0 else p
            token = taken_from(p, uniforms[0])
        else:
            token = taken_from(p, uniforms[at] if uniforms is not None else 0)
            found = next((i for i in children if tokens[i] == token), None)
        if found is None:
            return path, token
        path.append(found)


def run_verify(ctx, logits, tokens, parents, counts, uniforms, draft=None, temperature=1.0, draft_temperature=None, vocab=None):
    ints = [dev(ctx, np.asarray(a, np.int32)) if a is not None else None for a in (tokens, parents, counts)]
    floats = [dev(ctx, a.astype(f32)) if a is not None else None for a in (logits, uniforms, draft)]
    out = ctx.verify_drafts(floats[0], *ints, uniforms=floats[1], draft_logits=floats[2], temperature=temperature, draft_temperature=draft_temperature,
                            vocab=vocab)
    got = [t.get_data().reshape(t.dims) for t in out]
    dispose(*out, *ints, *floats)
    return got


def assert_verdicts(got, logits, tokens, parents, counts, uniforms, draft, temperature, draft_temperature=None):
    path, accepted, following = got
    batch, n = tokens.shape
    draft_temperature = temperature if draft_temperature is None else draft_temperature
    for b in range(batch):
        mine = parents[b] if parents is not None else np.arange(-1, n - 1)
        count = counts[b] if counts is not None else n
        want, token = reference_verdict(logits[b], tokens[b], mine, count, uniforms[b] if uniforms is not None else None,
                                        draft[b] if draft is not None else None, temperature, draft_temperature)
        assert path[b].tolist() == want + [-1] * (n - len(want)), b
        assert accepted[b] == len(want) and following[b] == token, b


def drafted(rng, batch, n, vocab, kind, with_draft, width=None, spread=2.0):
    width = width or vocab
    logits = (rng.standard_normal((batch, n, width)) * spread).astype(f32)
    guess = (logits + rng.standard_normal(logits.shape) * 0.5).astype(f32)
    parents = np.stack([random_tree(rng, n, kind) for _ in range(batch)]).astype(np.int32)
    parents[:, 1:] = np.maximum(parents[:, 1:], 0)
    tokens = rng.integers(0, vocab, (batch, n)).astype(np.int32)
    for b in range(batch):
        taken = {}
        for i in range(1, n):
            row = guess[b, parents[b, i], :vocab].astype(np.float64)
            if with_draft:
                tokens[b, i] = (row - np.log(-np.log(rng.random(vocab)))).argmax()
            else:
                taken[parents[b, i]] = taken.get(parents[b, i], -1) + 1
                tokens[b, i] = np.argsort(-row)[min(taken[parents[b, i]], vocab - 1)]
    return logits, guess if with_draft else None, parents, tokens, rng.random((batch, n)).astype(f32)


@pytest.mark.parametrize("batch,n,vocab,kind,with_draft,temperature", [
    (1, 1, 1, "chain", False, 1.0), (3, 4, 2, "chain", True, 1.0), (40, 6, 5, "any", True, 1.0), (40, 9, 7, "star", True, 0.7),
    (30, 12, 33, "any", False, 1.0), (9, 5, 1000, "chain", True, 1.3), (5, 16, 1003, "any", True, 1.0), (7, 16, 4098, "any", False, 0.8),
    (2, 8, 50001, "any", True, 1.0), (1, 5, 100003, "chain", True, 1.0), (3, 24, 32000, "star", True, 1.0), (3, 30, 32001, "any", False, 0.0),
    (70, 6, 20011, "any", True, 1.0), (300, 3, 999, "chain", False, 1.0), (20, 6, 300, "any", True, 0.0), (2, 100, 150, "any", True, 1.0),
    (2, 700, 40, "any", False, 1.0), (1, 3, 300007, "chain", True, 1.0)])
def test_verdicts(cuda_context, batch, n, vocab, kind, with_draft, temperature):
    rng = np.random.default_rng(batch + n + vocab)
    logits, draft, parents, tokens, uniforms = drafted(rng, batch, n, vocab, kind, with_draft)
    counts = np.array([max(0, n - int(rng.integers(0, 3)) * (i % 2)) for i in range(batch)], np.int32)
    got = run_verify(cuda_context, logits, tokens, parents, counts, uniforms, draft, temperature)
    cuda_context.sync()
    assert_verdicts(got, logits, tokens, parents, counts, uniforms, draft, temperature)


@pytest.mark.parametrize("with_draft", [False, True])
def test_verdicts_of_rows_that_are_cut_off_masked_or_missing(cuda_context, with_draft):
    ctx, rng = cuda_context, np.random.default_rng(11)
    batch, n, vocab, width = 12, 7, 517, 519
    logits, draft, parents, tokens, uniforms = drafted(rng, batch, n, vocab, "any", with_draft, width)
    logits[..., vocab:] = 1e30                        # columns behind the vocabulary
    logits[:6][rng.random(logits[:6].shape) < 0.6] = -np.inf
    logits[0, 0, :] = -np.inf
    logits[1, 0, 3] = np.nan
    logits[2, 0, vocab - 1] = np.inf
    logits[3, 0, :] = -np.inf
    logits[3, 0, 400] = np.finfo(f32).min
    logits[..., vocab:] = 1e30
    if with_draft:
        draft[4, 0, 9] = np.nan
        draft[5, 0, rng.random(width) < 0.5] = -np.inf
        draft[..., vocab:] = np.inf
    tokens[6, 1:] = -1
    tokens[7, 1:] = vocab
    counts = np.full(batch, n)
    counts[8], counts[9], counts[10] = 0, 1, 2
    uniforms[11], uniforms[10] = 0, 1 - 2.0 ** -24
    got = run_verify(ctx, logits, tokens, parents, counts, uniforms, draft, 1.0, vocab=vocab)
    ctx.sync()
    cut = [a[..., :vocab] if a is not None else None for a in (logits, draft)]
    assert_verdicts(got, cut[0], tokens, parents, counts, uniforms, cut[1], 1.0)


def test_verdicts_without_trees_counts_or_random_numbers(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(12)
    logits, draft, _, tokens, uniforms = drafted(rng, 5, 6, 40, "chain", True)
    got = run_verify(ctx, logits, tokens, None, None, uniforms, draft)
    assert_verdicts(got, logits, tokens, None, None, uniforms, draft, 1.0)
    got = run_verify(ctx, logits, tokens, None, None, None, None, 0.0)
    assert_verdicts(got, logits, tokens, None, None, None, None, 0.0)
    # the largest logit is there several times: the first
    logits[:, :, 7] = logits[:, :, 30] = logits[:, :, 31] = 50
    got = run_verify(ctx, logits, np.full((5, 6), 7), None, None, None, None, 0.0)
    assert (got[1] == 6).all() and (got[2] == 7).all()
    # drafts with a distribution that are decided by the largest logit, and the other way round
    for t, dt in ((0.0, 1.0), (1.0, 0.0), (0.0, 0.0), (0.5, 2.0)):
        got = run_verify(ctx, logits, tokens, None, None, uniforms, draft, t, dt)
        assert_verdicts(got, logits, tokens, None, None, uniforms, draft, t, dt)


@pytest.mark.parametrize("with_draft", [False, True])
def test_drafts_do_not_change_what_is_said(cuda_context, with_draft):
    """The first new token has the target's distribution, whatever was drafted: 30000 sequences, each share within five standard deviations."""
    ctx, rng = cuda_context, np.random.default_rng(13)
    batch, n, vocab = 30000, 4, 6
    row, guess = rng.standard_normal(vocab).astype(f32), rng.standard_normal(vocab).astype(f32)
    logits, draft = np.broadcast_to(row, (batch, n, vocab)), np.broadcast_to(guess, (batch, n, vocab))
    q = chances(guess, 1.0)
    tokens = rng.choice(vocab, (batch, n), p=q)
    parents = np.tile(np.array([-1, 0, 0, 0]), (batch, 1))
    path, accepted, following = run_verify(ctx, logits, tokens, parents, None, rng.random((batch, n)).astype(f32), draft if with_draft else None)
    first = np.where(accepted > 1, tokens[np.arange(batch), np.maximum(path[:, 1], 0)], following)
    p = chances(row, 1.0)
    share = np.bincount(first, minlength=vocab) / batch
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / batch)).all()
    assert with_draft is False or (accepted > 1).mean() > 0.3


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab,spread", [(3001, 0.1), (3001, 3.0), (40009, 0.5)])
def test_verdicts_beside_the_borders_of_tokens(cuda_context, vocab, spread, with_draft):
    """Random numbers that are the float32 numbers next to a border of the running sum, and those that a draft stands or falls by: 32 bits
    do not tell on which side they are."""
    rng = np.random.default_rng(vocab)
    batch, n = 60, 3
    logits, draft, parents, tokens, uniforms = drafted(rng, batch, n, vocab, "chain", with_draft, spread=spread)
    for b in range(batch):
        p, u = chances(logits[b, 0], 1.0), rng.integers(-1, 2)
        if with_draft and b % 2:
            q = chances(draft[b, 0], 1.0)
            tokens[b, 1] = np.where(p < q, q, 0).argmax()
            border = p[tokens[b, 1]] / q[tokens[b, 1]]
            uniforms[b, 1] = f32(border) * f32(1 + u * 2.0 ** -23)
        else:
            left = p
            if with_draft:
                tokens[b, 1], q = vocab, chances(draft[b, 0], 1.0)               # (never stands: a rejection, then a draw)
                left = np.maximum(p - q, 0)
            border = np.cumsum(left)[rng.integers(0, vocab)] / left.sum()
            uniforms[b, 0] = min(f32(border) * f32(1 + u * 2.0 ** -23), f32(1 - 2.0 ** -24))
    got = run_verify(cuda_context, logits, tokens, parents, None, uniforms, draft, 1.0)
    cuda_context.sync()
    assert_verdicts(got, logits, tokens, parents, None, uniforms, draft, 1.0)


def test_results_of_verdicts_overlap_nothing(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(15)
    logits, _, parents, tokens, uniforms = drafted(rng, 3, 5, 50, "chain", False)
    ints = [dev(ctx, np.asarray(a, np.int32)) for a in (tokens, parents, np.full(3, 5))]
    floats = [dev(ctx, logits), dev(ctx, uniforms)]
    out = [ctx.empty_tensor(d, "int32") for d in ([3, 5], [3], [3])]
    for bad in ((ints[0], out[1], out[2]), (ints[1], out[1], out[2]), (out[0], ints[2], out[2]), (out[0], out[1], ints[2]), (out[0], out[1], out[1])):
        with pytest.raises(CudaBackendError, match="overlaps"):
            ctx.verify_drafts(floats[0], *ints, uniforms=floats[1], out=bad)
    ctx.verify_drafts(floats[0], *ints, uniforms=floats[1], out=out)
    ctx.sync()
    assert_verdicts([t.get_data().reshape(t.dims) for t in out], logits, tokens, parents, None, uniforms, None, 1.0)
    dispose(*out, *ints, *floats)


def test_bad_parents_and_counts_of_verdicts_are_reported(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(14)
    logits, _, parents, tokens, uniforms = drafted(rng, 3, 5, 50, "chain", False)
    fixed = parents.copy()
    parents[0] = [3, 0, 2, -5, 100]
    fixed[0] = [-1, 0, -1, -1, -1]
    counts = np.array([5, -1, 6])
    ints = [dev(ctx, np.asarray(a, np.int32)) for a in (tokens, parents, counts)]
    floats = [dev(ctx, logits), dev(ctx, uniforms)]
    out = ctx.verify_drafts(floats[0], *ints, uniforms=floats[1])
    with pytest.raises(CudaBackendError, match="parent"):
        ctx.sync()
    got = [t.get_data().reshape(t.dims) for t in out]
    assert_verdicts(got, logits, tokens, fixed, np.array([5, 0, 0]), uniforms, None, 1.0)
    dispose(*out, *ints, *floats)


# -------------------------------------------------------------------------------------------------- kept paths
def reference_keep(codes, scales, table, lengths, counts, path, accepted, size):
    """Pools [layers, pages, 2, heads, size, c] and [layers, pages, 2, heads], in place, in the 32-bit steps of the definition."""
    for b, (length, count) in enumerate(zip(lengths, counts)):
        start, kept = length - count, accepted[b]
        if kept == 0 or all(path[b][i] == i for i in range(kept)):
            continue
        for p in range(start // size, (start + kept - 1) // size + 1):
            page = table[b][p]
            before = scales[:, page].copy()
            scale, moves = before.copy(), []
            for i in range(kept):
                if (start + i) // size != p:
                    continue
                at = start + path[b][i]
                of = table[b][at // size]
                x, by = codes[:, of, :, :, at % size].copy(), scales[:, of].copy()
                moves.append(((start + i) % size, of == page, x, by))
                if of != page:
                    scale = np.maximum(scale, np.abs(x.astype(f32)).max(-1) * by / f32(127))
            grown = (scale > before)[..., None, None]
            safe = np.where(scale > 0, scale, f32(1))[..., None]
            old = max(start - p * size, 0)
            again = np.clip(np.rint(codes[:, page, :, :, :old].astype(f32) * before[..., None, None] / safe[..., None]), -127, 127)
            codes[:, page, :, :, :old] = np.where(grown, again, codes[:, page, :, :, :old])
            for slot, stays, x, by in moves:
                again = np.clip(np.rint(x.astype(f32) * by[..., None] / safe), -127, 127)
                codes[:, page, :, :, slot] = np.where(stays & ~grown[..., 0], x, again)
            scales[:, page] = scale


def run_keep(ctx, cache, table, lengths, counts, path, accepted):
    ts = [dev(ctx, np.asarray(a, np.int32)) for a in (table, lengths, counts, path, accepted)]
    cache.keep_paths(*ts)
    dispose(*ts)


@pytest.mark.parametrize("size,c,heads,layers,lengths,counts,accepted", [
    (16, 32, 1, 1, [5], [5], [3]), (16, 64, 3, 4, [40, 33, 16], [9, 20, 16], [4, 12, 9]), (32, 128, 2, 3, [100, 64, 95], [13, 64, 40], [6, 40, 1]),
    (64, 64, 8, 2, [300, 10, 0, 129], [40, 10, 0, 33], [17, 10, 0, 0]), (128, 128, 2, 2, [700, 333], [200, 250], [150, 129]),
    (16, 128, 5, 7, [90 + i for i in range(12)], [30] * 12, [5] * 12), (16, 32, 2, 1, [600], [512], [300])])
def test_kept_paths(cuda_context, size, c, heads, layers, lengths, counts, accepted):
    ctx, rng = cuda_context, np.random.default_rng(size + c + heads)
    cache = PagedCache(ctx, layers, sum(-(-n // size) for n in lengths) + 3, heads, c, size)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    path = np.full((len(lengths), max(counts)), -1)
    for b, (n, k) in enumerate(zip(counts, accepted)):
        path[b, :k] = np.sort(rng.choice(n, k, replace=False))
    run_keep(ctx, cache, table, lengths, counts, path, accepted)
    ctx.sync()
    reference_keep(codes, scales, table, lengths, counts, path, accepted, size)
    assert np.array_equal(pool_scales(cache), scales)
    assert np.array_equal(pool_codes(cache), codes)
    cache.dispose()


def test_kept_paths_of_pages_without_numbers(cuda_context):
    """A page that stands for NaN stays one; a token of such a page makes its new page one; zeros move as they are."""
    ctx, rng = cuda_context, np.random.default_rng(3)
    for nan, value in ((0, np.nan), (1, np.nan), (1, np.inf), (1, 0.0), (0, 0.0)):
        cache = PagedCache(ctx, 1, 4, 1, 32, 16)
        codes, scales = random_pool(rng, cache)
        table = np.array([[0, 1]])
        scales[0, nan] = value
        if value == 0:
            codes[0, nan] = 0
        set_pool(cache, codes, scales)
        run_keep(ctx, cache, table, [30], [20], [[0, 9, 12] + [-1] * 17], [3])
        got, by = pool_codes(cache)[0, 0].astype(np.float64), pool_scales(cache)[0, 0].astype(np.float64)
        if value != 0:
            assert not np.isfinite(by).any() and (nan == 0 or np.isnan(by).all())
            assert nan == 1 or not np.array_equal(got[:, :, 11], codes[0, 1][:, :, 3])
        elif nan == 1:
            assert np.array_equal(by, scales[0, 0]) and not got[:, :, 11:13].any()
        else:
            want = codes[0, 1][:, :, [3, 6]] * scales[0, 1].astype(np.float64)[..., None, None]
            # (half a step, and the quotient's two roundings: 127 * 2^-23 of a step)
            assert np.abs(got[:, :, 11:13] * by[..., None, None] - want).max() <= (by.max() / 2) * (1 + 2.0 ** -14)
        ctx.sync()
        cache.dispose()


def test_kept_paths_of_numbers_of_any_magnitude(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(8)
    cache = PagedCache(ctx, 1, 30, 2, 64, 16)
    codes, scales = random_pool(rng, cache)
    lengths, counts, accepted = [30] * 9, [20] * 9, [12] * 9
    table = tables(rng, cache, lengths)
    path = np.stack([np.pad(np.sort(rng.choice(20, 12, replace=False)), (0, 8), constant_values=-1) for _ in lengths])
    for b, (first, second) in enumerate(((1e36, 1e35), (1e35, 1e36), (2e36, 1e30), (1e-30, 1e-36), (1e-36, 1e-30), (1e-40, 1e-42), (1e29, 1e31), (1e-29, 1e-31), (1e-45, 1e36))):
        scales[0, table[b][0]], scales[0, table[b][1]] = first, second
    set_pool(cache, codes, scales)
    run_keep(ctx, cache, table, lengths, counts, path, accepted)
    ctx.sync()
    reference_keep(codes, scales, table, lengths, counts, path, accepted, 16)
    assert np.array_equal(pool_scales(cache), scales) and np.array_equal(pool_codes(cache), codes)
    cache.dispose()


def test_paths_that_do_not_fit_leave_their_sequence_alone(cuda_context):
    ctx, rng = cuda_context, np.random.default_rng(6)
    cache = PagedCache(ctx, 2, 20, 2, 64, 16)
    codes, scales = random_pool(rng, cache)
    lengths, counts = [30, 30, 30, 30, 30, 30], [8, 8, 8, 8, 8, 8]
    table = tables(rng, cache, lengths)
    path = np.array([[0, 2, 2, -1], [0, 3, 1, -1], [0, 2, 8, -1], [-1, 2, 3, -1], [0, 2, 4, 6], [0, 3, 5, 7]])
    path = np.pad(path, [(0, 0), (0, 4)], constant_values=-1)
    accepted = [3, 3, 3, 3, 9, 4]
    run_keep(ctx, cache, table, lengths, counts, path, accepted)
    with pytest.raises(CudaBackendError, match="path"):
        ctx.sync()
    ctx.sync()
    reference_keep(codes, scales, table, lengths, counts, path, [0, 0, 0, 0, 0, 4], 16)
    assert np.array_equal(pool_scales(cache), scales) and np.array_equal(pool_codes(cache), codes)
    run_keep(ctx, cache, table, lengths, counts, path, [0, -1, 0, 0, 0, 0])
    with pytest.raises(CudaBackendError, match="path"):
        ctx.sync()
    assert np.array_equal(pool_scales(cache), scales) and np.array_equal(pool_codes(cache), codes)
    cache.dispose()


# -------------------------------------------------------------------------------------------------- verdicts: what has no say
@pytest.mark.parametrize("batch,n,vocab,temperature,whole", [
    (40, 2, 50, 1.0, False), (40, 5, 1003, 0.7, False), (30, 4, 1000, 1.0, True), (8, 6, 40009, 1.0, False), (3, 3, 300007, 1.3, False)])
def test_drafts_that_never_stand_leave_the_target_where_both_are_equal(cuda_context, batch, n, vocab, temperature, whole):
    """max(p - q, 0) of equal distributions is 0 everywhere, and p stays, however often a draft that never stands (a token outside of the
    vocabulary, or one that weighs nothing on either side) is rejected: the next token is drawn from p."""
    ctx, rng = cuda_context, np.random.default_rng(batch + vocab)
    logits = (rng.standard_normal((batch, n, vocab)) * 2).astype(f32)
    draft = logits.copy()
    if whole:                                        # (whole numbers: equal distributions of different logits)
        logits = np.rint(logits)
        draft = logits + f32(5)
    logits[:, :, 7] = draft[:, :, 7] = -np.inf
    parents = np.tile(np.where(np.arange(n) == 0, -1, 0), (batch, 1))
    tokens = rng.choice([-1, vocab, 7, 1 << 30], (batch, n))
    uniforms = rng.random((batch, n)).astype(f32)
    for wider in (0, 1):                             # (rows of the draft's that begin elsewhere in their 16 bytes)
        got = run_verify(ctx, logits, tokens, parents, None, uniforms, np.pad(draft, [(0, 0), (0, 0), (0, wider)]), temperature, vocab=vocab)
        ctx.sync()
        assert_verdicts(got, logits, tokens, parents, None, uniforms, draft, temperature)
        for b in range(batch):
            assert got[1][b] == 1 and got[2][b] == taken_from(chances(logits[b, 0], temperature), uniforms[b, 0])


@pytest.mark.parametrize("with_draft", [False, True])
def test_verdicts_of_sequences_without_tokens(cuda_context, with_draft):
    """No rows are there, and no memory of them: nothing is asked for."""
    ctx = cuda_context
    empty = lambda *dims: ctx.empty_tensor(list(dims))  # noqa: E731
    ints = [ctx.empty_tensor([3, 0], "int32"), ctx.empty_tensor([3, 0], "int32"), dev(ctx, np.zeros(3, np.int32))]
    floats = [empty(3, 0, 40000), empty(3, 0), empty(3, 0, 40000)]
    for counts in (None, ints[2]):
        out = ctx.verify_drafts(floats[0], ints[0], ints[1], counts, floats[1], floats[2] if with_draft else None)
        assert out[0].dims == [3, 0] and out[1].get_data().tolist() == [0] * 3 and out[2].get_data().tolist() == [-1] * 3
        dispose(*out)
    ctx.sync()
    dispose(*ints, *floats)


@pytest.mark.parametrize("missing", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("vocab", [5, 3001, 40009])
def test_rows_of_drafts_behind_tokens_without_children_have_no_say(cuda_context, vocab, missing):
    """A drafter need not run behind its last tokens.  Random numbers beside a border of a leaf's running sum, so that 32 bits do not decide
    there; and sequences whose first token has no children, though others are there."""
    ctx, rng = cuda_context, np.random.default_rng(vocab)
    batch, n = 24, 4
    logits, draft, _, tokens, uniforms = drafted(rng, batch, n, vocab, "star", True)
    parents = np.tile([-1, 0, 1, 1], (batch, 1))
    parents[::4] = -1
    parents[1::4] = [-1, 0, 0, 0]
    for b in range(batch):
        for i in range(n):
            if not (parents[b, i + 1:] == i).any():
                draft[b, i] = missing
        uniforms[b, 1:] = 0                          # (every draft that weighs anything stands)
        leaf = 0 if b % 4 == 0 else 1 if b % 4 == 1 else 2
        run = np.cumsum(chances(logits[b, leaf], 1.0))
        uniforms[b, 0] = min(f32(run[rng.integers(0, vocab)] / run[-1]), f32(1 - 2.0 ** -24))
    got = run_verify(ctx, logits, tokens, parents, None, uniforms, draft, 1.0)
    ctx.sync()
    assert_verdicts(got, logits, tokens, parents, None, uniforms, draft, 1.0)
    assert got[1].tolist() == [1, 2, 3, 3] * (batch // 4) and (got[2] >= 0).all()


# -------------------------------------------------------------------------------------------------- results beside operands
def test_heads_that_overlap_others_are_refused(cuda_context):
    """What groups write in no order must not be what others still read; columns of one buffer are no overlap."""
    ctx, rng = cuda_context, np.random.default_rng(21)
    rows, heads, c, wide = 700, 3, 32, 200
    x = rng.standard_normal((rows, wide)).astype(f32)
    room = dev(ctx, np.concatenate([x.reshape(-1), np.zeros(4 * wide, f32)]))
    cos, sin = tables_of(rows, 16)
    tc, ts = dev(ctx, cos), dev(ctx, sin)

    def call(y, y_st=wide, y_sh=c, n=rows):
        desc = lib.RotateDesc(n, heads, c, 32, rows, wide, c, y_st, y_sh, 1e-6, 0)
        ctx._call("wdc_rotate_heads", byref(desc), room.ptr, None, tc.ptr, ts.ptr, None, room.ptr + 4 * y)

    width = heads * c
    for bad in (dict(y=4), dict(y=c), dict(y=width - 4), dict(y=wide), dict(y=5 * wide), dict(y=5 * wide + width - 4), dict(y=wide - 4), dict(y=0, y_st=width),
                dict(y=0, y_st=wide + 4), dict(y=width, y_st=width), dict(y=0, y_sh=c + 4), dict(y=width, y_sh=2 * c), dict(y=c, n=1)):
        with pytest.raises(CudaBackendError, match="overlaps"):
            call(**bad)
    borrowed = ctx.borrow_tensor(room.ptr + 16, [rows, wide], "float32", owner=room)
    whole = ctx.borrow_tensor(room.ptr, [rows, wide], "float32", owner=room)
    with pytest.raises(CudaBackendError, match="overlaps"):
        ctx.rotate_heads(whole, wide // 40, 40, out=borrowed)
    ctx.sync()
    assert np.array_equal(room.get_data()[:rows * wide].reshape(rows, wide), x)
    want = x.copy()
    call(width)                                      # beside x, and then in its place
    got = room.get_data()[:rows * wide].reshape(rows, wide)
    assert_heads(got[:, width:2 * width].reshape(rows, heads, c), x[:, :width].reshape(rows, heads, c), None, cos, sin, 1e-6, False)
    want[:, width:2 * width] = got[:, width:2 * width]
    assert np.array_equal(got, want)
    call(0)
    assert np.array_equal(room.get_data()[:rows * wide].reshape(rows, wide)[:, :width], got[:, width:2 * width])
    call(wide, n=1)                                  # (one row, behind itself)
    ctx.sync()
    dispose(borrowed, whole, room, tc, ts)


def test_queries_of_an_append_that_overlap_its_operands_are_refused(cuda_context):
    """Keys are read by other groups than those that write queries.  Results that are columns of the operands' buffer are no overlap."""
    ctx, rng = cuda_context, np.random.default_rng(22)
    batch, tokens, heads, kv_heads, c, size = 3, 40, 4, 2, 32, 16
    width, wide = heads * c, (2 * heads + 2 * kv_heads) * c
    fused = rng.standard_normal((batch, tokens, wide)).astype(f32)          # q, k, v, and a place for the result
    k0, v0, y0 = width, width + kv_heads * c, width + 2 * kv_heads * c
    lengths, counts = [50, 40, 45], [40, 33, 1]
    cache = PagedCache(ctx, 1, 20, kv_heads, c, size)
    codes, scales = random_pool(rng, cache)
    room, table = dev(ctx, np.concatenate([fused.reshape(-1), np.zeros(batch * tokens * wide, f32)])), tables(rng, cache, lengths)
    where = [dev(ctx, np.asarray(a, np.int32)) for a in (table, lengths, counts)]
    cos, sin = tables_of(60, 16)
    tc, ts = dev(ctx, cos), dev(ctx, sin)

    def call(y, q=0, y_sb=tokens * wide, y_st=wide, y_sh=c):
        append = lib.CacheAppendDesc(20, kv_heads, size, c, batch, tokens, table.shape[1], tokens * wide, c, wide, tokens * wide, c, wide)
        desc = lib.CacheAppendRotaryDesc(append, heads, tokens * wide, c, wide, y_sb, y_sh, y_st, 32, 60, 1e-6, 0)
        ctx._call("wdc_cache_append_rotary", byref(desc), room.ptr + 4 * q, room.ptr + 4 * k0, room.ptr + 4 * v0, None, None, tc.ptr, ts.ptr, None,
                  cache.codes.ptr, cache.scales.ptr, *[t.ptr for t in where], room.ptr + 4 * y)

    behind = batch * tokens * wide
    for bad in (dict(y=4), dict(y=k0), dict(y=k0 - c), dict(y=v0), dict(y=v0 + 4), dict(y=y0 - 4), dict(y=wide), dict(y=0, y_st=width), dict(y=0, y_sb=tokens * wide + 4),
                dict(y=y0, y_st=width, y_sb=tokens * width), dict(y=behind - width - 4, y_st=width, y_sb=tokens * width), dict(y=y0, q=y0 - 4)):
        with pytest.raises(CudaBackendError, match="overlaps"):
            call(**bad)
    # the call of a program whose queries come out where its keys are
    whole = ctx.borrow_tensor(room.ptr, [batch, tokens, wide], "float32", owner=room)
    out = ctx.borrow_tensor(room.ptr, [batch, tokens, width], "float32", owner=room)
    keys = ctx.borrow_tensor(room.ptr, [batch, tokens, width], "float32", owner=room)
    for args in (dict(q=whole, heads=heads, out=out), dict(q=dev(ctx, np.zeros((batch, tokens, width), f32)), out=keys)):
        with pytest.raises((CudaBackendError, ValueError)):
            cache.append_rotary(0, whole, whole, *where, cos=tc, sin=ts, k_column=k0, v_column=v0, **args)
    ctx.sync()
    assert np.array_equal(room.get_data()[:behind], fused.reshape(-1)) and np.array_equal(pool_codes(cache), codes)
    positions = np.minimum((np.array(lengths) - counts)[:, None] + np.arange(tokens), 59)
    there = np.arange(tokens) < np.array(counts)[:, None]
    heads_of = lambda a, at, n: a[..., at:at + n * c].reshape(batch, tokens, n, c)  # noqa: E731
    turned = rotated(heads_of(fused, k0, kv_heads), None, cos[positions], sin[positions], 0.0, False).astype(f32)
    reference_append(codes[0], scales[0], turned, heads_of(fused, v0, kv_heads), table, lengths, counts, size)
    results = []
    for args in (dict(y=y0), dict(y=behind), dict(y=0)):     # beside the operands, behind them, in the queries' place
        call(**args)
        got = room.get_data()
        results.append(heads_of(got[args["y"] // behind * behind:][:behind].reshape(fused.shape), args["y"] % behind, heads))
        assert np.array_equal(pool_codes(cache), codes) and np.array_equal(pool_scales(cache), scales)
        kept = got[:behind].reshape(fused.shape)
        assert np.array_equal(kept[..., k0:y0], fused[..., k0:y0])
    assert_heads(results[0][there], heads_of(fused, 0, heads)[there], None, cos[positions][there], sin[positions][there], 0.0, False)
    assert not results[0][~there].any() and all(np.array_equal(results[0], r) for r in results[1:])
    ctx.sync()
    dispose(whole, out, keys, room, tc, ts, *where)
    cache.dispose()


@pytest.mark.parametrize("wider", [1, 2, 3])
@pytest.mark.parametrize("vocab", [37, 1002, 20011, 120001])
def test_verdicts_of_rows_that_begin_at_different_places_in_16_bytes(cuda_context, vocab, wider):
    rng = np.random.default_rng(vocab + wider)
    logits, draft, parents, tokens, uniforms = drafted(rng, 6, 7, vocab, "any", True)
    counts = np.array([7, 7, 6, 5, 7, 1], np.int32)
    wide = np.concatenate([draft, np.full((6, 7, wider), np.nan, f32)], 2)
    got = run_verify(cuda_context, logits, tokens, parents, counts, uniforms, wide, 0.9, vocab=vocab)
    cuda_context.sync()
    assert_verdicts(got, logits, tokens, parents, counts, uniforms, draft, 0.9)


@pytest.mark.parametrize("c,heads,kv_heads,lengths,counts,width", [
    (128, 32, 8, [900], [13], 512), (64, 16, 4, [900, 31], [11, 11], 700), (128, 16, 8, [300, 40, 0], [64, 40, 0], 300), (32, 4, 2, [70], [33], 900)])
def test_trees_with_tables_that_are_wider_than_their_texts(cuda_context, c, heads, kv_heads, lengths, counts, width):
    """Most parts of a tile have nothing to do, as with the tables of a program that has them as wide as its longest text may be."""
    rng = np.random.default_rng(c + width)
    cache = PagedCache(cuda_context, 1, sum(-(-n // 64) for n in lengths) + 3, kv_heads, c, 64)
    codes, scales = random_pool(rng, cache)
    table = tables(rng, cache, lengths)
    table = np.pad(table, [(0, 0), (0, width - table.shape[1])], constant_values=-1)
    q = rng.standard_normal((len(lengths), max(counts), heads, c)).astype(f32)
    for kind in ("any", "chain"):
        parents = np.stack([random_tree(rng, max(counts), kind) for _ in lengths])
        got = run_tree(cuda_context, cache, q, table, lengths, counts, parents)
        cuda_context.sync()
        want, room = reference_tree(q, codes[0], scales[0], table, lengths, counts, 64, c ** -0.5, parents)
        assert np.abs(got - want).max() <= room
        for b, n in enumerate(counts):
            assert not got[b, n:].any()
    cache.dispose()
