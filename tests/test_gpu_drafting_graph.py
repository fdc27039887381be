"""The operators of a decoder that drafts as nodes of a graph, in captured graphs, and together in the loop that drafts and decides; and
what the device library refuses.  Tolerances are those of the operators (test_gpu_drafting) and of a whole decoder (test_gpu_decode).
"""
from ctypes import byref

import numpy as np
import pytest

from test_gpu_decode import model_of
from test_gpu_drafting import (assert_heads, assert_verdicts, dispose, drafted, random_tree, reference_tree, rotated, tables_of)
from test_gpu_paged_cache import dev, pool_codes, pool_scales, random_pool, reference_append, tables
from util import run_cuda, single_op_model
from webdnn_b200 import lib
from webdnn_b200.backend import CPUTensor
from webdnn_b200.decode import Decoder
from webdnn_b200.lib import CudaBackendError
from webdnn_b200.onnx_io import FLOAT, INT32, make_node
from webdnn_b200.paged_cache import PagedCache
from webdnn_b200.runner import load

pytestmark = pytest.mark.gpu
f32 = np.float32


# -------------------------------------------------------------------------------------------------- nodes
@pytest.mark.parametrize("rank", [3, 4])
@pytest.mark.parametrize("ids", [True, False])
@pytest.mark.parametrize("size,rotary,interleaved", [(64, 0, 0), (80, 32, 1), (256, 128, 0)])
def test_rotary_embedding_node(cuda_context, rank, ids, size, rotary, interleaved):
    rng = np.random.default_rng(size + rank)
    batch, heads, tokens, pairs = 3, 2, 5, (rotary or size) // 2
    x = rng.standard_normal((batch, tokens, heads, size)).astype(f32)
    cos, sin = tables_of(40, pairs)
    places = rng.integers(0, 40, (batch, tokens)).astype(np.int32)
    given = x.reshape(batch, tokens, -1) if rank == 3 else np.ascontiguousarray(x.transpose(0, 2, 1, 3))
    attrs = dict(interleaved=interleaved, rotary_embedding_dim=rotary, _opset=23, **(dict(num_heads=heads) if rank == 3 else {}))
    inputs = [given, cos, sin, places] if ids else [given, cos[places], sin[places]]
    (got,) = run_cuda(single_op_model("RotaryEmbedding", attrs, inputs), inputs, cuda_context)
    got = got.reshape(batch, tokens, heads, size) if rank == 3 else got.reshape(batch, heads, tokens, size).transpose(0, 2, 1, 3)
    assert_heads(got, x, None, cos[places], sin[places], 0.0, bool(interleaved))


def test_rotate_heads_node(cuda_context):
    rng = np.random.default_rng(2)
    x, weight, places = rng.standard_normal((2, 7, 160)).astype(f32), rng.standard_normal(32).astype(f32), rng.integers(0, 20, (2, 7)).astype(np.int32)
    cos, sin = tables_of(20, 8)
    attrs = dict(extras="weight,positions,cos,sin", heads=3, head_size=32, column=64, epsilon=1e-5)
    inputs = [x, weight, places, cos, sin]
    (got,) = run_cuda(single_op_model("CudaRotateHeads", attrs, inputs), inputs, cuda_context)
    assert_heads(got.reshape(2, 7, 3, 32), x[..., 64:].reshape(2, 7, 3, 32), weight, cos[places], sin[places], 1e-5, False)


@pytest.mark.parametrize("replay", [True, False])
def test_cache_attention_node_of_rotated_trees_run_after_run(cuda_context, replay):
    ctx, rng = cuda_context, np.random.default_rng(1)
    b, t, heads, kv, c, size = 3, 6, 4, 2, 32, 16
    cache = PagedCache(ctx, 2, 40, kv, c, size)
    name = f"trees {replay}"
    ctx.add_cache(name, cache)
    cache.codes.set_data(np.zeros(cache.codes.dims, np.int32))
    cache.scales.set_data(np.zeros(cache.scales.dims, f32))
    codes, scales = np.zeros((40, 2, kv, size, c), np.int8), np.zeros((40, 2, kv), f32)
    cos, sin = tables_of(100, 16)
    qw, kw = ((1 + rng.standard_normal(c) * 0.2).astype(f32) for _ in range(2))
    shapes = dict(q=[b, t, heads * c], k=[b, t, kv * c], v=[b, t, kv * c], table=[b, 6], lengths=[b], counts=[b], positions=[b, t], cos=[100, 16],
                  sin=[100, 16], q_weight=[c], k_weight=[c], parents=[b, t])
    kinds = {n: INT32 if n in ("table", "lengths", "counts", "positions", "parents") else FLOAT for n in shapes}
    node = make_node("CudaCacheAttention", list(shapes), ["y"], cache=name, layer=1, extras="positions,cos,sin,q_weight,k_weight,parents")
    runner = load(model_of(node, [(n, kinds[n], d) for n, d in shapes.items()], [("y", FLOAT)]), backend_order=["cuda", "cpu"],
                  backend_options={"cuda": {"context": ctx, "graphReplay": replay}})
    lengths, table = np.zeros(b, np.int32), tables(rng, cache, [96] * b, 0)
    for step in range(7):
        counts = rng.integers(0, t + 1, b).astype(np.int32)
        lengths = lengths + counts
        q, k, v = (rng.standard_normal((b, t, n, c)).astype(f32) for n in (heads, kv, kv))
        positions = rng.integers(0, 100, (b, t)).astype(np.int32)
        parents = np.stack([random_tree(rng, t, "any") for _ in range(b)]).astype(np.int32)
        given = (q.reshape(b, t, -1), k.reshape(b, t, -1), v.reshape(b, t, -1), table, lengths, counts, positions, cos, sin, qw, kw, parents)
        (y,) = runner.run([CPUTensor.from_array(a) for a in given])
        turned = [rotated(x, w, cos[positions], sin[positions], 1e-6, False) for x, w in ((q, qw), (k, kw))]
        reference_append(codes, scales, turned[1].astype(f32), v, table, lengths, counts, size)
        want, room = reference_tree(turned[0], codes, scales, table, lengths, counts, size, c ** -0.5, parents)
        # (queries are 2^-20 off, twice that in a score's weight: as much again as the attention's own)
        assert np.abs(y.numpy().reshape(q.shape) - want).max() <= 2 * room
    assert np.array_equal(pool_codes(cache)[1], codes) and np.array_equal(pool_scales(cache)[1], scales)
    assert not runner.nodes_on("cpu") and bool(runner.graph_replays) == replay
    runner.dispose()


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_node_run_after_run(cuda_context, with_draft):
    rng = np.random.default_rng(3)
    batch, n, vocab = 5, 6, 300
    names = ["logits", "tokens", "parents", "counts", "uniforms"] + (["draft"] if with_draft else [])
    dims = [[batch, n, vocab], [batch, n], [batch, n], [batch], [batch, n], [batch, n, vocab]]
    kinds = [FLOAT, INT32, INT32, INT32, FLOAT, FLOAT]
    node = make_node("CudaVerifyDrafts", names, ["path", "accepted", "next"], extras="parents,counts,uniforms" + (",draft_logits" if with_draft else ""),
                     temperature=0.75)
    model = model_of(node, list(zip(names, kinds, dims)), [("path", INT32), ("accepted", INT32), ("next", INT32)])
    runner = load(model, backend_order=["cuda", "cpu"], backend_options={"cuda": {"context": cuda_context}})
    for step in range(5):
        logits, draft, parents, tokens, uniforms = drafted(rng, batch, n, vocab, "any", with_draft)
        counts = rng.integers(0, n + 1, batch).astype(np.int32)
        given = [logits, tokens, parents, counts, uniforms] + ([draft] if with_draft else [])
        got = [t.numpy().copy() for t in runner.run([CPUTensor.from_array(a) for a in given])]
        assert_verdicts(got, logits, tokens, parents, counts, uniforms, draft, 0.75)
    runner.dispose()


# -------------------------------------------------------------------------------------------------- captured
def test_a_captured_step_repeats_with_new_inputs(cuda_context):
    """Rotation, append, attention of the tree and the verdict in one captured graph, two of them in turn, with results of their own."""
    ctx, rng = cuda_context, np.random.default_rng(4)
    b, t, heads, kv, c, size, vocab = 2, 20, 32, 8, 128, 64, 4099
    cache = PagedCache(ctx, 1, 30, kv, c, size)
    random_pool(rng, cache)
    lengths, counts = [700, 333], [20, 13]
    table = tables(rng, cache, lengths)
    cos, sin = tables_of(800, c // 2)
    fixed = [dev(ctx, np.asarray(a, np.int32)) for a in (table, lengths, counts)]
    tc, ts = dev(ctx, cos), dev(ctx, sin)

    def inputs():
        logits, _, parents, tokens, uniforms = drafted(rng, b, t, vocab, "any", False)
        q, k, v = (rng.standard_normal((b, t, n * c)).astype(f32) for n in (heads, kv, kv))
        return dict(q=q, k=k, v=v, parents=parents, logits=logits, tokens=tokens, uniforms=uniforms)

    first = inputs()
    up = {n: dev(ctx, a) for n, a in first.items()}

    def step():
        q = cache.append_rotary(0, up["k"], up["v"], *fixed, cos=tc, sin=ts, q=up["q"])
        y = cache.attention(0, q, *fixed, parents=up["parents"])
        return q, y, *ctx.verify_drafts(up["logits"], up["tokens"], up["parents"], counts=fixed[2], uniforms=up["uniforms"])

    dispose(*step())                                     # (once normally first)
    graphs = []
    for _ in range(2):
        ctx.capture_begin()
        outs = step()
        graphs.append((ctx.capture_end(), outs))
    for round_ in range(4):
        new = inputs()
        for n, a in new.items():
            up[n].set_data(a)
        graph, outs = graphs[round_ % 2]
        ctx.graph_launch(graph)
        replayed = [o.get_data().copy() for o in outs]
        direct = step()
        for got, want in zip(replayed, direct):
            assert np.array_equal(got, want.get_data(), equal_nan=True)
        got = [o.get_data().reshape(o.dims) for o in direct[2:]]
        assert_verdicts(got, new["logits"], new["tokens"], new["parents"], counts, new["uniforms"], None, 1.0)
        dispose(*direct)
    for graph, outs in graphs:
        dispose(*outs)
        ctx.graph_destroy(graph)
    ctx.sync()
    dispose(tc, ts, *fixed, *up.values())
    cache.dispose()


# -------------------------------------------------------------------------------------------------- the loop
@pytest.mark.parametrize("rotary", [False, True])
def test_drafted_texts_are_the_decoders_own(cuda_context, rotary):
    """At temperature 0 every token is the likeliest behind the text so far, whatever was drafted, but for rounding to 8 bits: that differs
    with the way in which a text comes into the cache, and rounding every number at random by half a step moves a log probability
    by 0.2 (test_gpu_decode, whose 0.02 is a tenth of it); two of them by 0.4.  All pages come back."""
    rng = np.random.default_rng(6)
    shape = dict(vocab=300, d=128, heads=4, kv_heads=2, ffn=128, positions=256, top=4, pages=60, page_tokens=16)
    target = Decoder(cuda_context, layers=2, name=f"target {rotary}", rotary=rotary, **shape)
    draft = Decoder(cuda_context, layers=1, name=f"draft {rotary}", **shape)
    prompts = [rng.integers(0, 300, n).tolist() for n in (1, 30, 17)]
    for drafter, depth, width in ((draft, 3, 2), (target, 4, 3), (draft, 0, 1)):
        found = target.generate(prompts, 20, drafter, depth, width)
        assert target.cache.used_pages == 0 and draft.cache.used_pages == 0
        for prompt, text in zip(prompts, found):
            assert len(text) == 20
            s = target.cache.add_sequence()
            wanted = [(0, len(prompt) - 1 + i) for i in range(20)]
            logprob, _, _, best = target.step([s], [prompt + text[:-1]], wanted, text)
            assert (logprob >= best[:, 0] - 0.4).all()
            target.cache.release(s)
    # with random numbers: the same ones give the same texts, others others
    texts = [target.generate(prompts, 12, draft, 3, 2, temperature=1.0, seed=seed) for seed in (1, 1, 2)]
    assert texts[0] == texts[1] != texts[2] and all(0 <= x < 300 for t in texts[0] for x in t)
    target.close()
    draft.close()


def test_drafts_of_the_decoder_itself_stand(cuda_context):
    """A decoder's own likeliest tokens are what it says at temperature 0, so whole chains stand: as many steps as a chain makes of a text."""
    shape = dict(vocab=300, d=128, heads=4, kv_heads=2, ffn=128, positions=256, top=4, pages=60, page_tokens=16, layers=2)
    target = Decoder(cuda_context, name="its own", rotary=True, **shape)
    steps = []
    decide = target.decide
    target.decide = lambda *a: steps.append(decide(*a)) or steps[-1]
    (text,) = target.generate([[5, 6, 7]], 40, target, depth=4, width=1)
    assert len(text) == 40 and len(steps) <= 40 // 5 + 4         # (8, were there no rounding to 8 bits)
    target.close()


# -------------------------------------------------------------------------------------------------- refusals
def test_the_library_refuses_what_does_not_fit(cuda_context):
    ctx = cuda_context
    x = dev(ctx, np.zeros(4096, f32))
    p = x.ptr

    def refused(status, name, desc, *pointers):
        with pytest.raises(CudaBackendError) as e:
            ctx._call(name, byref(desc), *pointers)
        assert e.value.status == status

    def with_fields(kind, base, **other):
        return kind(*[other.get(n, v) for (n, _), v in zip(kind._fields_, base)])

    heads = (2, 2, 64, 64, 8, 128, 64, 128, 64, 1e-6, 0)
    D = lambda **other: with_fields(lib.RotateDesc, heads, **other)  # noqa: E731
    call = ("wdc_rotate_heads",)
    for bad in (dict(head_size=62), dict(head_size=260), dict(rotary=60)):
        refused(lib.WDC_ERR_UNSUPPORTED, *call, D(**bad), p, None, p, p, None, p)
    for bad in (dict(rows=-1), dict(heads=70000), dict(rotary=72), dict(places=0), dict(x_st=126), dict(y_sh=-4), dict(epsilon=-1.0), dict(epsilon=float("nan"))):
        refused(lib.WDC_ERR_INVALID, *call, D(**bad), p, None, p, p, None, p)
    for pointers in ((None, None, p, p, None, p), (p, None, None, p, None, p), (p, None, p, None, None, p), (p, None, p, p, None, None),
                     (p + 4, None, p, p, None, p), (p, p + 4, p, p, None, p), (p, None, p + 8, p, None, p), (p, None, p, p, p + 2, p)):
        refused(lib.WDC_ERR_INVALID, *call, D(), *pointers)
    ctx._call(*call, byref(D(rows=0)), None, None, None, None, None, None)

    append = lib.CacheAppendDesc(4, 1, 16, 32, 1, 1, 4, 32, 32, 32, 32, 32, 32)
    A = lambda **other: with_fields(lib.CacheAppendRotaryDesc, (append, 1, 32, 32, 32, 32, 32, 32, 32, 8, 1e-6, 0), **other)  # noqa: E731
    good = [p, p, p, None, None, p, p, None, p, p, p, p, None, p]
    refused(lib.WDC_ERR_UNSUPPORTED, "wdc_cache_append_rotary", A(rotary=12), *good)
    for bad in (dict(heads=-1), dict(rotary=40), dict(places=0), dict(q_st=30), dict(epsilon=-1.0),
                dict(append=lib.CacheAppendDesc(4, 0, 16, 32, 1, 1, 4, 32, 32, 32, 32, 32, 32))):
        refused(lib.WDC_ERR_INVALID, "wdc_cache_append_rotary", A(**bad), *good)
    for i in (0, 1, 2, 5, 6, 8, 9, 10, 11, 13):
        refused(lib.WDC_ERR_INVALID, "wdc_cache_append_rotary", A(), *[None if j == i else a for j, a in enumerate(good)])
    refused(lib.WDC_ERR_INVALID, "wdc_cache_append_rotary", A(), *[p + 4 if j == 0 else a for j, a in enumerate(good)])

    T = lambda **other: with_fields(lib.CacheAttentionDesc, (4, 1, 16, 32, 1, 2, 4, 1, 64, 32, 32, 64, 32, 32, 0.5), **other)  # noqa: E731
    refused(lib.WDC_ERR_UNSUPPORTED, "wdc_cache_attention_tree", T(tokens=1025), p, p, p, p, p, None, p, p)
    refused(lib.WDC_ERR_INVALID, "wdc_cache_attention_tree", T(), p, p, p, p, p, None, None, p)
    refused(lib.WDC_ERR_INVALID, "wdc_cache_attention_tree", T(), p, p, p, p, p, None, p + 2, p)

    V = lambda **other: with_fields(lib.VerifyDesc, (1, 2, 50, 100, 50, 100, 50, 1.0, 1.0), **other)  # noqa: E731
    for bad in (dict(batch=65536), dict(tokens=1025), dict(vocab=1 << 30)):
        refused(lib.WDC_ERR_UNSUPPORTED, "wdc_verify_drafts", V(**bad), p, None, p, None, None, p, p, p, p)
    for bad in (dict(batch=-1), dict(tokens=-1), dict(vocab=0), dict(logits_st=-1), dict(temperature=-1.0), dict(temperature=1e-7),
                dict(draft_temperature=float("inf"))):
        refused(lib.WDC_ERR_INVALID, "wdc_verify_drafts", V(**bad), p, None, p, None, None, p, p, p, p)
    good = [p, None, p, None, None, p, p, p, p]
    for i in (0, 2, 5, 6, 7, 8):
        refused(lib.WDC_ERR_INVALID, "wdc_verify_drafts", V(), *[None if j == i else a for j, a in enumerate(good)])
    refused(lib.WDC_ERR_INVALID, "wdc_verify_drafts", V(), p + 2, *good[1:])

    K = lambda **other: with_fields(lib.CacheKeepDesc, (1, 4, 1, 16, 32, 1, 2, 4), **other)  # noqa: E731
    refused(lib.WDC_ERR_UNSUPPORTED, "wdc_cache_keep_paths", K(page_tokens=48), p, p, p, p, None, p, p)
    for bad in (dict(layers=0), dict(pages=0), dict(batch=-1), dict(batch=70000)):
        refused(lib.WDC_ERR_INVALID, "wdc_cache_keep_paths", K(**bad), p, p, p, p, None, p, p)
    good = [p, p, p, p, None, p, p]
    for i in (0, 1, 2, 3, 5, 6):
        refused(lib.WDC_ERR_INVALID, "wdc_cache_keep_paths", K(), *[None if j == i else a for j, a in enumerate(good)])
    ctx.sync()
    x.dispose()


def test_a_tape_that_moves_paths_is_not_repeated(cuda_context):
    """Moving a path a second time would move what has been moved."""
    ctx = cuda_context
    cache = PagedCache(ctx, 1, 4, 1, 32, 16)
    ts = [dev(ctx, np.array(a, np.int32)) for a in ([[0, 1]], [8], [4], [[0, 2, -1, -1]], [2])]
    ctx.tape_begin(ts)
    cache.keep_paths(*ts)
    assert ctx.tape_end([]) is None
    ctx.sync()
    dispose(*ts)
    cache.dispose()


# -------------------------------------------------------------------------------------------------- what the cache holds behind a decision
@pytest.mark.parametrize("rotary", [False, True])
def test_what_stands_is_where_its_text_has_it(cuda_context, rotary):
    """Keys and values of the first layer, which only tokens and their places make, are those of the same text without drafts.  A number is
    rounded to its page's scale when it comes, when that grows with a tree, when it is moved, and when that makes it grow: four times half a
    step, and half of one in the other cache; S is the largest scale."""
    rng = np.random.default_rng(9)
    target = Decoder(cuda_context, vocab=300, d=128, heads=4, kv_heads=2, layers=2, ffn=128, positions=256, top=4, pages=200, page_tokens=16,
                     name=f"stands {rotary}", rotary=rotary)
    texts = [rng.integers(0, 300, n).tolist() for n in (12, 15, 16, 17, 31, 40)]
    mine = [target.cache.add_sequence() for _ in texts]
    target.step(mine, [t[:-1] for t in texts], [], [])
    moved = 0
    for step in range(3):
        # the likeliest four behind each text, the likeliest last, and the same again behind each of those
        trees, parents = [], []
        for t in texts:
            tree, above, level = [t[-1]], [-1], [(0, t)]
            for _ in range(2):
                probes = [target.cache.add_sequence() for _ in level]
                *_, best, _ = target.step(probes, [x for _, x in level], [(i, len(x) - 1) for i, (_, x) in enumerate(level)], [0] * len(level))
                for probe in probes:
                    target.cache.release(probe)
                following = []
                for (at, x), ids in zip(level, best):
                    for token in ids[::-1].tolist():
                        following.append((len(tree), x + [token]))
                        tree.append(token)
                        above.append(at)
                level = following
            trees.append(tree)
            parents.append(above)
        found = target.decide(mine, trees, parents, np.zeros((len(texts), len(trees[0]))), 0.0)
        for i, (path, token) in enumerate(found):
            moved += path != list(range(len(path)))
            texts[i] = texts[i] + [trees[i][j] for j in path[1:]] + [token]
    assert moved >= 9                                # (of 18)
    plain = [target.cache.add_sequence() for _ in texts]
    target.step(plain, [t[:-1] for t in texts], [], [])
    codes, scales = pool_codes(target.cache)[0].astype(np.float64), pool_scales(target.cache)[0].astype(np.float64)
    whole = codes * scales[..., None, None]
    for a, b, text in zip(mine, plain, texts):
        assert target.cache.length(a) == target.cache.length(b) == len(text) - 1
        rows = []
        for s in (a, b):
            pages = target.cache.sequence_pages(s)
            rows.append(whole[pages].transpose(1, 2, 0, 3, 4).reshape(2, 2, -1, 32)[:, :, :len(text) - 1])
        most = scales[target.cache.sequence_pages(a) + target.cache.sequence_pages(b)].max(0)[..., None, None]
        assert (np.abs(rows[0] - rows[1]) <= 2.5 * most + 1e-5 * np.abs(rows[1]).max()).all()
        # (and tokens that are elsewhere would not pass)
        assert (np.abs(rows[0][:, :, 1:] - rows[1][:, :, :-1]) > 2.5 * most).any((0, 1, 3)).all()
    for s in (*mine, *plain):
        target.cache.release(s)
    target.close()


def test_texts_are_drafted_up_to_the_last_place(cuda_context):
    target = Decoder(cuda_context, vocab=300, d=128, heads=4, kv_heads=2, layers=1, ffn=128, positions=64, top=4, pages=60, page_tokens=16, name="last place")
    prompts = [[1, 2, 3], list(range(40)), list(range(63))]
    found = [target.generate([p], 64 - len(p), target, depth=5, width=4, temperature=t)[0] for p in prompts for t in (0.0, 1.0)]
    assert [len(t) for t in found] == [61, 61, 24, 24, 1, 1] and all(0 <= x < 300 for t in found for x in t)
    assert target.cache.used_pages == 0
    target.close()
