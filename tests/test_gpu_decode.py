"""The decoder's operators as nodes of a graph, and the loop around them: run after run (node by node, from a tape, from a replayed
graph) with new inputs, against the definitions in numpy.

A whole decoder is compared with the same layers in 64 bits whose keys and values go through the same 8-bit rounding.  Numbers that
differ by 1e-6 before that rounding may end one code apart now and then, a step of 1/127 of the page's largest number; the tolerance
of 0.02 on log probabilities is a tenth of what rounding every number at random by half a step does to them.
"""
import numpy as np
import pytest

from test_gpu_paged_cache import pool_codes, pool_scales, reference_append, reference_attention, tables
from webdnn_b200 import onnx_io
from webdnn_b200.backend import CPUTensor
from webdnn_b200.decode import Decoder
from webdnn_b200.onnx_io import FLOAT, INT32, Graph, Model, ValueInfo, make_node
from webdnn_b200.paged_cache import PagedCache
from webdnn_b200.runner import load

pytestmark = pytest.mark.gpu
f32 = np.float32


def model_of(node, inputs, outputs):
    g = Graph("g", [node], [], [ValueInfo(n, k, d) for n, k, d in inputs], [ValueInfo(n, k, []) for n, k in outputs])
    return Model(g, opset_import=[("", 13)])


@pytest.mark.parametrize("replay", ["auto", False])
def test_cache_attention_node_run_after_run(cuda_context, replay):
    ctx = cuda_context
    rng = np.random.default_rng(1)
    b, t, heads, kv, c, size = 3, 4, 4, 2, 32, 16
    cache = PagedCache(ctx, 2, 40, kv, c, size)
    name = f"nodes {replay}"
    ctx.add_cache(name, cache)
    codes, scales = np.zeros((40, 2, kv, size, c), np.int8), np.zeros((40, 2, kv), f32)
    cache.codes.set_data(np.zeros(cache.codes.dims, np.int32))
    cache.scales.set_data(np.zeros(cache.scales.dims, f32))
    ints = [("table", INT32, [b, 6]), ("lengths", INT32, [b]), ("counts", INT32, [b])]
    node = make_node("CudaCacheAttention", ["q", "k", "v", "table", "lengths", "counts"], ["y"], cache=name, layer=1, scale=0.25)
    model = model_of(node, [("q", FLOAT, [b, t, heads * c]), ("k", FLOAT, [b, t, kv * c]), ("v", FLOAT, [b, t, kv * c])] + ints,
                     [("y", FLOAT)])
    runner = load(model, backend_order=["cuda", "cpu"], backend_options={"cuda": {"context": ctx, "graphReplay": replay}})
    lengths = np.zeros(b, np.int32)
    table = tables(rng, cache, [96] * b, 0)
    for step in range(7):
        counts = rng.integers(0, t + 1, b).astype(np.int32)
        lengths = lengths + counts
        q, k, v = (rng.standard_normal((b, t, n, c)).astype(f32) for n in (heads, kv, kv))
        (y,) = runner.run([CPUTensor.from_array(a) for a in (q.reshape(b, t, -1), k.reshape(b, t, -1), v.reshape(b, t, -1), table,
                                                             lengths, counts)])
        reference_append(codes, scales, k, v, table, lengths, counts, size)
        want, tol = reference_attention(q, codes, scales, table, lengths, counts, size, 0.25)
        assert np.abs(y.numpy().reshape(q.shape) - want).max() <= tol
    assert np.array_equal(pool_codes(cache)[1], codes) and np.array_equal(pool_scales(cache)[1], scales)
    assert not pool_codes(cache)[0].any()
    assert not runner.nodes_on("cpu")
    if replay == "auto":
        assert runner.graph_replays > 0
    runner.dispose()


def test_cache_attention_node_refuses_unknown_caches_and_wrong_inputs(cuda_context):
    inputs = [("q", FLOAT, [1, 1, 32]), ("k", FLOAT, [1, 1, 32]), ("v", FLOAT, [1, 1, 32]), ("t", INT32, [1, 1]), ("l", INT32, [1])]
    data = [np.zeros((1, 1, 32), f32)] * 3 + [np.zeros((1, 1), np.int32), np.ones(1, np.int32)]
    for names, match in ((["q", "k", "v", "t", "l"], "no cache"), (["q", "k", "v", "t"], "inputs are")):
        model = model_of(make_node("CudaCacheAttention", names, ["y"], cache="nobody's"), inputs, [("y", FLOAT)])
        runner = load(model, backend_order=["cuda", "cpu"], backend_options={"cuda": {"context": cuda_context}})
        with pytest.raises(Exception, match=match):
            runner.run([CPUTensor.from_array(a) for a in data])
        runner.dispose()


@pytest.mark.parametrize("with_tokens,top", [(True, 5), (True, 0), (False, 3), (False, 0)])
def test_token_logprobs_node(cuda_context, with_tokens, top):
    rng = np.random.default_rng(2)
    outs = (["logprob"] if with_tokens else []) + ["entropy"] + (["ids", "best"] if top else [])
    node = make_node("CudaTokenLogProbs", ["x", "t"][:1 + with_tokens], outs, top=top)
    model = model_of(node, [("x", FLOAT, [2, 3, 77])] + ([("t", INT32, [2, 3])] if with_tokens else []),
                     [(o, INT32 if o == "ids" else FLOAT) for o in outs])
    runner = load(model, backend_order=["cuda", "cpu"], backend_options={"cuda": {"context": cuda_context}})
    for _ in range(4):
        x, t = rng.standard_normal((2, 3, 77)).astype(f32), rng.integers(0, 77, (2, 3)).astype(np.int32)
        got = dict(zip(outs, (o.numpy() for o in runner.run([CPUTensor.from_array(a) for a in (x, t)[:1 + with_tokens]]))))
        x = x.astype(np.float64)
        logs = x - np.log(np.exp(x).sum(-1, keepdims=True))
        np.testing.assert_allclose(got["entropy"], -(np.exp(logs) * logs).sum(-1), rtol=1e-6)
        if with_tokens:
            np.testing.assert_allclose(got["logprob"], np.take_along_axis(logs, t[..., None], -1)[..., 0], rtol=1e-6)
        if top:
            ids = np.argsort(-x, -1, kind="stable")[..., :top]
            assert got["ids"].dtype == np.int32 and np.array_equal(got["ids"], ids)
            np.testing.assert_allclose(got["best"], np.take_along_axis(logs, ids, -1), rtol=1e-6)
    runner.dispose()


SHAPE = dict(vocab=300, d=128, heads=4, kv_heads=2, layers=2, ffn=256, positions=256, top=6)


class Reference:
    """zoo.decoder in 64 bits, keys and values through the cache's 8 bits; one text at a time, a list of new tokens a step."""

    def __init__(self, model, page_tokens):
        self.w = {t.name: np.asarray(t.array, np.float64) for t in model.graph.initializer if t.data_type == FLOAT}
        self.names = [t.name for t in model.graph.initializer if t.name.split("_")[0] in ("w", "b", "ln")]
        self.size, pages = page_tokens, -(-SHAPE["positions"] // page_tokens)
        c = SHAPE["d"] // SHAPE["heads"]
        self.codes = [np.zeros((pages, 2, SHAPE["kv_heads"], page_tokens, c), np.int8) for _ in range(SHAPE["layers"])]
        self.scales = [np.zeros((pages, 2, SHAPE["kv_heads"]), f32) for _ in range(SHAPE["layers"])]
        self.length, self.table = 0, [list(range(pages))]

    def step(self, tokens):
        """Log probabilities [tokens, vocab] behind each new token."""
        names = [n for n in self.names if not n.startswith("ln_eps")]
        take = iter(names)

        def linear(x):
            return x @ self.w[next(take)] + self.w[next(take)]

        def norm(x):
            g, b = self.w[next(take)], self.w[next(take)]
            x = x - x.mean(-1, keepdims=True)
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * g + b

        n, self.length = len(tokens), self.length + len(tokens)
        c = SHAPE["d"] // SHAPE["heads"]
        h = self.w["embedding"][tokens] + self.w["place_embedding"][self.length - n:self.length]
        for codes, scales in zip(self.codes, self.scales):
            q, k, v = (linear(h).reshape(1, n, -1, c) for _ in range(3))
            reference_append(codes, scales, k.astype(f32), v.astype(f32), self.table, [self.length], [n], self.size)
            a, _ = reference_attention(q, codes, scales, self.table, [self.length], [n], self.size, c ** -0.5)
            h = norm(h + linear(a.reshape(n, -1)))
            h = norm(h + linear(np.maximum(linear(h), 0)))
        logits = linear(h)
        logits -= logits.max(-1, keepdims=True)
        return logits - np.log(np.exp(logits).sum(-1, keepdims=True))


@pytest.fixture(scope="module")
def decoder(cuda_context):
    d = Decoder(cuda_context, pages=64, page_tokens=16, name="decoder", **SHAPE)
    yield d
    d.close()


def reference_of(decoder):
    from webdnn_b200 import zoo
    return Reference(zoo.decoder(cache="decoder", **SHAPE), 16)


def test_scores_of_texts(decoder):
    rng = np.random.default_rng(3)
    texts = [rng.integers(0, SHAPE["vocab"], n).tolist() for n in (40, 2, 17, 120)]
    got = decoder.score(texts)
    for text, logs in zip(texts, got):
        want = reference_of(decoder).step(text)
        np.testing.assert_allclose(logs, want[np.arange(len(text) - 1), text[1:]], atol=0.02)
    assert decoder.cache.used_pages == 0


def test_steps_of_uneven_sequences(decoder):
    """Sequences of several lengths in one call, some with a prompt and some with a token, again and again."""
    rng = np.random.default_rng(4)
    sequences = [decoder.cache.add_sequence() for _ in range(3)]
    references = [reference_of(decoder) for _ in sequences]
    for lengths in ((5, 30, 1), (1, 1, 1), (1, 1, 1), (1, 1, 1), (3, 1, 20), (1, 1, 1)):
        new = [rng.integers(0, SHAPE["vocab"], n).tolist() for n in lengths]
        targets = rng.integers(0, SHAPE["vocab"], 3)
        logprob, entropy, ids, best = decoder.step(sequences, new, [(i, n - 1) for i, n in enumerate(lengths)], targets)
        for i, reference in enumerate(references):
            logs = reference.step(new[i])[-1]
            np.testing.assert_allclose(logprob[i], logs[targets[i]], atol=0.02)
            np.testing.assert_allclose(entropy[i], -(np.exp(logs) * logs).sum(), atol=0.02)
            np.testing.assert_allclose(best[i], logs[ids[i]], atol=0.02)
            np.testing.assert_allclose(best[i], np.sort(logs)[::-1][:6], atol=0.02)
    for s in sequences:
        decoder.cache.release(s)


def test_beam_search(decoder):
    """Every continuation has the log probability that the reference gives it, no two are alike, the first is as good as the
    greedy one, and all pages come back."""
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, SHAPE["vocab"], 37).tolist()
    found = decoder.beam_search(prompt, 9, beams=5)
    assert decoder.cache.used_pages == 0 and len(found) == 5
    assert len({tuple(t) for _, t in found}) == 5 and [s for s, _ in found] == sorted((s for s, _ in found), reverse=True)
    for score, tokens in found:
        reference = reference_of(decoder)
        logs = reference.step(prompt)[-1]
        total = 0.0
        for token in tokens:
            total += logs[token]
            logs = reference.step([token])[-1]
        assert abs(total - score) <= 0.02 * len(tokens)
    ((greedy, _),) = decoder.beam_search(prompt, 9, beams=1)
    assert found[0][0] >= greedy - 0.02 * 9


def test_steps_that_want_nothing_and_texts_without_scores(decoder):
    """A prompt may be appended without asking for anything; the next step sees it."""
    rng = np.random.default_rng(6)
    cache, reference = decoder.cache, reference_of(decoder)
    a = cache.add_sequence()
    prompt = rng.integers(0, SHAPE["vocab"], 21).tolist()
    for _ in range(3):                               # (node by node, recorded, replayed)
        got = decoder.step([a], [prompt], [], [])
        assert [o.shape for o in got] == [(0,), (0,), (0, 6), (0, 6)]
    logs = [reference.step(t)[-1] for t in (prompt, prompt, prompt, [7])][-1]
    logprob, *_ = decoder.step([a], [[7]], [(0, 0)], [5])
    np.testing.assert_allclose(logprob[0], logs[5], atol=0.02)
    cache.release(a)
    got = decoder.score([[], prompt, [3]])
    want = reference_of(decoder).step(prompt)
    assert [len(s) for s in got] == [0, 20, 0]
    np.testing.assert_allclose(got[1], want[np.arange(20), prompt[1:]], atol=0.02)
    assert cache.used_pages == 0
