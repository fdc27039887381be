"""A decoder that drafts, without a GPU: what its operators refuse before a call reaches the device, and the loop that drafts, decides and
goes on, around graphs that are stood in for."""
import numpy as np
import pytest

from test_decode_loop import FakeTensor
from test_paged_cache import FakeContext, make
from webdnn_b200 import decode, zoo
from webdnn_b200.onnx_io import make_node
from webdnn_b200.operators import cuda as operators


def rows(context, batch=2, tokens=3):
    ints = lambda *dims: context.empty_tensor(list(dims), "int32")  # noqa: E731
    return ints(batch, 5), ints(batch), ints(batch), ints(batch, tokens)


# -------------------------------------------------------------------------------------------------- refusals
def test_heads_that_do_not_fit_are_refused():
    context, other = FakeContext(), FakeContext()
    t = context.empty_tensor
    x, cos, sin, weight, places = t([2, 3, 128]), t([50, 16]), t([50, 16]), t([64]), t([2, 3], "int32")
    y = context.rotate_heads(x, 2, 64, cos, sin, places, weight)
    assert y.dims == [2, 3, 128] and context.rotate_heads(x, 1, 64, column=64, weight=weight).dims == [2, 3, 64]
    assert context.rotate_heads(x, 2, 64, cos, sin, out=x) is x
    calls = len(context.calls)
    for bad in (dict(heads=0), dict(heads=3), dict(head_size=63), dict(head_size=260, heads=1), dict(column=2), dict(column=-4), dict(column=64),
                dict(cos=None), dict(sin=None), dict(cos=None, sin=None), dict(cos=t([50, 15]), sin=t([50, 15])), dict(cos=t([50, 36]), sin=t([50, 36])),
                dict(sin=t([49, 16])), dict(cos=t([0, 16]), sin=t([0, 16])), dict(weight=t([32])), dict(positions=t([5], "int32")),
                dict(out=t([2, 3, 64])), dict(out=t([2, 3, 128], "int32")), dict(out=other.empty_tensor([2, 3, 128])),
                dict(heads=1, column=64, out=x), dict(x=t([4, 6, 128]), positions=places)):
        with pytest.raises(ValueError):
            context.rotate_heads(**{**dict(x=x, heads=2, head_size=64, cos=cos, sin=sin, positions=places, weight=weight), **bad})
    for bad in (dict(x=t([2, 128], "int32")), dict(cos=t([50, 16], "int32")), dict(positions=t([2, 3])), dict(x=other.empty_tensor([2, 3, 128])),
                dict(weight=other.empty_tensor([64])), dict(x=t([2, 3, 4, 128], layout="nhwc"), positions=None)):
        with pytest.raises(TypeError):
            context.rotate_heads(**{**dict(x=x, heads=2, head_size=64, cos=cos, sin=sin, positions=places, weight=weight), **bad})
    assert len(context.calls) == calls
    assert context.rotate_heads(t([0, 128]), 2, 64, cos, sin).dims == [0, 128] and len(context.calls) == calls


def test_appends_of_rotated_keys_that_do_not_fit_are_refused():
    context, cache = make(page_tokens=16)                                        # 2 heads of 32
    t = context.empty_tensor
    table, lengths, counts, places = rows(context)
    good = dict(layer=0, k=t([2, 3, 64]), v=t([2, 3, 64]), page_table=table, lengths=lengths, counts=counts, cos=t([9, 16]), sin=t([9, 16]),
                positions=places, q=t([2, 3, 128]), q_weight=t([32]), k_weight=t([32]))
    assert cache.append_rotary(**good).dims == [2, 3, 128]
    assert cache.append_rotary(**{**good, "q": None, "q_weight": None}) is None
    assert cache.append_rotary(**{**good, "heads": 1, "q_column": 4}).dims == [2, 3, 32]
    calls = len(context.calls)
    for bad in (dict(layer=2), dict(k=t([2, 3, 60])), dict(v=t([2, 4, 64])), dict(positions=t([2, 4], "int32")), dict(q=t([2, 3, 30])), dict(q=t([6, 128])),
                dict(heads=5), dict(heads=0), dict(q_column=-4), dict(q_column=2), dict(k_column=4), dict(cos=None), dict(positions=None, cos=None),
                dict(cos=t([9, 20]), sin=t([9, 20])), dict(q_weight=t([64])), dict(k_weight=t([31])), dict(out=t([2, 3, 64])), dict(out=t([2, 3, 128], "int32")),
                dict(q=None, heads=2, q_weight=None), dict(q=None), dict(q=None, q_weight=None, out=t([2, 3, 128])), dict(lengths=t([3], "int32")),
                dict(heads=3, out=good["q"])):
        with pytest.raises(ValueError):
            cache.append_rotary(**{**good, **bad})
    for bad in (dict(q=t([2, 3, 128], "int32")), dict(counts=t([2])), dict(positions=t([2, 3])), dict(cos=FakeContext().empty_tensor([9, 16]))):
        with pytest.raises(TypeError):
            cache.append_rotary(**{**good, **bad})
    assert len(context.calls) == calls


def test_trees_and_paths_that_do_not_fit_are_refused():
    context, cache = make(page_tokens=16)
    t = context.empty_tensor
    table, lengths, counts, parents = rows(context)
    q = t([2, 3, 128])
    cache.attention(0, q, table, lengths, counts, parents=parents)
    cache.attention(0, q, table, lengths, counts)
    cache.keep_paths(table, lengths, counts, parents, lengths)
    cache.keep_paths(table, lengths, None, parents, lengths)
    assert [name for name, _ in context.calls] == ["wdc_cache_attention_tree", "wdc_cache_attention", "wdc_cache_keep_paths", "wdc_cache_keep_paths"]
    for bad in (t([2, 4], "int32"), t([3, 3], "int32"), t([6], "int32")):
        with pytest.raises(ValueError):
            cache.attention(0, q, table, lengths, counts, parents=bad)
    with pytest.raises(TypeError):
        cache.attention(0, q, table, lengths, counts, parents=t([2, 3]))
    for bad in (dict(path=t([6], "int32")), dict(path=t([3, 3], "int32")), dict(accepted=t([3], "int32")), dict(counts=t([1], "int32")),
                dict(page_table=t([2], "int32"))):
        with pytest.raises(ValueError):
            cache.keep_paths(**{**dict(page_table=table, lengths=lengths, counts=counts, path=parents, accepted=lengths), **bad})
    for bad in (dict(path=t([2, 3])), dict(accepted=t([2])), dict(lengths=t([2]))):
        with pytest.raises(TypeError):
            cache.keep_paths(**{**dict(page_table=table, lengths=lengths, counts=counts, path=parents, accepted=lengths), **bad})
    assert len(context.calls) == 4


def test_verdicts_that_do_not_fit_are_refused():
    context = FakeContext()
    t = context.empty_tensor
    ints = lambda *dims: t(list(dims), "int32")  # noqa: E731
    good = dict(logits=t([2, 3, 50]), tokens=ints(2, 3), parents=ints(2, 3), counts=ints(2), uniforms=t([2, 3]), draft_logits=t([2, 3, 60]), vocab=50)
    assert [o.dims for o in context.verify_drafts(**good)] == [[2, 3], [2], [2]]
    context.verify_drafts(t([2, 3, 50]), ints(2, 3), temperature=0)
    for bad in (dict(logits=t([6, 50])), dict(tokens=ints(2, 4)), dict(parents=ints(3, 3)), dict(counts=ints(3)), dict(uniforms=t([2, 4])), dict(uniforms=None),
                dict(draft_logits=t([2, 3, 49])), dict(draft_logits=t([2, 4, 50])), dict(draft_logits=t([6, 50])), dict(vocab=51), dict(vocab=0),
                dict(temperature=-1.0), dict(temperature=1e-9), dict(temperature=float("nan")), dict(draft_temperature=1e7),
                dict(temperature=0.0, uniforms=None), dict(out=(ints(2, 3), ints(2))), dict(out=(ints(2, 3), ints(2), ints(3)))):
        with pytest.raises(ValueError):
            context.verify_drafts(**{**good, **bad})
    for bad in (dict(logits=ints(2, 3, 50)), dict(tokens=t([2, 3])), dict(uniforms=ints(2, 3)), dict(out=(ints(2, 3), ints(2), t([2]))),
                dict(draft_logits=FakeContext().empty_tensor([2, 3, 50]))):
        with pytest.raises(TypeError):
            context.verify_drafts(**{**good, **bad})
    assert [name for name, _ in context.calls] == ["wdc_verify_drafts"] * 2


@pytest.mark.parametrize("kind,known", [(operators.CudaCacheAttention, "positions"), (operators.CudaRotateHeads, "weight"),
                                        (operators.CudaVerifyDrafts, "uniforms")])
def test_extras_of_a_node_are_known_and_there(kind, known):
    for extras in ("nobody", f"{known},{known}", f"{known},,nobody"):
        with pytest.raises(ValueError):
            kind().initialize(make_node("X", [], ["y"], extras=extras).attribute)
    op = kind()
    op.initialize(make_node("X", [], ["y"], extras=known, cache="c").attribute)
    context, cache = make()
    context.add_cache("c", cache)
    with pytest.raises(ValueError, match=known):
        op.run(context, [context.empty_tensor([2, 3, 64]) for _ in range(5)], 1)


def test_the_graph_that_decides_keeps_its_operators():
    from webdnn_b200 import onnx_io
    from webdnn_b200.model_transform import model_transform
    model = onnx_io.decode_model(onnx_io.encode_model(zoo.decoder(50, 64, 2, 1, 2, 64, 128, 4, rotary=True, drafts=True, temperature=0.5)))
    model_transform(model, ["cuda", "cpu"])
    types = [n.op_type for n in model.graph.node]
    assert types.count("CudaCacheAttention") == 2 and types.count("CudaVerifyDrafts") == 1 and types.count("CudaLayerNorm") == 4
    node = next(n for n in model.graph.node if n.op_type == "CudaVerifyDrafts")
    op = operators.CudaVerifyDrafts()
    op.initialize(node.attribute)
    assert op.temperature == op.draft_temperature == 0.5 and op.extras == ["parents", "counts", "uniforms"]


# -------------------------------------------------------------------------------------------------- the loop
VOCAB, TOP, POSITIONS = 50, 3, 70


def following(token):
    return (token * 7 + 3) % VOCAB


class Model:
    """Stands in for the graphs of a decoder that always says `following`; its drafts are that for tokens below `knows`, and something
    else for others.  Keeps what it was called with."""

    def __init__(self, drafts, knows):
        self.drafts, self.knows, self.calls, self.fail = drafts, knows, [], False

    def run(self, inputs):
        arrays = [t.numpy().copy() for t in inputs]
        self.calls.append(arrays)
        if self.fail:
            raise RuntimeError("the graph failed")
        if not self.drafts:
            ids, rows = arrays[0].reshape(-1), arrays[5]
            best = [[following(t) if t < self.knows else (following(t) + 1) % VOCAB, following(t), (t + 1) % VOCAB] for t in ids[rows]]
            n = len(rows)
            return [FakeTensor(a) for a in (np.zeros(n), np.zeros(n), np.array(best, np.int32).reshape(n, TOP), np.zeros((n, TOP)))]
        ids, places, _, lengths, counts, parents, _ = arrays
        path, accepted, after = np.full(ids.shape, -1, np.int32), [], []
        for b, n in enumerate(counts):
            at, walk = 0, [0]
            for i in range(1, n):
                assert places[b, i] == places[b, parents[b, i]] + 1
                if parents[b, i] == at and ids[b, i] == following(ids[b, at]):
                    at = i
                    walk.append(i)
            assert places[b, 0] == lengths[b] - n
            path[b, :len(walk)] = walk
            accepted.append(len(walk))
            after.append(following(ids[b, at]))
        return [FakeTensor(a) for a in (path, np.array(accepted, np.int32), np.array(after, np.int32))]

    def dispose(self):
        pass


class Context(FakeContext):
    """Moves host tensors to addresses, and keeps what they hold."""

    def move_tensor(self, tensor, option=None):
        t = self.empty_tensor(tensor.dims, tensor.data_type)
        self.moved = getattr(self, "moved", []) + [tensor.numpy().copy()]
        return t


def decoders(monkeypatch, knows, pages=12):
    made = []

    def load(model, **kw):
        made.append(Model(any(n.op_type == "CudaVerifyDrafts" for n in model.graph.node), knows))
        return made[-1]

    monkeypatch.setattr(decode, "load", load)
    context = Context()
    common = dict(vocab=VOCAB, d=64, heads=2, kv_heads=1, layers=1, ffn=64, positions=POSITIONS, top=TOP, pages=pages, page_tokens=16)
    return decode.Decoder(context, **common), decode.Decoder(context, **common, name="draft"), made


@pytest.mark.parametrize("knows", [0, 20, 50])
@pytest.mark.parametrize("depth,width", [(0, 1), (1, 1), (4, 1), (4, 2), (3, 3), (40, 2)])
def test_drafts_of_any_quality_give_the_same_texts(monkeypatch, knows, depth, width):
    target, draft, made = decoders(monkeypatch, knows)
    prompts = [[5], [1, 2, 3], list(range(20))]
    got = target.generate(prompts, 9, draft, depth, width)
    for prompt, text in zip(prompts, got):
        want = [prompt[-1]]
        for _ in range(9):
            want.append(following(want[-1]))
        assert text == want[1:]
    for decoder in (target, draft):
        assert decoder.cache.used_pages == 0 and not decoder.cache._sequences
    # good drafts are worth steps, and the draft is never shown a token that does not stand
    decisions = next(m for m in made if m.drafts).calls
    if knows == 50:
        assert len(decisions) <= -(-9 // (min(depth, 8) + 1)) + 1
    elif width > 1:                                  # (an alternative stands, and the token behind it)
        assert len(decisions) <= 5
    assert all(c[4].max() <= 1 + min(depth, 8) * width for c in decisions)


def test_kept_paths_are_moved_only_where_they_are_not_in_place(monkeypatch):
    target, draft, _ = decoders(monkeypatch, 0)
    s = target.cache.add_sequence()
    tree, parents = [4, 9, following(4), 1], [-1, 0, 0, 2]
    assert target.decide([s], [tree], [parents], np.zeros((1, 4))) == [([0, 2], following(following(4)))]
    assert target.cache.length(s) == 2 and target.context.calls[-1][0] == "wdc_cache_keep_paths"
    assert target.context.moved[-2].tolist() == [[0, 2, -1, -1]] and target.context.moved[-1].tolist() == [2]
    calls = len(target.context.calls)
    assert target.decide([s], [[4, following(4)]], [[-1, 0]], np.zeros((1, 2))) == [([0, 1], following(following(4)))]
    assert target.cache.length(s) == 4 and len(target.context.calls) == calls


def test_a_decision_that_fails_leaves_the_sequences_as_long_as_they_were(monkeypatch):
    target, draft, made = decoders(monkeypatch, 50)
    s = target.cache.add_sequence()
    target.decide([s], [[4]], [[-1]], np.zeros((1, 1)))
    held = target.cache.used_pages
    made[-1].fail = True
    with pytest.raises(RuntimeError):
        target.decide([s], [[4] * 30], [[-1] + [0] * 29], np.zeros((1, 30)))
    assert target.cache.length(s) == 1 and target.cache.used_pages == held
    target.cache.release(s)
    with pytest.raises(RuntimeError):
        target.generate([[5, 6]], 5, draft, temperature=1.0)
    for decoder in (target, draft):
        assert decoder.cache.used_pages == 0 and not decoder.cache._sequences


def test_temperatures_are_checked_and_few_graphs_are_kept(monkeypatch):
    target, draft, made = decoders(monkeypatch, 50)
    s = target.cache.add_sequence()
    disposed = []
    monkeypatch.setattr(Model, "dispose", lambda self: disposed.append(self))
    for bad in (-1.0, 1e-9, 1e7, float("nan")):
        with pytest.raises(ValueError):
            target.decide([s], [[4]], [[-1]], np.zeros((1, 1)), bad)
    assert len(made) == 2 and target.cache.length(s) == 0
    for temperature in (0.0, 0.5, 1.0, 0.5, 1.5, 0.5, 2.0, 0.0):
        target.decide([s], [[4]], [[-1]], np.zeros((1, 1)), temperature)
    # (0.5 was used again before a fifth came, 0 was not)
    assert len(made) == 2 + 6 and disposed == [made[2], made[4]] and list(target._deciding) == [1.5, 0.5, 2.0, 0.0]
    target.close()
    assert len(disposed) == 2 + 5


def test_trees_that_do_not_fit_together_are_refused(monkeypatch):
    target, draft, made = decoders(monkeypatch, 50)
    s, r = target.cache.add_sequence(), target.cache.add_sequence()
    u = lambda *shape: np.zeros(shape)  # noqa: E731
    for bad in (([s], [[]], [[]], u(1, 0)), ([s, s], [[1], [2]], [[-1], [-1]], u(2, 1)), ([s], [[1], [2]], [[-1], [-1]], u(2, 1)), ([s], [[1]], [], u(1, 1)),
                ([s], [[1, 2]], [[-1]], u(1, 2)), ([s], [[1, 2]], [[-1, -1]], u(1, 2)), ([s], [[1, 2]], [[-1, 1]], u(1, 2)), ([s], [[1, 2]], [[0, 0]], u(1, 2)),
                ([s], [[1]], [[-1]], u(1, 2)), ([s], [[1]], [[-1]], np.ones((1, 1))), ([s], [[1]], [[-1]], u(1, 1) - 1), ([s], [[1]], [[-1]], u(1, 1) * np.nan),
                ([s], [[VOCAB]], [[-1]], u(1, 1)), ([s], [[-1]], [[-1]], u(1, 1)), ([s], [[1] * 71], [list(range(-1, 70))], u(1, 71))):
        with pytest.raises(ValueError):
            target.decide(*bad)
    for bad in (dict(prompts=[[]]), dict(width=0), dict(width=TOP + 1), dict(depth=-1)):
        with pytest.raises(ValueError):
            target.generate(**{**dict(prompts=[[1]], new_tokens=2, draft=draft), **bad})
    assert target.cache.length(s) == 0 and target.generate([[1], [2]], 0, draft) == [[], []]
    # texts up to the last place
    assert [len(t) for t in target.generate([list(range(40))], 30, draft, depth=8)] == [30]
    with pytest.raises(ValueError):
        target.generate([list(range(40))], 32, draft, depth=8)
    target.cache.release(s)
    target.cache.release(r)
    assert target.cache.used_pages == 0 and draft.cache.used_pages == 0


@pytest.mark.parametrize("depth,width", [(8, 3), (30, 2), (2, 3)])
def test_trees_beside_the_last_places_have_room(monkeypatch, depth, width):
    """A tree has several tokens for a place: its pages may be more than those of a text that takes every place."""
    target, draft, made = decoders(monkeypatch, 50, pages=30)
    for prompt in (list(range(40)), list(range(49)) + [1] * 12, [3] * 69):
        (text,) = target.generate([prompt], 70 - len(prompt), draft, depth, width)
        want = [prompt[-1]]
        while len(want) <= 70 - len(prompt):
            want.append(following(want[-1]))
        assert text == want[1:]
    assert target.cache.used_pages == 0 and draft.cache.used_pages == 0
    # and the table of every other call is as wide as before
    s = target.cache.add_sequence()
    tree = [4] * 70, [-1] + [0] * 69
    assert target.decide([s], [tree[0]], [tree[1]], np.zeros((1, 70)))[0][0] == [0]
    assert made[-1].calls[-1][2].shape == (1, 5)
    for _ in range(60):
        target.decide([s], [[4]], [[-1]], np.zeros((1, 1)))
    assert target.decide([s], [tree[0]], [tree[1]], np.zeros((1, 70)))[0][0] == [0] and target.cache.length(s) == 62
    assert made[-1].calls[-1][2].shape == (1, 9)
    target.cache.release(s)


@pytest.mark.parametrize("temperature", [1e-6, 1e6, 0.0, float(np.float32(1e-6))])
def test_the_ends_of_temperatures_pass_through_a_graph(monkeypatch, temperature):
    """A graph has them as float32, and 1e-6 is a little less there."""
    from webdnn_b200 import onnx_io
    model = onnx_io.decode_model(onnx_io.encode_model(zoo.decoder(50, 64, 2, 1, 1, 64, 128, 4, drafts=True, temperature=temperature)))
    op = operators.CudaVerifyDrafts()
    op.initialize(next(n for n in model.graph.node if n.op_type == "CudaVerifyDrafts").attribute)
    context = FakeContext()
    ints = lambda *dims: context.empty_tensor(list(dims), "int32")  # noqa: E731
    given = [context.empty_tensor([2, 3, 50]), ints(2, 3), ints(2, 3), ints(2), context.empty_tensor([2, 3])]
    assert len(op.run(context, given, 3)) == 3
    op.temperature = op.draft_temperature = temperature
    assert len(op.run(context, given, 3)) == 3
    target, _, _ = decoders(monkeypatch, 50)
    assert target.decide([target.cache.add_sequence()], [[4]], [[-1]], np.zeros((1, 1)), temperature) == [([0], following(4))]
    for bad in (9.9e-7, 1.0001e6, 1e-50, 1e300, -1e-6, float("nan"), float("inf")):
        op.temperature = bad
        with pytest.raises(ValueError):
            op.run(context, given, 3)


@pytest.mark.parametrize("ids", [False, True])
@pytest.mark.parametrize("dims", [[0, 5, 128], [2, 0, 128], [0, 2, 5, 64], [2, 2, 0, 64], [2, 0, 5, 64]])
def test_rotary_embeddings_of_nothing_are_nothing(dims, ids):
    op = operators.CudaRotaryEmbedding()
    op.initialize(make_node("X", [], ["y"], num_heads=2).attribute)
    context = FakeContext()
    t = context.empty_tensor
    tokens = [dims[0], dims[2] if len(dims) == 4 else dims[1]]
    tables = [t([40, 32]), t([40, 32]), t(tokens, "int32")] if ids else [t([*tokens, 32]), t([*tokens, 32])]
    (y,) = op.run(context, [t(dims), *tables], 1)
    assert y.dims == dims and y.data_type == "float32" and not context.calls
    with pytest.raises(ValueError):
        op.run(context, [t(dims), t([40, 31]), *tables[1:]], 1)


def test_random_numbers_in_64_bits_are_all_below_1(monkeypatch):
    target, _, made = decoders(monkeypatch, 50)
    s = target.cache.add_sequence()
    given = np.array([[1 - 2.0 ** -25, np.nextafter(1.0, 0.0), 0.25]])
    target.decide([s], [[4, 1, 2]], [[-1, 0, 0]], given)
    assert made[-1].calls[-1][6].dtype == np.float32 and made[-1].calls[-1][6].tolist() == [[1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.25]]
    target.decide([s], [[4]], [[-1]], [[0]])
    for bad in (1.0, 1 + 1e-12, -1e-300, np.nan):
        with pytest.raises(ValueError):
            target.decide([s], [[4]], [[-1]], [[bad]])
    assert target.cache.length(s) == 2
