"""The host side of the paged cache and of the decoder around it, without a GPU: which pages belong to which sequence, what is
copied when, and what is refused before a call reaches the device."""
import random

import numpy as np
import pytest

from webdnn_b200 import zoo
from webdnn_b200.backend import CudaTensor, WebDNNCPUContext, WebDNNCudaContext
from webdnn_b200.paged_cache import PagedCache


class FakeContext(WebDNNCudaContext):
    """Hands out addresses and writes down the calls."""

    def __init__(self):
        super().__init__(WebDNNCPUContext())
        self.calls, self.next = [], 1 << 20

    def _alloc(self, nbytes):
        self.next += (nbytes + 511) // 512 * 512
        return self.next

    def _free(self, ptr):
        pass

    def _call(self, name, *args):
        self.calls.append((name, args))

    def copies(self):
        """The (from, to) pairs of the page copies since the last call."""
        pairs = [p for name, a in self.calls if name == "wdc_cache_copy_pages" for p in zip(list(a[4]), list(a[5]))]
        self.calls.clear()
        return pairs


def make(pages=20, page_tokens=16):
    context = FakeContext()
    return context, PagedCache(context, 2, pages, 2, 32, page_tokens)


def test_sequences_take_the_lowest_pages_and_give_them_back():
    context, cache = make()
    a, b = cache.add_sequence(), cache.add_sequence()
    cache.extend({a: 17, b: 1})
    assert cache.sequence_pages(a) == [0, 1] and cache.sequence_pages(b) == [2] and cache.free_pages == 17
    cache.extend({b: 15})
    assert cache.sequence_pages(b) == [2] and cache.length(b) == 16
    cache.extend({b: 1, a: 0})
    assert cache.sequence_pages(b) == [2, 3] and cache.length(a) == 17
    cache.release(a)
    c = cache.add_sequence()
    cache.extend({c: 40})
    assert cache.sequence_pages(c) == [0, 1, 4]
    assert not context.copies()


def test_a_fork_shares_pages_until_one_writes():
    context, cache = make()
    a = cache.add_sequence()
    cache.extend({a: 20})
    b, c = cache.fork(a), cache.fork(a)
    assert cache.sequence_pages(b) == cache.sequence_pages(c) == [0, 1] and cache.used_pages == 2
    cache.extend({b: 1})
    assert context.copies() == [(1, 2)] and cache.sequence_pages(b) == [0, 2]
    cache.extend({a: 1, c: 2})                      # the last one that keeps the page writes to it where it is
    assert context.copies() == [(1, 3)] and cache.sequence_pages(a) == [0, 3] and cache.sequence_pages(c) == [0, 1]
    cache.release(a)
    cache.release(c)
    assert cache.used_pages == 2 and cache.sequence_pages(b) == [0, 2]
    d = cache.fork(b)
    cache.extend({d: 11})                           # 21 tokens: the shared page is filled up, so a copy of it is
    assert context.copies() == [(2, 1)] and cache.sequence_pages(d) == [0, 1]
    e = cache.fork(d)
    cache.extend({e: 1})                            # 32 tokens: a page of its own begins, nothing is copied
    assert context.copies() == [] and cache.sequence_pages(e) == [0, 1, 3]


def test_room_is_given_to_all_or_to_none():
    context, cache = make(pages=4)
    a = cache.add_sequence()
    cache.extend({a: 20})
    b = cache.fork(a)
    with pytest.raises(MemoryError):
        cache.extend({a: 1, b: 33})                 # one copy (the other keeps the page) and two pages more
    assert cache.length(a) == cache.length(b) == 20 and cache.free_pages == 2 and not context.copies()
    cache.extend({a: 1, b: 13})                     # one copy and one page
    assert cache.free_pages == 0 and cache.length(b) == 33
    with pytest.raises(MemoryError):
        cache.extend({a: 12})
    with pytest.raises(ValueError):
        cache.extend({a: -1})


def test_truncation_and_compaction():
    context, cache = make()
    seqs = [cache.add_sequence() for _ in range(4)]
    for s in seqs:
        cache.extend({s: 48})
    cache.truncate(seqs[3], 17)
    assert cache.sequence_pages(seqs[3]) == [9, 10] and cache.length(seqs[3]) == 17
    cache.truncate(seqs[3], 0)
    assert cache.sequence_pages(seqs[3]) == []
    cache.release(seqs[0])
    fork = cache.fork(seqs[2])
    assert cache.compact() == 3
    assert sorted(context.copies()) == [(6, 0), (7, 1), (8, 2)]
    assert cache.sequence_pages(seqs[2]) == cache.sequence_pages(fork) == [0, 1, 2]
    assert cache.sequence_pages(seqs[1]) == [3, 4, 5] and cache.free_pages == 14
    assert cache.compact() == 0 and not context.calls
    with pytest.raises(ValueError):
        cache.truncate(seqs[1], 49)


def test_any_history_keeps_pages_apart():
    """Sequences against a model that copies whole texts: the same contents, page by page, after whatever happened."""
    rng = random.Random(1)
    for _ in range(30):
        context, cache = make(pages=rng.randint(6, 40), page_tokens=16)
        memory = {}                                  # page -> tokens
        texts = {}
        for step in range(60):
            what = rng.random()
            if what < 0.15 or not texts:
                texts[cache.add_sequence()] = []
            elif what < 0.3:
                s = rng.choice(list(texts))
                texts[cache.fork(s)] = list(texts[s])
            elif what < 0.4:
                s = rng.choice(list(texts))
                cache.release(s)
                del texts[s]
            elif what < 0.5:
                cache.compact()
            elif what < 0.55:
                s = rng.choice(list(texts))
                n = rng.randint(0, len(texts[s]))
                cache.truncate(s, n)
                del texts[s][n:]
            else:
                which = {s: rng.randint(0, 20) for s in rng.sample(list(texts), rng.randint(1, len(texts)))}
                try:
                    cache.extend(which)
                except MemoryError:
                    which = {}
                for a, b in context.copies():
                    memory[b] = list(memory.get(a, []))
                for s, n in which.items():
                    for i in range(n):
                        at = len(texts[s])
                        page = cache.sequence_pages(s)[at // 16]
                        tokens = memory.setdefault(page, [])
                        tokens[at % 16:] = [(s, step, i)]
                        texts[s].append((s, step, i))
            for a, b in context.copies():
                memory[b] = list(memory.get(a, []))
            used = set()
            for s, text in texts.items():
                pages = cache.sequence_pages(s)
                used |= set(pages)
                assert cache.length(s) == len(text) and len(pages) == -(-len(text) // 16)
                for at, token in enumerate(text):
                    assert memory[pages[at // 16]][at % 16] == token
            assert cache.used_pages == len(used)


def test_batch_gives_tables_of_a_fixed_width():
    context, cache = make()
    a, b = cache.add_sequence(), cache.add_sequence()
    cache.extend({a: 33, b: 2})
    table, lengths, counts = (t.numpy() for t in cache.batch([b, a], [2, 1], 5))
    assert table.tolist() == [[3, -1, -1, -1, -1], [0, 1, 2, -1, -1]] and table.dtype == np.int32
    assert lengths.tolist() == [2, 33] and counts.tolist() == [2, 1]
    assert cache.batch([b], [2])[0].dims == [1, 1] and cache.batch([], [])[0].dims == [0, 1]
    with pytest.raises(ValueError):
        cache.batch([a], [1], 2)
    with pytest.raises(ValueError):
        cache.batch([a], [])


def test_calls_reach_the_library_with_the_layers_addresses():
    context, cache = make()
    x = context.empty_tensor([3, 5, 160])
    table, lengths = context.empty_tensor([3, 4], "int32"), context.empty_tensor([3], "int32")
    cache.append(1, x, x, table, lengths, k_column=64, v_column=96)
    name, args = context.calls.pop()
    d = args[0]._obj
    assert name == "wdc_cache_append" and (d.batch, d.tokens, d.table_pages, d.k_sb, d.k_sh, d.k_st) == (3, 5, 4, 800, 32, 160)
    assert args[1:5] == (x.ptr + 256, x.ptr + 384, cache.codes.ptr + 20 * 2 * 2 * 16 * 32, cache.scales.ptr + 20 * 2 * 2 * 4)
    assert args[-1] is None
    y = cache.attention(0, x, table, lengths, lengths, heads=4, q_column=32)
    name, args = context.calls.pop()
    d = args[0]._obj
    assert (d.heads, d.q_st, d.y_sb, d.y_sh, d.y_st) == (4, 160, 640, 32, 128) and abs(d.scale - 32 ** -0.5) < 1e-7
    assert args[1] == x.ptr + 128 and args[-1] == y.ptr and y.dims == [3, 5, 128]
    cache.copy_pages(np.array([1, 2]), [3, 4])
    assert context.copies() == [(1, 3), (2, 4)]


def test_refusals():
    context, cache = make()
    x = context.empty_tensor([3, 5, 160])
    table, lengths = context.empty_tensor([3, 4], "int32"), context.empty_tensor([3], "int32")
    other = FakeContext().empty_tensor([3, 5, 160])
    flat, two = context.empty_tensor([15, 160]), context.empty_tensor([2, 4], "int32")
    for bad in ((x, x, two, lengths), (x, x, table, two), (flat, x, table, lengths), (x, flat, table, lengths),
                (x, context.empty_tensor([3, 4, 160]), table, lengths), (x, x, table, lengths, two)):
        with pytest.raises(ValueError):
            cache.append(0, *bad)
    for bad in ((other, x, table, lengths), (x, table, table, lengths), (x, x, x, lengths), (x, x, table, flat),
                (np.zeros(3), x, table, lengths)):
        with pytest.raises((TypeError, AttributeError)):
            cache.append(0, *bad)
    for kw in (dict(k_column=100), dict(v_column=-4), dict(k_column=2)):
        with pytest.raises(ValueError):
            cache.append(0, x, x, table, lengths, **kw)
    for kw in (dict(heads=3), dict(heads=6), dict(q_column=34), dict(heads=4, q_column=64), dict(heads=0)):
        with pytest.raises(ValueError):
            cache.attention(0, x, table, lengths, **kw)
    for layer in (-1, 2):
        with pytest.raises(ValueError):
            cache.append(layer, x, x, table, lengths)
        with pytest.raises(ValueError):
            cache.attention(layer, x, table, lengths, heads=4)
    with pytest.raises(ValueError):
        cache.attention(0, x, table, lengths, heads=4, out=context.empty_tensor([3, 5, 160]))
    for pair in (([0], [20]), ([-1], [0]), ([0, 1], [2]), ([2 ** 32], [1])):
        with pytest.raises(ValueError):
            cache.copy_pages(*pair)
    for shape in (dict(page_tokens=24), dict(head_size=48), dict(pages=0), dict(layers=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            PagedCache(context, **{**dict(layers=1, pages=1, kv_heads=1, head_size=32, page_tokens=16), **shape})
    with pytest.raises(ValueError):
        PagedCache(context, 1, 4, 1, 32, 16, codes=context.empty_tensor([1, 4, 2, 1, 16, 32], "int32"))
    assert not context.calls


def test_borrowed_memory_is_left_to_its_owner():
    context = FakeContext()
    owner = object()
    t = context.borrow_tensor(1 << 16, [4, 8], "int32", owner)
    alias = t.alias([32])
    assert isinstance(t, CudaTensor) and t.ptr == alias.ptr == 1 << 16 and t.shared_buffer.owner is owner
    t.dispose()
    assert alias.shared_buffer.owner is owner
    alias.dispose()
    assert alias.shared_buffer.owner is None
    for address, dims in ((8, [1]), (0, [3]), (16, [-1])):
        with pytest.raises(ValueError):
            context.borrow_tensor(address, dims)


def test_caches_of_a_context_have_names_of_their_own():
    context, cache = make()
    context.add_cache("layers", cache)
    with pytest.raises(ValueError):
        context.add_cache("layers", PagedCache(context, 1, 1, 1, 32, 16))
    with pytest.raises(ValueError):
        FakeContext().add_cache("layers", cache)
    with pytest.raises(RuntimeError):
        cache.dispose()


def test_the_decoder_graph_keeps_its_operators():
    """The load-time rewrite leaves the cache's nodes alone and fuses what is around them."""
    from webdnn_b200 import onnx_io
    from webdnn_b200.model_transform import model_transform
    model = onnx_io.decode_model(onnx_io.encode_model(zoo.decoder(50, 64, 2, 1, 2, 64, 128, 4)))
    model_transform(model, ["cuda", "cpu"])
    types = [n.op_type for n in model.graph.node]
    assert types.count("CudaCacheAttention") == 2 and types.count("CudaTokenLogProbs") == 1
    assert types.count("CudaLayerNorm") == 4 and "ReduceMean" not in types


def test_a_copy_that_fails_gives_no_room():
    context, cache = make()
    a = cache.add_sequence()
    cache.extend({a: 20})
    b, c = cache.fork(a), cache.fork(a)
    state = lambda: ([cache.sequence_pages(s) for s in (a, b, c)], [cache.length(s) for s in (a, b, c)], sorted(cache._free), cache._users[:])  # noqa: E731
    before = state()

    def fails(name, *args):
        raise RuntimeError(name)

    context._call, call = fails, context._call
    with pytest.raises(RuntimeError, match="copy_pages"):
        cache.extend({a: 1, b: 30, c: 0})
    assert state() == before
    context._call = call
    cache.extend({a: 1, b: 30, c: 0})
    assert cache.sequence_pages(c) == [0, 1] and context.copies() == [(1, 2), (1, 3)]
    assert cache.sequence_pages(a) == [0, 2] and cache.sequence_pages(b) == [0, 3, 4, 5] and cache.used_pages == 6


def test_results_are_row_major():
    """A result in another order of memory would be read as something else."""
    context, cache = make()
    logits, tokens = context.empty_tensor([2, 3, 4, 5, 9]), context.empty_tensor([2, 3, 4, 5], "int32")
    good = [context.empty_tensor([2, 3, 4, 5]), context.empty_tensor([2, 3, 4, 5]), None, None]
    context.token_logprobs(logits, tokens, out=good)
    for i in (0, 1):
        out = list(good)
        out[i] = context.empty_tensor([2, 3, 4, 5], layout="nhwc")
        with pytest.raises(ValueError):
            context.token_logprobs(logits, tokens, out=out)
    assert [name for name, _ in context.calls] == ["wdc_token_logprobs"]
