"""The loop around a decoder graph without a GPU: what a step hands to the graph, what it refuses, and that a step that fails, wherever it
fails, leaves the cache as it was."""
import numpy as np
import pytest

from test_paged_cache import FakeContext
from webdnn_b200 import decode

VOCAB, TOP, POSITIONS = 50, 3, 70


class FakeRunner:
    """Gives every wanted row the same alternatives, and raises in the call that it is told to."""

    def __init__(self):
        self.calls, self.fail_in = [], None

    def run(self, inputs):
        self.calls.append([t.numpy().copy() for t in inputs])
        if len(self.calls) == self.fail_in:
            raise RuntimeError("the graph failed")
        n = len(self.calls[-1][5])
        logs = np.log(np.arange(1, TOP + 1) / 6.0)[::-1]
        outs = np.zeros(n), np.zeros(n), np.tile(np.arange(TOP, dtype=np.int32), (n, 1)), np.tile(logs, (n, 1))
        return [FakeTensor(o) for o in outs]

    def dispose(self):
        pass


class FakeTensor:
    def __init__(self, array):
        self.array = array

    def numpy(self):
        return self.array


@pytest.fixture
def decoder(monkeypatch):
    monkeypatch.setattr(decode, "load", lambda *a, **kw: FakeRunner())
    return decode.Decoder(FakeContext(), vocab=VOCAB, d=64, heads=2, kv_heads=1, layers=1, ffn=64, positions=POSITIONS, top=TOP, pages=8,
                          page_tokens=16)


def nothing_is_held(decoder):
    return decoder.cache.used_pages == 0 and not decoder.cache._sequences


def test_a_step_gives_the_graph_ids_places_and_rows(decoder):
    a, b = decoder.cache.add_sequence(), decoder.cache.add_sequence()
    decoder.step([a], [[7, 8, 9]], [(0, 2)], [1])
    decoder.step([a, b], [[1], [4, 5]], [(0, 0), (1, 0), (1, 1)], [2, 3, 4])
    ids, places, table, lengths, counts, rows, targets = decoder.runner.calls[-1]
    assert ids.tolist() == [[1, 0], [4, 5]] and places.tolist() == [[3, 0], [0, 1]]
    assert table.shape == (2, 5) and lengths.tolist() == [4, 2] and counts.tolist() == [1, 2]
    assert rows.tolist() == [0, 2, 3] and targets.tolist() == [2, 3, 4]


def test_a_step_that_fails_leaves_the_sequences_as_long_as_they_were(decoder):
    cache = decoder.cache
    a = cache.add_sequence()
    decoder.step([a], [list(range(20))], [(0, 19)], [0])
    b = cache.fork(a)
    pages = cache.sequence_pages(a)
    decoder.runner.fail_in = 2
    with pytest.raises(RuntimeError, match="the graph failed"):
        decoder.step([a, b], [[1] * 20, [2]], [(0, 0), (1, 0)], [0, 0])
    assert cache.length(a) == cache.length(b) == 20 and cache.used_pages <= 3
    assert cache.sequence_pages(a)[0] == cache.sequence_pages(b)[0] == pages[0]
    rest = cache.add_sequence()
    cache.extend({rest: 16 * cache.free_pages})
    with pytest.raises(MemoryError):
        decoder.step([a], [[1] * 30], [(0, 0)], [0])
    assert cache.length(a) == 20
    cache.release(rest)
    cache.release(a)
    cache.release(b)
    assert nothing_is_held(decoder)


def test_scores_that_fail_give_their_pages_back(decoder):
    with pytest.raises(MemoryError):
        decoder.score([[1] * 60, [2] * 60, [3] * 60])
    assert nothing_is_held(decoder)
    with pytest.raises(ValueError):                  # more than the table has pages for
        decoder.score([[1] * 100])
    assert nothing_is_held(decoder)
    decoder.runner.fail_in = 1
    with pytest.raises(RuntimeError):
        decoder.score([[1, 2, 3]])
    assert nothing_is_held(decoder)
    assert [len(s) for s in decoder.score([[1, 2, 3], [4, 5]])] == [2, 1] and nothing_is_held(decoder)


@pytest.mark.parametrize("fail_in", [1, 2, 3, 5])
def test_a_search_that_fails_gives_its_pages_back(decoder, fail_in):
    decoder.runner.fail_in = fail_in
    with pytest.raises(RuntimeError):
        decoder.beam_search([1] * 20, 6, beams=3)
    assert nothing_is_held(decoder)


def test_a_search_that_fills_the_pool_gives_its_pages_back(decoder):
    with pytest.raises(MemoryError):
        decoder.beam_search([1] * 47, 20, beams=6)   # (three pages, and six copies of the last)
    assert nothing_is_held(decoder)
    found = decoder.beam_search([1] * 20, 6, beams=3)
    assert nothing_is_held(decoder) and len(found) == 3 and [len(t) for _, t in found] == [6] * 3


def test_texts_beyond_the_places_are_refused(decoder):
    """70 places in pages of 16: the table has room for 80 tokens."""
    cache = decoder.cache
    with pytest.raises(ValueError, match="places"):
        decoder.score([[1] * 71])
    with pytest.raises(ValueError, match="places"):
        decoder.beam_search([1] * 68, 4, beams=1)    # (three tokens are appended)
    assert nothing_is_held(decoder) and len(decoder.runner.calls) == 3
    decoder.beam_search([1] * 68, 3, beams=1)
    a = cache.add_sequence()
    decoder.step([a], [[1] * 70], [(0, 0)], [0])
    calls = len(decoder.runner.calls)
    with pytest.raises(ValueError, match="places"):
        decoder.step([a], [[1]], [(0, 0)], [0])
    assert cache.length(a) == 70 and len(decoder.runner.calls) == calls


def test_texts_without_a_second_token_have_no_scores(decoder):
    decoder.runner.run = lambda inputs, run=decoder.runner.run: [FakeTensor(np.arange(inputs[5].length))] + run(inputs)[1:]
    got = decoder.score([[], [1, 2, 3], [4], [5, 6], []])
    assert [s.tolist() for s in got] == [[], [0, 1], [], [2], []]
    assert decoder.runner.calls[0][4].tolist() == [3, 2]          # (the graph sees the others only)
    assert [s.tolist() for s in decoder.score([[7], []])] == [[], []] and decoder.score([]) == []
    assert len(decoder.runner.calls) == 1 and nothing_is_held(decoder)
    with pytest.raises(ValueError):
        decoder.beam_search([], 3)
    assert nothing_is_held(decoder)


def test_steps_that_do_not_fit_together_are_refused(decoder):
    cache = decoder.cache
    a, b = cache.add_sequence(), cache.add_sequence()
    good = [a, b], [[1, 2], [3]], [(0, 1), (1, 0)], [0, 0]
    for change in ({0: [a, a]}, {0: [a]}, {0: [], 1: [], 2: [], 3: []}, {1: [[1, 2]]}, {1: [[], []], 2: [], 3: []},  # one sequence twice ...
                   {1: [[1, VOCAB], [3]]}, {1: [[1, -1], [3]]},                    # (Gather would take the last token's embedding)
                   {2: [(0, 1)]}, {3: [0]}, {2: [(0, 2), (1, 0)]}, {2: [(0, 1), (1, 1)]}, {2: [(2, 0), (1, 0)]}, {2: [(0, -1), (1, 0)]}):
        with pytest.raises(ValueError):
            decoder.step(*[change.get(i, v) for i, v in enumerate(good)])
        assert cache.length(a) == cache.length(b) == cache.used_pages == 0 and not decoder.runner.calls, change
    decoder.step(*good)
    decoder.step([a, b], [[], [VOCAB - 1]], [], [])
    assert cache.length(a) == 2 and cache.length(b) == 2
