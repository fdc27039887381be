"""Scoring and generation with a decoder graph over a paged 8-bit cache.

The loop around a graph such as ``zoo.decoder``: every step appends the new tokens of some sequences, attends and returns log
probabilities; between steps sequences fork, end and are compacted.  The reference has no counterpart (its runner executes
one graph on one set of inputs, ``core/runnerImpl.ts:315-596``).

    python -m webdnn_b200.decode        # a small decoder with random weights: scores a text, then searches with beams
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import numpy as np

from . import zoo
from .backend import CPUTensor, WebDNNCudaContext
from .paged_cache import PagedCache
from .runner import load


class Decoder:
    """A decoder with random weights (``zoo.decoder``) and its cache, which the context knows as ``name`` and keeps for its own life: a
    second decoder of one context needs another name."""

    def __init__(self, context: Optional[WebDNNCudaContext] = None, vocab: int = 1000, d: int = 256, heads: int = 8,
                 kv_heads: int = 2, layers: int = 4, ffn: int = 1024, positions: int = 4096, top: int = 8, pages: int = 512,
                 page_tokens: int = 32, name: str = "cache"):
        self.owns_context = context is None
        if context is None:
            context = WebDNNCudaContext()
            context.initialize()
        self.context, self.vocab, self.top, self.positions = context, vocab, top, positions
        self.cache = PagedCache(context, layers, pages, kv_heads, d // heads, page_tokens)
        context.add_cache(name, self.cache)
        self.table_pages = -(-positions // page_tokens)      # the same for every call, so that calls repeat
        self.runner = load(zoo.decoder(vocab, d, heads, kv_heads, layers, ffn, positions, top, name),
                           backend_order=["cuda", "cpu"], backend_options={"cuda": {"context": context}})

    def close(self) -> None:
        self.runner.dispose()
        if self.owns_context:
            self.context.close()

    def step(self, sequences: Sequence[int], new_tokens: Sequence[Sequence[int]], wanted: Sequence[Tuple[int, int]],
             targets: Sequence[int]):
        """Appends new_tokens[i] to sequences[i]; (logprob of targets[j], entropy, top ids, top logprobs) behind the new token
        wanted[j] = (which sequence of the call, which of its new tokens).  A step that fails leaves the sequences as long as they were."""
        counts = [len(t) for t in new_tokens]
        width = max(counts, default=0)
        # (two rows of one sequence would write to the same page at a time)
        if width == 0 or len(counts) != len(sequences) or len(set(sequences)) != len(sequences):
            raise ValueError("Decoder.step: some new tokens, one list for each of different sequences")
        if len(wanted) != len(targets) or not all(0 <= i < len(counts) and 0 <= j < counts[i] for i, j in wanted):
            raise ValueError("Decoder.step: one target for each wanted token, which is a new one")
        before = [self.cache.length(s) for s in sequences]
        ids, places = np.zeros((len(sequences), width), np.int32), np.zeros((len(sequences), width), np.int32)
        for i, (n, t) in enumerate(zip(before, new_tokens)):
            ids[i, :len(t)] = t
            places[i, :len(t)] = np.arange(n, n + len(t))
        # (Gather would take the first or the last)
        if places.max() >= self.positions:
            raise ValueError(f"Decoder.step: there are places for {self.positions} tokens")
        if ids.min() < 0 or ids.max() >= self.vocab:
            raise ValueError(f"Decoder.step: tokens are 0 .. {self.vocab - 1}")
        rows = np.array([i * width + j for i, j in wanted], np.int32)
        self.cache.extend(dict(zip(sequences, counts)))
        try:
            inputs = [CPUTensor.from_array(ids), CPUTensor.from_array(places),
                      *self.cache.batch(sequences, counts, self.table_pages),
                      CPUTensor.from_array(rows), CPUTensor.from_array(np.array(targets, np.int32))]
            return tuple(t.numpy().copy() for t in self.runner.run(inputs))
        except BaseException:
            for s, length in zip(sequences, before):         # (what was written behind that is written again)
                self.cache.truncate(s, length)
            raise

    def score(self, texts: Sequence[Sequence[int]]) -> List[np.ndarray]:
        """Log probability of every token of each text but its first, given those before it."""
        scored = [t for t in texts if len(t) > 1]
        if not scored:
            return [np.zeros(0, np.float32) for _ in texts]
        sequences = [self.cache.add_sequence() for _ in scored]
        wanted = [(i, j) for i, t in enumerate(scored) for j in range(len(t) - 1)]
        try:
            logprob = self.step(sequences, scored, wanted, [scored[i][j + 1] for i, j in wanted])[0]
        finally:
            for s in sequences:
                self.cache.release(s)
        ends = np.cumsum([max(len(t) - 1, 0) for t in texts])
        return np.split(logprob, ends[:-1])

    def beam_search(self, prompt: Sequence[int], new_tokens: int, beams: int = 4) -> List[Tuple[float, List[int]]]:
        """The ``beams`` continuations with the highest log probability that the search finds: (log probability, tokens), best
        first.  A beam that has several successors forks; one that has none gives its pages back."""
        if not len(prompt):
            raise ValueError("Decoder.beam_search: a prompt has a token")
        first = self.cache.add_sequence()
        held = {first}
        try:
            *_, ids, logs = self.step([first], [prompt], [(0, len(prompt) - 1)], [0])
            alive = [(0.0, [], first)]
            for step in range(new_tokens):
                found = sorted(((score + float(logs[i, j]), i, int(ids[i, j])) for i, (score, _, _) in enumerate(alive)
                                for j in range(self.top)), reverse=True)[:beams]
                heirs = {}
                following = []
                for score, i, token in found:
                    _, text, sequence = alive[i]
                    heirs[i] = heirs.get(i, 0) + 1
                    if heirs[i] > 1:
                        sequence = self.cache.fork(sequence)
                        held.add(sequence)
                    following.append((score, text + [token], sequence))
                for i, (_, _, sequence) in enumerate(alive):
                    if i not in heirs:
                        held.remove(sequence)
                        self.cache.release(sequence)
                alive = following
                if step + 1 < new_tokens:
                    n = len(alive)
                    *_, ids, logs = self.step([s for _, _, s in alive], [t[-1:] for _, t, _ in alive], [(i, 0) for i in range(n)],
                                              [0] * n)
        finally:
            for sequence in held:
                self.cache.release(sequence)
        return [(score, text) for score, text, _ in alive]


def main() -> None:
    decoder = Decoder()
    text = [int(t) for t in np.random.default_rng(0).integers(0, 1000, 200)]
    print("mean log probability of a text:", float(decoder.score([text])[0].mean()))
    for score, tokens in decoder.beam_search(text[:50], 12):
        print(f"{score:9.4f}", tokens)
    decoder.close()


if __name__ == "__main__":
    main()
