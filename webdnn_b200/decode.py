"""Scoring and generation with a decoder graph over a paged 8-bit cache.

The loop around a graph such as ``zoo.decoder``: every step appends the new tokens of some sequences, attends and returns log
probabilities; between steps sequences fork, end and are compacted.  Or a smaller decoder drafts trees of continuations, and a step
decides which of their tokens stand.  The reference has no counterpart (its runner executes one graph on one set of inputs,
``core/runnerImpl.ts:315-596``).

    python -m webdnn_b200.decode        # a small decoder with random weights: scores a text, searches with beams, has texts drafted
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from . import zoo
from .backend import CPUTensor, WebDNNCudaContext, is_temperature
from .paged_cache import PagedCache
from .runner import load


class Decoder:
    """A decoder with random weights (``zoo.decoder``) and its cache, which the context knows as ``name`` and keeps for its own life: a
    second decoder of one context needs another name."""

    def __init__(self, context: Optional[WebDNNCudaContext] = None, vocab: int = 1000, d: int = 256, heads: int = 8,
                 kv_heads: int = 2, layers: int = 4, ffn: int = 1024, positions: int = 4096, top: int = 8, pages: int = 512,
                 page_tokens: int = 32, name: str = "cache", rotary: bool = False):
        self.owns_context = context is None
        if context is None:
            context = WebDNNCudaContext()
            context.initialize()
        self.context, self.vocab, self.top, self.positions = context, vocab, top, positions
        self.cache = PagedCache(context, layers, pages, kv_heads, d // heads, page_tokens)
        context.add_cache(name, self.cache)
        self.table_pages = -(-positions // page_tokens)      # the same for every call, so that calls repeat
        self._graph = (vocab, d, heads, kv_heads, layers, ffn, positions, top, name, rotary)
        self.runner = self._load()
        self._deciding: Dict[float, object] = {}             # runners that decide on drafts, by their temperature: the last ones used

    MAX_DECIDING = 4

    def _load(self, **how):
        return load(zoo.decoder(*self._graph, **how), backend_order=["cuda", "cpu"], backend_options={"cuda": {"context": self.context}})

    def close(self) -> None:
        for runner in (self.runner, *self._deciding.values()):
            runner.dispose()
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

    def decide(self, sequences: Sequence[int], trees: Sequence[Sequence[int]], parents: Sequence[Sequence[int]], uniforms: np.ndarray,
               temperature: float = 1.0) -> List[Tuple[List[int], int]]:
        """Appends to sequences[i] those tokens of trees[i] that stand: its first, which is decided already, and a path of drafts
        behind it (``parents``: which token of the tree each continues, -1 for the first).  Returns that path, as indices into the
        tree, and the token that follows it, which is not appended.  ``uniforms`` [sequences, tokens of the largest tree] are random
        numbers in [0, 1).  A step that fails leaves the sequences as long as they were."""
        counts = [len(t) for t in trees]
        width = max(counts, default=0)
        if min(counts, default=0) == 0 or len(counts) != len(sequences) or len(set(sequences)) != len(sequences):
            raise ValueError("Decoder.decide: a tree for each of different sequences, of a token or more")
        if len(parents) != len(trees) or not all(len(p) == n and p[0] == -1 and all(0 <= a < i for i, a in enumerate(p) if i)
                                                 for p, n in zip(parents, counts)):
            raise ValueError("Decoder.decide: a token of a tree continues one before it, the first the text")
        uniforms = np.asarray(uniforms)
        if uniforms.shape != (len(trees), width) or not ((uniforms >= 0) & (uniforms < 1)).all():
            raise ValueError(f"Decoder.decide: uniforms are [{len(trees)}, {width}], from 0 to below 1")
        # (numbers next to 1 would be 1 as float32)
        uniforms = np.minimum(uniforms.astype(np.float32), np.float32(1 - 2.0 ** -24))
        before = [self.cache.length(s) for s in sequences]
        ids, places, above = (np.zeros((len(trees), width), np.int32) for _ in range(3))
        for i, (n, tokens, tree) in enumerate(zip(before, trees, parents)):
            ids[i, :counts[i]], above[i, :counts[i]] = tokens, tree
            for j, parent in enumerate(tree):
                places[i, j] = n if j == 0 else places[i, parent] + 1
        if places.max() >= self.positions:
            raise ValueError(f"Decoder.decide: there are places for {self.positions} tokens")
        if ids.min() < 0 or ids.max() >= self.vocab:
            raise ValueError(f"Decoder.decide: tokens are 0 .. {self.vocab - 1}")
        if not is_temperature(temperature):
            raise ValueError("Decoder.decide: a temperature is 0, or 1e-6 to 1e6")
        runner = self._deciding.pop(temperature, None) or self._load(drafts=True, temperature=temperature)
        while len(self._deciding) >= self.MAX_DECIDING:      # (each has the weights once more)
            self._deciding.pop(next(iter(self._deciding))).dispose()
        self._deciding[temperature] = runner
        self.cache.extend(dict(zip(sequences, counts)))
        try:
            # (a tree beside the last places has more tokens than there are places)
            pages = max(len(self.cache.sequence_pages(s)) for s in sequences)
            where = self.cache.batch(sequences, counts, max(self.table_pages, pages))
            outs = runner.run([CPUTensor.from_array(ids), CPUTensor.from_array(places), *where, CPUTensor.from_array(above),
                                                    CPUTensor.from_array(uniforms)])
            path, accepted, following = (t.numpy().copy() for t in outs)
            if (following < 0).any():
                raise RuntimeError("Decoder.decide: the logits behind a token are no distribution")
            # (a path that is the front of its tree is where it has to be)
            if any(path[i, j] != j for i, n in enumerate(accepted) for j in range(n)):
                moved = [self.context.move_tensor(t) for t in (*where, CPUTensor.from_array(path), CPUTensor.from_array(accepted))]
                self.cache.keep_paths(*moved)
                for t in moved:
                    t.dispose()
        except BaseException:
            for s, length in zip(sequences, before):
                self.cache.truncate(s, length)
            raise
        for s, length, n in zip(sequences, before, accepted):
            self.cache.truncate(s, length + int(n))
        return [(path[i, :n].tolist(), int(following[i])) for i, n in enumerate(accepted)]

    def generate(self, prompts: Sequence[Sequence[int]], new_tokens: int, draft: "Decoder", depth: int = 4, width: int = 2,
                 temperature: float = 0.0, seed: int = 0) -> List[List[int]]:
        """``new_tokens`` tokens behind each prompt, distributed as this decoder has them at ``temperature`` (0: the likeliest), whatever
        ``draft``, a smaller decoder of the same tokens, makes of it: that one drafts ``depth`` tokens a step and their likeliest
        ``width`` - 1 alternatives, and this one decides on all of them at once."""
        if not all(len(p) for p in prompts):
            raise ValueError("Decoder.generate: a prompt has a token")
        if draft.vocab != self.vocab or not 1 <= width <= draft.top or depth < 0:
            raise ValueError("Decoder.generate: decoders of the same tokens, 1 to top alternatives, a depth of 0 or more")
        rng = np.random.default_rng(seed)
        texts = [list(p) for p in prompts]
        wanted = [len(p) + new_tokens for p in prompts]
        mine, theirs = [self.cache.add_sequence() for _ in prompts], [draft.cache.add_sequence() for _ in prompts]
        try:
            long = [i for i, t in enumerate(texts) if len(t) > 1]
            if new_tokens and long:
                self.step([mine[i] for i in long], [texts[i][:-1] for i in long], [], [])
            while True:
                alive = [i for i, t in enumerate(texts) if len(t) < wanted[i]]
                if not alive:
                    return [t[len(p):] for t, p in zip(texts, prompts)]
                trees, parents = {i: [texts[i][-1]] for i in alive}, {i: [-1] for i in alive}
                chains = {i: [0] for i in alive}                                 # the drafts that the next ones continue
                for level in range(depth):
                    # (the token that follows a path needs no draft of its own)
                    going = [i for i in alive if len(texts[i]) + level < min(wanted[i] - 1, self.positions, draft.positions)]
                    if not going:
                        break
                    # what the draft has not seen of the text, then what it drafted last
                    fed = [texts[i][draft.cache.length(theirs[i]):] if level == 0 else [trees[i][chains[i][-1]]] for i in going]
                    *_, best, _ = draft.step([theirs[i] for i in going], fed, [(k, len(f) - 1) for k, f in enumerate(fed)], [0] * len(fed))
                    for i, tokens in zip(going, best):
                        parents[i] += [chains[i][-1]] * width
                        chains[i].append(len(trees[i]))
                        trees[i] += [int(t) for t in tokens[:width]]
                uniforms = rng.random((len(alive), max(len(trees[i]) for i in alive)), dtype=np.float32)
                found = self.decide([mine[i] for i in alive], [trees[i] for i in alive], [parents[i] for i in alive], uniforms, temperature)
                for i, (path, following) in zip(alive, found):
                    # the draft has seen the chain but for its last token; what of that stands is a part of the text
                    seen = sum(1 for a, b in zip(path, chains[i]) if a == b)
                    draft.cache.truncate(theirs[i], min(draft.cache.length(theirs[i]), len(texts[i]) - 1 + seen))
                    texts[i] = (texts[i] + [trees[i][j] for j in path[1:]] + [following])[:wanted[i]]
        finally:
            for cache, sequences in ((self.cache, mine), (draft.cache, theirs)):
                for sequence in sequences:
                    cache.release(sequence)

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
    draft = Decoder(decoder.context, layers=1, name="draft")
    print("drafted and decided:", decoder.generate([text[:50]], 12, draft)[0])
    draft.close()
    decoder.close()


if __name__ == "__main__":
    main()
