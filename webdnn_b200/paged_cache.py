"""Keys and values of a decoder in 8 bits, in pages of one pool.

The reference's graphs keep nothing between runs (``core/runnerImpl.ts:315-596``), so a decoder in it attends to whatever
its inputs bring along.  ``PagedCache`` is the state that such a graph needs: the pool on the device (``codes``, int8, four
to an int32 word, and a float32 scale for each page, head and side), and on the host which pages belong to which
sequence.

* device: ``append`` writes new tokens (``append_rotary`` with their keys and queries normalised and rotated), ``attention`` lets
  them attend to their sequences, ``keep_paths`` moves those of a tree that stand to its front, ``copy_pages`` moves pages.  They
  take the page table, lengths and counts as int32 tensors, so a recorded run (tape or graph) repeats with new ones; the pool
  stays where it is.
* host: sequences are numbers.  ``extend`` gives one room for new tokens, ``fork`` shares its pages with a new one, ``release``
  gives them back, ``compact`` moves the pages in use to the front of the pool.  A shared page is copied the moment a
  sequence is about to write to it.

A page has the same index in every layer.
"""
from __future__ import annotations

import ctypes
import heapq
from ctypes import byref
from typing import Dict, List, Optional, Sequence

import numpy as np

from .backend import CPUTensor, CudaTensor, WebDNNCudaContext
from .lib import CacheAppendDesc, CacheAppendRotaryDesc, CacheAttentionDesc, CacheKeepDesc, CachePagesDesc


class PagedCache:
    def __init__(self, context: WebDNNCudaContext, layers: int, pages: int, kv_heads: int, head_size: int,
                 page_tokens: int = 64, codes: Optional[CudaTensor] = None, scales: Optional[CudaTensor] = None):
        """``codes`` (int32 words) and ``scales`` (float32) are the pool's memory, taken over by the cache; it allocates its
        own otherwise."""
        if min(layers, pages, kv_heads) < 1:
            raise ValueError("PagedCache: layers, pages and kv_heads are at least 1")
        if page_tokens not in (16, 32, 64, 128) or head_size not in (32, 64, 128):
            raise ValueError("PagedCache: page_tokens is 16, 32, 64 or 128 and head_size 32, 64 or 128")
        self.context = context
        self.layers, self.pages, self.kv_heads = int(layers), int(pages), int(kv_heads)
        self.head_size, self.page_tokens = int(head_size), int(page_tokens)
        shape = [self.layers, self.pages, 2, self.kv_heads, self.page_tokens, self.head_size // 4]
        for t, dims, kind in ((codes, shape, "int32"), (scales, shape[:4], "float32")):
            if t is not None:
                context.asserts_cuda_tensor(t)
                if t.dims != dims or t.data_type != kind:
                    raise ValueError(f"PagedCache: a pool of this shape is {kind} {dims}, not {t.data_type} {t.dims}")
        self.codes = codes if codes is not None else context.empty_tensor(shape, "int32")
        self.scales = scales if scales is not None else context.empty_tensor(shape[:4])
        self._layer_bytes, self._layer_scale_bytes = self.codes.length // self.layers * 4, self.scales.length // self.layers * 4
        self._descs: Dict[tuple, tuple] = {}                 # of the shapes seen
        self._pages_desc = byref(CachePagesDesc(self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_size))
        self.registered = False                              # by WebDNNCudaContext.add_cache
        self._sequences: Dict[int, List[int]] = {}           # pages of each sequence
        self._lengths: Dict[int, int] = {}
        self._users = [0] * self.pages                       # sequences that hold a page
        self._free = list(range(self.pages))                 # a heap: the lowest page first
        self._next = 0

    def dispose(self) -> None:
        if self.registered:
            raise RuntimeError("PagedCache: graphs of the context may use it: it lives as long as the context")
        self.codes.dispose()
        self.scales.dispose()

    # ---------------------------------------------------------------------------------- on the device
    MAX_SHAPES = 1024

    def _keep(self, key, desc):
        """The description of a call of these shapes, checked once and kept by its shapes alone."""
        if len(self._descs) >= self.MAX_SHAPES:
            self._descs.clear()
        self._descs[key] = kept = (byref(desc), desc)
        return kept

    def _at(self, layer: int):
        if not 0 <= layer < self.layers:
            raise ValueError(f"PagedCache: layer {layer} of {self.layers}")
        return self.codes.ptr + layer * self._layer_bytes, self.scales.ptr + layer * self._layer_scale_bytes

    def _operands(self, who: str, rows: Sequence[CudaTensor], page_table: CudaTensor, lengths: CudaTensor,
                  counts: Optional[CudaTensor]) -> None:
        """Tensors of this context, of the types and in the order of memory that a call takes."""
        for tensors, kind in ((rows, "float32"), ((page_table, lengths) if counts is None else (page_table, lengths, counts), "int32")):
            for t in tensors:
                if t.__class__ is not CudaTensor or t.context is not self.context:
                    self.context.asserts_cuda_tensor(t)
                if t.data_type != kind or t.layout != "nchw":
                    raise TypeError(f"{who}: operands are float32, page_table, lengths and counts int32, all row-major")

    @staticmethod
    def _batch(who: str, rows: Sequence[CudaTensor], page_table: CudaTensor, lengths: CudaTensor, counts: Optional[CudaTensor]):
        """(batch, tokens) of a call: of its [batch, tokens, width] tensors and the int32 ones beside them."""
        for t in rows:
            if t.ndim != 3 or t.dims[:2] != rows[0].dims[:2]:
                raise ValueError(f"{who}: operands are [batch, tokens, width]")
        batch = rows[0].dims[0]
        PagedCache._batch_ints(who, batch, page_table, lengths, counts)
        return batch, rows[0].dims[1]

    @staticmethod
    def _batch_ints(who: str, batch: int, page_table: CudaTensor, lengths: CudaTensor, counts: Optional[CudaTensor]) -> None:
        if page_table.ndim != 2 or page_table.dims[0] != batch or lengths.dims != [batch] or (
                counts is not None and counts.dims != [batch]):
            raise ValueError(f"{who}: page_table is [{batch}, pages], lengths and counts are [{batch}]")

    def append(self, layer: int, k: CudaTensor, v: CudaTensor, page_table: CudaTensor, lengths: CudaTensor,
               counts: Optional[CudaTensor] = None, k_column: int = 0, v_column: int = 0) -> None:
        """Writes new tokens to one layer (``wdc_cache_append``).  k, v: [batch, tokens, width], of which kv_heads *
        head_size columns from ``k_column`` / ``v_column`` on are the heads side by side; ``lengths`` counts the tokens of each
        sequence with the new ones, ``counts`` the new ones (without: all are).  The same call again changes nothing."""
        self._operands("PagedCache.append", (k, v), page_table, lengths, counts)
        key = ("append", *map(tuple, (k.dims, v.dims, page_table.dims, lengths.dims)), counts is not None and tuple(counts.dims), k_column,
               v_column)
        kept = self._descs.get(key) or self._append_desc(key, k, v, page_table, lengths, counts, k_column, v_column)
        if k.length and v.length:
            self.context._call("wdc_cache_append", kept[0], k.ptr + 4 * k_column, v.ptr + 4 * v_column, *self._at(layer),
                               page_table.ptr, lengths.ptr, counts.ptr if counts is not None else None)

    def _append_desc(self, key, k, v, page_table, lengths, counts, k_column, v_column):
        return self._keep(key, self._append_fields("PagedCache.append", k, v, page_table, lengths, counts, k_column, v_column))

    def _append_fields(self, who, k, v, page_table, lengths, counts, k_column, v_column):
        batch, tokens = self._batch(who, (k, v), page_table, lengths, counts)
        width = self.kv_heads * self.head_size
        for t, c in ((k, k_column), (v, v_column)):
            if c < 0 or c % 4 or c + width > t.dims[2] or t.dims[2] % 4:
                raise ValueError(f"{who}: {width} columns from {c} on, of {t.dims[2]} (multiples of 4)")
        kw, vw, c = k.dims[2], v.dims[2], self.head_size
        return CacheAppendDesc(self.pages, self.kv_heads, self.page_tokens, c, batch, tokens, page_table.dims[1],
                               tokens * kw, c, kw, tokens * vw, c, vw)

    def append_rotary(self, layer: int, k: CudaTensor, v: CudaTensor, page_table: CudaTensor, lengths: CudaTensor,
                      counts: Optional[CudaTensor] = None, cos: Optional[CudaTensor] = None, sin: Optional[CudaTensor] = None,
                      positions: Optional[CudaTensor] = None, q: Optional[CudaTensor] = None, heads: Optional[int] = None,
                      q_weight: Optional[CudaTensor] = None, k_weight: Optional[CudaTensor] = None, epsilon: float = 1e-6,
                      interleaved: bool = False, q_column: int = 0, k_column: int = 0, v_column: int = 0,
                      out: Optional[CudaTensor] = None) -> Optional[CudaTensor]:
        """``append`` of keys whose heads are normalised (``k_weight``) and rotated (``cos``, ``sin``) on the way, like
        ``WebDNNCudaContext.rotate_heads`` (``wdc_cache_append_rotary``).  ``positions``: int32 [batch, tokens], without: a token's
        place in its sequence.  With ``q``, whose ``heads`` * head_size columns from ``q_column`` on count, its heads are too
        (``q_weight``); the result is [batch, tokens, heads * head_size], rows of padding 0."""
        who = "PagedCache.append_rotary"
        if q is None and (heads or q_column or out is not None or q_weight is not None):
            raise ValueError(f"{who}: heads, q_column, q_weight and out are of queries")
        self.context.asserts_rows(who, (k, v, q, cos, sin, q_weight, k_weight), (page_table, lengths, counts, positions))
        key = ("append_rotary", *(t is not None and tuple(t.dims) for t in (k, v, q, page_table, lengths, counts, cos, sin, positions, q_weight, k_weight)),
               heads, epsilon, bool(interleaved), q_column, k_column, v_column)
        kept = self._descs.get(key) or self._append_rotary_desc(who, key, k, v, page_table, lengths, counts, cos, sin, positions, q, heads,
                                                                (q_weight, k_weight), epsilon, interleaved, q_column, k_column, v_column)
        codes, scales = self._at(layer)
        if q is not None:
            d = kept[1]
            shape = [d.append.batch, d.append.tokens, d.heads * self.head_size]
            if out is None:
                out = self.context.empty_tensor(shape)
            elif out.__class__ is not CudaTensor or out.context is not self.context or out.dims != shape or out.data_type != "float32" or (
                    out.layout != "nchw" or (out.ptr == q.ptr and (q_column or out.dims != q.dims))):
                raise ValueError(f"{who}: the result is float32 {shape}, row-major, in this context, and q only where that has its shape")
        if k.length and v.length:
            self.context._call("wdc_cache_append_rotary", kept[0], q.ptr + 4 * q_column if q is not None else None, k.ptr + 4 * k_column, v.ptr + 4 * v_column,
                               q_weight.ptr if q_weight is not None else None, k_weight.ptr if k_weight is not None else None,
                               cos.ptr if cos is not None else None, sin.ptr if sin is not None else None,
                               positions.ptr if positions is not None else None, codes, scales, page_table.ptr, lengths.ptr,
                               counts.ptr if counts is not None else None, out.ptr if q is not None else None)
        return out

    def _append_rotary_desc(self, who, key, k, v, page_table, lengths, counts, cos, sin, positions, q, heads, weights, epsilon, interleaved,
                            q_column, k_column, v_column):
        self.context.asserts_rotation(who, self.head_size, cos, sin, positions, weights)
        fields = self._append_fields(who, k, v, page_table, lengths, counts, k_column, v_column)
        c, batch, tokens = self.head_size, fields.batch, fields.tokens
        if positions is not None and positions.dims != [batch, tokens]:
            raise ValueError(f"{who}: positions are [{batch}, {tokens}]")
        if q is None:
            heads = width = 0
        else:
            width = q.dims[2] if q.ndim == 3 else 0
            heads = (width - q_column) // c if heads is None else heads
            if q.ndim != 3 or q.dims[:2] != [batch, tokens] or heads < 1 or q_column < 0 or q_column % 4 or q_column + heads * c > width or width % 4:
                raise ValueError(f"{who}: {heads} heads of {c} from column {q_column} on, of {q.dims}")
        row = heads * c
        return self._keep(key, CacheAppendRotaryDesc(fields, heads, tokens * width, c, width, tokens * row, c, row,
                                                     2 * cos.dims[1] if cos is not None else 0, cos.dims[0] if cos is not None else 0,
                                                     epsilon, interleaved))

    def attention(self, layer: int, q: CudaTensor, page_table: CudaTensor, lengths: CudaTensor,
                  counts: Optional[CudaTensor] = None, heads: Optional[int] = None, q_column: int = 0,
                  scale: Optional[float] = None, out: Optional[CudaTensor] = None,
                  parents: Optional[CudaTensor] = None) -> CudaTensor:
        """Attention of the new tokens over their sequences, themselves and what is before them (``wdc_cache_attention``), after
        ``append``.  q: [batch, tokens, width], of which ``heads`` * head_size columns from ``q_column`` on count (without
        ``heads``: all from there on); the result is [batch, tokens, heads * head_size], rows of padding 0.  ``scale``:
        1 / sqrt(head_size) unless given.  ``parents``: int32 [batch, tokens], the new tokens are a tree
        (``wdc_cache_attention_tree``): which of the new ones, before it, each continues, -1: the text before them; a token then
        sees that text, its ancestors and itself."""
        self._operands("PagedCache.attention", (q,), page_table, lengths, counts)
        if parents is not None:
            self.context.asserts_int_rows("PagedCache.attention", "parents", parents, q.dims[:2])
        key = (*map(tuple, (q.dims, page_table.dims, lengths.dims)), counts is not None and tuple(counts.dims), heads, q_column, scale)
        kept = self._descs.get(key) or self._attention_desc(key, q, page_table, lengths, counts, heads, q_column, scale)
        d = kept[1]
        dims = [d.batch, d.tokens, d.heads * d.head_size]
        if out is None:
            out = self.context.empty_tensor(dims)
        elif out.__class__ is not CudaTensor or out.context is not self.context or out.dims != dims or out.data_type != "float32":
            raise ValueError(f"PagedCache.attention: the result is float32 {dims} of this context")
        if out.length:
            tree = () if parents is None else (parents.ptr,)
            self.context._call("wdc_cache_attention_tree" if tree else "wdc_cache_attention", kept[0], q.ptr + 4 * q_column, *self._at(layer),
                               page_table.ptr, lengths.ptr, counts.ptr if counts is not None else None, *tree, out.ptr)
        return out

    def _attention_desc(self, key, q, page_table, lengths, counts, heads, q_column, scale):
        batch, tokens = self._batch("PagedCache.attention", (q,), page_table, lengths, counts)
        c, width = self.head_size, q.dims[2]
        heads = (width - q_column) // c if heads is None else heads
        if heads < 1 or heads % self.kv_heads or q_column < 0 or q_column % 4 or q_column + heads * c > width or width % 4:
            raise ValueError(f"PagedCache.attention: {heads} heads of {c} from column {q_column} on, of {width}; "
                             f"{self.kv_heads} key heads")
        row = heads * c
        return self._keep(key, CacheAttentionDesc(self.pages, self.kv_heads, self.page_tokens, c, batch, tokens, page_table.dims[1],
                                                  heads, tokens * width, c, width, tokens * row, c, row,
                                                  c ** -0.5 if scale is None else scale))

    def keep_paths(self, page_table: CudaTensor, lengths: CudaTensor, counts: Optional[CudaTensor], path: CudaTensor,
                   accepted: CudaTensor) -> None:
        """Moves the new tokens that stand to the front of their sequences' new ones, in every layer (``wdc_cache_keep_paths``): ``path``
        int32 [batch, tokens] and ``accepted`` int32 [batch] as ``WebDNNCudaContext.verify_drafts`` gives them; the other operands are
        those of the step.  ``truncate`` then takes the sequences to length - count + accepted."""
        self._operands("PagedCache.keep_paths", (), page_table, lengths, counts)
        if path.ndim != 2:
            raise ValueError("PagedCache.keep_paths: path is [batch, tokens]")
        batch, tokens = path.dims
        self.context.asserts_int_rows("PagedCache.keep_paths", "path", path, [batch, tokens])
        self.context.asserts_int_rows("PagedCache.keep_paths", "accepted", accepted, [batch])
        self._batch_ints("PagedCache.keep_paths", batch, page_table, lengths, counts)
        key = ("keep", batch, tokens, page_table.dims[1])
        kept = self._descs.get(key) or self._keep(key, CacheKeepDesc(self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_size,
                                                                     batch, tokens, page_table.dims[1]))
        if path.length:
            self.context._call("wdc_cache_keep_paths", kept[0], self.codes.ptr, self.scales.ptr, page_table.ptr, lengths.ptr,
                               counts.ptr if counts is not None else None, path.ptr, accepted.ptr)

    def copy_pages(self, sources: Sequence[int], targets: Sequence[int]) -> None:
        """Page sources[i] to page targets[i], in every layer (``wdc_cache_copy_pages``)."""
        n = len(sources)
        if n != len(targets):
            raise ValueError("PagedCache.copy_pages: as many sources as targets")
        if n and (min(min(sources), min(targets)) < 0 or max(max(sources), max(targets)) >= self.pages):
            raise ValueError(f"PagedCache.copy_pages: pages are 0 .. {self.pages - 1}")
        array = ctypes.c_int32 * n                       # (in range: nothing is cut off)
        self.context._call("wdc_cache_copy_pages", self._pages_desc, self.codes.ptr, self.scales.ptr, n, array(*sources),
                           array(*targets))

    # ---------------------------------------------------------------------------------- on the host
    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def used_pages(self) -> int:
        return self.pages - len(self._free)

    def length(self, sequence: int) -> int:
        return self._lengths[sequence]

    def sequence_pages(self, sequence: int) -> List[int]:
        return list(self._sequences[sequence])

    def add_sequence(self) -> int:
        """A new, empty sequence."""
        sequence, self._next = self._next, self._next + 1
        self._sequences[sequence], self._lengths[sequence] = [], 0
        return sequence

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._users[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            heapq.heappush(self._free, page)

    def extend(self, new_tokens: Dict[int, int]) -> None:
        """Room for new tokens: {sequence: how many}.  All of it is given or, where the pool has too few free pages, none
        (MemoryError).  Afterwards no page that an append of these tokens writes is shared."""
        need = []
        shared: Dict[int, int] = {}
        wanted = 0
        for s, n in new_tokens.items():
            if n < 0:
                raise ValueError("PagedCache.extend: negative number of tokens")
            pages, length = self._sequences[s], self._lengths[s]
            need.append(-(-(length + n) // self.page_tokens) - len(pages))
            wanted += max(need[-1], 0)
            if n and length % self.page_tokens:              # the page that is partly filled is written to
                shared[pages[length // self.page_tokens]] = shared.get(pages[length // self.page_tokens], 0) + 1
        # of the sequences that write to a shared page all take a copy, but for one if nobody else keeps it
        wanted += sum(w if self._users[p] > w else w - 1 for p, w in shared.items())
        if wanted > len(self._free):
            raise MemoryError(f"PagedCache: {wanted} pages are needed, {len(self._free)} are free")
        sources, targets, copied = [], [], []
        for (s, n), more in zip(new_tokens.items(), need):
            pages, length = self._sequences[s], self._lengths[s]
            at = length // self.page_tokens
            if n and length % self.page_tokens and self._users[pages[at]] > 1:
                sources.append(pages[at])
                self._users[pages[at]] -= 1
                pages[at] = self._take()
                targets.append(pages[at])
                copied.append((pages, at))
            pages.extend(self._take() for _ in range(more))
            self._lengths[s] = length + n
        if sources:
            try:
                self.copy_pages(sources, targets)
            except BaseException:
                for s, n in new_tokens.items():
                    self.truncate(s, self._lengths[s] - n)
                for (pages, at), page in zip(copied, sources):
                    self._drop(pages[at])
                    pages[at] = page
                    self._users[page] += 1
                raise

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens, on the same pages."""
        pages = self._sequences[sequence]
        for p in pages:
            self._users[p] += 1
        new = self.add_sequence()
        self._sequences[new], self._lengths[new] = list(pages), self._lengths[sequence]
        return new

    def truncate(self, sequence: int, length: int) -> None:
        """Forgets the tokens from ``length`` on (a draft that was not accepted)."""
        if not 0 <= length <= self._lengths[sequence]:
            raise ValueError(f"PagedCache.truncate: {length} of {self._lengths[sequence]} tokens")
        pages = self._sequences[sequence]
        keep = -(-length // self.page_tokens)
        for p in pages[keep:]:
            self._drop(p)
        del pages[keep:]
        self._lengths[sequence] = length

    def release(self, sequence: int) -> None:
        for p in self._sequences.pop(sequence):
            self._drop(p)
        del self._lengths[sequence]

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool; returns how many were moved."""
        used = self.used_pages
        holes = sorted(p for p in self._free if p < used)
        moved = [p for p in range(used, self.pages) if self._users[p]]
        if not moved:
            return 0
        self.copy_pages(moved, holes)
        to = dict(zip(moved, holes))
        for pages in self._sequences.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(used, self.pages))
        return len(moved)

    def batch(self, sequences: Sequence[int], new_tokens: Sequence[int], table_pages: Optional[int] = None):
        """(page_table, lengths, counts) of a call for these sequences, the last ``new_tokens[i]`` of each being new, as host
        tensors.  ``table_pages``: the width of the table, where it shall be the same for every call."""
        widest = max([len(self._sequences[s]) for s in sequences] or [0])
        width = max(widest, 1) if table_pages is None else table_pages
        if width < widest or len(sequences) != len(new_tokens):
            raise ValueError("PagedCache.batch: one count a sequence, and a table that is wide enough")
        table = np.full((len(sequences), width), -1, np.int32)
        for row, s in zip(table, sequences):
            row[:len(self._sequences[s])] = self._sequences[s]
        lengths = np.array([self._lengths[s] for s in sequences], np.int32)
        return tuple(CPUTensor.from_array(a) for a in (table, lengths, np.array(new_tokens, np.int32)))
