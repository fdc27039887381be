"""The operators of a decoder that drafts, as measured cases.

A decoder with rotary positions normalises and rotates the heads of its queries and keys ("rotate"), or does so on the way to the
8-bit paged cache ("append").  To gain several tokens a step it lets a smaller model draft some: a tree of candidate
continuations whose first token is the last one decided.  All of the tree attends at once, each token to the text before and to its
ancestors ("tree").  The logits behind every token then decide, with given random numbers, which path of the tree stands and
which token follows it ("verify"), and the tokens of that path move to the front of the cache's new ones ("keep").

Everything a step takes and gives is float32 or int32, the types of the runtime.

A page of the pool is [2 (keys, values)][kv_heads][page_tokens][head_size] int8, its scales [2][kv_heads] float32; a number
is code * scale.  A page table row names the pages of one sequence in order.  `lengths` counts the tokens of each sequence
with the new ones, `counts` the new ones, which are the last; rows of a call behind a sequence's count are padding.  `parents` holds
for each new token which of the new ones it continues, -1: the text before them.
"""
import functools
import math

import torch

own = False

_DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
_SPREAD = 40.0        # standard deviation of the codes: +-127 is about three of them
_BASE = 10000.0       # of the rotation's angles: position * _BASE ** (-2 i / rotary)
_EPSILON = 1e-6


def listed():
    return [
        # the queries of the next token of one conversation, a long way into it: launches and latency are all there is
        dict(name="rotate_1x40", op="rotate", rows=1, heads=40, head_size=128, rotary=128, interleaved=False, norm=True, places=40000),
        # the heads of a long prompt, a part of their channels rotated
        dict(name="rotate_9001x24", op="rotate", rows=9001, heads=24, head_size=80, rotary=32, interleaved=False, norm=True,
             places=9001),
        # the new token of each sequence of a serving batch
        dict(name="append_64x1", op="append", batch=64, tokens=1, shortest=5, longest=3000, heads=32, kv_heads=8, head_size=128,
             page_tokens=64, rotary=128, interleaved=False, norm=True),
        # prompts of uneven lengths, neighbouring channels rotated together, no norms
        dict(name="append_5x2001", op="append", batch=5, tokens=2001, shortest=900, longest=2500, heads=24, kv_heads=8, head_size=64,
             page_tokens=32, rotary=64, interleaved=True, norm=False),
        # one conversation, a small tree
        dict(name="tree_1x900_11", op="tree", batch=1, tokens=11, shortest=900, longest=900, heads=16, kv_heads=4, head_size=64,
             page_tokens=16),
        # a serving batch of uneven conversations, trees of up to 13 tokens, four query heads to a key head
        dict(name="tree_24x2500_13", op="tree", batch=24, tokens=13, shortest=100, longest=2500, heads=32, kv_heads=8, head_size=128,
             page_tokens=64),
        # a few long documents, large trees
        dict(name="tree_3x20001_61", op="tree", batch=3, tokens=61, shortest=9000, longest=20001, heads=32, kv_heads=8, head_size=128,
             page_tokens=128),
        # one conversation, a chain of drafts from a smaller model's distribution
        dict(name="verify_1x32000_5", op="verify", batch=1, tokens=5, vocab=32000, draft=True, chain=True, temperature=1.0),
        # a batch of trees whose drafts are the likeliest tokens
        dict(name="verify_16x100003_25", op="verify", batch=16, tokens=25, vocab=100003, draft=False, chain=False, temperature=0.8),
        # a large batch of trees of sampled drafts
        dict(name="verify_64x50001_9", op="verify", batch=64, tokens=9, vocab=50001, draft=True, chain=False, temperature=1.0),
        # two conversations, a small model
        dict(name="keep_2x12", op="keep", batch=2, tokens=12, accepted=4, shortest=100, longest=300, layers=6, kv_heads=4, head_size=64,
             page_tokens=16),
        # a serving batch, all layers of a larger model
        dict(name="keep_40x32", op="keep", batch=40, tokens=32, accepted=9, shortest=40, longest=250, layers=30, kv_heads=8,
             head_size=128, page_tokens=32),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotate", "append", "tree", "tree", "verify", "verify", "keep"])
    if op == "verify":
        vocab, tokens, kind = _log(rng, 300, 200000), _log(rng, 1, 32), rng.choice(["draft", "draft", "target", "greedy"])
        return dict(op=op, batch=_log(rng, 1, max(1, min(64, 28_000_000 // (vocab * tokens)))), tokens=tokens, vocab=vocab,
                    draft=kind == "draft", chain=rng.random() < 0.5,
                    temperature=0.0 if kind == "greedy" else rng.choice([0.6, 1.0, 1.0, 1.3]))
    how = dict(interleaved=rng.random() < 0.5, norm=rng.random() < 0.5)
    if op == "rotate":
        heads, head_size = rng.choice([1, 3, 5, 8, 16, 24, 32]), rng.choice([32, 40, 64, 80, 96, 128, 256])
        rows = _log(rng, 1, max(1, min(20000, 17_000_000 // (heads * head_size))))
        rotary = rng.choice([head_size, head_size, head_size // 16 * 8])
        return dict(op=op, rows=rows, heads=heads, head_size=head_size, rotary=rotary, places=rows + _log(rng, 1, 30000), **how)
    kv_heads, head_size = rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([32, 64, 128])
    page_tokens, width = rng.choice([16, 32, 64, 128]), kv_heads * head_size
    if op == "keep":
        tokens, layers = _log(rng, 2, 64), rng.randint(1, 30)
        longest = tokens + _log(rng, 1, 200)
        batch = _log(rng, 1, max(1, min(64, 300_000_000 // (layers * longest * width))))
        return dict(op=op, batch=batch, tokens=tokens, accepted=rng.randint(1, min(tokens, 12)), shortest=rng.randint(tokens, longest),
                    longest=longest, layers=layers, kv_heads=kv_heads, head_size=head_size, page_tokens=page_tokens)
    group = rng.choice([1, 2, 3, 4, 6, 8])
    if op == "append":
        tokens = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2001)])
        batch = _log(rng, 1, max(1, min(128, 15_000_000 // (tokens * width * (group + 2)))))
        longest = tokens + _log(rng, 1, 2000)
        return dict(op=op, batch=batch, tokens=tokens, shortest=min(longest, tokens // 2 + 1), longest=longest, heads=group * kv_heads,
                    kv_heads=kv_heads, head_size=head_size, page_tokens=page_tokens,
                    rotary=rng.choice([head_size, head_size, head_size // 2]), **how)
    tokens = rng.choice([_log(rng, 1, 8), _log(rng, 4, 64), _log(rng, 4, 64), _log(rng, 64, 200)])
    longest = tokens + _log(rng, 1, 20000)
    batch = _log(rng, 1, max(1, min(64, 60_000_000 // (longest * width), 6_000_000_000 // (tokens * longest * width * group))))
    return dict(op=op, batch=batch, tokens=tokens, shortest=rng.randint(max(1, tokens // 2), longest), longest=longest,
                heads=group * kv_heads, kv_heads=kv_heads, head_size=head_size, page_tokens=page_tokens)


def _lengths(case):
    """(tokens of each sequence, new ones of them): spread evenly between the shortest and the longest."""
    b, lo, hi = case["batch"], case.get("shortest", 1 << 20), case.get("longest", 1 << 20)
    lengths = [hi - (hi - lo) * i // max(b - 1, 1) for i in range(b)]
    # the last sequences bring fewer new tokens than the call has room for
    counts = [min(n, max(1, case["tokens"] - (case["tokens"] * i) // (2 * b))) for i, n in enumerate(lengths)]
    return lengths, counts


# ------------------------------------------------------------------------------------------------ what a program has
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEVICE)


def _tables(places, rotary):
    """Cosines and sines [places, rotary / 2] of the angles, which are far beyond 2 pi: in 64 bits, rounded at the end."""
    at = torch.arange(places, dtype=torch.float64, device=_DEVICE)[:, None]
    angle = at * _BASE ** (-2 * torch.arange(rotary // 2, dtype=torch.float64, device=_DEVICE) / rotary)
    return dict(cos=torch.cos(angle).float(), sin=torch.sin(angle).float())


def _pool(case, g):
    """Codes and scales of a pool, and a page table of it: pages in no order, -1 behind a sequence's last."""
    lengths, counts = _lengths(case)
    need = [-(-n // case["page_tokens"]) for n in lengths]
    pages = sum(need) + 7
    layers = [case["layers"]] if "layers" in case else []
    shape = (*layers, pages + 1 - len(layers), 2, case["kv_heads"], case["page_tokens"], case["head_size"])
    codes = torch.empty(shape, dtype=torch.int8, device=_DEVICE)        # (of one layer: the last page is in no table)
    for part in codes.split(max(1, (1 << 26) // codes[0].numel())):
        part.copy_((torch.randn(part.shape, generator=g, device=_DEVICE) * _SPREAD).round_().clamp_(-127, 127))
    scales = torch.exp(0.3 * torch.randn(shape[:-2], generator=g, device=_DEVICE)) / _SPREAD
    order = torch.randperm(pages, generator=g, device=_DEVICE).to(torch.int32)
    table = torch.full((case["batch"], max(need) + 3), -1, dtype=torch.int32, device=_DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return dict(codes=codes, scales=scales, table=table, lengths=_ints(lengths), counts=_ints(counts))


def _parents(case, g):
    """[batch, tokens]: a chain, or trees in which a token continues the one before it or any earlier one."""
    b, n = case["batch"], case["tokens"]
    chain = torch.arange(-1, n - 1, device=_DEVICE).expand(b, n)
    if case.get("chain"):
        return chain.int().contiguous()
    any_of = (torch.rand((b, n), generator=g, device=_DEVICE) * torch.arange(n, device=_DEVICE)).long()
    parents = torch.where(torch.rand((b, n), generator=g, device=_DEVICE) < 0.4, chain, any_of)
    parents[:, 0] = -1
    return parents.int()


def _logits(rows, vocab, g):
    """A language model's: most tokens unlikely, a few of each row that are not."""
    x = torch.randn((rows, vocab), generator=g, device=_DEVICE) * 2
    ids = torch.randint(0, vocab, (rows, 6), generator=g, device=_DEVICE)
    return x.scatter_(1, ids, 10 + 7 * torch.rand((rows, 6), generator=g, device=_DEVICE))


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    state = dict(case=case)
    randn = lambda *shape: torch.randn(shape, generator=g, device=_DEVICE)  # noqa: E731
    op = case["op"]
    if op == "rotate":
        state.update(_tables(case["places"], case["rotary"]))
        state["x"] = randn(case["rows"], case["heads"] * case["head_size"])
        first = case["places"] - case["rows"]
        state["positions"] = _ints(list(range(first, first + case["rows"])))
        state["weight"] = 1 + 0.2 * randn(case["head_size"])
        state["y"] = torch.empty_like(state["x"])
    elif op == "append":
        state.update(_pool(case, g))
        state.update(_tables(case["longest"], case["rotary"]))
        b, n, d = case["batch"], case["tokens"], case["head_size"]
        state["q"] = randn(b, n, case["heads"] * d)
        state["k"], state["v"] = (randn(b, n, case["kv_heads"] * d) for _ in range(2))
        state["positions"] = (state["lengths"] - state["counts"])[:, None] + torch.arange(n, dtype=torch.int32, device=_DEVICE)
        state["positions"].clamp_(max=case["longest"] - 1)                     # (rows of padding)
        state["q_weight"], state["k_weight"] = 1 + 0.2 * randn(d), 1 + 0.2 * randn(d)
        state["y"] = torch.empty_like(state["q"])
    elif op == "tree":
        state.update(_pool(case, g))
        state["parents"] = _parents(case, g)
        state["q"] = randn(case["batch"], case["tokens"], case["heads"] * case["head_size"])
        state["y"] = torch.empty_like(state["q"])
    elif op == "keep":
        state.update(_pool(case, g))
        n = case["tokens"]
        # token 0, and some of the others in order
        chosen = torch.rand((case["batch"], n), generator=g, device=_DEVICE) + (torch.arange(n, device=_DEVICE) >= state["counts"][:, None])
        chosen[:, 0] = -1
        most = torch.randint(1, case["accepted"] + 1, (case["batch"],), generator=g, device=_DEVICE)
        state["accepted"] = torch.minimum(most, state["counts"].long()).int()
        rank = chosen.argsort(1).argsort(1)
        path = torch.where(rank < state["accepted"][:, None], torch.arange(n, device=_DEVICE), n).sort(1).values
        state["path"] = torch.where(path < n, path, -1).int()
    else:
        b, n, vocab = case["batch"], case["tokens"], case["vocab"]
        state["parents"], state["counts"] = _parents(case, g), _ints(_lengths(case)[1])
        state["logits"] = _logits(b * n, vocab, g).view(b, n, vocab)
        state["uniforms"] = torch.rand((b, n), generator=g, device=_DEVICE)
        guess = state["logits"] + 0.7 * randn(b, n, vocab)                      # what a smaller model makes of it
        tokens = torch.randint(0, vocab, (b, n), generator=g, device=_DEVICE)
        every = torch.arange(b, device=_DEVICE)
        taken = torch.zeros((b, n), dtype=torch.long, device=_DEVICE)           # children that a token has
        for i in range(1, n):
            parent = state["parents"][:, i].long()
            if case["draft"]:
                noise = torch.rand((b, vocab), generator=g, device=_DEVICE).clamp_min(1e-12)
                tokens[:, i] = (guess[every, parent] / case["temperature"] - torch.log(-torch.log(noise))).argmax(1)
            else:
                best = guess[every, parent].topk(min(n, vocab), 1).indices
                tokens[:, i] = best[every, taken[every, parent].clamp_max(best.shape[1] - 1)]
                taken[every, parent] += 1
        state["tokens"] = tokens.int()
        if case["draft"]:
            state["draft_logits"] = guess
        state["path"] = torch.empty((b, n), dtype=torch.int32, device=_DEVICE)
        state["accepted"], state["next"] = (torch.empty(b, dtype=torch.int32, device=_DEVICE) for _ in range(2))
    if own:
        _bind(state)
    return state


# ------------------------------------------------------------------------------------------------ the framework's calls
@functools.lru_cache(maxsize=1)
def _context():
    from webdnn_b200.backend import WebDNNCudaContext
    context = WebDNNCudaContext()
    context.initialize()
    return context


def _bind(state):
    """The tensors and the cache of the framework over a program's device memory, which it keeps."""
    from webdnn_b200.paged_cache import PagedCache
    context, case = _context(), state["case"]
    names = {torch.float32: "float32", torch.int32: "int32"}

    def tensor(t, dims=None):
        return context.borrow_tensor(t.data_ptr(), dims or list(t.shape), names.get(t.dtype, "int32"), owner=t)

    state["own"] = {n: tensor(t) for n, t in state.items() if torch.is_tensor(t) and n not in ("codes", "scales")}
    if "codes" in state:
        layers = case.get("layers", 1)
        pages = state["codes"].shape[1] if "layers" in case else state["codes"].shape[0] - 1
        words = [layers, pages, 2, case["kv_heads"], case["page_tokens"], case["head_size"] // 4]   # four codes each
        state["cache"] = PagedCache(context, layers, pages, case["kv_heads"], case["head_size"], case["page_tokens"],
                                    codes=tensor(state["codes"], words), scales=tensor(state["scales"], words[:4]))


def _run_own(state):
    case, t = state["case"], state["own"]
    op = case["op"]
    if op == "rotate":
        _context().rotate_heads(t["x"], case["heads"], case["head_size"], cos=t["cos"], sin=t["sin"], positions=t["positions"],
                                weight=t["weight"] if case["norm"] else None, epsilon=_EPSILON, interleaved=case["interleaved"],
                                out=t["y"])
    elif op == "append":
        state["cache"].append_rotary(0, t["k"], t["v"], t["table"], t["lengths"], t["counts"], cos=t["cos"], sin=t["sin"],
                                     positions=t["positions"], q=t["q"], q_weight=t["q_weight"] if case["norm"] else None,
                                     k_weight=t["k_weight"] if case["norm"] else None, epsilon=_EPSILON,
                                     interleaved=case["interleaved"], out=t["y"])
    elif op == "tree":
        state["cache"].attention(0, t["q"], t["table"], t["lengths"], t["counts"], parents=t["parents"], out=t["y"])
    elif op == "keep":
        state["cache"].keep_paths(t["table"], t["lengths"], t["counts"], t["path"], t["accepted"])
    else:
        _context().verify_drafts(t["logits"], t["tokens"], t["parents"], counts=t["counts"], uniforms=t["uniforms"],
                                 draft_logits=t.get("draft_logits"), temperature=case["temperature"],
                                 draft_temperature=case["temperature"], out=(t["path"], t["accepted"], t["next"]))


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_rotated(x, weight, cos, sin, interleaved):
    """Heads [..., heads, head_size] normalised and rotated by cos, sin [..., 1, rotary / 2]; in 64 bits, rounded once: the keys' codes
    hang on the last bit."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPSILON) * weight.double()
    half = cos.shape[-1]
    cos, sin = cos.double(), sin.double()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1).float()


def _plain_rotate(state):
    case = state["case"]
    at = state["positions"].long()
    x = state["x"].view(case["rows"], case["heads"], case["head_size"])
    y = _plain_rotated(x, state["weight"] if case["norm"] else None, state["cos"][at][:, None], state["sin"][at][:, None],
                       case["interleaved"])
    return y.flatten(1)


def _plain_append(state):
    case = state["case"]
    b, n, h, d, size = case["batch"], case["tokens"], case["kv_heads"], case["head_size"], case["page_tokens"]
    at = state["positions"].long()
    cos, sin = state["cos"][at][:, :, None], state["sin"][at][:, :, None]
    turned = lambda name: _plain_rotated(state[name].view(b, n, -1, d), state[name + "_weight"] if case["norm"] else None, cos,  # noqa: E731
                                         sin, case["interleaved"])
    there = torch.arange(n, device=_DEVICE) < state["counts"].long()[:, None]
    y = turned("q").flatten(2).masked_fill(~there[..., None], 0)
    # the rotated keys and the values, as codes: a page's scale is its largest number / 127, and only grows while it holds older tokens
    spare = state["codes"].shape[0] - 1
    start = state["lengths"].long() - state["counts"].long()
    slots = (n + size - 2) // size + 1                                                 # pages a sequence may touch
    page = start[:, None] // size + torch.arange(slots, device=_DEVICE)                # [batch, slot]
    token = (page * size - start[:, None])[..., None] + torch.arange(size, device=_DEVICE)     # which new one is there
    new = (token >= 0) & (token < state["counts"].long()[:, None, None])
    kept = page * size < start[:, None]                                                # the page holds older tokens
    ids = torch.where(new.any(-1), state["table"].long().gather(1, page.clamp_max(state["table"].shape[1] - 1)), spare)
    x = torch.stack([turned("k"), state["v"].view(b, n, h, d)])
    x = x[:, torch.arange(b, device=_DEVICE)[:, None, None], token.clamp(0, n - 1)]    # [2, batch, slot, token, head, d]
    x = x.permute(1, 2, 0, 4, 3, 5)                                                    # like a page: [.., 2, head, token, d]
    is_new, is_old = new[:, :, None, None, :, None], ~new[:, :, None, None, :, None]
    top = torch.full((), 127.0, device=_DEVICE)
    fresh = x.abs().masked_fill(is_old, 0).amax((-1, -2)) / top
    before = state["scales"][ids]
    scale = torch.where(kept[:, :, None, None], torch.maximum(before, fresh), fresh)
    old = state["codes"][ids]
    by = torch.where(scale > 0, scale, 1.0)[..., None, None]
    again = (old.float() * before[..., None, None] / by).round().clamp(-127, 127).to(torch.int8)
    grown = (kept[:, :, None, None] & (scale > before))[..., None, None]
    older = (token < 0)[:, :, None, None, :, None]
    codes = torch.where(is_new, (x / by).round().clamp(-127, 127).to(torch.int8), torch.where(grown & older, again, old))
    state["codes"][ids] = codes
    state["scales"][ids] = scale
    return y


def _seen(parents):
    """[batch, n, n]: whether new token j is i itself or above it, by doubling the steps that are looked at."""
    b, n = parents.shape
    up = torch.zeros((b, n, n + 1), device=_DEVICE).scatter_(2, parents.long()[..., None] % (n + 1), 1.0)[..., :n]
    reach = torch.eye(n, device=_DEVICE) + up
    for _ in range(max(1, n.bit_length())):
        reach = (reach @ reach).clamp_max(1.0)
    return reach > 0


def _plain_tree(state):
    case, table = state["case"], state["table"].long().clamp_min(0)
    b, n, h, d = case["batch"], case["tokens"], case["kv_heads"], case["head_size"]
    keys, values = ((state["codes"][table, i].float() * state["scales"][table, i][..., None, None])
                    .transpose(1, 2).reshape(b, h, -1, d) for i in (0, 1))            # [batch, kv head, token, channel]
    group, room = case["heads"] // h, keys.shape[2]
    q = state["q"].view(b, n, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, n * group, d)
    scores = (q @ keys.transpose(2, 3)) / math.sqrt(d)
    start = state["lengths"].long() - state["counts"].long()
    new = torch.arange(room, device=_DEVICE) - start[:, None]                          # which new token a place holds
    above = _seen(state["parents"]).gather(2, new.clamp(0, n - 1)[:, None].expand(b, n, room)) & (new >= 0)[:, None] & (new < n)[:, None]
    seen = above | (new < 0)[:, None]
    seen &= (torch.arange(n, device=_DEVICE) < state["counts"].long()[:, None])[..., None]
    seen = seen[:, None, :, None].expand(b, 1, n, group, room).reshape(b, 1, n * group, -1)
    scores = scores.masked_fill(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    y = (weights @ values) / weights.sum(-1, keepdim=True).clamp_min(1e-30)
    return y.view(b, h, n, group, d).permute(0, 2, 1, 3, 4).reshape(b, n, -1)


def _plain_keep(state):
    """A token that stays in its page keeps its code unless the page's scale has to grow for one that comes from another page."""
    case = state["case"]
    b, n, size = case["batch"], case["tokens"], case["page_tokens"]
    start, accepted = (state["lengths"] - state["counts"]).long(), state["accepted"].long()
    index = torch.arange(n, device=_DEVICE)
    source = start[:, None] + torch.where(index < accepted[:, None], state["path"].long(), index)
    slots = (n + size - 2) // size + 1
    place = start[:, None] // size * size + torch.arange(slots * size, device=_DEVICE)           # of the pages that are written to
    which = place - start[:, None]
    kept = (which >= 0) & (which < accepted[:, None])
    comes_from = torch.where(kept, source.gather(1, which.clamp(0, n - 1)), place)
    pages = state["table"].long()
    page_of = lambda at: pages.gather(1, (at // size).clamp_max(pages.shape[1] - 1)).clamp_min(0)  # noqa: E731
    to, of = page_of(place), page_of(comes_from)
    scales_of = state["scales"][:, of]                                                 # [layer, batch, place, 2, head]
    x = state["codes"][:, of, :, :, comes_from % size].permute(2, 0, 1, 3, 4, 5)       # [layer, batch, place, 2, head, d]
    moved = (kept & (of != to))[None, :, :, None, None]
    top = torch.full((), 127.0, device=_DEVICE)
    peak = torch.where(moved, x.float().abs().amax(-1) * scales_of / top, 0.0)
    peak = peak.unflatten(2, (slots, size)).amax(3)                                    # of a page: [layer, b, slot, 2, h]
    ids = to.view(b, slots, size)[..., 0]
    before = state["scales"][:, ids]
    scale = torch.maximum(before, peak)
    written = kept.view(b, slots, size).any(-1)
    live = (which < accepted[:, None])[None, :, :, None, None, None]                   # the rest of a page stays as it is
    wide = scale.repeat_interleave(size, 2)
    again = (x.float() * scales_of[..., None] / torch.where(wide > 0, wide, 1.0)[..., None]).round().clamp(-127, 127).to(torch.int8)
    same = ((of == to)[None, :, :, None, None] & (wide == scales_of))[..., None]
    codes = torch.where(live & ~same, again, x).unflatten(2, (slots, size)).permute(0, 1, 2, 4, 5, 3, 6)   # like pages
    state["codes"][:, ids[written]] = codes[:, written]
    state["scales"][:, ids[written]] = scale[:, written]


def _weights(x, temperature):
    """Probabilities of rows of logits; at temperature 0 all of it is the first of the largest."""
    x = x.double()
    if temperature == 0:
        return torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
    return torch.softmax(x / temperature, 1)


def _sample(w, u):
    """The first index whose running sum passes u of the whole; borders between tokens are as near as 64 bits tell them apart."""
    run = w.cumsum(1)
    return (run <= u.double()[:, None] * run[:, -1:]).sum(1).clamp_max(w.shape[1] - 1)


def _plain_verify(state):
    """The tree's tokens in their order: a child of the token that the walk stands at is tried, and taken or not."""
    case = state["case"]
    b, n = case["batch"], case["tokens"]
    every = torch.arange(b, device=_DEVICE)
    at = torch.zeros(b, dtype=torch.long, device=_DEVICE)
    length = torch.ones(b, dtype=torch.long, device=_DEVICE)
    path = torch.full((b, n + 1), -1, device=_DEVICE)
    path[:, 0] = 0
    row = lambda name, i: _weights(state[name][every, i], case["temperature"])  # noqa: E731
    p = row("logits", at)
    wanted = None if case["draft"] else _sample(p, state["uniforms"][:, 0])
    for i in range(1, n):
        token = state["tokens"][:, i].long()
        tried = (state["parents"][:, i] == at) & (i < state["counts"])
        if case["draft"]:
            q = row("draft_logits", at)
            taken = tried & (state["uniforms"][:, i].double() * q[every, token] * p.sum(1) < p[every, token])
            left = (p / p.sum(1, keepdim=True) - q).clamp_min(0)
            left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
            p = torch.where((tried & ~taken)[:, None], left, p)
        else:
            taken = tried & (token == wanted)
        at = torch.where(taken, i, at)
        path.scatter_(1, torch.where(taken, length, n)[:, None], i)
        length = length + taken
        path[:, n] = -1
        p = torch.where(taken[:, None], row("logits", at), p)
        if not case["draft"]:
            wanted = torch.where(taken, _sample(p, state["uniforms"][every, at]), wanted)
    following = _sample(p, state["uniforms"][:, 0]) if case["draft"] else wanted
    return [path[:, :n].int(), length.int(), following.int()]


def run(state):
    op = state["case"]["op"]
    if own:
        _run_own(state)
        result = [state[n] for n in ("path", "accepted", "next")] if op == "verify" else state.get("y")
    else:
        result = {"rotate": _plain_rotate, "append": _plain_append, "tree": _plain_tree, "keep": _plain_keep,
                  "verify": _plain_verify}[op](state)
    if op == "append":
        # the queries, and the pool as it stands now, codes in units of the page's scale and those scales; without the page of no table
        return [result, state["codes"][:-1], state["scales"][:-1]]
    return [state["codes"], state["scales"]] if op == "keep" else result


# ------------------------------------------------------------------------------------------------ from the definitions
def _exact_rotated(x, weight, angle_cos, angle_sin, interleaved):
    """x [rows, heads, head_size], in 64 bits: pairs as complex numbers, times the unit number of their angle."""
    x = x.double()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPSILON) * weight.double()
    unit = torch.complex(angle_cos.double(), angle_sin.double())[:, None]
    half = unit.shape[-1]
    pairs = x[..., :2 * half].reshape(*x.shape[:2], half, 2) if interleaved else x[..., :2 * half].reshape(*x.shape[:2], 2, half).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    return torch.cat([(turned if interleaved else turned.transpose(-1, -2)).reshape(*x.shape[:2], 2 * half), x[..., 2 * half:]], -1)


def _exact_append(state):
    case = state["case"]
    size, h, d = case["page_tokens"], case["kv_heads"], case["head_size"]
    scales = state["scales"].double()
    y = torch.zeros(state["y"].shape, dtype=torch.float64, device=_DEVICE)
    for b, (length, count) in enumerate(zip(*_lengths(case))):
        start = length - count
        cos, sin = (state[name][start:length] for name in ("cos", "sin"))
        turned = lambda name: _exact_rotated(state[name][b, :count].view(count, -1, d), state[name + "_weight"] if case["norm"] else None,  # noqa: E731
                                             cos, sin, case["interleaved"])
        y[b, :count] = turned("q").flatten(1)
        sides = turned("k"), state["v"][b, :count].double().view(count, h, d)
        for p in range(start // size, (length - 1) // size + 1):
            lo, hi = max(start, p * size), min(length, (p + 1) * size)
            page = int(state["table"][b, p])
            for i, side in enumerate(sides):
                peak = side[lo - start:hi - start].abs().amax((0, 2)) / 127
                scales[page, i] = torch.maximum(scales[page, i], peak) if lo > p * size else peak
    return [y, None, scales[:-1]]     # (codes are whole numbers, rounded by the 32-bit scale that stands beside them)


def _exact_tree(state):
    case = state["case"]
    size, h, d = case["page_tokens"], case["kv_heads"], case["head_size"]
    out = torch.zeros(state["y"].shape, dtype=torch.float64, device=_DEVICE)
    parents = state["parents"].tolist()
    for b, (length, count) in enumerate(zip(*_lengths(case))):
        ids = state["table"][b, :-(-length // size)].long()
        page = state["codes"][ids].double() * state["scales"][ids].double()[..., None, None]
        k, v = (page[:, i].permute(1, 0, 2, 3).reshape(h, -1, d)[:, :length] for i in (0, 1))
        hidden = torch.ones(count, count, dtype=torch.bool)
        for i in range(count):
            j = i
            while j >= 0:
                hidden[i, j] = False
                j = parents[b][j]
        hidden = torch.cat([torch.zeros(count, length - count, dtype=torch.bool), hidden], 1).to(_DEVICE)
        for head in range(case["heads"]):
            q = state["q"][b, :count, head * d:(head + 1) * d].double()
            s = (q @ k[head * h // case["heads"]].T * d ** -0.5).masked_fill(hidden, -math.inf)
            out[b, :count, head * d:(head + 1) * d] = torch.softmax(s, -1) @ v[head * h // case["heads"]]
    return out


def _exact_keep(state):
    case = state["case"]
    size = case["page_tokens"]
    scales, table = state["scales"].double(), state["table"].tolist()
    new = scales.clone()
    path, accepted = state["path"].tolist(), state["accepted"].tolist()
    for b, (length, count) in enumerate(zip(*_lengths(case))):
        start = length - count
        for i in range(accepted[b]):
            to, of = start + i, start + path[b][i]
            if to // size != of // size:
                a, z = table[b][of // size], table[b][to // size]
                peak = state["codes"][:, a, :, :, of % size].double().abs().amax(-1) * scales[:, a] / 127
                new[:, z] = torch.maximum(new[:, z], peak)
    return [None, new]


def _exact_verify(state):
    case = state["case"]
    paths, lengths, following = [], [], []
    tokens, parents, counts = state["tokens"].tolist(), state["parents"].tolist(), state["counts"].tolist()
    uniforms = state["uniforms"].double().tolist()

    def chances(name, b, i):
        x = state[name][b, i].double()
        if case["temperature"] == 0:
            return (torch.arange(len(x), device=_DEVICE) == int(x.argmax())).double()
        e = torch.exp((x - x.max()) / case["temperature"])
        return e / e.sum()

    def drawn(p, u):
        run = torch.cumsum(p, 0)
        return int(torch.searchsorted(run, u * run[-1], right=True).clamp_max(len(p) - 1))

    for b in range(case["batch"]):
        path, p = [0], chances("logits", b, 0)
        token = None if case["draft"] else drawn(p, uniforms[b][0])
        while True:
            children = [i for i in range(1, counts[b]) if parents[b][i] == path[-1]]
            found = None
            if case["draft"] and children:
                q = chances("draft_logits", b, path[-1])
                for i in children:
                    if uniforms[b][i] * float(q[tokens[b][i]]) < float(p[tokens[b][i]]):
                        found = i
                        break
                    left = (p - q).clamp_min(0)
                    p = left / left.sum() if float(left.sum()) > 0 else p
            else:
                found = next((i for i in children if tokens[b][i] == token), None)
            if found is None:
                break
            path.append(found)
            p = chances("logits", b, found)
            if not case["draft"]:
                token = drawn(p, uniforms[b][found])
        paths.append(path + [-1] * (case["tokens"] - len(path)))
        lengths.append(len(path))
        following.append(drawn(p, uniforms[b][0]) if case["draft"] else token)
    return [_ints(paths), _ints(lengths), _ints(following)]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotate":
        at = state["positions"].long()
        x = state["x"].view(case["rows"], case["heads"], case["head_size"])
        return _exact_rotated(x, state["weight"] if case["norm"] else None, state["cos"][at], state["sin"][at], case["interleaved"]).flatten(1)
    return {"append": _exact_append, "tree": _exact_tree, "keep": _exact_keep, "verify": _exact_verify}[case["op"]](state)


def work(case):
    op = case["op"]
    if op == "rotate":
        # the heads in and out, a row of the tables for each; a sum of squares, three products, a rotation
        n = case["rows"] * case["heads"] * case["head_size"]
        return {"bytes": 8 * n + case["rows"] * (4 * case["rotary"] + 4) + 4 * case["head_size"], "flops": 8 * n}
    lengths, counts = _lengths(case)
    if op == "verify":
        # the logits behind the token that the walk begins with: every sequence needs those, the drafts decide what else
        rows = case["batch"] * (2 if case["draft"] and case["tokens"] > 1 else 1)
        return {"bytes": 4 * rows * case["vocab"] + 16 * case["batch"] * case["tokens"], "flops": 4 * rows * case["vocab"]}
    row, size = case["kv_heads"] * case["head_size"], case["page_tokens"]
    if op == "keep":
        # of each sequence half of the path on the average is elsewhere: read and written, keys and values, in every layer
        moved = case["batch"] * case["accepted"] / 2
        return {"bytes": int(2 * moved * 2 * row * case["layers"]), "flops": 0}
    width = case["heads"] * case["head_size"]
    if op == "append":
        # queries in and out, new keys and values in, their codes out, and a scale of each page they lie in
        touched = sum((n - 1) // size - (n - c) // size + 1 for n, c in zip(lengths, counts))
        table = sum(counts) * 4 * case["rotary"]
        return {"bytes": sum(counts) * (2 * row * (4 + 1) + 8 * width) + touched * 2 * case["kv_heads"] * 4 + table,
                "flops": sum(counts) * (8 * (width + row) + 4 * row)}
    pages = sum(-(-n // size) for n in lengths)
    # the text before, and of the new tokens about as many as a path is long
    pairs = sum(c * (n - c) + c * max(1, c.bit_length()) for n, c in zip(lengths, counts))
    return {"bytes": 2 * sum(lengths) * row + pages * 2 * case["kv_heads"] * 4 + 4 * width * (sum(counts) + case["batch"] * case["tokens"]),
            "flops": 4 * pairs * width}
