"""The operators of a decoder that keeps its keys and values in 8 bits, as measured cases.

A program that generates or scores text holds the keys and values of every sequence in pages of one pool, 8 bits a number
with a float32 scale for each page and head.  Every step it writes the new tokens' keys and values there ("append"), lets
the new tokens attend to the pages of their sequence ("attention"), and turns the logits into log probabilities of given
tokens, their entropy and the best alternatives ("logprobs").  Between steps it copies pages: a sequence that forks takes
its last page along, and a pool that has become sparse is compacted ("pages").

Everything a step takes and gives is float32 or int32, the types of the runtime.

A page of the pool is [2 (keys, values)][kv_heads][page_tokens][head_size] int8, its scales [2][kv_heads] float32; a number
is code * scale.  A page table row names the pages of one sequence in order.  `lengths` counts the tokens of each sequence
with the new ones, `counts` the new ones, which are the last; rows of a call behind a sequence's count are padding.
"""
import functools
import math

import torch

own = False

_SPREAD = 40.0        # standard deviation of the codes: +-127 is about three of them


def listed():
    return [
        # one conversation, the next token: launches and latency are all there is
        dict(name="attention_1x700", op="attention", batch=1, tokens=1, shortest=700, longest=700, heads=16, kv_heads=4,
             head_size=64, page_tokens=16),
        # a serving batch of uneven conversations, one token each, four query heads to a key head
        dict(name="attention_48x4100", op="attention", batch=48, tokens=1, shortest=1, longest=4100, heads=32, kv_heads=8,
             head_size=128, page_tokens=64),
        # a few long documents, every query head with its own keys
        dict(name="attention_3x40001", op="attention", batch=3, tokens=1, shortest=12000, longest=40001, heads=16,
             kv_heads=16, head_size=128, page_tokens=128),
        # drafts of up to five tokens that are checked at once
        dict(name="attention_20x1500_5", op="attention", batch=20, tokens=5, shortest=100, longest=1500, heads=24,
             kv_heads=8, head_size=64, page_tokens=32),
        # prompts, the later part of them behind pages that are there already
        dict(name="attention_prompt_3x900", op="attention", batch=3, tokens=900, shortest=450, longest=1800, heads=16,
             kv_heads=4, head_size=128, page_tokens=64),
        # the new token of each sequence of a batch
        dict(name="append_64x1", op="append", batch=64, tokens=1, shortest=5, longest=3000, kv_heads=8, head_size=128,
             page_tokens=64),
        # prompts of uneven lengths
        dict(name="append_6x1999", op="append", batch=6, tokens=1999, shortest=800, longest=2500, kv_heads=8,
             head_size=128, page_tokens=32),
        # four sequences fork: the partly filled page of each, in all layers
        dict(name="pages_fork_4", op="pages", count=4, pages=200, layers=12, kv_heads=4, head_size=64, page_tokens=32),
        # a pool is compacted
        dict(name="pages_compact_150", op="pages", count=150, pages=400, layers=24, kv_heads=8, head_size=128,
             page_tokens=64),
        # the next token of one sequence
        dict(name="logprobs_1x32000", op="logprobs", rows=1, vocab=32000, pad=0, top=5, masked=0.0),
        # a batch of beams, some tokens ruled out
        dict(name="logprobs_36x100003", op="logprobs", rows=36, vocab=100003, pad=1, top=20, masked=0.3),
        # scoring of given texts
        dict(name="logprobs_3000x50001", op="logprobs", rows=3000, vocab=50001, pad=3, top=1, masked=0.0),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "pages", "logprobs"])
    if op == "logprobs":
        vocab = _log(rng, 300, 200000)
        return dict(op=op, rows=_log(rng, 1, max(1, min(4096, 120_000_000 // vocab))), vocab=vocab, pad=rng.randint(0, 5),
                    top=rng.choice([0, 1, 3, 8, 20, 32]), masked=rng.choice([0.0, 0.0, 0.5]))
    kv_heads, head_size = rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([32, 64, 128])
    page_tokens = rng.choice([16, 32, 64, 128])
    if op == "pages":
        page = 2 * kv_heads * page_tokens * head_size
        layers = rng.randint(1, 32)
        count = _log(rng, 1, max(1, min(300, 400_000_000 // (page * layers))))
        return dict(op=op, count=count, pages=2 * count + _log(rng, 1, 200), layers=layers, kv_heads=kv_heads,
                    head_size=head_size, page_tokens=page_tokens)
    width = kv_heads * head_size
    if op == "append":
        tokens = rng.choice([1, _log(rng, 1, 2048)])
        batch = _log(rng, 1, max(1, min(128, 9_000_000 // (tokens * width))))
        longest = tokens + _log(rng, 1, 2000)
        return dict(op=op, batch=batch, tokens=tokens, shortest=min(longest, tokens // 2 + 1), longest=longest,
                    kv_heads=kv_heads, head_size=head_size, page_tokens=page_tokens)
    group = rng.choice([1, 2, 3, 4, 6, 8, 12])
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 16, 512)])
    longest = tokens + _log(rng, 1, 40000 if tokens == 1 else 2000)
    batch = _log(rng, 1, max(1, min(64, 100_000_000 // (longest * width),
                                    2_000_000_000 // (tokens * longest * width * group))))
    return dict(op=op, batch=batch, tokens=tokens, shortest=rng.randint(max(1, tokens // 2), longest), longest=longest,
                heads=group * kv_heads, kv_heads=kv_heads, head_size=head_size, page_tokens=page_tokens)


def _lengths(case):
    """(tokens of each sequence, new ones of them): spread evenly between the shortest and the longest."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    lengths = [hi - (hi - lo) * i // max(b - 1, 1) for i in range(b)]
    # the last sequences bring fewer new tokens than the call has room for
    counts = [min(n, max(1, case["tokens"] - (case["tokens"] * i) // (2 * b))) for i, n in enumerate(lengths)]
    return lengths, counts


# ------------------------------------------------------------------------------------------------ what a program has
def _pool(case, g):
    """Codes and scales of a pool, and a page table of it: pages in no order, -1 behind a sequence's last."""
    lengths, counts = _lengths(case)
    need = [-(-n // case["page_tokens"]) for n in lengths]
    pages = sum(need) + 7
    shape = (pages + 1, 2, case["kv_heads"], case["page_tokens"], case["head_size"])   # the last page is in no table
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    for part in codes.split(max(1, (1 << 26) // codes[0].numel())):
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * _SPREAD).round_().clamp_(-127, 127))
    scales = torch.exp(0.3 * torch.randn(shape[:3], generator=g, device="cuda")) / _SPREAD
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], max(need) + 3), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(codes=codes, scales=scales, table=table, lengths=as_int(lengths), counts=as_int(counts))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "attention":
        state.update(_pool(case, g))
        state["q"] = randn(case["batch"], case["tokens"], case["heads"] * case["head_size"])
        state["y"] = torch.empty_like(state["q"])
    elif case["op"] == "append":
        state.update(_pool(case, g))
        width = case["kv_heads"] * case["head_size"]
        state["k"], state["v"] = (randn(case["batch"], case["tokens"], width) for _ in range(2))
    elif case["op"] == "pages":
        shape = (case["layers"], case["pages"], 2, case["kv_heads"], case["page_tokens"], case["head_size"])
        state["codes"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        state["scales"] = torch.rand(shape[:4], generator=g, device="cuda") / _SPREAD
        order = torch.randperm(case["pages"], generator=g, device="cuda")[:2 * case["count"]].tolist()
        state["sources"], state["targets"] = order[::2], order[1::2]
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = randn(rows, vocab + case["pad"]) * 3
        if case["masked"]:
            logits[torch.rand(logits.shape, generator=g, device="cuda") < case["masked"]] = -math.inf
        state["logits"] = logits
        state["tokens"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        state["logprob"], state["entropy"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        state["top_ids"] = torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda")
        state["top_logprobs"] = torch.empty((rows, case["top"]), device="cuda")
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
        pages = case["pages"] if case["op"] == "pages" else state["codes"].shape[0] - 1
        words = [layers, pages, 2, case["kv_heads"], case["page_tokens"], case["head_size"] // 4]   # four codes each
        state["cache"] = PagedCache(context, layers, pages, case["kv_heads"], case["head_size"], case["page_tokens"],
                                    codes=tensor(state["codes"], words), scales=tensor(state["scales"], words[:4]))


def _run_own(state):
    op, t = state["case"]["op"], state["own"]
    if op == "attention":
        state["cache"].attention(0, t["q"], t["table"], t["lengths"], t["counts"], out=t["y"])
    elif op == "append":
        state["cache"].append(0, t["k"], t["v"], t["table"], t["lengths"], t["counts"])
    elif op == "pages":
        state["cache"].copy_pages(state["sources"], state["targets"])
    else:
        _context().token_logprobs(t["logits"], t["tokens"], state["case"]["top"], vocab=state["case"]["vocab"],
                                  out=(t["logprob"], t["entropy"], t["top_ids"], t["top_logprobs"]))


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_attention(state):
    case, table = state["case"], state["table"].long().clamp_min(0)
    b, n, h, d = case["batch"], case["tokens"], case["kv_heads"], case["head_size"]
    keys, values = ((state["codes"][table, i].float() * state["scales"][table, i][..., None, None])
                    .transpose(1, 2).reshape(b, h, -1, d) for i in (0, 1))            # [batch, kv head, token, channel]
    group = case["heads"] // h
    q = state["q"].view(b, n, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, n * group, d)
    scores = (q @ keys.transpose(2, 3)) / math.sqrt(d)
    lengths, counts = state["lengths"].long(), state["counts"].long()
    at = (lengths - counts)[:, None] + torch.arange(n, device="cuda")                  # a query's own place
    seen = torch.arange(keys.shape[2], device="cuda") <= at[..., None]
    seen &= (torch.arange(n, device="cuda") < counts[:, None])[..., None]
    seen = seen[:, None, :, None].expand(b, 1, n, group, keys.shape[2]).reshape(b, 1, n * group, -1)
    scores = scores.masked_fill(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    y = (weights @ values) / weights.sum(-1, keepdim=True).clamp_min(1e-30)
    return y.view(b, h, n, group, d).permute(0, 2, 1, 3, 4).reshape(b, n, -1)


def _plain_append(state):
    case = state["case"]
    b, n, h, d, size = case["batch"], case["tokens"], case["kv_heads"], case["head_size"], case["page_tokens"]
    spare = state["codes"].shape[0] - 1
    start = state["lengths"].long() - state["counts"].long()
    slots = (n + size - 2) // size + 1                                                 # pages a sequence may touch
    page = start[:, None] // size + torch.arange(slots, device="cuda")                 # [batch, slot]
    token = (page * size - start[:, None])[..., None] + torch.arange(size, device="cuda")      # which new one is there
    new = (token >= 0) & (token < state["counts"].long()[:, None, None])
    touched = new.any(-1)
    kept = (page * size < start[:, None])                                              # the page holds older tokens
    ids = torch.where(touched, state["table"].long().gather(1, page.clamp_max(state["table"].shape[1] - 1)), spare)
    x = torch.stack([state["k"], state["v"]]).view(2, b, n, h, d)
    x = x[:, torch.arange(b, device="cuda")[:, None, None], token.clamp(0, n - 1)]     # [2, batch, slot, token, head, d]
    x = x.permute(1, 2, 0, 4, 3, 5)                                                    # like a page: [.., 2, head, token, d]
    is_new, is_old = new[:, :, None, None, :, None], ~new[:, :, None, None, :, None]
    top = torch.full((), 127.0, device="cuda")
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


def _plain_pages(state):
    for name in ("codes", "scales"):
        state[name][:, state["targets"]] = state[name][:, state["sources"]]


def _plain_logprobs(state):
    case = state["case"]
    x = state["logits"][:, :case["vocab"]]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    logs = x - top - torch.log(total)
    logprob = logs.gather(1, state["tokens"].long()[:, None])[:, 0]
    entropy = -torch.where(e > 0, e * logs, 0.0).sum(1) / total[:, 0]
    # a key that orders by value, then by the lower index
    bits = (x + 0.0).contiguous().view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32
    key += torch.arange(case["vocab"] - 1, -1, -1, device="cuda")
    ids = case["vocab"] - 1 - (key.topk(case["top"], 1).values & 0xffffffff)
    return [logprob, entropy, ids.int(), logs.gather(1, ids)]


def run(state):
    op = state["case"]["op"]
    if own:
        _run_own(state)
        result = [state[n] for n in ("logprob", "entropy", "top_ids", "top_logprobs")] if op == "logprobs" else state.get("y")
    else:
        result = {"attention": _plain_attention, "append": _plain_append, "pages": _plain_pages,
                  "logprobs": _plain_logprobs}[op](state)
    if op == "append":
        # the pool as it stands now, as codes in units of the page's scale and those scales; without the page of no table
        return [state["codes"][:-1], state["scales"][:-1]]
    return [state["codes"], state["scales"]] if op == "pages" else result


# ------------------------------------------------------------------------------------------------ from the definitions
def _exact_attention(state):
    case = state["case"]
    size, h, d = case["page_tokens"], case["kv_heads"], case["head_size"]
    out = torch.zeros(state["y"].shape, dtype=torch.float64, device="cuda")
    for b, (length, count) in enumerate(zip(*_lengths(case))):
        ids = state["table"][b, :-(-length // size)].long()
        page = state["codes"][ids].double() * state["scales"][ids].double()[..., None, None]
        k, v = (page[:, i].permute(1, 0, 2, 3).reshape(h, -1, d)[:, :length] for i in (0, 1))
        causal = torch.ones(count, length, dtype=torch.bool, device="cuda").tril(length - count)
        for head in range(case["heads"]):
            q = state["q"][b, :count, head * d:(head + 1) * d].double()
            s = (q @ k[head * h // case["heads"]].T * d ** -0.5).masked_fill(~causal, -math.inf)
            out[b, :count, head * d:(head + 1) * d] = torch.softmax(s, -1) @ v[head * h // case["heads"]]
    return out


def _exact_append(state):
    case = state["case"]
    size, h, d = case["page_tokens"], case["kv_heads"], case["head_size"]
    scales = state["scales"].double()
    for b, (length, count) in enumerate(zip(*_lengths(case))):
        start = length - count
        for p in range(start // size, (length - 1) // size + 1):
            lo, hi = max(start, p * size), min(length, (p + 1) * size)
            page = int(state["table"][b, p])
            for i, name in enumerate("kv"):
                peak = state[name][b, lo - start:hi - start].double().view(-1, h, d).abs().amax((0, 2)) / 127
                scales[page, i] = torch.maximum(scales[page, i], peak) if lo > p * size else peak
    return [None, scales[:-1]]     # (codes are whole numbers, rounded by the 32-bit scale that stands beside them)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(state)
    if case["op"] == "append":
        return _exact_append(state)
    if case["op"] == "pages":
        scales = state["scales"].double()
        for s, t in zip(state["sources"], state["targets"]):
            scales[:, t] = scales[:, s]
        return [None, scales]
    logprob, entropy, best = [], [], []
    for row, token in zip(state["logits"], state["tokens"].tolist()):
        p = torch.log_softmax(row[:case["vocab"]].double(), 0)
        some = p[p > -math.inf]
        logprob.append(p[token])
        entropy.append(-(some.exp() * some).sum())
        best.append(p.topk(case["top"]).values)
    return [torch.stack(logprob), torch.stack(entropy), None, torch.stack(best)]


def work(case):
    op = case["op"]
    if op == "logprobs":
        # the logits once; a maximum, a difference, an exponential and two sums of each
        return {"bytes": 4 * case["rows"] * (case["vocab"] + 3 + 2 * case["top"]), "flops": 6 * case["rows"] * case["vocab"]}
    page = 2 * case["kv_heads"] * (case["page_tokens"] * case["head_size"] + 4)
    if op == "pages":
        return {"bytes": 2 * case["count"] * case["layers"] * page, "flops": 0}
    lengths, counts = _lengths(case)
    row = case["kv_heads"] * case["head_size"]
    if op == "append":
        # new keys and values in, their codes out, and a scale of each page they lie in
        touched = sum((n - 1) // case["page_tokens"] - (n - c) // case["page_tokens"] + 1 for n, c in zip(lengths, counts))
        return {"bytes": 2 * sum(counts) * row * (4 + 1) + touched * 2 * case["kv_heads"] * 4, "flops": 4 * sum(counts) * row}
    pages = sum(-(-n // case["page_tokens"]) for n in lengths)
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lengths, counts))
    width = case["heads"] * case["head_size"]
    return {"bytes": 2 * sum(lengths) * row + pages * 2 * case["kv_heads"] * 4 + 4 * width * (sum(counts) + case["batch"] * case["tokens"]),
            "flops": 4 * pairs * width}
