"""Attention over a paged cache of keys and values, and what belongs to it: the plain forms of the operators, and their workloads.

A decoder keeps the keys and values of its tokens in pages. Every step appends the new tokens' rows (`append`), reads back the recent
ones in full (`attention`), reads of the far ones those that a search over the keys named (`attend_candidates`), and joins the two reads
(`merge_parts`). A slot is a token's place in the cache: page * page_size + place in the page; it is the source id under which the
token's key is in the search index.

`own` chooses between the plain forms (elementary operations in 32 bits) and the framework's entry points.
"""
import math

import torch

own = False

_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
_TYPE = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_NONE = 2**63 - 1  # the id that a search gives where it found fewer rows than it was asked for


def _append(name, dtype, n_sequences, n_tokens, heads, group, dim, rotated, page_size, *, far, interleaved=False, padding=0):
    """`rotated`: how many of the columns the rotation turns; `far`: positions begin below this; `padding`: trailing tokens without a
    position, as in a batch that is padded to a fixed size."""
    return {"name": name, "op": "append", "dtype": dtype, "n_sequences": n_sequences, "n_tokens": n_tokens, "heads": heads,
            "group": group, "dim": dim, "rotated": rotated, "page_size": page_size, "far": far, "interleaved": interleaved,
            "padding": padding}


def _attention(name, dtype, n_sequences, longest, heads, group, dim, page_size, *, window=0, kept=1.0, empty=0):
    """`window`: only so many last positions are attended (0: all); `kept` < 1: a bitset filter lets that fraction of the slots
    through; `empty`: so many of the sequences have no token."""
    return {"name": name, "op": "attention", "dtype": dtype, "n_sequences": n_sequences, "longest": longest, "heads": heads,
            "group": group, "dim": dim, "page_size": page_size, "window": window, "kept": kept, "empty": empty}


def _candidates(name, dtype, n_tokens, n_candidates, n_slots, heads, group, dim, page_size, *, missing=0):
    """`missing`: so many of the last candidates of every other list are the search's "no such neighbour"."""
    return {"name": name, "op": "candidates", "dtype": dtype, "n_tokens": n_tokens, "n_candidates": n_candidates,
            "n_slots": n_slots, "heads": heads, "group": group, "dim": dim, "page_size": page_size, "missing": missing}


def _merge(name, dtype, n_parts, n_tokens, n_heads, dim, *, empty=0.0):
    """`empty`: the share of the parts' rows that attended to nothing."""
    return {"name": name, "op": "merge", "dtype": dtype, "n_parts": n_parts, "n_tokens": n_tokens, "n_heads": n_heads, "dim": dim,
            "empty": empty}


def listed():
    return [
        # a step of eight requests: one new token each, the latency of the call
        _append("append 8 new tokens", "bfloat16", 8, 8, 8, 4, 128, 128, 16, far=30_000),
        # the prompts of several requests in one go
        _append("append 20k prompt tokens", "float16", 7, 20_000, 8, 4, 128, 128, 64, far=4000),
        # full precision, adjacent pairs, half of the columns rotated, far positions, pages of 24, a padded batch
        _append("append 3k tokens, f32", "float32", 5, 3001, 3, 3, 96, 48, 24, far=1_000_000, interleaved=True, padding=9),
        # one request with a short context: latency
        _attention("one request, 1.5k tokens", "float16", 1, 1500, 8, 4, 128, 16),
        # a batch of requests of very different lengths
        _attention("32 requests up to 16k", "bfloat16", 32, 16_384, 8, 8, 128, 16),
        # one very long context, seven query heads to a key head
        _attention("one request, 250k tokens", "float16", 1, 250_001, 4, 7, 128, 64),
        # full precision, every head with keys of its own, a window, pages of 20, erased slots, an empty request
        _attention("f32, window, filter", "float32", 9, 9000, 12, 1, 64, 20, window=4000, kept=0.75, empty=1),
        # the rows that a search named for one new token: latency
        _candidates("one token, 100 candidates", "float16", 1, 100, 100_000, 8, 4, 128, 16),
        # a batch of tokens, a thousand candidates for every query head
        _candidates("64 tokens, 1000 candidates", "bfloat16", 64, 1000, 400_000, 8, 4, 128, 16, missing=50),
        # full precision, rows of 96, lists that are not full
        _candidates("16 tokens, 333 candidates, f32", "float32", 16, 333, 100_003, 3, 3, 96, 7, missing=33),
        # the recent tokens' part and the candidates' part of one step
        _merge("merge 2 parts of 8 tokens", "float16", 2, 8, 32, 128, empty=0.1),
        # the parts of a cache that is dealt out over eight GPUs, for a large batch
        _merge("merge 8 parts of 4k tokens", "bfloat16", 8, 4096, 32, 128),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    size = _SIZE[dtype]
    op = rng.choice(["append", "attention", "attention", "candidates", "merge"])
    dim = rng.choice([32, 48, 64, 72, 80, 96, 104, 112, 128, 128, 160, 192, 256])
    if size == 4:
        dim = rng.choice([dim, dim - 4])
    heads = rng.choice([1, 2, 3, 4, 5, 8, 12])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    page_size = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 128, 256])
    case = None
    if op == "append":
        most = 240_000_000 // (size * dim * heads * (group + 2))
        n_tokens = _spread(rng, 1, max(2, min(20_000, most)))
        rotated = rng.choice([dim, dim, 2 * (dim // 4), 2 * rng.randint(1, dim // 2)])
        case = _append("", dtype, rng.randint(1, min(64, n_tokens)), n_tokens, heads, group, dim, rotated, page_size,
                       far=_spread(rng, 1, 1_000_000), interleaved=rng.random() < 0.5, padding=rng.choice([0, 0, min(3, n_tokens - 1)]))
    elif op == "attention":
        n_sequences = _spread(rng, 1, 64)
        # no more bytes and products than the largest listed case, were all sequences of the longest one's length
        most = 880_000_000 // (n_sequences * heads * dim * max(2 * size, group // 2))
        longest = _spread(rng, 1, max(2, min(200_000, most)))
        case = _attention("", dtype, n_sequences, longest, heads, group, dim, page_size,
                          window=rng.choice([0, 0, 0, rng.randint(1, longest)]), kept=rng.choice([1.0, 1.0, 0.5, 0.9]),
                          empty=rng.choice([0, 0, 1]) if n_sequences > 1 else 0)
    elif op == "candidates":
        n_candidates = _spread(rng, 1, 2000)
        most = 370_000_000 // (size * n_candidates * heads * group * dim)
        n_slots = _spread(rng, n_candidates, max(n_candidates, min(400_000, 1_600_000_000 // (size * heads * dim))))
        case = _candidates("", dtype, _spread(rng, 1, max(2, min(128, most))), n_candidates, n_slots, heads, group, dim, page_size,
                           missing=rng.choice([0, n_candidates // 3, n_candidates]))
    else:
        n_parts = rng.randint(1, 16)
        n_heads = heads * group
        most = 300_000_000 // (size * (n_parts + 1) * n_heads * (dim + 2))
        case = _merge("", dtype, n_parts, _spread(rng, 1, max(2, min(8192, most))), n_heads, dim, empty=rng.choice([0.0, 0.3]))
    del case["name"]
    return case


def _lengths(case):
    """The lengths of a batch's sequences, longest first: the longest, then ever shorter ones; the last `empty` of them are 0."""
    b = case["n_sequences"]
    return [0 if i >= b - case["empty"] else max(1, int(case["longest"] * (1 - i / b) ** 1.5)) for i in range(b)]


def _table_width(case):
    return -(-case["longest"] // case["page_size"])


def _cache(case, n_pages, g):
    """A cache as a program lays it out: the tokens of a page that belong to one head lie together."""
    shape = (n_pages, case["heads"], case["page_size"], case["dim"])
    keys, values = (torch.randn(shape, generator=g, device="cuda", dtype=_TYPE[case["dtype"]]) for _ in range(2))
    return keys.permute(0, 2, 1, 3), values.permute(0, 2, 1, 3)


def _prepare_append(case, g):
    b, t, ps = case["n_sequences"], case["n_tokens"], case["page_size"]
    dtype = _TYPE[case["dtype"]]
    each = -(-t // b)
    pages_each = each // ps + 2
    keys, values = _cache(case, b * pages_each + 3, g)
    start = torch.randint(0, case["far"], (b,), generator=g, device="cuda")
    sequences = torch.arange(t, device="cuda") * b // t
    first = -(-(torch.arange(b, device="cuda") * t) // b)
    positions = start[sequences] + torch.arange(t, device="cuda") - first[sequences]
    if case["padding"]:
        positions[t - case["padding"]:] = -1
    width = (case["far"] + each) // ps + 3
    order = torch.randperm(b * pages_each + 3, generator=g, device="cuda")[:b * pages_each].view(b, pages_each)
    pages = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    pages.scatter_(1, start[:, None] // ps + torch.arange(pages_each, device="cuda"), order.int())
    heads, queries = case["heads"], case["heads"] * case["group"]
    # what a fused projection leaves: the rows of queries, keys and values side by side
    rows = torch.randn((t, queries + 2 * heads, case["dim"]), generator=g, device="cuda", dtype=dtype)
    half = case["rotated"] // 2
    frequencies = torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
    return {"case": case, "keys": keys, "values": values, "queries": rows[:, :queries], "new_keys": rows[:, queries:queries + heads],
            "new_values": rows[:, queries + heads:], "sequences": sequences.int(), "positions": positions.int(), "pages": pages,
            "frequencies": frequencies}


def _prepare_attention(case, g):
    ps = case["page_size"]
    longest_first = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    lengths = longest_first[torch.randperm(case["n_sequences"], generator=g, device="cuda")]
    used = (lengths + ps - 1) // ps
    n_pages = sum(-(-n // ps) for n in _lengths(case)) + 2
    keys, values = _cache(case, n_pages, g)
    # pages were handed out as requests came and went: in no order
    column = torch.arange(_table_width(case), device="cuda")
    rank = (used.cumsum(0) - used)[:, None] + column
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    pages = torch.where(column < used[:, None], order[rank.clamp(max=n_pages - 1)], -1)
    # a head's queries and keys are not independent: some of the keys answer to it
    queries = 1.5 * torch.randn((case["n_sequences"], case["heads"] * case["group"], case["dim"]), generator=g, device="cuda")
    bits = None
    if case["kept"] < 1.0:
        keep = torch.rand((-(-n_pages * ps // 32), 32), generator=g, device="cuda") < case["kept"]
        bits = (keep.long() << torch.arange(32, device="cuda")).sum(1).to(torch.uint32)
    return {"case": case, "keys": keys, "values": values, "queries": queries.to(_TYPE[case["dtype"]]), "pages": pages,
            "lengths": lengths, "window": case["window"] or None, "filter": bits}


def _prepare_candidates(case, g):
    n_pages = -(-case["n_slots"] // case["page_size"])
    keys, values = _cache(case, n_pages, g)
    n, n_heads, k = case["n_tokens"], case["heads"] * case["group"], case["n_candidates"]
    # best first, as a search gives them; which slots they are is as good as random
    candidates = torch.randint(0, case["n_slots"], (n, n_heads, k), generator=g, device="cuda")
    if case["missing"]:
        candidates.view(-1, k)[::2, k - case["missing"]:] = _NONE
    queries = 1.5 * torch.randn((n, n_heads, case["dim"]), generator=g, device="cuda")
    return {"case": case, "keys": keys, "values": values, "queries": queries.to(_TYPE[case["dtype"]]), "candidates": candidates}


def _prepare_merge(case, g):
    shape = (case["n_parts"], case["n_tokens"], case["n_heads"], case["dim"])
    parts = torch.randn(shape, generator=g, device="cuda", dtype=_TYPE[case["dtype"]])
    lse = 8.0 + 2.0 * torch.randn(shape[:3], generator=g, device="cuda")
    if case["empty"]:
        nothing = torch.rand(shape[:3], generator=g, device="cuda") < case["empty"]
        lse = lse.masked_fill(nothing, -math.inf)
        parts = parts.masked_fill(nothing[..., None], 0.0)
    return {"case": case, "parts": parts, "lse": lse}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "candidates": _prepare_candidates,
            "merge": _prepare_merge}[case["op"]](case, g)


# ---- plain forms --------------------------------------------------------------------------------------------------------------

def _rotate(x, positions, frequencies, interleaved):
    """Pairs of columns turned by position * frequency; rows without a position and columns behind the pairs stay."""
    half = frequencies.shape[0]
    angle = positions.double()[:, None] * frequencies
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float()
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
    else:
        a, b = y[..., :half], y[..., half:2 * half]
    u, v = a * c - b * s, b * c + a * s
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    turned = torch.cat((turned, y[..., 2 * half:]), -1)
    return torch.where(positions[:, None, None] >= 0, turned, y).to(x.dtype)


def _plain_append(s):
    ps = s["keys"].shape[1]
    positions = s["positions"].long()
    known = positions >= 0
    page = s["pages"][s["sequences"].long(), positions.clamp(min=0) // ps].long()
    slots = torch.where(known, page * ps + positions % ps, -1)
    keys = _rotate(s["new_keys"], s["positions"], s["frequencies"], s["case"]["interleaved"])
    queries = _rotate(s["queries"], s["positions"], s["frequencies"], s["case"]["interleaved"])
    at = slots[known]
    s["keys"][at // ps, at % ps] = keys[known]
    s["values"][at // ps, at % ps] = s["new_values"][known]
    return {"keys": s["keys"], "values": s["values"], "slots": slots, "queries": queries}


def _softmax_sum(scores, allowed, values, equation):
    """Sum of the value rows by the softmax of the allowed scores, and the logarithm of its denominator."""
    scores = scores.masked_fill(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = torch.einsum(equation, weights / torch.where(total == 0, 1.0, total), values)
    return out, (top + torch.log(total)).squeeze(-1)


def _plain_attention(s):
    case, queries = s["case"], s["queries"]
    b, n_heads, dim = queries.shape
    heads, ps = s["keys"].shape[2], s["keys"].shape[1]
    position = torch.arange(s["pages"].shape[1] * ps, device="cuda")
    lengths = s["lengths"].long()[:, None]
    page = s["pages"][:, position // ps].long()
    allowed = (position < lengths) & (page >= 0)
    if s["window"]:
        allowed &= position >= lengths - s["window"]
    page = page.clamp(min=0)
    if s["filter"] is not None:
        slot = page * ps + position % ps
        allowed &= (s["filter"].to(torch.int64)[slot // 32] >> (slot % 32) & 1).bool()
    keys = s["keys"][page, position % ps].float()
    scores = torch.einsum("bhgd,blhd->bhgl", queries.float().view(b, heads, -1, dim), keys) / math.sqrt(dim)
    del keys
    values = s["values"][page, position % ps].float()
    out, lse = _softmax_sum(scores, allowed[:, None, None], values, "bhgl,blhd->bhgd")
    return out.reshape(b, n_heads, dim).to(queries.dtype), lse.reshape(b, n_heads)


def _plain_candidates(s):
    queries, candidates = s["queries"], s["candidates"]
    n, n_heads, dim = queries.shape
    n_pages, ps, heads, _ = s["keys"].shape
    allowed = (candidates >= 0) & (candidates < n_pages * ps)
    slot = torch.where(allowed, candidates, 0)
    head = (torch.arange(n_heads, device="cuda") // (n_heads // heads))[:, None]
    keys = s["keys"][slot // ps, slot % ps, head].float()
    scores = torch.einsum("nhd,nhkd->nhk", queries.float(), keys) / math.sqrt(dim)
    del keys
    values = s["values"][slot // ps, slot % ps, head].float()
    out, lse = _softmax_sum(scores, allowed, values, "nhk,nhkd->nhd")
    return out.to(queries.dtype), lse


def _plain_merge(s):
    lse = s["lse"]
    top = lse.amax(0)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(lse - top)
    total = weights.sum(0)
    weights = weights / torch.where(total == 0, 1.0, total)
    out = (weights[..., None] * s["parts"].float().masked_fill(weights[..., None] == 0, 0.0)).sum(0)
    return out.to(s["parts"].dtype), top + torch.log(total)


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        from cuvs_b200 import kv_cache
        if op == "append":
            slots, queries = kv_cache.append(state["keys"], state["values"], state["new_keys"], state["new_values"], state["pages"],
                                             state["positions"], sequences=state["sequences"], queries=state["queries"],
                                             frequencies=state["frequencies"], interleaved=state["case"]["interleaved"], sync=False)
            return {"keys": state["keys"], "values": state["values"], "slots": slots, "queries": queries}
        if op == "attention":
            return kv_cache.attention(state["keys"], state["values"], state["queries"], state["pages"], state["lengths"],
                                      window=state["window"], filter=state["filter"], sync=False)
        if op == "candidates":
            return kv_cache.attend_candidates(state["keys"], state["values"], state["queries"], state["candidates"], sync=False)
        return kv_cache.merge_parts(state["parts"], state["lse"], sync=False)
    return {"append": _plain_append, "attention": _plain_attention, "candidates": _plain_candidates, "merge": _plain_merge}[op](state)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "append":
        t, half = case["n_tokens"], case["rotated"] // 2
        heads, n_heads = case["heads"], case["heads"] * case["group"]
        return {"bytes": 2 * t * (n_heads + 2 * heads) * case["dim"] * size + 16 * t + 8 * half,
                "flops": t * half * (6 * (n_heads + heads) + 3)}
    if case["op"] == "attention":
        attended = sum(min(n, case["window"] or n) for n in _lengths(case)) * case["kept"]
        heads, n_heads = case["heads"], case["heads"] * case["group"]
        rows = case["n_sequences"] * n_heads
        return {"bytes": int(2 * attended * heads * case["dim"] * size) + rows * (2 * case["dim"] * size + 4),
                "flops": int(4 * attended * n_heads * case["dim"])}
    if case["op"] == "candidates":
        n_heads = case["heads"] * case["group"]
        lists = case["n_tokens"] * n_heads
        n = lists * case["n_candidates"] - (lists + 1) // 2 * case["missing"]
        # a row that several lists name is read once: so many different rows of a head do n / heads random names reach
        rows = case["heads"] * case["n_slots"] * -math.expm1(-n / case["heads"] / case["n_slots"])
        return {"bytes": int(2 * rows * case["dim"] * size) + 8 * lists * case["n_candidates"] + lists * (2 * case["dim"] * size + 4),
                "flops": 4 * n * case["dim"]}
    rows = case["n_tokens"] * case["n_heads"]
    return {"bytes": (case["n_parts"] + 1) * rows * (case["dim"] * size + 4), "flops": 2 * case["n_parts"] * rows * case["dim"]}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _exact_append(s):
    """A pair of columns is a complex number, its rotation a product with exp(i * position * frequency)."""
    keys, values = s["keys"].double(), s["values"].double()
    ps, half = keys.shape[1], s["frequencies"].shape[0]
    turned = {}
    for name in ("new_keys", "queries"):
        x = s[name].double()
        pairs = x[..., :2 * half]
        pairs = pairs.unflatten(-1, (half, 2)) if s["case"]["interleaved"] else pairs.unflatten(-1, (2, half)).transpose(-1, -2)
        angle = torch.outer(s["positions"].clamp(min=0).double(), s["frequencies"])
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None])
        x[..., :2 * half] = z.flatten(-2) if s["case"]["interleaved"] else z.transpose(-1, -2).flatten(-2)
        turned[name] = x
    place = s["positions"].long()
    real = (place >= 0).nonzero()[:, 0]
    page = s["pages"][s["sequences"][real].long(), place[real] // ps].long()
    keys[page, place[real] % ps] = turned["new_keys"][real]
    values[page, place[real] % ps] = s["new_values"][real].double()
    return {"keys": keys, "values": values, "slots": None, "queries": turned["queries"]}


def _exact_rows(query, keys, values):
    """query [h, d], keys and values [n, h, d] -> [h, d], [h]"""
    scores = (keys * query).sum(-1) / math.sqrt(query.shape[-1])
    lse = torch.logsumexp(scores, 0)
    return (torch.exp(scores - lse)[..., None] * values).sum(0), lse


def _exact_attention(s):
    queries = s["queries"].double()
    b, n_heads, dim = queries.shape
    ps, heads = s["keys"].shape[1], s["keys"].shape[2]
    out = torch.zeros((b, heads, n_heads // heads, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((b, heads, n_heads // heads), -math.inf, dtype=torch.float64, device="cuda")
    words = None if s["filter"] is None else s["filter"].to(torch.int64)
    for i, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(max(0, n - (s["window"] or n)), n, device="cuda")
        slot = s["pages"][i, at // ps].long() * ps + at % ps
        if words is not None:
            slot = slot[(words[slot // 32] >> (slot % 32)) % 2 == 1]
        if slot.numel() == 0:
            continue
        keys, values = (s[name][slot // ps, slot % ps].double() for name in ("keys", "values"))
        for j in range(n_heads // heads):
            out[i, :, j], lse[i, :, j] = _exact_rows(queries[i].view(heads, -1, dim)[:, j], keys, values)
    return out.view(b, n_heads, dim), lse.view(b, n_heads)


def _exact_candidates(s):
    queries, candidates = s["queries"].double(), s["candidates"]
    n, n_heads, dim = queries.shape
    n_pages, ps, heads, _ = s["keys"].shape
    head = torch.arange(n_heads, device="cuda").div(n_heads // heads, rounding_mode="floor")
    out, lse = torch.zeros_like(queries), torch.full((n, n_heads), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(n):
        there = candidates[i] < n_pages * ps
        slot = candidates[i].clamp(max=n_pages * ps - 1).t()
        keys, values = (s[name][slot // ps, slot % ps, head].double() for name in ("keys", "values"))
        scores = (keys * queries[i]).sum(-1) / math.sqrt(dim)
        scores[~there.t()] = -math.inf
        lse[i] = torch.logsumexp(scores, 0)
        full = lse[i] > -math.inf
        out[i, full] = (torch.exp(scores[:, full] - lse[i, full])[..., None] * values[:, full]).sum(0)
    return out, lse


def _exact_merge(s):
    lse = torch.logsumexp(s["lse"].double(), 0)
    share = torch.exp(s["lse"].double() - lse).nan_to_num(0.0)
    return torch.einsum("pnh,pnhd->nhd", share, s["parts"].double()), lse


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "candidates": _exact_candidates,
            "merge": _exact_merge}[case["op"]](prepare(case, seed))
