"""Drafted tokens over a paged cache of keys and values: the plain forms of the operators, and their workloads.

A decoder that drafts a tree of tokens per sequence checks all of them in one step. The tree's parents become ancestors' bits and positions
(`draft_tree`), the tokens' rows are appended at places of their own but turned by the positions that they would have (`append` with `turns`,
which also turns images' and videos' tokens by several axes), every drafted token attends to its sequence's tokens and to its ancestors
(`attend_tree`), the rows of the path that was accepted move up to follow the sequence (`keep_path`), and where a sequence goes on in several
ways its last page is copied (`copy_pages`).

`own` chooses between the plain forms (elementary operations in 32 bits) and the framework's entry points.
"""
import math

import torch

own = False

_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
_TYPE = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def _tree(name, n_sequences, n_drafted, *, padding=0):
    """`padding`: so many of the last tokens of every other sequence's tree are none."""
    return {"name": name, "op": "tree", "n_sequences": n_sequences, "n_drafted": n_drafted, "padding": padding}


def _append(name, dtype, n_sequences, n_tokens, heads, group, dim, rotated, page_size, axes, *, blocks=True, interleaved=False, padding=0):
    """`rotated`: how many of the columns are turned; `axes`: by so many positions of a token; `blocks`: neighbouring pairs of columns go by the
    same axis, else they take turns."""
    return {"name": name, "op": "append", "dtype": dtype, "n_sequences": n_sequences, "n_tokens": n_tokens, "heads": heads, "group": group,
            "dim": dim, "rotated": rotated, "page_size": page_size, "axes": axes, "blocks": blocks, "interleaved": interleaved,
            "padding": padding}


def _attend(name, dtype, n_sequences, longest, n_drafted, heads, group, dim, page_size, *, window=0, cap=0.0, slopes=False, kept=1.0, padding=0):
    """`longest`: tokens of the longest sequence before the drafted ones; `kept` < 1: a bitset filter lets that fraction of the slots through;
    `padding` as in `_tree`."""
    return {"name": name, "op": "attend", "dtype": dtype, "n_sequences": n_sequences, "longest": longest, "n_drafted": n_drafted,
            "heads": heads, "group": group, "dim": dim, "page_size": page_size, "window": window, "cap": cap, "slopes": slopes, "kept": kept,
            "padding": padding}


def _keep(name, dtype, n_sequences, n_drafted, deepest, heads, dim, page_size):
    """`deepest`: entries of a path, at most."""
    return {"name": name, "op": "keep", "dtype": dtype, "n_sequences": n_sequences, "n_drafted": n_drafted, "deepest": deepest,
            "heads": heads, "dim": dim, "page_size": page_size}


def _copy(name, dtype, n_pairs, heads, dim, page_size):
    return {"name": name, "op": "copy", "dtype": dtype, "n_pairs": n_pairs, "heads": heads, "dim": dim, "page_size": page_size}


def listed():
    return [
        # eight requests that draft a small tree each: latency
        _tree("trees of 8 x 16 tokens", 8, 16),
        # a large batch that drafts wide trees, some of them not full
        _tree("trees of 64 x 255 tokens", 64, 255, padding=30),
        # the drafted tokens of eight requests: turned by one position, which is not their place
        _append("append 8 x 16 drafted tokens", "bfloat16", 8, 128, 8, 4, 128, 128, 16, 1, padding=5),
        # images and videos between text: three positions for each token, the axes take turns
        _append("append 9k tokens of 3 axes", "float16", 3, 9001, 8, 4, 128, 128, 64, 3, blocks=False),
        # one request with a short context that drafts a few tokens: latency
        _attend("one request, 1.5k + 8 tokens", "float16", 1, 1500, 8, 8, 4, 128, 16),
        # a batch of requests of very different lengths, capped scores, trees that are not full
        _attend("16 requests up to 16k + 32", "bfloat16", 16, 16_384, 32, 8, 8, 128, 16, cap=30.0, padding=7),
        # one very long context, a wide tree, seven query heads to a key head
        _attend("one request, 250k + 64 tokens", "float16", 1, 250_001, 64, 4, 7, 128, 64),
        # full precision, every head with keys of its own, a bias by distance, a window, pages of 20, erased slots
        _attend("f32, window, slopes, filter", "float32", 9, 9000, 5, 12, 1, 64, 20, window=4000, slopes=True, kept=0.75),
        # the accepted paths of eight requests: latency
        _keep("keep 8 paths", "bfloat16", 8, 16, 5, 8, 128, 16),
        # the accepted paths of a large batch
        _keep("keep 256 paths of up to 17", "float16", 256, 64, 17, 8, 128, 64),
        # four ways on from each of two requests
        _copy("copy 6 pages", "bfloat16", 6, 8, 128, 16),
        # a batch that is forked whole, full precision
        _copy("copy 700 pages, f32", "float32", 700, 3, 96, 100),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    size = _SIZE[dtype]
    op = rng.choice(["tree", "append", "attend", "attend", "attend", "keep", "copy"])
    dim = rng.choice([32, 48, 64, 72, 80, 96, 104, 112, 128, 128, 160, 192, 256])
    if size == 4:
        dim = rng.choice([dim, dim - 4])
    heads = rng.choice([1, 2, 3, 4, 5, 8, 12])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    page_size = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 128, 256])
    if op == "tree":
        n_drafted = _spread(rng, 1, 300)
        case = _tree("", _spread(rng, 1, min(300, 4_000_000 // n_drafted**2)), n_drafted, padding=rng.choice([0, 0, n_drafted // 3]))
    elif op == "append":
        most = 240_000_000 // (size * dim * heads * (group + 2))
        n_tokens = _spread(rng, 1, max(2, min(9000, most)))
        rotated = rng.choice([dim, dim, 2 * (dim // 4), 2 * rng.randint(1, dim // 2)])
        case = _append("", dtype, rng.randint(1, min(64, n_tokens)), n_tokens, heads, group, dim, rotated, page_size, rng.choice([1, 2, 3, 3, 4]),
                       blocks=rng.random() < 0.5, interleaved=rng.random() < 0.5, padding=rng.choice([0, 0, min(3, n_tokens - 1)]))
    elif op == "attend":
        n_sequences = _spread(rng, 1, 64)
        n_drafted = _spread(rng, 1, max(2, min(130, 100_000_000 // (n_sequences * heads * group * dim * size))))
        # no more bytes and products than the largest listed case, were all sequences of the longest one's length; 32-bit products cost more
        most = 800_000_000 // (n_sequences * heads * dim * max(2 * size, group * n_drafted // (6 if size == 4 else 60)))
        longest = _spread(rng, 1, max(2, min(200_000, most)))
        case = _attend("", dtype, n_sequences, longest, n_drafted, heads, group, dim, page_size,
                       window=rng.choice([0, 0, 0, rng.randint(1, longest + n_drafted)]), cap=rng.choice([0.0, 0.0, rng.uniform(5.0, 60.0)]),
                       slopes=rng.random() < 0.25, kept=rng.choice([1.0, 1.0, 0.5, 0.9]), padding=rng.choice([0, 0, n_drafted // 3]))
    elif op == "keep":
        deepest = _spread(rng, 1, 20)
        n_drafted = deepest + _spread(rng, 1, 100)
        most = 500_000_000 // (size * dim * heads * (n_drafted + 2 * page_size))
        case = _keep("", dtype, _spread(rng, 1, max(2, min(300, most))), n_drafted, deepest, heads, dim, page_size)
    else:
        most = 80_000_000 // (size * dim * heads * page_size)
        case = _copy("", dtype, _spread(rng, 1, max(2, min(3000, most))), heads, dim, page_size)
    del case["name"]
    return case


def _lengths(case):
    """The lengths of a batch's sequences before the drafted tokens, longest first: the longest, then ever shorter ones."""
    b = case["n_sequences"]
    return [int(case["longest"] * (1 - i / b) ** 1.5) for i in range(b)]


def _cache(case, n_pages, g):
    """A cache as a program lays it out: the tokens of a page that belong to one head lie together."""
    shape = (n_pages, case["heads"], case["page_size"], case["dim"])
    keys, values = (torch.randn(shape, generator=g, device="cuda", dtype=_TYPE[case["dtype"]]) for _ in range(2))
    return keys.permute(0, 2, 1, 3), values.permute(0, 2, 1, 3)


def _parents(case, g):
    """Every token follows one before it, mostly one not far before: -1 is the sequence's last token, -2 no token."""
    b, t = case["n_sequences"], case["n_drafted"]
    u = torch.rand((b, t), generator=g, device="cuda").sqrt()
    parents = (u * torch.arange(t, device="cuda")).int() - 1
    if case["padding"]:
        parents[::2, t - case["padding"]:] = -2
    return parents


def _table(used, n_pages, width, g):
    """Pages in no order, as they are handed out while requests come and go: `used` [n_sequences] of them for each."""
    column = torch.arange(width, device="cuda")
    rank = (used.cumsum(0) - used)[:, None] + column
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    return torch.where(column < used[:, None], order[rank.clamp(max=n_pages - 1)], -1)


def _prepare_tree(case, g):
    lengths = torch.randint(0, 100_000, (case["n_sequences"],), generator=g, device="cuda", dtype=torch.int32)
    return {"case": case, "parents": _parents(case, g), "lengths": lengths}


def _prepare_append(case, g):
    b, t, ps = case["n_sequences"], case["n_tokens"], case["page_size"]
    each = -(-t // b)
    far = 4000
    pages_each = each // ps + 2
    keys, values = _cache(case, b * pages_each + 3, g)
    start = torch.randint(0, far, (b,), generator=g, device="cuda")
    sequences = torch.arange(t, device="cuda") * b // t
    first = -(-(torch.arange(b, device="cuda") * t) // b)
    place = torch.arange(t, device="cuda") - first[sequences]
    positions = start[sequences] + place
    if case["padding"]:
        positions[t - case["padding"]:] = -1
    width = (far + each) // ps + 3
    order = torch.randperm(b * pages_each + 3, generator=g, device="cuda")[:b * pages_each].view(b, pages_each)
    pages = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    pages.scatter_(1, start[:, None] // ps + torch.arange(pages_each, device="cuda"), order.int())
    if case["axes"] == 1:  # depths of a tree
        turns = (start[sequences] + (torch.rand(t, generator=g, device="cuda") * (place + 1)).long())[:, None]
    else:  # frames of 24 x 17 patches, their rows and columns, and whatever further axis there is
        turns = torch.stack([start[sequences] + place // 408, start[sequences] + place // 17 % 24, start[sequences] + place % 17, place], 1)
        turns = turns[:, :case["axes"]]
    heads, queries = case["heads"], case["heads"] * case["group"]
    # what a fused projection leaves: the rows of queries, keys and values side by side
    rows = torch.randn((t, queries + 2 * heads, case["dim"]), generator=g, device="cuda", dtype=_TYPE[case["dtype"]])
    half = case["rotated"] // 2
    frequencies = torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
    pair = torch.arange(half, device="cuda")
    axes = pair * case["axes"] // half if case["blocks"] else pair % case["axes"]
    return {"case": case, "keys": keys, "values": values, "queries": rows[:, :queries], "new_keys": rows[:, queries:queries + heads],
            "new_values": rows[:, queries + heads:], "sequences": sequences.int(), "positions": positions.int(), "pages": pages,
            "frequencies": frequencies, "turns": turns.int(), "axes": axes.int() if case["axes"] > 1 else None}


def _prepare_attend(case, g):
    ps, t = case["page_size"], case["n_drafted"]
    longest_first = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    lengths = longest_first[torch.randperm(case["n_sequences"], generator=g, device="cuda")]
    used = (lengths + t + ps - 1) // ps
    n_pages = sum(-(-(n + t) // ps) for n in _lengths(case)) + 2
    keys, values = _cache(case, n_pages, g)
    pages = _table(used, n_pages, -(-(case["longest"] + t) // ps), g)
    queries = 1.5 * torch.randn((case["n_sequences"], t, case["heads"] * case["group"], case["dim"]), generator=g, device="cuda")
    mask, positions = _plain_tree({"parents": _parents(case, g), "lengths": lengths})
    n_heads = case["heads"] * case["group"]
    slopes = None
    if case["slopes"]:
        slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / n_heads) for i in range(n_heads)], device="cuda")
    bits = None
    if case["kept"] < 1.0:
        keep = torch.rand((-(-n_pages * ps // 32), 32), generator=g, device="cuda") < case["kept"]
        bits = (keep.long() << torch.arange(32, device="cuda")).sum(1).to(torch.uint32)
    return {"case": case, "keys": keys, "values": values, "queries": queries.to(_TYPE[case["dtype"]]), "pages": pages, "lengths": lengths,
            "positions": positions, "mask": mask.view(torch.uint32), "window": case["window"] or None, "cap": case["cap"] or None,
            "slopes": slopes, "filter": bits}


def _prepare_keep(case, g):
    b, t, deepest, ps = case["n_sequences"], case["n_drafted"], case["deepest"], case["page_size"]
    lengths = torch.randint(0, 5000, (b,), generator=g, device="cuda", dtype=torch.int32)
    first = lengths // ps
    used = (lengths + t + ps - 1) // ps - first
    pages_each = t // ps + 2
    keys, values = _cache(case, b * pages_each, g)
    order = torch.randperm(b * pages_each, generator=g, device="cuda").int().view(b, pages_each)
    column = torch.arange(5000 // ps + pages_each + 1, device="cuda") - first[:, None]
    pages = torch.where((column >= 0) & (column < used[:, None]), order.gather(1, column.clamp(0, pages_each - 1)), -1)
    # the first tokens of a path stay in place, the others come from behind all places that are written, so that every pass finds the same rows
    step = torch.arange(deepest, device="cuda")
    stay = torch.randint(0, deepest + 1, (b, 1), generator=g, device="cuda")
    behind = torch.rand((b, t - deepest), generator=g, device="cuda").argsort(1)[:, :deepest].sort(1).values + deepest
    behind = torch.nn.functional.pad(behind, (0, deepest - behind.shape[1]), value=-1)
    index = torch.where(step < stay, step, behind.gather(1, (step - stay).clamp(min=0)))
    kept = torch.randint(1, deepest + 1, (b, 1), generator=g, device="cuda")
    return {"case": case, "keys": keys, "values": values, "pages": pages.int(), "lengths": lengths,
            "paths": torch.where(step < kept, index, -1).int()}


def _prepare_copy(case, g):
    n = case["n_pairs"]
    keys, values = _cache(case, 2 * n + 5, g)
    order = torch.randperm(2 * n + 5, generator=g, device="cuda").int()
    return {"case": case, "keys": keys, "values": values, "sources": order[:n].contiguous(), "targets": order[n:2 * n].contiguous()}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"tree": _prepare_tree, "append": _prepare_append, "attend": _prepare_attend, "keep": _prepare_keep,
            "copy": _prepare_copy}[case["op"]](case, g)


# ---- plain forms --------------------------------------------------------------------------------------------------------------

def _plain_tree(s):
    """Who reaches whom in at most 1, 2, 4, .. steps, until that is all."""
    parents = s["parents"].long()
    b, t = parents.shape
    token = torch.arange(t, device="cuda")
    reach = ((token == parents[..., None]) | (token == token[:, None])).float()
    steps = 1
    while steps < t:
        reach = (torch.bmm(reach, reach) > 0).float()
        steps *= 2
    reach = reach > 0
    # a token that reaches one which follows the sequence itself
    known = (reach & (parents == -1)[:, None]).any(-1)
    reach &= known[..., None]
    words = -(-t // 32)
    bits = torch.nn.functional.pad(reach, (0, 32 * words - t)).view(b, t, words, 32)
    mask = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(mask >= 2**31, mask - 2**32, mask).int()
    positions = torch.where(known, s["lengths"].long()[:, None] + reach.sum(-1) - 1, -1).int()
    return mask, positions


def _rotate(x, known, angle, interleaved):
    """Pairs of columns turned by angles [n_tokens, n_pairs]; rows of no tokens and columns behind the pairs stay."""
    half = angle.shape[1]
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float()
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
    else:
        a, b = y[..., :half], y[..., half:2 * half]
    u, v = a * c - b * s, b * c + a * s
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    turned = torch.cat((turned, y[..., 2 * half:]), -1)
    return torch.where(known[:, None, None], turned, y).to(x.dtype)


def _plain_append(s):
    ps = s["keys"].shape[1]
    positions = s["positions"].long()
    known = positions >= 0
    page = s["pages"][s["sequences"].long(), positions.clamp(min=0) // ps].long()
    slots = torch.where(known, page * ps + positions % ps, -1)
    turns = s["turns"].double()
    angle = (turns if s["axes"] is None else turns[:, s["axes"].long()]) * s["frequencies"]
    keys = _rotate(s["new_keys"], known, angle, s["case"]["interleaved"])
    queries = _rotate(s["queries"], known, angle, s["case"]["interleaved"])
    at = slots[known]
    s["keys"][at // ps, at % ps] = keys[known]
    s["values"][at // ps, at % ps] = s["new_values"][known]
    return {"keys": s["keys"], "values": s["values"], "slots": slots, "queries": queries}


def _plain_attend(s):
    queries, positions = s["queries"], s["positions"].long()
    b, t, n_heads, dim = queries.shape
    heads, ps = s["keys"].shape[2], s["keys"].shape[1]
    place = torch.arange(s["pages"].shape[1] * ps, device="cuda")
    lengths = s["lengths"].long()[:, None]
    page = s["pages"][:, place // ps].long()
    there = page >= 0
    page = page.clamp(min=0)
    if s["filter"] is not None:
        slot = page * ps + place % ps
        there &= (s["filter"].to(torch.int64)[slot // 32] >> (slot % 32) & 1).bool()
    drafted = (place >= lengths) & (place < lengths + t)
    index = (place - lengths).clamp(0, t - 1)
    at = torch.where(drafted, positions.gather(1, index), place)
    words = s["mask"].view(torch.int32).long().gather(2, (index // 32)[:, None].expand(b, t, -1))
    allowed = (words >> (index % 32)[:, None] & 1).bool() & drafted[:, None]
    del words
    allowed |= (place < lengths)[:, None]
    distance = positions[..., None] - at[:, None]
    allowed &= (there & (at >= 0))[:, None] & (positions >= 0)[..., None]
    if s["window"]:
        allowed &= distance < s["window"]
    keys = s["keys"][page, place % ps].float()
    scores = torch.einsum("bthgd,blhd->bhgtl", queries.float().view(b, t, heads, -1, dim), keys) / math.sqrt(dim)
    del keys
    if s["cap"]:
        scores = s["cap"] * torch.tanh(scores / s["cap"])
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(heads, -1, 1, 1) * distance[:, None, None].float()
    scores = scores.masked_fill(~allowed[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    scores = torch.exp(scores - top)
    total = scores.sum(-1, keepdim=True)
    scores = scores / torch.where(total == 0, 1.0, total)
    values = s["values"][page, place % ps].float()
    out = torch.einsum("bhgtl,blhd->bthgd", scores, values)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)
    return out.reshape(b, t, n_heads, dim).to(queries.dtype), lse.reshape(b, t, n_heads)


def _plain_keep(s):
    ps = s["keys"].shape[1]
    lengths, paths = s["lengths"].long()[:, None], s["paths"].long()
    kept = paths >= 0

    def slots(at):
        return s["pages"].gather(1, (at // ps).long()).long() * ps + at % ps

    source = slots(torch.where(kept, lengths + paths, lengths))[kept]
    target = slots(torch.where(kept, lengths + torch.arange(paths.shape[1], device="cuda"), lengths))[kept]
    for rows in (s["keys"], s["values"]):
        rows[target // ps, target % ps] = rows[source // ps, source % ps]
    return {"keys": s["keys"], "values": s["values"], "lengths": s["lengths"] + kept.sum(1, dtype=torch.int32)}


def _plain_copy(s):
    sources, targets = s["sources"].long(), s["targets"].long()
    s["keys"][targets] = s["keys"][sources]
    s["values"][targets] = s["values"][sources]
    return {"keys": s["keys"], "values": s["values"]}


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        from cuvs_b200 import kv_cache
        if op == "tree":
            mask, positions = kv_cache.draft_tree(state["parents"], state["lengths"], sync=False)
            return mask.view(torch.int32), positions
        if op == "append":
            slots, queries = kv_cache.append(state["keys"], state["values"], state["new_keys"], state["new_values"], state["pages"],
                                             state["positions"], sequences=state["sequences"], queries=state["queries"],
                                             frequencies=state["frequencies"], interleaved=state["case"]["interleaved"],
                                             turns=state["turns"], axes=state["axes"], sync=False)
            return {"keys": state["keys"], "values": state["values"], "slots": slots, "queries": queries}
        if op == "attend":
            return kv_cache.attend_tree(state["keys"], state["values"], state["queries"], state["pages"], state["lengths"],
                                        state["positions"], state["mask"], window=state["window"], cap=state["cap"],
                                        slopes=state["slopes"], filter=state["filter"], sync=False)
        if op == "keep":
            lengths = kv_cache.keep_path(state["keys"], state["values"], state["pages"], state["lengths"], state["paths"], sync=False)
            return {"keys": state["keys"], "values": state["values"], "lengths": lengths}
        kv_cache.copy_pages(state["keys"], state["values"], state["sources"], state["targets"], sync=False)
        return {"keys": state["keys"], "values": state["values"]}
    return {"tree": _plain_tree, "append": _plain_append, "attend": _plain_attend, "keep": _plain_keep, "copy": _plain_copy}[op](state)


def work(case):
    if case["op"] == "tree":
        n, t = case["n_sequences"], case["n_drafted"]
        return {"bytes": n * (8 * t + 4 + 4 * t * -(-t // 32)), "flops": 0}
    size = _SIZE[case["dtype"]]
    row = case["heads"] * case["dim"] * size  # of a token's keys, or its values
    if case["op"] == "append":
        t, half = case["n_tokens"], case["rotated"] // 2
        heads, n_heads = case["heads"], case["heads"] * case["group"]
        return {"bytes": 2 * t * (case["group"] + 2) * row + t * (16 + 4 * case["axes"]) + 12 * half,
                "flops": t * half * (6 * (n_heads + heads) + 3)}
    if case["op"] == "attend":
        t, group = case["n_drafted"], case["group"]
        read = sum(min(n + t, case["window"] or n + t) for n in _lengths(case)) * case["kept"]
        attended = sum(min(n, case["window"] or n) + 1 for n in _lengths(case)) * t * case["kept"]
        rows = case["n_sequences"] * t
        return {"bytes": int(2 * read * row) + rows * group * (2 * row + 4 * case["heads"]) + rows * (4 + 4 * -(-t // 32)),
                "flops": int(4 * attended * case["heads"] * group * case["dim"])}
    if case["op"] == "keep":
        moved = case["n_sequences"] * (case["deepest"] + 1) / 4  # of a path's (deepest + 1) / 2 tokens every other one is not in its place
        return {"bytes": int(4 * moved * row) + 4 * case["n_sequences"] * (case["deepest"] + 2), "flops": 0}
    return {"bytes": case["n_pairs"] * (4 * case["page_size"] * row + 8), "flops": 0}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _exact_append(s):
    """A pair of columns is a complex number, its rotation a product with exp(i * turn * frequency)."""
    keys, values = s["keys"].double(), s["values"].double()
    ps, half = keys.shape[1], s["frequencies"].shape[0]
    axis = [0] * half if s["axes"] is None else s["axes"].tolist()
    angle = torch.stack([s["turns"][:, a].double() * f for a, f in zip(axis, s["frequencies"].tolist())], 1)
    angle[s["positions"] < 0] = 0
    turned = {}
    for name in ("new_keys", "queries"):
        x = s[name].double()
        pairs = x[..., :2 * half]
        pairs = pairs.unflatten(-1, (half, 2)) if s["case"]["interleaved"] else pairs.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None])
        x[..., :2 * half] = z.flatten(-2) if s["case"]["interleaved"] else z.transpose(-1, -2).flatten(-2)
        turned[name] = x
    place = s["positions"].long()
    real = (place >= 0).nonzero()[:, 0]
    page = s["pages"][s["sequences"][real].long(), place[real] // ps].long()
    keys[page, place[real] % ps] = turned["new_keys"][real]
    values[page, place[real] % ps] = s["new_values"][real].double()
    return {"keys": keys, "values": values, "slots": None, "queries": turned["queries"]}


def _exact_attend(s):
    """Sequence by sequence: the slots that any of its drafted tokens may attend to, their positions, and who may."""
    queries = s["queries"].double()
    b, t, n_heads, dim = queries.shape
    ps, heads = s["keys"].shape[1], s["keys"].shape[2]
    group = n_heads // heads
    out = torch.zeros_like(queries)
    lse = torch.full((b, t, n_heads), -math.inf, dtype=torch.float64, device="cuda")
    words = None if s["filter"] is None else s["filter"].to(torch.int64)
    for i, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n + t, device="cuda")
        slot = s["pages"][i, at // ps].long() * ps + at % ps
        own_at = s["positions"][i].long()
        at = torch.cat((at[:n], own_at))
        unpacked = s["mask"][i].view(torch.uint8)[..., None] >> torch.arange(8, device="cuda", dtype=torch.uint8) & 1
        tree = unpacked.reshape(t, -1)[:, :t].bool()
        may = torch.cat((torch.ones((t, n), dtype=torch.bool, device="cuda"), tree), 1) & (own_at >= 0)[:, None]
        if s["window"]:
            may &= own_at[:, None] - at < s["window"]
        if words is not None:
            may &= (words[slot // 32] >> (slot % 32)) % 2 == 1
        for h in range(heads):
            keys, values = (s[name][slot // ps, slot % ps, h].double() for name in ("keys", "values"))
            for j in range(h * group, h * group + group):
                scores = queries[i, :, j] @ keys.t() / math.sqrt(dim)
                if s["cap"]:
                    scores = s["cap"] * torch.tanh(scores / s["cap"])
                if s["slopes"] is not None:
                    scores -= s["slopes"][j].double() * (own_at[:, None] - at)
                scores[~may] = -math.inf
                lse[i, :, j] = torch.logsumexp(scores, 1)
                some = lse[i, :, j] > -math.inf
                out[i, some, j] = torch.exp(scores[some] - lse[i, some, j][:, None]) @ values
    return out, lse


def _exact_tree(s):
    """Every token's way up, step by step."""
    masks, positions = [], []
    for parents, n in zip(s["parents"].tolist(), s["lengths"].tolist()):
        for j in range(len(parents)):
            bits, at, depth = 0, j, -1
            while 0 <= at < len(parents) and depth < len(parents):
                bits |= 1 << at
                at, depth = parents[at], depth + 1
            masks.append(bits.to_bytes(4 * -(-len(parents) // 32), "little") if at == -1 else bytes(4 * -(-len(parents) // 32)))
            positions.append(n + depth if at == -1 else -1)
    mask = torch.frombuffer(bytearray(b"".join(masks)), dtype=torch.int32).view(*s["parents"].shape, -1)
    return mask.cuda(), torch.tensor(positions, dtype=torch.int32, device="cuda").view(s["parents"].shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    keys, values = s["keys"].double(), s["values"].double()
    if case["op"] == "copy":
        for a, b in zip(s["sources"].tolist(), s["targets"].tolist()):
            keys[b], values[b] = keys[a], values[a]
        return {"keys": keys, "values": values}
    ps, pages = case["page_size"], s["pages"].tolist()
    for row, n, path in zip(pages, s["lengths"].tolist(), s["paths"].tolist()):
        for i, index in enumerate(path):
            if index < 0:
                break
            a, b = n + index, n + i
            for rows in (keys, values):
                rows[row[b // ps], b % ps] = rows[row[a // ps], a % ps]
    return {"keys": keys, "values": values, "lengths": None}
