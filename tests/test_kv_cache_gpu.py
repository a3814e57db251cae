"""GPU tests of attention over a paged cache against the definitions in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of 32 bits.  A score, scale * sum of dim products, is off by at most
(dim + 4) u * scale * sum |q k|; a weight exp(score - top) by twice that (score and top), and by 2^-21 for the exponential and what goes
into it; a sum of n weights or weighted values in 32 bits by at most n u of the sum of their magnitudes, where n counts the additions
that follow one another: a unit's rows go to four warps at least, in turn, and one warp adds at most a quarter of them, plus those of its
lanes, of the warps and of the parts (fewer than 592).  Both come in twice, in the sum of values and in the sum of weights.  The output is
rounded once to its type: half a step, eps / 2 of its magnitude (and 2^-25 for fp16's smallest numbers).
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
NONE = 2 ** 63 - 1
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(shape, dtype, g, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def layout(shape, dtype, g, how):
    """A cache's keys and values [n_pages, page_size, n_heads, dim] in one of the layouts that programs use."""
    p, t, h, d = shape
    if how == "tokens":        # the heads of a token together
        return rows(shape, dtype, g), rows(shape, dtype, g)
    if how == "heads":         # the tokens of a head together
        return (rows((p, h, t, d), dtype, g).permute(0, 2, 1, 3) for _ in range(2))
    both = rows((p, 2, t, h, d), dtype, g)      # keys and values of a page side by side
    return both[:, 0], both[:, 1]


def half_step(want, dtype):
    return torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def attend(query, keys, values, scale, dtype):
    """One head in 64 bits: out, lse, and what a 32-bit computation may be off by."""
    q, k, v = query.double(), keys.double(), values.double()
    n, dim = k.shape
    if n == 0:
        return torch.zeros(dim, dtype=torch.float64, device="cuda"), -math.inf, 0.0, 0.0
    s = scale * (k @ q)
    lse = torch.logsumexp(s, 0)
    p = torch.exp(s - lse)
    out = p @ v
    weight = 2 * (dim + 4) * U * abs(scale) * (k.abs() @ q.abs()).max().item() + 2.0 ** -21
    total = weight + (n / 4 + 592) * U
    return out, lse.item(), 2 * total * (p @ v.abs()).max().item() + half_step(out, dtype), total + 4 * U * (1 + abs(lse.item()))


def check(got, got_lse, want):
    """`want`: [[attend(...)]] of every row and head."""
    for i, row in enumerate(want):
        for j, (out, lse, tol, lse_tol) in enumerate(row):
            d = (got[i, j].double() - out).abs()
            assert (d <= tol).all(), (i, j, d.max().item(), float(torch.as_tensor(tol).max()))
            g = got_lse[i, j].item()
            assert g == lse if lse == -math.inf else abs(g - lse) <= lse_tol, (i, j, g, lse, lse_tol)


def slots_of(pages, n_pages, page_size, first, end):
    at = torch.arange(first, max(first, min(end, pages.shape[0] * page_size)))
    page = pages.cpu()[at // page_size].long()
    slot = page * page_size + at % page_size
    return slot[(page >= 0) & (page < n_pages)].cuda()


def allowed(slots, bits):
    if bits is None:
        return slots
    words = torch.from_numpy(bits.cpu().numpy().astype(np.int64)).cuda()
    return slots[(words[slots // 32] >> (slots % 32)) % 2 == 1]


def want_attention(keys, values, queries, pages, lengths, scale=None, window=None, bits=None):
    n_pages, ps, heads, dim = keys.shape
    scale = dim ** -0.5 if scale is None else scale
    found = []
    for i, n in enumerate(lengths.tolist()):
        n = max(n, 0)
        slots = allowed(slots_of(pages[i], n_pages, ps, max(0, n - (window or n)), n), bits)
        k, v = keys[slots // ps, slots % ps], values[slots // ps, slots % ps]
        group = queries.shape[1] // heads
        found.append([attend(queries[i, j], k[:, j // group], v[:, j // group], scale, queries.dtype) for j in range(queries.shape[1])])
    return found


def tables(lengths, page_size, n_pages, g, width=None):
    need = [-(-max(n, 0) // page_size) for n in lengths]
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    pages = torch.full((len(lengths), width or max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        pages[i, :n] = order[at:at + n]
        at += n
    assert at <= n_pages
    return pages


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def random_bits(n_slots, keep, g):
    b = torch.rand((-(-n_slots // 32), 32), generator=g, device="cuda") < keep
    return (b.long() << torch.arange(32, device="cuda")).sum(1).to(torch.uint32)


# lengths, heads, group, dim, page size, layout, window
SHAPES = [
    ([1], 1, 1, 128, 16, "heads", None),
    ([0, 1, 2, 17, 500], 2, 4, 64, 16, "tokens", None),
    ([1000, 3, 0, 129, 128, 127], 4, 8, 128, 32, "both", None),
    ([700, 65, 64, 63], 1, 7, 96, 24, "heads", 100),
    ([333, 40], 3, 3, 40, 5, "tokens", 1),
    ([15, 16, 17, 4099], 2, 16, 80, 1, "tokens", None),
    ([300, 299], 1, 33, 128, 64, "heads", 250),
    ([50, 2000], 2, 20, 256, 128, "both", None),
    ([77], 5, 2, 200, 100, "heads", 70),
    ([260] * 40, 3, 1, 8, 7, "tokens", None),
    ([2500], 8, 1, 160, 256, "heads", None),
    ([90, 11], 1, 128, 64, 16, "tokens", None),
    ([400, 31, 32, 33], 2, 5, 16, 16, "heads", None),
    ([1000], 1, 2, 32, 20, "tokens", 700),
    ([64, 63], 1, 8, 24, 16, "both", None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,group,dim,page_size,how,window", SHAPES)
@pytest.mark.parametrize("keep", [1.0, 0.4])
def test_attention(dtype, lengths, heads, group, dim, page_size, how, window, keep):
    from cuvs_b200 import kv_cache
    g = generator(dim + len(lengths))
    n_pages = sum(-(-n // page_size) for n in lengths) + 3
    keys, values = layout((n_pages, page_size, heads, dim), dtype, g, how)
    queries = rows((len(lengths), heads * group, dim), dtype, g, 2.0)
    pages = tables(lengths, page_size, n_pages, g)
    bits = random_bits(n_pages * page_size, keep, g) if keep < 1 else None
    out, lse = kv_cache.attention(keys, values, queries, pages, ints(lengths), window=window, filter=bits)
    assert out.dtype == dtype and lse.dtype == torch.float32
    check(out, lse, want_attention(keys, values, queries, pages, ints(lengths), window=window, bits=bits))
    again, lse_again = kv_cache.attention(keys, values, queries, pages, ints(lengths), window=window, filter=bits)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)       # no order of arrival in the result


# Work that no single block or warp finishes: parts of one unit by the hundred, of many units with one long one among short and empty ones, of
# all units at once; several eights of heads; more units than blocks.
LONG = [([60000], 1, 4, 64, 16, None), ([30001], 2, 16, 128, 64, None), ([20000, 0, 17], 3, 1, 128, 20, None), ([9000], 4, 40, 64, 16, None),
        ([1, 0, 40000, 5, 300, 0, 77] + [10] * 60, 4, 2, 64, 16, None), ([700 + 13 * i for i in range(40)], 4, 8, 128, 16, None),
        ([3000] * 20, 8, 1, 40, 32, 2000), ([25000] * 3, 1, 5, 256, 32, None), ([1500] * 80, 2, 3, 96, 24, None),
        ([60] * 150 + [20000] + [130] * 60, 8, 1, 64, 16, None), ([300, 40, 0, 1, 90] * 100, 4, 9, 128, 16, 200), ([5000] + [200] * 180, 3, 4, 200, 48, None),
        ([9000, 3], 1, 4, 32, 16, None), ([15000, 700, 31], 2, 2, 8, 20, None), ([300] * 200, 2, 8, 16, 16, None)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,group,dim,page_size,window", LONG)
def test_attention_shared_by_many(dtype, lengths, heads, group, dim, page_size, window):
    from cuvs_b200 import kv_cache
    g = generator(dim + len(lengths))
    n_pages = sum(-(-n // page_size) for n in lengths) + 1
    keys, values = layout((n_pages, page_size, heads, dim), dtype, g, "heads")
    queries = rows((len(lengths), heads * group, dim), dtype, g, 2.0)
    pages, n = tables(lengths, page_size, n_pages, g), ints(lengths)
    out, lse = kv_cache.attention(keys, values, queries, pages, n, window=window)
    check(out, lse, want_attention(keys, values, queries, pages, n, window=window))
    for _ in range(5):
        again, lse_again = kv_cache.attention(keys, values, queries, pages, n, window=window)
        assert torch.equal(out, again) and torch.equal(lse, lse_again)
    need = kv_cache.attention_workspace(keys, queries, pages, window)
    own = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")       # what a workspace held before does not matter
    again, lse_again = kv_cache.attention(keys, values, queries, pages, n, window=window, workspace=own[:need] if need else None)
    assert torch.equal(out, again) and torch.equal(lse, lse_again) and (own[need:] == 255).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page_size", [16, 20])
def test_what_may_not_be_attended_is_not_read(dtype, page_size):
    """Slots behind the length, before the window, left out by the filter, of pages that belong to nobody, hold NaN and infinities."""
    from cuvs_b200 import kv_cache
    g = generator(5)
    lengths, heads, group, dim, window = [300, 45, 0, 1, 100], 2, 4, 64, 150
    n_pages = 60
    keys, values = layout((n_pages, page_size, heads, dim), dtype, g, "heads")
    queries = rows((5, heads * group, dim), dtype, g)
    pages = tables(lengths, page_size, n_pages, g, width=21)
    bits = random_bits(n_pages * page_size, 0.7, g)
    used = torch.zeros(n_pages * page_size, dtype=torch.bool, device="cuda")
    for i, n in enumerate(lengths):
        used[allowed(slots_of(pages[i], n_pages, page_size, max(0, n - window), n), bits)] = True
    bad = (~used).view(n_pages, page_size)
    for t in (keys, values):
        t[bad] = float("nan")
        t[bad & (torch.rand(bad.shape, generator=g, device="cuda") < 0.5)] = float("inf")
    pages[4, 2] = n_pages          # pages that are none, in the middle of a sequence
    pages[4, 3] = -7
    pages[1, 3:] = 2 ** 31 - 1     # and behind the end of one
    out, lse = kv_cache.attention(keys, values, queries, pages, ints(lengths), window=window, filter=bits)
    assert torch.isfinite(out).all()
    check(out, lse, want_attention(keys, values, queries, pages, ints(lengths), window=window, bits=bits))
    # a filter that lets nothing through; lengths that are none, or more than the table holds
    nothing = torch.zeros_like(bits)
    out, lse = kv_cache.attention(keys, values, queries, pages, ints(lengths), filter=nothing)
    assert (out == 0).all() and (lse == -math.inf).all()
    far = ints([-3, 10 ** 9, -2 ** 31, 2 ** 31 - 1, 0])
    clean_k, clean_v = layout((n_pages, page_size, heads, dim), dtype, g, "heads")
    out, lse = kv_cache.attention(clean_k, clean_v, queries, pages, far)
    check(out, lse, want_attention(clean_k, clean_v, queries, pages, far))
    out, lse = kv_cache.attention(clean_k, clean_v, queries, pages, far, window=10 ** 9 - 30)
    check(out, lse, want_attention(clean_k, clean_v, queries, pages, far, window=10 ** 9 - 30))


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_no_numbers_come_through(dtype):
    from cuvs_b200 import kv_cache
    g = generator(6)
    keys, values = layout((8, 16, 1, 64), dtype, g, "tokens")
    queries = rows((3, 2, 64), dtype, g)
    pages = torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2)
    values[0, 3, 0, 5] = float("nan")
    values[2, 3, 0, 6] = float("inf")
    keys[4, 1] = float("nan")
    out, lse = kv_cache.attention(keys, values, queries, pages, ints([32, 32, 32]))
    assert torch.isnan(out[0, :, 5]).all() and torch.isfinite(out[0, :, :5]).all() and torch.isfinite(lse[:2]).all()
    assert (out[1, :, 6] == float("inf")).all() and torch.isfinite(out[1, :, 7:]).all()
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_far_apart_and_other_scales(dtype):
    """Scores of hundreds: one row takes all; a scale of zero: the mean; a negative one: the least alike."""
    from cuvs_b200 import kv_cache
    g = generator(7)
    keys, values = layout((21, 16, 2, 64), dtype, g, "heads")
    queries = rows((2, 4, 64), dtype, g, 30.0)
    pages = tables([150, 170], 16, 21, g, width=11)
    lengths = ints([150, 170])
    for scale in (1.0, 0.0, -0.5, None):
        out, lse = kv_cache.attention(keys, values, queries, pages, lengths, scale=scale)
        check(out, lse, want_attention(keys, values, queries, pages, lengths, scale=scale))


def test_strided_queries_outputs_tables_and_streams():
    from cuvs_b200 import Resources, kv_cache
    g = generator(8)
    keys, values = layout((40, 16, 2, 96), torch.bfloat16, g, "both")
    fused = rows((6, 12, 96), torch.bfloat16, g)
    queries = fused[:, 1:9:2]
    wide = torch.full((6, 50), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    lengths = [100, 1, 0, 37, 96, 5]
    wide[:, 3:10] = tables(lengths, 16, 40, g, width=7)
    pages = wide[:, 3:10]
    want = want_attention(keys, values, queries, pages, ints(lengths))
    frame = torch.full((6, 4, 3, 96), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((6, 4), device="cuda")
    out, same = kv_cache.attention(keys, values, queries, pages, ints(lengths), out=frame[:, :, 1], lse=lse)
    assert out.data_ptr() == frame[:, :, 1].data_ptr() and same is lse
    check(frame[:, :, 1], lse, want)
    assert (frame[:, :, 0] == 7).all() and (frame[:, :, 2] == 7).all()
    # a stream of torch's, a handle with a stream of its own, and the output over the queries
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = kv_cache.attention(keys, values, queries, pages, ints(lengths), sync=False)
    side.synchronize()
    check(out, lse, want)
    torch.cuda.synchronize()
    out, lse = kv_cache.attention(keys, values, queries, pages, ints(lengths), resources=Resources(side.cuda_stream))
    check(out, lse, want)
    kv_cache.attention(keys, values, queries, pages, ints(lengths), out=queries, lse=lse)
    check(queries, lse, want)


def test_calls_on_several_streams_at_once():
    from cuvs_b200 import kv_cache
    g = generator(9)
    keys, values = layout((400, 16, 2, 64), torch.float16, g, "heads")
    lengths = [3000, 1500, 900]
    pages = tables(lengths, 16, 400, g)
    queries = [rows((3, 8, 64), torch.float16, g) for _ in range(6)]
    want = [kv_cache.attention(keys, values, q, pages, ints(lengths)) for q in queries]
    n = ints(lengths)
    streams = [torch.cuda.Stream() for _ in queries]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for q, s in zip(queries, streams):
            with torch.cuda.stream(s):
                got.append(kv_cache.attention(keys, values, q, pages, n, sync=False))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and torch.equal(b, d)


def test_captured_steps_follow_their_inputs():
    """Two graphs, replayed in turn with changed lengths, tables and tokens, agree with calls; a captured call cannot wait."""
    from cuvs_b200 import kv_cache
    from cuvs_b200._lib import CuvsError
    g = generator(10)
    dtype, b, heads, n_heads, dim, ps = torch.float16, 3, 2, 8, 64, 16
    f = torch.tensor([100.0 ** (-i / 32) for i in range(32)], dtype=torch.float64, device="cuda")

    def step(c):
        slots, q = kv_cache.append(c["k"], c["v"], c["nk"], c["nv"], c["pages"], c["pos"], queries=c["q"], frequencies=f, sync=False)
        near = kv_cache.attention(c["k"], c["v"], q, c["pages"], c["len"], window=600, sync=False)
        far = kv_cache.attend_candidates(c["k"], c["v"], q, c["cand"], sync=False)
        return (slots, *kv_cache.merge_parts(torch.stack((near[0], far[0])), torch.stack((near[1], far[1])), sync=False))

    def inputs(c, lengths):
        c["len"].copy_(ints(lengths))
        c["pos"].copy_(ints(lengths) - 1)
        c["pages"].copy_(tables(lengths, ps, 500, g, width=180))
        c["cand"].copy_(torch.randint(0, 8000, (b, n_heads, 33), generator=g, device="cuda"))
        for name, heads_of in (("nk", heads), ("nv", heads), ("q", n_heads)):
            c[name].copy_(rows((b, heads_of, dim), dtype, g))

    cases, graphs, outs = [], [], []
    for _ in range(2):
        k, v = layout((500, ps, heads, dim), dtype, g, "heads")
        c = {"k": k, "v": v, "nk": rows((b, heads, dim), dtype, g), "nv": rows((b, heads, dim), dtype, g),
             "q": rows((b, n_heads, dim), dtype, g), "pos": ints([0] * b), "len": ints([1] * b),
             "pages": torch.zeros((b, 180), dtype=torch.int32, device="cuda"),
             "cand": torch.zeros((b, n_heads, 33), dtype=torch.int64, device="cuda")}
        inputs(c, [5, 2000, 70])
        step(c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(c)
        cases.append(c)
        graphs.append(graph)
        outs.append(out)
    for lengths in ([5, 2000, 70], [1, 1, 1], [2800, 16, 17], [640, 641, 1]):
        for c in cases:
            inputs(c, lengths)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for out in outs]
        for c, have in zip(cases, got):
            for a, w in zip(have, step(c)):
                assert torch.equal(a, w)
    c = cases[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(CuvsError, match="sync=False"):
            kv_cache.attention(c["k"], c["v"], c["q"], c["pages"], c["len"])
        out = step(c)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[1], got[0][1])


def test_shared_units_on_several_streams_and_in_graphs():
    """Work that leaves parts in a workspace: calls on several streams and from several threads at once, two graphs that are replayed side by
    side while calls go on, each with the lengths of the moment."""
    import threading
    from cuvs_b200 import kv_cache
    g = generator(12)
    n_pages = 6000
    keys, values = layout((n_pages, 16, 2, 64), torch.bfloat16, g, "heads")
    lengths = [40000, 20000, 7000, 30]
    pages = tables(lengths, 16, n_pages, g)
    queries = [rows((4, 8, 64), torch.bfloat16, g) for _ in range(4)]
    assert kv_cache.attention_workspace(keys, queries[0], pages) > 0
    n = ints(lengths)
    want = [kv_cache.attention(keys, values, q, pages, n) for q in queries]
    check(*want[0], want_attention(keys, values, queries[0], pages, n))
    moment = [ints(lengths), ints(lengths)]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kv_cache.attention(keys, values, queries[i], pages, moment[i], sync=False))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    shorter = [39000, 1, 0, 30]
    want_shorter = [kv_cache.attention(keys, values, q, pages, ints(shorter)) for q in queries[:2]]
    torch.cuda.synchronize()
    for turn in range(10):
        for m in moment:
            m.copy_(ints(lengths if turn % 2 else shorter))
        torch.cuda.synchronize()
        got = []
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        for q, s in zip(queries, streams[2:] * 2):
            with torch.cuda.stream(s):
                got.append(kv_cache.attention(keys, values, q, pages, n, sync=False))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and torch.equal(b, d)
        for (a, b), (c, d) in zip(outs, want if turn % 2 else want_shorter):
            assert torch.equal(a, c) and torch.equal(b, d)
    wrong = []

    def work(q, w):
        for _ in range(30):
            a, b = kv_cache.attention(keys, values, q, pages, n)        # all threads on the default stream, through one handle
            if not (torch.equal(a, w[0]) and torch.equal(b, w[1])):
                wrong.append(1)

    threads = [threading.Thread(target=work, args=x) for x in zip(queries, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_parameters_and_other_subclasses():
    from cuvs_b200 import kv_cache
    g = generator(13)
    keys, values = layout((9, 16, 2, 64), torch.float16, g, "tokens")
    q, pages, n = rows((1, 4, 64), torch.float16, g), ints([[3, 1, 7]]), ints([44])
    want = kv_cache.attention(keys, values, q, pages, n)
    got = kv_cache.attention(torch.nn.Parameter(keys), values, torch.nn.Parameter(q), pages, n)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # tensors that require gradients are read all the same; the results have none
    got = kv_cache.attention(keys, values, q.clone().requires_grad_(), pages, n)
    assert torch.equal(got[0], want[0]) and not got[0].requires_grad


def test_offsets_that_pass_32_bits():
    """A cache of more than 2^32 elements: rows of its last pages."""
    from cuvs_b200 import kv_cache
    g = generator(11)
    dim, ps, heads = 128, 64, 4
    n_pages = 2 ** 32 // (dim * ps * heads) + 9
    keys, values = (torch.empty((n_pages, heads, ps, dim), dtype=torch.float16, device="cuda").permute(0, 2, 1, 3) for _ in range(2))
    pages = ints([[n_pages - 1, 3], [n_pages - 5, n_pages - 2]])
    new_k, new_v = rows((256, heads, dim), torch.float16, g), rows((256, heads, dim), torch.float16, g)
    order = ints(list(range(128)) * 2)
    sequences = ints([0] * 128 + [1] * 128)
    slots, _ = kv_cache.append(keys, values, new_k, new_v, pages, order, sequences=sequences)
    want = (pages.long()[sequences.long(), order.long() // ps] * ps + order.long() % ps)
    assert torch.equal(slots, want)
    assert torch.equal(keys[slots // ps, slots % ps], new_k) and torch.equal(values[slots // ps, slots % ps], new_v)
    queries = rows((2, 8, dim), torch.float16, g)
    lengths = ints([100, 128])
    out, lse = kv_cache.attention(keys, values, queries, pages, lengths)
    check(out, lse, want_attention(keys, values, queries, pages, lengths))
    candidates = slots.view(2, 1, 128).expand(2, 8, 128).contiguous()
    out, lse = kv_cache.attend_candidates(keys, values, queries, candidates)
    check(out, lse, want_attention(keys, values, queries, pages, ints([128, 128])))


# ---- append -------------------------------------------------------------------------------------------------------------------

def turned(x, positions, f, interleaved):
    """x [n, heads, dim] turned in 64 bits, and what 32 bits may be off by."""
    y, half = x.double().clone(), f.shape[0]
    tol = torch.zeros_like(y)
    angle = positions.clamp(min=0).double()[:, None, None] * f.double()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * angle.cos() - q * angle.sin(), q * angle.cos() + p * angle.sin()
    # two products, a sum, and sine and cosine: off by two steps of 32 bits and by pi times the rounding of the reduced angle
    tol[..., a] = tol[..., b] = (p.abs() + q.abs()) * 10 * U
    return y, tol + half_step(y, x.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,pairs,heads,group,page_size,how", [
    (128, 64, 8, 4, 16, "heads"), (64, 32, 2, 1, 20, "tokens"), (96, 24, 3, 3, 24, "both"), (80, 40, 1, 5, 1, "tokens"),
    (256, 128, 1, 16, 64, "heads"), (256, 101, 2, 2, 3, "heads"), (40, 7, 2, 3, 16, "both"), (128, 63, 2, 2, 16, "heads"), (8, 4, 5, 1, 2, "tokens"),
    (112, 0, 2, 2, 16, "tokens"), (72, 1, 2, 2, 16, "heads")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(dtype, dim, pairs, heads, group, page_size, how, interleaved):
    from cuvs_b200 import kv_cache
    g = generator(dim + pairs)
    n_pages, width = 50, 70000
    keys, values = layout((n_pages, page_size, heads, dim), dtype, g, how)
    before_k, before_v = keys.clone(), values.clone()
    fused = rows((23, heads * group + 2 * heads, dim), dtype, g)
    q, k, v = fused[:, :heads * group], fused[:, heads * group:heads * group + heads], fused[:, heads * group + heads:]
    # tokens of three sequences, in no order: short, far, up to the page's end and over it; padding; what is nowhere
    places = [(0, 0), (0, 1), (0, 2), (1, 1000), (1, 1001), (2, 65535), (2, 65536), (0, page_size), (0, page_size - 1 + 5), (1, 999)]
    places = list(dict.fromkeys(places))
    nowhere = [(0, -1), (1, -2 ** 31), (3, 5), (-1, 5), (2, 2 ** 31 - 1), (0, 40000 * page_size)]
    places = (places + nowhere + [(1, 5000 + i) for i in range(23)])[:23]
    order = torch.randperm(23, generator=g, device="cuda").tolist()
    places = [places[i] for i in order]
    sequences, positions = ints([s for s, _ in places]), ints([p for _, p in places])
    pages = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    free, slots_want = torch.randperm(n_pages, generator=g, device="cuda").tolist(), []
    for s, p in places:
        c = p // page_size
        if not (0 <= s < 3 and 0 <= p and c < width) or (s, p) in nowhere:
            slots_want.append(-1)
            continue
        if pages[s, c] < 0:
            pages[s, c] = free.pop()
        slots_want.append(int(pages[s, c]) * page_size + p % page_size)
    f = torch.tensor([10000.0 ** (-i / max(1, pairs)) for i in range(pairs)], dtype=torch.float64, device="cuda")
    rotated = torch.full((23, heads * group, 2, dim), 3.0, dtype=dtype, device="cuda")
    slots, got = kv_cache.append(keys, values, k, v, pages, positions, sequences=sequences, queries=q, frequencies=f,
                                 interleaved=interleaved, rotated=rotated[:, :, 1])
    assert slots.tolist() == slots_want
    written = (slots >= 0).nonzero()[:, 0]
    at = slots[written]
    want, tol = turned(k[written], positions[written], f, interleaved)
    assert ((keys[at // page_size, at % page_size].double() - want).abs() <= tol).all()
    assert torch.equal(values[at // page_size, at % page_size], v[written])
    want, tol = turned(q, positions, f, interleaved)
    want[positions < 0] = q[positions < 0].double()
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[positions < 0], q[positions < 0]) and (rotated[:, :, 0] == 3).all()
    # nothing else in the cache has changed
    left = torch.ones(n_pages * page_size, dtype=torch.bool, device="cuda")
    left[at] = False
    left = left.view(n_pages, page_size)
    assert torch.equal(keys[left], before_k[left]) and torch.equal(values[left], before_v[left])
    # over the queries themselves, with frequencies of 32 bits, gives the same to 32 bits' rounding of the angles at near positions
    kv_cache.append(keys, values, k, v, pages, positions, sequences=sequences, queries=q, frequencies=f, interleaved=interleaved, rotated=q)
    assert torch.equal(q, got)


def test_append_without_rotation_or_queries_and_many_tokens():
    from cuvs_b200 import kv_cache
    g = generator(21)
    n, heads, dim, ps = 30011, 2, 64, 32
    keys, values = layout((1000, ps, heads, dim), torch.bfloat16, g, "heads")
    k, v = rows((n, heads, dim), torch.bfloat16, g), rows((n, heads, dim), torch.bfloat16, g)
    pages = torch.randperm(1000, generator=g, device="cuda").int().view(1, 1000)
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    slots, rotated = kv_cache.append(keys, values, k, v, pages, positions, sequences=torch.zeros_like(positions))
    assert rotated is None
    assert torch.equal(keys[slots // ps, slots % ps], k) and torch.equal(values[slots // ps, slots % ps], v)
    # one token of every sequence; frequencies of 32 bits are taken as they are
    f32 = torch.rand(32, generator=g, device="cuda")
    slots, _ = kv_cache.append(keys, values, k[:7], v[:7], pages.view(10, 100)[:7], positions[:7] + 90, frequencies=f32)
    want, tol = turned(k[:7], positions[:7] + 90, f32, False)
    assert ((keys[slots // ps, slots % ps].double() - want).abs() <= tol).all()
    # no tokens
    slots, _ = kv_cache.append(keys, values, k[:0], v[:0], pages, positions[:0], sequences=positions[:0])
    assert slots.shape == (0,)


def test_far_positions_keep_their_angles():
    from cuvs_b200 import kv_cache
    g = generator(22)
    keys, values = layout((4, 16, 1, 64), torch.float32, g, "tokens")
    k, v = rows((3, 1, 64), torch.float32, g), rows((3, 1, 64), torch.float32, g)
    q = rows((3, 2, 64), torch.float32, g)
    positions = ints([2 ** 31 - 1, 2 ** 31 - 2, 123456789])
    f = torch.tensor([1.0 / (1 + i) for i in range(32)], dtype=torch.float64, device="cuda")
    pages = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    slots, got = kv_cache.append(keys, values, k, v, pages, positions, queries=q, frequencies=f)
    assert (slots == -1).all()                           # no table reaches that far; the queries are turned all the same
    want, tol = turned(q, positions, f, False)
    # the product of position and frequency is rounded in 64 bits, there and here: 2^31 * 2^-52 of an angle
    assert ((got.double() - want).abs() <= tol + 2.0 ** -20 * want.abs().max()).all()


# ---- candidates ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,group,dim,page_size,k,how,keep", [
    (1, 1, 1, 128, 16, 1, "heads", 1.0), (3, 2, 4, 64, 20, 100, "tokens", 1.0), (2, 3, 1, 96, 7, 33, "both", 0.6),
    (1, 1, 16, 256, 128, 1000, "heads", 1.0), (5, 2, 2, 40, 1, 65, "tokens", 0.3), (1, 2, 1, 200, 16, 4000, "heads", 1.0),
    (200, 4, 2, 32, 16, 17, "heads", 1.0), (4, 1, 2, 8, 16, 31, "heads", 1.0)])
def test_candidates(dtype, n, heads, group, dim, page_size, k, how, keep):
    from cuvs_b200 import kv_cache
    g = generator(dim + k)
    n_pages = 1500 // page_size + 1
    n_slots = n_pages * page_size
    keys, values = layout((n_pages, page_size, heads, dim), dtype, g, how)
    queries = rows((n, heads * group, dim), dtype, g, 2.0)
    candidates = torch.randint(0, n_slots, (n, heads * group, k), generator=g, device="cuda")
    lists = candidates.view(-1, k)
    lists[::3, k // 2:] = NONE                       # lists that are not full
    lists[1::4, ::2] = -1
    lists[-1] = torch.tensor([NONE, -1, n_slots, -2 ** 63, 2 ** 40, 2 ** 32], device="cuda").repeat(k)[:k]       # nothing at all
    lists[0, :] = lists[0, 0] if k > 1 else lists[0, :]          # the same slot again and again
    bits = random_bits(n_slots, keep, g) if keep < 1 else None
    out, lse = kv_cache.attend_candidates(keys, values, queries, candidates, filter=bits)
    want = []
    for i in range(n):
        want.append([])
        for j in range(heads * group):
            slots = candidates[i, j]
            slots = allowed(slots[(slots >= 0) & (slots < n_slots)], bits)
            want[-1].append(attend(queries[i, j], keys[slots // page_size, slots % page_size, j // group],
                                   values[slots // page_size, slots % page_size, j // group], dim ** -0.5, dtype))
    check(out, lse, want)
    again, lse_again = kv_cache.attend_candidates(keys, values, queries, candidates, filter=bits)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)


def test_empty_calls():
    from cuvs_b200 import kv_cache
    g = generator(30)
    keys, values = layout((4, 16, 2, 64), torch.float16, g, "heads")
    q = rows((3, 4, 64), torch.float16, g)
    none = torch.empty((3, 4, 0), dtype=torch.int64, device="cuda")
    for out, lse in (kv_cache.attend_candidates(keys, values, q, none),
                     kv_cache.attention(keys, values, q, torch.empty((3, 0), dtype=torch.int32, device="cuda"), ints([5, 0, 7])),
                     kv_cache.attention(keys[:0], values[:0], q, ints([[0], [0], [0]]), ints([5, 0, 7])),
                     kv_cache.merge_parts(rows((0, 3, 4, 64), torch.float16, g), torch.empty((0, 3, 4), device="cuda"))):
        assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = kv_cache.attend_candidates(keys, values, q[:0], none[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = kv_cache.attention(keys, values, q[:0], ints([[0]])[:0], ints([5])[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = kv_cache.merge_parts(rows((2, 0, 4, 64), torch.float16, g), torch.empty((2, 0, 4), device="cuda"))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


# ---- joining parts ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_parts,n,heads,dim", [(1, 1, 1, 8), (2, 8, 32, 128), (3, 5, 7, 96), (17, 33, 3, 200), (8, 1000, 4, 64), (5, 2, 2, 256)])
def test_merge_parts(dtype, n_parts, n, heads, dim):
    from cuvs_b200 import kv_cache
    g = generator(dim + n_parts)
    # blocks as they are gathered: every part with its lse and with something between them
    parts = rows((n_parts, n + 2, heads, dim), dtype, g)[:, :n]
    lse = (10.0 + 5.0 * torch.randn((n_parts, heads, n + 1), generator=g, device="cuda")).transpose(1, 2)[:, :n]
    empty = torch.rand(lse.shape, generator=g, device="cuda") < 0.3
    empty[:, 0, 0] = True                              # a row with nothing at all
    lse[empty] = -math.inf
    parts[empty] = float("nan")                        # what a part left where it attended to nothing is not read
    out, got = kv_cache.merge_parts(parts, lse)
    share = torch.exp(lse.double() - torch.logsumexp(lse.double(), 0)).nan_to_num(0.0)
    clean = torch.where(empty[..., None], 0.0, parts.double())
    want = torch.einsum("pnh,pnhd->nhd", share, clean)
    want_lse = torch.logsumexp(lse.double(), 0)
    # weights: 2^-21 as above and the rounding of differences of up to 40; n_parts additions
    total = 2.0 ** -21 + 40 * U + n_parts * U
    tol = 2 * total * torch.einsum("pnh,pnhd->nhd", share, clean.abs()) + half_step(want, dtype)
    assert ((out.double() - want).abs() <= tol).all()
    there = want_lse > -math.inf
    assert (got[~there] == -math.inf).all() and (out[~there] == 0).all()
    assert ((got.double() - want_lse)[there].abs() <= total + 4 * U * (1 + want_lse[there].abs())).all()


# ---- together -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_step_with_a_search_over_the_far_keys(dtype):
    """Append a prompt, index its far keys by their slots, then decode: append, search, attend to the near tokens and to the found far
    ones, join.  With every far key found, the step is attention to all tokens; with few, to the near ones and those."""
    from cuvs_b200 import ivf_pq, kv_cache
    g = generator(40)
    heads, group, dim, ps, n, window = 2, 3, 64, 16, 2200, 200
    keys, values = layout((160, ps, heads, dim), dtype, g, "heads")
    pages = torch.randperm(160, generator=g, device="cuda").int().view(1, 160)
    f = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64, device="cuda")
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    slots, _ = kv_cache.append(keys, values, rows((n, heads, dim), dtype, g), rows((n, heads, dim), dtype, g), pages, at,
                               sequences=torch.zeros_like(at), frequencies=f)
    far = slots[:n + 1 - window]
    indexes = []
    for h in range(heads):
        params = ivf_pq.IndexParams(n_lists=16, metric="inner_product", pq_dim=32, kmeans_n_iters=4, add_data_on_build=False)
        own = keys[far // ps, far % ps, h].contiguous()
        indexes.append(ivf_pq.extend(ivf_pq.build(params, own), own, far))
    new = [rows((1, heads, dim), dtype, g) for _ in range(2)]
    q = rows((1, heads * group, dim), dtype, g)
    slot, q = kv_cache.append(keys, values, *new, pages, ints([n]), queries=q, frequencies=f)
    lengths = ints([n + 1])
    everything = want_attention(keys, values, q, pages, lengths)
    for k, n_probes in ((far.shape[0], 16), (50, 8)):
        candidates = torch.stack([ivf_pq.search(ivf_pq.SearchParams(n_probes=n_probes), indexes[h], q[0, h * group:(h + 1) * group].contiguous(),
                                                k)[1] for h in range(heads)]).view(1, heads * group, k)
        near = kv_cache.attention(keys, values, q, pages, lengths, window=window)
        named = kv_cache.attend_candidates(keys, values, q, candidates)
        out, lse = kv_cache.merge_parts(torch.stack((near[0], named[0])), torch.stack((near[1], named[1])))
        recent = slots_of(pages[0], 160, ps, n + 1 - window, n + 1)
        want = []
        for j in range(heads * group):
            found = candidates[0, j]
            found = found[found < 160 * ps]
            assert found.unique().numel() == found.numel()
            both = torch.cat((recent, found))
            # the parts are rounded to their type before they are joined: half a step of either, by its share
            o, l, tol, lse_tol = attend(q[0, j], keys[both // ps, both % ps, j // group], values[both // ps, both % ps, j // group],
                                        dim ** -0.5, dtype)
            parts = torch.stack((near[0][0, j], named[0][0, j])).double().abs().amax(0)
            want.append((o, l, 2 * tol + torch.finfo(dtype).eps / 2 * parts + 2.0 ** -24, 2 * lse_tol))
        check(out, lse, [want])
        if k == far.shape[0]:
            for j in range(heads * group):
                assert (out[0, j].double() - everything[0][j][0]).abs().max() <= want[j][2].max()


def test_c_entries_take_described_tensors():
    """The C interface with DLPack tensors, and the handle's own workspace."""
    import ctypes as C
    from cuvs_b200 import _lib as L
    from cuvs_b200 import kv_cache
    from cuvs_b200.common import DLTensorRef, default_resources
    g = generator(50)
    keys, values = rows((30, 16, 2, 64), torch.float16, g), rows((30, 16, 2, 64), torch.float16, g)
    q = rows((2, 8, 64), torch.float16, g)
    pages, lengths = tables([200, 233], 16, 30, g), ints([200, 233])
    lib, res = L.load(), default_resources()
    res.use_current_stream()
    out, lse = torch.empty_like(q), torch.empty((2, 8), device="cuda")
    refs = [DLTensorRef(t) for t in (keys, values, q, pages, lengths, out, lse)]
    k, v, qq, p, n, o, l = (r.ref() for r in refs)
    size = C.c_size_t()
    L.check(lib.cuvsKvCacheAttentionWorkspace(res.handle, k, qq, p, 0, C.byref(size)))
    L.check(lib.cuvsKvCacheAttention(res.handle, k, v, qq, p, n, 0.125, 0, L.FilterStruct(0, 0), o, l, None))
    res.sync()
    want = kv_cache.attention(keys, values, q, pages, lengths, scale=0.125)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    if size.value:
        small = torch.empty(16, dtype=torch.uint8, device="cuda")
        w = DLTensorRef(small)
        with pytest.raises(L.CuvsError, match="are needed"):
            L.check(lib.cuvsKvCacheAttention(res.handle, k, v, qq, p, n, 0.125, 0, L.FilterStruct(0, 0), o, l, w.ref()))
    bits = DLTensorRef(random_bits(480, 0.5, g))
    flt = L.FilterStruct(C.addressof(bits.managed), 1)
    L.check(lib.cuvsKvCacheAttention(res.handle, k, v, qq, p, n, 0.125, 100, flt, o, l, None))
    res.sync()
    check(out, lse, want_attention(keys, values, q, pages, lengths, scale=0.125, window=100, bits=bits._keep))
    with pytest.raises(L.CuvsError, match="Unsupported sample filter"):
        L.check(lib.cuvsKvCacheAttention(res.handle, k, v, qq, p, n, 0.125, 100, L.FilterStruct(1, 2), o, l, None))
    cand = torch.randint(0, 480, (2, 8, 10), generator=g, device="cuda")
    c = DLTensorRef(cand)
    L.check(lib.cuvsKvCacheAttendCandidates(res.handle, k, v, qq, c.ref(), 0.125, L.FilterStruct(0, 0), o, l))
    res.sync()
    want = kv_cache.attend_candidates(keys, values, q, cand)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    parts, parts_lse = torch.stack((q, out)), torch.stack((lse, lse))
    a, b = DLTensorRef(parts), DLTensorRef(parts_lse)
    joined, joined_lse = torch.empty_like(q), torch.empty_like(lse)
    j, jl = DLTensorRef(joined), DLTensorRef(joined_lse)
    L.check(lib.cuvsKvCacheMergeParts(res.handle, a.ref(), b.ref(), j.ref(), jl.ref()))
    res.sync()
    want = kv_cache.merge_parts(parts, parts_lse)
    assert torch.equal(joined, want[0]) and torch.equal(joined_lse, want[1])
    new = rows((2, 2, 64), torch.float16, g)
    slots = torch.empty(2, dtype=torch.int64, device="cuda")
    a, s = DLTensorRef(new), DLTensorRef(slots)
    L.check(lib.cuvsKvCacheAppend(res.handle, k, v, a.ref(), a.ref(), p, n, None, None, None, False, s.ref(), None))
    res.sync()
    at = (lengths // 16).long()
    inside = at < pages.shape[1]
    page = pages[torch.arange(2, device="cuda"), at.clamp(max=pages.shape[1] - 1)].long()
    assert torch.equal(slots, torch.where(inside & (page >= 0), page * 16 + lengths % 16, -1))
