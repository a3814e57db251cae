"""GPU tests of how the calls of a step of drafted tokens may be made: as a step, captured, by words, from C, on several streams and threads."""
import ctypes as C
import math
import textwrap
import threading

import pytest
import torch

from cuvs_b200 import Resources, kv_cache
from cuvs_b200 import _lib as L
from test_kv_tree_gpu import DTYPES, U, WEIGHT, Step, generator, ints, needs_a_gpu, pack, random_parents, tree_of  # noqa: F401

pytestmark = pytest.mark.gpu


def rows(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def step_of(dtype, seed=1, lengths=(300, 17, 2000), n_drafted=12, heads=2, group=4, dim=64, page=16):
    """What the documented step has in hand."""
    g = generator(seed)
    n = len(lengths)
    width = (max(lengths) + n_drafted) // page + 1
    has = {"keys": rows((n * width, page, heads, dim), dtype, g), "values": rows((n * width, page, heads, dim), dtype, g),
           "pages": torch.randperm(n * width, generator=g, device="cuda").int().view(n, width), "lengths": ints(lengths),
           "parents": random_parents(n, n_drafted, g, spread=0.3), "n_drafted": n_drafted, "torch": torch, "kv_cache": kv_cache,
           "new_keys": rows((n, n_drafted, heads, dim), dtype, g), "new_values": rows((n, n_drafted, heads, dim), dtype, g),
           "queries": rows((n, n_drafted, heads * group, dim), dtype, g),
           "sequences": torch.arange(n, device="cuda").repeat_interleave(n_drafted).int(),
           "frequencies": torch.tensor([10000.0 ** (-i / (dim // 2)) for i in range(dim // 2)], dtype=torch.float64, device="cuda")}
    # the deepest path of every tree
    paths = []
    for up in has["parents"].tolist():
        best = []
        for j in range(n_drafted):
            way = []
            while j >= 0:
                way.append(j)
                j = up[j]
            best = max(best, way[::-1], key=len)
        paths.append(best + [-1] * (n_drafted - len(best)))
    has["paths"] = ints(paths)
    return has


def documented():
    doc = kv_cache.__doc__
    return textwrap.dedent(doc[doc.index("has as its step::") + 17:doc.index("The drafted token ``j``")])


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_documented_step(dtype):
    """The last token of a path that stays: attention of one token to the sequence as it is then says the same."""
    has = step_of(dtype)
    before = has["lengths"].clone()
    exec(documented(), has)
    torch.cuda.synchronize()
    n_kept = (has["paths"] >= 0).sum(1)
    assert torch.equal(has["lengths"], (before + n_kept).int())
    last = has["paths"].gather(1, (n_kept - 1)[:, None].long())[:, 0].long()
    i = torch.arange(3, device="cuda")
    q = has["q"].view(has["queries"].shape)[i, last]
    assert torch.equal(has["positions"][i, last] + 1, has["lengths"])
    near, near_lse = kv_cache.attention(has["keys"], has["values"], q.contiguous(), has["pages"], has["lengths"])
    # each is within its rounding and that of a 32-bit softmax of the exact answer: products of 64 terms, weights, sums of as many terms as there are keys
    size = 64 ** -0.5 * has["q"].double().norm(dim=-1).max() * has["keys"].double().norm(dim=-1).max()
    total = 70 * U * size + 2.0 ** -20 + (has["lengths"].max() + 600) * U
    off = torch.finfo(dtype).eps * near.double().abs() * 1.01 + 2 * (2 * total + WEIGHT[dtype]) * has["values"].double().abs().max() + 2.0 ** -24
    assert ((has["out"][i, last].double() - near.double()).abs() <= off).all()
    assert ((has["lse"][i, last] - near_lse).double().abs() <= 2 * (total + 4 * U * (1 + near_lse.abs()))).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("by_words", [False, True])
def test_a_captured_step_follows_its_inputs(dtype, by_words, monkeypatch):
    if by_words:
        monkeypatch.setattr(kv_cache, "_tensors", None)
    has = step_of(dtype, lengths=(30_000, 5, 9000))
    sources, targets = ints([int(has["pages"][0, 0])]), ints([int(has["pages"][1, 200])])

    def step():
        mask, positions = kv_cache.draft_tree(has["parents"], has["lengths"], sync=False)
        places = has["lengths"][:, None] + torch.arange(has["n_drafted"], dtype=torch.int32, device="cuda")
        slots, q = kv_cache.append(has["keys"], has["values"], has["new_keys"].flatten(0, 1), has["new_values"].flatten(0, 1), has["pages"],
                                   torch.where(positions >= 0, places, -1).flatten(), sequences=has["sequences"],
                                   queries=has["queries"].flatten(0, 1), frequencies=has["frequencies"], turns=positions.flatten(), sync=False)
        out, lse = kv_cache.attend_tree(has["keys"], has["values"], q.view(has["queries"].shape), has["pages"], has["lengths"], positions, mask,
                                        cap=20.0, window=20_000, sync=False)
        kept = kv_cache.keep_path(has["keys"], has["values"], has["pages"], has["lengths"], has["paths"], sync=False)
        kv_cache.copy_pages(has["keys"], has["values"], sources, targets, sync=False)
        return mask.view(torch.int32), positions, slots, q, out, lse, kept, has["keys"], has["values"]

    start = has["keys"].clone(), has["values"].clone(), has["parents"].clone(), has["lengths"].clone(), has["queries"].clone()

    def reset(seed):
        for name, t in zip(("keys", "values", "parents", "lengths", "queries"), start):
            has[name].copy_(t)
        if seed:
            g = generator(seed)
            has["parents"].copy_(random_parents(3, has["n_drafted"], g, padding=2))
            has["lengths"].copy_(ints([20_001, 700, 3]))
            has["queries"].copy_(rows(has["queries"].shape, dtype, g))

    graphs = []
    for _ in range(2):  # two graphs, each with what it allocated while it was captured
        reset(0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(L.CuvsError, match="sync=False"):
                kv_cache.draft_tree(has["parents"], has["lengths"])
            got = step()
        graphs.append((graph, got))
    for seed in (0, 5, 6):
        reset(seed)
        want = [t.clone() for t in step()]
        for graph, got in graphs:
            reset(seed)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_graphs_at_once():
    """Both need a workspace of their own: they are replayed on two streams at a time."""
    steps = [Step(torch.bfloat16, lengths, 20, 1, 8, 128, 16, seed) for seed, lengths in enumerate(([40_000], [25_000, 3000]))]
    want = [[t.clone() for t in s.call()] for s in steps]
    graphs = []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = s.call(sync=False)
        graphs.append((graph, got))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for (graph, got), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                got[0].zero_(), got[1].zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_streams_and_threads():
    """Four threads with a stream each, through one handle."""
    steps = [Step(dtype, [9000 + 1000 * i, 40], 8 + i, 2, 4, 64, 16, i) for i, dtype in enumerate((torch.float16, torch.bfloat16, torch.float32, torch.float16))]
    want = [s.call() for s in steps]
    resources = Resources()
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for k in range(20):
                    got = steps[i].call(resources=resources, sync=k % 2 == 0)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        failed.append((i, k))
        except Exception as e:  # noqa: BLE001
            failed.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_another_stream_than_the_current_one():
    """The handle's stream, while the current one is another: results belong to it."""
    step = Step(torch.float16, [20_000, 100], 10, 2, 4, 128, 16)
    want = step.call()
    stream = torch.cuda.Stream()
    resources = Resources(stream=stream.cuda_stream)
    torch.cuda.synchronize()
    got = step.call(resources=resources, sync=False)
    kept = kv_cache.keep_path(step.keys.clone(), step.values.clone(), step.pages, step.lengths, ints([[0, 1], [2, -1]]), resources=resources, sync=False)
    mask, positions = kv_cache.draft_tree(step.parents, step.lengths, resources=resources, sync=False)
    resources.sync()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert kept.tolist() == [20_002, 101]
    assert torch.equal(mask.view(torch.int32), step.mask.view(torch.int32)) and torch.equal(positions, step.positions)


def test_workspaces_and_c_entries():
    """Every call from C; the handle's workspace, one of just the size that is asked for, one byte less, and a captured call."""
    from cuvs_b200.common import DLTensorRef
    step = Step(torch.float16, [30_000, 4000], 10, 2, 4, 64, 16, heads_outside=False)
    slopes = torch.linspace(0.001, 0.1, 8, device="cuda")
    want = step.call(scale=0.125, cap=9.0, slopes=slopes)
    lib, res = L.load(), Resources()
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    mask, positions = torch.empty_like(step.mask), torch.empty_like(step.positions)
    kept = [DLTensorRef(t) for t in (step.keys, step.values, step.queries, step.pages, step.lengths, step.positions, step.mask, slopes, out, lse)]
    k, v, q, p, n, at, m, s, o, l = (t.ref() for t in kept)
    size = C.c_size_t()
    L.check(lib.cuvsKvCacheAttendTreeWorkspace(res.handle, k, q, p, 0, C.byref(size)))
    assert size.value == kv_cache.attend_tree_workspace(step.keys, step.queries, step.pages) > 0

    def call(workspace):
        L.check(lib.cuvsKvCacheAttendTree(res.handle, k, v, q, p, n, at, m, 0.125, 0, 9.0, s, L.FilterStruct(0, 0), o, l, workspace))

    def good():
        torch.cuda.synchronize()
        found = torch.equal(out, want[0]) and torch.equal(lse, want[1])
        out.zero_(), lse.zero_()
        return found

    res.use_current_stream()
    call(None)
    assert good()
    frame = torch.full((size.value + 16,), 255, dtype=torch.uint8, device="cuda")
    exact, short = DLTensorRef(frame[:size.value]), DLTensorRef(frame[:size.value - 1])
    call(exact.ref())
    assert good() and (frame[size.value:] == 255).all()
    frame.fill_(255)
    with pytest.raises(L.CuvsError, match=f"{size.value - 1} bytes, but {size.value} are needed"):
        call(short.ref())
    torch.cuda.synchronize()
    assert (frame == 255).all() and (out == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res.use_current_stream()
        with pytest.raises(L.CuvsError, match="workspace of its own"):
            call(None)
        call(exact.ref())
    graph.replay()
    assert good()
    res.use_current_stream()

    refs = [DLTensorRef(t) for t in (step.parents, step.lengths, mask, positions)]
    L.check(lib.cuvsKvCacheDraftTree(res.handle, *(t.ref() for t in refs)))
    paths, lengths = ints([[1, 4], [0, -1]]), torch.empty_like(step.lengths)
    keys, values = step.keys.clone(), step.values.clone()
    wanted = kv_cache.keep_path(keys, values, step.pages, step.lengths, paths)
    refs2 = [DLTensorRef(t) for t in (step.keys, step.values, step.pages, step.lengths, paths, lengths)]
    L.check(lib.cuvsKvCacheKeepPath(res.handle, *(t.ref() for t in refs2)))
    torch.cuda.synchronize()
    assert torch.equal(mask.view(torch.int32), step.mask.view(torch.int32)) and torch.equal(positions, step.positions)
    assert torch.equal(lengths, wanted) and torch.equal(step.keys, keys) and torch.equal(step.values, values)
    sources, targets = ints([3]), ints([5])
    kv_cache.copy_pages(keys, values, sources, targets)
    refs3 = [DLTensorRef(t) for t in (step.keys, step.values, sources, targets)]
    L.check(lib.cuvsKvCacheCopyPages(res.handle, *(t.ref() for t in refs3)))
    new, turns, f = rows((2, 2, 64), torch.float16, generator(3)), ints([[7, 9], [1, 0]]), torch.rand(32, device="cuda")
    axes, where, slots = ints([i % 2 for i in range(32)]), ints([50, 60]), torch.empty(2, dtype=torch.int64, device="cuda")
    want_slots, _ = kv_cache.append(keys, values, new, new, step.pages, where, frequencies=f, turns=turns, axes=axes, interleaved=True)
    refs4 = [DLTensorRef(t) for t in (step.keys, step.values, new, new, step.pages, where)]
    more = [DLTensorRef(t) for t in (f, slots, turns, axes)]
    L.check(lib.cuvsKvCacheAppendTurned(res.handle, *(t.ref() for t in refs4), None, None, more[0].ref(), True, more[1].ref(), None, more[2].ref(),
                                        more[3].ref()))
    torch.cuda.synchronize()
    assert torch.equal(slots, want_slots) and torch.equal(step.keys, keys) and torch.equal(step.values, values)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_offsets_that_pass_32_bits(dtype):
    """Pages behind 4 GB of a cache, in every call that reads or writes one."""
    n_pages, page, dim = 5_000_000 if dtype == torch.float16 else 2_500_000, 16, 64
    keys, values = (torch.empty((n_pages, page, 1, dim), dtype=dtype, device="cuda") for _ in range(2))
    used = ints([n_pages - 1 - 3 * i for i in range(60)])
    g = generator(2)
    for t in (keys, values):
        t[used.long()] = rows((60, page, 1, dim), dtype, g)
    step = Step(dtype, [900], 9, 1, 4, dim, page)
    step.keys, step.values, step.pages = keys[used.long()], values[used.long()], torch.arange(60, dtype=torch.int32, device="cuda")[None]
    small = step.call()
    step.keys, step.values, step.pages = keys, values, used[None]
    assert all(torch.equal(a, b) for a, b in zip(small, step.call()))
    row = keys[used[57].long(), 3].clone()
    kept = kv_cache.keep_path(keys, values, step.pages, step.lengths, ints([[57 * 16 + 3 - 900]]))
    assert kept.tolist() == [901] and torch.equal(keys[used[56].long(), 4], row)
    kv_cache.copy_pages(keys, values, used[:2], ints([n_pages - 2, n_pages - 3]))
    assert torch.equal(keys[n_pages - 2], keys[used[0].long()]) and torch.equal(values[n_pages - 3], values[used[1].long()])


def test_parameters_and_other_subclasses():
    step = Step(torch.float16, [100], 4, 2, 2, 64, 16)
    want = step.call()
    with torch.no_grad():
        got = step.call(queries=torch.nn.Parameter(step.queries), keys=torch.nn.Parameter(step.keys))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and type(got[0]) is torch.Tensor


def test_refused_calls_do_nothing():
    step = Step(torch.float16, [100], 4, 2, 2, 64, 16)
    for options, message in (({"mask": step.mask[:, :3]}, "mask: expected shape"), ({"positions": step.positions.long()}, "expected int32"),
                             ({"slopes": torch.ones(3, device="cuda")}, "slopes"), ({"values": step.values[1:]}, "same shape"),
                             ({"workspace": torch.empty(16, device="cuda")}, "uint8")):
        out = torch.full_like(step.queries, 7.0)
        with pytest.raises(L.CuvsError, match=message):
            step.call(out=out, **options)
        assert (out == 7).all()
    for cap in (0.0, -1.0, math.inf, math.nan, 1e-40):
        with pytest.raises(ValueError, match="cap"):
            step.call(cap=cap)
    with pytest.raises(ValueError, match="axes go with turns"):
        kv_cache.append(step.keys, step.values, step.keys[0], step.values[0], step.pages, step.lengths, axes=ints([0]))
    with pytest.raises(L.CuvsError, match="lengths' own memory"):
        kv_cache.keep_path(step.keys, step.values, step.pages, step.lengths, ints([[0]]), kept=step.lengths)
