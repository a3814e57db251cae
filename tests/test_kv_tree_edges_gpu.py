"""GPU tests of attention of drafted tokens at the ends of its ranges: very long sequences, values and scores that are no numbers."""
import ctypes as C
import math
import threading

import pytest
import torch

from cuvs_b200 import Resources
from cuvs_b200 import _lib as L
from cuvs_b200 import kv_cache
from test_kv_tree_gpu import DTYPES, Step, U, check, generator, ints, needs_a_gpu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,n_sequences,m,group,dim", [
    (torch.float16, 1, 1024, 40, 64),    # more blocks of 256 rows than SMs: each of them goes through all keys
    (torch.bfloat16, 1, 1024, 20, 256),  # of 128 rows
    (torch.float16, 300, 2, 4, 128),     # more sequences than SMs, every other tile for each of two sums
    (torch.float16, 150, 50, 4, 72)])    # a tile for both
def test_sums_of_long_sequences_lose_nothing(dtype, n_sequences, m, group, dim):
    """Values around 1, so that whatever a sum loses on its way shows: outputs are not too small on average."""
    n, page = 200_000, 64
    g = generator(dim)
    n_pages = (n + m) // page + 1
    keys = torch.randn((n_pages, page, 1, dim), generator=g, device="cuda").to(dtype)
    columns = 1 + torch.rand(dim, generator=g, device="cuda")
    values = (columns * (1 + 0.25 * torch.rand((n_pages, page, 1, dim), generator=g, device="cuda"))).to(dtype)
    pages = torch.arange(n_pages, device="cuda", dtype=torch.int32).expand(n_sequences, n_pages)
    lengths = ints([n] * n_sequences)
    queries = torch.randn((n_sequences, m, group, dim), generator=g, device="cuda").to(dtype)
    mask, positions = kv_cache.draft_tree(ints([[-1] * m]).expand(n_sequences, m), lengths)
    out, lse = kv_cache.attend_tree(keys, values, queries, pages, lengths, positions, mask)
    off, lse_off = [], []
    for i, j in ((0, 0), (n_sequences - 1, m // 2), (n_sequences // 2, m - 1)):
        sees = torch.cat((torch.arange(n, device="cuda"), torch.tensor([n + j], device="cuda")))
        k, v = (t.view(-1, dim)[sees].double() for t in (keys, values))
        s = queries[i, j].double() @ k.t() * dim ** -0.5
        l = torch.logsumexp(s, 1)
        o = torch.exp(s - l[:, None]) @ v
        off.append((out[i, j].double() - o) / o)
        lse_off.append(lse[i, j].double() - l)
    # A product with tensor cores adds 16 terms to a sum, and may cut off 2^-24 of it for each of 17: 32 tiles of 64 keys in pairs of weights are 256 of them.
    chain = 256 * 17 * U
    # scores of up to 7, in powers of two, from products of `dim` terms; exponentials to 2^-21; a sum of 3,200 tiles of 64
    total = (dim + 6) * U * 30 + 2.0 ** -20 + (n / 64 + 100) * U
    half = torch.finfo(dtype).eps / 2
    off, lse_off = torch.stack(off), torch.stack(lse_off)
    assert off.abs().max() <= 1.01 * (half + chain + 2 * total)
    # roundings are spread evenly over half a step either way, those of different columns independently
    assert off.mean().abs() <= chain + 6 * half / math.sqrt(3 * dim)
    assert lse_off.abs().max() <= total + 4 * U * 14


# ---- waits that run out -------------------------------------------------------------------------------------------------------

@pytest.fixture
def giving_up():
    """Sets a limit of about a millisecond, and a tile of each block whose keys nobody is told of; what it yields does so, or ends it with 0."""
    def wait_test(tile):
        L.check(L.load().cuvsB200SetTreeWaitTest(1000 if tile else 0, tile))

    yield wait_test
    torch.cuda.synchronize()
    wait_test(0)


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256)])
@pytest.mark.parametrize("lengths,m", [([(7 * i) % 700 for i in range(200)], 10),   # more units than blocks
                                       ([(7 * i) % 700 for i in range(200)], 80),
                                       ([40_000, 5, 9000], 10), ([40_000, 5, 9000], 80)])
@pytest.mark.parametrize("tile", [1, 2, 5])
def test_a_call_that_gives_up_writes_nothing_elsewhere(giving_up, dtype, dim, lengths, m, tile):
    """What the workspace holds from before must not say where outputs go."""
    step = Step(dtype, lengths, m, 2, 4, dim, 16)
    want = step.call()
    n = len(lengths)
    frame, lse_frame = torch.full((n + 2, m, 8, dim), 7.0, dtype=dtype, device="cuda"), torch.full((n + 2, m, 8), 7.0, device="cuda")
    out, lse = frame[1:-1], lse_frame[1:-1]
    words = kv_cache.attend_tree_workspace(step.keys, step.queries, step.pages) // 4
    # entries of units behind the last sequence, with parts
    workspace = ints([n, 1, 1, 0]).repeat(words // 4 + 1)[:words].view(torch.uint8)
    giving_up(tile)
    with pytest.raises(L.CuvsError, match="gave up on a wait"):
        step.call(out=out, lse=lse, workspace=workspace)
    giving_up(0)
    for t in (frame, lse_frame):
        assert (t[0] == 7).all() and (t[-1] == 7).all()
    got = step.call(out=out, lse=lse, workspace=workspace)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_limits_that_a_busy_gpu_would_reach_are_refused():
    with pytest.raises(L.CuvsError, match="at least 1000"):
        L.check(L.load().cuvsB200SetTreeWaitTest(999, 0))


def small_step(seed=0, **options):
    return Step(torch.float16, [3000, 100], 9, 2, 4, 64, 16, seed, **options)


def test_who_gave_up_is_told(giving_up):
    """Two streams of one handle: a call of one of them gives up, whoever waits first."""
    step, resources = small_step(), Resources()
    want = step.call()
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def on(stream, **options):
        with torch.cuda.stream(stream):
            return step.call(resources=resources, **options)

    giving_up(1)
    on(one, sync=False)
    torch.cuda.synchronize()
    giving_up(0)
    assert all(torch.equal(a, b) for a, b in zip(on(other), want))
    with torch.cuda.stream(other):
        kv_cache.draft_tree(step.parents, step.lengths, resources=resources)
    with pytest.raises(L.CuvsError, match="gave up on a wait: the results of a call on this stream"):
        on(one)
    assert all(torch.equal(a, b) for a, b in zip(on(one), want))
    # another call that waits, and the handle's own wait
    for wait in (lambda: kv_cache.draft_tree(step.parents, step.lengths, resources=resources), resources.sync):
        giving_up(1)
        on(one, sync=False)
        torch.cuda.synchronize()
        giving_up(0)
        with torch.cuda.stream(one), pytest.raises(L.CuvsError, match="gave up on a wait"):
            wait()
    assert all(torch.equal(a, b) for a, b in zip(on(one), want))


def test_threads_are_told_of_their_own_calls(giving_up):
    """Three threads with a stream each, through one handle; the calls of all of them give up."""
    steps, resources = [small_step(i) for i in range(3)], Resources()
    torch.cuda.synchronize()
    giving_up(1)
    told, barrier = [None] * 3, threading.Barrier(3)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            steps[i].call(resources=resources, sync=False)
            torch.cuda.synchronize()
            barrier.wait()
            try:
                kv_cache.draft_tree(steps[i].parents, steps[i].lengths, resources=resources)
            except L.CuvsError as e:
                told[i] = str(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(t is not None and "a call on this stream" in t for t in told)


def test_a_c_caller_is_told(giving_up):
    from cuvs_b200.common import DLTensorRef
    step, resources, lib = small_step(heads_outside=False), Resources(), L.load()
    want = step.call()
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    refs = [DLTensorRef(t) for t in (step.keys, step.values, step.queries, step.pages, step.lengths, step.positions, step.mask, out, lse)]
    resources.use_current_stream()

    def call():
        L.check(lib.cuvsKvCacheAttendTree(resources.handle, *(r.ref() for r in refs[:7]), 0.125, 0, 0.0, None, L.FilterStruct(0, 0), refs[7].ref(),
                                          refs[8].ref(), None))

    giving_up(1)
    call()
    torch.cuda.synchronize()
    giving_up(0)
    with pytest.raises(L.CuvsError, match="gave up on a wait"):
        L.check(lib.cuvsStreamSync(resources.handle))
    L.check(lib.cuvsStreamSync(resources.handle))
    call()
    L.check(lib.cuvsStreamSync(resources.handle))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_captured_call_that_gives_up(giving_up):
    """It may be replayed on any stream: the next wait of the handle is told, and says what it was."""
    step, resources = small_step(), Resources()
    want = step.call(resources=resources)
    graph = torch.cuda.CUDAGraph()
    giving_up(1)
    with torch.cuda.graph(graph):
        step.call(resources=resources, sync=False)
    giving_up(0)
    assert all(torch.equal(a, b) for a, b in zip(step.call(resources=resources), want))
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(L.CuvsError, match="results of a captured call"):
        step.call(resources=resources)
    assert all(torch.equal(a, b) for a, b in zip(step.call(resources=resources), want))


def test_more_streams_than_there_are_words(giving_up):
    """A page has a word for each of 1,008 streams; those behind share one."""
    from cuvs_b200.common import DLTensorRef
    step, resources, lib = small_step(heads_outside=False), Resources(), L.load()
    want = step.call()
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    workspace = torch.empty(kv_cache.attend_tree_workspace(step.keys, step.queries, step.pages), dtype=torch.uint8, device="cuda")
    refs = [DLTensorRef(t) for t in (step.keys, step.values, step.queries, step.pages, step.lengths, step.positions, step.mask, out, lse, workspace)]
    torch.cuda.synchronize()
    cudart = torch.cuda.cudart()

    def call():
        L.check(lib.cuvsKvCacheAttendTree(resources.handle, *(r.ref() for r in refs[:7]), 0.125, 0, 0.0, None, L.FilterStruct(0, 0), refs[7].ref(),
                                          refs[8].ref(), refs[9].ref()))

    for i in range(1050):
        stream = C.c_uint64()
        assert int(cudart.cudaStreamCreate(C.addressof(stream))) == 0
        L.check(lib.cuvsStreamSet(resources.handle, stream.value))
        for fails in ((True, False) if i in (0, 1007, 1008, 1049) else (False,)):
            giving_up(1 if fails else 0)
            call()
            giving_up(0)
            if fails:
                with pytest.raises(L.CuvsError, match="gave up on a wait"):
                    L.check(lib.cuvsStreamSync(resources.handle))
            else:
                L.check(lib.cuvsStreamSync(resources.handle))
        L.check(lib.cuvsStreamSet(resources.handle, None))
        assert int(cudart.cudaStreamDestroy(stream.value)) == 0
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


# ---- what is no number --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim", [(2, 2, 64), (9, 8, 64), (40, 8, 128), (9, 5, 256)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_token_that_is_none_attends_to_nothing(dtype, m, group, dim, bad):
    """Beside values of its sequence that are no numbers, in tiles that all other tokens see whole; in one share and in several."""
    for lengths in ([300, 40, 300], [20_000], [130] * 300):
        step = Step(dtype, lengths, m, 2, group, dim, 16, padding=1)
        slot = step.allowed()[1][0]
        assert lengths[0] >= 128  # place 70 lies in a tile before the drafted tokens
        step.values[slot[70] // 16, slot[70] % 16] = bad
        out, lse = step.call()
        none = step.positions < 0
        assert none.any() and (out[none] == 0).all() and (lse[none] == -math.inf).all()
        assert not out[0][~none[0]].isfinite().any() and lse[~none].isfinite().all()
        assert out[1:][~none[1:]].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim", [(2, 2, 64), (9, 8, 64), (40, 8, 128), (9, 5, 256)])
@pytest.mark.parametrize("lengths", [[300, 40], [20_000, 300], [130] * 300])
def test_scores_that_are_no_numbers(dtype, m, group, dim, lengths):
    """Of a token's query, and of all keys that one share of many has: whoever has such a score has no answer, in as many parts as it comes."""
    step = Step(dtype, lengths, m, 2, group, dim, 16)
    want, want_lse = step.call()
    step.queries[0, 1, 3 % (2 * group)] = math.nan
    out, lse = step.call()
    touched = torch.zeros_like(lse, dtype=torch.bool)
    touched[0, 1, 3 % (2 * group)] = True
    assert out[touched].isnan().all() and lse[touched].isnan().all()
    assert torch.equal(out[~touched], want[~touched]) and torch.equal(lse[~touched], want_lse[~touched])
    slot = step.allowed()[1][0, :lengths[0] * 3 // 4]
    step.keys[slot // 16, slot % 16, 0] = math.nan  # of the first key head
    out, lse = step.call()
    touched[0, :, :group] = True
    assert out[touched].isnan().all() and lse[touched].isnan().all()
    assert torch.equal(out[~touched], want[~touched]) and torch.equal(lse[~touched], want_lse[~touched])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim", [(1, 2, 64), (3, 8, 128), (20, 8, 64), (20, 8, 128), (3, 8, 256)])
def test_an_infinite_value_of_a_small_weight(dtype, m, group, dim):
    """Weights from 1 down to 2^-30 of the largest, in a tile that all rows see whole: the output is infinite, of the value's sign."""
    n = 300
    step = Step(dtype, [200] * n, m, 1, group, dim, 16)
    slot = step.allowed()[1]
    step.queries.zero_()
    step.queries[..., 0] = 1.0
    step.keys.zero_()
    step.keys[..., 0] = -100.0
    row = torch.arange(n, device="cuda")
    first, small = slot[:, 5], slot[:, 70]
    step.keys[first // 16, first % 16, 0, 0] = 0.0
    weight = torch.linspace(0.0, 29.9 * math.log(2), n, device="cuda").to(dtype)
    weight = torch.where(weight.float() > 29.95 * math.log(2), 29.9 * math.log(2) - 0.05, weight.float()).to(dtype)  # (rounded up)
    step.keys[small // 16, small % 16, 0, 0] = -weight
    step.values[small // 16, small % 16, 0, 3] = torch.where(row % 2 == 0, math.inf, -math.inf).to(dtype)
    out, lse = step.call(scale=1.0)
    want = torch.where(row % 2 == 0, math.inf, -math.inf)[:, None, None].expand(n, m, group)
    assert torch.equal(out[..., 3].float(), want) and out[..., :3].isfinite().all() and out[..., 4:].isfinite().all() and lse.isfinite().all()


# ---- sums that are set aside --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,group,dim", [(3, 4, 128), (20, 8, 64), (20, 8, 104), (9, 4, 256)])
@pytest.mark.parametrize("rising", [False, True])
def test_lengths_around_the_turns_at_setting_sums_aside(dtype, m, group, dim, rising):
    """More units than blocks, of about 16, 32, 48, .. tiles; scores whose largest stays, or grows by many powers of two on the way."""
    lengths = [64 * tiles + more for tiles in (15, 16, 17, 31, 32, 33, 47, 48, 64, 65, 96, 97) for more in (-m, -1, 0, 17)]
    step = Step(dtype, lengths, m, 5, group, dim, 16, dim, padding=1)
    if rising:
        slot = step.allowed()[1]
        step.queries.abs_()
        for i, n in enumerate(lengths):
            s = slot[i, :n + m]
            rise = torch.linspace(0.0, 40.0 / dim ** 0.5, n + m, device="cuda")
            step.keys[s // 16, s % 16] = (step.keys[s // 16, s % 16].float() * 0.1 + rise[:, None, None]).to(dtype)
    check(step)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_no_numbers_beside_sums_that_were_set_aside(dtype):
    """In the tiles around a turn, of a sequence's last tokens and of drafted ones that only some rows see."""
    for m, group, dim in ((3, 4, 128), (20, 8, 64), (9, 4, 256)):
        lengths = [64 * tiles - 20 for tiles in (17, 33, 49, 65)] * 20
        step = Step(dtype, lengths, m, 3, group, dim, 16, padding=1, spread=0.1)
        seen, slot, _ = step.allowed()
        touched = torch.zeros_like(step.positions, dtype=torch.bool)
        for i, n in enumerate(lengths):
            if i % 3 == 0:
                step.values[slot[i, n + 1] // 16, slot[i, n + 1] % 16] = math.inf
                touched[i] = seen[i, :, n + 1]
        exact, exact_lse, off, lse_off = step.exact()
        out, lse = step.call()
        none = step.positions < 0
        clean = ~touched & ~none
        assert touched.any() and clean.any() and (out[none] == 0).all() and not out[touched].isfinite().any()
        assert ((out[clean].double() - exact[clean]).abs() <= off[clean]).all()
        assert ((lse[~none].double() - exact_lse[~none]).abs() <= lse_off[~none]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sums_set_aside_in_calls_of_several_streams_and_graphs(dtype):
    """Calls of one handle at a time on several streams, and captured ones, each with room of its own for what it sets aside."""
    steps = [Step(dtype, [30_000 + 7000 * i] * 2, 40, 1, 8, 128, 16, i) for i in range(3)]
    want = [s.call() for s in steps]
    graphs = []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = s.call(sync=False)
        graphs.append((graph, got))
    streams = [torch.cuda.Stream() for _ in range(6)]
    torch.cuda.synchronize()
    for _ in range(5):
        live = []
        for i in range(3):
            with torch.cuda.stream(streams[i]):
                live.append(steps[i].call(sync=False))
            with torch.cuda.stream(streams[3 + i]):
                graphs[i][0].replay()
        torch.cuda.synchronize()
        for i in range(3):
            assert all(torch.equal(a, b) for a, b in zip(live[i], want[i]))
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want[i]))
