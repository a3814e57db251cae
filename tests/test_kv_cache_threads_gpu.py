"""GPU tests of attention over a paged cache called from several threads and on several streams through one handle, beside searches."""
import ctypes as C
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(shape, dtype, g, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def shared(lengths, g, n_queries=1, heads=2, n_heads=8, dim=64, page_size=16, dtype=torch.float16):
    """A cache with sequences whose units lie in several blocks' shares, so that the call needs a workspace; [queries], pages, lengths."""
    from cuvs_b200 import kv_cache
    used = [-(-n // page_size) for n in lengths]
    keys, values = (rows((sum(used), page_size, heads, dim), dtype, g) for _ in range(2))
    pages = torch.full((len(lengths), max(used)), -1, dtype=torch.int32, device="cuda")
    order, at = torch.randperm(sum(used), generator=g, device="cuda").int(), 0
    for i, n in enumerate(used):
        pages[i, :n] = order[at:at + n]
        at += n
    queries = [rows((len(lengths), n_heads, dim), dtype, g) for _ in range(n_queries)]
    assert kv_cache.attention_workspace(keys, queries[0], pages) > 0
    return keys, values, queries, pages, ints(lengths)


def handle_stream(resources):
    from cuvs_b200 import _lib as L
    at = C.c_void_p()
    L.check(L.load().cuvsStreamGet(resources.handle, C.byref(at)))
    return at.value or 0


def test_calls_leave_the_stream_of_the_handle_alone():
    """It belongs to the thread that searches through the handle; `sync` waits for the calls of the thread that asks all the same."""
    from cuvs_b200 import Resources, kv_cache
    g = generator(1)
    keys, values, (q,), pages, n = shared([200_000, 100_000], g)
    resources = Resources()
    resources.use_current_stream()
    before = handle_stream(resources)
    side = torch.cuda.Stream()
    want = kv_cache.attention(keys, values, q, pages, n)
    slots = torch.randint(0, 1000, (2, 8, 20), generator=g, device="cuda")
    torch.cuda.synchronize()
    for sync in (True, False):
        with torch.cuda.stream(side):
            for _ in range(20):
                got = kv_cache.attention(keys, values, q, pages, n, resources=resources, sync=sync)
                kv_cache.attend_candidates(keys, values, q, slots, resources=resources, sync=sync)
                kv_cache.merge_parts(torch.stack((got[0], got[0])), torch.stack((got[1], got[1])), resources=resources, sync=sync)
                kv_cache.append(keys, values, keys[0, :2], values[0, :2], pages, ints([-1, -1]), resources=resources, sync=sync)
            got = kv_cache.attention(keys, values, q, pages, n, resources=resources, sync=sync)
        assert handle_stream(resources) == before
        resources.sync()
        assert side.query()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_search_and_attention_through_one_handle_at_once():
    """One thread searches on its stream, others attend on theirs, all through the default handle of the device."""
    from cuvs_b200 import ivf_pq, kv_cache
    rng = np.random.default_rng(0)
    data = torch.from_numpy(rng.standard_normal((20_000, 32), dtype=np.float32)).cuda()
    asked = [torch.from_numpy(rng.standard_normal((m, 32), dtype=np.float32)).cuda() for m in (1, 100, 3000)]
    index = ivf_pq.build(ivf_pq.IndexParams(n_lists=64, pq_dim=16, kmeans_n_iters=4), data)
    params = ivf_pq.SearchParams(n_probes=16)
    want_found = [ivf_pq.search(params, index, q, 10) for q in asked]
    g = generator(2)
    keys, values, queries, pages, n = shared([30_000, 4000, 70], g, n_queries=3)
    want = [kv_cache.attention(keys, values, q, pages, n) for q in queries]
    torch.cuda.synchronize()
    wrong, done = [], threading.Event()

    def search():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(300):
                    d, found = ivf_pq.search(params, index, asked[i % 3], 10)
                    if not (torch.equal(d, want_found[i % 3][0]) and torch.equal(found, want_found[i % 3][1])):
                        wrong.append(f"search {i}")
        except Exception as e:
            wrong.append(repr(e))
        done.set()

    def attend(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not done.is_set():
                    out, lse = kv_cache.attention(keys, values, queries[i], pages, n)
                    if not (torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])):
                        wrong.append(f"attention of {i}")
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=search)] + [threading.Thread(target=attend, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:5]


PER_THREAD = 2  # cudaStreamPerThread: one value for a stream of every thread


def test_the_stream_of_each_thread():
    """cudaStreamPerThread through one handle: every thread's stream has a workspace to itself."""
    from cuvs_b200 import Resources, kv_cache
    g = generator(3)
    keys, values, queries, pages, n = shared([60_000, 9000, 20, 0, 30_000], g, n_queries=4, dim=128)
    want = [kv_cache.attention(keys, values, q, pages, n) for q in queries]
    resources = Resources(PER_THREAD)
    places = [[(torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")) for _ in range(10)] for q in queries]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(queries)), []

    def work(i):
        try:
            start.wait(60)
            for _ in range(20):
                for out, lse in places[i]:
                    kv_cache.attention(keys, values, queries[i], pages, n, out=out, lse=lse, resources=resources, sync=False)
                resources.sync()
                wrong.extend(i for out, lse in places[i] if not (torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])))
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(queries))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:5]


class NewStream:
    """A stream of the runtime's own making, not one of torch's pool."""

    def __init__(self):
        at = C.c_uint64()
        assert int(torch.cuda.cudart().cudaStreamCreate(C.addressof(at))) == 0
        self.value = at.value

    def current(self):
        return torch.cuda.stream(torch.cuda.ExternalStream(self.value))

    def destroy(self):
        assert int(torch.cuda.cudart().cudaStreamDestroy(self.value)) == 0


def test_streams_that_are_destroyed_with_work_in_them():
    """The next stream may get the handle of one whose work goes on; more streams than the handle has workspaces for."""
    from cuvs_b200 import kv_cache
    g = generator(4)
    keys, values, queries, pages, n = shared([60_000, 9000, 20, 30_000], g, n_queries=5)
    want = [kv_cache.attention(keys, values, q, pages, n) for q in queries]
    places = [(torch.empty_like(queries[0]), torch.empty(queries[0].shape[:2], device="cuda")) for _ in range(150)]
    torch.cuda.synchronize()
    alive = []
    for i, (out, lse) in enumerate(places):
        stream = NewStream()
        with stream.current():
            kv_cache.attention(keys, values, queries[i % 5], pages, n, out=out, lse=lse, sync=False)
        if i % 2:
            stream.destroy()
        else:
            alive.append(stream)
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(places):
        assert torch.equal(out, want[i % 5][0]) and torch.equal(lse, want[i % 5][1]), i
    for stream in alive:
        stream.destroy()


def test_a_workspace_that_grows_behind_queued_work():
    from cuvs_b200 import Resources, kv_cache
    g = generator(5)
    small, large = shared([30_000], g), shared([60_000, 50_000, 40_000], g, heads=4, n_heads=16, dim=128)
    need = [kv_cache.attention_workspace(c[0], c[2][0], c[3]) for c in (small, large)]
    assert 0 < need[0] < need[1]
    want = [kv_cache.attention(c[0], c[1], c[2][0], c[3], c[4]) for c in (small, large)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        resources = Resources()
        with torch.cuda.stream(side):
            got = [kv_cache.attention(c[0], c[1], c[2][0], c[3], c[4], resources=resources, sync=False) for c in (small, small, small, large, small)]
        resources.sync()
        for a, w in zip(got, [want[0]] * 3 + [want[1], want[0]]):
            assert torch.equal(a[0], w[0]) and torch.equal(a[1], w[1])


@pytest.mark.parametrize("elsewhere", [False, True])
def test_calls_on_other_streams_while_a_graph_is_captured(elsewhere):
    """A call that is not captured may need a workspace of its stream just then: neither it nor the capture fails, whether the capturing
    thread makes it or another one."""
    from cuvs_b200 import Resources, kv_cache
    g = generator(6)
    small, large = shared([30_000], g), shared([60_000, 50_000, 40_000], g, heads=4, n_heads=16, dim=128)
    want = [kv_cache.attention(c[0], c[1], c[2][0], c[3], c[4]) for c in (small, large)]
    places = [(torch.empty_like(w[0]), torch.empty_like(w[1])) for w in want]
    resources, side, raised = Resources(), torch.cuda.Stream(), []
    torch.cuda.synchronize()

    def calls():
        try:
            with torch.cuda.stream(side):
                for c, (out, lse) in zip((small, large), places):        # the second one wants more
                    kv_cache.attention(c[0], c[1], c[2][0], c[3], c[4], out=out, lse=lse, resources=resources, sync=False)
        except Exception as e:
            raised.append(repr(e))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = kv_cache.attention(small[0], small[1], small[2][0], small[3], small[4], sync=False)
        if elsewhere:
            thread = threading.Thread(target=calls)
            thread.start()
            thread.join()
        else:
            calls()
        second = kv_cache.attention(large[0], large[1], large[2][0], large[3], large[4], sync=False)
    assert not raised, raised
    graph.replay()
    torch.cuda.synchronize()
    for got in (places, (first, second)):
        for a, w in zip(got, want):
            assert torch.equal(a[0], w[0]) and torch.equal(a[1], w[1])


FIRST = """
import torch
from cuvs_b200 import kv_cache
k, v = (torch.randn((4000, 16, 2, 64), device="cuda").bfloat16() for _ in range(2))
q, new = torch.randn((1, 8, 64), device="cuda").bfloat16(), torch.randn((1, 2, 64), device="cuda").bfloat16()
pages = torch.arange(4000, dtype=torch.int32, device="cuda")[None]
n, place = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (60_000, 61_000))
slots = torch.arange(1000, device="cuda").expand(1, 8, 1000).contiguous()
torch.cuda.synchronize()

def step():
    at, _ = kv_cache.append(k, v, new, new, pages, place, sync=False)
    near = kv_cache.attention(k, v, q, pages, n, sync=False)
    far = kv_cache.attend_candidates(k, v, q, slots, sync=False)
    return (at, *kv_cache.merge_parts(torch.stack((near[0], far[0])), torch.stack((near[1], far[1])), sync=False))

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("ok")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout + done.stderr
