"""GPU tests of the way to the library that does without DLPack's table of exchange functions: tensors described by words, as where torch has
no such table."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def rows(shape, dtype, g, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_the_four_calls_and_a_captured_step(dtype, monkeypatch):
    from cuvs_b200 import _lib as L
    from cuvs_b200 import kv_cache
    g = torch.Generator(device="cuda").manual_seed(1)
    n_pages, page, heads, n_heads, dim = 4000, 16, 2, 6, 64
    keys, values = (rows((n_pages, heads, page, dim), dtype, g).permute(0, 2, 1, 3) for _ in range(2))
    lengths = ints([40_000, 15_000, 30])
    pages = torch.full((3, 2600), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    pages[0, :2500], pages[1, :940], pages[2, :2] = order[:2500], order[2500:3440], order[3440:3442]
    fused = rows((3, n_heads + 2 * heads, dim), dtype, g)
    q, new_k, new_v = fused[:, :n_heads], fused[:, n_heads:n_heads + heads], fused[:, n_heads + heads:]
    f = torch.tensor([10000.0 ** (-i / 24) for i in range(24)], dtype=torch.float64, device="cuda")
    candidates = torch.randint(-5, n_pages * page + 100, (3, n_heads, 77), generator=g, device="cuda")
    bits = torch.randint(0, 2 ** 32, (n_pages * page // 32,), generator=g, device="cuda").to(torch.uint32)

    def step(sync=False):
        slots, turned = kv_cache.append(keys, values, new_k, new_v, pages, lengths - 1, queries=q, frequencies=f, interleaved=True, sync=sync)
        near = kv_cache.attention(keys, values, turned, pages, lengths, scale=0.2, window=25_000, filter=bits, sync=sync)
        far = kv_cache.attend_candidates(keys, values, turned, candidates, scale=0.2, filter=bits, sync=sync)
        return (slots, turned, *near, *far, *kv_cache.merge_parts(torch.stack((near[0], far[0])), torch.stack((near[1], far[1])), sync=sync))

    assert kv_cache.attention_workspace(keys, q, pages, 25_000) > 0
    want = step(True)
    monkeypatch.setattr(kv_cache, "_tensors", None)
    for got in (step(True), step(False)):
        kv_cache.default_resources().sync()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(L.CuvsError, match="sync=False"):
            kv_cache.attention(keys, values, q, pages, lengths)
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(L.CuvsError, match="same shape"):
        kv_cache.attention(keys, values[1:], q, pages, lengths)
