"""GPU tests of what the C entries of attention over a paged cache do with workspaces, and of frequencies of 32 bits."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def rows(shape, dtype, g, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def test_workspaces_of_c_calls():
    """A list that many blocks share: the handle's workspace, one of just the size that is asked for, one byte less, and a captured call."""
    from cuvs_b200 import Resources, kv_cache
    from cuvs_b200 import _lib as L
    from cuvs_b200.common import DLTensorRef
    g = torch.Generator(device="cuda").manual_seed(1)
    keys, values, q = (rows(shape, torch.float16, g) for shape in ((3800, 16, 2, 64), (3800, 16, 2, 64), (1, 8, 64)))
    pages, lengths = torch.arange(3800, dtype=torch.int32, device="cuda")[None], torch.tensor([60_000], dtype=torch.int32, device="cuda")
    want = kv_cache.attention(keys, values, q, pages, lengths, scale=0.125)
    lib, res = L.load(), Resources()
    out, lse = torch.empty_like(q), torch.empty((1, 8), device="cuda")
    kept = [DLTensorRef(t) for t in (keys, values, q, pages, lengths, out, lse)]
    k, v, qq, p, n, o, l = (t.ref() for t in kept)
    size = C.c_size_t()
    L.check(lib.cuvsKvCacheAttentionWorkspace(res.handle, k, qq, p, 0, C.byref(size)))
    assert size.value == kv_cache.attention_workspace(keys, q, pages) > 0

    def call(workspace):
        L.check(lib.cuvsKvCacheAttention(res.handle, k, v, qq, p, n, 0.125, 0, L.FilterStruct(0, 0), o, l, workspace))

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
    with pytest.raises(L.CuvsError, match="are needed"):
        kv_cache.attention(keys, values, q, pages, lengths, workspace=frame[:16])
    # captured: refused without a workspace of its own, and the capture goes on
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res.use_current_stream()
        with pytest.raises(L.CuvsError, match="workspace of its own"):
            call(None)
        call(exact.ref())
    graph.replay()
    assert good()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_frequencies_of_32_bits(dtype, interleaved):
    """They are taken as the numbers that they are: the same numbers in 64 bits give the same rows, over the queries themselves too."""
    from cuvs_b200 import kv_cache
    g = torch.Generator(device="cuda").manual_seed(2)
    keys, values = rows((20, 16, 2, 96), dtype, g), rows((20, 16, 2, 96), dtype, g)
    q, k, v = rows((40, 6, 96), dtype, g), rows((40, 2, 96), dtype, g), rows((40, 2, 96), dtype, g)
    pages = torch.full((2, 70_000), -1, dtype=torch.int32, device="cuda")
    pages[0, 62_500:62_510] = torch.arange(10, dtype=torch.int32, device="cuda")
    pages[1, :10] = torch.arange(10, 20, dtype=torch.int32, device="cuda")
    sequences = torch.arange(40, dtype=torch.int32, device="cuda") % 2
    positions = torch.arange(40, dtype=torch.int32, device="cuda") * 3 + torch.where(sequences == 0, 1_000_000, 0).int()
    f = torch.tensor([10000.0 ** (-i / 41) for i in range(41)], dtype=torch.float32, device="cuda")
    slots, want = kv_cache.append(keys, values, k, v, pages, positions, sequences=sequences, queries=q, frequencies=f.double(), interleaved=interleaved)
    assert (slots >= 0).all()
    written = keys.clone()
    keys.zero_()
    again, got = kv_cache.append(keys, values, k, v, pages, positions, sequences=sequences, queries=q, frequencies=f, interleaved=interleaved, rotated=q)
    assert got is q and torch.equal(q, want) and torch.equal(again, slots)
    at = slots
    assert torch.equal(keys[at // 16, at % 16], written[at // 16, at % 16])
