"""GPU tests of attention of drafted tokens at the ends of its ranges: very long sequences, values and scores that are no numbers."""
import math

import pytest
import torch

from cuvs_b200 import _lib as L
from cuvs_b200 import kv_cache
from test_kv_tree_gpu import Step, U, generator, ints, needs_a_gpu  # noqa: F401

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
