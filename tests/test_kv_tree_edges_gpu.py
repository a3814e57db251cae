"""GPU tests of attention of drafted tokens at the ends of its ranges: very long sequences, values and scores that are no numbers."""
import math

import pytest
import torch

from cuvs_b200 import kv_cache
from test_kv_tree_gpu import U, generator, ints, needs_a_gpu  # noqa: F401

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
