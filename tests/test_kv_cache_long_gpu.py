"""GPU tests of attention over a paged cache: sums of very long sequences."""
import math

import pytest
import torch

from cuvs_b200 import kv_cache

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of a 32-bit number


@pytest.mark.parametrize("dtype,n_sequences,group,dim", [(torch.float16, 300, 8, 128), (torch.float16, 200, 1, 64), (torch.float16, 150, 20, 256),
                                                         (torch.bfloat16, 300, 8, 128), (torch.float32, 300, 2, 64)])
def test_sums_of_long_sequences_lose_nothing(dtype, n_sequences, group, dim):
    """More sequences than SMs, of values around 1, so that whatever a sum loses on its way shows: outputs are not too small on average."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    n, page = 400_000, 64
    g = torch.Generator(device="cuda").manual_seed(dim)
    n_pages = n // page
    keys = torch.randn((n_pages, page, 1, dim), generator=g, device="cuda").to(dtype)
    columns = 1 + torch.rand(dim, generator=g, device="cuda")
    values = (columns * (1 + 0.25 * torch.rand((n_pages, page, 1, dim), generator=g, device="cuda"))).to(dtype)
    pages = torch.arange(n_pages, device="cuda", dtype=torch.int32).expand(n_sequences, n_pages)
    lengths = torch.full((n_sequences,), n, dtype=torch.int32, device="cuda")
    queries = torch.randn((n_sequences, group, dim), generator=g, device="cuda").to(dtype)
    out, lse = kv_cache.attention(keys, values, queries, pages, lengths)
    k, v = keys.view(-1, dim).double(), values.view(-1, dim).double()
    off, lse_off = [], []
    for i in range(0, n_sequences, n_sequences // 6):
        s = queries[i].double() @ k.t() * dim ** -0.5
        l = torch.logsumexp(s, 1)
        o = torch.exp(s - l[:, None]) @ v
        off.append((out[i].double() - o) / o)
        lse_off.append(lse[i].double() - l)
    off, lse_off = torch.stack(off), torch.stack(lse_off)
    # Products of 16 keys with up to three numbers of each weight may cut off 2^-24 of their sum for each of 17 terms; scores of up to 7 from products of
    # `dim` terms, exponentials to 2^-21, sums of 16 keys for each warp of a block and lane in 32 bits, rounded: their errors have no sign.
    products, half = 3 * 17 * U, torch.finfo(dtype).eps / 2
    total = (dim + 6) * U * 30 + 2.0 ** -20 + n / 16 * U
    assert off.mean().abs() <= products + 32 * math.sqrt(n / 16) * U + 6 * half / math.sqrt(3 * dim)
    assert off.abs().max() <= 1.01 * (half + products + 2 * total)
    assert lse_off.abs().max() <= total + 4 * U * 14
