"""GPU tests of what attention over a paged cache keeps of its numbers: digits of the weights, and the ends of the types' ranges.

u = 2^-24 is half a step of 32 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads", [(64, 1), (128, 8), (128, 16), (256, 3), (64, 20)])
def test_weights_keep_their_digits(dtype, dim, heads):
    """Two rows a sequence, whose values nearly cancel: what is left of a column is small, and so is its rounding, so that the error of the
    weight shows.  Scores are exact: 0 and -x with x of a few bits.  The weight w = exp(-x), x < 4, may be off, relative to itself, by the
    roundings of log2(e), of scale * log2(e) and of their product with x (3 u x <= 12 u), by 2^-22 = 4 u of the exponential, by 2^-22 of what
    goes into the product, and by the sum and its reciprocal (4 u)."""
    from cuvs_b200 import kv_cache
    g = generator(dim + heads)
    n, page = 500, 16
    x = (torch.randint(1, 250, (n,), generator=g, device="cuda") / 64.0).to(dtype).double()
    w = torch.exp(-x)
    keys = torch.zeros((n, page, 1, dim), dtype=dtype, device="cuda")
    values = torch.zeros_like(keys)
    keys[:, 1, 0, 3] = -x.to(dtype)
    # the nearest number of 8 bits, whatever the type, and neighbours of it in the other columns
    near = w.to(torch.bfloat16).double()[:, None] * (1 + torch.arange(dim, device="cuda") % 5 * 2.0 ** -7)
    values[:, 0, 0] = -near.to(dtype)
    values[:, 1, 0] = 1.0
    queries = torch.zeros((n, heads, dim), dtype=dtype, device="cuda")
    queries[:, :, 3] = 1.0
    out, lse = kv_cache.attention(keys, values, queries, torch.arange(n, dtype=torch.int32, device="cuda")[:, None], ints([2] * n), scale=1.0)
    share = (w / (1 + w))[:, None]
    want = share + values[:, 0, 0].double() / (1 + w)[:, None]
    tol = 24 * U * (share + values[:, 0, 0].double().abs() / (1 + w)[:, None]) + torch.finfo(dtype).eps / 2 * want.abs()
    tol += 2.0 ** -25 if dtype == torch.float16 else 0.0       # of its smallest numbers
    off = (out.double() - want[:, None]).abs() / tol[:, None]
    assert off.max() <= 1, (off.max().item(), (off > 1).double().mean().item())
    assert ((lse.double() - torch.log1p(w)[:, None]).abs() <= 24 * U).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_values_of_small_weights(dtype):
    """A row of infinite values makes the output infinite however small its weight is, as far as the weights reach: 2^-38 of the largest weight
    for fp16 (exp(-26) is 2^-37.5), 2^-126 else (exp(-87) is 2^-125.5)."""
    from cuvs_b200 import kv_cache
    n = 27 if dtype == torch.float16 else 88
    keys = torch.zeros((n, 16, 1, 64), dtype=dtype, device="cuda")
    values = torch.ones_like(keys)
    keys[:, 1, 0, 0] = -torch.arange(n, device="cuda").to(dtype)
    values[:, 1, 0, ::2] = float("inf")
    values[:, 1, 0, 1::4] = -float("inf")
    for heads in (1, 5, 12):
        queries = torch.zeros((n, heads, 64), dtype=dtype, device="cuda")
        queries[..., 0] = 1
        out, lse = kv_cache.attention(keys, values, queries, torch.arange(n, dtype=torch.int32, device="cuda")[:, None], ints([3] * n), scale=1.0)
        want = values[:, 1].expand_as(out)
        assert torch.equal(out[..., 0::4], want[..., 0::4]) and torch.equal(out[..., 1::4], want[..., 1::4]) and torch.equal(out[..., 2::4], want[..., 2::4])
        assert ((out[..., 3::4] - 1).abs() <= torch.finfo(dtype).eps).all()
