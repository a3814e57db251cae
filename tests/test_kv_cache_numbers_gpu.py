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
    for fp16 (exp(-26) is 2^-37.5), 2^-126 else in lists as short as these (exp(-87) is 2^-125.5)."""
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


WIDE = [torch.bfloat16, torch.float32]
LARGEST = 3.0e38   # of 3.4e38


def tables(lengths, page):
    """Pages in order, one sequence behind the other, and how many they are."""
    used = [-(-n // page) for n in lengths]
    pages = torch.full((len(lengths), max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        pages[i, :n] = torch.arange(at, at + n)
        at += n
    return pages, at


def near(out, want, n, dtype):
    """Sums of n equal terms: n / 4 + 592 additions follow one another at most, in the sum of values and in that of weights."""
    return ((out.double() - want.double()).abs() <= (2 * (n / 4 + 592) * U + torch.finfo(dtype).eps / 2) * want.double().abs()).all()


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("lengths,heads,group,dim,window", [
    ([1500], 1, 4, 64, None), ([1, 700, 0, 20], 3, 1, 128, None), ([3000, 20, 0, 700] * 20, 2, 3, 64, None), ([60000], 1, 1, 64, None),
    ([40000, 300], 2, 8, 128, 30000), ([5000] * 10, 2, 12, 256, None), ([900] * 300, 4, 1, 64, 700)])
def test_values_next_to_the_largest(dtype, lengths, heads, group, dim, window):
    """Rows of the same values have the same values as their mean, and finite ones."""
    from cuvs_b200 import kv_cache
    pages, n_pages = tables(lengths, 16)
    keys = torch.zeros((n_pages, 16, heads, dim), dtype=dtype, device="cuda")
    values = torch.full_like(keys, LARGEST)
    values[..., 1::2] = -LARGEST
    queries = torch.randn((len(lengths), heads * group, dim), generator=generator(1), device="cuda").to(dtype)
    out, lse = kv_cache.attention(keys, values, queries, pages, ints(lengths), window=window)
    for i, n in enumerate(lengths):
        n = min(n, window or n)
        assert near(out[i], values[0, 0, 0] if n else torch.zeros_like(out[i]), n, dtype), i
        assert ((lse[i].double() - math.log(n)).abs() <= (n / 4 + 600) * U).all() if n else (lse[i] == -math.inf).all()


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("n,k", [(1, 700), (1, 20_000), (300, 40)])
def test_values_next_to_the_largest_among_candidates(dtype, n, k):
    from cuvs_b200 import kv_cache
    g = generator(2)
    keys = torch.zeros((50, 16, 2, 64), dtype=dtype, device="cuda")
    values = torch.full_like(keys, -LARGEST)
    candidates = torch.randint(0, 800, (n, 4, k), generator=g, device="cuda")
    out, lse = kv_cache.attend_candidates(keys, values, torch.randn((n, 4, 64), generator=g, device="cuda").to(dtype), candidates)
    assert near(out, values[0, 0, 0], k, dtype) and ((lse.double() - math.log(k)).abs() <= (k / 4 + 600) * U).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_small_values_keep_their_digits(dtype):
    """The other end: the smallest normal numbers of fp16; 1e-25, which leaves room for 24 digits and lists of 2^15 rows above 2^-126."""
    from cuvs_b200 import kv_cache
    g = generator(3)
    lengths = [20_000, 300, 5]
    pages, n_pages = tables(lengths, 16)
    small = 6.2e-5 if dtype == torch.float16 else 1e-25
    keys = torch.zeros((n_pages, 16, 2, 64), dtype=dtype, device="cuda")
    values = (small * (1 + torch.rand((n_pages, 16, 2, 64), generator=g, device="cuda"))).to(dtype)
    queries = torch.randn((3, 4, 64), generator=g, device="cuda").to(dtype)
    out, _ = kv_cache.attention(keys, values, queries, pages, ints(lengths))
    at = 0
    for i, n in enumerate(lengths):
        used = -(-n // 16)
        mean = values[at:at + used].reshape(-1, 2, 64)[:n].double().mean(0).repeat_interleave(2, 0)
        at += used
        tol = (2 * (n / 4 + 592) * U + torch.finfo(dtype).eps / 2) * mean + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert ((out[i].double() - mean).abs() <= tol).all(), i


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_parts,dim", [(2, 128), (9, 64), (40, 256), (7, 24)])
def test_parts_next_to_the_largest(dtype, n_parts, dim):
    from cuvs_b200 import kv_cache
    parts = torch.full((n_parts, 5, 3, dim), 65000.0 if dtype == torch.float16 else LARGEST, dtype=dtype, device="cuda")
    parts[..., 1::2] *= -1
    lse = torch.full((n_parts, 5, 3), 4.0, device="cuda")
    lse[1:, 0] = -math.inf
    out, joined = kv_cache.merge_parts(parts, lse)
    # weights and their sum: n_parts additions each, 2^-22 for the exponentials, a few roundings
    tol = (2 * n_parts + 16) * U + torch.finfo(dtype).eps / 2
    assert ((out.double() - parts[0].double()).abs() <= tol * parts[0].double().abs()).all()
    want = torch.full((5, 3), 4.0 + math.log(n_parts), device="cuda").double()
    want[0] = 4.0
    assert ((joined.double() - want).abs() <= (n_parts + 16) * U * want).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_sine_and_cosine(interleaved):
    """Rows of (1, 0) pairs are turned into the cosine and the sine themselves.  A step of values below 1 is u at most: the 32-bit functions are
    within one of them, and turning them by the angle's last digits rounds once more, by half a step.  Errors spread evenly within that
    have a root mean square of sqrt(1/3 + 1/12) u = 0.65 u, were all values above 1/2; a third of them is not."""
    from cuvs_b200 import kv_cache
    g = generator(4)
    n, dim, half = 4000, 128, 64
    nothing = torch.zeros((n, 1, dim), device="cuda")
    keys, values = torch.zeros((2, 4, 16, 1, dim), device="cuda")
    positions = torch.cat((torch.arange(100, device="cuda"), torch.randint(0, 1_000_000, (n - 100,), generator=g, device="cuda"))).int()
    f = torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
    queries = nothing.clone()
    queries[..., slice(0, dim, 2) if interleaved else slice(0, half)] = 1
    _, turned = kv_cache.append(keys, values, nothing, nothing, torch.full((n, 1), -1, dtype=torch.int32, device="cuda"), positions, queries=queries,
                                frequencies=f, interleaved=interleaved)
    pairs = turned[:, 0].view(n, half, 2) if interleaved else turned[:, 0].view(n, 2, half).transpose(1, 2)
    angle = positions.double()[:, None] * f
    for got, want in ((pairs[..., 0], angle.cos()), (pairs[..., 1], angle.sin())):
        off = (got.double() - want).abs()
        # the product of position and frequency is rounded to 2^-53 of an angle of up to 2^20
        assert (off <= 1.5 * U + 2.0 ** -33).all(), off.max().item() / U
        assert off.square().mean().sqrt() <= 0.65 * U
