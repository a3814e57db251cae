"""GPU tests of a step of drafted tokens over a paged cache, against the definitions in 64 bits."""
import math

import pytest
import torch

from cuvs_b200 import kv_cache

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of a 32-bit number
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
# what a weight loses on its way into a product of 16-bit numbers, relative to itself
WEIGHT = {torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -17, torch.float32: 0.0}


@pytest.fixture(autouse=True)
def needs_a_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def random_parents(n, m, g, padding=0, spread=0.5):
    u = torch.rand((n, m), generator=g, device="cuda") ** spread
    parents = (u * torch.arange(m, device="cuda")).int() - 1
    if padding:
        parents[::2, m - padding:] = -2
    return parents


def tree_of(parents, lengths):
    """mask as bool [n, m, m], positions, by walking up from every token."""
    n, m = parents.shape
    up, length = parents.tolist(), lengths.tolist()
    mask, positions = torch.zeros((n, m, m), dtype=torch.bool), torch.full((n, m), -1, dtype=torch.int64)
    for i in range(n):
        for j in range(m):
            way, at = [], j
            while 0 <= at < m and len(way) <= m:
                way.append(at)
                at = up[i][at]
            position = max(length[i], 0) + len(way) - 1
            if at == -1 and position < 2 ** 31:
                mask[i, j, way] = True
                positions[i, j] = position
    return mask, positions


def pack(mask):
    m = mask.shape[-1]
    words = -(-m // 32)
    bits = torch.nn.functional.pad(mask.long(), (0, 32 * words - m)).view(*mask.shape[:-1], words, 32)
    return (bits << torch.arange(32, device=mask.device)).sum(-1).to(torch.uint32)


def cache_of(dtype, n_pages, page_size, n_heads, dim, g, heads_outside=True):
    shape = (n_pages, n_heads, page_size, dim) if heads_outside else (n_pages, page_size, n_heads, dim)
    keys, values = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    return (keys.permute(0, 2, 1, 3), values.permute(0, 2, 1, 3)) if heads_outside else (keys, values)


class Step:
    """Inputs of one call: sequences of the given lengths with m drafted tokens each, their pages in no order."""

    def __init__(self, dtype, lengths, m, n_heads, group, dim, page_size, seed=0, padding=0, heads_outside=True, spread=0.5):
        g = generator(seed)
        self.dtype, self.m, self.n_heads, self.group, self.dim, self.page_size = dtype, m, n_heads, group, dim, page_size
        n = len(lengths)
        used = [-(-(max(x, 0) + m) // page_size) for x in lengths]
        n_pages = sum(used) + 3
        self.keys, self.values = cache_of(dtype, n_pages, page_size, n_heads, dim, g, heads_outside)
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        self.pages = ints([[order.pop() if c < used[i] else -1 for c in range(max(used) + 1)] for i in range(n)])
        self.lengths = ints(lengths)
        self.queries = (1.5 * torch.randn((n, m, n_heads * group, dim), generator=g, device="cuda")).to(dtype)
        self.parents = random_parents(n, m, g, padding, spread)
        mask, positions = tree_of(self.parents, self.lengths)
        self.bool_mask, self.positions = mask.cuda(), positions.int().cuda()
        self.mask = pack(self.bool_mask)
        self.generator = g

    def call(self, **options):
        names = ("keys", "values", "queries", "pages", "lengths", "positions", "mask")
        tensors = [options.pop(name, getattr(self, name)) for name in names]
        return kv_cache.attend_tree(*tensors, **options)

    def allowed(self, window=None, filter=None):
        """[n, m, l] which places are seen, [n, l] their slots, [n, l] their positions"""
        n, ps = len(self.lengths), self.page_size
        place = torch.arange(self.pages.shape[1] * ps, device="cuda")
        length = self.lengths.long().clamp(min=0)[:, None]
        page = self.pages.long()[:, place // ps]
        there = (page >= 0) & (page < self.keys.shape[0])
        slot = torch.where(there, page, 0) * ps + place % ps
        if filter is not None:
            there &= (filter.to(torch.int64)[slot // 32] >> (slot % 32) & 1).bool()
        own = self.positions.long().expand(n, self.m)
        index = place - length
        drafted = (index >= 0) & (index < self.m)
        index = index.clamp(0, self.m - 1)
        at = torch.where(drafted, own.gather(1, index), place.expand(n, -1))
        seen = (place < length)[:, None] | (self.bool_mask.expand(n, self.m, self.m).gather(2, index[:, None].expand(n, self.m, -1)) &
                                            (drafted & (at >= length))[:, None])
        seen = seen & there[:, None] & (own >= length)[..., None]
        if window:
            seen &= own[..., None] - at[:, None] < window
        return seen, slot, at

    def exact(self, scale=None, window=None, cap=None, slopes=None, filter=None):
        """out, lse and how far a call may be off: two 32-bit products and a softmax, whose output is rounded once."""
        n, h, ps, dtype = len(self.lengths), self.group * self.n_heads, self.page_size, self.dtype
        scale = self.dim ** -0.5 if scale is None else scale
        seen, slot, at = self.allowed(window, filter)
        out = torch.zeros((n, self.m, h, self.dim), dtype=torch.float64, device="cuda")
        lse = torch.full((n, self.m, h), -math.inf, dtype=torch.float64, device="cuda")
        out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
        for i in range(n):
            for j in range(h):
                ok = seen[i].any(0).nonzero()[:, 0]
                if ok.numel() == 0:
                    continue
                slots, may = slot[i, ok], seen[i][:, ok]
                key, value = (t[slots // ps, slots % ps, j // self.group].double() for t in (self.keys, self.values))
                q = self.queries[i, :, j].double()
                s = scale * (q @ key.t())
                # a product of dim terms, in 32 bits, with its scale; the exponential's argument is rounded
                off = (self.dim + 6) * U * abs(scale) * (q.abs() @ key.abs().t()) + 4 * U * s.abs()
                if cap is not None:
                    s = cap * torch.tanh(s / cap)
                    off = off + 8 * U * cap
                if slopes is not None:
                    far = slopes[j].double() * (self.positions.expand(n, -1)[i].double()[:, None] - at[i, ok])
                    s = s - far
                    off = off + 4 * U * (far.abs() + s.abs())
                s = s.masked_fill(~may, -math.inf)
                some = may.any(1)
                l = torch.logsumexp(s[some], 1)
                p = torch.exp(s[some] - l[:, None])
                spread = torch.where(may[some], off[some], 0.0).amax(1)
                lse[i, some, j] = l
                # weights: 2^-21 of an exponential by powers of two, sums of n terms in 32 bits
                total = spread + 2.0 ** -20 + (slots.numel() + 600) * U
                lse_off[i, some, j] = total + 4 * U * (1 + l.abs())
                v = torch.where(torch.isfinite(value), value, 0.0)
                good = torch.einsum("mk,kd->md", p, v)
                size = torch.einsum("mk,kd->md", p, v.abs())
                out[i, some, j] = good
                out_off[i, some, j] = (2 * total[:, None] + WEIGHT[dtype]) * size + torch.finfo(dtype).eps / 2 * good.abs() + \
                    torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -30 * v.abs().max() * (dtype != torch.float32)
        return out, lse, out_off, lse_off


def check(step, rows=None, **options):
    out, lse = step.call(**options)
    exact, exact_lse, off, lse_off = step.exact(**{k: v for k, v in options.items() if k in ("scale", "window", "cap", "slopes", "filter")})
    none = exact_lse == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert (out[none] == 0).all()
    far = (out.double() - exact).abs()
    assert (far <= off).all(), (far / off).max().item()
    far = (lse.double() - exact_lse)[~none].abs()
    assert (far <= lse_off[~none]).all(), (far / lse_off[~none]).max().item()
    return out, lse


# ---- trees --------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,m", [(1, 1), (3, 2), (2, 31), (5, 32), (1, 33), (4, 64), (2, 255), (1, 1000), (1, 1024)])
@pytest.mark.parametrize("spread", [0.0, 0.1, 1.0])
def test_trees(n, m, spread):
    g = generator(m)
    parents = random_parents(n, m, g, padding=m // 3, spread=spread)
    lengths = torch.randint(0, 10_000, (n,), generator=g, device="cuda", dtype=torch.int32)
    mask, positions = kv_cache.draft_tree(parents, lengths)
    expected, at = tree_of(parents, lengths)
    assert mask.dtype == torch.uint32 and mask.shape == (n, m, -(-m // 32))
    assert torch.equal(mask.view(torch.int32).cpu(), pack(expected).view(torch.int32))
    assert torch.equal(positions.cpu(), at.int())


def test_trees_in_any_order_with_what_is_no_token():
    # 3 <- 0 <- 2; 1 alone; 4 and 5 in a circle, 6 follows them; 7 follows itself; 8 and 9: no tokens; 10 follows 9; 11: far out of range
    parents = ints([[3, -1, 0, -1, 5, 4, 4, 7, -2, 12, 9, 2 ** 31 - 1, 2]])
    for length in (0, 5, -3, 2 ** 31 - 1, 2 ** 31 - 2):
        lengths = ints([length])
        mask, positions = kv_cache.draft_tree(parents, lengths)
        expected, at = tree_of(parents, lengths)
        assert torch.equal(mask.view(torch.int32).cpu(), pack(expected).view(torch.int32))
        assert torch.equal(positions.cpu(), at.int())


def test_sequences_share_a_tree():
    parents = random_parents(1, 40, generator(1))
    lengths = ints([5, 0, 77])
    mask, positions = kv_cache.draft_tree(parents.expand(3, 40), lengths)
    alone, at = kv_cache.draft_tree(parents, ints([0]))
    assert all(torch.equal(mask[i].view(torch.int32), alone[0].view(torch.int32)) for i in range(3))
    assert torch.equal(positions, at + lengths[:, None])


# ---- attention ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim,page_size", [(1, 1, 64, 16), (1, 8, 128, 16), (2, 3, 128, 5), (5, 1, 80, 1), (8, 4, 128, 16), (16, 8, 128, 64),
                                                   (17, 8, 128, 100), (33, 7, 96, 24), (64, 4, 64, 256), (64, 5, 128, 16), (24, 2, 256, 16),
                                                   (70, 2, 192, 32), (3, 16, 256, 8), (130, 3, 48, 7), (9, 4, 8, 16), (40, 16, 128, 16)])
def test_sizes(dtype, m, group, dim, page_size):
    for seed, lengths in enumerate(([300, 1, 0, 127, 129], [1500], [5000, 3])):
        check(Step(dtype, lengths, m, 2, group, dim, page_size, seed, padding=m // 4, heads_outside=seed % 2 == 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [4, 8, 12, 16, 24, 32, 40, 56, 72, 88, 104, 112, 120, 136, 144, 160, 176, 200, 208, 240, 248, 252, 256])
def test_columns(dtype, dim):
    if dtype != torch.float32 and dim % 8:
        pytest.skip("rows of 16-byte pieces")
    check(Step(dtype, [200, 31], 6, 3, 2, dim, 16, dim))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", [{"window": 1}, {"window": 2}, {"window": 3}, {"window": 100}, {"window": 128}, {"window": 700},
                                     {"window": 10 ** 6}, {"cap": 2.0}, {"cap": 30.0}, {"cap": 1e4}, {"slopes": True},
                                     {"slopes": True, "cap": 5.0, "window": 333}, {"scale": -0.2}, {"scale": 0.0}, {"scale": 0.0, "cap": 3.0},
                                     {"scale": 1.0}])
def test_options(dtype, options):
    for m, group, dim in ((7, 4, 128), (40, 8, 64), (12, 3, 256)):
        step = Step(dtype, [900, 130, 0, 1], m, 2, group, dim, 16, m, padding=2, spread=0.2)
        given = dict(options)
        if given.get("slopes"):
            given["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / (2 * group)) for i in range(2 * group)], device="cuda")
        keep = torch.rand((-(-step.keys.shape[0] * 16 // 32), 32), generator=step.generator, device="cuda") < 0.6
        for bits in (None, (keep.long() << torch.arange(32, device="cuda")).sum(1).to(torch.uint32)):
            check(step, **given, filter=bits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences_in_many_parts(dtype):
    check(Step(dtype, [70_000], 3, 1, 2, 64, 16))
    check(Step(dtype, [30_011, 9, 20_000], 20, 1, 8, 128, 64))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_short_sequences(dtype):
    check(Step(dtype, [i % 37 for i in range(300)], 4, 1, 2, 64, 16))
    check(Step(dtype, [(7 * i) % 300 for i in range(90)], 20, 3, 4, 128, 16, padding=5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group", [(6, 4), (40, 8)])
def test_any_mask_and_positions(dtype, m, group):
    """Masks that are no tree's, rows that see nothing, positions with gaps; masks and positions that all sequences share."""
    step = Step(dtype, [200, 200, 200], m, 2, group, 128, 16)
    g = step.generator
    step.bool_mask = torch.rand((3, m, m), generator=g, device="cuda") < 0.5
    step.bool_mask[:, 3] = False
    step.mask = pack(step.bool_mask)
    step.positions = (200 + torch.randint(-3, 50, (3, m), generator=g, device="cuda")).int()
    check(step)
    check(step, window=30)
    step.bool_mask, step.positions = step.bool_mask[:1].expand(3, m, m), step.positions[:1].expand(3, m)
    step.mask = step.mask[:1].expand(3, m, step.mask.shape[2])
    check(step)
    # one row of the mask for all tokens, words to spare with bits that mean nothing
    step.bool_mask = step.bool_mask[:, :1].expand(3, m, m)
    wide = torch.full((3, 1, 5), 0xFFFFFFFF, dtype=torch.int64, device="cuda")
    words = -(-m // 32)
    bits = pack(step.bool_mask[:, :1]).to(torch.int64)
    spare = ~((1 << (m - 32 * (words - 1))) - 1) & 0xFFFFFFFF if m % 32 else 0
    bits[..., -1] |= spare
    wide[..., :words] = bits
    step.mask = wide.to(torch.uint32).expand(3, m, 5)
    check(step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim", [(5, 4, 128), (40, 8, 64), (9, 2, 256)])
def test_what_nobody_may_see_may_hold_anything(dtype, m, group, dim):
    step = Step(dtype, [300, 17, 0], m, 2, group, dim, 16, padding=2)
    keep = torch.rand((-(-step.keys.shape[0] * 16 // 32), 32), generator=step.generator, device="cuda") < 0.7
    bits = (keep.long() << torch.arange(32, device="cuda")).sum(1).to(torch.uint32)
    first = check(step, filter=bits)
    seen, slot, _ = step.allowed(filter=bits)
    used = torch.zeros(step.keys.shape[0] * 16, dtype=torch.bool, device="cuda")
    used[slot[seen.any(1)]] = True
    for bad in (math.nan, math.inf, -math.inf):
        step.keys.masked_fill_(~used.view(-1, 16, 1, 1), bad)
        step.values.masked_fill_(~used.view(-1, 16, 1, 1), bad)
        again = step.call(filter=bits)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim", [(5, 4, 128), (40, 8, 64), (64, 5, 128), (9, 2, 256)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_value_that_is_no_number_reaches_those_who_see_it(dtype, m, group, dim, bad):
    """One drafted token's values are bad, and one of the sequence's that falls out of the window of some: only rows that see them are touched."""
    step = Step(dtype, [300, 129], m, 2, group, dim, 16, spread=0.1)
    window = 250
    seen, slot, _ = step.allowed(window)
    for i, place in ((0, 300 + 2), (1, 129 + 1), (0, 300 - window + 1)):
        s = slot[i, place]
        step.values[s // 16, s % 16] = bad
        touched = torch.zeros_like(seen[..., 0])
        for b in range(2):
            touched[b] = seen[b][:, (step.values[slot[b] // 16, slot[b] % 16, 0, 0].float().isfinite()).logical_not()].any(1)
        out, lse = step.call(window=window)
        exact, exact_lse, off, lse_off = step.exact(window=window)
        assert not out[touched].isfinite().any()
        clean = ~touched
        assert clean.any() and ((out[clean].double() - exact[clean]).abs() <= off[clean]).all()
        assert ((lse.double() - exact_lse).abs() <= lse_off).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_that_are_no_numbers(dtype):
    """A drafted token's keys: its score is no number, for those who see it alone."""
    step = Step(dtype, [100], 12, 1, 4, 64, 16, spread=0.3)
    seen, slot, _ = step.allowed()
    s = slot[0, 103]
    exact, exact_lse, off, lse_off = step.exact()
    step.keys[s // 16, s % 16] = math.nan
    out, lse = step.call()
    touched = seen[0, :, 103]
    assert touched.any() and not touched.all()
    assert lse[0, touched].isnan().all() and out[0, touched].isnan().all()
    assert ((out[0, ~touched].double() - exact[0, ~touched]).abs() <= off[0, ~touched]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_none(dtype):
    step = Step(dtype, [300, 100, 64], 6, 2, 3, 64, 16)
    step.pages[0, 3] = -1
    step.pages[0, 18] = step.keys.shape[0]
    step.pages[1, :] = -7
    step.pages[2, 1] = 2 ** 31 - 1
    check(step)
    # a table that ends before the sequence does, and before it begins to be seen
    step.pages = step.pages[:, :3].contiguous()
    check(step)
    check(step, window=20)
    step.pages = step.pages[:, :0]
    check(step)


def test_negative_lengths_count_as_none():
    step = Step(torch.float16, [-5, 10, -2 ** 31], 4, 2, 2, 64, 16)
    check(step)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sums_stay_finite_where_the_answer_is(dtype):
    """Rows next to the type's largest value."""
    step = Step(dtype, [1500], 3, 1, 2, 64, 16)
    most = torch.finfo(dtype).max
    step.values.fill_(0.99 * most)
    out, _ = step.call()
    assert torch.isfinite(out).all() and ((out.double() / (0.99 * most) - 1).abs() < 0.01).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_small_weights_beside_a_large_one(dtype):
    """20,000 keys with weights of 2^-14 of the first one's: together they count as much as it does."""
    step = Step(dtype, [20_000], 2, 1, 1, 64, 16)
    slot = step.allowed()[1][0]
    step.queries.zero_()
    step.queries[..., 0] = 1.0
    step.keys.zero_()
    step.keys[slot[0] // 16, slot[0] % 16, :, 0] = 14 * math.log(2) * 8
    check(step)
    step.keys[slot[0] // 16, slot[0] % 16, :, 0] = 0
    step.keys[slot[19_990] // 16, slot[19_990] % 16, :, 0] = 14 * math.log(2) * 8
    check(step)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Queries and outputs as parts of larger tensors, keys and values between others."""
    step = Step(dtype, [300, 20], 9, 2, 3, 64, 16)
    plain = step.call()
    fused = torch.zeros((2, 9, 6 + 4, 64), dtype=dtype, device="cuda")
    fused[:, :, 2:8] = step.queries
    turned = torch.full((9, 6, 2, 72), math.nan, dtype=dtype, device="cuda").permute(2, 0, 1, 3)
    out, lse = step.call(queries=fused[:, :, 2:8], out=turned[..., :64])
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1]) and turned[..., 64:].isnan().all()
    both = torch.full((step.keys.shape[0], 2, 16, 2, 72), math.nan, dtype=dtype, device="cuda")
    both[:, 0, ..., :64], both[:, 1, ..., :64] = step.keys, step.values
    out, lse = step.call(keys=both[:, 0, ..., :64], values=both[:, 1, ..., :64])
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])


def test_one_token_is_attention():
    """A tree of one token per sequence and attention to one more position are the same thing."""
    for dtype in DTYPES:
        step = Step(dtype, [300, 0, 1000], 1, 2, 4, 128, 16)
        out, lse = check(step)
        near, near_lse = kv_cache.attention(step.keys, step.values, step.queries[:, 0], step.pages, step.lengths + 1)
        exact, _, off, lse_off = step.exact()
        assert ((out[:, 0].double() - near.double()).abs() <= 2 * off[:, 0]).all()
        assert ((lse[:, 0].double() - near_lse.double()).abs() <= 2 * lse_off[:, 0]).all()


def test_empty_calls():
    step = Step(torch.float16, [5], 3, 2, 2, 64, 16)
    out, lse = kv_cache.attend_tree(step.keys, step.values, step.queries[:0], step.pages[:0], step.lengths[:0], step.positions[:0], step.mask[:0])
    assert out.shape == (0, 3, 4, 64) and lse.shape == (0, 3, 4)
    mask, positions = kv_cache.draft_tree(step.parents[:0], step.lengths[:0])
    assert mask.shape == (0, 3, 1) and positions.shape == (0, 3)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    kv_cache.copy_pages(step.keys, step.values, none, none)
    assert kv_cache.keep_path(step.keys, step.values, step.pages[:0], none, none.view(0, 4)).shape == (0,)
    assert torch.equal(kv_cache.keep_path(step.keys, step.values, step.pages, step.lengths, none.view(1, 0)), step.lengths)


def test_the_same_call_gives_the_same_bits():
    for dtype in DTYPES:
        step = Step(dtype, [9000, 40, 333], 20, 2, 8, 128, 16)
        first = step.call()
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, step.call()))


# ---- turns and axes -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,n_pairs,interleaved", [(128, 64, False), (128, 64, True), (80, 20, False), (72, 25, False), (64, 3, True), (256, 128, False)])
@pytest.mark.parametrize("n_axes", [1, 3, 5])
def test_append_by_turns(dtype, dim, n_pairs, interleaved, n_axes):
    g = generator(dim + n_axes)
    n, heads, queries, ps = 37, 2, 6, 16
    keys, values = cache_of(dtype, 12, ps, heads, dim, g)
    before = keys.clone(), values.clone()
    pages = torch.randperm(12, generator=g, device="cuda").int().view(3, 4)
    sequences = ints([i % 3 for i in range(n)])
    positions = ints([i // 3 if i % 5 else -1 for i in range(n)])
    rows = torch.randn((n, queries + 2 * heads, dim), generator=g, device="cuda").to(dtype)
    turns = torch.randint(-100_000, 1_000_000, (n, n_axes), generator=g, device="cuda").int()
    axes = torch.randint(0, n_axes, (n_pairs,), generator=g, device="cuda").int()
    if n_pairs > 20:
        axes[7], axes[9] = n_axes, -1  # pairs that stay
    f = torch.tensor([10000.0 ** (-i / n_pairs) for i in range(n_pairs)], dtype=torch.float64, device="cuda")
    slots, rotated = kv_cache.append(keys, values, rows[:, queries:queries + heads], rows[:, queries + heads:], pages, positions, sequences=sequences,
                                     queries=rows[:, :queries], frequencies=f, interleaved=interleaved, turns=turns, axes=axes)
    place = positions.long().clamp(min=0)
    expected = torch.where(positions >= 0, pages[sequences.long(), place // ps].long() * ps + place % ps, -1)
    assert torch.equal(slots, expected)
    angle = torch.where((axes >= 0) & (axes < n_axes), turns.double().gather(1, axes.long().clamp(0, n_axes - 1).expand(n, -1)) * f, 0.0)

    def turned(x):
        x = x.double().clone()
        a, b = (slice(0, 2 * n_pairs, 2), slice(1, 2 * n_pairs, 2)) if interleaved else (slice(0, n_pairs), slice(n_pairs, 2 * n_pairs))
        u, v, c, s = x[..., a].clone(), x[..., b].clone(), angle.cos()[:, None], angle.sin()[:, None]
        x[..., a], x[..., b] = u * c - v * s, v * c + u * s
        return x

    known = positions >= 0
    # sines and cosines to 2^-22, products and their sum in 32 bits, one rounding (angles up to 10^6 in 64 bits: 2^-33)
    for got, source in ((rotated, rows[:, :queries]), (keys[slots.clamp(min=0) // ps, slots.clamp(min=0) % ps], rows[:, queries:queries + heads])):
        want, size = turned(source), source.double().abs()
        off = 2.0 ** -20 * 2 * size.amax(-1, keepdim=True) + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal
        assert ((got.double() - want).abs() <= off)[known].all()
    assert torch.equal(rotated[~known], rows[:, :queries][~known])
    kept = torch.ones(12 * ps, dtype=torch.bool, device="cuda")
    kept[slots[known]] = False
    for got, was in zip((keys, values), before):
        assert torch.equal(got.reshape(12 * ps, heads, dim)[kept], was.reshape(12 * ps, heads, dim)[kept])
    assert torch.equal(values[slots[known] // ps, slots[known] % ps], rows[:, queries + heads:][known])


def test_turns_by_the_positions_are_those_without():
    g = generator(5)
    keys, values = cache_of(torch.float16, 9, 16, 2, 64, g)
    pages, positions = torch.randperm(9, generator=g, device="cuda").int().view(3, 3), ints([3, 40, 17])
    rows = torch.randn((3, 2, 64), generator=g, device="cuda").half()
    f = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], device="cuda")
    slots, q = kv_cache.append(keys, values, rows, rows, pages, positions, queries=rows, frequencies=f)
    written = keys.clone()
    for turns, axes in ((positions, None), (positions[:, None], None), (positions[:, None].expand(3, 2).contiguous(), ints([i % 2 for i in range(32)]))):
        again, q2 = kv_cache.append(keys, values, rows, rows, pages, positions, queries=rows, frequencies=f, turns=turns, axes=axes)
        assert torch.equal(slots, again) and torch.equal(q, q2) and torch.equal(keys, written)


# ---- paths and pages ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads_outside", [True, False])
@pytest.mark.parametrize("heads,dim,page_size", [(2, 64, 16), (1, 8, 1), (5, 128, 5), (8, 256, 64)])
def test_paths(dtype, heads_outside, heads, dim, page_size):
    paths = [[0, 1, 2, 3], [0, 2, 5, -1], [3, 4, 6, 9], [-1, 2, 3, 4], [1, 2, 2, 3], [7, -1, 9, 10], [1, 3, 5, 7]]
    lengths = [0, 1, 15, 16, 31, 100, 3]
    step = Step(dtype, lengths, 12, heads, 1, dim, page_size, heads_outside=heads_outside)
    keys, values = step.keys.clone(), step.values.clone()
    kept = kv_cache.keep_path(step.keys, step.values, step.pages, step.lengths, ints(paths))
    n = [4, 3, 4, 0, 2, 1, 4]
    assert kept.tolist() == [a + b for a, b in zip(lengths, n)]
    table = step.pages.tolist()
    for i, path in enumerate(paths):
        for j in range(n[i]):
            a, b = lengths[i] + path[j], lengths[i] + j
            for now, was in ((keys, step.keys), (values, step.values)):
                # (entries ascend: what is read here has not been written before)
                now[table[i][b // page_size], b % page_size] = now[table[i][a // page_size], a % page_size]
    assert torch.equal(keys, step.keys) and torch.equal(values, step.values)


def test_long_paths_and_places_that_are_none():
    step = Step(torch.float16, [10, 20], 200, 2, 1, 64, 16)
    path = [[2 * i + 1 for i in range(100)], [i + i // 7 for i in range(100)]]
    step.pages[0, 3] = -1
    keys = step.keys.clone()
    table = step.pages.tolist()
    kept = kv_cache.keep_path(step.keys, step.values, step.pages, step.lengths, ints(path))
    assert kept.tolist() == [110, 120]
    for i, n in enumerate((10, 20)):
        for j in range(100):
            a, b = n + path[i][j], n + j
            if table[i][a // 16] >= 0 and table[i][b // 16] >= 0:
                keys[table[i][b // 16], b % 16] = keys[table[i][a // 16], a % 16]
    assert torch.equal(keys, step.keys)
    # beyond the last position, beyond the table, negative lengths
    kept = kv_cache.keep_path(step.keys, step.values, step.pages, ints([2 ** 31 - 3, -4]), ints([[0, 1, 2, 3], [0, 5000, -1, -1]]))
    assert kept.tolist() == [2 ** 31 - 1, 2]
    assert torch.equal(keys, step.keys)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads_outside", [True, False])
@pytest.mark.parametrize("heads,dim,page_size,n", [(2, 64, 16, 5), (1, 8, 1, 1), (3, 72, 5, 40), (8, 128, 64, 3), (4, 256, 1000, 2)])
def test_copies(dtype, heads_outside, heads, dim, page_size, n):
    g = generator(n)
    keys, values = cache_of(dtype, 2 * n + 4, page_size, heads, dim, g, heads_outside)
    order = torch.randperm(2 * n + 4, generator=g, device="cuda").int()
    sources, targets = torch.cat((order[:n], ints([-1, 2 * n + 4, int(order[0]), 2 ** 31 - 1]))), torch.cat((order[n:2 * n], order[2 * n:2 * n + 2], ints([-1, -5])))
    sources[0] = sources[n - 1]  # one page twice a source
    want = keys.clone(), values.clone()
    for t in want:
        t[targets[:n].long()] = t[sources[:n].long()]
    kv_cache.copy_pages(keys, values, sources, targets)
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,dim", [(2, 4, 128), (6, 1, 64), (40, 8, 64), (64, 4, 128), (9, 4, 256)])
def test_scores_that_rise_and_fall(dtype, m, group, dim):
    """A row's largest score so far grows with every tile of keys, by many powers of two; then all keys are far below it."""
    for falls in (False, True):
        step = Step(dtype, [1200, 700], m, 2, group, dim, 16)
        slot = step.allowed()[1]
        step.queries.abs_()
        for i, n in enumerate((1200, 700)):
            s = slot[i, :n + m]
            rise = torch.linspace(0.0, 60.0 / dim ** 0.5, n + m, device="cuda").to(dtype)
            rise = rise.flip(0) if falls else rise
            step.keys[s // 16, s % 16] = (step.keys[s // 16, s % 16].float() * 0.1 + rise.float()[:, None, None]).to(dtype)
        check(step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group", [(3, 4), (40, 8)])
def test_slots_that_are_all_left_out(dtype, m, group):
    step = Step(dtype, [500, 64], m, 2, group, 128, 16)
    n_words = -(-step.keys.shape[0] * 16 // 32)
    none = torch.zeros(n_words, dtype=torch.uint32, device="cuda")
    out, lse = step.call(filter=none)
    assert (out == 0).all() and (lse == -math.inf).all()
    # all but the drafted tokens' own
    bits = torch.zeros((n_words, 32), dtype=torch.int64, device="cuda")
    slot = step.allowed()[1]
    for i, n in enumerate((500, 64)):
        s = slot[i, n:n + m]
        bits[s // 32, s % 32] = 1
    check(step, filter=(bits << torch.arange(32, device="cuda")).sum(1).to(torch.uint32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group", [(1024, 1), (300, 4), (1, 16)])
def test_the_largest_trees(dtype, m, group):
    check(Step(dtype, [150, 0], m, 1, group, 64, 16, spread=0.1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_lengths_around_the_ends_of_tiles(dtype, dim):
    lengths = [15, 16, 17, 31, 33, 47, 61, 62, 63, 64, 65, 66, 126, 127, 128, 129, 191, 192, 193, 255, 256, 257]
    for m, group in ((1, 2), (2, 8), (33, 5)):
        check(Step(dtype, lengths, m, 1, group, dim, 16 if m != 2 else 24))


def test_groups_that_are_no_power_of_two_and_many_key_heads():
    for dtype in DTYPES:
        check(Step(dtype, [100, 40], 11, 13, 3, 64, 16))
        check(Step(dtype, [100, 40], 3, 40, 11, 32, 10))
