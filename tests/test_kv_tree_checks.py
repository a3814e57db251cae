"""CPU tests of the checks of a step of drafted tokens (no GPU): what keep_path writes is not what it reads, scales and caps whose ratio is a number."""
import pytest

from cuvs_b200 import _lib as L
from cuvs_b200 import kv_cache
from test_kv_tree import I, K, T, check
from test_kv_cache import Described

BASE = 1 << 41


@pytest.mark.parametrize("name", ["paths", "pages"])
def test_kept_lies_apart_from_rows(name):
    """Three integers against rows of seven, ten integers from one to the next: in a row, over an end of one, and between two."""
    where = {"pages": Described(I, (3, 7), (10, 1), address=BASE), "paths": Described(I, (3, 7), (10, 1), address=BASE)}[name]
    for at in range(-5, 32):
        kept = set(range(at, at + 3))
        shares = any(kept & set(range(10 * row, 10 * row + 7)) for row in range(3))
        change = {name: where, "kept": Described(I, (3,), address=BASE + 4 * at)}
        if shares:
            with pytest.raises(L.CuvsError, match="memory of the paths or the pages"):
                check(K, change)
        else:
            check(K, change)


def test_kept_and_rows_that_sequences_share():
    for at in range(-5, 12):
        change = {"paths": Described(I, (3, 6), (0, 1), address=BASE), "kept": Described(I, (3,), address=BASE + 4 * at)}
        if -3 < at < 6:
            with pytest.raises(L.CuvsError, match="memory of the paths or the pages"):
                check(K, change)
        else:
            check(K, change)


def test_empty_paths_share_nothing():
    check(K, {"paths": Described(I, (3, 0), address=BASE), "kept": Described(I, (3,), address=BASE)})


def scalars(scale, cap):
    return 0, kv_cache._bits(scale), kv_cache._bits(cap)


@pytest.mark.parametrize("scale,cap", [(1e9, 1e-30), (-1e9, 1e-30), (1e-10, 1e30), (1e-40, 1.0)])
def test_scales_that_no_32_bit_number_divides_by_the_cap(scale, cap):
    with pytest.raises(L.CuvsError, match="scale / cap"):
        check(T, scalars=scalars(scale, cap))
    check(T, scalars=scalars(scale, 0.0))


def test_scales_at_the_ends_of_their_range():
    for cap in (0.0, 1e-30, 50.0, 1e30):
        check(T, scalars=scalars(0.0, cap))
    for scale in (1e8, -1e8, 1e-7):
        for cap in (1e-30, 1e30):
            check(T, scalars=scalars(scale, cap))
    for scale in (3e38, -3e38):
        with pytest.raises(L.CuvsError, match="scale: too large"):
            check(T, scalars=scalars(scale, 0.0))
