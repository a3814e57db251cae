"""CPU tests: what keep_path writes must not be what it reads, as far as its checks can tell (no GPU)."""
import pytest

from cuvs_b200 import _lib as L
from test_kv_tree import I, K, check
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
