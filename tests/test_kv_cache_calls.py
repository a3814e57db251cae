"""CPU tests of what Python makes of the arguments of attention over a paged cache."""
import numpy as np
import pytest

from cuvs_b200 import kv_cache


def test_windows():
    assert kv_cache._window(None) == 0 and kv_cache._window(7) == 7 and kv_cache._window(np.int32(7)) == 7
    # no position is as far away as 2^31: what does not fit 64 bits is a window over everything, not over its last bits
    for far in (2 ** 31, 2 ** 63 - 1, 2 ** 63, 2 ** 64, 2 ** 64 + 5, 10 ** 30):
        assert kv_cache._window(far) == 2 ** 31
    for none in (0, -1, -2 ** 64, np.int64(-3)):
        with pytest.raises(ValueError, match="window"):
            kv_cache._window(none)
    with pytest.raises(TypeError):
        kv_cache._window(7.5)
