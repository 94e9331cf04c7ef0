"""The decode cache and the device's memory: a forecast that the cache leaves without memory runs without
the cache, what the cache holds is there for other forecasts, and switching it off gives all of it back.
Allocations that fail are injected (the next one fails as an exhausted device would)."""
import numpy as np
import pytest
import torch

import timestral_b200 as tb
from timestral_b200 import synthetic as sy

pytestmark = pytest.mark.gpu


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


class fail_next_allocation:
    def __enter__(self):
        assert tb.lib().tsb_test_fail_workspace_allocations(1) == tb.TSB_OK

    def __exit__(self, *_):
        tb.lib().tsb_test_fail_workspace_allocations(0)


def test_no_memory_for_the_cache_itself():
    path = sy.cached_model(sy.spec_small(), "f16")
    x = sy.series_random_walk(3, 640)
    m = tb.Model(path)
    off = m.forecast(x, 1500).copy()
    plain = m.last_geometry()
    m.decode_cache(True)
    with fail_next_allocation():                  # every other buffer is there already
        got = m.forecast(x, 1500).copy()
        assert same(got, off) and m.last_geometry() == plain
    on = m.forecast(x, 1500).copy()
    assert m.last_geometry() != plain and same(on, m.forecast(x, 1500))


def test_no_memory_beside_the_cache():
    """The cache is laid out and the first block's own buffers find no memory: once more without the cache."""
    path = sy.cached_model(sy.spec_small_long(), "f16")
    small, large = sy.series_random_walk(4, 320), sy.series_random_walk(4, 1280)
    other = tb.Model(path)
    off = other.forecast(large, 2080, symmetric=0).copy()
    plain, launches = other.last_geometry(), other.last_launch_count()
    other.decode_cache(True)
    on = other.forecast(large, 2080, symmetric=0).copy()
    assert other.last_geometry() != plain
    m = tb.Model(path)
    m.decode_cache(True)
    m.forecast(small, 4160, symmetric=0)           # a cache, contexts and results at least as large, fewer tokens a block
    with fail_next_allocation():
        got = m.forecast(large, 2080, symmetric=0).copy()
    assert same(got, off) and m.last_geometry() == plain and m.last_launch_count() == launches
    assert same(m.forecast(large, 2080, symmetric=0), on)          # served by the cache again


def test_the_cache_gives_way_to_other_forecasts():
    path = sy.cached_model(sy.spec_small(), "f16")
    x, wide = sy.series_random_walk(2, 640), sy.series_random_walk(16, 700)
    want = tb.Model(path).forecast(wide, 64).copy()
    m = tb.Model(path)
    m.decode_cache(True)
    on = m.forecast(x, 1500).copy()
    with fail_next_allocation():
        assert same(m.forecast(wide, 64), want)
    assert same(m.forecast(x, 1500), on)
    # with nothing to give, the error is what it was
    m.decode_cache(False)
    with fail_next_allocation():
        with pytest.raises(tb.TimestralError, match="cudaMalloc workspace: out of memory"):
            m.forecast(sy.series_random_walk(64, 700), 64)
    assert same(m.forecast(wide, 64), want)


def test_off_gives_back_what_the_cache_held():
    """All of its buffers: keys and values, and the later blocks' features and positions (8 MB here)."""
    path = sy.cached_model(sy.spec_small(), "f16")
    x = sy.series_random_walk(512, 640)
    m = tb.Model(path)

    def free():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]
    other = tb.Model(path)                        # (the kernels' code is loaded on their first use, into device memory)
    other.decode_cache(True)
    other.forecast(x, 1500)
    other.close()
    for _ in range(2):                            # (the two buffers of contexts change places with every block)
        m.forecast(x, 1500)
    before = free()
    m.decode_cache(True)
    m.forecast(x, 1500)
    assert free() < before - (16 << 20)
    m.decode_cache(False)
    assert free() >= before - (2 << 20)


def test_nothing_stays_of_a_cache_that_found_no_memory():
    """Its keys and values are to grow and cannot: the rest of it (8 MB here) goes too."""
    path = sy.cached_model(sy.spec_small(), "f16")
    x = sy.series_random_walk(512, 640)
    m, other = tb.Model(path), tb.Model(path)
    other.decode_cache(True)
    other.forecast(x, 2600)
    other.close()

    def free():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]
    for H in (2600, 1500, 2600):                  # (until both buffers of contexts are as large as they get)
        off = m.forecast(x, H).copy()
    plain, before = m.last_geometry(), free()
    m.decode_cache(True)
    m.forecast(x, 1500)
    assert free() < before - (16 << 20)
    with fail_next_allocation():
        got = m.forecast(x, 2600).copy()
    assert same(got, off) and m.last_geometry() == plain
    assert free() >= before - (2 << 20)
    m.forecast(x, 2600)
    assert m.last_geometry() != plain
    m.decode_cache(False)
    assert free() >= before - (2 << 20)
