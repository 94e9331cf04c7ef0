"""The decode cache and the device's memory: switching it off gives all of it back."""
import pytest
import torch

import timestral_b200 as tb
from timestral_b200 import synthetic as sy

pytestmark = pytest.mark.gpu


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
