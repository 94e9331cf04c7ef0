"""The decode cache where a row's positions change between blocks, and in the other norm modes of the 209M model."""
import numpy as np
import pytest

import oracle_py as op
import timestral_b200 as tb
from timestral_b200 import synthetic as sy

pytestmark = pytest.mark.gpu


def cached(m, x, H, **kw):
    m.decode_cache(True)
    try:
        tokens = m.last_geometry()
        on = m.forecast(x, H, **kw).copy()
        assert m.last_geometry() != tokens
    finally:
        m.decode_cache(False)
    return on


@pytest.mark.parametrize("T", [96, 320])
@pytest.mark.parametrize("symmetric", [0, 1])
def test_a_row_without_any_observation(T, symmetric):
    """Its first observations are the medians fed back after the first block: with them the positions of all its
    patches change, while keys turned to the old ones stand in the cache (of patches that stay unseen), over
    four blocks. The F16 bound of the other forecast tests (mean 1e-3, a value 3e-2) in units of the row's
    largest value, against the oracle and, twice that, against the forecast without the cache."""
    path = sy.cached_model(sy.spec_small(), "f16")
    m, o = tb.Model(path), op.OracleModel(path)
    x = sy.series_random_walk(3, T)
    x[1] = np.nan
    off = m.forecast(x, 3300, symmetric=symmetric).copy()
    on = cached(m, x, 3300, symmetric=symmetric)
    ref = o.forecast(x, 3300, symmetric=symmetric)
    assert np.isfinite(on).all() and m.last_geometry()[3] == 4
    largest = np.abs(ref[1]).max()
    assert largest > 0
    for other, factor in ((ref, 1), (off, 2)):
        d = np.abs(on[1] - other[1]) / largest
        print("mean %.3e worst %.3e" % (d.mean(), d.max()))
        assert d.mean() <= factor * 1e-3 and d.max() <= factor * 3e-2
    # the rows beside it as they are without it
    assert np.array_equal(on[[0, 2]].view(np.uint32), cached(m, x[[0, 2]], 3300, symmetric=symmetric).view(np.uint32))


@pytest.mark.parametrize("norm_mode", [0, 2])
def test_209m_each_block_in_the_other_norm_modes(norm_mode):
    """As test_209m_each_block_against_the_oracle_on_its_own_context, with its bounds: the norms of a cached
    forecast by kernels of their own (0), and run again with them (2)."""
    path = sy.cached_model(sy.spec_209m(), "f16")
    m, o = tb.Model(path), op.OracleModel(path)
    x = sy.series_random_walk(2, 512, nan_frac=0.05)
    median = m.num_quantiles // 2
    m.fused_norm(norm_mode)
    on = cached(m, x, 2100, symmetric=0, clip=0)
    for first in (0, 1024, 2048):
        context = np.concatenate([x, on[:, :, :first, median]], axis=-1)
        n = min(1024, 2100 - first)
        ref, plain = o.forecast(context, n, symmetric=0, clip=0), m.forecast(context, n, symmetric=0, clip=0)
        loc, sc = op.anchors(context, 32)
        (mean, worst), (pmean, pworst) = (op.normalized_deviation_rows(np.ascontiguousarray(g), ref, loc, sc)
                                          for g in (on[:, :, first:first + n], plain))
        print(f"block at {first}: mean {np.mean(mean):.3e} (plain {np.mean(pmean):.3e}) worst {np.max(worst):.3e} ({np.max(pworst):.3e})")
        assert np.mean(mean) <= 1.1 * np.mean(pmean) and np.max(mean) <= 1.25 * np.max(pmean) and np.max(worst) <= 2 * np.max(pworst)
