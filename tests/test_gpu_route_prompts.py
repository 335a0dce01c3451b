"""The router of many rows: experts of NaNs beside others."""
import numpy as np
import pytest

from mixcase import route_ref, typed
from test_gpu_route import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("e", [65, 130, 200, 256])
@pytest.mark.parametrize("nan", [None, 1, 2, 3])
def test_an_expert_of_nans(qkv, torch_gpu, name, e, nan):
    """Experts whose large terms cancel, so that fp32 sums lose what tells them apart; near each stand an expert of NaNs and small ones.  The choice among the
    others is that of 64-bit sums."""
    rows, dim = 1030, 128
    rng = np.random.default_rng(e + (nan or 0))
    xv = np.ones((rows, dim))
    xv[:, 32:96] = rng.integers(1, 9, (rows, 64)) / 8.0
    wv = rng.integers(-8, 9, (e, dim)) * 2.0 ** -12
    large = np.arange(0, e, 4)
    wv[large, 0], wv[large, 127] = 2.0 ** 14, -2.0 ** 14  # (the first and the last of the products that add up)
    wv[large, 1:127] = 0
    wv[large, 32:96] = rng.integers(0, 9, (len(large), 64)) * 2.0 ** -12 + 2.0 ** -6
    if nan:
        wv[np.arange(nan, e, 4)] = 0
    x, xv = typed(xv, name)
    w, wv = typed(wv, name)
    if nan:
        bad = np.arange(nan, e, 4)
        w[bad, 5] = 0x7e00 if name == "fp16" else 0x7fc0
        wv[bad] = np.nan
    _, ids, wt = run(qkv, torch_gpu, x, name, w, name, None, 1, 1.0, 8)
    _, ri, _ = route_ref(xv, wv, None, 1, 1.0, 8)
    assert np.array_equal(ids, ri) and np.isfinite(wt).all()
