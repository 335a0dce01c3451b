"""The router of many rows: experts of NaNs beside others, values below fp16's and bf16's smallest normal ones, a bias, unequal types."""
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
    rows, dim = 1600, 128
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


@pytest.mark.parametrize("name,least", [("fp16", -24), ("bf16", -133)])
def test_below_the_smallest_normal(qkv, torch_gpu, name, least):
    """Rows, or experts, of subnormal values alone, and mixed with normal ones: they count in the choice and the logits."""
    rows, dim, e = 1600, 256, 40
    rng = np.random.default_rng(3)
    small = rng.integers(-100, 101, (rows, dim)) * 2.0 ** least
    xs, xt = typed(small, name)
    assert np.array_equal(xt, small)
    wb, wt = typed(rng.integers(-64, 65, (e, dim)) / 64.0, name)
    logits, ids, _ = run(qkv, torch_gpu, xs, name, wb, name, None, 0, 1.0, 8)
    rl, ri, _ = route_ref(xt, wt, None, 0, 1.0, 8)
    assert np.array_equal(ids, ri)
    # (chains of 8 instructions: the bound of the many rows' sums; below fp32's smallest normal value steps of 2^-149, 256 terms)
    bound = 50 * 2.0 ** -22 * np.linalg.norm(xt, axis=1)[:, None] * np.linalg.norm(wt, axis=1) + 256 * 2.0 ** -149
    assert (np.abs(logits - xt @ wt.T) <= bound).all()
    # experts of subnormal weights that differ in them alone, beside a large common term
    xb, xt = typed(rng.integers(1, 9, (rows, dim)) / 8.0, name)
    wv = rng.integers(-100, 101, (e, dim)) * 2.0 ** least
    wv[:, 7] = 2.0 ** (least + 14)
    wb, wt = typed(wv, name)
    assert np.array_equal(wt, wv)
    _, ids, _ = run(qkv, torch_gpu, xb, name, wb, name, None, 0, 1.0, 8)
    assert np.array_equal(ids, route_ref(xt, wt, None, 0, 1.0, 8)[1])


@pytest.mark.parametrize("xname,wname,form,bias", [("bf16", "bf16", 3, True), ("fp16", "fp16", 2, True), ("bf16", "fp32", 3, True), ("fp32", "fp32", 0, False), ("bf16", "fp16", 1, False),
                                                   ("fp32", "bf16", 2, False)])
@pytest.mark.parametrize("rows,dim,e,top", [(1023, 320, 40, 4), (1536, 320, 40, 4), (1600, 2048, 256, 8), (1700, 100, 300, 8)])
def test_other_forms(qkv, torch_gpu, xname, wname, form, bias, rows, dim, e, top):
    """Prompts with a bias, fp32 weights, unequal types, more experts: the choice is that of 64-bit sums, the logits those sums rounded once."""
    rng = np.random.default_rng(rows + e)
    x, xv = typed(rng.standard_normal((rows, dim)), xname)
    w, wv = typed(rng.standard_normal((e, dim)) / np.sqrt(dim), wname)
    b = rng.standard_normal(e).astype(np.float32) if bias else None
    logits, ids, wt = run(qkv, torch_gpu, x, xname, w, wname, b, form, 2.0, top, pad=8)
    exact = xv @ wv.T
    many = xname == wname != "fp32" and not bias and e <= 256 and dim % 32 == 0 and rows >= 1536
    assert not many  # (the kernel of many rows does not take these)
    assert (np.abs(logits - exact) <= 2.0 ** -24 * np.abs(exact) + dim * 2.0 ** -52 * (np.abs(xv) @ np.abs(wv).T)).all()
    _, ri, rw = route_ref(logits.astype(np.float64), np.eye(e), b, form, 2.0, top)
    assert np.array_equal(ids, ri) and (np.abs(wt - rw) <= 2.0 ** -23 * rw).all()
    assert np.array_equal(ids, route_ref(xv, wv, b, form, 2.0, top)[1])
