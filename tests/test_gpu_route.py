"""The router (mk_moe_route) against 64 bits: the choice and its order are equal, ties go to the lowest index."""
import numpy as np
import pytest

from mixcase import route_ref, to_gpu, typed
from stepcase import CODE, ptr

pytestmark = pytest.mark.gpu


def run(qkv, torch, x, xname, w, wname, bias, form, scale, top, pad=0, stream=0, out=None, ws=None):
    rows, dim = x.shape
    e = w.shape[0]
    xd = torch.full((rows, dim + pad), float("nan"), device="cuda").to({"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[xname])
    xd[:, :dim] = to_gpu(torch, x, xname)
    wd = to_gpu(torch, w, wname)
    bd = None if bias is None else torch.from_numpy(bias).cuda()
    need = qkv.moe_route_ws(rows, dim, e)
    ws = torch.full((need // 4 + 4,), float("nan"), device="cuda")
    logits = torch.full((rows + 1, e), 7.0, device="cuda")
    ids = torch.full((rows + 1, top), -7, device="cuda", dtype=torch.int32)
    wt = torch.full((rows + 1, top), 7.0, device="cuda")
    qkv.moe_route(rows, dim, e, top, xd.data_ptr(), dim + pad, CODE[xname], wd.data_ptr(), CODE[wname], ptr(bd), form, scale, logits.data_ptr(), ids.data_ptr(),
                  wt.data_ptr(), ws.data_ptr(), need, stream)
    torch.cuda.synchronize()
    assert (logits[rows] == 7).all() and (ids[rows] == -7).all() and (wt[rows] == 7).all()
    return logits[:rows].cpu().numpy(), ids[:rows].cpu().numpy(), wt[:rows].cpu().numpy()


def grid(rng, shape, name):
    """Values of few bits: their sums are exact in 64 bits, in any order, and equal logits are met often."""
    return typed(rng.integers(-8, 9, shape) / 8.0, name)


@pytest.mark.parametrize("form,bias", [(0, False), (1, False), (2, False), (3, False), (2, True), (3, True)])
@pytest.mark.parametrize("rows,dim,e,top", [(1, 64, 8, 2), (1, 1, 1, 1), (5, 33, 17, 4), (16, 512, 64, 8), (17, 100, 65, 6), (64, 2048, 128, 8), (3, 7, 1024, 16),
                                            (130, 257, 200, 10), (1000, 96, 63, 6)])
def test_ties(qkv, torch_gpu, form, bias, rows, dim, e, top):
    rng = np.random.default_rng(rows + e)
    x, xv = grid(rng, (rows, dim), "bf16")
    w, wv = grid(rng, (e, dim), "bf16")
    b = (rng.integers(-2, 3, e) / 4.0).astype(np.float32) if bias else None
    logits, ids, wt = run(qkv, torch_gpu, x, "bf16", w, "bf16", b, form, 1.5, top)
    rl, ri, rw = route_ref(xv, wv, b, form, 1.5, top)
    assert np.array_equal(logits, rl)
    assert np.array_equal(ids, ri)
    assert (np.abs(wt - rw) <= 2.0 ** -23 * rw).all()


@pytest.mark.parametrize("xname", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("wname", ["fp32", "fp16", "bf16"])
def test_types(qkv, torch_gpu, xname, wname):
    """Normal values: sums of 64 bits differ by their order, 2^-52 of the terms a step; rounded to fp32 that is half a step and hardly ever another."""
    rng = np.random.default_rng(7)
    for rows, dim, e, top, pad in ((1, 5120, 128, 8, 0), (70, 3001, 100, 6, 5), (300, 640, 40, 2, 3)):
        x, xv = typed(rng.standard_normal((rows, dim)), xname)
        w, wv = typed(rng.standard_normal((e, dim)) / np.sqrt(dim), wname)
        logits, ids, wt = run(qkv, torch_gpu, x, xname, w, wname, None, 1, 1.0, top, pad)
        exact = xv @ wv.T
        assert (np.abs(logits - exact) <= 2.0 ** -24 * np.abs(exact) + dim * 2.0 ** -52 * (np.abs(xv) @ np.abs(wv).T)).all()
        # by the library's own logits the choice is exact
        _, ri, rw = route_ref(logits.astype(np.float64), np.eye(e), None, 1, 1.0, top)
        assert np.array_equal(ids, ri) and (np.abs(wt - rw) <= 2.0 ** -23 * rw).all()
        assert np.array_equal(ids, route_ref(xv, wv, None, 1, 1.0, top)[1])


def test_close(qkv, torch_gpu):
    """Logits that differ in the last bits of a 64-bit sum of large terms: fp32 sums would not see it."""
    rows, dim, e = 40, 512, 64
    rng = np.random.default_rng(8)
    xv = rng.integers(-2 ** 7, 2 ** 7, (rows, dim)).astype(np.float64)
    xv[:, 0] = 1
    half = rng.integers(-2 ** 7, 2 ** 7, (e, dim // 2)).astype(np.float64)
    wv = np.concatenate([half, half[:, ::-1]], 1)
    wv[:] = wv[0]
    wv[:, 0] = (rng.permutation(e) - e // 2) * 2.0 ** -8  # all but equal
    x, xv = typed(xv, "bf16")
    w, wv = typed(wv, "fp32")
    # (terms up to 2^14 that sum to about 2^18, in steps of 2^-8: more than 24 bits within the sum)
    logits, ids, _ = run(qkv, torch_gpu, x, "bf16", w, "fp32", None, 0, 1.0, 8)
    rl, ri, _ = route_ref(xv, wv, None, 0, 1.0, 8)
    assert np.array_equal(logits, rl) and np.array_equal(ids, ri)


def test_not_finite(qkv, torch_gpu):
    """Rows with infinities and NaNs: distinct experts all the same, other rows as without them."""
    rng = np.random.default_rng(9)
    x, xv = grid(rng, (40, 96), "bf16")
    w, wv = grid(rng, (33, 96), "bf16")
    clean = run(qkv, torch_gpu, x, "bf16", w, "bf16", None, 0, 1.0, 8)
    bad = x.copy()
    bad[3, 5], bad[4, 6], bad[5, :] = 0x7f80, 0x7fc0, 0xff80
    for form in (0, 1, 2, 3):
        _, ids, _ = run(qkv, torch_gpu, bad, "bf16", w, "bf16", None, form, 1.0, 8)
        for m in range(40):
            assert len(set(ids[m])) == 8 and (ids[m] >= 0).all() and (ids[m] < 33).all()
            if not 3 <= m <= 5:
                assert np.array_equal(ids[m], clean[1][m])
    w2 = w.copy()
    w2[7] = 0x7fc0  # an expert of NaNs is below everything
    logits, ids, wt = run(qkv, torch_gpu, x, "bf16", w2, "bf16", None, 1, 1.0, 8)
    assert not (ids == 7).any() and np.isfinite(wt).all() and np.isnan(logits[:, 7]).all()


def test_bias_masks(qkv, torch_gpu):
    """A bias of -infinity keeps experts out; where it leaves fewer than top_k, they follow by their index."""
    rng = np.random.default_rng(10)
    x, xv = grid(rng, (9, 64), "fp32")
    w, wv = grid(rng, (20, 64), "fp32")
    b = np.full(20, -np.inf, np.float32)
    b[[3, 9, 17]] = 0
    _, ids, _ = run(qkv, torch_gpu, x, "fp32", w, "fp32", b, 3, 1.0, 6)
    assert (np.sort(ids[:, :3], 1) == [3, 9, 17]).all() and (ids[:, 3:] == [0, 1, 2]).all()
