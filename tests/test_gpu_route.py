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


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,dim,e,top,form", [(1024, 2048, 63, 6, 0), (1030, 64, 16, 16, 1), (2001, 96, 8, 1, 2), (1500, 512, 130, 8, 3), (1100, 1024, 256, 10, 1), (1025, 32, 1, 1, 0),
                                                 (1040, 320, 72, 4, 2), (1024, 4096, 33, 16, 0)])
@pytest.mark.parametrize("pad", [8, 3])  # (rows that do not start at 16 bytes are summed in 64 bits)
def test_many(qkv, torch_gpu, name, rows, dim, e, top, form, pad):
    """Many rows of 16-bit types: logits to the error of fp32 sums (a chain of dim / 32 instructions, of parts of dim fewer, each off by up to four half
    steps of what it adds), the choice and its order as of 64-bit sums."""
    rng = np.random.default_rng(rows + e)
    x, xv = typed(rng.standard_normal((rows, dim)), name)
    w, wv = typed(rng.standard_normal((e, dim)) / np.sqrt(dim), name)
    x[5], xv[5] = 0, 0  # (a padded row)
    logits, ids, wt = run(qkv, torch_gpu, x, name, w, name, None, form, 2.0, top, pad=pad)
    exact = xv @ wv.T
    bound = (dim // 32 + 40) * 2.0 ** -22 * np.linalg.norm(xv, axis=1)[:, None] * np.linalg.norm(wv, axis=1)
    assert (np.abs(logits - exact) <= bound).all()
    rl, ri, rw = route_ref(xv, wv, None, form, 2.0, top)
    assert np.array_equal(ids, ri)
    # the weights are those of the logits given: to their own rounding
    _, _, gw = route_ref(logits.astype(np.float64), np.eye(e), None, form, 2.0, top)
    assert (np.abs(wt - gw) <= 2.0 ** -23 * gw).all()


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("e", [20, 100, 200])
def test_many_close(qkv, torch_gpu, name, e):
    """Experts whose logits differ past fp32's bits, equal ones among them: the choice is that of 64-bit sums, ties to the lowest index."""
    rows, dim = 1200, 256
    rng = np.random.default_rng(e)
    xv = rng.integers(-64, 65, (rows, dim)).astype(np.float64)
    xv[:, 1] = 2.0 ** -6
    wv = np.tile(rng.integers(-64, 65, (1, dim)).astype(np.float64), (e, 1))
    wv[:, 1] = rng.integers(-8, 9, e) * 2.0 ** -4  # logits of about 2^15 that differ by multiples of 2^-10
    wv[::7, 0] += 3  # some apart from the others
    x, xv = typed(xv, name)
    w, wv = typed(wv, name)
    logits, ids, _ = run(qkv, torch_gpu, x, name, w, name, None, 0, 1.0, 8)
    rl, ri, _ = route_ref(xv, wv, None, 0, 1.0, 8)
    assert np.array_equal(ids, ri)
    assert np.array_equal(np.take_along_axis(logits, ids, 1), np.take_along_axis(rl, ids.astype(np.int64), 1))


def test_many_small(qkv, torch_gpu):
    """Rows and experts whose squares, and whose products, are below fp32's smallest."""
    rows, dim, e = 1100, 256, 40
    rng = np.random.default_rng(4)
    xv = rng.integers(-64, 65, (rows, dim)).astype(np.float64)
    xv[:, 1] = 2.0 ** -6
    wv = np.tile(rng.integers(-64, 65, (1, dim)).astype(np.float64), (e, 1))
    wv[:, 1] = rng.integers(-8, 9, e) * 2.0 ** -4
    for by_x, by_w in ((-100, 0), (0, -100), (-70, -70), (60, 50)):
        x, xt = typed(xv * 2.0 ** by_x, "bf16")
        w, wt = typed(wv * 2.0 ** by_w, "bf16")
        x[7] = xt[7] = 0
        _, ids, _ = run(qkv, torch_gpu, x, "bf16", w, "bf16", None, 0, 1.0, 8)
        assert np.array_equal(ids, route_ref(xt, wt, None, 0, 1.0, 8)[1])


def test_many_not_finite(qkv, torch_gpu):
    rng = np.random.default_rng(11)
    x, xv = grid(rng, (1100, 96), "bf16")
    w, wv = grid(rng, (33, 96), "bf16")
    _, ri, _ = route_ref(xv, wv, None, 1, 1.0, 8)
    bad = x.copy()
    bad[3, 5], bad[4, 6], bad[5, :], bad[1099, 0] = 0x7f80, 0x7fc0, 0xff80, 0x7f80
    _, ids, _ = run(qkv, torch_gpu, bad, "bf16", w, "bf16", None, 1, 1.0, 8)
    for m in range(1100):
        assert len(set(ids[m])) == 8 and (ids[m] >= 0).all() and (ids[m] < 33).all()
        if m not in (3, 4, 5, 1099):
            assert np.array_equal(ids[m], ri[m])
    w2 = w.copy()
    w2[7, 3] = 0x7fc0  # an expert of NaNs is below everything
    _, ids, wt = run(qkv, torch_gpu, x, "bf16", w2, "bf16", None, 1, 1.0, 8)
    assert not (ids == 7).any() and np.isfinite(wt).all()
    w3, wv3 = w[[i for i in range(33) if i != 7]], wv[[i for i in range(33) if i != 7]]
    _, r3, _ = route_ref(xv, wv3, None, 1, 1.0, 8)
    assert np.array_equal(ids - (ids > 7), r3)


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


def test_same_bits_streams_graph(qkv, torch_gpu):
    """The same bits on two streams at once, each with its workspace, and on replays of a graph between other work."""
    torch = torch_gpu
    rng = np.random.default_rng(21)
    cs = []
    for rows, dim, e, top in ((40, 512, 100, 8), (1100, 96, 72, 4)):
        x, w = torch.from_numpy(rng.standard_normal((rows, dim))).to(torch.bfloat16).cuda(), torch.from_numpy(rng.standard_normal((e, dim))).to(torch.bfloat16).cuda()
        need = qkv.moe_route_ws(rows, dim, e)
        out = [torch.empty(rows, e, device="cuda"), torch.empty(rows, top, device="cuda", dtype=torch.int32), torch.empty(rows, top, device="cuda")]
        cs.append((x, w, top, out, torch.empty(need + 16, device="cuda", dtype=torch.uint8), need))

    def call(c, stream=0):
        x, w, top, out, ws, need = c
        qkv.moe_route(x.shape[0], x.shape[1], w.shape[0], top, x.data_ptr(), x.stride(0), 2, w.data_ptr(), 2, 0, 0, 1.5, *(t.data_ptr() for t in out), ws.data_ptr(), need, stream)
        return out

    want = [[t.clone() for t in call(c)] for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        for c, s in zip(cs, streams):
            call(c, s.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(cs, want):
        assert all(torch.equal(a, b) for a, b in zip(c[3], w))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in cs:
            call(c, torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        for c in cs:
            c[0].mul_(-1.5)
            c[3][0].zero_()
        g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in c[3]] for c in cs]
        for c, o in zip(cs, got):
            assert all(torch.equal(a, b) for a, b in zip(call(c), o))
        torch.cuda.synchronize()
