"""Products with 4-bit weights (mk_w4_units, mk_w4_rows) against the products in 64 bits, within the roundings that
stepcase.w4_bound counts."""
import numpy as np
import pytest

from stepcase import CODE, dtype_of, pack_codes, ptr, units_of, unpack_units, w4_bound, w4_ref

pytestmark = pytest.mark.gpu


def weights(rng, n, k, group, mins):
    c = rng.integers(0, 16, (n, k))
    gs = -(-k // group)
    s = (rng.uniform(0.2, 1.5, (n, gs)) * 0.01).astype(np.float16)
    m = (rng.standard_normal((n, gs)) * 0.02).astype(np.float16) if mins else None
    return c, s, m


def run(torch, qkv, rows, n, k, group, mins, x, seed=0, y_pad=0, x_pad=0, x_off=0, edit=None, scale=1.0):
    rng = np.random.default_rng(seed + 1000 * rows + n + k)
    c, s, m = weights(rng, n, k, group, mins)
    v = (rng.standard_normal((rows, k)) * scale).astype(np.float32)
    if edit:
        edit(v, s)
    codes = torch.from_numpy(pack_codes(c)).cuda()
    sd = torch.from_numpy(s).cuda()
    md = torch.from_numpy(m).cuda() if mins else None
    y = torch.full((rows + 1, n + y_pad), 77.0, device="cuda")
    if x == "units":
        a, b, meta = units_of(v)
        q, sc, _ = unpack_units(a, b, meta)
        v = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(rows, k)
        ad, bd, xm = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda(), torch.from_numpy(meta.view(np.int16)).cuda()
        qkv.w4_units(rows, n, k, group, codes.data_ptr(), sd.data_ptr(), ptr(md), ad.data_ptr(), bd.data_ptr(), xm.data_ptr(), y.data_ptr(), n + y_pad,
                     torch.cuda.current_stream().cuda_stream)
    else:
        t = torch.from_numpy(v).to(dtype_of(torch, x))
        v = t.double().numpy()
        buf = torch.full((rows * (k + x_pad) + x_off,), 3.0, dtype=t.dtype)
        buf[x_off:].view(rows, k + x_pad)[:, :k] = t
        xd = buf.cuda()
        qkv.w4_rows(rows, n, k, group, codes.data_ptr(), sd.data_ptr(), ptr(md), xd.data_ptr() + x_off * xd.element_size(), k + x_pad, CODE[x],
                    y.data_ptr(), n + y_pad, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    assert (got[rows] == 77).all() and (got[:, n:] == 77).all(), "written outside the result"
    with np.errstate(all="ignore"):
        ref, mag = w4_ref(c, s, m, group, v)
    return got[:rows, :n].astype(np.float64), ref, mag


def check(torch, qkv, rows, n, k, group, mins, x, **kw):
    got, ref, mag = run(torch, qkv, rows, n, k, group, mins, x, **kw)
    err = np.abs(got - ref)
    bad = err > w4_bound(k, mag, x != "units")
    assert not bad.any(), (np.argwhere(bad)[:4], err.max(), mag.max())


@pytest.mark.parametrize("x", ["units", "fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64])
def test_rows(qkv, torch_gpu, rows, x):
    check(torch_gpu, qkv, rows, 100, 1024, 32, False, x)
    check(torch_gpu, qkv, rows, 48, 704, 64, True, x)


@pytest.mark.parametrize("x", ["units", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
def test_groups(qkv, torch_gpu, group, mins, x):
    for rows in (1, 3, 8, 20):
        check(torch_gpu, qkv, rows, 33, 1088, group, mins, x)  # (1,088: the last group of 128 is half as long)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 127, 129, 1000])
@pytest.mark.parametrize("k", [64, 128, 192, 2240])
def test_shapes(qkv, torch_gpu, n, k):
    check(torch_gpu, qkv, 1, n, k, 32, False, "units")
    check(torch_gpu, qkv, 6, n, k, 64, True, "units")
    check(torch_gpu, qkv, 2, n, k, 128, False, "fp16")


@pytest.mark.parametrize("k", [32, 96, 160, 1056])
def test_plain_rows_of_odd_blocks(qkv, torch_gpu, k):
    for x in ("fp16", "bf16", "fp32"):
        for rows in (1, 7, 24):
            check(torch_gpu, qkv, rows, 40, k, 32, True, x, x_pad=5, x_off=3, y_pad=2)


@pytest.mark.parametrize("x,rows", [("units", 1), ("units", 8), ("units", 64), ("bf16", 1), ("fp32", 4), ("fp32", 64)])
def test_long_rows(qkv, torch_gpu, x, rows):
    """Rows of x that do not fit a workgroup's LDS at once."""
    check(torch_gpu, qkv, rows, 50, 25600, 128, True, x)


@pytest.mark.parametrize("x", ["units", "fp16"])
def test_many_weight_rows(qkv, torch_gpu, x):
    """More 16-row tiles than the launch has waves: every number of waves per tile, workgroups with several tiles."""
    for n in (3000, 9001, 20011, 70003):
        check(torch_gpu, qkv, 1, n, 256, 32, False, x)
        check(torch_gpu, qkv, 5, n, 128, 128, True, x)
        check(torch_gpu, qkv, 40, n, 128, 64, False, x)


@pytest.mark.parametrize("x", ["units", "bf16", "fp32"])
@pytest.mark.parametrize("n", [4090, 8000, 12000, 16001, 20000, 24500, 24600])
def test_tiles_per_workgroup(qkv, torch_gpu, n, x):
    """The dense form's one to six tiles a workgroup and its two workgroups a CU, of 16, 32, 64 rows and of several times that."""
    for rows, mins in ((9, False), (30, True), (64, False), (50, True), (130, False)):
        check(torch_gpu, qkv, rows, n, 192, 32 if mins else 64, mins, x)


@pytest.mark.parametrize("rows,x", [(1, "units"), (8, "bf16"), (20, "units"), (40, "bf16")])
def test_offsets_past_32_bits(qkv, torch_gpu, rows, x):
    """4.9 GB of codes, plain rows of x over 17 GB; the last weight rows and some on the way."""
    torch, n, k = torch_gpu, 300001, 32768
    rng = np.random.default_rng(rows)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    s = (torch.rand(n, k // 128, device="cuda") * 0.01 + 0.001).half()
    v = rng.standard_normal((rows, k)).astype(np.float32)
    y = torch.zeros(rows, n, device="cuda")
    if x == "units":
        a, b, meta = units_of(v)
        q, sc, _ = unpack_units(a, b, meta)
        v = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(rows, k)
        ad, bd, xm = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda(), torch.from_numpy(meta.view(np.int16)).cuda()
        qkv.w4_units(rows, n, k, 128, codes.data_ptr(), s.data_ptr(), 0, ad.data_ptr(), bd.data_ptr(), xm.data_ptr(), y.data_ptr(), n)
    else:
        stride = (1 << 33) // 2 // rows * 2 + 8
        buf = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
        buf.view(rows, stride)[:, :k] = torch.from_numpy(v).cuda()
        v = buf.view(rows, stride)[:, :k].double().cpu().numpy()
        qkv.w4_rows(rows, n, k, 128, codes.data_ptr(), s.data_ptr(), 0, buf.data_ptr(), stride, 2, y.data_ptr(), n)
    torch.cuda.synchronize()
    pick = np.r_[0:3, 131070:131075, 262142:262147, n - 20:n]
    words = codes[torch.from_numpy(pick).cuda()].cpu().numpy().reshape(len(pick), k // 8, 4)
    c = np.concatenate([words & 15, words >> 4], -1).reshape(len(pick), k)
    ref, mag = w4_ref(c, s[torch.from_numpy(pick).cuda()].cpu().numpy(), None, 128, v)
    assert (np.abs(y.cpu().numpy()[:, pick] - ref) <= w4_bound(k, mag, x != "units")).all()


@pytest.mark.parametrize("x", ["fp16", "bf16", "fp32"])
def test_value_ranges(qkv, torch_gpu, x):
    """Blocks of very different sizes, zeros, and the types' smallest values."""
    def edit(v, s):
        v[0, :32] *= 1e4
        v[0, 32:64] = 0
        v[0, 64:96] *= 2e-7
        v[1] *= 1e-6 if x == "fp16" else 1e-30
        v[2, ::2] *= 1e-5
    check(torch_gpu, qkv, 3, 64, 256, 32, True, x, edit=edit)
    if x != "fp16":
        check(torch_gpu, qkv, 2, 64, 256, 32, False, x, scale=1e30)


@pytest.mark.parametrize("x", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [4, 20])
def test_wild_values(qkv, torch_gpu, x, rows):
    """An infinity or a NaN in a row of x reaches that row alone; a weight row's infinite scale that column alone."""
    def edit(v, s):
        v[1, 40] = np.inf
        v[2, 50] = np.nan
        s[5, 1] = np.inf
    got, ref, mag = run(torch_gpu, qkv, rows, 37, 256, 64, False, x, edit=edit)
    ok = np.ones(rows, bool)
    ok[[1, 2]] = False
    cols = np.arange(37) != 5
    g, r = got[ok][:, cols], ref[ok][:, cols]
    assert np.isfinite(g).all() and (np.abs(g - r) <= w4_bound(256, mag[ok][:, cols], True)).all()
    assert np.isnan(got[2]).all()
    assert np.array_equal(np.isnan(got[1, cols]), np.isnan(ref[1, cols])) and np.array_equal(np.sign(got[1, cols]), np.sign(ref[1, cols]), equal_nan=True)
    assert not np.isfinite(got[ok][:, 5]).any()


@pytest.mark.parametrize("x", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 2, 8, 20])
def test_lone_values(qkv, torch_gpu, x, rows):
    """One value far above the rest of its block, at every place of it; an infinity in a last block that others pad."""
    def edit(v, s):
        for i in range(5 * 32):
            v[i % rows, i] = 4096.0 * (1 + i / 256) * (-1) ** i
    got, ref, mag = run(torch_gpu, qkv, rows, 37, 160, 32, rows == 2, x, edit=edit)
    assert (np.abs(got - ref) <= w4_bound(160, mag, True)).all()

    def last(v, s):
        v[0, 150] = np.inf
    got, ref, mag = run(torch_gpu, qkv, rows, 37, 160, 32, False, x, edit=last)
    assert np.isinf(ref[0]).any() and np.array_equal(np.isnan(got[0]), np.isnan(ref[0]))
    there = ~np.isnan(ref[0])
    assert np.array_equal(got[0][there], ref[0][there])


@pytest.mark.parametrize("x", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 256), (1, 2240), (2, 256), (2, 2240), (4, 256), (4, 2240), (8, 256), (8, 2240), (20, 2240), (40, 256)])
def test_infinities_with_minimums(qkv, torch_gpu, x, rows, k):
    """W x of an infinite x is infinite where W = s (c - 8) + m is not zero, whatever the signs of its two parts and also for c = 8;
    and finite values whose block's sum passes fp32's largest leave what their products sum to.  The same for the row beside it."""
    for kind in ("one", "two", "last", "nan", "large"):
        if kind == "large" and x == "fp16":
            continue

        def edit(v, s):
            m = min(1, rows - 1)
            if kind == "one":
                v[m, 70] = np.inf
            elif kind == "two":
                v[m, 70], v[m, 200] = -np.inf, np.inf
            elif kind == "last":
                v[m, k - 1] = -np.inf
            elif kind == "nan":
                v[m, 70], v[m, 71] = np.inf, np.nan
            else:
                v[m, 64:72] = 1.5e38
            s[3] = 0
        got, ref, mag = run(torch_gpu, qkv, rows, 300, k, 64, True, x, edit=edit, seed=len(kind))
        assert np.array_equal(np.isnan(got), np.isnan(ref)), kind
        wild = np.isinf(ref)
        assert np.array_equal(got[wild], ref[wild]) and (kind in ("nan", "large") or wild.any())
        fine = np.isfinite(ref)
        assert (np.abs(got[fine] - ref[fine]) <= w4_bound(k, mag, True)[fine]).all(), kind
        assert kind != "large" or fine.all()


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 40, 130])
@pytest.mark.parametrize("n,k", [(70003, 128), (9001, 640), (300001, 64)])
def test_infinities_over_many_tiles(qkv, torch_gpu, rows, n, k):
    """Workgroups of several tiles, the last of them short, rows of every kind beside each other, results with a stride; in a graph's
    replay too (the same bits)."""
    if rows * n > 8e6:
        n = 70003 if rows == 40 else 20011
    torch = torch_gpu
    rng = np.random.default_rng(rows + n)
    c, s, m = weights(rng, n, k, 32, True)
    v = rng.standard_normal((rows, k)).astype(np.float16)
    kinds = rng.permutation(rows)
    v[kinds[0], k - 3] = np.inf
    if rows > 2:
        v[kinds[1], 5], v[kinds[2], 17], v[kinds[2], 40] = np.nan, -np.inf, -np.inf
    dev = [torch.from_numpy(t).cuda() for t in (pack_codes(c), s, m, v)]
    y, y2 = (torch.full((rows + 1, n + 3), 77.0, device="cuda") for _ in range(2))

    def call(y, stream):
        qkv.w4_rows(rows, n, k, 32, *(t.data_ptr() for t in dev), k, CODE["fp16"], y.data_ptr(), n + 3, stream)
    call(y, torch.cuda.current_stream().cuda_stream)
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            call(y2, side.cuda_stream)
    for _ in range(3):
        y2[:rows, :n] = 5
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int32), y2.view(torch.int32))
    got = y.cpu().numpy()
    assert (got[rows] == 77).all() and (got[:, n:] == 77).all()
    got = got[:rows, :n].astype(np.float64)
    with np.errstate(all="ignore"):
        ref, mag = w4_ref(c, s, m, 32, v)
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
    assert (np.abs(got[fine] - ref[fine]) <= w4_bound(k, mag, True)[fine]).all() and np.isinf(ref).any()


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 4, 8, 20, 40])
def test_scales_that_are_not_finite(qkv, torch_gpu, rows, mins):
    """A unit's scale reaches its row alone, a weight's scale or minimum its column alone; both are then not finite."""
    torch, n, k, group = torch_gpu, 90, 320, 64
    rng = np.random.default_rng(rows)
    c, s, m = weights(rng, n, k, group, mins)
    c[c == 8] = 9
    (m if mins else s)[7, 2] = np.inf
    s[70, 1] = np.nan
    a, b, meta = units_of(rng.standard_normal((rows, k)).astype(np.float32))
    a[a == 0], b[b == 0] = 1, 1
    q, sc, _ = unpack_units(a, b, meta)
    sums = q.reshape(rows, k // 64, 2, 2, 16).astype(np.int16).sum(-1, dtype=np.int16)
    meta = meta.reshape(rows, k // 64, 2, 4)
    meta[..., 2:] = np.swapaxes(sums, 2, 3).view(np.uint16)
    bad = {rows - 1: np.inf, rows // 2: np.nan} if rows > 2 else {}
    for row, v in bad.items():
        meta[row, 3, :, 1] = np.float16(v).view(np.uint16)
    x = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(rows, k)
    y = torch.zeros(rows, n, device="cuda")
    dev = [torch.from_numpy(np.ascontiguousarray(t)).cuda() for t in (pack_codes(c), s, a, b, meta.reshape(rows, k // 32, 4).view(np.int16))]
    md = torch.from_numpy(m).cuda() if mins else None
    qkv.w4_units(rows, n, k, group, dev[0].data_ptr(), dev[1].data_ptr(), ptr(md), dev[2].data_ptr(), dev[3].data_ptr(), dev[4].data_ptr(), y.data_ptr(), n,
                 torch.cuda.current_stream().cuda_stream)
    got = y.cpu().numpy().astype(np.float64)
    fine_r, fine_c = ~np.isin(np.arange(rows), list(bad)), ~np.isin(np.arange(n), (7, 70))
    with np.errstate(all="ignore"):
        ref, mag = w4_ref(c, s, m, group, x)
    at = np.ix_(fine_r, fine_c)
    assert (np.abs(got[at] - ref[at]) <= w4_bound(k, mag[at], False)).all()
    assert not np.isfinite(got[~fine_r]).any() and not np.isfinite(got[:, ~fine_c]).any()


def test_no_rows_and_refusals(qkv, torch_gpu):
    torch = torch_gpu
    t = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    y = torch.full((64,), 5.0, device="cuda")
    p = t.data_ptr()
    qkv.w4_rows(0, 64, 64, 32, p, p, 0, p, 64, 1, y.data_ptr(), 64)
    qkv.w4_units(0, 64, 64, 32, p, p, 0, p, p, p, y.data_ptr(), 64)
    torch.cuda.synchronize()
    assert (y == 5).all()
    h = torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(qkv.KVError, match="codes is not device memory"):
        qkv.w4_rows(1, 16, 64, 32, (h.data_ptr() + 15) // 16 * 16, p, 0, p, 64, 1, y.data_ptr(), 64)
    torch.cuda.synchronize()
