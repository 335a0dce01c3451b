"""Residual norm and its int8 units (mk_norm_q32) against the definition in 64 bits.

The stored sum and the units are compared bit for bit: the sum is one fp32 addition and one rounding, the codes and scales follow
from single float32 operations and a factor whose sum is in 64 bits.  y carries three float32 roundings (the factor, two
products) and the output's."""
import numpy as np
import pytest

from stepcase import CODE, EPS_HALF, dtype_of, norm_ref, norm_units_ref, ptr, unpack_units

pytestmark = pytest.mark.gpu


def run(torch, qkv, rows, dim, dt, res=True, out="both", pad=0, off=0, inplace=False, eps=1e-6, edit=None, seed=0, stream=None):
    g = torch.Generator().manual_seed(seed)
    T = dtype_of(torch, dt)

    def rowsof(scale):
        buf = torch.zeros(rows * (dim + pad) + off + 64, dtype=T)
        v = buf[off:off + rows * (dim + pad)].view(rows, dim + pad)
        v[:, :dim] = (torch.randn(rows, dim, generator=g) * scale).to(T)
        return buf, v
    xb, x = rowsof(1.0)
    rb, r = rowsof(3.0)
    if edit:
        edit(x, r)
    w = 1 + 0.2 * torch.randn(dim, generator=g)
    want_h = ((x[:, :dim].float() + r[:, :dim].float()).to(T) if res else x[:, :dim].clone())
    xd, rd, wd = xb.cuda(), rb.cuda(), w.cuda()
    guard = 7.0
    sb = rd if inplace else torch.full_like(rb, guard, device="cuda")
    yb = torch.full_like(xb, guard, device="cuda")
    units = out != "rows"
    nu = dim // 32
    a = torch.full((rows + 1, nu, 16), 99, dtype=torch.int8, device="cuda") if units else None
    b = torch.full((rows + 1, nu, 16), 99, dtype=torch.int8, device="cuda") if units else None
    m = torch.full((rows + 1, nu, 4), 999, dtype=torch.int16, device="cuda") if units else None
    es = xd.element_size()
    st, ld = off * es, dim + pad
    s = stream or torch.cuda.current_stream()
    qkv.norm_q32(xd.data_ptr() + st, ld, rd.data_ptr() + st if res else 0, ld, wd.data_ptr(), rows, dim, eps, CODE[dt],
                 sb.data_ptr() + st if res else 0, ld, yb.data_ptr() + st if out != "units" else 0, ld, ptr(a), ptr(b), ptr(m), s.cuda_stream)
    torch.cuda.synchronize()
    h = want_h.float().numpy()
    y64, rs = norm_ref(h, w.numpy(), eps)

    def inner(buf):
        return buf.cpu()[off:off + rows * ld].view(rows, ld)
    if res:
        got = inner(sb)
        # the same bits (a NaN's payload is the hardware's own)
        ints, nan = torch.int16 if es == 2 else torch.int32, torch.isnan(want_h)
        assert torch.equal(torch.isnan(got[:, :dim]), nan)
        assert torch.equal(got[:, :dim].contiguous().view(ints)[~nan], want_h.contiguous().view(ints)[~nan])
        if pad and not inplace:
            assert (got[:, dim:] == guard).all(), "columns behind the row were written"
    if out != "units":
        got = inner(yb)[:, :dim].float().numpy().astype(np.float64)
        ok = np.isfinite(y64)
        assert np.array_equal(np.isfinite(got), ok)
        tol = np.abs(y64[ok]) * (3.01 * 2.0 ** -24 + EPS_HALF[dt]) + {"fp32": 1e-44, "bf16": 1e-40, "fp16": 2.0 ** -25}[dt]
        assert (np.abs(got[ok] - y64[ok]) <= tol).all()
        if pad:
            assert (inner(yb)[:, dim:] == guard).all()
    if units:
        q, sc, sums = unpack_units(a[:rows].cpu().numpy(), b[:rows].cpu().numpy(), m[:rows].cpu().numpy().view(np.uint16))
        eq, es_ = norm_units_ref(h, w.numpy(), rs)
        fine = np.isfinite(h).all(1)
        assert np.array_equal(q[fine], eq[fine])
        assert np.array_equal(sc.view(np.uint16)[fine], es_.view(np.uint16)[fine])
        assert np.array_equal(sums, q.reshape(rows, nu, 2, 16).astype(np.int16).sum(-1, dtype=np.int16))
        # the values stand within half a code and the scale's half step of y
        val = q.astype(np.float64) * sc.astype(np.float64)[..., None]
        yb_ = y64.reshape(rows, nu, 32)
        step = np.abs(yb_).max(-1, keepdims=True) / 127
        assert (np.abs(val - yb_)[fine] <= (step * (0.5 + 127 * 2.0 ** -11 + 1e-3) + 127 * 2.0 ** -25)[fine]).all()
        for t, v in ((a, 99), (b, 99), (m, 999)):
            assert (t[rows] == v).all(), "written behind the last row"
        return q, sc
    return None


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(1, 64), (3, 128), (2, 1984), (5, 2048), (1, 2112), (4, 5120), (2, 8192), (3, 8256), (2, 16448), (2, 32768)])
def test_units_and_rows(qkv, torch_gpu, rows, dim, dt):
    run(torch_gpu, qkv, rows, dim, dt)


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,dim,pad,off", [(1, 1, 0, 0), (3, 7, 0, 0), (2, 8, 3, 1), (9, 1001, 0, 3), (17, 6143, 41, 0), (2, 20001, 5, 1), (1, 32767, 0, 0)])
def test_odd_rows(qkv, torch_gpu, rows, dim, pad, off, dt):
    run(torch_gpu, qkv, rows, dim, dt, out="rows", pad=pad, off=off)
    run(torch_gpu, qkv, rows, dim, dt, out="rows", res=False, pad=pad, off=off)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_unaligned_rows_with_units(qkv, torch_gpu, dt):
    run(torch_gpu, qkv, 6, 5120, dt, pad=13, off=1)
    run(torch_gpu, qkv, 6, 1024, dt, out="units", pad=1, off=5)


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
def test_in_place_and_many_rows(qkv, torch_gpu, dt):
    run(torch_gpu, qkv, 2500, 512, dt, inplace=True)
    run(torch_gpu, qkv, 1300, 5120, dt, inplace=True, out="units")


def test_offsets_past_32_bits(qkv, torch_gpu):
    """Rows 2^24 + 1 elements apart, 17 GB of them: every row's norm and sum, and nothing between them."""
    torch, rows, dim, ld = torch_gpu, 260, 100, (1 << 24) + 1
    buf = torch.zeros(rows * ld, device="cuda")
    x = torch.randn(rows, dim, device="cuda")
    v = buf.view(rows, ld)
    v[:, :dim] = x
    w = torch.ones(dim, device="cuda")
    y = torch.empty(rows, dim, device="cuda")
    qkv.norm_q32(x.data_ptr(), dim, buf.data_ptr(), ld, w.data_ptr(), rows, dim, 1e-6, 0, buf.data_ptr(), ld, y.data_ptr(), dim, 0, 0, 0)
    torch.cuda.synchronize()
    h = (2 * x).double()
    ref = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)
    assert torch.equal(v[:, :dim], 2 * x) and not v[:, dim:dim + 64].any() and not v[:, -64:].any()
    assert ((y.double() - ref).abs() <= ref.abs() * 4.01 * 2.0 ** -24).all()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_zero_tiny_and_wild_rows(qkv, torch_gpu, dt):
    def edit(x, r):
        x[0] = 0
        r[0] = 0              # a row of zeros
        x[1] = 0
        r[1] = 0
        x[1, :32] = 1e-38     # a block without a finite 127 / max
        r[2, 5] = float("inf")
        x[3, 100] = float("nan")
        x[4] *= 1e-20
        r[4] = 0
    run(torch_gpu, qkv, 6, 256, dt, edit=edit)


def test_wild_rows_units_propagate(qkv, torch_gpu):
    """A NaN in a row makes every scale of the row NaN; an infinity the scale of its block, the others zero."""
    def edit(x, r):
        x[0, 100] = float("nan")
        x[1, 40] = float("inf")
    q, sc = run(torch_gpu, qkv, 3, 256, "fp32", edit=edit)
    assert np.isnan(sc[0]).all() and np.isnan(sc[1, 1]) and (sc[1, [0, 2, 3, 4, 5, 6, 7]] == 0).all() and np.isfinite(sc[2]).all()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("eps", [0.0, 1e-38])
@pytest.mark.parametrize("dim", [256, 5120, 20032])
def test_rows_near_the_ends_of_the_type(qkv, torch_gpu, dim, eps, dt):
    """Rows whose factor 1 / sqrt(mean) is near fp32's largest or smallest number or past them: y and its units are ordinary.
    y carries three roundings and its own; a code the rounding to an integer and four (t, 127 / max, their product, the largest
    value's), a scale those and fp16's."""
    torch, T = torch_gpu, dtype_of(torch_gpu, dt)
    g = torch.Generator().manual_seed(dim)
    sizes = [1e-42 if dt == "fp32" else 5e-40, 3e-39, 1e-38, 1e-36, 1e-20, 1e-6, 1.0, 1e6, 1e12, 1e20, 1e30, 5e36, 1.0, 1.0]
    x = torch.randn(len(sizes), dim, generator=g).clamp(-4, 4).double() * torch.tensor(sizes, dtype=torch.float64)[:, None]
    x[-2] = 3e38 * torch.sign(x[-2])                              # close to the largest number everywhere
    x[-1, :32] *= 1e-38                                            # a block with next to nothing in an ordinary row
    x = x.to(T)
    w = 1 + 0.2 * torch.randn(dim, generator=g)
    w[64:96] *= 1e4                                                # (a block's products beyond the row's own range)
    rows, nu = len(sizes), dim // 32
    xd, wd = x.cuda(), w.cuda()
    y = torch.empty_like(xd)
    a, b = (torch.empty(rows, nu, 16, dtype=torch.int8, device="cuda") for _ in range(2))
    m = torch.empty(rows, nu, 4, dtype=torch.int16, device="cuda")
    qkv.norm_q32(xd.data_ptr(), dim, 0, 0, wd.data_ptr(), rows, dim, eps, CODE[dt], 0, 0, y.data_ptr(), dim, a.data_ptr(), b.data_ptr(), m.data_ptr(),
                 torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    h, wn = x.double().numpy(), w.double().numpy()
    rs = 1 / np.sqrt((h * h).mean(1, keepdims=True) + np.float64(np.float32(eps)))
    y64, got = h * rs * wn, y.double().cpu().numpy()
    assert (np.abs(got - y64) <= np.abs(y64) * (3.01 * 2.0 ** -24 + EPS_HALF[dt]) + (1e-44 if dt == "fp32" else 1e-40)).all()
    q, sc, sums = unpack_units(a.cpu().numpy(), b.cpu().numpy(), m.cpu().numpy().view(np.uint16))
    assert np.array_equal(sums, q.reshape(rows, nu, 2, 16).astype(np.int16).sum(-1, dtype=np.int16))
    t = (h * wn).reshape(rows, nu, 32)
    top = np.abs(t).max(-1)
    scale = top * rs / 127
    assert (np.abs(sc.astype(np.float64) - scale) <= scale * (2.0 ** -11 + 4.01 * 2.0 ** -24) + 2.0 ** -25).all()
    some = scale > 2.0 ** -25                                      # (a scale of zero leaves its codes without a meaning)
    want = t[some] * 127 / top[some][:, None]
    assert (np.abs(q[some] - want) <= 0.5 + 127 * 4.01 * 2.0 ** -24).all()
    assert some[:-1].all() == (eps == 0)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_rows_without_a_value(qkv, torch_gpu, dt):
    """Zeros over an eps of 0: NaN.  An infinity: NaN in its own place and its block's scale, zeros elsewhere.  A NaN: all of its row."""
    torch, T = torch_gpu, dtype_of(torch_gpu, dt)
    x = torch.randn(4, 128).to(T)
    x[0], x[1, 40], x[2, 3] = 0, -float("inf"), float("nan")
    xd, w = x.cuda(), torch.ones(128, device="cuda")
    y = torch.zeros_like(xd)
    a, b = (torch.zeros(4, 4, 16, dtype=torch.int8, device="cuda") for _ in range(2))
    m = torch.zeros(4, 4, 4, dtype=torch.int16, device="cuda")
    qkv.norm_q32(xd.data_ptr(), 128, 0, 0, w.data_ptr(), 4, 128, 0.0, CODE[dt], 0, 0, y.data_ptr(), 128, a.data_ptr(), b.data_ptr(), m.data_ptr(),
                 torch.cuda.current_stream().cuda_stream)
    got = y.float().cpu().numpy()
    _, sc, _ = unpack_units(a.cpu().numpy(), b.cpu().numpy(), m.cpu().numpy().view(np.uint16))
    assert np.isnan(got[[0, 2]]).all() and np.isnan(sc[[0, 2]]).all() and np.isfinite(got[3]).all() and np.isfinite(sc[3]).all()
    assert np.isnan(got[1, 40]) and (np.delete(got[1], 40) == 0).all() and np.isnan(sc[1, 1]) and (sc[1, [0, 2, 3]] == 0).all()


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,dim,pad", [(1, 64, 0), (3, 5120, 0), (2, 777, 3), (600, 1024, 8), (2, 32768, 1)])
def test_in_place_and_unstored(qkv, torch_gpu, rows, dim, pad, dt):
    """y in the place of x, the sum in the place of the residual or not stored at all: the bits of the call with outputs of its own."""
    torch, T, ld = torch_gpu, dtype_of(torch_gpu, dt), dim + pad
    x, r = (torch.randn(rows, ld, device="cuda").to(T) for _ in range(2))
    w = 1 + 0.2 * torch.randn(dim, device="cuda")
    units = dim % 64 == 0

    def call(x, r, sum, y):
        u = [torch.zeros(rows, dim // 32, k, dtype=t, device="cuda") for k, t in ((16, torch.int8), (16, torch.int8), (4, torch.int16))] if units else [None] * 3
        qkv.norm_q32(x.data_ptr(), ld, r.data_ptr(), ld, w.data_ptr(), rows, dim, 1e-6, CODE[dt], ptr(sum), ld, ptr(y), ld, *(ptr(t) for t in u),
                     torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return u
    sums, y = torch.zeros_like(x), torch.zeros_like(x)
    u0 = call(x, r, sums, y)
    assert torch.equal(sums[:, :dim], (x.float() + r.float()).to(T)[:, :dim])
    for inplace_x, inplace_r in ((True, False), (True, True), (False, False)):
        x1, r1 = x.clone(), r.clone()
        y1 = x1 if inplace_x else torch.zeros_like(x)
        u1 = call(x1, r1, r1 if inplace_r else None, y1)
        assert torch.equal(y1[:, :dim], y[:, :dim]) and torch.equal(y1[:, dim:], (x if inplace_x else torch.zeros_like(x))[:, dim:])
        assert torch.equal(r1[:, :dim], (sums if inplace_r else r)[:, :dim]) and torch.equal(r1[:, dim:], r[:, dim:])
        assert all(torch.equal(p, q) for p, q in zip(u0, u1)) if units else True


def test_no_rows(qkv, torch_gpu):
    torch = torch_gpu
    x = torch.ones(64, device="cuda")
    y = torch.full((64,), 5.0, device="cuda")
    qkv.norm_q32(x.data_ptr(), 64, 0, 0, x.data_ptr(), 0, 64, 1e-6, 0, 0, 0, y.data_ptr(), 64)
    torch.cuda.synchronize()
    assert (y == 5).all()


def test_host_memory_refused(qkv, torch_gpu):
    torch = torch_gpu
    x = torch.ones(64, device="cuda")
    for h in (torch.ones(64), torch.ones(64).pin_memory()):
        with pytest.raises(qkv.KVError, match="not device memory"):
            qkv.norm_q32(x.data_ptr(), 64, 0, 0, h.data_ptr(), 1, 64, 1e-6, 0, 0, 0, x.data_ptr(), 64)
        with pytest.raises(qkv.KVError, match="not device memory"):
            qkv.norm_q32(x.data_ptr(), 64, 0, 0, x.data_ptr(), 1, 64, 1e-6, 0, 0, 0, h.data_ptr(), 64)
    torch.zeros(1, device="cuda")  # (no error left behind)
    torch.cuda.synchronize()
