"""Adapters of many requests (mk_lora_rows, mk_lora_units) against 64 bits."""
import numpy as np
import pytest

from mixcase import bits16, lora_ref, to_gpu, typed
from stepcase import CODE, ptr, unpack_units, units_of

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, torch, rows, n, k, rank, na, xform="bf16", wname="bf16", ranks=False, scales=True, base=True, ids=None, seed=0, pad=0, x=None):
        rng = np.random.default_rng(seed)
        self.torch, self.n, self.k, self.rank, self.na, self.rows, self.xform, self.wname = torch, n, k, rank, na, rows, xform, wname
        ab, self.av = bits16(rng.standard_normal((na, rank, k)) / np.sqrt(k), wname)
        bb, self.bv = bits16(rng.standard_normal((na, n, rank)), wname)
        self.a, self.b = to_gpu(torch, ab, wname), to_gpu(torch, bb, wname)
        self.ranks = rng.integers(0, rank + 1, na).astype(np.int32) if ranks else None
        self.scales = (rng.random(na) + 0.5).astype(np.float32) if scales else None
        self.ids = (rng.integers(-1, na + 1, rows) if ids is None else np.asarray(ids)).astype(np.int32)
        x = rng.standard_normal((rows, k)) if x is None else x
        if xform == "units":
            u = units_of(x)
            q, sc, _ = unpack_units(*u)
            self.xv = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(rows, k)
            self.x = [torch.from_numpy(np.ascontiguousarray(t.view(np.int16) if t.dtype == np.uint16 else t)).cuda() for t in u]
        else:
            xb, self.xv = typed(x, xform)
            full = torch.full((rows, k + pad), float("nan"), device="cuda").to(to_gpu(torch, xb[:0], xform).dtype)
            full[:, :k] = to_gpu(torch, xb, xform)
            self.x = full
        self.base = rng.standard_normal((rows, n)).astype(np.float32) if base else None
        self.dev = [None if t is None else torch.from_numpy(t).cuda() for t in (self.ranks, self.scales, self.ids, self.base)]
        self.y = torch.full((rows + 2, n + 3), 7.0, device="cuda")

    def run(self, qkv, stream=0, ws=None, y=None, base=None):
        torch, (ranks, scales, ids, b0) = self.torch, self.dev
        self.need = qkv.lora_ws(self.rows, self.k, self.rank)
        self.ws = torch.full((self.need // 4 + 4,), float("nan"), device="cuda") if ws is None else ws
        y = self.y[1:self.rows + 1, 1:self.n + 1] if y is None else y
        base = b0 if base is None else base
        head = (self.rows, self.n, self.k, self.na, self.rank, self.a.data_ptr(), self.b.data_ptr(), CODE[self.wname], ptr(ranks), ptr(scales), ids.data_ptr())
        tail = (ptr(base), self.n if base is None else base.stride(0), y.data_ptr(), y.stride(0), self.ws.data_ptr(), self.need, stream)
        if self.xform == "units":
            qkv.lora_units(*head, *(t.data_ptr() for t in self.x), *tail)
        else:
            qkv.lora_rows(*head, self.x.data_ptr(), self.x.stride(0), CODE[self.xform], *tail)
        return y

    def want(self):
        chunks = max(1, self.need // (4 * max(self.rows, 1) * ((self.rank + 15) // 16 * 16)))
        return lora_ref(self.av, self.bv, self.ranks, self.scales, self.ids, self.xv, None if self.base is None else self.base.astype(np.float64), chunks)

    def check(self, qkv):
        y = self.run(qkv).cpu().numpy()
        ref, bound = self.want()
        err = np.abs(y - ref)
        assert (err <= bound).all(), (np.argwhere(~(err <= bound))[:5], float(np.nanmax(err / bound)))
        full = self.y.cpu().numpy()
        full[1:self.rows + 1, 1:self.n + 1] = 7
        assert (full == 7).all()  # what lies around y is left as it was
        return y


@pytest.mark.parametrize("xform", ["units", "fp32", "fp16", "bf16"])
@pytest.mark.parametrize("wname", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,n,k,rank,na", [(1, 64, 64, 16, 1), (1, 1, 64, 1, 3), (3, 33, 128, 7, 2), (16, 200, 320, 32, 5), (17, 95, 640, 16, 40),
                                              (64, 130, 1088, 65, 9), (300, 70, 192, 24, 3)])
def test_shapes(qkv, torch_gpu, xform, wname, rows, n, k, rank, na):
    Case(torch_gpu, rows, n, k, rank, na, xform, wname, ranks=rank > 1, seed=rows + rank, pad=0 if xform == "units" else rows % 4).check(qkv)


@pytest.mark.parametrize("rows,n,k,rank,na", [(1, 6144, 5120, 16, 2), (40, 4099, 5120, 64, 30), (1000, 1100, 2048, 128, 4), (2, 100, 32768, 256, 2), (257, 1500, 96, 16, 2)])
def test_larger(qkv, torch_gpu, rows, n, k, rank, na):
    Case(torch_gpu, rows, n, k, rank, na, "bf16" if rows % 2 else "fp32", "bf16", ranks=True, seed=rank).check(qkv)


@pytest.mark.parametrize("rows", [5, 64, 300])
def test_ids(qkv, torch_gpu, rows):
    """Runs, the same adapter everywhere, none anywhere, ids far outside."""
    for ids in (np.zeros(rows), np.full(rows, -1), np.full(rows, 2 ** 31 - 1), np.full(rows, -2 ** 31), np.arange(rows) // 7 % 4, (np.arange(rows) * 5) % 6 - 1):
        Case(torch_gpu, rows, 50, 96, 12, 4, ids=ids.astype(np.int64)).check(qkv)


def test_without(qkv, torch_gpu):
    """No base, no scales; then in place of base."""
    torch = torch_gpu
    c = Case(torch, 37, 75, 256, 16, 3, base=False, scales=False)
    y = c.check(qkv)
    assert (y[c.ids < 0] == 0).all()
    c = Case(torch, 37, 75, 256, 16, 3, "units")
    at = torch.full((37, 80), 5.0, device="cuda")[:, :75]
    at.copy_(c.dev[3])
    y = c.run(qkv, y=at, base=at).cpu().numpy()
    ref, bound = c.want()
    assert (np.abs(y - ref) <= bound).all()


def test_base_bits(qkv, torch_gpu):
    """Rows without an adapter, and rows of adapters of rank 0, are base to the bit, NaNs and infinities among them."""
    c = Case(torch_gpu, 20, 40, 64, 8, 2, ids=[-1, 0, 1, 5] * 5)
    c.dev[0] = torch_gpu.tensor([0, 8], dtype=torch_gpu.int32, device="cuda")
    c.dev[3][0, 3] = float("inf")
    c.dev[3][1, 4] = float("nan")
    y = c.run(qkv)
    for m in range(20):
        if m % 4 != 2:
            assert torch_gpu.equal(y[m].view(torch_gpu.int32), c.dev[3][m].view(torch_gpu.int32))


@pytest.mark.parametrize("xform", ["units", "fp32", "fp16", "bf16"])
@pytest.mark.parametrize("wname", ["fp16", "bf16"])
def test_not_finite(qkv, torch_gpu, xform, wname):
    """A row's infinities and NaNs stay in it, an adapter's in its rows."""
    torch = torch_gpu
    c = Case(torch, 40, 70, 128, 20, 3, xform, wname, ids=np.arange(40) % 4 - 1, seed=3)
    clean = c.run(qkv).clone()
    if xform == "units":
        c.x[2][5] = 0x7c00  # every scale of the row infinite
    else:
        c.x[5, 3], c.x[6, 100] = float("inf"), float("nan")
    y = c.run(qkv).clone()
    hit = [5] if xform == "units" else [5, 6]
    rest = [m for m in range(40) if m not in hit]
    assert torch.equal(y[rest], clean[rest])
    for m in hit:
        assert not torch.isfinite(y[m]).any()
    c = Case(torch, 40, 70, 128, 20, 3, xform, wname, ids=np.arange(40) % 4 - 1, seed=3)
    c.a[1, 4, 7] = float("nan")
    c.b[2, 9, 0] = float("inf")
    y = c.run(qkv)
    for m in range(40):
        i = m % 4 - 1
        if i == 1:
            assert torch.isnan(y[m]).all()
        elif i == 2:
            keep = [j for j in range(70) if j != 9]
            assert torch.equal(y[m, keep], clean[m, keep]) and not torch.isfinite(y[m, 9])
        else:
            assert torch.equal(y[m], clean[m])


def test_unused_ranks(qkv, torch_gpu):
    """What lies behind an adapter's ranks is not used, whatever it holds."""
    c = Case(torch_gpu, 30, 64, 96, 40, 2, ids=np.arange(30) % 2, seed=4)
    c.ranks = np.array([13, 33], np.int32)
    c.dev[0] = torch_gpu.from_numpy(c.ranks).cuda()
    for i, q in enumerate(c.ranks):
        c.a[i, q:] = float("nan")
        c.b[i, :, q:] = float("nan")
    c.check(qkv)


def test_extremes(qkv, torch_gpu):
    """fp32 rows of very large and very small values, and values that cancel."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 256)) * np.array([1e30, 1e-30, 1e4, 1e-4, 1, 1])[:, None]
    x[4, 1::2] = -x[4, ::2]
    Case(torch_gpu, 6, 50, 256, 16, 2, "fp32", "fp16", ids=[0, 1, 0, 1, 0, 1], x=x, base=False).check(qkv)


def test_same_bits_streams_graph(qkv, torch_gpu):
    """The same bits on every run, on two streams at once, and on replays of a graph between other work."""
    torch = torch_gpu
    cs = [Case(torch, r, 700, 512, 16, 6, "bf16", seed=r) for r in (9, 64)]
    want = [c.run(qkv).clone() for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                c.run(qkv, s.cuda_stream, ws=c.ws)
    torch.cuda.synchronize()
    for c, w in zip(cs, want):
        assert torch.equal(c.y[1:c.rows + 1, 1:c.n + 1], w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in cs:
            c.run(qkv, torch.cuda.current_stream().cuda_stream, ws=c.ws)
    for i in range(4):
        for c in cs:
            c.y.zero_()
            c.x.mul_(0.5)
        g.replay()
        torch.cuda.synchronize()
        got = [c.y[1:c.rows + 1, 1:c.n + 1].clone() for c in cs]
        for c, y in zip(cs, got):
            assert torch.equal(c.run(qkv, ws=c.ws), y)
        torch.cuda.synchronize()


def test_far_offsets(qkv, torch_gpu):
    """Adapters whose elements lie past 2^32 bytes."""
    torch = torch_gpu
    na, rank, k, n = 1100, 32, 65536, 64
    a = torch.zeros(na, rank, k, device="cuda", dtype=torch.bfloat16)
    b = torch.zeros(na, n, rank, device="cuda", dtype=torch.bfloat16)
    a[na - 1, rank - 1, k - 1] = 2
    b[na - 1, n - 1, rank - 1] = 3
    x = torch.zeros(1, k, device="cuda")
    x[0, k - 1] = 5
    ids = torch.tensor([na - 1], device="cuda", dtype=torch.int32)
    y = torch.empty(1, n, device="cuda")
    ws = torch.empty(qkv.lora_ws(1, k, rank), device="cuda", dtype=torch.uint8)
    qkv.lora_rows(1, n, k, na, rank, a.data_ptr(), b.data_ptr(), 2, 0, 0, ids.data_ptr(), x.data_ptr(), k, 0, 0, 0, y.data_ptr(), n, ws.data_ptr(), ws.numel())
    want = torch.zeros(1, n, device="cuda")
    want[0, n - 1] = 30
    assert torch.equal(y, want)


@pytest.mark.parametrize("xform", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("wname", ["fp16", "bf16"])
def test_wide_range(qkv, torch_gpu, xform, wname):
    """Values whose size differs from step to step, and in one."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((33, 256)) * 2.0 ** rng.integers(-8, 5, (33, 8)).repeat(32, 1) * 2.0 ** rng.integers(-5, 3, (33, 256))
    Case(torch_gpu, 33, 90, 256, 40, 3, xform, wname, x=x, seed=9).check(qkv)


@pytest.mark.parametrize("wname", ["fp16", "bf16"])
@pytest.mark.parametrize("rank", [64, 100, 256])
def test_many_rows_long_ranks(qkv, torch_gpu, wname, rank):
    """Tiles of 32 rows and more than one part of the ranks; runs of rows of one adapter, as of prompts."""
    Case(torch_gpu, 530, 70, 64, rank, 4, "bf16", wname, ranks=True, ids=np.arange(530) // 130 - 1, seed=rank).check(qkv)
