"""The experts of a layer with 4-bit weights (mk_moe_rows, mk_moe_units, mk_moe_layer) against 64 bits."""
import numpy as np
import pytest

from mixcase import moe_ref, to_gpu, typed, w4_values
from stepcase import CODE, pack_codes, ptr, units_of, unpack_units

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, torch, rows, dim, inner, e, top, group=32, mins=False, xform="bf16", ids=None, seed=0, pad=0, router=None, x=None):
        rng = np.random.default_rng(seed)
        self.torch, self.rows, self.dim, self.inner, self.e, self.top, self.group, self.xform = torch, rows, dim, inner, e, top, group, xform
        self.w, self.dev, self.mags = [], [], []
        for n, k in ((2 * inner, dim), (dim, inner)):
            gs = -(-k // group)
            c = rng.integers(0, 16, (e, n, k), dtype=np.uint8)
            s = ((rng.random((e, n, gs)) + 0.5) * 0.25 / np.sqrt(k)).astype(np.float16)
            m = (rng.standard_normal((e, n, gs)) * 0.2 / np.sqrt(k)).astype(np.float16) if mins else None
            self.w.append(w4_values(c, s, m, group))
            mag = np.abs(w4_values(c, s, None, group))
            self.mags.append(mag if m is None else mag + np.abs(m.astype(np.float64))[..., np.arange(k) // group])
            codes = pack_codes(c.reshape(e * n, k))
            self.dev.append([torch.from_numpy(codes).cuda(), torch.from_numpy(s).cuda(), None if m is None else torch.from_numpy(m).cuda()])
        x = rng.standard_normal((rows, dim)) if x is None else x
        if xform == "units":
            u = units_of(x)
            q, sc, _ = unpack_units(*u)
            self.xv = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(rows, dim)
            self.x = [torch.from_numpy(np.ascontiguousarray(t.view(np.int16) if t.dtype == np.uint16 else t)).cuda() for t in u]
            self.yname = "fp32"
        else:
            xb, self.xv = typed(x, xform)
            self.x = torch.full((rows, dim + pad), float("nan"), device="cuda").to(to_gpu(torch, xb[:0], xform).dtype)
            self.x[:, :dim] = to_gpu(torch, xb, xform)
            self.yname = xform
        if ids is None:
            ids = np.stack([rng.permutation(e)[:top] for _ in range(rows)]) if rows else np.zeros((0, top))
        self.ids = np.asarray(ids).astype(np.int32).reshape(rows, top)
        self.weights = rng.standard_normal((rows, top)).astype(np.float32)
        self.chosen = [torch.from_numpy(self.ids).cuda(), torch.from_numpy(self.weights).cuda()]
        ydt = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[self.yname]
        self.y = torch.full((rows + 2, dim + 3), 7.0, device="cuda").to(ydt)
        self.router = None
        if router:
            rb, self.rv = typed(rng.standard_normal((e, dim)) * 2 / np.sqrt(dim), router)
            self.router, self.rname = to_gpu(torch, rb, router), router
            self.logits = torch.empty(rows, e, device="cuda")

    def out(self):
        return self.y[1:self.rows + 1, 1:self.dim + 1]

    def run(self, qkv, stream=0, ws=None, layer=False):
        torch, y = self.torch, self.out()
        need = qkv.moe_ws(self.rows, self.dim, self.inner, self.e, self.top)
        self.ws = torch.full((need // 4 + 4,), float("nan"), device="cuda") if ws is None else ws
        head = (self.rows, self.dim, self.inner, self.e, self.top, self.group, *(ptr(t) for d in self.dev for t in d))
        tail = (self.chosen[0].data_ptr(), self.chosen[1].data_ptr(), y.data_ptr(), y.stride(0), self.ws.data_ptr(), need, stream)
        if self.xform == "units":
            qkv.moe_units(*head, *(t.data_ptr() for t in self.x), *tail)
        elif layer:
            qkv.moe_layer(*head, self.x.data_ptr(), self.x.stride(0), CODE[self.xform], self.router.data_ptr(), CODE[self.rname], 0, 1, 1.0, self.logits.data_ptr(), *tail)
        else:
            qkv.moe_rows(*head, self.x.data_ptr(), self.x.stride(0), CODE[self.xform], *tail)
        return y

    def want(self):
        return moe_ref(self.w[0], self.w[1], self.mags, self.xv, self.xform, self.ids, self.weights, self.yname, self.group)

    def check(self, qkv):
        y = self.run(qkv).double().cpu().numpy()
        ref, bound = self.want()
        err = np.abs(y - ref)
        assert (err <= bound).all(), (np.argwhere(~(err <= bound))[:5], float(np.nanmax(err / bound)))
        full = self.y.float().cpu().numpy()
        full[1:self.rows + 1, 1:self.dim + 1] = 7
        assert (full == 7).all()  # what lies around y is left as it was
        return y


FORMS = ["units", "fp32", "fp16", "bf16"]


@pytest.mark.parametrize("xform", FORMS)
@pytest.mark.parametrize("group,mins", [(32, False), (64, True), (128, False), (32, True), (128, True), (64, False)])
@pytest.mark.parametrize("rows,dim,inner,e,top", [(1, 64, 32, 1, 1), (1, 320, 96, 6, 3), (5, 192, 288, 4, 2), (17, 576, 64, 9, 4)])
def test_shapes(qkv, torch_gpu, xform, group, mins, rows, dim, inner, e, top):
    Case(torch_gpu, rows, dim, inner, e, top, group, mins, xform, seed=rows + group, pad=rows % 4).check(qkv)


@pytest.mark.parametrize("xform", FORMS[1:])
def test_dim_of_one_block_more(qkv, torch_gpu, xform):
    Case(torch_gpu, 3, 96, 32, 3, 2, xform=xform).check(qkv)
    Case(torch_gpu, 2, 32, 352, 2, 2, 64, True, xform=xform).check(qkv)


@pytest.mark.parametrize("xform,rows,dim,inner,e,top", [("bf16", 64, 256, 128, 16, 4), ("fp32", 65, 128, 64, 3, 2), ("units", 200, 128, 96, 5, 3), ("fp16", 130, 64, 64, 2, 1),
                                                        ("fp32", 2, 5120, 64, 2, 1), ("bf16", 3, 64, 5120, 2, 1), ("fp32", 1, 32, 32768, 1, 1), ("bf16", 1, 16384, 32, 1, 1),
                                                        ("bf16", 9, 64, 32, 1024, 16)])
def test_larger(qkv, torch_gpu, xform, rows, dim, inner, e, top):
    Case(torch_gpu, rows, dim, inner, e, top, xform=xform, seed=rows).check(qkv)


@pytest.mark.parametrize("xform", FORMS)
@pytest.mark.parametrize("group,mins,dim,inner,top", [(32, False, 64, 768, 2), (64, True, 4160, 288, 1), (128, True, 128, 2080, 3), (32, True, 192, 64, 16), (128, False, 4224, 544, 5)])
def test_one_row(qkv, torch_gpu, xform, group, mins, dim, inner, top):
    """A single row: parts of inner, two tiles of columns, the same expert twice, choices that are no expert, none at all."""
    rng = np.random.default_rng(dim)
    Case(torch_gpu, 1, dim, inner, max(5, top), top, group, mins, xform, ids=rng.integers(0, 5, (1, top)), seed=top).check(qkv)
    Case(torch_gpu, 1, dim, inner, max(5, top), top, group, mins, xform, ids=rng.integers(-3, 8, (1, top)), seed=top).check(qkv)
    y = Case(torch_gpu, 1, dim, inner, max(5, top), top, group, mins, xform, ids=np.full((1, top), 2 ** 31 - 1)).check(qkv)
    assert (y == 0).all()


@pytest.mark.parametrize("xform", FORMS)
def test_skewed(qkv, torch_gpu, xform):
    """All rows on one expert (several passes), the same expert twice in a row, choices that are no expert."""
    for rows in (16, 33, 64):
        Case(torch_gpu, rows, 128, 64, 4, 2, xform=xform, ids=np.tile([2, 0], (rows, 1)), seed=rows).check(qkv)
    Case(torch_gpu, 20, 128, 64, 4, 3, xform=xform, ids=np.tile([1, 1, 1], (20, 1))).check(qkv)
    rng = np.random.default_rng(1)
    c = Case(torch_gpu, 20, 128, 64, 4, 3, xform=xform, ids=rng.integers(-2, 7, (20, 3)))
    c.ids[4] = c.ids[11] = [-1, 4, 2 ** 31 - 1]
    c.chosen[0] = torch_gpu.from_numpy(c.ids).cuda()
    y = c.check(qkv)
    assert (y[4] == 0).all()
    y = Case(torch_gpu, 5, 64, 32, 2, 2, xform=xform, ids=np.full((5, 2), -1)).check(qkv)
    assert (y == 0).all()


@pytest.mark.parametrize("xform", FORMS)
@pytest.mark.parametrize("mins", [False, True])
def test_not_finite(qkv, torch_gpu, xform, mins):
    """A row of x with an infinity or a NaN is NaN in y, and alone; an expert's reach the rows that chose it alone."""
    torch = torch_gpu
    ids = np.arange(40).reshape(20, 2) % 5
    c = Case(torch, 20, 128, 96, 5, 2, mins=mins, xform=xform, ids=ids, seed=2)
    clean = c.run(qkv).clone()
    hit = [3, 8]
    if xform == "units":
        c.x[2][3] = 0x7c00
        c.x[2][8] = 0x7e00
    else:
        c.x[3, 70], c.x[8, 5] = float("inf"), float("nan")
    y = c.run(qkv)
    rest = [m for m in range(20) if m not in hit]
    assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[hit]).all()
    c = Case(torch, 20, 128, 96, 5, 2, mins=mins, xform=xform, ids=ids, seed=2)
    c.dev[0][1].view(torch.int16)[2, 40, 1] = 0x7e00  # a scale of expert 2
    y = c.run(qkv)
    for m in range(20):
        if 2 in ids[m]:
            assert torch.isnan(y[m]).all()
        else:
            assert torch.equal(y[m], clean[m])


def test_rows_apart(qkv, torch_gpu):
    """A row's result does not depend on the rows beside it."""
    torch = torch_gpu
    c = Case(torch, 40, 256, 96, 6, 2, xform="bf16", seed=6)
    all_rows = c.run(qkv).clone()
    for m in (0, 7, 39):
        one = Case(torch, 40, 256, 96, 6, 2, xform="bf16", seed=6)
        one.rows, one.x = 1, one.x[m:m + 1]
        one.chosen = [t[m:m + 1].contiguous() for t in one.chosen]
        assert torch.equal(one.run(qkv)[0], all_rows[m])


@pytest.mark.parametrize("xform", FORMS[1:])
@pytest.mark.parametrize("rows", [1, 8, 70])
def test_layer(qkv, torch_gpu, xform, rows):
    """The layer is the router and the experts, to the bit."""
    torch = torch_gpu
    c = Case(torch, rows, 320, 96, 20, 3, xform=xform, seed=rows, router="bf16" if xform == "bf16" else "fp32", pad=1)
    c.chosen[0].fill_(-5)
    y = c.run(qkv, layer=True).clone()
    ids, weights, logits = c.chosen[0].clone(), c.chosen[1].clone(), c.logits.clone()
    c.ids, c.weights = ids.cpu().numpy(), weights.cpu().numpy()
    ref, bound = c.want()
    assert (np.abs(y.double().cpu().numpy() - ref) <= bound).all()
    need = qkv.moe_route_ws(rows, 320, 20)
    ws = torch.empty(need + 16, device="cuda", dtype=torch.uint8)
    qkv.moe_route(rows, 320, 20, 3, c.x.data_ptr(), c.x.stride(0), CODE[xform], c.router.data_ptr(), CODE[c.rname], 0, 1, 1.0, c.logits.data_ptr(), c.chosen[0].data_ptr(),
                  c.chosen[1].data_ptr(), ws.data_ptr(), need)
    assert torch.equal(c.logits, logits) and torch.equal(c.chosen[0], ids) and torch.equal(c.chosen[1], weights)
    assert torch.equal(c.run(qkv), y)


def test_same_bits_streams_graph(qkv, torch_gpu):
    """The same bits on every run, on two streams at once, and on replays of a graph between other work."""
    torch = torch_gpu
    cs = [Case(torch, r, 512, 192, 12, 3, xform="bf16", seed=r, router="bf16") for r in (2, 50)]
    want = [c.run(qkv, layer=True).clone() for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                c.run(qkv, s.cuda_stream, ws=c.ws, layer=True)
    torch.cuda.synchronize()
    for c, w in zip(cs, want):
        assert torch.equal(c.out(), w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in cs:
            c.run(qkv, torch.cuda.current_stream().cuda_stream, ws=c.ws, layer=True)
    for _ in range(4):
        for c in cs:
            c.y.zero_()
            c.x.mul_(-1.5)  # (other experts)
        g.replay()
        torch.cuda.synchronize()
        got = [c.out().clone() for c in cs]
        for c, y in zip(cs, got):
            assert torch.equal(c.run(qkv, ws=c.ws, layer=True), y)
        torch.cuda.synchronize()


def test_far_offsets(qkv, torch_gpu):
    """Experts whose codes lie past 2^32 bytes."""
    torch = torch_gpu
    e, dim, inner = 40, 8192, 16384
    up = torch.full((e, 2 * inner, dim // 2), 0x88, device="cuda", dtype=torch.uint8)  # codes of 8: zeros
    down = torch.full((e, dim, inner // 2), 0x88, device="cuda", dtype=torch.uint8)
    us = torch.ones(e, 2 * inner, dim // 128, device="cuda", dtype=torch.float16)
    ds = torch.ones(e, dim, inner // 128, device="cuda", dtype=torch.float16)
    last = dim // 2 - 1  # byte 3 of the last word: value k - 1 in its high nibble
    up[e - 1, inner - 1, last] = 0xC8      # gate: 4
    up[e - 1, 2 * inner - 1, last] = 0xA8  # up: 2
    down[e - 1, dim - 1, inner // 2 - 1] = 0x98  # 1
    x = torch.zeros(1, dim, device="cuda")
    x[0, dim - 1] = 3
    ids = torch.tensor([[e - 1]], device="cuda", dtype=torch.int32)
    w, y = torch.ones(1, 1, device="cuda"), torch.empty(1, dim, device="cuda")
    need = qkv.moe_ws(1, dim, inner, e, 1)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    qkv.moe_rows(1, dim, inner, e, 1, 128, up.data_ptr(), us.data_ptr(), 0, down.data_ptr(), ds.data_ptr(), 0, x.data_ptr(), dim, 0, ids.data_ptr(), w.data_ptr(), y.data_ptr(),
                 dim, ws.data_ptr(), need)
    g = 12.0
    want = g / (1 + np.exp(-g)) * 6
    assert abs(float(y[0, dim - 1]) - want) <= 2.0 ** -20 * want and (y[0, :-1] == 0).all()


@pytest.mark.parametrize("xform", FORMS[1:])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_wide_range(qkv, torch_gpu, xform, group):
    """Values whose size differs from block to block, and in one: a block's small ones are off by its largest's steps."""
    rng = np.random.default_rng(group)
    size = 2.0 ** rng.integers(-9, 4, (6, 9)).repeat(32, 1) * 2.0 ** rng.integers(-3, 3, (6, 288))
    Case(torch_gpu, 6, 288, 160, 4, 2, group, True, xform, x=rng.standard_normal((6, 288)) * size).check(qkv)


@pytest.mark.parametrize("xform", FORMS)
@pytest.mark.parametrize("group,mins", [(32, True), (128, False)])
@pytest.mark.parametrize("dim,inner", [(8192, 32), (64, 6400)])
def test_long_rows_of_many(qkv, torch_gpu, xform, group, mins, dim, inner):
    """One expert's tokens past a workgroup's memory: k in parts."""
    Case(torch_gpu, 40, dim, inner, 2, 1, group, mins, xform, ids=np.zeros((40, 1)), seed=dim).check(qkv)


def test_layer_of_many_rows(qkv, torch_gpu):
    """Rows that the router takes in one kernel, 64 at a time through the experts."""
    torch = torch_gpu
    c = Case(torch, 1030, 64, 32, 6, 2, xform="fp16", seed=5, router="fp16")
    y = c.run(qkv, layer=True).clone()
    c.ids, c.weights = c.chosen[0].cpu().numpy(), c.chosen[1].cpu().numpy()
    logits = c.xv @ c.rv.T
    assert np.array_equal(c.ids, np.argsort(-logits, 1, kind="stable")[:, :2])
    ref, bound = c.want()
    assert (np.abs(y.double().cpu().numpy() - ref) <= bound).all()
    assert torch.equal(c.run(qkv), y)


def test_layer_many_experts(qkv, torch_gpu):
    """More experts than the choice beside the rows takes; runs of 64 rows."""
    torch = torch_gpu
    for rows in (3, 70):
        c = Case(torch, rows, 96, 32, 300, 4, xform="bf16", seed=rows, router="bf16")
        y = c.run(qkv, layer=True).clone()
        c.ids, c.weights = c.chosen[0].cpu().numpy(), c.chosen[1].cpu().numpy()
        ref, bound = c.want()
        assert (np.abs(y.double().cpu().numpy() - ref) <= bound).all()
        assert torch.equal(c.run(qkv), y)
