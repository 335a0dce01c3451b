"""The kernel that the router takes for many rows of 16-bit types (from 1536 on), and both sides of that number: sums in fp32, the choice of 64-bit ones."""
import numpy as np
import pytest

from mixcase import route_ref, typed
import test_gpu_route
from test_gpu_route import grid, run

pytestmark = pytest.mark.gpu
MANY = 1536


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,dim,e,top,form", [(MANY - 1, 256, 40, 4, 0), (MANY, 256, 40, 4, 0), (MANY, 2048, 63, 6, 0), (MANY + 6, 64, 16, 16, 1), (2001, 96, 8, 1, 2), (1600, 512, 130, 8, 3),
                                                 (1551, 1024, 256, 10, 1), (MANY + 1, 32, 1, 1, 0), (1552, 320, 72, 4, 2), (MANY, 4096, 33, 16, 0), (4099, 64, 200, 8, 1)])
@pytest.mark.parametrize("pad", [8, 3])  # (rows that do not start at 16 bytes are summed in 64 bits)
def test_sizes(qkv, torch_gpu, name, rows, dim, e, top, form, pad):
    test_gpu_route.test_many(qkv, torch_gpu, name, rows, dim, e, top, form, pad)


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("e", [20, 100, 200])
def test_close(qkv, torch_gpu, name, e):
    """Experts whose logits differ past fp32's bits, equal ones among them: the choice is that of 64-bit sums, ties to the lowest index."""
    rows, dim = 1700, 256
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


def test_small(qkv, torch_gpu):
    """Rows and experts whose squares, and whose products, are below fp32's smallest, or near its largest."""
    rows, dim, e = 1600, 256, 40
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


@pytest.mark.parametrize("e", [33, 100, 200])
def test_not_finite(qkv, torch_gpu, e):
    """Rows with infinities and NaNs: distinct experts all the same, other rows as without them."""
    rows = 1600
    rng = np.random.default_rng(11)
    x, xv = grid(rng, (rows, 96), "bf16")
    w, wv = grid(rng, (e, 96), "bf16")
    _, ri, _ = route_ref(xv, wv, None, 1, 1.0, 8)
    bad = x.copy()
    hit = (3, 4, 5, rows - 1)
    bad[3, 5], bad[4, 6], bad[5, :], bad[rows - 1, 0] = 0x7f80, 0x7fc0, 0xff80, 0x7f80
    _, ids, _ = run(qkv, torch_gpu, bad, "bf16", w, "bf16", None, 1, 1.0, 8)
    for m in range(rows):
        if m in hit:
            assert len(set(ids[m])) == 8 and (ids[m] >= 0).all() and (ids[m] < e).all()
        else:
            assert np.array_equal(ids[m], ri[m])


def test_graph(qkv, torch_gpu):
    """The same bits on replays of a graph between other work."""
    torch, rows, dim, e, top = torch_gpu, 1600, 96, 72, 4
    rng = np.random.default_rng(21)
    x, w = (torch.from_numpy(rng.standard_normal(s)).to(torch.bfloat16).cuda() for s in ((rows, dim), (e, dim)))
    need = qkv.moe_route_ws(rows, dim, e)
    ws = torch.empty(need + 16, device="cuda", dtype=torch.uint8)
    out = [torch.empty(rows, e, device="cuda"), torch.empty(rows, top, device="cuda", dtype=torch.int32), torch.empty(rows, top, device="cuda")]

    def call(stream=0):
        qkv.moe_route(rows, dim, e, top, x.data_ptr(), dim, 2, w.data_ptr(), 2, 0, 0, 1.5, *(t.data_ptr() for t in out), ws.data_ptr(), need, stream)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        x.mul_(-1.5)
        for t in out:
            t.zero_()
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        call()
        assert all(torch.equal(a, b) for a, b in zip(got, out))
        torch.cuda.synchronize()
