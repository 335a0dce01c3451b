"""The choice that a layer of up to 64 rows makes beside x (mk_moe_layer): logits, experts, weights and y are those of mk_moe_route and
mk_moe_rows to the bit, and the choice that of 64-bit sums; for every number of experts a lane can hold, form, bias, scale and number of parts of dim."""
import numpy as np
import pytest

from mixcase import route_ref, to_gpu, typed
from stepcase import CODE, ptr

pytestmark = pytest.mark.gpu
FORMS = [(0, False), (1, False), (2, False), (3, False), (2, True), (3, True)]


@pytest.mark.parametrize("xname,rname", [("fp32", "fp32"), ("fp16", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("e,top", [(20, 3), (64, 8), (65, 6), (128, 8), (129, 8), (256, 8), (256, 16), (257, 4)])
@pytest.mark.parametrize("dim", [320, 2048])
def test_choice(qkv, torch_gpu, xname, rname, e, top, dim):
    torch, inner, group, most = torch_gpu, 32, 32, 64
    rng = np.random.default_rng(e + dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(e)
    dev = []
    for n, k in ((2 * inner, dim), (dim, inner)):
        codes = torch.randint(0, 256, (e, n, k // 2), device="cuda", dtype=torch.uint8, generator=g)
        dev += [codes, ((0.5 + torch.rand(e, n, k // group, device="cuda", generator=g)) * 0.25 / k ** 0.5).half(), None]
    x, xv = typed(rng.standard_normal((most, dim)), xname)
    w, wv = typed(rng.standard_normal((e, dim)) * 2 / np.sqrt(dim), rname)
    w[e - 1], wv[e - 1] = w[2], wv[2]  # (equal logits, far apart)
    bias = rng.standard_normal(e).astype(np.float32)
    bias[e - 1] = bias[2]
    xd, wd, bd = to_gpu(torch, x, xname), to_gpu(torch, w, rname), torch.from_numpy(bias).cuda()
    need = qkv.moe_ws(most, dim, inner, e, top)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    exact = xv @ wv.T
    for rows in (1, 7, 40, 64):
        for form, biased in FORMS:
            b = bias if biased else None
            out = lambda: [torch.full(s, 7, device="cuda", dtype=t) for s, t in (((rows + 1, e), torch.float32), ((rows + 1, top), torch.int32), ((rows + 1, top), torch.float32),
                                                                                ((rows + 1, dim), xd.dtype))]
            one, two = out(), out()
            head = (rows, dim, inner, e, top, group, *(ptr(t) for t in dev), xd.data_ptr(), dim, CODE[xname])
            router = (ptr(bd) if biased else 0, form, 2.5)
            ws.fill_(0xff)
            qkv.moe_layer(*head, wd.data_ptr(), CODE[rname], *router, *(t.data_ptr() for t in one), dim, ws.data_ptr(), need)
            ws.fill_(0xff)
            qkv.moe_route(rows, dim, e, top, xd.data_ptr(), dim, CODE[xname], wd.data_ptr(), CODE[rname], *router, *(t.data_ptr() for t in two[:3]), ws.data_ptr(), need)
            ws.fill_(0xff)
            qkv.moe_rows(*head, two[1].data_ptr(), two[2].data_ptr(), two[3].data_ptr(), dim, ws.data_ptr(), need)
            for p, q in zip(one, two):
                assert torch.equal(p, q) and (p[rows] == 7).all()
            logits, ids, wt = (t[:rows].cpu().numpy() for t in one[:3])
            assert (np.abs(logits - exact[:rows]) <= 2.0 ** -24 * np.abs(exact[:rows]) + dim * 2.0 ** -52 * (np.abs(xv[:rows]) @ np.abs(wv).T)).all()
            _, ri, rw = route_ref(logits.astype(np.float64), np.eye(e), b, form, 2.5, top)
            assert np.array_equal(ids, ri) and (np.abs(wt - rw) <= 2.0 ** -23 * rw).all()
            assert np.array_equal(ids, route_ref(xv[:rows], wv, b, form, 2.5, top)[1])
