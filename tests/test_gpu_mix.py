"""The operators of a server of many requests as a layer runs them: norm, a projection with its adapters in place, norm, router and experts, whose
output the next layer's norm adds; in eager calls, in a graph, and two such layers at once."""
import numpy as np
import pytest

from mixcase import bits16, lora_ref, moe_ref, route_ref, to_gpu, w4_values
from stepcase import pack_codes, unpack_units

pytestmark = pytest.mark.gpu
N, K, RANK, NA, E, TOP, INNER = 320, 320, 20, 6, 24, 3, 96


def weights(torch, rng, e, n, k, group):
    c = rng.integers(0, 16, (e, n, k), dtype=np.uint8)
    s = ((rng.random((e, n, k // group)) + 0.5) * 0.25 / np.sqrt(k)).astype(np.float16)
    return w4_values(c, s, None, group), torch.from_numpy(pack_codes(c.reshape(e * n, k))).cuda(), torch.from_numpy(s).cuda()


class Layer:
    def __init__(self, torch, rows, seed):
        rng = np.random.default_rng(seed)
        self.torch, self.rows = torch, rows
        (ab, self.av), (bb, self.bv) = bits16(rng.standard_normal((NA, RANK, K)) / np.sqrt(K), "bf16"), bits16(rng.standard_normal((NA, N, RANK)), "bf16")
        rb, self.rv = bits16(rng.standard_normal((E, K)) * 2 / np.sqrt(K), "bf16")
        self.a, self.b, self.r = (to_gpu(torch, t, "bf16") for t in (ab, bb, rb))
        self.o, self.down = weights(torch, rng, 1, N, K, 32), weights(torch, rng, E, K, INNER, 32)
        self.up = weights(torch, rng, E, 2 * INNER, K, 32)
        self.ids = torch.from_numpy(rng.integers(-1, NA, rows).astype(np.int32)).cuda()
        self.scales = torch.from_numpy((rng.random(NA) + 0.5).astype(np.float32)).cuda()
        f = lambda *s, dt=torch.float32: torch.full(s, 3.0, device="cuda").to(dt)
        self.w, self.res, self.y, self.norm = f(K), f(rows, K), f(rows, N), f(rows, K, dt=torch.float32)
        self.x = torch.from_numpy(rng.standard_normal((rows, K)).astype(np.float32)).cuda()
        self.qa, self.qb, self.qm = f(rows * K // 2, dt=torch.int8), f(rows * K // 2, dt=torch.int8), f(rows * K // 32 * 4, dt=torch.int16)
        self.logits, self.chosen, self.wt, self.out = f(rows, E), f(rows, TOP, dt=torch.int32), f(rows, TOP), f(rows, K)

    def run(self, qkv, stream=0):
        m, p = self.rows, lambda t: t.data_ptr()
        if not hasattr(self, "ws"):
            need = max(qkv.lora_ws(m, K, RANK), qkv.moe_ws(m, K, INNER, E, TOP))
            self.ws, self.need = self.torch.empty(need, device="cuda", dtype=self.torch.uint8), need
        qkv.norm_q32(p(self.x), K, 0, 0, p(self.w), m, K, 1e-6, 0, p(self.res), K, 0, 0, p(self.qa), p(self.qb), p(self.qm), stream)
        qkv.w4_units(m, N, K, 32, p(self.o[1]), p(self.o[2]), 0, p(self.qa), p(self.qb), p(self.qm), p(self.y), N, stream)
        qkv.lora_units(m, N, K, NA, RANK, p(self.a), p(self.b), 2, 0, p(self.scales), p(self.ids), p(self.qa), p(self.qb), p(self.qm), p(self.y), N, p(self.y), N,
                       p(self.ws), self.need, stream)
        qkv.norm_q32(p(self.y), N, p(self.res), K, p(self.w), m, K, 1e-6, 0, p(self.res), K, p(self.norm), K, 0, 0, 0, stream)
        qkv.moe_layer(m, K, INNER, E, TOP, 32, p(self.up[1]), p(self.up[2]), 0, p(self.down[1]), p(self.down[2]), 0, p(self.norm), K, 0, p(self.r), 2, 0, 1, 1.0,
                      p(self.logits), p(self.chosen), p(self.wt), p(self.out), K, p(self.ws), self.need, stream)
        qkv.norm_q32(p(self.out), K, p(self.res), K, p(self.w), m, K, 1e-6, 0, p(self.res), K, 0, 0, p(self.qa), p(self.qb), p(self.qm), stream)

    def results(self):
        return [t.clone() for t in (self.y, self.norm, self.logits, self.chosen, self.wt, self.out, self.res, self.qa, self.qb, self.qm)]


@pytest.mark.parametrize("rows", [1, 7, 40])
def test_against_64_bits(qkv, torch_gpu, rows):
    """Each call's result from what the one before left, within its own bound."""
    torch, c = torch_gpu, Layer(torch_gpu, rows, rows)
    p = lambda t: t.data_ptr()
    qkv.norm_q32(p(c.x), K, 0, 0, p(c.w), rows, K, 1e-6, 0, 0, 0, 0, 0, p(c.qa), p(c.qb), p(c.qm))
    units = [t.cpu().numpy() for t in (c.qa, c.qb, c.qm)]
    base = torch.empty(rows, N, device="cuda")
    qkv.w4_units(rows, N, K, 32, p(c.o[1]), p(c.o[2]), 0, p(c.qa), p(c.qb), p(c.qm), p(base), N)
    c.run(qkv)
    q, s, _ = unpack_units(units[0].reshape(rows, K // 32, 16), units[1].reshape(rows, K // 32, 16), units[2].view(np.uint16).reshape(rows, K // 32, 4))
    xv = (q.astype(np.float64) * s.astype(np.float64)[..., None]).reshape(rows, K)
    y, bound = lora_ref(c.av, c.bv, None, c.scales.cpu().numpy(), c.ids.cpu().numpy(), xv, base.double().cpu().numpy(), 1)
    assert (np.abs(c.y.double().cpu().numpy() - y) <= bound).all()
    n = c.norm.double().cpu().numpy()
    logits, ids, wt = route_ref(n, c.rv, None, 1, 1.0, TOP)
    assert np.array_equal(c.chosen.cpu().numpy(), ids)
    assert (np.abs(c.wt.cpu().numpy() - wt) <= 2.0 ** -20 * wt).all()
    mags = [np.abs(c.up[0]), np.abs(c.down[0])]
    y, bound = moe_ref(c.up[0], c.down[0], mags, n, "fp32", ids, c.wt.cpu().numpy(), "fp32")
    assert (np.abs(c.out.double().cpu().numpy() - y) <= bound).all()


def test_graph(qkv, torch_gpu):
    """Replays between other work are the eager calls, to the bit."""
    torch, c = torch_gpu, Layer(torch_gpu, 9, 1)
    c.run(qkv)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(qkv, torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        c.x.mul_(-1.25).add_(0.1)
        c.ids.copy_((c.ids + 2) % (NA + 1) - 1)
        g.replay()
        got = c.results()
        torch.cuda.synchronize()
        c.run(qkv)
        for a, b in zip(got, c.results()):
            assert torch.equal(a, b)


def test_two_at_once(qkv, torch_gpu):
    """Two layers on streams of their own, each with its workspace."""
    torch = torch_gpu
    cs = [Layer(torch, 6, 3), Layer(torch, 33, 4)]
    want = []
    for c in cs:
        c.run(qkv)
        want.append(c.results())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(10):
        for c, s in zip(cs, streams):
            c.run(qkv, s.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(cs, want):
        for a, b in zip(c.results(), w):
            assert torch.equal(a, b)
