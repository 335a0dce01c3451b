"""The step operators together as a decoder runs them around the KV store: a verify step of one layer from the residual
stream to the accepted drafts (norm -> 4-bit q/k/v -> append and attention from raw projections -> 4-bit o_proj on the attention's own
units -> norm -> 4-bit head -> verification -> rewind), each stage against its restatement on the GPU's own inputs; the same step
captured into a graph and replayed; on other streams; two calls at once."""
import numpy as np
import pytest

from stepcase import norm_ref, norm_units_ref, pack_codes, unpack_units, verify_ref, w4_bound, w4_ref

pytestmark = pytest.mark.gpu

H, VOCAB, NQ, NKVD = 640, 1003, 24 * 512, 4 * 256


class W4:
    def __init__(self, torch, rng, n, k, group=32, mins=False, size=1.0):
        self.n, self.k, self.group = n, k, group
        self.c = rng.integers(0, 16, (n, k))
        self.s = (rng.uniform(0.5, 1.5, (n, -(-k // group))) * size / (4.6 * np.sqrt(k))).astype(np.float16)
        self.m = (rng.standard_normal(self.s.shape) * 0.1 * size / np.sqrt(k)).astype(np.float16) if mins else None
        self.cd, self.sd = torch.from_numpy(pack_codes(self.c)).cuda(), torch.from_numpy(self.s).cuda()
        self.md = torch.from_numpy(self.m).cuda() if mins else None

    def __call__(self, qkv, u, y, rows, stream):
        qkv.w4_units(rows, self.n, self.k, self.group, self.cd.data_ptr(), self.sd.data_ptr(), self.md.data_ptr() if self.m is not None else 0,
                     u[0].data_ptr(), u[1].data_ptr(), u[2].data_ptr(), y.data_ptr(), self.n, stream)

    def check(self, u, y):
        q, sc, _ = unpack_units(*(t.cpu().numpy().reshape(-1, t.shape[-2], t.shape[-1]) for t in u[:2]),
                                u[2].cpu().numpy().view(np.uint16).reshape(-1, u[2].shape[-2], 4))
        x = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(q.shape[0], -1)
        ref, mag = w4_ref(self.c, self.s, self.m, self.group, x)
        assert (np.abs(y.cpu().numpy().reshape(ref.shape) - ref) <= w4_bound(self.k, mag, False)).all()


def units(torch, rows, k):
    return (torch.zeros(rows, k // 32, 16, dtype=torch.int8, device="cuda"), torch.zeros(rows, k // 32, 16, dtype=torch.int8, device="cuda"),
            torch.zeros(rows, k // 32, 4, dtype=torch.int16, device="cuda"))


class Step:
    """Buffers and calls of one verify step of T tokens over a store of one layer."""

    def __init__(self, torch, qkv, T, L, seed=0):
        rng = np.random.default_rng(seed)
        self.torch, self.qkv, self.T = torch, qkv, T
        self.st = qkv.KVStore("K*=5r,V*=6", win=512, n_layers=1, ctx=L + 64)
        K, V = (torch.from_numpy(rng.standard_normal((L, 1, 4, 256)).astype(np.float32)).cuda() for _ in range(2))
        self.st.append(0, 0, 1, 0, L, K.data_ptr(), V.data_ptr(), 0)
        self.wq, self.wk, self.wv = W4(torch, rng, NQ, H), W4(torch, rng, NKVD, H, 64, True), W4(torch, rng, NKVD, H, 128)
        self.wo, self.head = W4(torch, rng, H, 6144, 32, True), W4(torch, rng, VOCAB, H, 64, size=3.0)

        def f(*shape):
            return torch.zeros(*shape, device="cuda")
        self.x, self.res = f(T, H), f(T, H)
        self.w1, self.w2 = (torch.from_numpy((1 + 0.1 * rng.standard_normal(H)).astype(np.float32)).cuda() for _ in range(2))
        self.nq, self.nk = (torch.from_numpy((1 + 0.1 * rng.standard_normal((1, 256))).astype(np.float32)).cuda() for _ in range(2))
        self.u1, self.ua, self.u2 = units(torch, T, H), units(torch, T, 6144), units(torch, T, H)
        self.qg, self.k, self.v, self.att, self.o, self.logits = f(T, NQ), f(T, NKVD), f(T, NKVD), f(T, 6144), f(T, H), f(T, VOCAB)
        self.drafts, self.u = torch.zeros(1, T - 1, dtype=torch.int32, device="cuda"), f(1, T)
        self.acc, self.tok = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, T, dtype=torch.int32, device="cuda")
        self.p = f(1, T - 1)
        self.ws = torch.zeros(qkv.verify_ws(1, T - 1, VOCAB), dtype=torch.uint8, device="cuda")
        self.h1, self.h2 = f(T, H), f(T, H)
        torch.cuda.synchronize()

    def set(self, seed):
        rng, t = np.random.default_rng(seed), self.torch
        for b, v in ((self.x, rng.standard_normal((self.T, H))), (self.res, 2 * rng.standard_normal((self.T, H))), (self.u, rng.random((1, self.T)))):
            b.copy_(t.from_numpy(v.astype(np.float32)))
        self.drafts.copy_(t.from_numpy(rng.integers(0, VOCAB, (1, self.T - 1)).astype(np.int32)))

    def run(self, pos, stream):
        q, T = self.qkv, self.T
        # the residual stream of this test stays as it is (h1, h2 beside it), so that a pass can be repeated
        q.norm_q32(self.x.data_ptr(), H, self.res.data_ptr(), H, self.w1.data_ptr(), T, H, 1e-6, 0, self.h1.data_ptr(), H, 0, 0,
                   *(t.data_ptr() for t in self.u1), stream)
        self.wq(q, self.u1, self.qg, T, stream)
        self.wk(q, self.u1, self.k, T, stream)
        self.wv(q, self.u1, self.v, T, stream)
        self.st.append_prep(0, 0, 1, pos, T, self.k.data_ptr(), self.v.data_ptr(), self.nk.data_ptr(), stream)
        self.st.attend_prep(0, 1, [0], [pos + T], T, self.qg.data_ptr(), self.nq.data_ptr(), self.att.data_ptr(), *(t.data_ptr() for t in self.ua), stream)
        self.wo(q, self.ua, self.o, T, stream)
        q.norm_q32(self.o.data_ptr(), H, self.h1.data_ptr(), H, self.w2.data_ptr(), T, H, 1e-6, 0, self.h2.data_ptr(), H, 0, 0,
                   *(t.data_ptr() for t in self.u2), stream)
        self.head(q, self.u2, self.logits, T, stream)
        q.verify_drafts(1, T - 1, VOCAB, self.logits.data_ptr(), VOCAB, 0, 0, 0, 0, self.drafts.data_ptr(), 0, self.u.data_ptr(), self.acc.data_ptr(),
                        self.tok.data_ptr(), self.p.data_ptr(), self.ws.data_ptr(), self.ws.numel(), stream)

    def results(self):
        self.torch.cuda.synchronize()
        return [t.cpu().numpy().copy() for t in (self.h1, *self.u1, self.qg, self.k, self.v, self.att, *self.ua, self.o, self.h2, *self.u2, self.logits,
                                                 self.acc, self.tok, self.p)]

    def check(self):
        self.torch.cuda.synchronize()
        for x, r, w, h, u in ((self.x, self.res, self.w1, self.h1, self.u1), (self.o, self.h1, self.w2, self.h2, self.u2)):
            want = x.cpu().numpy() + r.cpu().numpy()
            assert np.array_equal(h.cpu().numpy(), want)
            _, rs = norm_ref(want, w.cpu().numpy(), 1e-6)
            eq, es = norm_units_ref(want, w.cpu().numpy(), rs)
            q, sc, _ = unpack_units(u[0].cpu().numpy(), u[1].cpu().numpy(), u[2].cpu().numpy().view(np.uint16))
            assert np.array_equal(q, eq) and np.array_equal(sc.view(np.uint16), es.view(np.uint16))
        for w, u, y in ((self.wq, self.u1, self.qg), (self.wk, self.u1, self.k), (self.wv, self.u1, self.v), (self.wo, self.ua, self.o),
                        (self.head, self.u2, self.logits)):
            w.check(u, y)
        # the attention's units are its rows to half a code
        q, sc, _ = unpack_units(self.ua[0].cpu().numpy(), self.ua[1].cpu().numpy(), self.ua[2].cpu().numpy().view(np.uint16))
        val = (q.astype(np.float64) * sc.astype(np.float64)[..., None]).reshape(self.T, 6144)
        step = np.abs(val).reshape(self.T, 192, 32).max(-1).repeat(32, -1) / 127
        assert (np.abs(val - self.att.cpu().numpy()) <= step * (0.5 + 127 * 2.0 ** -11 + 1e-2) + 1e-7).all()
        acc, tok, p = verify_ref(self.logits.cpu().numpy().astype(np.float64)[None], None, False, None, self.drafts.cpu().numpy(), None, self.u.cpu().numpy())
        assert np.array_equal(self.acc.cpu().numpy(), acc) and np.array_equal(self.tok.cpu().numpy(), tok)
        assert (np.abs(self.p.cpu().numpy() - p) <= p * 2.0 ** -24 * (1 + 1e-6) + 1e-45).all()


@pytest.mark.parametrize("T", [2, 8])
def test_verify_step(qkv, torch_gpu, T):
    torch, L = torch_gpu, 1500
    s = Step(torch, qkv, T, L, seed=T)
    pos = L
    for i in range(3):
        s.set(10 * T + i)
        if i:  # a step with the drafts that the one before found likely
            s.drafts.copy_(s.logits[:-1].argmax(-1)[None].int())
            s.u.mul_(0.02)
        s.run(pos, torch.cuda.current_stream().cuda_stream)
        s.check()
        kept = pos + int(s.acc[0]) + 1
        s.st.rewind(0, kept)
        pos = kept
    s.st.close()


def test_verify_step_in_a_graph(qkv, torch_gpu):
    """Captured once, replayed on other inputs with eager work between the replays: the eager results, bit for bit."""
    torch, T, L = torch_gpu, 8, 1200
    s = Step(torch, qkv, T, L, seed=3)
    side = torch.cuda.Stream()
    s.set(1)
    s.run(L, torch.cuda.current_stream().cuda_stream)  # (the store's workspace and table)
    eager = {}
    for seed in range(2, 5):
        s.set(seed)
        s.run(L, torch.cuda.current_stream().cuda_stream)
        eager[seed] = s.results()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            s.run(L, side.cuda_stream)
    for seed in (4, 2, 3, 4):
        s.set(seed)
        torch.cuda.synchronize()
        graph.replay()
        for i, (a, b) in enumerate(zip(s.results(), eager[seed])):
            assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f"), (seed, i)
        s.set(1)
        s.run(L, torch.cuda.current_stream().cuda_stream)  # eager work between the replays
        torch.cuda.synchronize()
    s.st.close()


@pytest.mark.parametrize("rows", [1, 3, 8, 40, 64])
@pytest.mark.parametrize("x", ["units", "fp32"])
def test_products_in_a_graph(qkv, torch_gpu, rows, x):
    torch = torch_gpu
    rng = np.random.default_rng(rows)
    w = W4(torch, rng, 1000, 1024, 32, True)
    u = units(torch, rows, 1024)
    xs = torch.zeros(rows, 1024, device="cuda")
    y = torch.zeros(rows, 1000, device="cuda")

    def run(stream):
        if x == "units":
            w(qkv, u, y, rows, stream)
        else:
            qkv.w4_rows(rows, 1000, 1024, 32, w.cd.data_ptr(), w.sd.data_ptr(), w.md.data_ptr(), xs.data_ptr(), 1024, 0, y.data_ptr(), 1000, stream)
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            run(side.cuda_stream)  # (captured without a call before it)
    for seed in range(3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        xs.copy_(torch.randn(rows, 1024, device="cuda", generator=gen))
        qkv.norm_q32(xs.data_ptr(), 1024, 0, 0, torch.ones(1024, device="cuda").data_ptr(), rows, 1024, 0.0, 0, 0, 0, 0, 0, *(t.data_ptr() for t in u),
                     torch.cuda.current_stream().cuda_stream)
        run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want = y.clone()
        y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool(y.abs().sum() > 0)


def test_two_streams_at_once(qkv, torch_gpu):
    """Calls that overlap on two streams, each with its own outputs and workspace, give what they give alone."""
    torch = torch_gpu
    rng = np.random.default_rng(5)
    b, n, v = 16, 3, 60000
    logits = torch.from_numpy((3 * rng.standard_normal((b, n + 1, v))).astype(np.float32)).cuda()
    drafts = logits[:, :n].argmax(-1).int().contiguous()
    u = torch.from_numpy(rng.random((2, b, n + 1)).astype(np.float32)).cuda()
    w = W4(torch, rng, 20000, 2048)
    us = [units(torch, 8, 2048) for _ in range(2)]
    for k, t in enumerate(us):
        xs = torch.from_numpy(rng.standard_normal((8, 2048)).astype(np.float32)).cuda()
        qkv.norm_q32(xs.data_ptr(), 2048, 0, 0, torch.ones(2048, device="cuda").data_ptr(), 8, 2048, 1e-6, 0, 0, 0, 0, 0, *(z.data_ptr() for z in t), 0)
    torch.cuda.synchronize()

    def outs():
        return dict(acc=torch.zeros(b, dtype=torch.int32, device="cuda"), tok=torch.zeros(b, n + 1, dtype=torch.int32, device="cuda"),
                    p=torch.zeros(b, n, device="cuda"), ws=torch.zeros(qkv.verify_ws(b, n, v), dtype=torch.uint8, device="cuda"),
                    y=torch.zeros(8, 20000, device="cuda"))

    def run(k, o, stream):
        w(qkv, us[k], o["y"], 8, stream)
        qkv.verify_drafts(b, n, v, logits.data_ptr(), v, 0, 0, 0, 0, drafts.data_ptr(), 0, u[k].data_ptr(), o["acc"].data_ptr(), o["tok"].data_ptr(),
                          o["p"].data_ptr(), o["ws"].data_ptr(), o["ws"].numel(), stream)
    alone = [outs(), outs()]
    for k in range(2):
        run(k, alone[k], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
    assert not torch.equal(alone[0]["tok"], alone[1]["tok"])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    both = [outs(), outs()]
    torch.cuda.synchronize()
    for _ in range(5):
        for k in range(2):
            run(k, both[k], streams[k].cuda_stream)
    torch.cuda.synchronize()
    for k in range(2):
        for name in ("acc", "tok", "p", "y"):
            assert torch.equal(alone[k][name], both[k][name]), (k, name)


def test_same_bits_every_run(qkv, torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(6)
    for rows, n, k in ((1, 5000, 2048), (8, 3001, 4096), (33, 2000, 4096)):
        w, u = W4(torch, rng, n, k, 64, True), units(torch, rows, k)
        xs = torch.from_numpy(rng.standard_normal((rows, k)).astype(np.float32)).cuda()
        qkv.norm_q32(xs.data_ptr(), k, 0, 0, torch.ones(k, device="cuda").data_ptr(), rows, k, 1e-6, 0, 0, 0, 0, 0, *(z.data_ptr() for z in u), 0)
        torch.cuda.synchronize()
        ys = [torch.zeros(rows, n, device="cuda") for _ in range(6)]
        torch.cuda.synchronize()
        for y in ys:
            w(qkv, u, y, rows, 0)
        torch.cuda.synchronize()
        assert all(torch.equal(y, ys[0]) for y in ys)


def test_an_earlier_error_is_not_this_calls(qkv, torch_gpu):
    """A HIP call of the thread that failed before (here a device that does not exist) does not turn these calls into errors."""
    torch, hip = torch_gpu, qkv.lib()  # (the library's own HIP runtime)
    rng = np.random.default_rng(1)
    w, u = W4(torch, rng, 100, 256, 32), units(torch, 2, 256)
    x, y, one = torch.ones(2, 256, device="cuda"), torch.zeros(2, 100, device="cuda"), torch.ones(256, device="cuda")
    drafts, rnd = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, device="cuda")
    acc, tok = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1, 2), -7, dtype=torch.int32, device="cuda")
    ws = torch.zeros(qkv.verify_ws(1, 1, 100), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    try:
        for call in (lambda: qkv.norm_q32(x.data_ptr(), 256, 0, 0, one.data_ptr(), 2, 256, 1e-6, 0, 0, 0, 0, 0, *(t.data_ptr() for t in u), stream),
                     lambda: w(qkv, u, y, 2, stream),
                     lambda: qkv.w4_rows(2, 100, 256, 32, w.cd.data_ptr(), w.sd.data_ptr(), 0, x.data_ptr(), 256, 0, y.data_ptr(), 100, stream),
                     lambda: qkv.verify_drafts(1, 1, 100, y.data_ptr(), 100, 0, 0, 0, 0, drafts.data_ptr(), 0, rnd.data_ptr(), acc.data_ptr(),
                                               tok.data_ptr(), 0, ws.data_ptr(), ws.numel(), stream)):
            assert hip.hipSetDevice(1 << 20) != 0
            call()
    finally:
        hip.hipGetLastError()
    torch.cuda.synchronize()
    assert int(tok[0, 0]) >= 0 and bool(y.abs().sum() > 0)


def test_kinds_of_streams(qkv, torch_gpu):
    """The null stream, the thread's own (handle 2), a stream of torch's and the current one."""
    torch = torch_gpu
    x, w = torch.randn(3, 128, device="cuda"), torch.ones(128, device="cuda")
    side = torch.cuda.Stream()
    ys = [torch.zeros(3, 128, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    for y, s in zip(ys, (0, 2, side.cuda_stream, torch.cuda.current_stream().cuda_stream)):
        qkv.norm_q32(x.data_ptr(), 128, 0, 0, w.data_ptr(), 3, 128, 1e-6, 0, 0, 0, y.data_ptr(), 128, 0, 0, 0, s)
    torch.cuda.synchronize()
    assert all(torch.equal(y, ys[0]) for y in ys) and bool(ys[0].abs().sum() > 0)
