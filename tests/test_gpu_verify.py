"""Verification of drafted tokens (mk_verify_drafts) against a plain restatement in 64 bits: the same counts and tokens, and
probabilities to a float32 rounding."""
import numpy as np
import pytest

from stepcase import CODE, dtype_of, ptr, verify_ref

pytestmark = pytest.mark.gpu


def make(rng, b, n, v, q, spread=3.0):
    logits = rng.standard_normal((b, n + 1, v)) * spread
    temp = rng.uniform(0.5, 1.4, b).astype(np.float32)
    dl = (logits[:, :n] + rng.standard_normal((b, n, v))) / temp[:, None, None]
    dp = np.exp(dl - dl.max(-1, keepdims=True)) if n else np.zeros((b, n, v))
    if n:
        dp /= dp.sum(-1, keepdims=True)
    drafts = np.zeros((b, n), np.int32)
    for s in range(b):
        for i in range(n):
            drafts[s, i] = rng.choice(v, p=dp[s, i]) if q else int(dl[s, i].argmax())
    u = (rng.integers(0, 1 << 24, (b, n + 1)) / float(1 << 24)).astype(np.float32)
    return logits, temp, dp.astype(np.float32) if q else None, drafts, u


def run(torch, qkv, logits, temp, dp, drafts, u, dt="fp32", probs=False, counts=None, pad=0, off=0, with_p=True, stream=None):
    b, rows, v = logits.shape
    n = rows - 1
    t = torch.from_numpy(np.ascontiguousarray(logits, np.float32)).to(dtype_of(torch, dt))
    buf = torch.full((b * rows * (v + pad) + off,), float("nan"), dtype=t.dtype)
    buf[off:].view(b, rows, v + pad)[..., :v] = t
    target = buf.cuda()
    dev = [None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in
           (None if temp is None else temp.astype(np.float32), dp, drafts.astype(np.int32), None if counts is None else np.asarray(counts, np.int32),
            u.astype(np.float32))]
    acc = torch.full((b + 1,), -7, dtype=torch.int32, device="cuda")
    tok = torch.full((b + 1, n + 1), -7, dtype=torch.int32, device="cuda")
    p = torch.full((b + 1, n), -7.0, device="cuda") if with_p else None
    need = qkv.verify_ws(b, n, v)
    ws = torch.full((need,), 0xAA, dtype=torch.uint8, device="cuda")
    s = stream or torch.cuda.current_stream()
    qkv.verify_drafts(b, n, v, target.data_ptr() + off * target.element_size(), v + pad, CODE[dt], int(probs), ptr(dev[0]), ptr(dev[1]), ptr(dev[2]),
                      ptr(dev[3]), dev[4].data_ptr(), acc.data_ptr(), tok.data_ptr(), ptr(p), ws.data_ptr(), need, s.cuda_stream)
    torch.cuda.synchronize()
    assert acc[b] == -7 and (tok[b] == -7).all()
    want = verify_ref(t.double().numpy(), temp, probs, dp, drafts, counts, u)
    got = acc[:b].cpu().numpy(), tok[:b].cpu().numpy(), p[:b].cpu().numpy() if with_p else None
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    if with_p:
        assert (np.abs(got[2].astype(np.float64) - want[2]) <= want[2] * 2.0 ** -24 * (1 + 1e-6) + 1e-45).all()
    return got


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("v", [1, 2, 5, 100, 4095, 4096, 4097, 20000])
@pytest.mark.parametrize("q", [False, True])
def test_vocabularies(qkv, torch_gpu, v, dt, q):
    rng = np.random.default_rng(v + len(dt) + q)
    run(torch_gpu, qkv, *make(rng, 5, 3, v, q), dt=dt)


@pytest.mark.parametrize("n", [0, 1, 2, 7, 8, 33, 64])
@pytest.mark.parametrize("q", [False, True])
def test_drafts(qkv, torch_gpu, n, q):
    rng = np.random.default_rng(n + 100 * q)
    a = make(rng, 6, n, 300, q, spread=6.0)
    run(torch_gpu, qkv, *a)
    run(torch_gpu, qkv, *a, with_p=False)
    run(torch_gpu, qkv, *a, counts=rng.integers(-1, n + 3, 6))


def test_all_accepted_64(qkv, torch_gpu):
    """Sixty-four drafts that the target is sure of: every lane's vote counts."""
    rng = np.random.default_rng(3)
    logits, temp, _, drafts, u = make(rng, 2, 64, 50, False)
    for s in range(2):
        logits[s, np.arange(64), drafts[s]] += 60
    got = run(torch_gpu, qkv, logits, temp, None, drafts, u)
    assert (got[0] == 64).all()


@pytest.mark.parametrize("q", [False, True])
def test_large_vocabulary(qkv, torch_gpu, q):
    rng = np.random.default_rng(17 + q)
    run(torch_gpu, qkv, *make(rng, 3, 2, 150001, q), dt="bf16" if q else "fp32")


@pytest.mark.parametrize("q", [False, True])
def test_largest_vocabulary_and_strides(qkv, torch_gpu, q):
    """2^24 entries a row (64 slices a lane), then rows 2^25 elements apart, 8.6 GB of them."""
    rng = np.random.default_rng(23 + q)
    run(torch_gpu, qkv, *make(rng, 1, 1, 1 << 24, q, spread=4.0), dt="bf16")
    torch, b, n, v, stride = torch_gpu, 2, 31, 5000, 1 << 25
    logits, temp, dp, drafts, u = make(rng, b, n, v, q)
    logits[:, np.arange(n), drafts[0]] += 4
    t = torch.from_numpy(logits.astype(np.float32)).cuda()
    wide = torch.empty(b * (n + 1) * stride, device="cuda")
    wide.view(b, n + 1, stride)[..., :v] = t
    td, qd, dd, ud = (None if z is None else torch.from_numpy(np.ascontiguousarray(z)).cuda() for z in (temp, dp, drafts, u))
    acc, tok = torch.zeros(b, dtype=torch.int32, device="cuda"), torch.zeros(b, n + 1, dtype=torch.int32, device="cuda")
    ws = torch.empty(qkv.verify_ws(b, n, v), dtype=torch.uint8, device="cuda")
    qkv.verify_drafts(b, n, v, wide.data_ptr(), stride, 0, 0, ptr(td), ptr(qd), dd.data_ptr(), 0, ud.data_ptr(), acc.data_ptr(), tok.data_ptr(), 0,
                      ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    want = verify_ref(t.double().cpu().numpy(), temp, False, dp, drafts, None, u)
    assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])


def test_flat_distribution(qkv, torch_gpu):
    """Equal logits: the token is the entry that the random number points at, in every slice."""
    v, b = 30011, 40
    rng = np.random.default_rng(5)
    u = (rng.integers(0, 1 << 24, (b, 1)) / float(1 << 24)).astype(np.float32)
    u[0], u[1] = 0, np.float32(1 - 2.0 ** -24)
    got = run(torch_gpu, qkv, np.full((b, 1, v), 1.5), None, None, np.zeros((b, 0), np.int32), u)
    assert got[1][0, 0] == 0 and got[1][1, 0] == v - 1


@pytest.mark.parametrize("q", [False, True])
def test_probabilities(qkv, torch_gpu, q):
    rng = np.random.default_rng(9 + q)
    logits, temp, dp, drafts, u = make(rng, 6, 4, 9000, q)
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    run(torch_gpu, qkv, p, None, dp, drafts, u, probs=True)
    p[:, :, ::3] = 0
    p[1, 2] = 0            # a row without weight
    p[2, 1, 17] = np.nan
    p[3, 0, :] *= 1e-30    # not normalised
    run(torch_gpu, qkv, p, None, dp, drafts, u, probs=True)


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
def test_greedy_ties(qkv, torch_gpu, dt):
    """Temperature 0: the lowest index of equal logits, across slices; beside sequences that sample."""
    rng = np.random.default_rng(2)
    logits, temp, dp, drafts, u = make(rng, 6, 3, 10000, False)
    logits = np.round(logits)
    temp[::2] = 0
    for s in range(6):
        for i in range(3):
            drafts[s, i] = int(logits[s, i].argmax()) + (s == 4 and i == 1)
    run(torch_gpu, qkv, logits, temp, None, drafts, u, dt=dt)
    q = np.full((6, 3, 10000), 1e-4, np.float32)
    run(torch_gpu, qkv, logits, temp, q, drafts, u, dt=dt)


@pytest.mark.parametrize("q", [False, True])
def test_masked_and_wild_rows(qkv, torch_gpu, q):
    rng = np.random.default_rng(23 + q)
    b, n, v = 8, 2, 9000
    logits, temp, dp, drafts, u = make(rng, b, n, v, q)
    logits[:, :, 4096:8192] = -np.inf                 # a slice with nothing in it
    logits[1, 0] = -np.inf                            # a row with nothing in it
    logits[2, 2] = -np.inf
    logits[2, 0, drafts[2, 0]] = logits[2, 1, drafts[2, 1]] = 80  # (reached)
    logits[3, 0, 100] = np.nan
    logits[4, 1, 8999] = np.inf
    logits[4, 0, drafts[4, 0]] = 80
    logits[5, 0] = -np.inf
    logits[5, 0, drafts[5, 0]] = 1.0                  # the draft is all there is
    logits[6, 0] = np.finfo(np.float32).min           # masked by the type's lowest value: all alike
    drafts[7, 0] = v if not q else -1                 # outside the vocabulary
    u[5, 0] = 0.5
    run(torch_gpu, qkv, logits, temp, dp, drafts, u)
    temp[:] = 0
    run(torch_gpu, qkv, logits, temp, dp, drafts, u)


def test_residual_of_equal_distributions(qkv, torch_gpu):
    """Probabilities equal to the draft model's leave nothing over: a refused draft's successor comes from p."""
    v = 5000
    p = np.zeros((2, 2, v))
    p[:, :, 10] = p[:, :, 4500] = 0.5
    q = p[:, :1].astype(np.float32).copy()
    drafts = np.full((2, 1), 7, np.int32)  # (a draft that neither gives)
    u = np.array([[0.5, 0.25], [0.5, 0.75]], np.float32)
    got = run(torch_gpu, qkv, p, None, q, drafts, u, probs=True)
    assert got[1][:, 0].tolist() == [10, 4500]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_strides_and_alignment(qkv, torch_gpu, dt):
    rng = np.random.default_rng(31)
    run(torch_gpu, qkv, *make(rng, 3, 2, 5003, True), dt=dt, pad=7, off=3)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_temperatures(qkv, torch_gpu, dt):
    """Greedy at zero, below it and for a NaN; the smallest and very large ones; all in one batch."""
    rng = np.random.default_rng(41)
    logits, _, _, drafts, u = make(rng, 8, 3, 5000, False)
    temp = np.array([0.0, -1.0, np.nan, 1e-30, 1e-3, 0.05, 50.0, 1e30], np.float32)
    run(torch_gpu, qkv, logits, temp, None, drafts, u, dt=dt)


def test_weights_below_the_smallest(qkv, torch_gpu):
    """A refused draft whose slice holds entries of e^-748 beside it: each is nothing in 64 bits, their sum would not be."""
    logits = np.full((1, 2, 8192), -np.inf)
    logits[0, 0, :4096], logits[0, 0, 5], logits[0, 0, 5000] = -374.0, 0.0, 374.0
    logits[0, 1, 7] = 1.0
    got = run(torch_gpu, qkv, logits, None, None, np.array([[5]], np.int32), np.array([[0.5, 0.0]], np.float32))
    assert got[1].tolist() == [[5000, -1]]


def test_random_numbers_outside(qkv, torch_gpu):
    """u[n] of 1 or more: the last entry with a weight; nothing is read or written outside."""
    v = 9000
    logits = np.zeros((3, 1, v))
    logits[1, 0, 8000:] = -np.inf
    u = np.array([[1.0], [1.5], [-0.5]], np.float32)
    torch = torch_gpu
    t = torch.from_numpy(logits).float().cuda()
    ud = torch.from_numpy(u).cuda()
    acc, tok = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, 1, dtype=torch.int32, device="cuda")
    ws = torch.empty(qkv.verify_ws(3, 0, v), dtype=torch.uint8, device="cuda")
    qkv.verify_drafts(3, 0, v, t.data_ptr(), v, 0, 0, 0, 0, 0, 0, ud.data_ptr(), acc.data_ptr(), tok.data_ptr(), 0, ws.data_ptr(), ws.numel(),
                      torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert tok[:2, 0].tolist() == [v - 1, 7999] and 0 <= int(tok[2, 0]) < v


def test_workspace_refusals(qkv, torch_gpu):
    torch = torch_gpu
    t = torch.zeros(4096, device="cuda")
    p = t.data_ptr()
    need = qkv.verify_ws(1, 1, 100)
    for ws, size in ((p, need - 1), (0, need), (p + 8, need)):
        with pytest.raises(qkv.KVError):
            qkv.verify_drafts(1, 1, 100, p, 100, 0, 0, 0, 0, p, 0, p, p, p, 0, ws, size)
    with pytest.raises(qkv.KVError, match="ws is not device memory"):
        h = torch.zeros(1024)
        qkv.verify_drafts(1, 1, 100, p, 100, 0, 0, 0, 0, p, 0, p, p, p, 0, (h.data_ptr() + 15) // 16 * 16, need)
    qkv.verify_drafts(0, 1, 100, p, 100, 0, 0, 0, 0, p, 0, p, p, p, 0, 0, 0)
    torch.cuda.synchronize()
