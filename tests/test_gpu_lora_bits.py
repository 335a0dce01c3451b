"""How many bits of x and of A x the adapters keep (mk_lora_rows, mk_lora_units): results that have to be equal because every step is exact, and the
size of the errors against 64 bits (a worst case would not see a lost part)."""
import numpy as np
import pytest

from stepcase import pack_units
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -23


@pytest.mark.parametrize("xform,terms", [("fp32", 1), ("fp16", 2), ("bf16", 3), ("units", 3)])
@pytest.mark.parametrize("wname", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,rank", [(1, 16), (3, 40), (40, 8), (64, 100), (300, 33), (1030, 20)])
def test_exact(qkv, torch_gpu, xform, terms, wname, rows, rank):
    """Values of all the bits of their type; A takes one of them to each rank (of types of few bits several, one behind the other: up to 24 bits), B hands one on to
    each column.  bf16 adapters: exact.  fp16 adapters: values of up to 22 bits are exact, others (x, then A x) are off by 2^-23, or by 2^-39 of the largest beside them."""
    torch, k, n = torch_gpu, 512, 130
    rng = np.random.default_rng(rows + rank)
    bits = {"fp32": 24, "fp16": 11, "bf16": 8, "units": 7}[xform]
    v = (rng.integers(2 ** (bits - 1), 2 ** bits, (rows, k)) | 1) * rng.choice([-1, 1], (rows, k))
    x = v * 2.0 ** -bits * 2.0 ** rng.integers(-3, 4, (rows, k // 32)).repeat(32, 1)
    if terms == 1:
        x = x * 2.0 ** rng.integers(-4, 1, (rows, k))
    c = Case(torch, rows, n, k, rank, 2, xform, wname, scales=False, base=False, ids=np.arange(rows) % 2, x=x)
    if xform == "units":
        q = v.astype(np.int8).reshape(rows, k // 32, 32)
        sc = (2.0 ** rng.integers(-9, -3, (rows, k // 32))).astype(np.float16)
        c.x = [torch.from_numpy(np.ascontiguousarray(t.view(np.int16) if t.dtype == np.uint16 else t)).cuda() for t in pack_units(q, sc)]
        c.xv = x = (q * sc.astype(np.float64)[..., None]).reshape(rows, k)
    a, u = np.zeros((2, rank, k)), np.empty((rows, rank))
    # (a rank's terms are of one block, all of one power of two: one behind the other they keep their bits)
    for e in range(2):
        for i in range(rank):
            at = (5 * i + 32 * e) % (k - 4) // 8 * 8
            for t in range(terms):
                a[e, i, at + t] = 2.0 ** (-bits * t)
    b = np.zeros((2, n, rank))
    b[:, np.arange(n), np.arange(n) % rank] = 2
    c.a, c.b = torch.from_numpy(a).to(c.a.dtype).cuda(), torch.from_numpy(b).to(c.b.dtype).cuda()
    assert np.array_equal(c.a.double().cpu().numpy(), a)
    for m in range(rows):
        u[m] = a[m % 2] @ c.xv[m]
    assert np.array_equal(u.astype(np.float32), u)
    want = 2 * u[:, np.arange(n) % rank]
    y = c.run(qkv).double().cpu().numpy()
    if wname == "bf16":
        assert np.array_equal(y, want)
        return
    xs = np.abs(c.xv).reshape(rows, -1, 32).max(-1).max(-1)[:, None]  # (bounds the largest of any 32)
    bound = 2 * (2 * STEP * np.abs(u) + 2.0 ** -39 * (xs + np.abs(u).max(1, keepdims=True)))[:, np.arange(n) % rank]
    if xform == "fp32" or terms * bits > 22:
        assert (np.abs(y - want) <= bound).all()
    else:
        assert np.array_equal(y, want)


@pytest.mark.parametrize("xform", ["fp32", "fp16", "bf16", "units"])
@pytest.mark.parametrize("wname", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,rank", [(1, 16), (24, 64), (40, 24), (300, 32), (300, 100), (1030, 64)])
def test_errors(qkv, torch_gpu, xform, wname, rows, rank):
    """Errors as large as a step of fp32 for every instruction of a chain makes them (a sum's size: what its terms' squares add up to), to a factor of two."""
    k, n = 256, 200
    c = Case(torch_gpu, rows, n, k, rank, 3, xform, wname, scales=False, base=False, ids=np.arange(rows) % 3, seed=rank)
    y = c.run(qkv).double().cpu().numpy()
    px, pu = (2 if wname == "fp16" else 3) if xform == "fp32" else 2 if xform == "fp16" and wname == "bf16" else 1, 2 if wname == "fp16" else 3
    down, up = px + 8 + 1, -(-rank // 32) * pu + 2  # (a step a wave, 8 waves; parts of u, the result)
    err = 0.0
    for m in range(rows):
        A, B = c.av[m % 3], c.bv[m % 3]
        u = A @ c.xv[m]
        vu = (A ** 2) @ (c.xv[m] ** 2) * (down * STEP) ** 2
        sd = np.sqrt((B ** 2) @ (vu + (up * STEP) ** 2 * u * u))
        err += (((y[m] - B @ u) / sd) ** 2).mean()
    assert np.sqrt(err / rows) <= 2
