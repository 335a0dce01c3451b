"""How many bits of x and of h the experts keep (mk_moe_rows, mk_moe_units): results that have to be equal because every step is exact, and the
size of the errors against 64 bits, each rounding taken as independent of the others (a worst case would not see a lost plane)."""
import numpy as np
import pytest

from mixcase import bits16
from stepcase import pack_codes, pack_units
from test_gpu_moe import Case

pytestmark = pytest.mark.gpu
FORMS = ["units", "fp32", "fp16", "bf16"]
ULP = 2.0 ** -24  # half a step of fp32, relative


@pytest.mark.parametrize("xform", FORMS)
@pytest.mark.parametrize("group,mins", [(32, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_exact(qkv, torch_gpu, xform, group, mins, rows):
    """Values of all the bits that their type has, beside one of their block that is larger by as much as the header allows (fp32: 22 bits and none
    larger).  The gate is 32 (silu(32) = 32 in fp32: exp(-32) < 2^-24), the up projection selects a value, the down projection an h: every
    product and sum is exact, and so is y = 32 x."""
    torch, dim, inner, used = torch_gpu, 256, 64, 48
    rng = np.random.default_rng(rows + group)
    bits, larger = {"fp32": (22, 0), "fp16": (11, 11), "bf16": (8, 14), "units": (7, 0)}[xform]
    at = 128 + np.arange(used) // 24 * 32 + np.arange(used) % 24
    x = np.zeros((rows, dim))
    x[:, 0] = 32
    x[:, at] = (rng.integers(2 ** (bits - 1), 2 ** bits, (rows, used)) | 1) * 2.0 ** (1 - bits) * rng.choice([-1, 1], (rows, used))
    if larger:
        x[:, [159, 191]] = 2.0 ** larger
    ids = np.arange(rows)[:, None] % 2
    c = Case(torch, rows, dim, inner, 2, 1, group, mins, xform, ids=ids, x=x)
    if xform == "units":
        q = np.where(x == 32, 32, np.rint(x * 64)).astype(np.int8).reshape(rows, dim // 32, 32)
        sc = np.ones((rows, dim // 32), np.float16)
        sc[:, 4:6] = (1 + 2.0 ** -10) / 64  # (18 bits in x and h)
        c.x = [torch.from_numpy(np.ascontiguousarray(t.view(np.int16) if t.dtype == np.uint16 else t)).cuda() for t in pack_units(q, sc)]
        x = (q * sc.astype(np.float64)[..., None]).reshape(rows, dim)
    want = np.empty((rows, dim))
    up, down = np.full((2, 2 * inner, dim), 8, np.uint8), np.full((2, dim, inner), 8, np.uint8)
    for e in range(2):
        take = np.roll(np.arange(used), e)  # column i of inner has value take[i]
        up[e, np.arange(used), 0] = 9
        up[e, inner + np.arange(used), at[take]] = 9
        down[e, np.arange(dim), np.arange(dim) % used] = 9
        want[ids[:, 0] == e] = 32 * x[ids[:, 0] == e][:, at[take]][:, np.arange(dim) % used]
    for w, codes in zip(c.dev, (up, down)):
        w[0] = torch.from_numpy(pack_codes(codes.reshape(-1, codes.shape[2]))).cuda()
        w[1] = torch.ones_like(w[1])
        w[2] = None if w[2] is None else torch.zeros_like(w[2])
    c.chosen[1].fill_(1.0)
    assert np.array_equal(c.run(qkv).double().cpu().numpy(), want)


def _step2(v, block):
    """The variance of rounding to 2^-21 of the power of two of a block's largest."""
    rows, k = v.shape
    b = np.abs(np.pad(v, ((0, 0), (0, -k % block)))).reshape(rows, -1, block).max(-1)
    step = np.where(b > 0, 2.0 ** (np.floor(np.log2(np.maximum(b, 1e-300))) - 21), 0)
    return np.repeat(step * step / 12, block, 1)[:, :k]


def _spread(c):
    """y in 64 bits and the standard deviation of what roundings do to it."""
    adds = lambda k: (k // 32 + 28) * ULP * ULP / 3  # (of a sum's size: what its terms' squares add up to)
    y, var = np.zeros((c.rows, c.dim)), np.zeros((c.rows, c.dim))
    sx = np.zeros_like(c.xv) if c.xform == "units" else _step2(c.xv, c.group)
    for m in range(c.rows):
        for j, e in enumerate(c.ids[m]):
            up, down = c.w[0][e], c.w[1][e]
            x = c.xv[m]
            gu = up @ x
            v = (up ** 2) @ (sx[m] + adds(c.dim) * x * x)
            g, u, vg, vu = gu[:c.inner], gu[c.inner:], v[:c.inner], v[c.inner:]
            s = g / (1 + np.exp(-g))
            h = s * u
            vs = 1.1 ** 2 * vg + 16 * ULP ** 2 * s * s
            vh = u * u * vs + s * s * vu + ULP ** 2 * h * h + _step2(h[None], min(c.group, 64))[0]
            o = down @ h
            vo = (down ** 2) @ (vh + adds(c.inner) * h * h)
            w = float(c.weights[m, j])
            y[m] += w * o
            var[m] += w * w * (vo + 4 * ULP ** 2 * o * o)
    return y, np.sqrt(var)


@pytest.mark.parametrize("xform", FORMS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 24])
@pytest.mark.parametrize("outliers", [False, True])
def test_errors(qkv, torch_gpu, xform, group, rows, outliers):
    """fp32 results: the errors are as large as independent roundings make them, to a factor of two.  16-bit results: as many of them are the one beside
    the nearest value as such errors carry over a border (an error of d crosses one with probability d / step)."""
    rng = np.random.default_rng(group + rows)
    x = rng.standard_normal((rows, 1024))
    if outliers:
        x[:, 17::128] *= 256
    c = Case(torch_gpu, rows, 1024, 512, 4, 2, group, False, xform, x=x, seed=rows)
    y = c.run(qkv).double().cpu().numpy()
    ref, sd = _spread(c)
    if c.yname == "fp32":
        assert np.sqrt(np.mean(((y - ref) / sd) ** 2)) <= 2
        return
    nearest = bits16(ref, c.yname)[1]
    step = 2.0 ** np.floor(np.log2(np.abs(ref))) * (2.0 ** -10 if c.yname == "fp16" else 2.0 ** -7)
    want = np.minimum(sd / step, 1).sum()
    assert (y != nearest).sum() <= 2 * want + 6 * np.sqrt(want) + 3, ((y != nearest).sum(), want, y.size)
