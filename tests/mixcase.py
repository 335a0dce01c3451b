"""Plain restatements in 64 bits (numpy) of the adapters of many requests, the router and the mixture of experts, for their tests, each
with a bound on how far the library's result may be off."""
import numpy as np

from stepcase import EPS_HALF

STEP = 2.0 ** -23  # a whole step of fp32: the matrix instructions' additions may cut


def bits16(v, name):
    """float values -> (their 16-bit pattern uint16, the values it stands for)."""
    if name == "fp16":
        h = v.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float64)
    u = v.astype(np.float32).view(np.uint32)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return r, (r.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def typed(v, name):
    """float values -> (array to hand over, the values it stands for)."""
    if name == "fp32":
        f = v.astype(np.float32)
        return f, f.astype(np.float64)
    return bits16(v, name)


def to_gpu(torch, v, name):
    """typed()'s array on the GPU."""
    t = torch.from_numpy(np.ascontiguousarray(v if name == "fp32" else v.view(np.int16))).cuda()
    return t if name == "fp32" else t.view({"fp16": torch.float16, "bf16": torch.bfloat16}[name])


# ------------------------------------------------------------------------------------------------ adapters
def lora_ref(a, b, ranks, scales, ids, x, base, chunks):
    """a [na][r][k], b [na][n][r], x [rows][k] (float64) -> y and its bound.  A wave adds an eighth of a chunk's steps of 32 values, up to 5
    products of parts each and 33 additions in each; then 8 waves and the chunks add up; what is left out of the products is below 2^-23 of them, and of the largest value of
    x in a step (of u in 64 ranks) 2^-39 where those are made fp16."""
    rows, k = x.shape
    n, r = b.shape[1:]
    y, bound = np.zeros((rows, n)), np.zeros((rows, n))
    down = (-(-k // 32 // 8 // chunks) + 1) * 5 * 33 + 8 + chunks + 2
    up = -(-r // 32) * 5 * 33 + 4
    for m in range(rows):
        i = int(ids[m])
        if 0 <= i < a.shape[0]:
            q = r if ranks is None else int(min(max(ranks[i], 0), r))
            s = 1.0 if scales is None else float(scales[i])
            A, B = a[i, :q], b[i, :, :q]
            xs = np.abs(np.pad(x[m], (0, -k % 32))).reshape(-1, 32).max(1).repeat(32)[:k]
            u, du = A @ x[m], np.abs(A) @ (down * STEP * np.abs(x[m]) + 2.0 ** -39 * xs)
            y[m] = s * (B @ u)
            bound[m] = abs(s) * (np.abs(B) @ (du + up * STEP * (np.abs(u) + du) + 2.0 ** -39 * np.abs(u).max(initial=0)))
    if base is not None:
        y = y + base
    return y, bound + STEP * np.abs(y) + 1e-37


# ------------------------------------------------------------------------------------------------ router
def route_ref(x, w, bias, form, scale, top):
    """x [rows][dim], w [E][dim] (float64, sums exact or nearly) -> logits (float32), ids, weights (float64)."""
    with np.errstate(all="ignore"):
        logits = (x @ w.T).astype(np.float32)
        l = logits.astype(np.float64)
        s = 1.0 / (1.0 + np.exp(-l))
        key = l if bias is None else s + bias.astype(np.float64)
        key = np.where(np.isnan(key), -np.inf, key)
        ids = np.empty((x.shape[0], top), np.int64)
        for m in range(x.shape[0]):
            nan = np.isnan(l[m])  # behind everything, -infinity too
            ids[m] = np.lexsort((np.arange(key.shape[1]), -key[m], nan))[:top]
        got = np.take_along_axis(l, ids, 1)
        if form == 0:
            wt = np.exp(got - l.max(1, keepdims=True)) / np.exp(l - l.max(1, keepdims=True)).sum(1, keepdims=True)
        elif form == 1:
            wt = np.exp(got - got.max(1, keepdims=True))
            wt = wt / wt.sum(1, keepdims=True)
        else:
            wt = np.take_along_axis(s, ids, 1)
            if form == 3:
                wt = wt / wt.sum(1, keepdims=True)
        return logits, ids, wt * scale


# ------------------------------------------------------------------------------------------------ experts
def w4_values(c, scales, mins, group):
    """codes 0..15 [..][n][k], scales and mins fp16 [..][n][gs] -> W (float64)."""
    of = np.arange(c.shape[-1]) // group
    w = (c.astype(np.float64) - 8) * scales.astype(np.float64)[..., of]
    return w if mins is None else w + mins.astype(np.float64)[..., of]


def _rounded(v, bits, block=32):
    """How far an integer of v's block is off: half of the block's power of two times 2^-bits."""
    k = v.shape[1]
    b = np.abs(np.pad(v, ((0, 0), (0, -k % block)))).reshape(v.shape[0], -1, block).max(-1)
    with np.errstate(divide="ignore"):
        top = np.where(b > 0, 2.0 ** np.floor(np.log2(np.maximum(b, 1e-300))), 0)
    return np.repeat(np.maximum(top, 2.0 ** -101), block, 1)[:, :k] * 2.0 ** -(bits + 1)


def moe_ref(up, down, mags, x, xform, ids, weights, yname, group=32):
    """up [E][2 inner][dim], down [E][dim][inner] (float64), mags the sums of their terms' magnitudes (|scale (c - 8)| + |min|, of both),
    x [rows][dim] -> y and its bound.  Rounding: x and h to 13 bits below the power of two of their block of `group` values, which
    have one exponent (fp32: 21; h: 21 for units too), every block's term to three steps, its addition and those of lanes and waves."""
    rows, dim = x.shape
    inner = down.shape[2]
    xb, hb = {"units": (60, 21), "fp32": (21, 21)}.get(xform, (13, 13))
    ops = lambda k: (k // 32 + 24 + 4) * STEP
    dxr = _rounded(x, xb, group)
    y, bound = np.zeros((rows, dim)), np.zeros((rows, dim))
    for m in range(rows):
        for j, e in enumerate(ids[m]):
            if not 0 <= e < up.shape[0]:
                continue
            gu = up[e] @ x[m]
            dgu = mags[0][e] @ (dxr[m] + ops(dim) * np.abs(x[m]))
            g, u, dg, du = gu[:inner], gu[inner:], dgu[:inner], dgu[inner:]
            with np.errstate(over="ignore"):
                s = g / (1 + np.exp(-g))
            h = s * u
            ds = 1.1 * dg + 8 * STEP * np.abs(s)  # (the slope of silu is below 1.1; expf, a sum, a quotient)
            dh = ds * (np.abs(u) + du) + np.abs(s) * du + STEP * np.abs(h)
            dh = dh + _rounded(((np.abs(h) + dh) * 1.0)[None], hb, group)[0]
            o = down[e] @ h
            do = mags[1][e] @ (dh + ops(inner) * (np.abs(h) + dh))
            w = float(weights[m, j])
            y[m] += w * o
            bound[m] += abs(w) * (do + 4 * STEP * (np.abs(o) + do))
    half = 0 if yname == "fp32" else EPS_HALF[yname]
    return y, bound + 16 * STEP * (np.abs(y) + bound) + half * (np.abs(y) + bound) + 1e-37
