"""Plain restatements in 64 bits (numpy) of the operators of a decode step, for their GPU tests: residual norm and int8 units,
products with 4-bit weights, verification of drafted tokens."""
import numpy as np

EPS_HALF = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
CODE = {"fp32": 0, "fp16": 1, "bf16": 2}


def dtype_of(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def ptr(t):
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------ units
def units_of(v):
    """float rows [rows][k] -> units (a, b int8 [rows][k/32][16], meta uint16 [rows][k/32][4]) of amax / 127 per 32 values."""
    rows, k = v.shape
    b = v.astype(np.float32).reshape(rows, k // 32, 32)
    d = np.abs(b).max(-1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(d > 0, np.rint(b / d), 0).astype(np.int8)
    return pack_units(q, d[..., 0].astype(np.float16))


def pack_units(q, sc):
    """codes int8 [rows][blocks][32] and scales fp16 [rows][blocks] -> a, b, meta."""
    rows, nb = q.shape[:2]
    h = q.reshape(rows, nb // 2, 2, 2, 16)  # pair, block of the pair, half
    meta = np.empty((rows, nb // 2, 2, 4), np.uint16)
    meta[..., 0:2] = sc.reshape(rows, nb // 2, 1, 2).view(np.uint16)
    meta[..., 2:4] = np.swapaxes(h.astype(np.int16).sum(-1, dtype=np.int16), 2, 3).view(np.uint16)
    return (np.ascontiguousarray(h[:, :, 0].reshape(rows, nb, 16)), np.ascontiguousarray(h[:, :, 1].reshape(rows, nb, 16)), meta.reshape(rows, nb, 4))


def unpack_units(a, b, meta):
    """-> codes int8 [rows][blocks][32], scales fp16 [rows][blocks], sums of the codes' halves int16 [rows][blocks][2]."""
    rows, nb = a.shape[:2]
    q = np.stack([a.reshape(rows, nb // 2, 32), b.reshape(rows, nb // 2, 32)], 2).reshape(rows, nb, 32)
    m = meta.reshape(rows, nb // 2, 2, 4)
    assert np.array_equal(m[:, :, 0, :2], m[:, :, 1, :2])
    sc = np.ascontiguousarray(m[:, :, 0, :2]).view(np.float16).reshape(rows, nb)
    sums = np.ascontiguousarray(np.swapaxes(m[..., 2:4], 2, 3)).view(np.int16).reshape(rows, nb, 2)
    return q, sc, sums


# ------------------------------------------------------------------------------------------------ norm
def norm_ref(h, w, eps):
    """h [rows][dim] (the stored sum, as float32), w -> y in 64 bits, and the factor 1 / sqrt(mean + eps) as float32."""
    x = h.astype(np.float64)
    with np.errstate(all="ignore"):
        rs = 1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / x.shape[-1] + np.float64(np.float32(eps)))
        return x * rs * w.astype(np.float64), rs.astype(np.float32)


def norm_units_ref(h, w, rs):
    """Codes and scales of the units, from their definition: float32 products and quotients, each rounded once."""
    rows, dim = h.shape
    with np.errstate(all="ignore"):
        t = (h * w).reshape(rows, dim // 32, 32)
        am = np.abs(t).max(-1, keepdims=True)
        q = np.where(am < np.float32(4e-37), 0, np.rint(t * (np.float32(127) / am)))
        sc = (am[..., 0] * (rs / np.float32(127))).astype(np.float16)
    return np.nan_to_num(q, nan=0.0, posinf=0.0, neginf=0.0).astype(np.int8), sc


# ------------------------------------------------------------------------------------------------ 4-bit weights
def pack_codes(c):
    """codes 0..15 [n][k] -> bytes [n][k/2]: value 8 w + i in the low (i < 4) or high nibble of byte i % 4 of word w."""
    n, k = c.shape
    w = c.reshape(n, k // 8, 2, 4).astype(np.uint8)
    return (w[:, :, 0] | (w[:, :, 1] << 4)).reshape(n, k // 2)


def w4_ref(c, scales, mins, group, x):
    """-> y [rows][n] in 64 bits and the sum of the terms' magnitudes."""
    k = c.shape[1]
    of = np.arange(k) // group
    s = scales.astype(np.float64)[:, of]
    q = c.astype(np.float64) - 8
    W, A = q * s, np.abs(q * s)
    if mins is not None:
        m = mins.astype(np.float64)[:, of]
        W, A = W + m, A + np.abs(m)
    x = x.astype(np.float64)
    return x @ W.T, np.abs(x) @ A.T


def w4_bound(k, mag, plain):
    """How far a row's fp32 result may be off: every block's term is added once (mins: twice) in fp32, half a step each, a wave's
    four blocks at a time, then over lanes and waves; plain rows: 32 values per block (64 for fp32's two parts) summed inside the
    matrix instructions, a whole step each, x itself to a step (fp32: the first part, rounded to 11 bits, leaves at most 2^-11 of the
    value's power of two, in steps of 2^-23; the second has steps of 2^-22 there, and half of one is 2^-23)."""
    ops = k / 32 / 2 + 16 + (2 * 64 + 34 if plain else 0)
    return ops * 2.0 ** -24 * mag + 1e-38


# ------------------------------------------------------------------------------------------------ verification
def verify_ref(target, temp, probs, q, drafts, counts, u):
    """target float64 [b][n + 1][vocab] -> accepted [b], tokens [b][n + 1], p [b][n] (float64)."""
    b, rows, v = target.shape
    n = rows - 1
    acc, tokens, p = np.zeros(b, np.int64), np.full((b, n + 1), -1, np.int64), np.zeros((b, n))
    for s in range(b):
        cnt = n if counts is None else int(min(max(counts[s], 0), n))

        def dist(i):
            x = target[s, i]
            if not (x < np.inf).all():
                return None  # a NaN or +infinity
            if probs:
                w = np.maximum(x, 0)
            else:
                t = 1.0 if temp is None else float(temp[s])
                m = x.max()
                if m == -np.inf:
                    return None
                if t > 0:
                    w = np.exp((x - m) / t)
                    w = w / w.sum()
                else:
                    w = np.zeros(v)
                    w[int(np.argmax(x))] = 1
            return w if w.sum() > 0 else None

        def prob(i, w):
            d = int(drafts[s, i])
            return 0.0 if w is None or not 0 <= d < v else float(w[d])

        a, want, stop = 0, None, False
        for i in range(cnt):
            w = dist(i)
            p[s, i] = prob(i, w)
            if stop:
                continue
            d = int(drafts[s, i])
            qd = 1.0 if q is None or not 0 <= d < v else float(q[s, i, d])
            if float(u[s, i]) * qd < p[s, i]:
                a += 1
                continue
            stop, want = True, w
            if w is not None:
                less = w.copy()
                if q is not None:
                    less = np.maximum(w - q[s, i].astype(np.float64), 0)
                elif 0 <= d < v:
                    less[d] = 0
                want = less if less.sum() > 0 else w
        if not stop:
            want = dist(cnt)
        acc[s] = a
        tokens[s, :a] = drafts[s, :a]
        if want is not None:
            cum = np.cumsum(want)
            j = int(np.searchsorted(cum, float(u[s, n]) * cum[-1], side="right"))
            tokens[s, a] = j if j < v else int(np.nonzero(want > 0)[0][-1])
    return acc, tokens, p
