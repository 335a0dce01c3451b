"""The router's weights where the chosen experts' sigmoids are below 64 bits' smallest: they are defined all the same."""
import numpy as np
import pytest

from mixcase import typed
from test_gpu_moe import Case
from test_gpu_route import run

pytestmark = pytest.mark.gpu


def far(logits, ids):
    """sigmoid(l) over the chosen ones' sum, 64 bits: log sigmoid(l) = min(l, 0) - log(1 + exp(-|l|))."""
    l = np.take_along_axis(logits.astype(np.float64), ids.astype(np.int64), 1)
    s = np.minimum(l, 0) - np.log1p(np.exp(-np.abs(l)))
    e = np.exp(s - s.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


# (from 1536 rows on another kernel, which takes no bias)
@pytest.mark.parametrize("rows,dim,e,top,bias", [(1, 64, 8, 3, False), (70, 64, 40, 8, True), (5, 2048, 200, 8, True), (9, 96, 300, 16, False), (1030, 64, 40, 4, False), (1600, 64, 40, 4, False), (1600, 64, 40, 4, True)])
def test_far_below_zero(qkv, torch_gpu, rows, dim, e, top, bias):
    """Logits about -600, -700, -800 and -2000, close to each other and far apart; a bias that leaves such experts alone."""
    rng = np.random.default_rng(rows + e)
    at = rng.choice([-590.0, -640.0, -704.0, -800.0, -2000.0], (rows, 1))
    x = np.zeros((rows, dim))
    x[:, 0], x[:, 1] = 1, at[:, 0]
    x[:, 2:] = rng.integers(-8, 9, (rows, dim - 2)) / 8.0
    w = np.zeros((e, dim))
    w[:, 0], w[:, 1] = -rng.integers(0, 40, e) / 4.0, 1
    w[:, 2:] = rng.integers(-2, 3, (e, dim - 2)) / 16.0
    w[1::5, 0] -= 64
    b = np.where(rng.random(e) < 0.5, -np.inf, rng.random(e)).astype(np.float32) if bias else None
    if bias:
        w[0, 1], b[0] = 0, -np.inf  # (a large one that may not be chosen)
        b[-top:] = 0.5
    x, xv = typed(x, "bf16")
    w, wv = typed(w, "bf16")
    logits, ids, wt = run(qkv, torch_gpu, x, "bf16", w, "bf16", b, 3, 1.0, top)
    assert np.isfinite(logits).all()
    want = far(logits, ids)
    assert (np.abs(wt - want) <= 2.0 ** -23 * want + 2.0 ** -149).all(), np.argwhere(~np.isfinite(wt))[:5]


def test_layer(qkv, torch_gpu):
    """A layer's row of such weights has numbers in y."""
    torch = torch_gpu
    c = Case(torch, 4, 128, 64, 12, 3, xform="fp32", router="fp32", seed=3)
    c.router[:] = -8.0 + 0.001 * torch.arange(12, device="cuda")[:, None]
    c.x.abs_().add_(0.5)
    c.xv = c.x.double().cpu().numpy()
    head = (c.rows, c.dim, c.inner, c.e, c.top, c.group, *(t.data_ptr() if t is not None else 0 for d in c.dev for t in d))
    need = qkv.moe_ws(c.rows, c.dim, c.inner, c.e, c.top)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    y = c.out()
    qkv.moe_layer(*head, c.x.data_ptr(), c.x.stride(0), 0, c.router.data_ptr(), 0, 0, 3, 1.0, c.logits.data_ptr(), c.chosen[0].data_ptr(), c.chosen[1].data_ptr(), y.data_ptr(),
                  y.stride(0), ws.data_ptr(), need)
    logits, c.ids = c.logits.cpu().numpy(), c.chosen[0].cpu().numpy()
    assert (logits < -900).all()
    c.weights = far(logits, c.ids)
    assert (np.abs(c.chosen[1].cpu().numpy() - c.weights) <= 2.0 ** -23 * c.weights).all()
    ref, bound = c.want()
    assert (np.abs(y.double().cpu().numpy() - ref) <= bound + 2.0 ** -22 * np.abs(ref).max()).all()
