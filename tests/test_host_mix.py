"""Refusals of the adapters, the router and the experts, without a GPU: every call is turned down before a pointer is looked at, or, with
arguments that are right, because its addresses are no device memory."""
import pytest

A = 1 << 20  # (never read)
BIG = 1 << 40


def lora(qkv, units=False, **kw):
    a = dict(rows=2, n=64, k=64, na=2, rank=16, a=A, b=A, abt=2, ranks=A, scales=A, ids=A, x=A, xs=64, dtype=0, qb=A, qm=A, base=A, bs=64, y=2 * A, ys=64, ws=A, size=BIG)
    a.update(kw)
    head = [a[i] for i in ("rows", "n", "k", "na", "rank", "a", "b", "abt", "ranks", "scales", "ids", "x")]
    tail = [a[i] for i in ("base", "bs", "y", "ys", "ws", "size")]
    if units:
        qkv.lora_units(*head, a["qb"], a["qm"], *tail)
    else:
        qkv.lora_rows(*head, a["xs"], a["dtype"], *tail)


def route(qkv, **kw):
    a = dict(rows=2, dim=64, e=8, top=2, x=A, xs=64, dtype=2, w=A, wt=2, bias=0, form=0, scale=1.0, logits=A, ids=A, wts=A, ws=A, size=BIG)
    a.update(kw)
    qkv.moe_route(*[a[i] for i in ("rows", "dim", "e", "top", "x", "xs", "dtype", "w", "wt", "bias", "form", "scale", "logits", "ids", "wts", "ws", "size")])


def moe(qkv, form="rows", **kw):
    a = dict(rows=2, dim=64, inner=64, e=8, top=2, group=32, up=A, us=A, um=A, down=A, ds=A, dm=A, x=A, xs=64, dtype=2, qb=A, qm=A, router=A, rt=2, bias=0, rform=0, scale=1.0,
             logits=A, ids=A, wts=A, y=A, ys=64, ws=A, size=BIG)
    a.update(kw)
    head = [a[i] for i in ("rows", "dim", "inner", "e", "top", "group", "up", "us", "um", "down", "ds", "dm", "x")]
    tail = [a[i] for i in ("ids", "wts", "y", "ys", "ws", "size")]
    if form == "units":
        qkv.moe_units(*head, a["qb"], a["qm"], *tail)
    elif form == "layer":
        qkv.moe_layer(*head, *[a[i] for i in ("xs", "dtype", "router", "rt", "bias", "rform", "scale", "logits")], *tail)
    else:
        qkv.moe_rows(*head, a["xs"], a["dtype"], *tail)


@pytest.mark.parametrize("units,kw,msg", [
    (False, dict(rows=-1), "rows"), (False, dict(rows=(1 << 19) + 1), "rows"), (False, dict(k=48), "multiple of 32"), (True, dict(k=96), "multiple of 64"),
    (False, dict(k=0, xs=0), "multiple of 32"), (False, dict(k=(1 << 20) + 32, xs=BIG), "multiple of 32"), (False, dict(rank=0), "rank"), (False, dict(rank=257), "rank"),
    (True, dict(n=0), "n outside"), (True, dict(n=(1 << 24) + 1, bs=BIG, ys=BIG), "n outside"), (False, dict(na=0), "n_adapters"), (False, dict(abt=0), "ab_dtype"),
    (False, dict(abt=3), "ab_dtype"), (False, dict(dtype=3), "dtype"), (False, dict(dtype=-1), "dtype"), (False, dict(xs=63), "x_stride"), (False, dict(ys=63), "y_stride"),
    (False, dict(bs=63), "base_stride"), (False, dict(base=2 * A, bs=65), "stride"), (False, dict(rows=1 << 19, n=1 << 17, bs=BIG, ys=BIG), "too many"),
    (False, dict(x=0), "null x"), (True, dict(x=0), "q32a"), (True, dict(qb=0), "q32b"), (True, dict(qm=0), "q32meta"), (False, dict(a=0), "null a"), (False, dict(b=0), "null b"),
    (False, dict(ids=0), "null ids"), (False, dict(y=0), "null y"), (False, dict(a=A + 1), "a is not"), (False, dict(b=A + 1), "b is not"), (False, dict(ranks=A + 2), "aligned"),
    (False, dict(scales=A + 2), "aligned"), (False, dict(ids=A + 1), "aligned"), (False, dict(base=A + 2), "aligned"), (False, dict(y=A + 2), "aligned"),
    (False, dict(x=A + 2), "x is not"), (True, dict(x=A + 8), "q32a"), (True, dict(qm=A + 4), "q32meta"), (False, dict(ws=0), "workspace"), (False, dict(size=16), "workspace"),
    (False, dict(ws=A + 8), "ws is not"),
])
def test_lora_refusals(qkv, units, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        lora(qkv, units, **kw)


ROUTE = [
    (dict(rows=-1), "rows"), (dict(rows=(1 << 19) + 1), "rows"), (dict(dim=0), "dim"), (dict(dim=(1 << 17) + 1, xs=BIG), "dim"), (dict(e=0), "n_experts"), (dict(e=1025), "n_experts"),
    (dict(top=0), "top_k"), (dict(top=17, e=100), "top_k"), (dict(top=9), "top_k"), (dict(form=4), "form"), (dict(form=-1), "form"), (dict(form=1, bias=A), "bias"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(xs=63), "x_stride"), (dict(dtype=3), "dtype"), (dict(wt=-1), "dtype"), (dict(x=0), "null x"),
    (dict(w=0), "null w"), (dict(logits=0), "null logits"), (dict(ids=0), "null ids"), (dict(wts=0), "null weights"), (dict(x=A + 1), "x is not"), (dict(w=A + 1), "w is not"),
    (dict(form=2, bias=A + 2), "aligned"), (dict(logits=A + 2), "aligned"), (dict(ids=A + 1), "aligned"), (dict(wts=A + 3), "aligned"),
]


@pytest.mark.parametrize("kw,msg", ROUTE)
def test_route_refusals(qkv, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        route(qkv, **kw)


MOE = [
    (dict(rows=-1), "rows"), (dict(rows=4097), "rows"), (dict(dim=48, xs=64), "dim must"), (dict(dim=0), "dim must"), (dict(dim=16416, xs=BIG, ys=BIG), "dim must"),
    (dict(inner=0), "inner"), (dict(inner=40), "inner"), (dict(inner=32800), "inner"), (dict(e=0), "n_experts"), (dict(e=1025), "n_experts"), (dict(top=0), "top_k"),
    (dict(top=9), "top_k"), (dict(top=17, e=64), "top_k"), (dict(group=16), "group"), (dict(group=256), "group"), (dict(ys=63), "y_stride"), (dict(um=0), "minimums"),
    (dict(dm=0), "minimums"), (dict(up=0), "null up"), (dict(us=0), "up_scales"), (dict(down=0), "null down"), (dict(ds=0), "down_scales"), (dict(ids=0), "null ids"),
    (dict(wts=0), "null weights"), (dict(y=0), "null y"), (dict(up=A + 8), "up is not"), (dict(down=A + 8), "down is not"), (dict(us=A + 1), "scale array"), (dict(dm=A + 1), "scale array"),
    (dict(ids=A + 2), "aligned"), (dict(wts=A + 2), "aligned"), (dict(ws=0), "workspace"), (dict(size=1000), "workspace"), (dict(ws=A + 8), "ws is not"),
]


@pytest.mark.parametrize("form", ["rows", "units", "layer"])
@pytest.mark.parametrize("kw,msg", MOE)
def test_moe_refusals(qkv, form, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        moe(qkv, form, **kw)


@pytest.mark.parametrize("form,kw,msg", [
    ("rows", dict(dtype=3), "dtype"), ("rows", dict(xs=63), "x_stride"), ("rows", dict(x=0), "null x"), ("rows", dict(x=A + 1), "x is not"), ("rows", dict(y=A + 1), "y is not"),
    ("rows", dict(dtype=0, y=A + 2), "y is not"), ("units", dict(dim=96, ys=96), "multiple of 64"), ("units", dict(x=0), "q32a"), ("units", dict(qb=0), "q32b"),
    ("units", dict(qm=0), "q32meta"), ("units", dict(x=A + 8), "q32a"), ("units", dict(y=A + 2), "y is not"), ("layer", dict(router=0), "null w"), ("layer", dict(rt=3), "dtype"),
    ("layer", dict(rform=4), "form"), ("layer", dict(bias=A), "bias"), ("layer", dict(logits=0), "null logits"), ("layer", dict(scale=float("inf")), "scale"),
])
def test_moe_refusals_of_a_form(qkv, form, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        moe(qkv, form, **kw)


def test_empty_tensors(qkv):
    """No rows: the calls return without a look at their pointers (an empty tensor's are null), but not with wrong sizes."""
    for units in (False, True):
        lora(qkv, units, rows=0, x=0, qb=0, qm=0, ids=0, base=0, y=0, ws=0, size=0)
    route(qkv, rows=0, x=0, logits=0, ids=0, wts=0, ws=0, size=0)
    for form in ("rows", "units", "layer"):
        moe(qkv, form, rows=0, x=0, qb=0, qm=0, ids=0, wts=0, logits=0, y=0, ws=0, size=0)
        with pytest.raises(qkv.KVError):
            moe(qkv, form, rows=0, dim=48)
    with pytest.raises(qkv.KVError):
        lora(qkv, rows=0, k=0)
    with pytest.raises(qkv.KVError):
        route(qkv, rows=0, e=0)


def test_no_device_memory(qkv):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for call in (lambda: lora(qkv), lambda: lora(qkv, True), lambda: route(qkv), lambda: moe(qkv), lambda: moe(qkv, "units"), lambda: moe(qkv, "layer")):
        with pytest.raises(qkv.KVError):
            call()


def test_workspaces(qkv):
    """What the calls ask for is what the size functions give, and those refuse what the calls refuse."""
    for f, good, bad in ((qkv.lora_ws, (64, 5120, 16), ((-1, 64, 16), (1, 33, 16), (1, 64, 0), (1, 64, 257))),
                         (qkv.moe_route_ws, (64, 2048, 128), ((-1, 64, 8), (1, 0, 8), (1, 64, 1025))),
                         (qkv.moe_ws, (64, 2048, 768, 128, 8), ((-1, 64, 64, 8, 2), (1, 33, 64, 8, 2), (1, 64, 33, 8, 2), (1, 64, 64, 0, 1), (1, 64, 64, 8, 9)))):
        assert f(*good) >= 0
        for b in bad:
            with pytest.raises(qkv.KVError):
                f(*b)
    assert qkv.moe_ws(4096, 64, 64, 8, 2) >= qkv.moe_ws(64, 64, 64, 8, 2)
    need = qkv.lora_ws(2, 64, 16)
    with pytest.raises(qkv.KVError, match=f"needs {need} bytes"):
        lora(qkv, size=need - 1)


def test_the_header_states_the_limits(qkv):
    """The limits that include/qwen38_kv.h gives are not refused (they get as far as the addresses); one past each is, above."""
    for call in (lambda: lora(qkv, rows=1 << 19, n=1 << 16, bs=BIG, ys=BIG, size=1 << 60), lambda: lora(qkv, k=1 << 20, n=1 << 24, rank=256, xs=BIG, bs=BIG, ys=BIG),
                 lambda: route(qkv, rows=1 << 19, dim=1 << 17, e=1024, top=16, xs=BIG, size=1 << 60), lambda: moe(qkv, rows=4096, dim=16384, inner=32768, e=1024, top=16, xs=BIG, ys=BIG)):
        with pytest.raises(qkv.KVError) as e:
            call()
        assert "outside" not in str(e.value) and "must" not in str(e.value) and "workspace" not in str(e.value), e.value
