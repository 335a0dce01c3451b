"""The step operators' refusals, without a GPU: every call is turned down before a pointer is looked at, or, with arguments
that are right, because its addresses are no device memory."""
import pytest

A = 1 << 20  # (never read)


def norm(qkv, **kw):
    a = dict(x=A, xs=64, res=A, rs=64, w=A, rows=2, dim=64, eps=1e-6, dtype=0, sum=A, ss=64, y=A, ys=64, a=A, b=A, m=A)
    a.update(kw)
    qkv.norm_q32(a["x"], a["xs"], a["res"], a["rs"], a["w"], a["rows"], a["dim"], a["eps"], a["dtype"], a["sum"], a["ss"], a["y"], a["ys"], a["a"], a["b"],
                 a["m"])


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 21) + 1), "rows"), (dict(dim=0), "dim"), (dict(dim=32769, xs=40000), "dim"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(a=0), "set"), (dict(m=0), "set"),
    (dict(dim=96, xs=96, rs=96, ss=96, ys=96), "multiple of 64"), (dict(sum=0, y=0, a=0, b=0, m=0), "no output"), (dict(x=0), "null x"), (dict(w=0), "null w"),
    (dict(xs=63), "x_stride"), (dict(rs=1), "res_stride"), (dict(ss=0), "sum_stride"), (dict(ys=63), "y_stride"), (dict(ss=65), "stride"),
    (dict(res=0, ys=65, y=A), "stride"), (dict(x=A + 2), "x is not aligned"), (dict(w=A + 2), "w is not"), (dict(a=A + 8), "q32a"), (dict(m=A + 4), "q32meta"),
    (dict(dtype=1, y=A + 1), "y is not aligned"),
])
def test_norm_refusals(qkv, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        norm(qkv, **kw)


def w4(qkv, units=True, **kw):
    a = dict(rows=1, n=16, k=64, group=32, codes=A, scales=A, mins=0, x=A, b=A, m=A, xs=64, dtype=1, y=A, ys=16)
    a.update(kw)
    if units:
        qkv.w4_units(a["rows"], a["n"], a["k"], a["group"], a["codes"], a["scales"], a["mins"], a["x"], a["b"], a["m"], a["y"], a["ys"])
    else:
        qkv.w4_rows(a["rows"], a["n"], a["k"], a["group"], a["codes"], a["scales"], a["mins"], a["x"], a["xs"], a["dtype"], a["y"], a["ys"])


@pytest.mark.parametrize("units,kw,msg", [
    (True, dict(rows=-1), "rows"), (True, dict(rows=1 << 20), "rows"), (True, dict(n=0), "n outside"), (True, dict(k=0), "multiple of 64"),
    (True, dict(k=96), "multiple of 64"), (False, dict(k=48, xs=48), "multiple of 32"), (True, dict(group=16), "group"), (True, dict(group=256), "group"),
    (True, dict(ys=15), "y_stride"), (False, dict(xs=63), "x_stride"), (False, dict(dtype=3), "dtype"), (True, dict(codes=0), "codes"),
    (True, dict(scales=0), "scales"), (True, dict(y=0), "null y"), (True, dict(x=0), "q32a"), (True, dict(b=0), "q32b"), (True, dict(m=0), "q32meta"),
    (False, dict(x=0), "null x"), (True, dict(codes=A + 8), "codes"), (True, dict(x=A + 8), "q32a"), (False, dict(x=A + 1), "x is not"),
    (True, dict(mins=A + 1), "mins"), (True, dict(y=A + 2), "y is not"), (False, dict(k=1 << 21, xs=1 << 21), "2\\^20"),
])
def test_w4_refusals(qkv, units, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        w4(qkv, units, **kw)


def verify(qkv, **kw):
    a = dict(b=1, n=2, v=100, t=A, rs=100, dtype=0, probs=0, temp=0, q=0, d=A, nd=0, u=A, acc=A, tok=A, p=0, ws=A, size=1 << 20)
    a.update(kw)
    qkv.verify_drafts(a["b"], a["n"], a["v"], a["t"], a["rs"], a["dtype"], a["probs"], a["temp"], a["q"], a["d"], a["nd"], a["u"], a["acc"], a["tok"], a["p"],
                      a["ws"], a["size"])


@pytest.mark.parametrize("kw,msg", [
    (dict(b=-1), "n_seq"), (dict(b=65536), "n_seq"), (dict(n=-1), "n_draft"), (dict(n=65), "n_draft"), (dict(v=0), "vocab"), (dict(v=(1 << 24) + 1), "vocab"),
    (dict(b=60000, n=64, v=1 << 22, rs=1 << 22), "too many"), (dict(b=1 << 15, n=63, v=4 * 4096 + 1, rs=1 << 20), "too many"), (dict(dtype=3), "dtype"), (dict(probs=2), "probs"), (dict(probs=1, dtype=1), "fp32"),
    (dict(probs=1, temp=A), "temperature"), (dict(rs=99), "row_stride"), (dict(t=0), "target"), (dict(u=0), "null u"), (dict(acc=0), "accepted"),
    (dict(tok=0), "tokens"), (dict(d=0), "drafts"), (dict(t=A + 2), "target is not"), (dict(dtype=2, t=A + 1), "target is not"), (dict(u=A + 2), "aligned"),
    (dict(q=A + 1), "aligned"), (dict(ws=0), "workspace"), (dict(size=10), "workspace"), (dict(ws=A + 8), "ws is not"),
])
def test_verify_refusals(qkv, kw, msg):
    with pytest.raises(qkv.KVError, match=msg):
        verify(qkv, **kw)


def test_workspace_size(qkv):
    assert qkv.verify_ws(0, 3, 1000) == 0
    assert qkv.verify_ws(2, 3, 4096) == 2 * (4 * 16 + 4 * 8) and qkv.verify_ws(1, 0, 4097) == 2 * (16 + 8)
    for bad in ((-1, 0, 1), (1, 65, 10), (1, 1, 0)):
        with pytest.raises(qkv.KVError):
            qkv.verify_ws(*bad)


def test_empty_tensors(qkv):
    """No rows: the calls return without a look at their pointers (an empty tensor's are null), but not with wrong sizes."""
    norm(qkv, rows=0, x=0, res=0, sum=0, y=0, a=0, b=0, m=0)
    w4(qkv, True, rows=0, x=0, b=0, m=0, y=0)
    w4(qkv, False, rows=0, x=0, y=0)
    verify(qkv, b=0, t=0, d=0, u=0, acc=0, tok=0, ws=0, size=0)
    for f, kw in ((norm, dict(rows=0, dim=0)), (lambda q, **k: w4(q, True, **k), dict(rows=0, k=96)), (verify, dict(b=0, v=0))):
        with pytest.raises(qkv.KVError):
            f(qkv, **kw)


def test_no_device_memory(qkv):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for call in (lambda: norm(qkv), lambda: w4(qkv), lambda: w4(qkv, False), lambda: verify(qkv)):
        with pytest.raises(qkv.KVError):
            call()


def test_nothing_to_do(qkv):
    norm(qkv, rows=0)
    w4(qkv, rows=0)
    w4(qkv, False, rows=0)
    verify(qkv, b=0, ws=0, size=0)


def test_the_header_states_the_limits(qkv):
    """One past each limit that include/qwen38_kv.h gives is refused; the limits themselves are not (they get as far as the addresses)."""
    big = 1 << 40
    for call, at, past in (
            (lambda **k: norm(qkv, **{**dict(xs=big, rs=big, ss=big, ys=big), **k}), dict(rows=1 << 21, dim=32768), (dict(rows=(1 << 21) + 1), dict(dim=32769))),
            (lambda **k: w4(qkv, True, **{**dict(ys=big), **k}), dict(rows=1 << 19, n=1 << 28, k=1 << 20), (dict(rows=(1 << 19) + 1), dict(n=(1 << 28) + 1), dict(k=(1 << 20) + 64))),
            (lambda **k: w4(qkv, False, **{**dict(ys=big, xs=big), **k}), dict(rows=1 << 19, n=1 << 28, k=1 << 20), (dict(rows=(1 << 19) + 1), dict(n=(1 << 28) + 1), dict(k=(1 << 20) + 32))),
            (lambda **k: verify(qkv, **{**dict(rs=big, size=1 << 40), **k}), dict(b=65535, n=64), (dict(b=65536), dict(n=65), dict(v=(1 << 24) + 1)))):
        for kw in past:
            with pytest.raises(qkv.KVError, match="outside|multiple"):
                call(**kw)
        with pytest.raises(qkv.KVError) as e:
            call(**at)
        assert "outside" not in str(e.value) and "multiple" not in str(e.value), e.value
