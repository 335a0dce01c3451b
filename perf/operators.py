"""What a decoder runs between the KV store's calls, as its users call it: the residual norm that leaves int8 activation units,
the matrix-vector products of 4-bit weights that take them (or plain rows), and the verification of drafted tokens.  `own`
False computes each in elementary torch operations, True through the binding.

Fields of a case
  op      "norm":   rows, dim, dtype, res (residual added), out ("units": int8 units and their scales; "rows": the normed rows;
                    "both"), pad (elements between the rows of x)
          "w4":     rows, n, k (y[rows][n] = x[rows][k] W[n][k]^T), group (weights per scale), mins (asymmetric), x ("units",
                    or the type of plain rows)
          "verify": seqs, drafts, vocab, dtype, form ("logits" or "probs"), q ("one" for drafts without probabilities of their
                    own, "probs" for a draft model's), greedy (every 4th sequence decodes at temperature 0), ragged (sequences
                    with fewer drafts)
"""
import math
import os
import sys

import torch

own = False
_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_CODE = {"fp32": 0, "fp16": 1, "bf16": 2}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6


def _binding():
    """The framework's binding (only where `own` is true)."""
    m = sys.modules.get("qkv")
    if m is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38-megakernel_amd"))
        import qkv as m
    return m


def listed():
    return [
        # one token's residual norm in a decode step, units for the next projection: launch and latency
        dict(name="norm_step", op="norm", rows=1, dim=5120, dtype="fp32", res=True, out="units", pad=0),
        # a verify step of four sequences with seven drafts each
        dict(name="norm_verify32", op="norm", rows=32, dim=5120, dtype="bf16", res=True, out="both", pad=0),
        # one chunk of a prompt
        dict(name="norm_prompt", op="norm", rows=4096, dim=5120, dtype="bf16", res=True, out="units", pad=0),
        # normed rows of a wide slice of another tensor, no residual, an odd width
        dict(name="norm_rows_odd", op="norm", rows=1111, dim=6143, dtype="fp32", res=False, out="rows", pad=41),
        # a kv projection of one token: the smallest product
        dict(name="w4_kv_1", op="w4", rows=1, n=1024, k=5120, group=32, mins=False, x="units"),
        # o_proj of one token, on the units the attention leaves (24 heads of 256)
        dict(name="w4_o_1", op="w4", rows=1, n=5120, k=6144, group=32, mins=False, x="units"),
        # the q (with gate), k and v projections of a verify of 7 drafts
        dict(name="w4_qkv_8", op="w4", rows=8, n=14336, k=5120, group=64, mins=True, x="units"),
        # an output head on one plain row, an odd vocabulary
        dict(name="w4_head_1", op="w4", rows=1, n=150001, k=5120, group=128, mins=False, x="bf16"),
        # eight sequences with seven drafts each through a wide projection
        dict(name="w4_wide_64", op="w4", rows=64, n=17408, k=5120, group=32, mins=False, x="units"),
        # one sequence with seven drafts over a draft vocabulary
        dict(name="verify_1x7", op="verify", seqs=1, drafts=7, vocab=32768, dtype="fp32", form="logits", q="one", greedy=False, ragged=False),
        # four sequences with a draft model's probabilities
        dict(name="verify_4x3_q", op="verify", seqs=4, drafts=3, vocab=150001, dtype="bf16", form="logits", q="probs", greedy=False, ragged=False),
        # a full batch, some greedy, some with fewer drafts
        dict(name="verify_64x7", op="verify", seqs=64, drafts=7, vocab=150001, dtype="fp32", form="logits", q="one", greedy=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "w4", "w4", "verify"])
    if op == "norm":
        out = rng.choice(["units", "units", "rows", "both"])
        dim = 64 * _log(rng, 4, 256) if out != "rows" else _log(rng, 100, 16384)
        rows = min(_log(rng, 1, 8192), 20_000_000 // dim)
        return dict(op="norm", rows=rows, dim=dim, dtype=rng.choice(["fp32", "fp16", "bf16", "bf16"]), res=rng.random() < 0.7, out=out,
                    pad=rng.choice([0, 0, 0, 8, rng.randint(1, 99)]))
    if op == "w4":
        x = rng.choice(["units", "units", "units", "fp16", "bf16", "fp32"])
        k = 64 * _log(rng, 4, 400)
        n = min(_log(rng, 64, 150000), 700_000_000 // k)
        rows = rng.choice([1, 1, 1, 2, 3, 4, 5, 8, 8, 16, rng.randint(1, 64), rng.randint(1, 64)])
        while rows > 1 and rows * n * k > 64 * 17408 * 5120:
            rows = max(1, rows // 2)
        return dict(op="w4", rows=rows, n=n, k=k, group=rng.choice([32, 32, 64, 128]), mins=rng.random() < 0.4, x=x)
    form = rng.choice(["logits", "logits", "probs"])
    q, drafts, vocab = rng.choice(["one", "one", "probs"]), rng.randint(0, 8), _log(rng, 1000, 150000)
    seqs = min(_log(rng, 1, 64), 64 * 8 * 150001 // (2 * (drafts + 1) * vocab))
    return dict(op="verify", seqs=seqs, drafts=drafts, vocab=vocab, dtype="fp32" if form == "probs" else rng.choice(["fp32", "fp16", "bf16"]),
                form=form, q=q, greedy=form == "logits" and rng.random() < 0.5, ragged=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, what=0):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what) % (1 << 62))
    return g


def _norm_inputs(c, seed):
    g, rows, dim, dt = _gen(seed, 1), c["rows"], c["dim"], _DT[c["dtype"]]
    x = torch.randn(rows, dim + c["pad"], device="cuda", generator=g).to(dt)[:, :dim]
    # the residual stream: larger, with a few channels much larger than the others
    big = torch.ones(dim, device="cuda")
    big[torch.randint(0, dim, (4,), device="cuda", generator=g)] = 20.0
    r = (torch.randn(rows, dim, device="cuda", generator=g) * 3 * big).to(dt) if c["res"] else None
    w = 1 + 0.2 * torch.randn(dim, device="cuda", generator=g)
    return x, r, w


def _units(x):
    """fp32 rows [rows][k] -> int8 units: a, b [rows][k / 32][16] of the even and odd 32-value blocks, meta [rows][k / 32][4]."""
    rows, k = x.shape
    v = x.reshape(rows, k // 64, 2, 2, 16)  # [pair][block of the pair][half][16]
    d = v.abs().amax((-1, -2), keepdim=True) / 127.0
    q = torch.where(d > 0, torch.round(v / d), torch.zeros_like(v)).to(torch.int8)
    sums = q.sum(-1, dtype=torch.int32).to(torch.int16)  # [rows][pair][block][half]
    sc = d.to(torch.float16).view(torch.int16).expand(-1, -1, -1, 2, -1)[..., 0]
    meta = torch.cat([sc, sums], 2).permute(0, 1, 3, 2)  # [rows][pair][half][scale a, scale b, sum a, sum b]
    return (q[:, :, 0].reshape(rows, k // 32, 16).contiguous(), q[:, :, 1].reshape(rows, k // 32, 16).contiguous(),
            meta.reshape(rows, k // 32, 4).contiguous())


def _nibbles(g, n, k):
    """k 4-bit codes per row, two a byte, spread as quantized weights are (most near the middle)."""
    def one():
        return torch.randint(0, 9, (n, k // 2), device="cuda", dtype=torch.uint8, generator=g) + torch.randint(
            0, 8, (n, k // 2), device="cuda", dtype=torch.uint8, generator=g)
    return one() | (one() << 4)


def _w4_inputs(c, seed):
    g, rows, n, k, gs = _gen(seed, 2), c["rows"], c["n"], c["k"], -(-c["k"] // c["group"])
    codes = _nibbles(g, n, k)
    scales = ((0.5 + torch.rand(n, gs, device="cuda", generator=g)) * 0.01).half()
    mins = (torch.randn(n, gs, device="cuda", generator=g) * 0.01).half() if c["mins"] else None
    x = torch.randn(rows, k, device="cuda", generator=g)
    return codes, scales, mins, _units(x) if c["x"] == "units" else x.to(_DT[c["x"]])


def _verify_inputs(c, seed):
    g, b, n, v = _gen(seed, 3), c["seqs"], c["drafts"], c["vocab"]
    logits = torch.randn(b, n + 1, v, device="cuda", generator=g) * 3
    temp = 0.6 + 0.6 * torch.rand(b, device="cuda", generator=g)
    # the draft model: the target's logits with noise of its own
    dl = (logits[:, :n] + torch.randn(b, n, v, device="cuda", generator=g)) / temp[:, None, None]
    dp = torch.softmax(dl, -1)
    if c["q"] == "one" or not n:
        drafts = dl.argmax(-1)
    else:
        cum = dp.double().cumsum(-1)
        drafts = (cum <= torch.rand(b, n, 1, device="cuda", generator=g) * cum[..., -1:]).sum(-1).clamp(max=v - 1)
    if c["q"] == "one":
        dp = None
    u = torch.rand(b, n + 1, device="cuda", generator=g)
    if c["form"] == "probs":
        target, temp = torch.softmax(logits / temp[:, None, None], -1), None
    else:
        target = logits.to(_DT[c["dtype"]])
        if c["greedy"]:
            temp[::4] = 0
    nd = torch.randint(0, n + 1, (b,), device="cuda", dtype=torch.int32, generator=g) if c["ragged"] else None
    return target, temp, dp, drafts.to(torch.int32).contiguous(), nd, u


def prepare(case, seed):
    d = dict(c=dict(case))
    if case["op"] == "norm":
        x, r, w = _norm_inputs(case, seed)
        rows, dim = x.shape
        d.update(x=x, r=r, w=w)
        if r is not None:
            d["h"] = torch.empty_like(r)
        if case["out"] != "units":
            d["y"] = torch.empty(rows, dim, device="cuda", dtype=x.dtype)
        if case["out"] != "rows":
            d["a"], d["b"] = (torch.empty(rows, dim // 32, 16, device="cuda", dtype=torch.int8) for _ in range(2))
            d["meta"] = torch.empty(rows, dim // 32, 4, device="cuda", dtype=torch.int16)
    elif case["op"] == "w4":
        d["codes"], d["scales"], d["mins"], d["x"] = _w4_inputs(case, seed)
        d["y"] = torch.empty(case["rows"], case["n"], device="cuda")
    else:
        d["target"], d["temp"], d["dp"], d["drafts"], d["nd"], d["u"] = _verify_inputs(case, seed)
        b, n = case["seqs"], case["drafts"]
        d["acc"] = torch.empty(b, device="cuda", dtype=torch.int32)
        d["tokens"] = torch.empty(b, n + 1, device="cuda", dtype=torch.int32)
        d["p"] = torch.empty(b, n, device="cuda")
        # a workspace kept between calls: 64 bytes for every 1,024 entries of a row, and one more piece a row
        d["ws"] = torch.empty(b * (n + 1) * (case["vocab"] // 1024 + 2) * 64, device="cuda", dtype=torch.uint8)
    return d


# ------------------------------------------------------------------------------------------------ a pass
def _unit_values(a, b, meta):
    """The values that int8 units stand for: the even blocks' and the odd blocks', [rows][pairs][32]."""
    rows, nu = a.shape[:2]
    s = meta.view(torch.float16).view(rows, nu // 2, 2, 4)
    return a.view(rows, nu // 2, 32) * s[:, :, 0, 0:1], b.view(rows, nu // 2, 32) * s[:, :, 0, 1:2]


def _plain_norm(d):
    c, x, r, w = d["c"], d["x"], d["r"], d["w"]
    out = {}
    h = x
    if r is not None:
        h = (x.float() + r.float()).to(x.dtype)
        out["h"] = h
    h = h.float()
    # the row's sum in 64 bits: every rounding after it is then the same in any order of summation
    rs = (1.0 / (h.double().square().sum(-1, keepdim=True) / h.shape[-1] + EPS).sqrt()).float()
    if c["out"] != "units":
        out["y"] = (h * rs * w).to(x.dtype)
    if c["out"] != "rows":
        t = (h * w).view(x.shape[0], -1, 2, 32)
        am = t.abs().amax(-1, keepdim=True)
        q = torch.round(t * (127.0 / am)).nan_to_num(0.0)
        sc = (am * (rs[:, :, None, None] / 127.0)).half()
        out["even"], out["odd"] = (q[:, :, i].half() * sc[:, :, i] for i in (0, 1))
    return out


def _plain_weights(codes, scales, mins, group):
    n, k = codes.shape[0], codes.shape[1] * 2
    w = codes.view(n, k // 8, 1, 4)
    q = torch.cat([w & 15, w >> 4], 2).view(n, k).float() - 8
    s = scales.float().repeat_interleave(group, 1)[:, :k]
    return q * s if mins is None else q * s + mins.float().repeat_interleave(group, 1)[:, :k]


def _plain_w4(d):
    x = d["x"]
    if d["c"]["x"] == "units":
        a, b, meta = x
        rows, nu = a.shape[:2]
        s = meta.view(torch.float16).view(rows, nu // 2, 2, 4)[:, :, 0, :2].float()
        q = torch.stack([a.view(rows, nu // 2, 32), b.view(rows, nu // 2, 32)], 2).float()
        x = (q * s[..., None]).view(rows, nu * 32)
    return x.float() @ _plain_weights(d["codes"], d["scales"], d["mins"], d["c"]["group"]).T


def _plain_verify(d):
    c, target, temp, dp, drafts, nd, u = d["c"], d["target"], d["temp"], d["dp"], d["drafts"].long(), d["nd"], d["u"].double()
    b, n, v = c["seqs"], c["drafts"], c["vocab"]
    # in 64 bits: cumulative sums of 150,000 small values, compared with a random number
    if c["form"] == "probs":
        w = target.double()
        z = torch.ones(b, n + 1, 1, device=w.device, dtype=torch.float64)
    else:
        top, best = target.max(-1, keepdim=True)
        greedy = (temp == 0)[:, None, None]
        scale = torch.where(greedy, torch.ones_like(temp[:, None, None], dtype=torch.float64), 1.0 / temp.double()[:, None, None])
        w = torch.exp((target.double() - top.double()) * scale)
        # temperature 0: all the probability on the largest logit, the lowest index of equal ones
        first = torch.arange(v, device=w.device) == (target == top).to(torch.int8).argmax(-1, keepdim=True)
        w = torch.where(greedy, first.double(), w)
        z = w.sum(-1, keepdim=True)
    p = (w[:, :n].gather(2, drafts[..., None]) / z[:, :n]).squeeze(-1)
    qd = torch.ones_like(p) if dp is None else dp.gather(2, drafts[..., None]).squeeze(-1).double()
    count = torch.full((b,), n, device=w.device) if nd is None else nd.long()
    live = torch.arange(n, device=w.device) < count[:, None]
    ok = (u[:, :n] * qd < p) & live
    acc = ok.long().cumprod(-1).sum(-1)
    row = w.gather(1, acc[:, None, None].expand(-1, 1, v)).squeeze(1) / z.squeeze(-1).gather(1, acc[:, None])
    # a refused draft: what the target has more than the draft model
    refused = (acc < count)[:, None]
    at = acc.clamp(max=max(n - 1, 0))
    if n:
        if dp is None:
            less = row.scatter(1, drafts.gather(1, at[:, None]), 0.0)
        else:
            less = (row - dp.gather(1, at[:, None, None].expand(-1, 1, v)).squeeze(1).double()).clamp(min=0.0)
        less = torch.where(less.sum(-1, keepdim=True) > 0, less, row)
        row = torch.where(refused, less, row)
    cum = row.cumsum(-1)
    # by a random number of its own, the last: the one that refused a draft is not free any more
    token = (cum <= u[:, n:] * cum[:, -1:]).sum(-1)
    steps = torch.arange(n + 1, device=w.device)
    tokens = torch.cat([drafts, torch.full((b, 1), -1, device=w.device)], 1)
    tokens = torch.where(steps < acc[:, None], tokens, torch.where(steps == acc[:, None], token[:, None], -1))
    return dict(accepted=acc.int(), tokens=tokens.int(), p=(p * live).float())


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def run(d):
    c = d["c"]
    if not own:
        return {"norm": _plain_norm, "w4": _plain_w4, "verify": _plain_verify}[c["op"]](d)
    qkv, stream = _binding(), torch.cuda.current_stream().cuda_stream
    if c["op"] == "norm":
        x, out = d["x"], {}
        qkv.norm_q32(x.data_ptr(), x.stride(0), _ptr(d["r"]), c["dim"], d["w"].data_ptr(), c["rows"], c["dim"], EPS, _CODE[c["dtype"]],
                     _ptr(d.get("h")), c["dim"], _ptr(d.get("y")), c["dim"], _ptr(d.get("a")), _ptr(d.get("b")), _ptr(d.get("meta")), stream)
        if "h" in d:
            out["h"] = d["h"]
        if "y" in d:
            out["y"] = d["y"]
        if "a" in d:
            out["even"], out["odd"] = _unit_values(d["a"], d["b"], d["meta"])
        return out
    if c["op"] == "w4":
        x, y = d["x"], d["y"]
        if c["x"] == "units":
            qkv.w4_units(c["rows"], c["n"], c["k"], c["group"], d["codes"].data_ptr(), d["scales"].data_ptr(), _ptr(d["mins"]),
                         x[0].data_ptr(), x[1].data_ptr(), x[2].data_ptr(), y.data_ptr(), c["n"], stream)
        else:
            qkv.w4_rows(c["rows"], c["n"], c["k"], c["group"], d["codes"].data_ptr(), d["scales"].data_ptr(), _ptr(d["mins"]),
                        x.data_ptr(), c["k"], _CODE[c["x"]], y.data_ptr(), c["n"], stream)
        return y
    qkv.verify_drafts(c["seqs"], c["drafts"], c["vocab"], d["target"].data_ptr(), c["vocab"], _CODE[c["dtype"]], int(c["form"] == "probs"),
                      _ptr(d["temp"]), _ptr(d["dp"]), d["drafts"].data_ptr(), _ptr(d["nd"]), d["u"].data_ptr(), d["acc"].data_ptr(),
                      d["tokens"].data_ptr(), d["p"].data_ptr(), d["ws"].data_ptr(), d["ws"].numel(), stream)
    return dict(accepted=d["acc"], tokens=d["tokens"], p=d["p"])


def work(case):
    c = case
    if c["op"] == "norm":
        e, s = c["rows"] * c["dim"], _SIZE[c["dtype"]]
        moved = s * (1 + 2 * c["res"] + (c["out"] != "units")) + (1.25 if c["out"] != "rows" else 0)
        return {"bytes": e * moved + 4 * c["dim"], "flops": 6 * e}
    if c["op"] == "w4":
        w = c["n"] * c["k"] // 2 + c["n"] * -(-c["k"] // c["group"]) * 2 * (1 + c["mins"])
        x = c["rows"] * c["k"] * (1.25 if c["x"] == "units" else _SIZE[c["x"]])
        return {"bytes": w + x + 4 * c["rows"] * c["n"], "flops": 2 * c["rows"] * c["n"] * c["k"]}
    # every row of the target once; of a draft model's rows the drafts' own entries and the refused row
    rows = c["seqs"] * (c["drafts"] + 1) * c["vocab"]
    q = c["seqs"] * c["vocab"] * 4 if c["q"] == "probs" and c["drafts"] else 0
    return {"bytes": rows * _SIZE[c["dtype"]] + q, "flops": 10 * rows}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_norm(c, seed):
    x, r, w = _norm_inputs(c, seed)
    out = {}
    h = x.double()
    if r is not None:
        # the stored sum is the operator's own rounding to the stream's type: the norm is of what is stored
        h = h + r.double()
        out["h"] = h
        h = h.to(torch.float32).to(x.dtype).double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * w.double()
    if c["out"] != "units":
        out["y"] = y
    if c["out"] != "rows":
        blocks = y.reshape(c["rows"], c["dim"] // 64, 2, 32)
        step = blocks.abs().amax(-1, keepdim=True) / 127
        v = torch.round(blocks / step.clamp(min=1e-300)) * step
        out["even"], out["odd"] = v[:, :, 0], v[:, :, 1]
    return out


def _exact_w4(c, seed):
    codes, scales, mins, x = _w4_inputs(c, seed)
    n, k, rows, group = c["n"], c["k"], c["rows"], c["group"]
    if c["x"] == "units":
        a, b, meta = x
        v = torch.empty(rows, k, device="cuda", dtype=torch.float64)
        unit = torch.arange(k // 32, device="cuda")
        at = (unit // 2 * 64 + unit % 2 * 16)[:, None] + torch.arange(16, device="cuda")  # the even block's values of each unit
        sc = meta[..., :2].contiguous().view(torch.float16).double()
        v[:, at] = a.double() * sc[..., 0:1]
        v[:, at + 32] = b.double() * sc[..., 1:2]
    else:
        v = x.double()
    out = torch.empty(rows, n, device="cuda", dtype=torch.float64)
    for j in range(0, n, 16384):
        q = torch.empty(min(16384, n - j), k, device="cuda", dtype=torch.float64)
        byte = codes[j:j + 16384].to(torch.int32)
        for i in range(4):  # byte i of a word: value i in its low four bits, value i + 4 in its high ones
            q[:, i::8] = (byte[:, i::4] % 16).double() - 8
            q[:, i + 4::8] = torch.div(byte[:, i::4], 16, rounding_mode="floor").double() - 8
        of = torch.arange(k, device="cuda") // group
        q *= scales[j:j + 16384].double()[:, of]
        if mins is not None:
            q += mins[j:j + 16384].double()[:, of]
        out[:, j:j + 16384] = v @ q.T
    return out


def _exact_verify(c, seed):
    target, temp, dp, drafts, nd, u = _verify_inputs(c, seed)
    b, n = c["seqs"], c["drafts"]
    p = torch.zeros(b, n, device="cuda", dtype=torch.float64)
    acc, tokens = torch.zeros(b, dtype=torch.int32), torch.full((b, n + 1), -1, dtype=torch.int32)
    count, drafted, rnd = [n] * b if nd is None else nd.tolist(), drafts.tolist(), u.double().tolist()
    for s in range(b):
        rows = target[s].double()
        if c["form"] != "probs":
            t = float(temp[s])
            if t:
                rows = torch.softmax(rows / t, -1)
            else:
                best = [int((r == r.max()).nonzero()[0]) for r in rows]
                rows = torch.zeros_like(rows)
                rows[range(n + 1), best] = 1.0
        a, want = 0, None
        for i in range(count[s]):
            p[s, i] = rows[i, drafted[s][i]]
        for i in range(count[s]):
            qi = 1.0 if dp is None else float(dp[s, i, drafted[s][i]])
            if not rnd[s][i] * qi < float(p[s, i]):
                if dp is None:
                    want = rows[i].clone()
                    want[drafted[s][i]] = 0
                else:
                    want = torch.relu(rows[i] - dp[s, i].double())
                break
            a += 1
        if want is None or not float(want.sum()) > 0:
            want = rows[a]
        part = torch.cumsum(want, 0)
        acc[s] = a
        tokens[s, :a] = torch.tensor(drafted[s][:a], dtype=torch.int32)
        tokens[s, a] = int(torch.searchsorted(part, rnd[s][n] * part[-1], right=True))
    return dict(accepted=acc, tokens=tokens, p=p)


def exact(case, seed):
    return {"norm": _exact_norm, "w4": _exact_w4, "verify": _exact_verify}[case["op"]](case, seed)
