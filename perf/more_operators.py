"""What a server of several requests runs beside the 4-bit projections, as its users call it: low-rank adapters of many requests at
once, the router of a mixture of experts, and such a layer's experts with 4-bit weights.  `own` False computes each in elementary
torch operations, True through the binding.

Fields of a case
  op "lora":  rows, n, k (y[rows][n] = base + s B (A x[rows][k])), rank, adapters (loaded), per (consecutive rows of one request), dtype
              (x: plain rows of a type, or "units": int8 units), wtype (the adapters' type), ragged (adapters of fewer ranks), free
              (every 4th request without an adapter), base (added to a projection's result)
     "route": rows, dim, experts, top, dtype, wtype (the router's weights), form ("softmax": over all experts, "chosen": over the chosen
              ones, "sigmoid": divided by their sum), bias (added to the scores for the choice alone), pad (elements between rows of x)
     "moe":   rows, dim, inner, experts, top, group (weights per scale), mins (asymmetric), x ("units" or the type of plain rows), layer
              (the router included, else the choice is given)
"""
import math
import os
import sys

import torch

own = False
_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_CODE = {"fp32": 0, "fp16": 1, "bf16": 2}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "units": 1.25}
_FORM = {"softmax": 0, "chosen": 1, "sigmoid": 3}
SCALE = 2.5  # of the sigmoid's weights


def _binding():
    """The framework's binding (only where `own` is true)."""
    m = sys.modules.get("qkv")
    if m is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38-megakernel_amd"))
        import qkv as m
    return m


def listed():
    return [
        # one token of one request beside o_proj: launch and latency
        dict(name="lora_step", op="lora", rows=1, n=5120, k=6144, rank=16, adapters=8, per=1, dtype="fp32", wtype="bf16", ragged=False, free=False, base=True),
        # eight requests with seven drafts each beside the q (with gate), k and v projections, on their units
        dict(name="lora_verify", op="lora", rows=64, n=14336, k=5120, rank=16, adapters=32, per=8, dtype="units", wtype="bf16", ragged=False, free=True, base=True),
        # 61 requests, nearly as many adapters, of ranks up to 64
        dict(name="lora_many", op="lora", rows=61, n=17408, k=5120, rank=64, adapters=500, per=1, dtype="bf16", wtype="fp16", ragged=True, free=False, base=True),
        # chunks of four requests' prompts together
        dict(name="lora_prompt", op="lora", rows=4001, n=6144, k=5120, rank=32, adapters=8, per=1031, dtype="bf16", wtype="bf16", ragged=False, free=False, base=True),
        # the router of one token
        dict(name="route_step", op="route", rows=1, dim=5120, experts=128, top=8, dtype="bf16", wtype="bf16", form="chosen", bias=False, pad=0),
        # a full batch's, with a bias that balances the experts
        dict(name="route_batch", op="route", rows=64, dim=5120, experts=256, top=8, dtype="fp32", wtype="fp32", form="sigmoid", bias=True, pad=0),
        # a chunk of a prompt, an odd number of experts, a slice of wider rows
        dict(name="route_prompt", op="route", rows=4096, dim=2048, experts=63, top=6, dtype="bf16", wtype="bf16", form="softmax", bias=False, pad=8),
        # one token through a whole layer of many small experts
        dict(name="moe_step", op="moe", rows=1, dim=2048, inner=768, experts=128, top=8, group=32, mins=False, x="bf16", layer=True),
        # a verify of seven drafts through it
        dict(name="moe_verify", op="moe", rows=8, dim=2048, inner=768, experts=128, top=8, group=32, mins=False, x="bf16", layer=True),
        # three tokens through few wide experts, asymmetric weights, in fp32
        dict(name="moe_wide", op="moe", rows=3, dim=5120, inner=6144, experts=8, top=2, group=64, mins=True, x="fp32", layer=False),
        # a full batch on the norm's units: nearly every expert, a few tokens each
        dict(name="moe_batch", op="moe", rows=64, dim=2048, inner=768, experts=128, top=8, group=32, mins=False, x="units", layer=False),
        # a batch through few experts: many tokens each
        dict(name="moe_dense", op="moe", rows=47, dim=4096, inner=8192, experts=8, top=2, group=128, mins=False, x="fp16", layer=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lora", "route", "moe", "moe"])
    if op == "lora":
        n, k, rank = _log(rng, 500, 17408), 64 * _log(rng, 8, 272), rng.choice([8, 16, 16, 32, 64, rng.randint(1, 64)])
        rows = min(_log(rng, 1, 4096), 24_000_000 // max(n, k))
        per = 1 if rows <= 64 and rng.random() < 0.6 else rng.randint(max(1, rows // 60), max(8, rows // 2))
        return dict(op="lora", rows=rows, n=n, k=k, rank=rank, adapters=_log(rng, 1, 200) if rows <= 64 else rng.randint(1, 16), per=per,
                    dtype=rng.choice(["units", "fp32", "fp16", "bf16"]), wtype=rng.choice(["fp16", "bf16"]), ragged=rng.random() < 0.3, free=rng.random() < 0.3,
                    base=rng.random() < 0.8)
    if op == "route":
        dim, experts = 32 * _log(rng, 16, 200), rng.choice([8, 60, 64, 128, 128, 256, rng.randint(2, 300)])
        rows = min(_log(rng, 1, 4096), 1_000_000_000 // (dim * experts))
        form = rng.choice(["softmax", "chosen", "sigmoid"])
        return dict(op="route", rows=max(1, rows), dim=dim, experts=experts, top=min(experts, rng.choice([1, 2, 4, 6, 8, 8, 10])), dtype=rng.choice(["fp32", "fp16", "bf16"]),
                    wtype=rng.choice(["fp32", "fp16", "bf16"]), form=form, bias=form == "sigmoid" and rng.random() < 0.5, pad=rng.choice([0, 0, 8, rng.randint(1, 40)]))
    experts = rng.choice([4, 8, 16, 60, 64, 128, 128, 200])
    x = rng.choice(["units", "fp32", "fp16", "bf16", "bf16"])
    dim = 64 * _log(rng, 8, 80)
    inner = min(32 * _log(rng, 8, 256), 200_000_000 // (experts * dim) // 32 * 32)
    return dict(op="moe", rows=rng.choice([1, 1, 2, 4, 8, rng.randint(1, 64), rng.randint(1, 64)]), dim=dim, inner=inner, experts=experts,
                top=min(experts, rng.choice([1, 2, 2, 4, 6, 8])), group=rng.choice([32, 32, 64, 128]), mins=rng.random() < 0.4, x=x, layer=x != "units" and rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what) % (1 << 62))
    return g


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


def _rows_or_units(x, form):
    return _units(x) if form == "units" else x.to(_DT[form])


def _lora_inputs(c, seed):
    g, rows, n, k, r, na = _gen(seed, 1), c["rows"], c["n"], c["k"], c["rank"], c["adapters"]
    wt = _DT[c["wtype"]]
    a = (torch.randn(na, r, k, device="cuda", generator=g) / math.sqrt(k)).to(wt)
    b = (torch.randn(na, n, r, device="cuda", generator=g) * 0.5).to(wt)
    ranks = torch.randint(1, r + 1, (na,), device="cuda", dtype=torch.int32, generator=g) if c["ragged"] else None
    scales = 0.5 + 1.5 * torch.rand(na, device="cuda", generator=g)
    reqs = -(-rows // c["per"])
    ids = torch.randint(0, na, (reqs,), device="cuda", dtype=torch.int32, generator=g)
    if c["free"]:
        ids[::4] = -1
    ids = ids.repeat_interleave(c["per"])[:rows].contiguous()
    x = _rows_or_units(torch.randn(rows, k, device="cuda", generator=g), c["dtype"])
    base = torch.randn(rows, n, device="cuda", generator=g) if c["base"] else None
    return a, b, ranks, scales, ids, x, base


def _router_weights(g, experts, dim, wtype):
    return (torch.randn(experts, dim, device="cuda", generator=g) * (1.5 / math.sqrt(dim))).to(_DT[wtype])


def _route_inputs(c, seed):
    g = _gen(seed, 2)
    x = torch.randn(c["rows"], c["dim"] + c["pad"], device="cuda", generator=g).to(_DT[c["dtype"]])[:, :c["dim"]]
    w = _router_weights(g, c["experts"], c["dim"], c["wtype"])
    bias = torch.randn(c["experts"], device="cuda", generator=g) * 0.1 if c["bias"] else None
    return x, w, bias


def _nibbles(g, shape):
    """4-bit codes, two a byte, spread as quantized weights are (most near the middle)."""
    def one():
        return torch.randint(0, 9, shape, device="cuda", dtype=torch.uint8, generator=g) + torch.randint(0, 8, shape, device="cuda", dtype=torch.uint8, generator=g)
    return one() | (one() << 4)


def _w4(g, e, n, k, group, mins):
    gs = -(-k // group)
    codes = _nibbles(g, (e, n, k // 2))
    scales = ((0.5 + torch.rand(e, n, gs, device="cuda", generator=g)) * (0.3 / math.sqrt(k))).half()
    return codes, scales, (torch.randn(e, n, gs, device="cuda", generator=g) * (0.2 / math.sqrt(k))).half() if mins else None


def _moe_inputs(c, seed):
    g, rows, dim, inner, e = _gen(seed, 3), c["rows"], c["dim"], c["inner"], c["experts"]
    up = _w4(g, e, 2 * inner, dim, c["group"], c["mins"])
    down = _w4(g, e, dim, inner, c["group"], c["mins"])
    x = _rows_or_units(torch.randn(rows, dim, device="cuda", generator=g), c["x"])
    if c["layer"]:
        return up, down, x, _router_weights(g, e, dim, "bf16" if c["x"] == "bf16" else "fp32")
    # some experts are asked for more often than others
    l = torch.randn(rows, e, device="cuda", generator=g) + 0.5 * torch.randn(e, device="cuda", generator=g)
    top, ids = l.topk(c["top"], -1)
    return up, down, x, (ids.to(torch.int32).contiguous(), torch.softmax(top, -1))


def prepare(case, seed):
    c, rows = dict(case), case["rows"]
    d = dict(c=c)
    if c["op"] == "lora":
        d["a"], d["b"], d["ranks"], d["scales"], d["ids"], d["x"], d["base"] = _lora_inputs(c, seed)
        d["y"] = torch.empty(rows, c["n"], device="cuda")
        # kept between calls: up to 16 partial sums of A x
        d["ws"] = torch.empty(4096 + 64 * rows * (c["rank"] + 15), device="cuda", dtype=torch.uint8)
        return d
    if c["op"] == "route":
        d["x"], d["w"], d["bias"] = _route_inputs(c, seed)
    else:
        d["up"], d["down"], d["x"], chosen = _moe_inputs(c, seed)
        if c["layer"]:
            d["w"], d["bias"] = chosen, None
        else:
            d["ids"], d["weights"] = chosen
        d["y"] = torch.empty(rows, c["dim"], device="cuda", dtype=torch.float32 if c["x"] == "units" else d["x"].dtype)
    # kept between calls: partial sums of the logits, and the experts' values within and behind the layer
    room = 65536 + 64 * min(rows, 256) * c["experts"]
    if c["op"] == "moe":
        room += rows * c["top"] * (8 * c["inner"] + 4 * c["dim"] + 1024)
    d["ws"] = torch.empty(room, device="cuda", dtype=torch.uint8)
    if "w" in d:
        d["logits"] = torch.empty(rows, c["experts"], device="cuda")
        d["ids"] = torch.empty(rows, c["top"], device="cuda", dtype=torch.int32)
        d["weights"] = torch.empty(rows, c["top"], device="cuda")
    return d


# ------------------------------------------------------------------------------------------------ a pass
def _plain_x(x, k):
    if not isinstance(x, tuple):
        return x.float()
    a, b, meta = x
    rows, nu = a.shape[:2]
    s = meta.view(torch.float16).view(rows, nu // 2, 2, 4)[:, :, 0, :2].float()
    q = torch.stack([a.view(rows, nu // 2, 32), b.view(rows, nu // 2, 32)], 2).float()
    return (q * s[..., None]).view(rows, k)


def _plain_lora(d):
    c, a, b, ids = d["c"], d["a"], d["b"], d["ids"].long()
    x = _plain_x(d["x"], c["k"])
    y = torch.zeros(c["rows"], c["n"], device=x.device) if d["base"] is None else d["base"]
    steps = torch.arange(c["rank"], device=x.device)
    if c["rows"] <= 64:  # every row's adapter by its index
        at = ids.clamp(min=0)
        u = torch.bmm(a[at].float(), x[:, :, None]).squeeze(-1) * (d["scales"][at] * (ids >= 0))[:, None]
        if d["ranks"] is not None:
            u = torch.where(steps < d["ranks"][at][:, None], u, 0.0)
        return y + torch.bmm(b[at].float(), u[:, :, None]).squeeze(-1)
    for i in range(c["adapters"]):  # every adapter's rows by a mask
        u = (x @ a[i].float().T) * (d["scales"][i] * (ids == i))[:, None]
        if d["ranks"] is not None:
            u = torch.where(steps < d["ranks"][i], u, 0.0)
        y = y + u @ b[i].float().T
    return y


def _plain_route(d):
    c = d["c"]
    # in 64 bits: the choice compares values that lie close to each other
    logits = (d["x"].double() @ d["w"].double().T).float()
    score = logits.double()
    if c.get("form") == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-score))
    key = logits.double() if d["bias"] is None else score + d["bias"].double()
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
    if c.get("form") == "softmax":
        e = torch.exp(score - score.amax(-1, keepdim=True))
        w = (e / e.sum(-1, keepdim=True)).gather(1, ids)
    elif c.get("form") == "sigmoid":
        w = score.gather(1, ids)
        w = w / w.sum(-1, keepdim=True) * SCALE
    else:
        e = score.gather(1, ids)
        e = torch.exp(e - e.amax(-1, keepdim=True))
        w = e / e.sum(-1, keepdim=True)
    return dict(logits=logits, ids=ids.int(), weights=w.float())


def _plain_weights(codes, scales, mins, group):
    n, k = codes.shape[0], codes.shape[1] * 2
    w = codes.view(n, k // 8, 1, 4)
    q = torch.cat([w & 15, w >> 4], 2).view(n, k).float() - 8
    s = scales.float().repeat_interleave(group, 1)[:, :k]
    return q * s if mins is None else q * s + mins.float().repeat_interleave(group, 1)[:, :k]


def _expert(t, i):
    return t[0][i], t[1][i], None if t[2] is None else t[2][i]


def _plain_moe(d):
    c = d["c"]
    out = _plain_route(d) if "w" in d else {}
    ids, weights = (out["ids"], out["weights"]) if out else (d["ids"], d["weights"])
    x = _plain_x(d["x"], c["dim"])
    y = torch.zeros(c["rows"], c["dim"], device=x.device)
    for i in ids.unique().tolist():
        row, slot = (ids == i).nonzero(as_tuple=True)
        gu = x[row] @ _plain_weights(*_expert(d["up"], i), c["group"]).T
        gate, up = gu[:, :c["inner"]], gu[:, c["inner"]:]
        h = gate / (1.0 + torch.exp(-gate)) * up
        y[row] += weights[row, slot][:, None] * (h @ _plain_weights(*_expert(d["down"], i), c["group"]).T)
    out["y"] = y.to(d["y"].dtype)
    return out


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def run(d):
    c = d["c"]
    if not own:
        return {"lora": _plain_lora, "route": _plain_route, "moe": _plain_moe}[c["op"]](d)
    qkv, stream = _binding(), torch.cuda.current_stream().cuda_stream
    x = d["x"]
    if c["op"] == "lora":
        y, n = d["y"], c["n"]
        head = (c["rows"], n, c["k"], c["adapters"], c["rank"], d["a"].data_ptr(), d["b"].data_ptr(), _CODE[c["wtype"]], _ptr(d["ranks"]),
                d["scales"].data_ptr(), d["ids"].data_ptr())
        tail = (_ptr(d["base"]), n, y.data_ptr(), n, d["ws"].data_ptr(), d["ws"].numel(), stream)
        if c["dtype"] == "units":
            qkv.lora_units(*head, x[0].data_ptr(), x[1].data_ptr(), x[2].data_ptr(), *tail)
        else:
            qkv.lora_rows(*head, x.data_ptr(), c["k"], _CODE[c["dtype"]], *tail)
        return y
    if c["op"] == "route":
        qkv.moe_route(c["rows"], c["dim"], c["experts"], c["top"], x.data_ptr(), x.stride(0), _CODE[c["dtype"]], d["w"].data_ptr(), _CODE[c["wtype"]],
                      _ptr(d["bias"]), _FORM[c["form"]], SCALE if c["form"] == "sigmoid" else 1.0, d["logits"].data_ptr(), d["ids"].data_ptr(),
                      d["weights"].data_ptr(), d["ws"].data_ptr(), d["ws"].numel(), stream)
        return dict(logits=d["logits"], ids=d["ids"], weights=d["weights"])
    head = (c["rows"], c["dim"], c["inner"], c["experts"], c["top"], c["group"], *map(_ptr, d["up"]), *map(_ptr, d["down"]))
    chosen = (d["ids"].data_ptr(), d["weights"].data_ptr())
    tail = (*chosen, d["y"].data_ptr(), c["dim"], d["ws"].data_ptr(), d["ws"].numel(), stream)
    if c["layer"]:
        qkv.moe_layer(*head, x.data_ptr(), c["dim"], _CODE[c["x"]], d["w"].data_ptr(), 2 if c["x"] == "bf16" else 0, 0, _FORM["chosen"], 1.0,
                      d["logits"].data_ptr(), *tail)
        return dict(logits=d["logits"], ids=d["ids"], weights=d["weights"], y=d["y"])
    if c["x"] == "units":
        qkv.moe_units(*head, *(t.data_ptr() for t in x), *tail)
    else:
        qkv.moe_rows(*head, x.data_ptr(), c["dim"], _CODE[c["x"]], *tail)
    return dict(y=d["y"])


def _distinct(of, asked):
    """How many of `of` things are met in `asked` draws, on average."""
    return of * (1 - (1 - 1 / of) ** asked)


def work(case):
    c, rows = case, case["rows"]
    if c["op"] == "lora":
        reqs, r = -(-rows // c["per"]), (c["rank"] + 1) / 2 if c["ragged"] else c["rank"]
        live = reqs - (-(-reqs // 4) if c["free"] else 0)
        share = live / reqs
        return {"bytes": _distinct(c["adapters"], live) * r * (c["n"] + c["k"]) * 2 + share * rows * c["k"] * _SIZE[c["dtype"]] + rows * c["n"] * 4 * (1 + c["base"]),
                "flops": 2 * share * rows * r * (c["n"] + c["k"])}
    route = rows * c["dim"] * _SIZE[c["dtype"] if c["op"] == "route" else c["x"]], c["experts"] * c["dim"], 2 * rows * c["experts"] * c["dim"]
    if c["op"] == "route":
        return {"bytes": route[0] + route[1] * _SIZE[c["wtype"]] + 4 * rows * (c["experts"] + 2 * c["top"]), "flops": route[2]}
    w = 3 * c["dim"] * c["inner"]
    met = c["experts"] * (1 - (1 - c["top"] / c["experts"]) ** rows)
    out = {"bytes": met * (w // 2 + 2 * w // c["group"] * (1 + c["mins"])) + route[0] + rows * c["dim"] * (4 if c["x"] == "units" else _SIZE[c["x"]]), "flops": 2 * rows * c["top"] * w}
    if c["layer"]:
        out["bytes"] += route[1] * (2 if c["x"] == "bf16" else 4) + 4 * rows * c["experts"]
        out["flops"] += route[2]
    return out


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_x(x):
    if not isinstance(x, tuple):
        return x.double()
    a, b, meta = x
    rows, nu = a.shape[:2]
    v = torch.empty(rows, nu * 32, device=a.device, dtype=torch.float64)
    unit = torch.arange(nu, device=a.device)
    at = (unit // 2 * 64 + unit % 2 * 16)[:, None] + torch.arange(16, device=a.device)  # the even block's values of each unit
    sc = meta[..., :2].contiguous().view(torch.float16).double()
    v[:, at] = a.double() * sc[..., 0:1]
    v[:, at + 32] = b.double() * sc[..., 1:2]
    return v


def _exact_lora(c, seed):
    a, b, ranks, scales, ids, x, base = _lora_inputs(c, seed)
    x, of = _exact_x(x), ids.tolist()
    y = torch.zeros(c["rows"], c["n"], device="cuda", dtype=torch.float64) if base is None else base.double()
    m = 0
    while m < len(of):  # runs of rows with one adapter
        e = m
        while e < len(of) and of[e] == of[m]:
            e += 1
        if of[m] >= 0:
            r = c["rank"] if ranks is None else int(ranks[of[m]])
            y[m:e] += float(scales[of[m]]) * ((x[m:e] @ a[of[m], :r].double().T) @ b[of[m], :, :r].double().T)
        m = e
    return y


def _exact_choice(x, w, bias, form, top):
    """-> logits, ids, weights of rows x by a router w."""
    logits = _exact_x(x) @ w.double().T
    key = logits if form != "sigmoid" else torch.sigmoid(logits)
    pick = key if bias is None else key + bias.double()
    ids = torch.empty(x.shape[0], top, device="cuda", dtype=torch.int64)
    left = pick.clone()
    for j in range(top):  # the largest that is left, the first of equal ones
        ids[:, j] = (left == left.amax(1, keepdim=True)).to(torch.int8).argmax(1)
        left.scatter_(1, ids[:, j:j + 1], -math.inf)
    if form == "softmax":
        weights = torch.softmax(logits, 1).gather(1, ids)
    elif form == "chosen":
        weights = torch.softmax(logits.gather(1, ids), 1)
    else:
        weights = key.gather(1, ids)
        weights = SCALE * weights / weights.sum(1, keepdim=True)
    return logits, ids.int(), weights


def _exact_weights(t, i, group):
    codes, scales, mins = _expert(t, i)
    n, k = codes.shape[0], codes.shape[1] * 2
    q = torch.empty(n, k, device=codes.device, dtype=torch.float64)
    byte = codes.to(torch.int32)
    for j in range(4):  # byte j of a word: value j in its low four bits, value j + 4 in its high ones
        q[:, j::8] = (byte[:, j::4] % 16).double() - 8
        q[:, j + 4::8] = torch.div(byte[:, j::4], 16, rounding_mode="floor").double() - 8
    of = torch.arange(k, device=codes.device) // group
    q *= scales.double()[:, of]
    return q if mins is None else q + mins.double()[:, of]


def _exact_moe(c, seed):
    up, down, x, chosen = _moe_inputs(c, seed)
    out = {}
    if c["layer"]:
        out["logits"], ids, weights = _exact_choice(x, chosen, None, "chosen", c["top"])
        out["ids"], out["weights"] = ids, weights
    else:
        ids, weights = chosen[0], chosen[1].double()
    v, y = _exact_x(x), torch.zeros(c["rows"], c["dim"], device="cuda", dtype=torch.float64)
    asked = ids.tolist()
    for i in sorted({e for row in asked for e in row}):
        hit = [(m, j) for m, row in enumerate(asked) for j, e in enumerate(row) if e == i]
        m, j = ([h[t] for h in hit] for t in (0, 1))
        gu = v[m] @ _exact_weights(up, i, c["group"]).T
        h = torch.nn.functional.silu(gu[:, :c["inner"]]) * gu[:, c["inner"]:]
        y[m] += weights[m, j][:, None] * (h @ _exact_weights(down, i, c["group"]).T)
    out["y"] = y
    return out


def exact(case, seed):
    if case["op"] == "lora":
        return _exact_lora(case, seed)
    if case["op"] == "route":
        x, w, bias = _route_inputs(case, seed)
        return dict(zip(("logits", "ids", "weights"), _exact_choice(x, w, bias, case["form"], case["top"])))
    return _exact_moe(case, seed)
