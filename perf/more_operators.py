"""Cases for the operators of a decoder layer that serves many requests, around its block-quantised products: the
residual's addition with the norm and its 8-bit rows (`norm`), the choice of experts by score, bias and group
(`route`), the low-rank adapters of the requests beside a shared projection (`lora`).

`own` chooses between the plain torch forms and the library's calls.  Both read the same buffers, laid out as
include/qlinear_b200.h says.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
F32, BF16, F16 = "f32", "bf16", "f16"
TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
BLOCK = 32  # values with one scale in an 8-bit row

# Projections of the decoders that the benchmark and the tests of this repository run: inputs, outputs side by side.
PROJ = {"7b.qkv": (3584, (3584, 512, 512)), "7b.gate_up": (3584, (18944, 18944)), "7b.down": (18944, (3584,)),
        "72b.qkv": (8192, (8192, 1024, 1024)), "72b.o": (8192, (8192,)), "0.5b.qkv": (896, (896, 128, 128)),
        "moe.shared": (2048, (2816, 2816))}


def listed():
    return [
        # one conversation's next token, the row that a projection reads: latency
        dict(name="norm_token", op="norm", rows=1, hidden=3584, type=F32, residual=True, y=True, q8="rows", raw=False),
        # a batch of 64 single tokens, bf16 activations
        dict(name="norm_tokens_64", op="norm", rows=64, hidden=8192, type=BF16, residual=True, y=True, q8="rows", raw=False),
        # chunks of prompts with an odd number of rows, the packed layout, no 32-bit copy of the normed rows
        dict(name="norm_chunk", op="norm", rows=777, hidden=2048, type=F32, residual=True, y=False, q8="mmq", raw=True),
        # a long prompt; its normed rows also go to a router and to adapters
        dict(name="norm_prompt", op="norm", rows=4096, hidden=8192, type=F32, residual=True, y=True, q8="rows", raw=False),
        # one token, 64 experts by softmax (the layer that the grouped experts are tested on): latency
        dict(name="route_token", op="route", tokens=1, experts=64, k=6, score="softmax", bias=False, groups=1, top=1, best=1,
             renorm=False, scale=1.0, ties=False),
        # a batch of single tokens, sigmoid scores, a bias for balance, 4 of 8 groups by their two best
        dict(name="route_tokens_64", op="route", tokens=64, experts=256, k=8, score="sigmoid", bias=True, groups=8, top=4, best=2,
             renorm=True, scale=2.5, ties=False),
        # long prompts of a layer with many small experts, logits from a 16-bit product (equal ones are common)
        dict(name="route_prompt", op="route", tokens=8191, experts=384, k=8, score="softmax", bias=False, groups=1, top=1, best=1,
             renorm=True, scale=1.0, ties=True),
        # long prompts, the grouped choice
        dict(name="route_prompt_groups", op="route", tokens=8192, experts=256, k=8, score="sigmoid", bias=True, groups=8, top=4,
             best=2, renorm=True, scale=2.5, ties=False),
        # one conversation's next token with its adapter on q, k and v: latency
        dict(name="lora_token", op="lora", proj="7b.qkv", type=F16, seqs=1, q=0, adapters=8, max_rank=16, spread=0),
        # a batch of single tokens over 16 adapters of unlike ranks, some rows without one
        dict(name="lora_tokens_64", op="lora", proj="7b.gate_up", type=BF16, seqs=64, q=0, adapters=16, max_rank=64, spread=1),
        # four prompts of unlike, odd lengths, narrow heads, adapters kept in 32 bits
        dict(name="lora_chunks", op="lora", proj="0.5b.qkv", type=F32, seqs=4, q=1021, adapters=3, max_rank=32, spread=1),
        # one long prompt
        dict(name="lora_prompt", op="lora", proj="72b.qkv", type=BF16, seqs=1, q=4096, adapters=4, max_rank=64, spread=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "route", "lora")}
    while True:
        op = rng.choice(["norm", "route", "lora", "lora"])
        if op == "norm":
            q8 = rng.choice(["rows", "rows", "mmq", "none"])
            c = dict(op=op, rows=_log(rng, 1, 8192), hidden=_log(rng, 64, 18944), type=rng.choice([F32, BF16]),
                     residual=rng.random() < 0.8, y=q8 == "none" or rng.random() < 0.6, q8=q8, raw=rng.random() < 0.5)
            if rng.random() < 0.6:
                c["hidden"] = max(64, c["hidden"] // 64 * 64)
        elif op == "route":
            groups = rng.choice([1, 1, 4, 8])
            per = _log(rng, 8, 512) if groups == 1 else _log(rng, 4, 512 // groups)
            top = rng.randint(1, groups)
            c = dict(op=op, tokens=_log(rng, 1, 8192), experts=groups * per, k=rng.randint(1, min(16, top * per)),
                     score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, top=top,
                     best=rng.choice([1, 2]), renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5, 16.0]),
                     ties=rng.random() < 0.3)
        else:
            token = rng.random() < 0.5
            c = dict(op=op, proj=rng.choice(sorted(PROJ)), type=rng.choice([F32, BF16, F16]), seqs=_log(rng, 1, 128 if token else 8),
                     q=0 if token else _log(rng, 2, 4096), adapters=_log(rng, 1, 32), max_rank=rng.choice([8, 16, 32, 64, 128]),
                     spread=rng.randrange(2))
            n_in, outs = PROJ[c["proj"]]
            wide = n_in + sum(outs)
            # what the plain form holds at once: every sequence's adapter in 32 bits, and rows filled up to the longest
            if c["seqs"] * len(outs) * c["max_rank"] * wide > 1 << 28 or c["seqs"] * max(1, c["q"]) * wide > 1 << 28 or \
                    c["adapters"] * len(outs) * c["max_rank"] * wide > 1 << 28:
                continue
        if _cost(c) <= most[op]:
            return c


# ---- sizes -------------------------------------------------------------------------------------------------------

def _lengths(case):
    """Rows of each sequence.  q = 0: one token a sequence."""
    n = case["seqs"]
    if not case["q"]:
        return [1] * n
    return [max(1, int(case["q"] * (1.0 - 0.75 * ((i * 5) % n) / n))) if case["spread"] else case["q"] for i in range(n)]


def _ranks(case):
    r = case["max_rank"]
    return [max(1, (r >> (i % 4)) - (1 if i % 5 == 3 else 0)) if case["spread"] else r for i in range(case["adapters"])]


def _adapters(case):
    """The adapter of each sequence; where they are unlike, every eighth has none."""
    n = case["seqs"]
    return [-1 if case["spread"] and i % 8 == 7 else (i * 7 + 3) % case["adapters"] for i in range(n)]


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        el = 4 if case["type"] == F32 else 2
        b = n * el * (1 + 2 * case["residual"] + case["y"]) + 4 * case["hidden"]
        if case["q8"] != "none":
            b += n * 36 / 32
        return {"bytes": float(b), "flops": 8.0 * n}
    if case["op"] == "route":
        n = case["tokens"]
        return {"bytes": n * (4.0 * case["experts"] + 8.0 * case["k"]), "flops": 8.0 * n * case["experts"]}
    n_in, outs = PROJ[case["proj"]]
    el = 4 if case["type"] == F32 else 2
    ranks, adapter, q = _ranks(case), _adapters(case), _lengths(case)
    rows = sum(q)
    b = 4.0 * rows * (n_in + 2 * sum(outs))
    b += sum(ranks[i] * (len(outs) * n_in + sum(outs)) * el for i in set(adapter) if i >= 0)
    f = sum(2.0 * m * ranks[i] * (len(outs) * n_in + sum(outs)) for m, i in zip(q, adapter) if i >= 0)
    return {"bytes": b, "flops": f}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    s = {"case": dict(case)}

    def randn(*size):
        return torch.randn(*size, generator=g, device=DEV)

    if case["op"] == "norm":
        n, h, dt = case["rows"], case["hidden"], TORCH[case["type"]]
        # a few channels of the residual stream are much larger than the others
        x = randn(n, h)
        r = randn(n, h)
        r[:, ::53] *= 12.0
        s["x"] = x.to(dt)
        if case["residual"]:
            s["residual"] = r.to(dt)
            s["sum"] = torch.empty(n, h, dtype=dt, device=DEV)
        s["gamma"] = 1.0 + 0.2 * randn(h)
        if case["y"]:
            s["y"] = torch.empty(n, h, dtype=dt, device=DEV)
        if case["q8"] != "none":
            nb = (h + BLOCK - 1) // BLOCK
            size = (n, nb, 36) if case["q8"] == "rows" else ((nb + 3) // 4, n, 144)
            s["xq"] = torch.zeros(size, dtype=torch.uint8, device=DEV)
        return s
    if case["op"] == "route":
        n, e, k = case["tokens"], case["experts"], case["k"]
        # some experts are liked more than others by every token
        x = randn(n, e) * 1.5 + randn(e) * 0.7
        s["logits"] = x.bfloat16().float() if case["ties"] else x
        if case["bias"]:
            s["bias"] = 0.05 * randn(e)
        s["idx"] = torch.empty(n, k, dtype=torch.int32, device=DEV)
        s["w"] = torch.empty(n, k, device=DEV)
        return s
    n_in, outs = PROJ[case["proj"]]
    dt, m, r = TORCH[case["type"]], case["adapters"], case["max_rank"]
    q = _lengths(case)
    s["rows"], s["max_q"] = sum(q), max(q)
    s["q_start"] = _i32([sum(q[:i]) for i in range(len(q) + 1)]) if case["q"] else None
    s["adapter"] = _i32(_adapters(case))
    s["rank"] = _i32(_ranks(case))
    s["scale"] = 0.5 + torch.rand(m, generator=g, device=DEV)
    # what stands behind an adapter's last rank is of no meaning (an earlier tenant's)
    s["a"] = [(randn(m, r, n_in) * n_in ** -0.5).to(dt) for _ in outs]
    s["b"] = [(randn(m, o, r) * (0.3 * r ** -0.5)).to(dt) for o in outs]
    s["x"] = randn(s["rows"], n_in)
    s["base"] = randn(s["rows"], sum(outs))
    s["y"] = torch.empty(s["rows"], sum(outs), device=DEV)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _norm_plain(s):
    c = s["case"]
    n, h = s["x"].shape
    v = s["x"].float()
    if c["residual"]:
        v = (v + s["residual"].float()).to(s["x"].dtype)  # what is stored is what is normed
        s["sum"] = v
        v = v.float()
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * s["gamma"]
    if c["y"]:
        s["y"] = y.to(s["x"].dtype)
    if c["q8"] == "none":
        return None
    nb = (h + BLOCK - 1) // BLOCK
    z = torch.zeros(n, nb * BLOCK, device=DEV)
    z[:, :h] = y
    z = z.view(n, nb, BLOCK)
    d = z.abs().amax(-1, keepdim=True) / 127.0
    q = (z / torch.where(d > 0, d, torch.ones_like(d))).round().clamp(-127, 127)
    total = z.sum(-1) if c["raw"] else d[..., 0] * q.sum(-1)
    return {"values": (q * d.half().float()).half(), "sum": total.half()}


def _route_plain(s):
    c = s["case"]
    n, e = s["logits"].shape
    x = s["logits"].double()  # two scores may be near: 64 bits decide
    if c["score"] == "softmax":
        p = (x - x.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    choice = p + s["bias"].double() if c["bias"] else p
    rank = choice if c["bias"] else x
    if c["groups"] > 1:
        per = e // c["groups"]
        best = choice.view(n, c["groups"], per).sort(dim=-1, descending=True)[0][..., :c["best"]].sum(-1)
        taken = best.sort(dim=-1, descending=True, stable=True)[1][:, :c["top"]]
        there = torch.zeros(n, c["groups"], dtype=torch.bool, device=DEV).scatter_(1, taken, True)
        rank = torch.where(there[..., None], rank.view(n, c["groups"], per), torch.full((), -math.inf, device=DEV, dtype=x.dtype))
        rank = rank.view(n, e)
    idx = rank.sort(dim=-1, descending=True, stable=True)[1][:, :c["k"]]  # the lowest id among equals
    w = p.gather(1, idx)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    s["idx"] = idx.to(torch.int32)
    s["w"] = (w * c["scale"]).float()


def _sequences(s):
    """(sequence, place in it) of each row."""
    r = torch.arange(s["rows"], device=DEV)
    if s["q_start"] is None:
        return r, torch.zeros_like(r)
    start = s["q_start"].long()
    seq = torch.searchsorted(start[1:], r, right=True)
    return seq, r - start[seq]


def _lora_plain(s):
    n_in, outs = PROJ[s["case"]["proj"]]
    seq, at = _sequences(s)
    x = torch.zeros(s["case"]["seqs"], s["max_q"], n_in, device=DEV)  # rows filled up to the longest
    x[seq, at] = s["x"]
    i = s["adapter"].clamp(min=0).long()
    used = (torch.arange(s["case"]["max_rank"], device=DEV) < s["rank"][i][:, None]) & (s["adapter"] >= 0)[:, None]
    k = torch.where(used, s["scale"][i][:, None], torch.zeros((), device=DEV))[:, None]
    d = [torch.matmul(torch.matmul(x, a[i].float().transpose(1, 2)) * k, b[i].float().transpose(1, 2)) for a, b in zip(s["a"], s["b"])]
    s["y"] = s["base"] + torch.cat(d, -1)[seq, at]


# ---- a pass --------------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm_own(Q, s):
    c = s["case"]
    n, h = s["x"].shape
    layout = {"none": Q.Q8_NONE, "rows": Q.Q8_ROWS, "mmq": Q.Q8_MMQ}[c["q8"]]
    Q.add_rms_norm(Q.F32 if c["type"] == F32 else Q.BF16, _ptr(s["x"]), h, _ptr(s.get("residual")), h, _ptr(s.get("sum")), h,
                   _ptr(s["gamma"]), 1e-6, _ptr(s.get("y")), h, _ptr(s.get("xq")), layout, c["raw"], n, h)
    if c["q8"] == "none":
        return None
    # the rows as the values that they stand for: scale times code, and the blocks' sums
    nb = (h + BLOCK - 1) // BLOCK
    if c["q8"] == "rows":
        return {"values": s["xq"][..., 4:].view(torch.int8) * s["xq"][..., :2].view(torch.float16),
                "sum": s["xq"][..., 2:4].view(torch.float16)[..., 0]}
    ds = s["xq"][..., :16].view(torch.float16).unflatten(-1, (4, 2))
    q = s["xq"][..., 16:].view(torch.int8).unflatten(-1, (4, BLOCK))
    return {"values": (q * ds[..., :1]).transpose(0, 1).flatten(1, 2)[:, :nb], "sum": ds[..., 1].transpose(0, 1).flatten(1, 2)[:, :nb]}


def _route_own(Q, s):
    c = s["case"]
    n, e = s["logits"].shape
    rule = s.get("rule")
    if rule is None:
        rule = s["rule"] = Q.moe_route_rule(Q.ROUTE_SOFTMAX if c["score"] == "softmax" else Q.ROUTE_SIGMOID, bias=_ptr(s.get("bias")),
                                            n_groups=c["groups"], top_groups=c["top"], group_best=c["best"],
                                            renormalise=c["renorm"], scale=c["scale"])
    Q.moe_route(_ptr(s["logits"]), e, _ptr(s["idx"]), _ptr(s["w"]), n, e, c["k"], rule)


def _lora_own(Q, s):
    c = s["case"]
    n_in, outs = PROJ[c["proj"]]
    pool = s.get("pool")
    if pool is None:
        pool = s["pool"] = Q.lora_pool({F32: Q.F32, BF16: Q.BF16, F16: Q.F16}[c["type"]], [_ptr(t) for t in s["a"]],
                                       [_ptr(t) for t in s["b"]], outs, n_in, c["adapters"], c["max_rank"],
                                       rank=_ptr(s["rank"]), scale=_ptr(s["scale"]))
    Q.lora_add(pool, _ptr(s["x"]), n_in, _ptr(s["base"]), sum(outs), _ptr(s["y"]), sum(outs), _ptr(s["adapter"]), c["seqs"],
               _ptr(s["q_start"]), s["rows"])


def run(state):
    op = state["case"]["op"]
    if own:
        import blog_b200 as Q
        Q.set_stream(torch.cuda.current_stream().cuda_stream)
        q8 = {"norm": _norm_own, "route": _route_own, "lora": _lora_own}[op](Q, state)
    else:
        q8 = {"norm": _norm_plain, "route": _route_plain, "lora": _lora_plain}[op](state)
    if op == "route":
        return {"idx": state["idx"], "w": state["w"]}
    if op == "lora":
        return {"y": state["y"]}
    return {"sum": state.get("sum"), "y": state.get("y"), "q8": q8}


# ---- 64 bits -------------------------------------------------------------------------------------------------------

def _exact_route(case, s):
    """Token by token on the host."""
    x = s["logits"].cpu().numpy().astype(np.float64)
    bias = s["bias"].cpu().numpy().astype(np.float64) if case["bias"] else None
    n, e = x.shape
    k, groups = case["k"], case["groups"]
    w = np.empty((n, k))
    for t in range(n):
        z = np.exp(x[t] - x[t].max())
        p = z / z.sum() if case["score"] == "softmax" else 0.5 * (1.0 + np.tanh(0.5 * x[t]))
        c = p if bias is None else p + bias
        key = x[t] if bias is None else c
        ids = np.arange(e)
        if groups > 1:
            best = np.sort(c.reshape(groups, -1), axis=1)[:, ::-1][:, :case["best"]].sum(1)
            taken = np.lexsort((np.arange(groups), -best))[:case["top"]]
            ids = ids[np.isin(ids // (e // groups), taken)]
        pick = ids[np.lexsort((ids, -key[ids]))[:k]]
        w[t] = p[pick] / (p[pick].sum() if case["renorm"] else 1.0) * case["scale"]
    return {"idx": None, "w": torch.from_numpy(w)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, s)
    if case["op"] == "lora":
        n_in, outs = PROJ[case["proj"]]
        y = s["base"].double()
        row = 0
        for m, i in zip(_lengths(case), _adapters(case)):
            if i >= 0:
                r, col = _ranks(case)[i], 0
                z = s["x"][row:row + m].double()
                for a, b, o in zip(s["a"], s["b"], outs):
                    h = torch.einsum("mk,rk->mr", z, a[i, :r].double())
                    y[row:row + m, col:col + o] += s["scale"][i].double() * torch.einsum("mr,or->mo", h, b[i, :, :r].double())
                    col += o
            row += m
        return {"y": y}
    n, h = case["rows"], case["hidden"]
    v = s["x"].double()
    out = {"sum": None, "y": None, "q8": None}
    if case["residual"]:
        v = v + s["residual"].double()
        out["sum"] = v
        if case["type"] == BF16:
            v = v.to(torch.bfloat16).double()
    y = v / (v.pow(2).sum(-1, keepdim=True) / h + 1e-6).sqrt() * s["gamma"].double()
    if case["y"]:
        out["y"] = y
    if case["q8"] != "none":
        nb = (h + BLOCK - 1) // BLOCK
        z = torch.nn.functional.pad(y, (0, nb * BLOCK - h)).view(n, nb, BLOCK)
        d = z.abs().max(-1).values / 127.0
        q = torch.floor(z / d[..., None].clamp(min=1e-300) + 0.5)
        out["q8"] = {"values": q * d[..., None], "sum": z.sum(-1) if case["raw"] else d * q.sum(-1)}
    return out
