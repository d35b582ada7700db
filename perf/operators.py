"""Cases for the serving operators around the 8-bit KV cache: the append (norms and rotation of q and k, the block
quantised store), the attention that reads the cache, and the logits rules (penalties, biases, masks, greedy token).

`own` chooses between the plain torch forms and the library's calls.  Both read the same buffers: the cache as
include/qlinear_b200.h lays it out (pages of 32 tokens, codes + 128 in bytes, one f32 scale for each page and KV head,
the rows of the unfinished block in f32).
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32
DEV = "cuda:0"
F32, BF16 = "f32", "bf16"
TORCH = {F32: torch.float32, BF16: torch.bfloat16}

# Head layouts of the decoders that the benchmark and the tests of this repository run: query heads, KV heads, head
# dimension, rotated dimensions.
HEADS = {"7b": (28, 4, 128, 128), "72b": (64, 8, 128, 128), "0.5b": (14, 2, 64, 64), "hybrid": (16, 4, 256, 64)}


def listed():
    return [
        # one new token of one conversation: a launch's latency
        dict(name="append_token", op="append", heads="7b", type=F32, seqs=1, q=0, past=1000, spread=0),
        # one new token of each of 64 conversations, gated hybrid layout (partial rotation), bf16 activations
        dict(name="append_tokens_64", op="append", heads="hybrid", type=BF16, seqs=64, q=0, past=2048, spread=1),
        # one long prompt
        dict(name="append_prompt", op="append", heads="7b", type=F32, seqs=1, q=4096, past=0, spread=0),
        # eight prompts of unlike lengths, each a later chunk of its conversation
        dict(name="append_prompts_8", op="append", heads="72b", type=BF16, seqs=8, q=1500, past=1024, spread=1),
        # one conversation's next token early on: latency
        dict(name="decode_short", op="attend", heads="7b", type=F32, seqs=1, q=0, past=200, spread=0, gate=False),
        # one long document's next token: the cache of one sequence over the whole GPU
        dict(name="decode_long", op="attend", heads="7b", type=F32, seqs=1, q=0, past=32767, spread=0, gate=False),
        # a full batch of unlike lengths, gated
        dict(name="decode_batch", op="attend", heads="72b", type=BF16, seqs=64, q=0, past=8192, spread=1, gate=True),
        # a prompt of ordinary length, f32 as the engine's activations are
        dict(name="prompt", op="attend", heads="7b", type=F32, seqs=1, q=2048, past=0, spread=0, gate=False),
        # a long prompt in bf16
        dict(name="prompt_long", op="attend", heads="7b", type=BF16, seqs=1, q=8192, past=0, spread=0, gate=False),
        # later chunks of four conversations, narrow heads, odd sizes
        dict(name="prompt_chunks", op="attend", heads="0.5b", type=BF16, seqs=4, q=1021, past=1536, spread=1, gate=False),
        # one row, short history: what a single conversation pays before its token
        dict(name="logits_one", op="logits", rows=1, vocab=32001, history=200, bias=16, mask=True, spread=0),
        # a serving batch: unlike histories, half the rows under a grammar
        dict(name="logits_batch", op="logits", rows=64, vocab=152064, history=4096, bias=300, mask=True, spread=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed() if c["op"] != "logits")
    while True:
        op = rng.choice(["append", "attend", "attend", "logits"])
        if op == "logits":
            c = dict(op=op, rows=_log(rng, 1, 128), vocab=_log(rng, 1000, 160000), history=_log(rng, 1, 8192),
                     bias=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.6, spread=rng.randrange(2))
            if c["rows"] * c["vocab"] > 64 * 152064:
                continue
        else:
            heads = rng.choice(sorted(HEADS))
            token = rng.random() < 0.5
            c = dict(op=op, heads=heads, type=rng.choice([F32, BF16]), seqs=_log(rng, 1, 64 if token else 8),
                     q=0 if token else _log(rng, 2, 8192), past=_log(rng, 1, 32768) - 1, spread=rng.randrange(2))
            if not token:
                c["past"] = c["past"] // 4 // BLOCK * BLOCK
            if op == "attend":
                c["gate"] = rng.random() < 0.3
            # what the plain forms hold at once: scores, and the cache in 32 bits
            nh, kvh, hd, _ = HEADS[heads]
            keys = c["past"] + max(1, c["q"])
            if c["seqs"] * nh * max(1, c["q"]) * keys > 28 * 8192 * 8192 or c["seqs"] * keys * kvh * hd > 64 * 8192 * 8 * 128:
                continue
        if _cost(c) <= most and 3072 not in c.values():
            return c


# ---- sizes -------------------------------------------------------------------------------------------------------

def _lengths(case):
    """(tokens of this call, tokens in the cache after it) for each sequence.  q = 0: one token a sequence."""
    n = case["seqs"]
    q, past = [], []
    for i in range(n):
        part = 1.0 if not case["spread"] or n == 1 else 1.0 - 0.75 * ((i * 7) % n) / n
        q.append(max(1, int(case["q"] * part)) if case["q"] else 1)
        p = int(case["past"] * part)
        past.append(p // BLOCK * BLOCK if case["q"] else p)
    return q, [a + b for a, b in zip(past, q)]


def _histories(case):
    n = case["rows"]
    return [case["history"] if not case["spread"] or n == 1 else case["history"] * ((i * 5) % n + 1) // n for i in range(n)]


def work(case):
    if case["op"] == "logits":
        n, v = case["rows"], case["vocab"]
        b = 8.0 * n * v + 4.0 * sum(_histories(case)) + 8.0 * n * case["bias"]
        if case["mask"]:
            b += n * v / 16.0  # half the rows have a mask
        return {"bytes": b, "flops": 4.0 * n * v}
    nh, kvh, hd, _ = HEADS[case["heads"]]
    el = 4 if case["type"] == F32 else 2
    q, kv = _lengths(case)
    if case["op"] == "append":
        b = f = 0.0
        for a, t in zip(q, kv):
            full = t // BLOCK * BLOCK - (t - a) // BLOCK * BLOCK  # tokens of blocks that this call fills
            b += a * ((2 * nh + 2 * kvh) * hd * el)                # q, k, v in, q out
            b += 2 * kvh * hd * (full * 1.0 + min(a, t % BLOCK) * 4)  # codes and open rows out
            b += 2 * kvh * hd * 4 * max(0, full - a)               # earlier open rows of a block that fills
            b += 2 * kvh * hd * 2 * (t - (t - a) // BLOCK * BLOCK)    # the touched rows read back in bf16
            f += a * (nh + kvh) * hd * 8.0
        return {"bytes": b, "flops": f}
    b = f = 0.0
    for a, t in zip(q, kv):
        b += 2 * kvh * hd * (t // BLOCK * BLOCK * 1.0 + t % BLOCK * 4) + a * nh * hd * el * (3 if case["gate"] else 2)
        f += 4.0 * nh * hd * (a * (t - a) + a * (a + 1) / 2)
    return {"bytes": b, "flops": f}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(case, g, filled):
    """A cache whose pages lie in a shuffled order.  filled: earlier tokens are there, codes as a quantiser leaves them
    (near normal, the largest of a block +-127), scales of unlike sizes."""
    nh, kvh, hd, _ = HEADS[case["heads"]]
    n = case["seqs"]
    _, kv = _lengths(case)
    per = max((t + BLOCK - 1) // BLOCK for t in kv)
    used = [(t + BLOCK - 1) // BLOCK for t in kv]
    pages = sum(used)
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
    table = torch.zeros(n, per, dtype=torch.int32, device=DEV)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u

    def codes():
        c = torch.empty(pages, kvh, BLOCK, hd, dtype=torch.uint8, device=DEV)
        if filled:
            for lo in range(0, pages, 4096):
                x = torch.randn(c[lo:lo + 4096].shape, generator=g, device=DEV).mul_(36.0).round_().clamp_(-127, 127)
                x[:, :, 0, 0] = 127.0
                c[lo:lo + 4096] = (x + 128.0).to(torch.uint8)
        else:
            c.fill_(128)
        return c

    def scales(size):
        u = torch.rand(pages, kvh, generator=g, device=DEV)
        return torch.exp((u - 0.5) * 1.4) * (size / 36.0) if filled else torch.zeros(pages, kvh, device=DEV)

    kc, vc = codes(), codes()
    ko, vo = (torch.randn(n, 2, kvh, BLOCK, hd, generator=g, device=DEV) for _ in range(2))
    return dict(k_codes=kc, v_codes=vc, k_scale=scales(1.0), v_scale=scales(0.5), k_open=ko, v_open=vo, table=table)


def _ragged(case):
    q, kv = _lengths(case)
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    return int(start[-1]), max(q), max(kv), _i32(start) if case["q"] else None, _i32(kv)


def _rope_table(positions, rotary, theta=1e6):
    """[positions][rotary]: the cosines of a position's rotary / 2 angles, then the sines."""
    inv = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    if case["op"] == "logits":
        n, v = case["rows"], case["vocab"]
        lens = _histories(case)
        s["logits"] = torch.randn(n, v, generator=g, device=DEV) * 3.0
        # text repeats itself: ids near a power law
        u = torch.rand(n, max(1, max(lens)), generator=g, device=DEV)
        s["history"] = (torch.exp(u * math.log(v + 1.0)).long() - 1).clamp(0, v - 1).to(torch.int32)
        s["history_len"] = _i32(lens)
        s["prompt_len"] = _i32([h // 3 for h in lens])
        s["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=g, device=DEV)
        s["frequency"] = 0.2 * torch.rand(n, generator=g, device=DEV)
        s["presence"] = 0.5 * torch.rand(n, generator=g, device=DEV)
        if case["bias"]:
            m = min(case["bias"], v)
            s["bias_ids"] = torch.cat([torch.randperm(v, generator=g, device=DEV)[:m] for _ in range(n)]).to(torch.int32)
            s["bias_values"] = torch.randn(n * m, generator=g, device=DEV) * 4.0
            s["bias_start"] = _i32([i * m for i in range(n + 1)])
        if case["mask"]:  # the first half of the rows: a state of the grammar allows few tokens, or many
            m = max(1, n // 2)
            words = (v + 31) // 32
            w = torch.randint(-2 ** 31, 2 ** 31, (m, words), generator=g, device=DEV, dtype=torch.int64)
            w2 = torch.randint(-2 ** 31, 2 ** 31, (m, words), generator=g, device=DEV, dtype=torch.int64)
            few = (torch.arange(m, device=DEV) % 2 == 0)[:, None]
            s["mask"] = torch.where(few, w & w2 & w2.roll(1, 1) & w.roll(1, 1), w).to(torch.int32)
            s["mask_row"] = _i32([i if i < m else -1 for i in range(n)])
        s["out"] = torch.empty(n, v, device=DEV)
        s["token"] = torch.empty(n, dtype=torch.int32, device=DEV)
        s["workspace"] = torch.zeros(16 * n, dtype=torch.uint8, device=DEV)
        return s
    nh, kvh, hd, rot = HEADS[case["heads"]]
    dt = TORCH[case["type"]]
    rows, max_q, max_kv, start, kv = _ragged(case)
    s.update(rows=rows, max_q=max_q, max_kv=max_kv, q_start=start, kv_len=kv, cache=_cache(case, g, case["op"] == "attend"))
    if case["op"] == "append":
        # one projection's stacked output: q, k and v of a token side by side, a few channels of k much larger
        x = torch.randn(rows, (nh + 2 * kvh) * hd, generator=g, device=DEV)
        x[:, nh * hd:(nh + kvh) * hd:17] *= 6.0
        s["x"] = x.to(dt)
        s["q_gamma"] = 1.0 + 0.2 * torch.randn(hd, generator=g, device=DEV)
        s["k_gamma"] = 1.0 + 0.2 * torch.randn(hd, generator=g, device=DEV)
        s["rope"] = _rope_table(max_kv, rot)
        s["q_out"] = torch.empty(rows, nh * hd, dtype=dt, device=DEV)
        # the rows that the call touches, whole blocks of them, read back
        q, t = _lengths(case)
        first = [(b - a) // BLOCK * BLOCK for a, b in zip(q, t)]
        s["count"] = max(b - f for b, f in zip(t, first))
        s["first"] = _i32(first)
        s["rows_out"] = [torch.empty(case["seqs"], s["count"], kvh, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        return s
    s["q"] = (torch.randn(rows, nh * hd, generator=g, device=DEV) * 1.5).to(dt)
    if case["gate"]:
        s["gate"] = torch.randn(rows, nh * hd, generator=g, device=DEV).to(dt)
    s["out"] = torch.empty(rows, nh * hd, dtype=dt, device=DEV)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _norm_rope(x, gamma, eps, cos, sin):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * gamma
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _positions(s, device_rows):
    """(sequence, position) of each row of the call."""
    kv = s["kv_len"].long()
    if s["q_start"] is None:
        return torch.arange(device_rows, device=DEV), kv - 1
    start = s["q_start"].long()
    r = torch.arange(device_rows, device=DEV)
    seq = torch.searchsorted(start[1:], r, right=True)
    return seq, kv[seq] - (start[seq + 1] - r)


def _plain_rows(codes, scale, opened, table, kv, first, count):
    """[sequences][count][KV heads][head dim]: positions first .. first + count - 1 of each sequence, 0 past its end."""
    n = table.shape[0]
    pos = first[:, None] + torch.arange(count, device=DEV)
    there = pos < kv[:, None]
    page = table.long().gather(1, (pos // BLOCK).clamp(max=table.shape[1] - 1))
    x = (codes.permute(0, 2, 1, 3)[page, pos % BLOCK].float() - 128.0) * scale[page][..., None]
    block = kv // BLOCK
    o = opened[torch.arange(n, device=DEV), block % 2].transpose(1, 2)  # [n][32][KV heads][hd]
    o = o[torch.arange(n, device=DEV)[:, None], pos % BLOCK]
    x = torch.where((pos // BLOCK == block[:, None])[..., None, None], o, x)
    return torch.where(there[..., None, None], x, torch.zeros((), device=DEV))


def _append_plain(s):
    c = s["cache"]
    nh, kvh, hd, rot = HEADS[s["case"]["heads"]]
    rows = s["rows"]
    x = s["x"].float().view(rows, nh + 2 * kvh, hd)
    seq, pos = _positions(s, rows)
    table = s["rope"][pos]
    cos, sin = table[:, None, :rot // 2], table[:, None, rot // 2:]
    q = _norm_rope(x[:, :nh], s["q_gamma"], 1e-6, cos, sin)
    k = _norm_rope(x[:, nh:nh + kvh], s["k_gamma"], 1e-6, cos, sin)
    v = x[:, nh + kvh:]
    s["q_out"].copy_(q.view(rows, nh * hd))
    kv, first, count = s["kv_len"].long(), s["first"].long(), s["count"]
    blocks = (count + BLOCK - 1) // BLOCK
    n = kv.shape[0]
    at = pos - first[seq]
    b = first[:, None] // BLOCK + torch.arange(blocks, device=DEV)  # blocks that the call touches
    full = (b + 1) * BLOCK <= kv[:, None]
    page = c["table"].long().gather(1, b.clamp(max=c["table"].shape[1] - 1))
    last = (kv - 1) // BLOCK
    ns = torch.arange(n, device=DEV)
    for new, codes, scale, opened in ((k, "k_codes", "k_scale", "k_open"), (v, "v_codes", "v_scale", "v_open")):
        y = torch.zeros(n, blocks * BLOCK, kvh, hd, device=DEV)
        y[:, :BLOCK] = c[opened][ns, (first // BLOCK) % 2].transpose(1, 2)  # earlier rows of the first block
        y[seq, at] = new
        y = y.view(n, blocks, BLOCK, kvh, hd).transpose(2, 3)  # [n][blocks][KV heads][32][hd]
        sc = y.abs().amax((-1, -2)) / 127.0
        z = torch.where(sc > 0, sc, torch.ones_like(sc))[..., None, None]
        code = torch.where((sc > 0)[..., None, None], (y / z).round().clamp(-127, 127), torch.zeros((), device=DEV)) + 128.0
        c[codes][page[full]] = code[full].to(torch.uint8)
        c[scale][page[full]] = sc[full]
        # the rows of the last block, and of the one before it
        for back in (1, 0):
            i = last - back - first // BLOCK
            ok = (i >= 0) if back == 0 else (i >= 0) & (last > 0)
            w = ns[ok]
            c[opened][w, (last[ok] - back) % 2] = torch.where(
                (torch.arange(BLOCK, device=DEV) + (last[ok] - back)[:, None] * BLOCK < kv[ok, None])[:, None, :, None],
                y[w, i[ok]], c[opened][w, (last[ok] - back) % 2])
    for out, codes, scale, opened in zip(s["rows_out"], ("k_codes", "v_codes"), ("k_scale", "v_scale"), ("k_open", "v_open")):
        out.copy_(_plain_rows(c[codes], c[scale], c[opened], c["table"], kv, first, count))


def _attend_plain(s):
    c = s["cache"]
    nh, kvh, hd, _ = HEADS[s["case"]["heads"]]
    rows, n, g = s["rows"], s["kv_len"].shape[0], nh // kvh
    kv = s["kv_len"].long()
    zero = torch.zeros_like(kv)
    k, v = (_plain_rows(c[x + "_codes"], c[x + "_scale"], c[x + "_open"], c["table"], kv, zero, s["max_kv"]).transpose(1, 2)
            for x in "kv")  # [n][KV heads][keys][hd]
    seq, pos = _positions(s, rows)
    mq = s["max_q"]
    at = pos - (kv - mq)[seq]  # rows lie at the end of a padded window
    q = torch.zeros(n, mq, nh, hd, device=DEV)
    q[seq, at] = s["q"].float().view(rows, nh, hd)
    q = q.view(n, mq, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * mq, hd)
    sc = torch.matmul(q, k.transpose(-1, -2)).mul_(hd ** -0.5).view(n, kvh, g, mq, -1)
    qpos = kv[:, None] - mq + torch.arange(mq, device=DEV)
    seen = torch.arange(sc.shape[-1], device=DEV) <= qpos[:, :, None]  # [n][mq][keys]
    sc.masked_fill_(~seen[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kvh, g * mq, -1), v).view(n, kvh, g, mq, hd) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(n, mq, nh * hd)[seq, at]
    if "gate" in s:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    s["out"].copy_(o)


def _logits_plain(s):
    x = s["logits"]
    n, v = x.shape
    h = s["history"].long()
    i = torch.arange(h.shape[1], device=DEV)
    there = i < s["history_len"][:, None]
    out = there & (i >= s["prompt_len"][:, None])
    seen = torch.zeros(n, v, device=DEV).scatter_add_(1, h, there.float())
    count = torch.zeros(n, v, device=DEV).scatter_add_(1, h, out.float())
    r = s["repetition"][:, None]
    y = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    y = y - s["frequency"][:, None] * count
    y = y - s["presence"][:, None] * (count > 0).float()
    if "bias_ids" in s:
        m = s["bias_ids"].shape[0] // n
        y = y.scatter_add(1, s["bias_ids"].long().view(n, m), s["bias_values"].view(n, m))
    if "mask" in s:
        t = torch.arange(v, device=DEV)
        bits = (s["mask"][s["mask_row"].clamp(min=0).long()][:, t // 32] >> (t % 32)) & 1
        y = torch.where((bits == 0) & (s["mask_row"] >= 0)[:, None], torch.full((), -math.inf, device=DEV), y)
    s["out"].copy_(y)
    best = y.amax(1, keepdim=True)
    first = torch.where(y == best, torch.arange(v, device=DEV), v).amin(1)
    s["token"].copy_(torch.where(best[:, 0] > -math.inf, first, -1))


# ---- a pass --------------------------------------------------------------------------------------------------------

def _own(s):
    import blog_b200 as Q
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if s["case"]["op"] == "logits":
        n, v = s["logits"].shape
        rules = Q.logits_rules(
            history=p(s["history"]), history_stride=s["history"].shape[1], history_len=p(s["history_len"]),
            prompt_len=p(s["prompt_len"]), repetition=p(s["repetition"]), frequency=p(s["frequency"]),
            presence=p(s["presence"]), bias_ids=p(s.get("bias_ids")), bias_values=p(s.get("bias_values")),
            bias_start=p(s.get("bias_start")), mask=p(s.get("mask")),
            mask_stride=s["mask"].shape[1] if "mask" in s else 0, mask_rows=s["mask"].shape[0] if "mask" in s else 0,
            mask_row=p(s.get("mask_row")))
        Q.logits_apply(p(s["logits"]), v, p(s["out"]), v, n, v, rules, p(s["token"]), p(s["workspace"]),
                       s["workspace"].numel())
        return
    c = s["cache"]
    nh, kvh, hd, rot = HEADS[s["case"]["heads"]]
    t = Q.F32 if s["case"]["type"] == F32 else Q.BF16
    n, per = c["table"].shape
    cache = Q.kv8_cache(p(c["k_codes"]), p(c["v_codes"]), p(c["k_scale"]), p(c["v_scale"]), p(c["k_open"]), p(c["v_open"]),
                        p(c["table"]), None, c["k_codes"].shape[0], n, n, per, kvh, hd)
    if s["case"]["op"] == "append":
        w, el = (nh + 2 * kvh) * hd, s["x"].element_size()
        x = p(s["x"])
        Q.kv8_append(cache, t, x, w, x + nh * hd * el, w, x + (nh + kvh) * hd * el, w, p(s["q_out"]), nh * hd, nh,
                     p(s["q_gamma"]), p(s["k_gamma"]), 1e-6, p(s["rope"]), rot, s["rope"].shape[0], p(s["kv_len"]),
                     p(s["q_start"]), s["rows"], s["max_q"])
        Q.kv8_gather(cache, Q.BF16, p(s["rows_out"][0]), p(s["rows_out"][1]), p(s["first"]), s["count"], p(s["kv_len"]))
        return
    if "workspace" not in s:  # kept by the caller, zero before its first use
        s["workspace"] = torch.zeros(Q.kv8_attend_workspace(nh, kvh, hd, n, s["rows"], s["max_q"], s["max_kv"]),
                                     dtype=torch.uint8, device=DEV)
    Q.kv8_attend(cache, t, p(s["q"]), nh * hd, p(s.get("gate")), nh * hd, p(s["out"]), nh * hd, nh, hd ** -0.5,
                 p(s["kv_len"]), p(s["q_start"]), s["rows"], s["max_q"], s["max_kv"], p(s["workspace"]),
                 s["workspace"].numel())


def run(state):
    op = state["case"]["op"]
    if own:
        _own(state)
    else:
        {"append": _append_plain, "attend": _attend_plain, "logits": _logits_plain}[op](state)
    if op == "logits":
        return {"logits": state["out"], "token": state["token"]}
    if op == "attend":
        return {"out": state["out"]}
    c = state["cache"]
    return {"q": state["q_out"], "k": state["rows_out"][0], "v": state["rows_out"][1], "k_scale": c["k_scale"],
            "v_scale": c["v_scale"]}


# ---- 64 bits -------------------------------------------------------------------------------------------------------

def _exact_rows(c, which, i, table, t):
    """The t rows of sequence i as they stand in the cache: [t][KV heads][hd]."""
    full = t // BLOCK
    parts = []
    if full:
        pg = table[i, :full].long()
        x = (c[which + "_codes"][pg].double() - 128.0) * c[which + "_scale"][pg].double()[..., None, None]
        parts.append(x.transpose(1, 2).reshape(full * BLOCK, *x.shape[1:2], x.shape[-1]))
    if t % BLOCK:
        parts.append(c[which + "_open"][i, full % 2, :, :t % BLOCK].double().transpose(0, 1))
    return torch.cat(parts)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        n, v = case["rows"], case["vocab"]
        y = s["logits"].double()
        lens, pl = s["history_len"].tolist(), s["prompt_len"].tolist()
        for r in range(n):
            h = s["history"][r, :lens[r]].long()
            seen = torch.bincount(h, minlength=v) > 0
            made = torch.bincount(h[pl[r]:], minlength=v).double()
            rep = s["repetition"][r].double()
            y[r] = torch.where(seen & (y[r] > 0), y[r] / rep, torch.where(seen, y[r] * rep, y[r]))
            y[r] -= s["frequency"][r].double() * made + s["presence"][r].double() * (made > 0)
            if "bias_ids" in s:
                a, b = s["bias_start"][r:r + 2].tolist()
                y[r].index_add_(0, s["bias_ids"][a:b].long(), s["bias_values"][a:b].double())
            if "mask" in s and int(s["mask_row"][r]) >= 0:
                w = s["mask"][int(s["mask_row"][r])].cpu().numpy().view(np.uint8)
                allowed = np.unpackbits(w, bitorder="little")[:v].astype(bool)
                y[r][~torch.from_numpy(allowed).to(DEV)] = -math.inf
        return {"logits": y, "token": None}
    nh, kvh, hd, rot = HEADS[case["heads"]]
    q_len, kv_len = _lengths(case)
    c = s["cache"]
    rows, at = s["rows"], np.concatenate([[0], np.cumsum(q_len)])
    if case["op"] == "append":
        x = s["x"].double().view(rows, nh + 2 * kvh, hd)
        q_out = torch.empty(rows, nh, hd, dtype=torch.float64, device=DEV)
        outs = [torch.zeros(case["seqs"], s["count"], kvh, hd, dtype=torch.float64, device=DEV) for _ in range(2)]
        scales = [c["k_scale"].double().clone(), c["v_scale"].double().clone()]
        for i, (a, t) in enumerate(zip(q_len, kv_len)):
            z = x[at[i]:at[i + 1]]
            ang = s["rope"][t - a:t].double()
            turn = torch.complex(ang[:, :rot // 2], ang[:, rot // 2:])[:, None]
            new = []
            for part, gamma in ((z[:, :nh], "q_gamma"), (z[:, nh:nh + kvh], "k_gamma")):
                y = part / (part.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * s[gamma].double()
                w = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
                new.append(torch.cat([w.real, w.imag, y[..., rot:]], -1))
            q_out[at[i]:at[i + 1]] = new[0]
            first = (t - a) // BLOCK * BLOCK
            for j, (which, y) in enumerate((("k", new[1]), ("v", z[:, nh + kvh:]))):
                old = c[which + "_open"][i, (first // BLOCK) % 2, :, :(t - a) - first].double().transpose(0, 1)
                y = torch.cat([old, y])
                full = y.shape[0] // BLOCK
                if full:
                    b = y[:full * BLOCK].view(full, BLOCK, kvh, hd)
                    sc = b.abs().amax((1, 3)) / 127.0
                    pg = c["table"][i, first // BLOCK:first // BLOCK + full].long()
                    scales[j][pg] = sc
                    y[:full * BLOCK] = ((b / sc[:, None, :, None]).round() * sc[:, None, :, None]).view(full * BLOCK, kvh, hd)
                outs[j][i, :t - first] = y
        return {"q": q_out.view(rows, nh * hd), "k": outs[0], "v": outs[1], "k_scale": scales[0], "v_scale": scales[1]}
    out = torch.empty(rows, nh, hd, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(rows, nh, hd)
    for i, (a, t) in enumerate(zip(q_len, kv_len)):
        k, v = (_exact_rows(c, w, i, c["table"], t) for w in "kv")
        for lo in range(0, a, 1024):
            m = min(1024, a - lo)
            qs = q[at[i] + lo:at[i] + lo + m]
            qpos = t - a + lo + torch.arange(m, device=DEV)
            hide = torch.arange(t, device=DEV)[None] > qpos[:, None]
            for h in range(nh):
                w = torch.softmax((qs[:, h] @ k[:, h // (nh // kvh)].T / math.sqrt(hd)).masked_fill(hide, -math.inf), -1)
                out[at[i] + lo:at[i] + lo + m, h] = w @ v[:, h // (nh // kvh)]
    out = out.view(rows, nh * hd)
    if "gate" in s:
        out = out * torch.sigmoid(s["gate"].double())
    return {"out": out}
