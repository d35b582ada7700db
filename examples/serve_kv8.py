"""Serving with the 8-bit KV cache: ragged prompts, then greedy tokens under rules, one CUDA graph per step.

    python examples/serve_kv8.py [--layers N] [--tokens N]

A small decoder with random-init Q4_K weights (norm - q/k/v - attention - o, norm - SwiGLU - down, LM head).  Per
layer the library's calls are the stacked q/k/v projection with its norm, ql_kv8_append (per-head q/k norms, rotation,
the 8-bit store), ql_kv8_attend, the output projection into the residual, and the SwiGLU pair; ql_logits_apply takes
the token (repetition and presence penalties, a bias, a mask for one of the sequences).  torch allocates memory and
captures the graph.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import blog_b200 as Q  # noqa: E402

DEV = "cuda:0"


class Decoder:
    def __init__(self, layers=4, hidden=1024, ffn=2048, n_heads=8, kv_heads=2, head_dim=128, vocab=8192, seqs=3,
                 max_tokens=512, seed=1):
        self.L, self.H, self.F, self.nh, self.kvh, self.hd, self.V = layers, hidden, ffn, n_heads, kv_heads, head_dim, vocab
        self.n, self.max_tokens = seqs, max_tokens
        self.seed = seed

        def w(rows, cols):
            self.seed += 1
            t = torch.empty(rows, Q.row_bytes(Q.Q4_K, cols), dtype=torch.uint8, device=DEV)
            Q.synth_quantized(Q.Q4_K, self.seed, rows, cols, 1.5 / cols ** 0.5, t.data_ptr())
            return t
        self.wide = (n_heads + 2 * kv_heads) * head_dim
        self.emb, self.head = w(vocab, hidden), w(vocab, hidden)
        self.layers = [dict(q=w(n_heads * head_dim, hidden), k=w(kv_heads * head_dim, hidden),
                            v=w(kv_heads * head_dim, hidden), o=w(hidden, n_heads * head_dim), gate=w(ffn, hidden),
                            up=w(ffn, hidden), down=w(hidden, ffn)) for _ in range(layers)]
        self.ones = torch.ones(hidden, device=DEV)
        self.gamma = torch.ones(head_dim, device=DEV)
        pos = torch.arange(max_tokens, dtype=torch.float64, device=DEV)[:, None]
        ang = pos * 10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=DEV) / head_dim)
        self.rope = torch.cat([ang.cos(), ang.sin()], 1).float()
        # one cache per layer; all layers share the page table (a page number names a page of each)
        per = (max_tokens + 31) // 32
        pages = seqs * per
        self.table = torch.randperm(pages, device=DEV, dtype=torch.int32).view(seqs, per).contiguous()
        self.buffers, self.caches = [], []
        for _ in range(layers):
            codes = [torch.zeros(pages, kv_heads, 32, head_dim, dtype=torch.uint8, device=DEV) for _ in range(2)]
            scales = [torch.zeros(pages, kv_heads, device=DEV) for _ in range(2)]
            opened = [torch.zeros(seqs, 2, kv_heads, 32, head_dim, device=DEV) for _ in range(2)]
            b = codes + scales + opened
            self.buffers.append(b)
            self.caches.append(Q.kv8_cache(*(t.data_ptr() for t in b), self.table.data_ptr(), None, pages, seqs, seqs, per,
                                           kv_heads, head_dim))
        self.kv_len = torch.zeros(seqs, dtype=torch.int32, device=DEV)
        self.ws = torch.zeros(max(Q.kv8_attend_workspace(n_heads, kv_heads, head_dim, seqs, r, q, max_tokens)
                                  for r, q in ((seqs, 1), (seqs * max_tokens, max_tokens))), dtype=torch.uint8, device=DEV)

    def forward(self, ids, q_start=None, max_q=1, last=None):
        """ids [rows] int32 on the device; kv_len already counts them.  The logits of rows `last` (all by default)."""
        m, H, hd = ids.numel(), self.H, self.hd
        p = lambda t: t.data_ptr()  # noqa: E731
        rb = lambda c: Q.row_bytes(Q.Q4_K, c)  # noqa: E731
        x = torch.empty(m, H, device=DEV)
        Q.quant_embedding(Q.Q4_K, p(ids), p(x), p(self.emb), rb(H), H, m)
        qkv = torch.empty(m, self.wide, device=DEV)
        attn = torch.empty(m, self.nh * hd, device=DEV)
        act = torch.empty(m, self.F, device=DEV)
        for w, cache in zip(self.layers, self.caches):
            Q.quant_gemv_stacked_ex(Q.Q4_K, [p(w["q"]), p(w["k"]), p(w["v"])], [rb(H)] * 3,
                                    [self.nh * hd, self.kvh * hd, self.kvh * hd], p(x), H, p(qkv), self.wide, H, m,
                                    p(self.ones), 1e-6)
            q, k, v = (p(qkv) + 4 * hd * i for i in (0, self.nh, self.nh + self.kvh))
            Q.kv8_append(cache, Q.F32, q, self.wide, k, self.wide, v, self.wide, q, self.wide, self.nh, p(self.gamma),
                         p(self.gamma), 1e-6, p(self.rope), hd, self.max_tokens, p(self.kv_len),
                         None if q_start is None else p(q_start), m, max_q)
            Q.kv8_attend(cache, Q.F32, q, self.wide, None, 0, p(attn), self.nh * hd, self.nh, hd ** -0.5, p(self.kv_len),
                         None if q_start is None else p(q_start), m, max_q, self.max_tokens, p(self.ws), self.ws.numel())
            Q.quant_gemv_ex(Q.Q4_K, p(w["o"]), rb(self.nh * hd), p(attn), self.nh * hd, p(x), H, H, self.nh * hd, m,
                            accumulate=True)
            Q.quant_swiglu_ex(Q.Q4_K, p(w["gate"]), p(w["up"]), rb(H), rb(H), p(x), H, p(act), self.F, self.F, H, m,
                              p(self.ones), 1e-6)
            Q.quant_gemv_ex(Q.Q4_K, p(w["down"]), rb(self.F), p(act), self.F, p(x), H, H, self.F, m, accumulate=True)
        if last is not None:
            x = x[last].contiguous()
        logits = torch.empty(x.shape[0], self.V, device=DEV)
        Q.quant_gemv_ex(Q.Q4_K, p(self.head), rb(H), p(x), H, p(logits), self.V, self.V, H, x.shape[0], p(self.ones), 1e-6)
        return logits


def check_request(lens, steps, seqs, max_tokens):
    """Raises ValueError for prompts of `lens` tokens and `steps` new ones that a Decoder's cache does not hold."""
    if len(lens) != seqs or min(lens, default=0) < 1:
        raise ValueError("need %d prompts of at least one token each" % seqs)
    if steps < 2:
        raise ValueError("need at least 2 tokens: the prompts' and one step's")
    if max(lens) + steps - 1 > max_tokens:  # (the last token's key is never stored)
        raise ValueError("%d prompt tokens and %d new ones do not fit a cache of %d" % (max(lens), steps, max_tokens))


def generate(model, prompts, steps):
    """Greedy tokens [sequences][steps] after the prompts (lists of ids), the logits of the last step, us per
    replayed step (None: there was none)."""
    n, V = model.n, model.V
    lens = [len(q) for q in prompts]
    check_request(lens, steps, n, model.max_tokens)
    room = max(lens) + steps
    history = torch.zeros(n, room, dtype=torch.int32, device=DEV)
    for i, q in enumerate(prompts):
        history[i, :lens[i]] = torch.tensor(q, dtype=torch.int32)
    h_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    p_len = h_len.clone()
    full = lambda v: torch.full((n,), v, device=DEV)  # noqa: E731
    rep, pres = full(1.1), full(0.2)
    allowed = torch.full((1, V // 32), -1, dtype=torch.int32, device=DEV)  # the first sequence: ids below V / 2 alone
    allowed[:, V // 64:] = 0
    mask_row = torch.tensor([0] + [-1] * (n - 1), dtype=torch.int32, device=DEV)
    bias_ids = torch.tensor([7], dtype=torch.int32, device=DEV)
    bias = torch.tensor([-100.0], device=DEV)  # the last sequence never says 7
    b_start = torch.tensor([0] * n + [1], dtype=torch.int32, device=DEV)
    p = lambda t: t.data_ptr()  # noqa: E731
    rules = Q.logits_rules(history=p(history), history_stride=room, history_len=p(h_len), prompt_len=p(p_len),
                           repetition=p(rep), presence=p(pres), bias_ids=p(bias_ids), bias_values=p(bias),
                           bias_start=p(b_start), mask=p(allowed), mask_stride=V // 32, mask_rows=1, mask_row=p(mask_row))
    token = torch.zeros(n, dtype=torch.int32, device=DEV)
    lws = torch.zeros(16 * n, dtype=torch.uint8, device=DEV)

    def take(logits):  # in place: the rules, the token, its place in the history
        Q.logits_apply(p(logits), V, p(logits), V, n, V, rules, p(token), p(lws), lws.numel())
        history.scatter_(1, h_len.long()[:, None], token[:, None])
        h_len.add_(1)

    # the prompts, all at once
    starts = [0]
    for k in lens:
        starts.append(starts[-1] + k)
    ids = torch.tensor([t for q in prompts for t in q], dtype=torch.int32, device=DEV)
    q_start = torch.tensor(starts, dtype=torch.int32, device=DEV)
    model.kv_len.copy_(h_len)
    take(model.forward(ids, q_start, max(lens), last=torch.tensor([s - 1 for s in starts[1:]], device=DEV)))

    def step():
        model.kv_len.add_(1)
        logits = model.forward(token)
        raw = logits.clone()
        take(logits)
        return raw

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    before = Q.lib().ql_get_stream()
    try:
        with torch.cuda.stream(stream):
            Q.set_stream(stream.cuda_stream)
            raw = step()  # sizes every workspace before the capture
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                raw = step()
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record(stream)
            for _ in range(steps - 2):  # (history has room for these and no more)
                graph.replay()
            end.record(stream)
        torch.cuda.synchronize()
    finally:
        Q.set_stream(before)
    Q.check_device()
    out = [history[i, lens[i]:lens[i] + steps].tolist() for i in range(n)]
    return out, raw, start.elapsed_time(end) * 1e3 / (steps - 2) if steps > 2 else None


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=64, help="new tokens per sequence (at least 2)")
    a = ap.parse_args()
    Q.init(0)
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    model = Decoder(layers=a.layers, max_tokens=max(512, 100 + a.tokens))
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, model.V, (k,), generator=g).tolist() for k in (100, 33, 7)]
    out, _, us = generate(model, prompts, a.tokens)
    for i, t in enumerate(out):
        print("sequence %d (%d prompt tokens): %s ..." % (i, len(prompts[i]), t[:12]))
    if us is not None:
        print("%.0f us per step of %d sequences, %d layers" % (us, model.n, a.layers))


if __name__ == "__main__":
    main()
