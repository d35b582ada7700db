"""Plain 64-bit restatements of the 8-bit cache's operators (numpy), written from their formulas."""
import numpy as np

BLOCK = 32


def bf16_round(x):
    """f32 values rounded to the nearest bf16 (ties to even), as f32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32)


def rope_table(positions, rotary, theta=10000.0):
    a = np.arange(positions)[:, None] * theta ** (-np.arange(0, rotary, 2) / max(rotary, 1))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def norm_rope(x, gamma, eps, table, pos, rotary):
    """x [heads][hd] in 64 bits."""
    y = x.astype(np.float64)
    if gamma is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)
    if rotary:
        h = rotary // 2
        c, s = table[pos, :h].astype(np.float64), table[pos, h:].astype(np.float64)
        a, b = y[:, :h].copy(), y[:, h:rotary].copy()
        y[:, :h], y[:, h:rotary] = a * c - b * s, b * c + a * s
    return y


def quantize(x):
    """x [32][hd] of one head: (bytes, scale)."""
    x = np.asarray(x, np.float64)
    if not np.isfinite(x).all():
        return np.full(x.shape, 128), np.nan
    scale = np.abs(x).max() / 127.0
    if scale == 0:
        return np.full(x.shape, 128), 0.0
    return np.rint(x / scale).clip(-127, 127) + 128, scale


def attend(q, k, v, pos, scale, gate=None):
    """One row: q [nh][hd], k and v [kvh][keys][hd], the keys 0 .. pos (pos < 0: none)."""
    nh, hd = q.shape
    g = nh // k.shape[0]
    out = np.zeros((nh, hd))
    for h in range(nh):
        if pos >= 0:
            kk, vv = k[h // g, :pos + 1], v[h // g, :pos + 1]
            s = kk @ q[h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[h] = (p @ vv) / p.sum()
    if gate is not None:
        out = out / (1 + np.exp(-gate.astype(np.float64)))
    return out


def logits_rules(x, history=(), prompt_len=0, repetition=None, frequency=0.0, presence=0.0, bias=(), allowed=None):
    """One row, each step rounded to f32 as the rules are defined."""
    f = np.float32
    y = np.array(x, f)
    v = len(y)
    made, seen = {}, set()
    for i, t in enumerate(history):
        if 0 <= t < v:
            seen.add(t)
            if i >= prompt_len:
                made[t] = made.get(t, 0) + 1
    with np.errstate(all="ignore"):
        for t in seen:
            if repetition is not None:
                y[t] = y[t] / f(repetition) if y[t] > 0 else y[t] * f(repetition)
        for t, n in made.items():
            y[t] = y[t] - f(f(frequency) * f(n))
            y[t] = y[t] - f(presence)
        for t, b in bias:
            if 0 <= t < v:
                y[t] = y[t] + f(b)
    if allowed is not None:
        y[~allowed] = -np.inf
    z = np.where(np.isnan(y), -np.inf, y)
    return y, (int(np.argmax(z)) if z.max() > -np.inf else -1)


def attend_rows(q, k, v, pos0, scale, gate=None):
    """Rows q [n][nh][hd] at positions pos0, pos0 + 1, ..; k and v [kvh][keys][hd]."""
    n, nh, hd = q.shape
    g = nh // k.shape[0]
    out = np.zeros((n, nh, hd))
    pos = pos0 + np.arange(n)
    seen = np.arange(k.shape[1])[None] <= pos[:, None]
    for h in range(nh):
        s = q[:, h].astype(np.float64) @ k[h // g].T * scale
        s = np.where(seen, s, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(m), m, 0))
        t = p.sum(1, keepdims=True)
        out[:, h] = p @ v[h // g] / np.where(t > 0, t, 1)
    if gate is not None:
        out = out / (1 + np.exp(-gate.astype(np.float64)))
    return out
