"""The choice of experts by score, bias and group, against the definition in 64 bits."""
import numpy as np
import pytest

import blog_b200 as Q

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -18  # of the token's largest score, times scale (twice that where the weights are renormalised)


def _reference(x, k, sigmoid, bias=None, groups=1, top=1, best=1, renorm=False, scale=1.0):
    x = x.astype(np.float64)
    n, e = x.shape
    ok = np.isfinite(x)
    with np.errstate(all="ignore"):
        if sigmoid:
            s = np.where(ok, 1.0 / (1.0 + np.exp(-np.where(ok, x, 0))), 0.0)
        else:
            m = np.where(ok, x, -np.inf).max(1, keepdims=True)
            z = np.where(ok, np.exp(np.where(ok, x, 0) - np.where(np.isfinite(m), m, 0)), 0.0)
            s = z / np.where(z.sum(1, keepdims=True) > 0, z.sum(1, keepdims=True), 1)
    c = s if bias is None else s + bias.astype(np.float64)
    ok &= c > -np.inf  # (not NaN either)
    key = np.where(ok, x if bias is None else c, -np.inf)
    idx, w = np.full((n, k), -1, np.int32), np.zeros((n, k))
    unit = s.max(1)
    for t in range(n):
        ids = np.nonzero(ok[t])[0]
        if groups > 1:
            per = e // groups
            score = []
            for g in range(groups):
                mine = np.sort(c[t, [i for i in ids if i // per == g]])[::-1][:best]
                score.append(mine.sum() if len(mine) else -np.inf)
            order = [g for g in np.lexsort((np.arange(groups), -np.array(score))) if score[g] > -np.inf][:top]
            ids = np.array([i for i in ids if i // per in order], int)
        pick = ids[np.lexsort((ids, -key[t, ids]))[:k]] if len(ids) else ids
        idx[t, :len(pick)] = pick
        p = s[t, pick]
        if renorm and len(pick):
            p = p / p.sum() if p.sum() > 0 else p * 0
        w[t, :len(pick)] = p * scale
    return idx, w, unit


def _run(x, k, sigmoid, bias=None, groups=1, top=1, best=1, renorm=False, scale=1.0, pad=0, lead=0):
    import torch
    n, e = x.shape
    st = e + pad
    buf = torch.full((lead + n * st + 8,), 50.0, device="cuda:0")
    torch.as_strided(buf, (n, e), (st, 1), lead).copy_(torch.from_numpy(x))
    tb = None if bias is None else torch.from_numpy(bias.astype(np.float32)).cuda()
    idx = torch.full((n * k + 8,), 77, dtype=torch.int32, device="cuda:0")
    w = torch.full((n * k + 8,), 77.0, device="cuda:0")
    rule = Q.moe_route_rule(Q.ROUTE_SIGMOID if sigmoid else Q.ROUTE_SOFTMAX, None if tb is None else tb.data_ptr(), groups, top,
                            best, renorm, scale)
    Q.set_stream(None)
    Q.moe_route(buf.data_ptr() + 4 * lead, st, idx.data_ptr(), w.data_ptr(), n, e, k, rule)
    Q.check_device()
    assert bool((idx[n * k:] == 77).all()) and bool((w[n * k:] == 77).all())
    return idx[:n * k].view(n, k).cpu().numpy(), w[:n * k].view(n, k).cpu().numpy()


def _check(x, k, sigmoid, **a):
    pad, lead = a.pop("pad", 0), a.pop("lead", 0)
    gi, gw = _run(x, k, sigmoid, pad=pad, lead=lead, **a)
    ri, rw, unit = _reference(x, k, sigmoid, **a)
    assert np.array_equal(gi, ri), (np.argwhere(gi != ri)[:4], gi[gi != ri][:4], ri[gi != ri][:4])
    size = np.ones(len(x)) * 2 if a.get("renorm") else unit
    assert np.all(np.abs(gw - rw) <= TOL * size[:, None] * abs(a.get("scale", 1.0)) + 1e-38)
    assert np.all(gw[gi < 0] == 0)


def _logits(n, e, seed, spread=1.5):
    r = np.random.default_rng(seed)
    return (r.standard_normal((n, e)) * spread + r.standard_normal(e)).astype(np.float32)


@pytest.mark.parametrize("e", [1, 2, 7, 31, 32, 33, 64, 65, 96, 127, 160, 256, 300, 384, 385, 512, 513, 1000, 1024])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_experts(e, sigmoid, bias):
    for k in sorted({1, min(e, 6), min(e, 32)}):
        b = (np.random.default_rng(k).standard_normal(e) * 0.1).astype(np.float32) if bias else None
        _check(_logits(37, e, e + k), k, sigmoid, bias=b, renorm=k > 1, scale=2.5)


@pytest.mark.parametrize("groups,per", [(2, 3), (3, 5), (4, 32), (5, 13), (8, 32), (8, 20), (16, 16), (17, 9), (32, 1), (32, 32)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_groups(groups, per, best, sigmoid, bias):
    e = groups * per
    b = (np.random.default_rng(e).standard_normal(e) * 0.1).astype(np.float32) if bias else None
    for top in sorted({1, (groups + 1) // 2, groups}):
        _check(_logits(41, e, e + top), min(8, top * per), sigmoid, bias=b, groups=groups, top=top, best=best, renorm=True)


def test_many_tokens_and_the_first_rule():
    """The reference's rule on 64 experts: the same experts as ql_moe_router_topk."""
    import torch
    x = _logits(5000, 64, 5)
    _check(x, 6, False, scale=16.0)
    t = torch.from_numpy(x).cuda()
    idx, w = torch.empty(5000, 6, dtype=torch.int32, device="cuda:0"), torch.empty(5000, 6, device="cuda:0")
    Q.moe_router_topk(t.data_ptr(), idx.data_ptr(), w.data_ptr(), 5000, 64, 6, 16.0)
    gi, gw = _run(x, 6, False, scale=16.0)
    assert np.array_equal(gi, idx.cpu().numpy())
    # (that one's exponential is a fast one)
    assert np.allclose(gw, w.cpu().numpy(), rtol=1e-4, atol=16 * TOL)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 8])
def test_equal_logits(bias, groups):
    """bf16 logits have many equal ones; a row of zeros nothing else."""
    import torch
    x = torch.from_numpy(_logits(400, 256, 9, 0.5)).bfloat16().float().numpy()
    x[:7] = 0.0
    x[7] = -0.0
    b = np.repeat(np.float32([0.1, 0.1, -0.2, 0.1]), 64) if bias else None
    for best in (1, 2):
        _check(x, 8, True, bias=b, groups=groups, top=max(1, groups // 2), best=best, renorm=True)
        _check(x, 8, False, bias=b, groups=groups, top=max(1, groups // 2), best=best)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_scores_nearer_than_fp32(sigmoid):
    """Biases that bring the sums of neighbours within 1e-8 of each other, so that fp32 cannot tell which is larger."""
    r = np.random.default_rng(11)
    e = 64
    x = _logits(1, e, 12)
    s = 1 / (1 + np.exp(-x.astype(np.float64))) if sigmoid else np.exp(x.astype(np.float64)) / np.exp(x.astype(np.float64)).sum()
    level = np.repeat(np.linspace(2.0, 1.0, e // 4), 4)
    b = (level - s[0] + r.uniform(-1, 1, e) * 3e-8).astype(np.float32)
    gaps = np.diff(np.sort(s[0] + b.astype(np.float64)))
    assert (gaps < 1e-7).sum() > 20 and gaps[gaps > 0].min() > 1e-13
    for k in (1, 2, 3, 6, 13):
        _check(x, k, sigmoid, bias=b, renorm=True)
        _check(x, k, sigmoid, bias=b, groups=8, top=3, best=2)
    # groups that all but tie
    y = np.tile(_logits(1, 16, 13), (50, 4)) + (r.integers(-1, 2, (50, 64)) * 2e-7).astype(np.float32)
    for best in (1, 2):
        for top in (1, 2, 3):
            _check(y.astype(np.float32), 5, sigmoid, groups=4, top=top, best=best)


def test_not_finite_and_not_to_be_chosen():
    x = _logits(60, 96, 14)
    r = np.random.default_rng(15)
    x[r.random(x.shape) < 0.3] = -np.inf
    x[r.random(x.shape) < 0.1] = np.nan
    x[r.random(x.shape) < 0.1] = np.inf
    x[5] = -np.inf
    x[6] = np.nan
    x[7, 1:] = -np.inf
    x[8, 48:] = -np.inf
    x[9] = -3.4028235e38
    x[10, ::2] = 3.4028235e38
    b = (r.standard_normal(96) * 0.1).astype(np.float32)
    b[3], b[4], b[50:60], b[70] = -np.inf, np.nan, -np.inf, np.inf
    for bias in (None, b):
        for sigmoid in (False, True):
            for renorm in (False, True):
                _check(x, 12, sigmoid, bias=bias, renorm=renorm)
                _check(x, 12, sigmoid, bias=bias, renorm=renorm, groups=6, top=2, best=2)
                _check(x, 12, sigmoid, bias=bias, renorm=renorm, groups=32, top=5, best=1)


def test_far_scores():
    """Scores of 1e-60: their quotients are in range."""
    x = np.full((3, 40), -200.0, np.float32) - np.arange(40, dtype=np.float32) * 0.25
    x[1] -= 400
    gi, gw = _run(x, 4, True, renorm=True)
    ri, rw, _ = _reference(x, 4, True, renorm=True)
    assert np.array_equal(gi, ri) and np.allclose(gw, rw, rtol=1e-6)


@pytest.mark.parametrize("pad,lead", [(1, 0), (0, 1), (4, 0), (3, 3), (4, 4)])
def test_strides_and_starts(pad, lead):
    b = (np.random.default_rng(1).standard_normal(256) * 0.1).astype(np.float32)
    _check(_logits(33, 256, 16), 8, True, bias=b, groups=8, top=4, best=2, renorm=True, pad=pad, lead=lead)


def test_replay():
    import torch
    x = torch.from_numpy(_logits(64, 128, 17)).cuda()
    idx, w = torch.empty(64, 4, dtype=torch.int32, device="cuda:0"), torch.empty(64, 4, device="cuda:0")
    rule = Q.moe_route_rule(Q.ROUTE_SOFTMAX, renormalise=True)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        call = lambda: Q.moe_route(x.data_ptr(), 128, idx.data_ptr(), w.data_ptr(), 64, 128, 4, rule)  # noqa: E731
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call()
        new = _logits(64, 128, 18)
        x.copy_(torch.from_numpy(new))
        g.replay()
        st.synchronize()
    Q.set_stream(None)
    ri, rw, _ = _reference(new, 4, False, renorm=True)
    assert np.array_equal(idx.cpu().numpy(), ri) and np.all(np.abs(w.cpu().numpy() - rw) <= 2 * TOL)
