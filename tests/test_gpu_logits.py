"""Rules on logits (ql_logits_apply) against a step-by-step restatement: bit-equal, since every step is one fp32
operation in a fixed order."""
import numpy as np
import pytest

import blog_b200 as Q
import kv8_util as U
from gpu_util import dev, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _stream():
    import torch
    torch.cuda.init()
    Q.init(0)
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    Q.check_device()


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def _run(x, stride=None, hist=None, lens=None, prompt=None, rep=None, freq=None, pres=None, bias=None, mask=None,
         mask_row=None, in_place=False, out=True, token=True, ws=None):
    import torch
    n, v = x.shape
    stride = stride or v
    buf = np.zeros((n, stride), np.float32)
    buf[:, :v] = x
    xd = dev(buf)
    od = xd if in_place else torch.full((n, stride), 5.0, device="cuda:0")
    p = lambda a: None if a is None else dev(a).data_ptr()  # noqa: E731
    f = lambda a: None if a is None else np.asarray(a, np.float32)  # noqa: E731
    kw = {}
    if hist is not None:
        kw.update(history=p(hist), history_stride=hist.shape[1], history_len=p(np.asarray(lens, np.int32)),
                  prompt_len=p(None if prompt is None else np.asarray(prompt, np.int32)))
    if bias is not None:
        ids = np.concatenate([np.asarray([i for i, _ in b], np.int32) for b in bias] + [np.zeros(1, np.int32)])
        val = np.concatenate([np.asarray([w for _, w in b], np.float32) for b in bias] + [np.zeros(1, np.float32)])
        kw.update(bias_ids=p(ids), bias_values=p(val),
                  bias_start=p(np.concatenate([[0], np.cumsum([len(b) for b in bias])]).astype(np.int32)))
    if mask is not None:
        words = (v + 31) // 32
        bits = np.zeros((len(mask), words * 32), bool)
        bits[:, :v] = mask
        w = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
        kw.update(mask=p(w), mask_stride=words, mask_rows=len(mask),
                  mask_row=p(None if mask_row is None else np.asarray(mask_row, np.int32)))
    rules = Q.logits_rules(repetition=p(f(rep)), frequency=p(f(freq)), presence=p(f(pres)), **kw)
    tok = torch.full((n,), -7, dtype=torch.int32, device="cuda:0")
    ws = torch.zeros(16 * n, dtype=torch.uint8, device="cuda:0") if ws is None else ws
    Q.logits_apply(xd.data_ptr(), stride, od.data_ptr() if out else None, stride, n, v, rules,
                   tok.data_ptr() if token else None, ws.data_ptr() if token else None, ws.numel())
    assert Q.last_launch_count() == 1
    got = host(od)
    assert (host(ws) == 0).all()
    if stride > v and out and not in_place:
        assert (got[:, v:] == 5.0).all()
    return got[:, :v], host(tok)


def _want(x, hist=None, lens=None, prompt=None, rep=None, freq=None, pres=None, bias=None, mask=None, mask_row=None):
    ys, ts = [], []
    for r in range(len(x)):
        m = None
        if mask is not None:
            i = r if mask_row is None else mask_row[r]
            m = mask[i] if i >= 0 else None
        y, t = U.logits_rules(x[r], hist[r][:lens[r]] if hist is not None else (), prompt[r] if prompt is not None else 0,
                              rep[r] if rep is not None else None, freq[r] if freq is not None else 0.0,
                              pres[r] if pres is not None else 0.0, bias[r] if bias is not None else (), m)
        ys.append(y)
        ts.append(t)
    return np.stack(ys), np.asarray(ts)


@pytest.mark.parametrize("n,v,stride", [(1, 1, 1), (1, 31, 31), (3, 33, 33), (2, 4096, 4096), (5, 4097, 4097),
                                        (4, 32001, 32004), (3, 50257, 50257), (2, 152064, 152064)])
@pytest.mark.parametrize("in_place", [False, True])
def test_all_rules(n, v, stride, in_place):
    rng = np.random.default_rng(v + n)
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    x[0, :min(v, 5)] = x[0].max()  # ties
    h = 700
    hist = (rng.integers(-2, v + 2, (n, h)) % max(1, min(v, 97) + 3) - 1).astype(np.int32)
    hist[:, 5] = v - 1
    hist[:, 6] = v + 5
    lens = rng.integers(0, h + 1, n)
    lens[0] = h
    prompt = [int(a * f) for a, f in zip(lens, rng.random(n))]
    kw = dict(hist=hist, lens=lens, prompt=prompt, rep=1 + rng.random(n), freq=rng.random(n), pres=rng.random(n),
              bias=[[(int(rng.integers(0, v)), float(b)) for b in rng.standard_normal(r % 3 * 40)] +
                    [(0, 0.3), (0, 1e-7), (v - 1, -1.0), (v, 3.0), (-1, 3.0)] for r in range(n)],
              mask=rng.random((max(1, n - 1), v)) < 0.7, mask_row=[r - 1 for r in range(n)])
    for a in ("rep", "freq", "pres"):
        kw[a] = kw[a].astype(np.float32)
    got, tok = _run(x, stride, in_place=in_place, **kw)
    y, t = _want(x, **kw)
    assert _same(got, y)
    assert (tok == t).all()


@pytest.mark.parametrize("drop", ["hist", "prompt", "rep", "freq", "pres", "bias", "mask", "mask_row"])
def test_each_rule_may_be_absent(drop):
    rng = np.random.default_rng(3)
    n, v = 4, 5003
    x = rng.standard_normal((n, v)).astype(np.float32)
    kw = dict(hist=rng.integers(0, v, (n, 64)).astype(np.int32), lens=[64, 1, 0, 30], prompt=[10, 0, 0, 30],
              rep=np.full(n, 1.3, np.float32), freq=np.full(n, 0.1, np.float32), pres=np.full(n, 0.4, np.float32),
              bias=[[(7, 2.0)], [], [(9, -3.0), (9, 1.0)], [(5002, 50.0)]], mask=rng.random((n, v)) < 0.5,
              mask_row=[3, -1, 0, 1])
    kw.pop(drop)
    if drop == "hist":
        kw.pop("lens"), kw.pop("prompt")
    if drop == "mask":
        kw.pop("mask_row")
    got, tok = _run(x, **kw)
    y, t = _want(x, **kw)
    assert _same(got, y) and (tok == t).all()


def test_rows_with_nothing_left_and_values_out_of_the_ordinary():
    """A mask that allows nothing (token -1), logits of -inf only, NaN and infinities under the rules and the mask, the
    type's lowest value, signed zeros (the lower index), a single allowed token."""
    v = 2100
    x = np.random.default_rng(4).standard_normal((8, v)).astype(np.float32)
    x[1] = -np.inf
    x[2, 10], x[2, 2000] = np.nan, np.inf
    x[3, ::2] = np.nan
    x[4] = np.finfo(np.float32).min
    x[5] = 0.0
    x[5, 0] = -0.0
    x[6] = np.nan
    mask = np.ones((8, v), bool)
    mask[0] = False
    mask[2, 2000] = False
    mask[7] = False
    mask[7, 2099] = True
    hist = np.tile(np.asarray([10, 2000, 2000, 0, 5], np.int32), (8, 1))
    kw = dict(hist=hist, lens=[5] * 8, prompt=[1] * 8, rep=np.full(8, 1.2, np.float32), freq=np.full(8, 0.25, np.float32),
              pres=np.full(8, 0.5, np.float32), mask=mask)
    got, tok = _run(x, **kw)
    y, t = _want(x, **kw)
    assert _same(got, y) and (tok == t).all()
    assert tok[0] == -1 and tok[1] == -1 and tok[6] == -1 and tok[7] == 2099
    got, tok = _run(x[5:6])
    assert tok[0] == 0


def test_token_only_and_logits_only():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 9001)).astype(np.float32)
    y, t = _want(x)
    got, tok = _run(x, out=False)
    assert (tok == t).all()
    got, tok = _run(x, token=False)
    assert _same(got, y) and (tok == -7).all()


def test_the_workspace_serves_call_after_call():
    import torch
    rng = np.random.default_rng(6)
    ws = torch.zeros(16 * 7, dtype=torch.uint8, device="cuda:0")
    for n in (7, 3, 7, 1):
        x = rng.standard_normal((n, 20000)).astype(np.float32)
        got, tok = _run(x, ws=ws)
        assert (tok == x.argmax(1)).all()


def test_many_repetitions_of_one_token():
    n = 20000
    hist = np.full((1, n), 3, np.int32)
    x = np.full((1, 100), 2.0, np.float32)
    kw = dict(hist=hist, lens=[n], prompt=[0], rep=[1.5], freq=np.asarray([0.01], np.float32), pres=[0.0])
    got, tok = _run(x, **kw)
    y, t = _want(x, **kw)
    assert _same(got, y) and (tok == t).all()


def test_a_mask_row_outside_the_masks_allows_nothing_and_is_reported():
    x = np.random.default_rng(8).standard_normal((2, 100)).astype(np.float32)
    got, tok = _run(x, mask=np.ones((1, 100), bool), mask_row=[0, 1])
    assert tok[0] == x[0].argmax() and tok[1] == -1 and np.isneginf(got[1]).all()
    with pytest.raises(Q.QLError, match="mask row"):
        Q.check_device()


def test_refusals():
    import torch
    x = torch.zeros(4096, device="cuda:0")
    p = x.data_ptr()
    none = Q.logits_rules()

    def call(**k):
        a = dict(x=p, xs=100, o=p, os=100, n=2, v=100, r=none, t=p, w=p, wb=64)
        a.update(k)
        Q.logits_apply(a["x"], a["xs"], a["o"], a["os"], a["n"], a["v"], a["r"], a["t"], a["w"], a["wb"])
    for bad in (dict(x=None), dict(xs=99), dict(os=50), dict(os=200), dict(n=-1), dict(n=70000), dict(v=-1), dict(v=0),
                dict(x=p + 2), dict(w=None), dict(wb=31), dict(w=p + 8),
                dict(r=Q.logits_rules(history=p)), dict(r=Q.logits_rules(bias_ids=p)),
                dict(r=Q.logits_rules(mask=p, mask_stride=3, mask_rows=2)),
                dict(r=Q.logits_rules(mask=p, mask_stride=4, mask_rows=1))):
        with pytest.raises(Q.QLError) as e:
            call(**bad)
        assert e.value.status == Q.QL_EINVAL, bad
    call(n=0)
