"""The residual's addition with the RMS norm and its 8-bit rows, against 64-bit numpy and the Q8_1 quantiser."""
import numpy as np
import pytest

import blog_b200 as Q

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# y in f32 against the exact norm of the stored sum: squares (fma and product, 2 roundings, 8 groups per thread and 10
# levels of the tree: 21), the mean and eps (2) count half under the root; rsqrtf 2 units in the last place (4),
# two products: 11.5 + 4 + 2 < 18
Y_TOL = 18 * U


def _torch(type_):
    import torch
    return torch.float32 if type_ == Q.F32 else torch.bfloat16


def _bf16(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).bfloat16().float().numpy()


def _padded(a, stride, type_, lead=0):
    """Device rows of a, `stride` elements apart, `lead` elements past an aligned address; the buffer and its rows."""
    import torch
    n, h = a.shape
    buf = torch.full((lead + n * stride + 64,), 7.0, dtype=_torch(type_), device="cuda:0")
    rows = torch.as_strided(buf, (n, h), (stride, 1), lead)
    rows.copy_(torch.from_numpy(np.ascontiguousarray(a, np.float32)))
    return buf, rows


def _run(type_, n, h, *, residual=True, gamma=True, y=True, layout=Q.Q8_ROWS, raw=False, pad=0, lead=0, eps=1e-6, seed=0,
         x=None, r=None):
    import torch
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, h)).astype(np.float32) if x is None else x
    r = (rng.standard_normal((n, h)) * 3).astype(np.float32) if r is None else r
    g = (1 + 0.3 * rng.standard_normal(h)).astype(np.float32)
    if type_ == Q.BF16:
        x, r = _bf16(x), _bf16(r)
    st = h + pad
    bx, tx = _padded(x, st, type_, lead)
    br, tr = _padded(r, st, type_, lead)
    bs, ts = _padded(np.zeros((n, h)), st, type_, lead)
    by, ty = _padded(np.zeros((n, h)), st, type_, lead)
    tg = torch.from_numpy(g).cuda()
    nb = (h + 31) // 32
    size = n * Q.q8_1_row_bytes(h) if layout != Q.Q8_MMQ else n * Q.q8_1_mmq_row_bytes(h)
    xq = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda:0")
    Q.set_stream(None)
    Q.add_rms_norm(type_, tx.data_ptr(), st, tr.data_ptr() if residual else None, st, ts.data_ptr(), st,
                   tg.data_ptr() if gamma else None, eps, ty.data_ptr() if y else None, st,
                   xq.data_ptr() if layout else None, layout, raw, n, h)
    Q.check_device()
    with np.errstate(all="ignore"):
        v = x + r if residual else x
        if type_ == Q.BF16:
            v = _bf16(v)
        w = v.astype(np.float64)
        ref = w / np.sqrt((w ** 2).mean(1, keepdims=True) + eps) * (g.astype(np.float64) if gamma else 1.0)
    # what lies between and behind the rows is left as it was
    for b in (bs, by):
        keep = torch.ones_like(b, dtype=torch.bool)
        torch.as_strided(keep, (n, h), (st, 1), lead).fill_(False)
        assert bool((b[keep] == 7.0).all())
    assert bool((xq[size:] == 0xA5).all())
    return dict(v=v, ref=ref, sum=ts.float().cpu().numpy(), y=ty.float().cpu().numpy(), xq=xq[:size].cpu().numpy(), nb=nb, h=h,
                n=n)


def _q8(y, raw):
    """Codes, d and sums of the Q8_1 definition for f32 rows y, each operation rounded as there."""
    n, h = y.shape
    nb = (h + 31) // 32
    z = np.zeros((n, nb * 32), np.float32)
    z[:, :h] = y
    z = z.reshape(n, nb, 32)
    amax = np.abs(z).max(-1)
    d = (amax / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d > 0, np.float32(1) / np.where(d > 0, d, 1), 0).astype(np.float32)
    q = np.clip(np.rint(z * inv[..., None]), -127, 127).astype(np.int32)
    if raw:
        t = z.copy()
        for o in (16, 8, 4, 2, 1):
            t = t[..., :o] + t[..., o:2 * o]
        s = t[..., 0]
    else:
        s = d * q.sum(-1).astype(np.float32)
    return q.astype(np.int8), d.astype(np.float16), s.astype(np.float16)


def _codes(o, layout):
    n, nb = o["n"], o["nb"]
    if layout == Q.Q8_ROWS:
        b = o["xq"].reshape(n, nb, 36)
        ds = b[..., :4].copy().view(np.float16)
        return b[..., 4:].copy().view(np.int8), ds[..., 0], ds[..., 1]
    b = o["xq"].reshape((nb + 3) // 4, n, 144)
    ds = b[..., :16].copy().view(np.float16).reshape(-1, n, 4, 2)
    q = b[..., 16:].copy().view(np.int8).reshape(-1, n, 4, 32)
    flat = lambda a: np.swapaxes(a, 0, 1).reshape(n, -1, *a.shape[3:])[:, :nb]  # noqa: E731
    return flat(q), flat(ds[..., 0]), flat(ds[..., 1])


def _check(o, type_, y=True, layout=Q.Q8_NONE, raw=False):
    assert np.array_equal(o["sum"], o["v"])
    tol = Y_TOL + (2.0 ** -8 if type_ == Q.BF16 else 0)
    if y:
        assert np.all(np.abs(o["y"] - o["ref"]) <= tol * np.abs(o["ref"]))
    if layout and type_ == Q.F32 and y:
        q, d, s = _codes(o, layout)
        eq, ed, es = _q8(o["y"], raw)
        assert np.array_equal(d, ed) and np.array_equal(q, eq) and np.array_equal(s, es)
    elif layout:  # y in f32 is not stored: within half a code, and d within its f16 and y's error
        q, d, s = _codes(o, layout)
        z = np.zeros((o["n"], o["nb"] * 32))
        z[:, :o["h"]] = o["ref"]
        z = z.reshape(o["n"], o["nb"], 32)
        ed = np.abs(z).max(-1) / 127
        assert np.all(np.abs(d - ed) <= ed * (2.0 ** -11 + 20 * U) + 2.0 ** -25)
        assert np.all(np.abs(q * ed[..., None] - z) <= ed[..., None] * (0.5 + 127 * 40 * U))


@pytest.mark.parametrize("h", [1, 5, 31, 32, 33, 96, 127, 1000, 2048, 3584, 4096, 4100, 8192, 8200, 16384, 18944, 32768])
@pytest.mark.parametrize("type_", [Q.F32, Q.BF16])
def test_widths(h, type_):
    for n in (1, 3):
        o = _run(type_, n, h, layout=Q.Q8_ROWS, seed=h)
        _check(o, type_, layout=Q.Q8_ROWS)


@pytest.mark.parametrize("n,h", [(297, 96), (300, 2048), (401, 8192), (299, 12288), (298, 20000)])
@pytest.mark.parametrize("type_", [Q.F32, Q.BF16])
def test_many_rows(n, h, type_):
    o = _run(type_, n, h, layout=Q.Q8_MMQ, raw=True, seed=n)
    _check(o, type_, layout=Q.Q8_MMQ, raw=True)


@pytest.mark.parametrize("pad,lead", [(4, 0), (1, 0), (0, 1), (3, 2), (8, 4)])
@pytest.mark.parametrize("type_", [Q.F32, Q.BF16])
@pytest.mark.parametrize("n", [3, 310])
def test_strides_and_starts(pad, lead, type_, n):
    o = _run(type_, n, 640, pad=pad, lead=lead, layout=Q.Q8_ROWS, raw=True, seed=pad)
    _check(o, type_, layout=Q.Q8_ROWS, raw=True)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("gamma", [False, True])
@pytest.mark.parametrize("y", [False, True])
@pytest.mark.parametrize("layout", [Q.Q8_NONE, Q.Q8_ROWS, Q.Q8_MMQ])
def test_parts(residual, gamma, y, layout):
    o = _run(Q.F32, 5, 352, residual=residual, gamma=gamma, y=y, layout=layout)
    _check(o, Q.F32, y=y, layout=layout)
    if not y:
        assert np.all(o["y"] == 0)


@pytest.mark.parametrize("raw", [False, True])
@pytest.mark.parametrize("mmq", [False, True])
def test_bytes_of_the_quantiser(raw, mmq):
    """The same bytes as the norm's y through ql_quantize_q8_1(_mmq), odd values among them."""
    import torch
    n, h = 9, 1024
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((n, h)) * np.exp(rng.standard_normal((n, h)) * 3)).astype(np.float32)
    x[1] = 0
    x[2, :64] = 1e-30
    x[3, 5] = np.inf
    x[4, 40] = np.nan
    x[5] = 1e-42
    x[6] = 3e18
    o = _run(Q.F32, n, h, residual=False, x=x, layout=Q.Q8_MMQ if mmq else Q.Q8_ROWS, raw=raw)
    yt = torch.from_numpy(o["y"]).cuda()
    want = torch.zeros(len(o["xq"]), dtype=torch.uint8, device="cuda:0")
    (Q.quantize_q8_1_mmq if mmq else Q.quantize_q8_1)(yt.data_ptr(), want.data_ptr(), h, n, raw)
    assert np.array_equal(o["xq"], want.cpu().numpy())
    fine = [0, 1, 2, 5, 6, 7, 8]
    err = np.abs(o["y"][fine] - o["ref"][fine])
    assert np.all(err <= Y_TOL * np.abs(o["ref"][fine]) + 2.0 ** -149)
    assert np.all(np.isnan(o["y"][4])) and np.isnan(o["y"][3, 5]) and np.all(np.delete(o["y"][3], 5) == 0)


def test_in_place():
    import torch
    n, h = 6, 777
    for type_ in (Q.F32, Q.BF16):
        g = torch.Generator(device="cuda:0").manual_seed(1)
        x = torch.randn(n, h, generator=g, device="cuda:0").to(_torch(type_))
        r = torch.randn(n, h, generator=g, device="cuda:0").to(_torch(type_))
        s, y = torch.empty_like(x), torch.empty_like(x)
        Q.set_stream(None)
        call = lambda a, b, c, d: Q.add_rms_norm(type_, a.data_ptr(), h, b.data_ptr(), h, c.data_ptr(), h, None, 1e-5,  # noqa: E731
                                                 d.data_ptr(), h, None, Q.Q8_NONE, False, n, h)
        call(x, r, s, y)
        for sum_in_x in (True, False):
            a, b = x.clone(), r.clone()
            if sum_in_x:
                call(a, b, a, b)
                assert torch.equal(a, s) and torch.equal(b, y)
            else:
                call(a, b, b, a)
                assert torch.equal(b, s) and torch.equal(a, y)


def test_offsets_past_32_bits():
    import torch
    h, st = 64, (1 << 30) + 8
    x = torch.zeros(2 * st + h, device="cuda:0")
    rows = torch.as_strided(x, (3, h), (st, 1))
    want = torch.randn(3, h, device="cuda:0")
    rows.copy_(want)
    y = torch.empty(3, h, device="cuda:0")
    Q.set_stream(None)
    Q.add_rms_norm(Q.F32, x.data_ptr(), st, x.data_ptr(), st, x.data_ptr(), st, None, 0.0, y.data_ptr(), h, None, Q.Q8_NONE, False,
                   3, h)
    assert torch.equal(rows, want + want)
    ref = want.double() / want.double().pow(2).mean(1, keepdim=True).sqrt()
    assert bool(((y - ref).abs() <= Y_TOL * ref.abs()).all())


def test_replay_and_stream():
    import torch
    n, h = 64, 3584
    x, r = torch.randn(n, h, device="cuda:0"), torch.randn(n, h, device="cuda:0")
    s, y = torch.empty_like(x), torch.empty_like(x)
    xq = torch.zeros(n * Q.q8_1_row_bytes(h), dtype=torch.uint8, device="cuda:0")
    st = torch.cuda.Stream()
    call = lambda: Q.add_rms_norm(Q.F32, x.data_ptr(), h, r.data_ptr(), h, s.data_ptr(), h, None, 1e-6, y.data_ptr(), h,  # noqa: E731
                                  xq.data_ptr(), Q.Q8_ROWS, False, n, h)
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call()
        x.copy_(torch.randn(n, h, device="cuda:0"))
        g.replay()
        st.synchronize()
        first = (s.clone(), y.clone(), xq.clone())
        call()
        st.synchronize()
    Q.set_stream(None)
    assert all(torch.equal(a, b) for a, b in zip(first, (s, y, xq))) and torch.equal(s, x + r)
    assert Q.last_launch_count() == 1


@pytest.mark.parametrize("size,eps", [(1e-30, 0.0), (1e-38, 0.0), (1e-43, 0.0), (1e-20, 1e-6), (1e25, 1e-6), (1e38, 1.0), (1e-12, 1e-24)])
@pytest.mark.parametrize("type_", [Q.F32, Q.BF16])
def test_squares_outside_the_range(size, eps, type_):
    """Rows whose squares fp32 does not hold.  (bf16 rounds 1e-43 to zeros: 0 / 0.)"""
    rng = np.random.default_rng(7)
    x = (rng.uniform(0.5, 1.5, (4, 1504)) * rng.choice([-1, 1], (4, 1504)) * size).astype(np.float32)
    o = _run(type_, 4, 1504, residual=False, x=x, eps=eps, layout=Q.Q8_NONE)
    tol = Y_TOL + (2.0 ** -8 if type_ == Q.BF16 else 0)
    none = np.isnan(o["ref"])
    assert np.array_equal(none, np.isnan(o["y"])) and (not none.any() or (type_ == Q.BF16 and size == 1e-43))
    assert np.all((np.abs(o["y"] - o["ref"]) <= tol * np.abs(o["ref"]) + 2.0 ** -149) | none)
