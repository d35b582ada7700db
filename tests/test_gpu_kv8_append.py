"""ql_kv8_append where its blocks, lengths or arguments are out of the ordinary."""
import numpy as np
import pytest

import blog_b200 as Q
import kv8_util as U
from gpu_util import dev, host, rel_l2
from test_gpu_kv8 import TOL, Cache, _append, _check_cache, _i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _stream():
    import torch
    torch.cuda.init()
    Q.init(0)
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    Q.check_device()


def test_codes_of_the_smallest_blocks():
    """Largest magnitudes of 1 to 2^20 units of 2^-149: a subnormal scale is rounded so coarsely that x / scale may pass
    127, and the code stays at +-127."""
    kvh, hd = 2, 64
    most = [1, 2, 63, 64, 100, 127, 190, 191, 254, 318, 1330, 5000, 1 << 20]
    n = 32 * len(most)
    rng = np.random.default_rng(81)
    x = np.concatenate([rng.integers(-m, m + 1, (32, 2, kvh, hd)) for m in most]).astype(np.float64)
    for b, m in enumerate(most):
        x[32 * b, :, :, 0], x[32 * b, :, :, 1] = m, -m
    x = (x * 2.0 ** -149).astype(np.float32)
    c = Cache(1, n, kvh, hd, seed=82)
    _append(c, "f32", dev(x.reshape(n, -1)), 0, None, _i32([n]), _i32([0, n]), n)
    for j, (codes, scales) in enumerate(((c.kc, c.ks), (c.vc, c.vs))):
        codes, scales = host(codes), host(scales)
        for b in range(len(most)):
            for h in range(kvh):
                z = x[32 * b:32 * b + 32, j, h]
                scale = np.abs(z).max() / np.float32(127)
                want = np.rint(z / scale).clip(-127, 127) + 128 if scale else np.full(z.shape, 128)
                page = c.table[0, b]
                assert scales[page, h] == scale
                assert np.array_equal(codes[page, h], want), most[b]
    Q.check_device()


@pytest.mark.parametrize("bad,what", [(2 ** 31 - 1, "page"), (2 ** 31 - 32, "page"), (-1, "more rows"), (-2 ** 31, "more rows")])
@pytest.mark.parametrize("ragged", [False, True])
def test_lengths_at_the_ends_of_their_type_are_reported(bad, what, ragged):
    """Nothing of that sequence is stored, the other's token is."""
    kvh, hd = 2, 64
    c = Cache(2, 64, kvh, hd, seed=89)
    c.ko.zero_()
    x = np.random.default_rng(90).standard_normal((2, 2 * kvh * hd)).astype(np.float32)
    _append(c, "f32", dev(x), 0, None, _i32([bad, 3]), _i32([0, 1, 2]) if ragged else None, 1)
    with pytest.raises(Q.QLError, match=what):
        Q.check_device()
    want = np.zeros(c.ko.shape, np.float32)
    want[c.slot[1], 0, :, 2] = x[1, :kvh * hd].reshape(kvh, hd)
    assert np.array_equal(host(c.ko), want)
    assert (host(c.kc) == 77).all()


def test_rows_before_the_first_sequence_are_nobodys():
    """q_start[0] = 70 (it should be 0): the 70 rows' tiles touch no page, and the sequences' own rows are stored."""
    kvh, hd = 2, 64
    c = Cache(2, 64, kvh, hd, seed=91)
    x = np.random.default_rng(92).standard_normal((75, 2 * kvh * hd)).astype(np.float32)
    _append(c, "f32", dev(x), 0, None, _i32([2, 3]), _i32([70, 72, 75]), 70)
    ko = host(c.ko)
    for s, (row, n) in enumerate(((70, 2), (72, 3))):
        assert np.array_equal(ko[c.slot[s], 0, :, :n], x[row:row + n, :kvh * hd].reshape(n, kvh, hd).transpose(1, 0, 2))
    assert (host(c.kc) == 77).all()
    Q.check_device()


def test_speculative_cycles():
    """Calls of up to 33 draft tokens of which some are taken back each time, over ten pages: as if the rejected ones
    had never been."""
    kvh, hd = 2, 64
    rng = np.random.default_rng(93)
    c = Cache(1, 400, kvh, hd, seed=94)
    text, pos = np.zeros((0, 2 * kvh * hd), np.float32), 0
    for step in range(60):
        n = int(rng.integers(1, 34))
        x = rng.standard_normal((n, 2 * kvh * hd)).astype(np.float32)
        if pos + n > 400:
            break
        _append(c, "f32", dev(x), 0, None, _i32([pos + n]), _i32([0, n]), n)
        keep = int(rng.integers(1, n + 1))
        text, pos = np.concatenate([text, x[:keep]]), pos + keep
        z = text.reshape(pos, 2, kvh, hd).astype(np.float64)
        _check_cache(c, [z[:, 0]], [z[:, 1]], [pos], exact_bytes=True)
    assert pos > 320
    Q.check_device()


@pytest.mark.parametrize("back", [0, 32, 64, 96, 129, 140, 150])
def test_going_back_to_a_page_and_into_the_last_two(back):
    """From 180 tokens to a multiple of 32 or into the last two pages (from 128 on), then 90 others."""
    kvh, hd = 2, 64
    rng = np.random.default_rng(95)
    x = rng.standard_normal((180, 2 * kvh * hd)).astype(np.float32)
    y = rng.standard_normal((90, 2 * kvh * hd)).astype(np.float32)
    c = Cache(1, 300, kvh, hd, seed=96)
    _append(c, "f32", dev(x), 0, None, _i32([180]), _i32([0, 180]), 180)
    _append(c, "f32", dev(y), 0, None, _i32([back + 90]), _i32([0, 90]), 90)
    z = np.concatenate([x[:back], y]).reshape(back + 90, 2, kvh, hd).astype(np.float64)
    _check_cache(c, [z[:, 0]], [z[:, 1]], [back + 90], exact_bytes=True)
    Q.check_device()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_pages_beyond_4_gb(t):
    """Pages on both sides of the 2^32nd byte of the codes: append, read-back, and both kernels of the attention."""
    import torch
    nh, kvh, hd, n = 64, 8, 128, 700
    pages = (1 << 32) // (kvh * 32 * hd) + 200
    per = (n + 31) // 32
    rng = np.random.default_rng(97)
    table = np.stack([rng.permutation(400)[:per] + pages - 400, rng.permutation(per)]).astype(np.int32)
    kc, vc = (torch.zeros((pages, kvh, 32, hd), dtype=torch.uint8, device="cuda:0") for _ in range(2))
    ks, vs = (torch.zeros((pages, kvh), device="cuda:0") for _ in range(2))
    ko, vo = (torch.zeros((2, 2, kvh, 32, hd), device="cuda:0") for _ in range(2))
    td = dev(table)
    cache = Q.kv8_cache(*(x.data_ptr() for x in (kc, vc, ks, vs, ko, vo, td)), None, pages, 2, 2, per, kvh, hd)
    el, code = (4, Q.F32) if t == "f32" else (2, Q.BF16)
    x = torch.randn((2 * n, (nh + 2 * kvh) * hd), device="cuda:0", generator=torch.Generator(device="cuda:0").manual_seed(98))
    x = x.to(torch.float32 if t == "f32" else torch.bfloat16)
    w, p = x.shape[1], x.data_ptr()
    kv, st = _i32([n, n]), _i32([0, n, 2 * n])
    Q.kv8_append(cache, code, None, 0, p + nh * hd * el, w, p + (nh + kvh) * hd * el, w, None, 0, 0, None, None, 1e-6, None, 0,
                 0, kv.data_ptr(), st.data_ptr(), 2 * n, n)
    back = [torch.zeros((2, n, kvh, hd), device="cuda:0") for _ in range(2)]
    Q.kv8_gather(cache, Q.F32, back[0].data_ptr(), back[1].data_ptr(), None, n, kv.data_ptr())
    k, v = (host(b).astype(np.float64) for b in back)
    raw = host(x.float()).reshape(2, n, nh + 2 * kvh, hd)
    for got, at in ((k, nh), (v, nh + kvh)):
        assert np.abs(got - raw[:, :, at:at + kvh]).max() < np.abs(raw).max() / 250
    ws = torch.zeros(Q.kv8_attend_workspace(nh, kvh, hd, 2, 2 * n, n, n), dtype=torch.uint8, device="cuda:0")
    out = torch.zeros((2 * n, nh * hd), dtype=x.dtype, device="cuda:0")
    for rows, form in ((2 * n, Q.KV8_FORM_TILES), (2, Q.KV8_FORM_SPLIT)):
        q_len = rows // 2
        Q.kv8_attend(cache, code, p, w, None, 0, out.data_ptr(), nh * hd, nh, hd ** -0.5, kv.data_ptr(),
                     st.data_ptr() if q_len > 1 else None, rows, q_len, n, ws.data_ptr(), ws.numel())
        assert Q.kv8_attend_form()[0] == form
        got = host(out.float())
        for s in range(2):
            for i in (0, q_len // 2, q_len - 1):
                row = s * q_len + i
                q = raw.reshape(2 * n, -1, hd)[row, :nh]
                want = U.attend(q, k[s].transpose(1, 0, 2), v[s].transpose(1, 0, 2), n - q_len + i, hd ** -0.5)
                assert rel_l2(got[row], want.ravel()) < TOL[t], (form, s, i)
    Q.check_device()
