"""ql_kv8_attend by the kernel that takes the call: each case is sized for the tiles on tcgen05 or for the split over the
keys and asserts which of the two ran, so that a change of the rule between them cannot move a case to the other.

Tolerances as in test_gpu_kv8.py; a score of size S carries an error of 2^-22 S into the exponent, so extreme scores
add S 2^-21."""
import numpy as np
import pytest

import blog_b200 as Q
import kv8_util as U
from gpu_util import dev, host, rel_l2
from test_gpu_kv8 import TOL, Cache, _attend, _dev, _filled, _i32

pytestmark = pytest.mark.gpu
WIDTHS = [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128), ("bf16", 256)]  # that the tiles take


@pytest.fixture(scope="module", autouse=True)
def _stream():
    import torch
    torch.cuda.init()
    Q.init(0)
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    Q.check_device()


def _tiles(ctas=None):
    form, n = Q.kv8_attend_form()
    assert form == Q.KV8_FORM_TILES
    assert ctas is None or n == ctas, n


def _starts(q_len):
    return np.concatenate([[0], np.cumsum(q_len)])


def _check_rows(got, q, stands, lens, q_len, nh, tol, scale=None, rows=None):
    """Every row (or those for which rows(s, i) holds) against the restatement."""
    st, hd = _starts(q_len), q.shape[1] // nh
    for s in range(len(lens)):
        r = slice(st[s], st[s + 1])
        if q_len[s] == 0:
            continue
        want = U.attend_rows(q[r].reshape(-1, nh, hd), *stands[s], lens[s] - q_len[s],
                             hd ** -0.5 if scale is None else scale).reshape(-1, nh * hd)
        for i in range(q_len[s]):
            if rows is None or rows(s, i):
                assert rel_l2(got[r][i], want[i]) < tol, (s, i)


@pytest.mark.parametrize("t,hd,nh,kvh,q_len,past,ctas", [
    ("f32", 64, 28, 4, 300, 1030, 2), ("f32", 64, 14, 2, 513, 1030, 3), ("f32", 64, 14, 2, 300, 2100, 4),
    ("f32", 64, 8, 1, 400, 2600, 5), ("f32", 64, 14, 2, 200, 3100, 6), ("f32", 64, 32, 2, 64, 3650, 7),
    ("f32", 64, 28, 4, 64, 4200, 8), ("f32", 128, 14, 2, 200, 1500, 3), ("f32", 128, 32, 2, 64, 2100, 4),
    ("f32", 128, 8, 1, 200, 2600, 5), ("f32", 128, 14, 2, 100, 3100, 6), ("f32", 128, 8, 1, 150, 3650, 7),
    ("f32", 128, 16, 1, 64, 4200, 8), ("bf16", 64, 8, 1, 513, 1500, 3), ("bf16", 64, 14, 2, 150, 2600, 5),
    ("bf16", 64, 28, 4, 64, 3100, 6), ("bf16", 64, 8, 1, 200, 3650, 7), ("bf16", 128, 8, 1, 400, 1030, 2),
    ("bf16", 128, 32, 2, 64, 1500, 3), ("bf16", 128, 8, 1, 150, 2600, 5), ("bf16", 128, 16, 1, 64, 3100, 6),
    ("bf16", 128, 8, 1, 100, 3650, 7), ("bf16", 128, 8, 1, 100, 4200, 8), ("bf16", 256, 8, 1, 300, 1030, 2),
    ("bf16", 256, 14, 2, 100, 1500, 3), ("bf16", 256, 16, 1, 64, 2100, 4), ("bf16", 256, 14, 2, 64, 2600, 5),
    ("bf16", 256, 8, 1, 100, 3100, 6), ("bf16", 256, 8, 1, 100, 3650, 7), ("bf16", 256, 8, 1, 64, 4200, 8)])
def test_keys_over_clusters_of_every_size(t, hd, nh, kvh, q_len, past, ctas):
    """A chunk over a long cache, its keys split over 2 to 8 CTAs (shares of 256 or 128 rows that do not divide), and a
    short one beside it, most of whose CTAs have no tiles."""
    q_lens, lens = [q_len, q_len // 3], [past + q_len, 17 + q_len // 3]
    c, stands = _filled(lens, max(lens), kvh, hd, seed=61)
    qd, q = _dev(np.random.default_rng(62).standard_normal((sum(q_lens), nh * hd)) * 1.5, t)
    got = _attend(c, t, qd, nh, _i32(lens), _i32(_starts(q_lens)), q_len, max(lens))
    _tiles(ctas)
    _check_rows(got, q, stands, lens, q_lens, nh, TOL[t])
    Q.check_device()


@pytest.mark.parametrize("t,hd", WIDTHS)
def test_tiles_scores_of_every_size_and_signs(t, hd):
    """Scores of +-1e3 and 1e30, equal scores, tiny and huge queries, values whose scales lie 1e12 apart, blocks of zeros
    (K, V), positive and negative softmax scales."""
    nh, kvh, n = 64, 1, 700
    c = Cache(1, n, kvh, hd, seed=63)
    rng = np.random.default_rng(64)
    k, v = rng.standard_normal((2, n, kvh, hd))
    v[:64] *= 1e-6
    v[64:96] *= 1e6
    v[96:128] = 0
    k[128:160] = 0
    stands = [z.transpose(1, 0, 2) for z in c.set(0, k, v)]
    q = rng.standard_normal((n, nh, hd))
    q[:, 1] *= 100
    q[:, 2] = 0
    q[:, 3] *= 1e-30
    q[:, 4] = -q[:, 1]
    q[:, 5] *= 1e30
    qd, q = _dev(q.reshape(n, -1), t)
    q = q.reshape(n, nh, hd)
    for scale in (hd ** -0.5, -hd ** -0.5):
        got = _attend(c, t, qd, nh, _i32([n]), _i32([0, n]), n, n, scale=scale).reshape(n, nh, hd)
        _tiles(1)
        want = U.attend_rows(q, *stands, 0, scale)
        for h in (0, 1, 2, 3, 4, 5, 40, 63):
            s = np.abs(stands[0][0] @ q[:, h].T.astype(np.float64)).max() * hd ** -0.5
            tol = TOL[t] + (0 if s > 1e6 else s * 2.0 ** -21)
            for i in range(n):
                assert rel_l2(got[i, h], want[i, h]) < tol, (h, i)
    Q.check_device()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 96, 256])
def test_split_scores_of_every_size_where_the_heaviest_keys_have_no_value(hd, t):
    """The same in few rows, eight blocks to a warp: blocks of zero and of large values among keys whose
    scores lie 0 to 1e30 apart."""
    nh, kvh, n = 8, 1, 1000
    c = Cache(1, n, kvh, hd, seed=77)
    rng = np.random.default_rng(78)
    k, v = rng.standard_normal((2, n, kvh, hd))
    v[640:] *= 1e6
    v[320:640] = 0
    stands = [z.transpose(1, 0, 2) for z in c.set(0, k, v)]
    q = rng.standard_normal((16, nh, hd)) * 10.0 ** np.asarray([0, 1, 2, 4, 7, 12, 20, 30])[None, :, None]
    qd, q = _dev(q.reshape(16, -1), t)
    q = q.reshape(16, nh, hd)
    got = _attend(c, t, qd, nh, _i32([n]), _i32([0, 16]), 16, 32).reshape(16, nh, hd)  # (a short bound: one CTA)
    assert Q.kv8_attend_form() == (Q.KV8_FORM_SPLIT, 1)
    want = U.attend_rows(q, *stands, n - 16, hd ** -0.5)
    for h in range(nh):
        s = np.abs(stands[0][0] @ q[:, h].T.astype(np.float64)).max() * hd ** -0.5
        for i in range(16):
            if s < 1e6:
                assert rel_l2(got[i, h], want[i, h]) < TOL[t] + s * 2.0 ** -21, (h, i)
            else:  # (one key has it all: its value, or zeros)
                top = np.argmax(stands[0][0][:n - 15 + i] @ q[i, h].astype(np.float64))
                assert rel_l2(got[i, h], stands[1][0][top]) < TOL[t], (h, i)
    Q.check_device()


@pytest.mark.parametrize("t,hd", WIDTHS)
def test_tiles_where_the_heaviest_keys_have_no_value(t, hd):
    """Keys 60 to 80 nats above all others with values of zero: what is left of the others is 1e-26 and less, and still
    relatively right (weights below the range of a 2^(s - m))."""
    nh, kvh, n = 64, 1, 700
    c = Cache(1, n, kvh, hd, seed=65)
    rng = np.random.default_rng(66)
    k, v = rng.standard_normal((2, n, kvh, hd)) * 0.5
    u = np.sign(rng.standard_normal(hd))
    k[32:64] = 4 * u
    v[32:64] = 0
    stands = [z.transpose(1, 0, 2) for z in c.set(0, k, v)]
    q = rng.standard_normal((n, nh, hd)) * 0.1 + (15 + 5 * rng.random((n, nh, 1))) * u / 4 / hd * hd ** 0.5
    q *= 4
    qd, q = _dev(q.reshape(n, -1), t)
    q = q.reshape(n, nh, hd)
    got = _attend(c, t, qd, nh, _i32([n]), _i32([0, n]), n, n).reshape(n, nh, hd)
    _tiles(1)
    want = U.attend_rows(q, *stands, 0, hd ** -0.5)
    s = np.abs(np.einsum("ihd,kd->ihk", q[::50].astype(np.float64), stands[0][0])).max() * hd ** -0.5
    assert 40 < s < 200
    for i in range(n):
        for h in (0, 31, 63):
            if 32 <= i < 64:  # (these see the block's first tokens: nothing but what lies under them)
                assert np.abs(want[i, h]).max() < 1e-10
            assert rel_l2(got[i, h], want[i, h]) < TOL[t] + s * 2.0 ** -21, (i, h)
    Q.check_device()


@pytest.mark.parametrize("t,hd", WIDTHS)
def test_tiles_nan_and_infinity(t, hd):
    """What is not finite, in open rows or as a page's scale, reaches exactly the rows that see it; past the end, none."""
    nh, kvh = 32, 2
    lens, q_len = [847] * 4, [800] * 4
    c, stands = _filled(lens, 864, kvh, hd, seed=67)
    c.ko[int(c.slot[0]), 0, :, 10, 3] = float("nan")   # token 842
    c.vo[int(c.slot[1]), 0, :, 10, 3] = float("-inf")  # token 842
    c.vs[int(c.table[2, 3])] = float("nan")            # tokens 96 .. 127
    c.ks[int(c.table[3, 20])] = float("nan")           # tokens 640 .. 671
    c.ko[int(c.slot[3]), 0, :, 15:] = float("nan")     # past the end
    c.vo[int(c.slot[3]), 0, :, 15:] = float("inf")
    qd, q = _dev(np.random.default_rng(68).standard_normal((3200, nh * hd)), t)
    got = _attend(c, t, qd, nh, _i32(lens), _i32(_starts(q_len)), 800, 847)
    _tiles()
    first_bad = [842, 842, 96, 640]
    _check_rows(got, q, stands, lens, q_len, nh, TOL[t], rows=lambda s, i: 47 + i < first_bad[s])
    for s in range(4):
        assert np.isnan(got[800 * s + first_bad[s] - 47:800 * s + 800]).all(), s
    Q.check_device()


@pytest.mark.parametrize("t,hd", WIDTHS)
def test_tiles_report_what_lies_outside_the_cache(t, hd):
    """A page, a slot, a length out of range and rows beyond max_q_len: reported, the other sequences' rows are right."""
    nh, kvh = 32, 2
    lens, q_len = [607, 607, 602, 607], [400, 450, 400, 400]
    rng = np.random.default_rng(69)
    qd, q = _dev(rng.standard_normal((sum(q_len), nh * hd)), t)

    def run(change, expect, max_q=450):
        c, stands = _filled(lens, 608, kvh, hd, seed=70)
        kv = _i32(lens)
        change(c, kv)
        got = _attend(c, t, qd, nh, kv, _i32(_starts(q_len)), max_q, 607)
        _tiles()
        with pytest.raises(Q.QLError) as e:
            Q.check_device()
        assert e.value.status == Q.QL_EDEVICE and expect in str(e.value)
        _check_rows(got, q, stands, lens, q_len, nh, TOL[t], rows=lambda s, i: s != 1 and i % 7 == 0)

    run(lambda c, kv: c.td.__setitem__((1, 5), c.pages), "page")
    run(lambda c, kv: c.td.__setitem__((1, 5), -1), "page")
    run(lambda c, kv: c.sd.__setitem__(1, -1), "slot")
    run(lambda c, kv: kv.__setitem__(1, 609), "page")
    run(lambda c, kv: None, "more rows", max_q=413)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("tiles", [False, True])
def test_lengths_above_the_bound_are_read(t, tiles):
    """max_kv_len sizes the launch; longer sequences are read to their ends all the same."""
    nh, kvh, hd = 64, 8, 128
    q_len, lens = ([256, 100], [700, 1300]) if tiles else ([1, 3], [700, 2000])
    c, stands = _filled(lens, max(lens), kvh, hd, seed=71)
    qd, q = _dev(np.random.default_rng(72).standard_normal((sum(q_len), nh * hd)) * 1.5, t)
    for bound in (256, 0):
        got = _attend(c, t, qd, nh, _i32(lens), _i32(_starts(q_len)), max(q_len), bound)
        if bound:
            assert Q.kv8_attend_form()[0] == (Q.KV8_FORM_TILES if tiles else Q.KV8_FORM_SPLIT)
        _check_rows(got, q, stands, lens, q_len, nh, TOL[t])
    Q.check_device()


def test_overlapping_calls_with_a_workspace_each():
    """Two streams, each with its workspace, over and over: the bits of the calls alone."""
    import torch
    nh, kvh, hd, n = 14, 2, 128, 12000
    c, stands = _filled([n], n, kvh, hd, seed=73)
    rng = np.random.default_rng(74)
    q = [dev(rng.standard_normal((1, nh * hd)).astype(np.float32)) for _ in range(2)]
    kv = _i32([n])
    size = Q.kv8_attend_workspace(nh, kvh, hd, 1, 1, 1, n)
    ws = [torch.zeros(size, dtype=torch.uint8, device="cuda:0") for _ in range(2)]
    alone = [_attend(c, "f32", x, nh, kv, None, 1, n, ws=ws[0]) for x in q]
    form, ctas = Q.kv8_attend_form()
    assert form == Q.KV8_FORM_SPLIT and ctas > 8  # (several clusters: partials and counters in the workspace)
    outs = torch.full((2, 40, nh * hd), float("nan"), device="cuda:0")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    try:
        for i in range(40):
            for j, s in enumerate(streams):
                Q.set_stream(s.cuda_stream)
                Q.kv8_attend(c.view, Q.F32, q[j].data_ptr(), nh * hd, None, 0, outs[j, i].data_ptr(), nh * hd, nh, hd ** -0.5,
                             kv.data_ptr(), None, 1, 1, n, ws[j].data_ptr(), size)
        torch.cuda.synchronize()
    finally:
        Q.set_stream(torch.cuda.current_stream().cuda_stream)
    got = host(outs)
    for j in range(2):
        assert rel_l2(alone[j][0], U.attend(host(q[j]).reshape(nh, hd), *stands[0], n - 1, hd ** -0.5).ravel()) < TOL["f32"]
        assert (got[j] == alone[j][0]).all()


@pytest.mark.parametrize("nh,kvh,hd,n_seqs", [(16, 2, 64, 1), (16, 2, 128, 1)])
def test_tiles_one_heavy_key_over_many_light_ones(nh, kvh, hd, n_seqs):
    """One key 23.2 nats above 32799 others whose values all point the other way: each weighs 2^-33 of it, their sum
    3e-6.  Sums are fp32 and go tile by tile of 64 keys: one rounding of 2^-24 of the sum for each tile at most, in the
    sums and in the total, beside a weight's own 2^-32 of the heaviest."""
    n, rows = 32800, 1280
    c = Cache(1, n, kvh, hd, seed=75)
    k, v = np.zeros((2, n, kvh, hd))
    u = np.sign(np.random.default_rng(76).standard_normal(hd))
    k[0], v[0], v[1:] = 4 * u, u, -u
    stands = [z.transpose(1, 0, 2) for z in c.set(0, k, v)]
    q = np.tile(23.2 / 4 * hd ** -0.5 * u, (rows, nh)).astype(np.float32)
    got = _attend(c, "f32", dev(q), nh, _i32([n]), _i32([0, rows]), rows, n)
    _tiles(1)
    for i in (0, 700, rows - 1):
        want = U.attend(q[i].reshape(nh, hd), *stands, n - rows + i, hd ** -0.5)
        assert rel_l2(got[i], want.ravel()) < 2e-6 + n / 64 * 2.0 ** -23 + n * 2.0 ** -32, i
    Q.check_device()


def test_one_workspace_serves_every_head_dim():
    """Calls of head_dim 256, 128 and 64 with several key clusters each, in turn over one workspace that was zeroed once."""
    import torch
    bound = 1 << 16
    calls = []
    for hd, nh, kvh, n in ((256, 16, 4, 1), (128, 8, 1, 24), (64, 14, 2, 9), (256, 8, 2, 1), (128, 28, 4, 5), (64, 4, 1, 30)):
        lens = [3000 - 97 * s for s in range(n)]
        c, stands = _filled(lens, max(lens), kvh, hd, seed=79 + hd)
        q = np.random.default_rng(hd).standard_normal((n, nh * hd)).astype(np.float32)
        calls.append((hd, nh, kvh, n, lens, c, stands, q))
    ws = torch.zeros(max(Q.kv8_attend_workspace(x[1], x[2], x[0], x[3], x[3], 1, bound) for x in calls), dtype=torch.uint8,
                     device="cuda:0")
    for _ in range(2):
        for hd, nh, kvh, n, lens, c, stands, q in calls:
            got = _attend(c, "f32", dev(q), nh, _i32(lens), None, 1, bound, ws=ws)
            form, ctas = Q.kv8_attend_form()
            assert form == Q.KV8_FORM_SPLIT and ctas >= 16  # (two clusters or more)
            for s in range(n):
                want = U.attend(q[s].reshape(nh, hd), *stands[s], lens[s] - 1, hd ** -0.5)
                assert rel_l2(got[s], want.ravel()) < TOL["f32"], (hd, s)
    Q.check_device()


@pytest.mark.parametrize("t,hd", WIDTHS)
def test_tiles_under_a_wide_bound_of_rows(t, hd):
    """max_q_len of 2^20 (more tiles of rows than a grid's second and third dimension hold) for a call of 600 rows."""
    nh, kvh = 16, 1
    q_len, lens = [500, 100], [900, 333]
    c, stands = _filled(lens, max(lens), kvh, hd, seed=83)
    qd, q = _dev(np.random.default_rng(84).standard_normal((600, nh * hd)), t)
    got = _attend(c, t, qd, nh, _i32(lens), _i32(_starts(q_len)), 1 << 20, 1 << 20)
    _tiles()
    _check_rows(got, q, stands, lens, q_len, nh, TOL[t])
    Q.check_device()


def test_tiles_of_more_rows_than_a_grid_dimension():
    """65600 tiles of rows in one call, all but the last of them before the cache's first token (zeros)."""
    import torch
    nh, kvh, hd, rows, n = 64, 1, 64, 262400, 900
    c, stands = _filled([n], n, kvh, hd, seed=85)
    g = torch.Generator(device="cuda:0").manual_seed(86)
    q = torch.randn(rows, nh * hd, device="cuda:0", generator=g, dtype=torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    ws = torch.zeros(Q.kv8_attend_workspace(nh, kvh, hd, 1, rows, rows, 300000), dtype=torch.uint8, device="cuda:0")
    kv, st = _i32([n]), _i32([0, rows])
    Q.kv8_attend(c.view, Q.BF16, q.data_ptr(), nh * hd, None, 0, out.data_ptr(), nh * hd, nh, hd ** -0.5, kv.data_ptr(),
                 st.data_ptr(), rows, rows, 300000, ws.data_ptr(), ws.numel())
    _tiles()
    assert Q.last_launch_count() == 2
    torch.cuda.synchronize()
    assert not bool(out[:rows - n].any())
    got, qh = host(out[rows - n:].float()), host(q[rows - n:].float())
    _check_rows(got, qh, stands, [n], [n], nh, TOL["bf16"], rows=lambda s, i: i % 50 == 0 or i > n - 5)
    Q.check_device()


@pytest.mark.parametrize("bad", [2 ** 31 - 1, 2 ** 31 - 32, -1, -40, -2 ** 31])
@pytest.mark.parametrize("tiles", [False, True])
def test_lengths_at_the_ends_of_their_type_are_reported(tiles, bad):
    """A length no cache holds: no key is read (zeros), it is reported, and the other sequences' rows are right."""
    nh, kvh, hd = 32, 2, 128
    lens, q_len = ([607] * 4, [400] * 4) if tiles else ([607] * 4, [3] * 4)
    c, stands = _filled(lens, 608, kvh, hd, seed=87)
    qd, q = _dev(np.random.default_rng(88).standard_normal((sum(q_len), nh * hd)), "f32")
    got = _attend(c, "f32", qd, nh, _i32([607, bad, 607, 607]), _i32(_starts(q_len)), max(q_len), 607)
    assert Q.kv8_attend_form()[0] == (Q.KV8_FORM_TILES if tiles else Q.KV8_FORM_SPLIT)
    with pytest.raises(Q.QLError, match="page"):
        Q.check_device()
    assert not got[q_len[0]:2 * q_len[0]].any()
    _check_rows(got, q, stands, lens, q_len, nh, TOL["f32"], rows=lambda s, i: s != 1 and i % 7 == 0)


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
def test_f32_scores_over_open_rows(hd):
    """The scores themselves, from the weight that one token has against another of score 0, both in the open rows: two
    limbs of 22 bits (2^-23 of the rows' largest, three times their size), eight truncating additions of 2^-25 and an
    exponential of 2^-22 add up to less than 2^-21 of the scores' size, in the root of the mean square."""
    nh, kvh, n = 64, 1, 2
    rng = np.random.default_rng(hd + n)
    c = Cache(1, n, kvh, hd, seed=3)
    k, v = np.zeros((2, n, kvh, hd))
    k[0], v[0] = rng.standard_normal((kvh, hd)), 1
    stands = c.set(0, k, v)
    q = (rng.standard_normal((nh, hd)) * 2).astype(np.float32)
    got = _attend(c, "f32", dev(q.reshape(1, -1)), nh, _i32([n]), None, 1, n)[0].reshape(nh, hd)
    assert Q.kv8_attend_form()[0] == Q.KV8_FORM_SPLIT
    s = q.astype(np.float64) @ stands[0][0, 0] * hd ** -0.5
    p = got.mean(-1).astype(np.float64)
    good = (p > 0.002) & (p < 0.9)
    assert good.sum() > 20
    err = (np.log(p / (1 - p)) - s)[good]
    assert np.sqrt((err ** 2).mean()) < 2.0 ** -21 * np.sqrt((s[good] ** 2).mean())
    Q.check_device()


@pytest.mark.parametrize("t,hd", WIDTHS)
@pytest.mark.parametrize("tiles", [False, True])
def test_queries_that_are_not_finite_and_a_scale_of_zero(t, hd, tiles):
    """NaN and infinity in a head of a query reach that head of that row alone; a softmax scale of zero gives the mean."""
    nh, kvh = 32, 2
    lens, q_len = ([640, 607], [450, 400]) if tiles else ([640, 607], [3, 2])
    c, stands = _filled(lens, 640, kvh, hd, seed=99)
    q = np.random.default_rng(100).standard_normal((sum(q_len), nh, hd))
    bad = [(1, 3, np.nan), (2, 31, np.inf), (q_len[0], 16, -np.inf)]
    for row, h, x in bad:
        q[row, h, 5] = x
    qd, q = _dev(q.reshape(len(q), -1), t)
    for row, h, x in bad:  # (as they are, whatever the rounding makes of them)
        qd[row, h * hd + 5] = float(x)
    for scale in (hd ** -0.5, 0.0):
        got = _attend(c, t, qd, nh, _i32(lens), _i32(_starts(q_len)), max(q_len), 640, scale=scale).reshape(-1, nh, hd)
        assert Q.kv8_attend_form()[0] == (Q.KV8_FORM_TILES if tiles else Q.KV8_FORM_SPLIT)
        z = q.reshape(-1, nh, hd).copy()
        for row, h, _ in bad:
            assert np.isnan(got[row, h]).all(), (row, h)
            got[row, h] = z[row, h] = 0
        st = _starts(q_len)
        for s in range(2):
            want = U.attend_rows(z[st[s]:st[s + 1]], *stands[s], lens[s] - q_len[s], scale)
            for i in range(0, q_len[s], 7 if tiles else 1):
                for h in range(nh):
                    if not any(r == st[s] + i and b == h for r, b, _ in bad):
                        # (the mean of random values is small beside them: relative to these, too)
                        v = stands[s][1][h // 16][:lens[s] - q_len[s] + i + 1]
                        size = np.linalg.norm(want[i, h]) + (np.linalg.norm(np.abs(v).mean(0)) * 2.0 ** -9 if t == "bf16" else 0)
                        assert np.linalg.norm(got[st[s] + i, h] - want[i, h]) < 2 * TOL[t] * size, (scale, s, i, h)
    Q.check_device()
