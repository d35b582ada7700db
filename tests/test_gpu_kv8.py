"""The 8-bit KV cache's operators (ql_kv8_append, ql_kv8_attend, ql_kv8_gather) against 64-bit restatements.

Tolerances.  f32: a norm, a rotation or a softmax-weighted sum has tens to thousands of fp32 roundings of 2^-24
that add like a random walk, and weights from a 2^-22 exponential: 2e-6 relative L2 (a few 2^-22).  bf16 outputs:
one rounding of at most 2^-9 (2e-3 in L2), or of operands of 16 bits besides: 4e-3.  Bytes: a value within 2^-20 of
its own size of a tie may round either way, so a byte differs by at most one, in at most 1 of 2000 values."""
import numpy as np
import pytest

import blog_b200 as Q
import kv8_util as U
from gpu_util import dev, host, rel_l2

pytestmark = pytest.mark.gpu
TOL = {"f32": 2e-6, "bf16": 4e-3}


@pytest.fixture(scope="module", autouse=True)
def _stream():
    import torch
    torch.cuda.init()
    Q.init(0)
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    yield
    Q.check_device()


class Cache:
    """A cache on the device, its pages in a shuffled order with spare ones between, slots permuted."""

    def __init__(self, n_seqs, max_tokens, kvh, hd, seed=0, slots=True):
        import torch
        rng = np.random.default_rng(seed)
        self.per = (max_tokens + 31) // 32 or 1
        self.n, self.kvh, self.hd = n_seqs, kvh, hd
        self.pages = n_seqs * self.per + 3
        self.table = rng.permutation(self.pages)[:n_seqs * self.per].reshape(n_seqs, self.per).astype(np.int32)
        self.slot = rng.permutation(n_seqs + 2)[:n_seqs].astype(np.int32) if slots else np.arange(n_seqs, dtype=np.int32)
        shape = (self.pages, kvh, 32, hd)
        self.kc, self.vc = (torch.full(shape, 77, dtype=torch.uint8, device="cuda:0") for _ in range(2))
        self.ks, self.vs = (torch.full(shape[:2], float("nan"), device="cuda:0") for _ in range(2))
        self.ko, self.vo = (torch.full((n_seqs + 2, 2, kvh, 32, hd), float("nan"), device="cuda:0") for _ in range(2))
        self.td, self.sd = dev(self.table), dev(self.slot) if slots else None
        self.view = Q.kv8_cache(self.kc.data_ptr(), self.vc.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(),
                                self.ko.data_ptr(), self.vo.data_ptr(), self.td.data_ptr(),
                                self.sd.data_ptr() if slots else None, self.pages, n_seqs + 2, n_seqs, self.per, kvh, hd)

    def set(self, seq, k, v):
        """Contents written from the host: k, v [tokens][kvh][hd]; returns what stands there, in 64 bits."""
        import torch
        t = len(k)
        out = []
        for x, c, s, o in ((k, self.kc, self.ks, self.ko), (v, self.vc, self.vs, self.vo)):
            x = np.array(x, np.float64)
            for b in range(t // 32):
                for h in range(self.kvh):
                    code, sc = U.quantize(x[32 * b:32 * b + 32, h].astype(np.float32))
                    sc = np.float32(sc)
                    c[int(self.table[seq, b]), h] = torch.from_numpy(code.astype(np.uint8)).cuda()
                    s[int(self.table[seq, b]), h] = float(sc)
                    x[32 * b:32 * b + 32, h] = (code - 128.0) * np.float64(sc)
            if t % 32:
                r = x[t // 32 * 32:].astype(np.float32)
                o[int(self.slot[seq]), (t // 32) % 2, :, :t % 32] = torch.from_numpy(r).cuda().transpose(0, 1)
                x[t // 32 * 32:] = r
            out.append(x)
        return out


def _i32(v):
    return dev(np.asarray(v, np.int32))


def _dev(x, t):
    """A device array of type t ("f32" or "bf16") and its values in f32."""
    import torch
    x = np.asarray(x, np.float32)
    if t == "f32":
        return dev(x), x
    return torch.from_numpy(x).cuda().to(torch.bfloat16), U.bf16_round(x)


def _code(t):
    return Q.F32 if t == "f32" else Q.BF16


def _append(cache, t, x, nh, q_out, kv_len, q_start, max_q, gq=None, gk=None, eps=1e-6, rope=None, rot=0, pad=0):
    """x: device [rows][(nh + 2 kvh) hd + pad], q, k and v side by side."""
    kvh, hd = cache.kvh, cache.hd
    w, el = x.shape[1], x.element_size()
    p = x.data_ptr() + (el * pad if pad else 0)
    rows = x.shape[0]
    Q.kv8_append(cache.view, _code(t), p if nh else None, w, p + nh * hd * el, w, p + (nh + kvh) * hd * el, w,
                 q_out.data_ptr() if nh else None, q_out.shape[1] if nh else 0, nh, gq.data_ptr() if gq is not None else None,
                 gk.data_ptr() if gk is not None else None, eps, rope.data_ptr() if rope is not None else None, rot,
                 rope.shape[0] if rope is not None else 0, kv_len.data_ptr(),
                 q_start.data_ptr() if q_start is not None else None, rows, max_q)


def _gather(cache, t, start, count, kv_len):
    import torch
    dt = torch.float32 if t == "f32" else torch.bfloat16
    outs = [torch.full((cache.n, count, cache.kvh, cache.hd), 9.0, dtype=dt, device="cuda:0") for _ in range(2)]
    Q.kv8_gather(cache.view, _code(t), outs[0].data_ptr(), outs[1].data_ptr(), start.data_ptr() if start is not None else None,
                 count, kv_len.data_ptr())
    return [host(o.float()) for o in outs]


def _check_cache(cache, k, v, lens, exact_bytes=False):
    """The cache holds k, v (lists of [tokens][kvh][hd] in 64 bits): bytes, scales and open rows."""
    kc, vc, ks, vs, ko, vo = (host(x) for x in (cache.kc, cache.vc, cache.ks, cache.vs, cache.ko, cache.vo))
    off = total = 0
    for s in range(cache.n):
        t = lens[s]
        for x, c, sc, o in ((k[s], kc, ks, ko), (v[s], vc, vs, vo)):
            for b in range(t // 32):
                pg = cache.table[s, b]
                for h in range(cache.kvh):
                    code, want = U.quantize(x[32 * b:32 * b + 32, h])
                    assert abs(sc[pg, h] - want) <= 2e-6 * want
                    d = np.abs(code - c[pg, h].astype(int))
                    assert d.max() <= 1
                    off += int(d.sum())
                    total += d.size
            if t % 32:
                got = o[cache.slot[s], (t // 32) % 2, :, :t % 32].transpose(1, 0, 2)
                assert rel_l2(got, x[t // 32 * 32:]) < TOL["f32"]
    assert off <= (0 if exact_bytes else total / 2000)


LAYOUTS = [(28, 4, 128, 128), (16, 4, 256, 64), (14, 2, 64, 64), (6, 3, 96, 48), (5, 1, 32, 0), (8, 2, 160, 80),
           (4, 4, 192, 192), (2, 1, 224, 28)]


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("nh,kvh,hd,rot", LAYOUTS)
def test_append_prompts_then_tokens(nh, kvh, hd, rot, t):
    """Prompts of 1, 31, 32, 33 and 100 tokens and an empty one, then a second call that continues each
    (the first blocks' earlier rows come from the open rows, which the call's last block overwrites), then one
    token each: q, bytes, scales and open rows."""
    import torch
    rng = np.random.default_rng(hd + nh)
    cache = Cache(6, 320, kvh, hd, seed=hd)
    gq, gk = rng.standard_normal(hd).astype(np.float32), 1 + 0.3 * rng.standard_normal(hd).astype(np.float32)
    gqd, gkd = dev(gq), dev(gk)
    table = U.rope_table(320, rot) if rot else None
    rd = dev(table) if rot else None
    k, v = [np.zeros((0, kvh, hd)) for _ in range(6)], [np.zeros((0, kvh, hd)) for _ in range(6)]
    lens = np.zeros(6, int)
    for step, q_len in enumerate([[1, 31, 32, 33, 0, 100], [70, 2, 0, 95, 64, 130], None]):
        single = q_len is None
        q_len = [1] * 6 if single else q_len
        lens = lens + q_len
        rows = sum(q_len)
        x = rng.standard_normal((rows, (nh + 2 * kvh) * hd)) * np.exp(rng.standard_normal((rows, 1)))
        xd, x = _dev(x, t)
        q_out = torch.full((rows, nh * hd), float("nan"), dtype=xd.dtype, device="cuda:0")
        starts = np.concatenate([[0], np.cumsum(q_len)])
        _append(cache, t, xd, nh, q_out, _i32(lens), None if single else _i32(starts), max(q_len), gqd, gkd, 1e-6, rd, rot)
        assert Q.last_launch_count() == 1
        want = np.zeros((rows, nh * hd))
        for s in range(6):
            for i in range(q_len[s]):
                r, pos = starts[s] + i, lens[s] - q_len[s] + i
                z = x[r].reshape(-1, hd)
                want[r] = U.norm_rope(z[:nh], gq, 1e-6, table, pos, rot).ravel()
                k[s] = np.concatenate([k[s], U.norm_rope(z[nh:nh + kvh], gk, 1e-6, table, pos, rot)[None]])
                v[s] = np.concatenate([v[s], z[nh + kvh:].astype(np.float64)[None]])
        assert rel_l2(host(q_out.float()), want) < TOL[t]
        _check_cache(cache, k, v, lens)
    Q.check_device()


def test_append_does_not_depend_on_the_cuts():
    """300 tokens in one call, in calls of 7, and token by token: the same bytes, scales and open rows, bit for bit."""
    import torch
    kvh, hd, n = 2, 128, 300
    rng = np.random.default_rng(7)
    x = dev(rng.standard_normal((n, 2 * kvh * hd)).astype(np.float32))
    gk, rd = dev(np.ones(hd, np.float32)), dev(U.rope_table(n, hd))
    got = []
    for step in (n, 7, 1):
        c = Cache(1, n, kvh, hd, seed=1)
        for lo in range(0, n, step):
            m = min(step, n - lo)
            _append(c, "f32", x[lo:lo + m], 0, None, _i32([lo + m]), _i32([0, m]) if step > 1 else None, m, None, gk, 1e-6,
                    rd, hd)
        Q.check_device()
        used = torch.from_numpy(c.table.ravel().astype(np.int64)).cuda()[:n // 32]
        got.append([host(z) for z in (c.kc[used], c.vc[used], c.ks[used], c.vs[used],
                                      c.ko[int(c.slot[0]), (n // 32) % 2, :, :n % 32], c.vo[int(c.slot[0]), (n // 32) % 2, :, :n % 32])])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert np.array_equal(a, b)


def test_tokens_taken_back():
    """kv_len goes back by 32 (over a block's end) and other tokens follow: as if the first had never been."""
    kvh, hd = 2, 64
    rng = np.random.default_rng(9)
    x = rng.standard_normal((140, 2 * kvh * hd)).astype(np.float32)
    y = rng.standard_normal((40, 2 * kvh * hd)).astype(np.float32)
    c = Cache(1, 200, kvh, hd, seed=2)
    _append(c, "f32", dev(x), 0, None, _i32([140]), _i32([0, 140]), 140)
    _append(c, "f32", dev(y), 0, None, _i32([148]), _i32([0, 40]), 40)  # tokens 108 .. 147 anew
    z = np.concatenate([x[:108], y]).reshape(148, 2, kvh, hd)
    _check_cache(c, [z[:, 0].astype(np.float64)], [z[:, 1].astype(np.float64)], [148], exact_bytes=True)
    Q.check_device()


@pytest.mark.parametrize("what", ["nan", "inf", "zero", "tiny", "huge"])
def test_append_blocks_out_of_the_ordinary(what):
    """A block with NaN or infinity has a NaN scale, one of zeros scale 0 and bytes 128, the smallest and the
    largest magnitudes keep their bytes; the neighbouring heads and blocks are not touched."""
    kvh, hd = 2, 64
    rng = np.random.default_rng(11)
    x = rng.standard_normal((96, 2, kvh, hd)).astype(np.float32)
    b = slice(32, 64)
    if what == "nan":
        x[40, 0, 1, 3] = np.nan
    elif what == "inf":
        x[40, 0, 1, 3] = -np.inf
    elif what == "zero":
        x[b, 0, 1] = 0
    else:
        x[b, 0, 1] *= {"tiny": 1e-36, "huge": 5e37}[what]
    c = Cache(1, 96, kvh, hd, seed=3)
    _append(c, "f32", dev(x.reshape(96, -1)), 0, None, _i32([96]), _i32([0, 96]), 96)
    kc, ks = host(c.kc), host(c.ks)
    for blk in range(3):
        for h in range(kvh):
            code, sc = U.quantize(x[32 * blk:32 * blk + 32, 0, h])
            pg = c.table[0, blk]
            if np.isnan(sc):
                assert np.isnan(ks[pg, h])
                continue
            assert abs(ks[pg, h] - sc) <= 2e-7 * sc
            assert np.abs(code - kc[pg, h]).max() <= (1 if sc else 0)
    Q.check_device()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_append_odd_strides_and_alignment(t):
    """Rows a few elements longer than their heads, starting one element off: the element-wise accesses."""
    import torch
    nh, kvh, hd, rot = 6, 2, 128, 128
    rng = np.random.default_rng(13)
    w = (nh + 2 * kvh) * hd + 5
    xd, x = _dev(rng.standard_normal((37, w)), t)
    c = Cache(1, 64, kvh, hd, seed=4, slots=False)
    out = torch.zeros((37, nh * hd + 3), dtype=xd.dtype, device="cuda:0")
    table = U.rope_table(64, rot)
    g = np.ones(hd, np.float32)
    _append(c, t, xd, nh, out, _i32([37]), _i32([0, 37]), 37, dev(g), dev(g), 1e-6, dev(table), rot, pad=1)
    x = x[:, 1:1 + (nh + 2 * kvh) * hd].reshape(37, -1, hd)
    want = np.stack([U.norm_rope(x[i, :nh], g, 1e-6, table, i, rot) for i in range(37)])
    k = np.stack([U.norm_rope(x[i, nh:nh + kvh], g, 1e-6, table, i, rot) for i in range(37)])
    assert rel_l2(host(out.float())[:, :nh * hd], want.reshape(37, -1)) < TOL[t]
    assert (host(out.float())[:, nh * hd:] == 0).all()
    _check_cache(c, [k], [x[:, nh + kvh:].astype(np.float64)], [37])


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1.0, 1e-20, 1e-34, 1e32])
def test_codes_are_the_rounded_quotients(size, t):
    """V is stored as it comes: its bytes are rint(x / scale) + 128 of the f32 quotient, bit for bit, ties of bf16
    values and of halves of the largest among them."""
    kvh, hd, n = 2, 128, 640
    rng = np.random.default_rng(17)
    x = rng.standard_normal((n, 2, kvh, hd)) * size
    x[:, :, :, ::7] = rng.integers(-254, 255, x[:, :, :, ::7].shape) * (size / 254)
    xd, x = _dev(x, t)
    c = Cache(1, n, kvh, hd, seed=6)
    _append(c, t, xd.reshape(n, -1), 0, None, _i32([n]), _i32([0, n]), n)
    vc, vs = host(c.vc), host(c.vs)
    for b in range(n // 32):
        for h in range(kvh):
            z = x[32 * b:32 * b + 32, 1, h]
            scale = np.abs(z).max() / np.float32(127)
            assert vs[c.table[0, b], h] == scale
            assert np.array_equal(vc[c.table[0, b], h], np.rint(z / scale) + 128)
    Q.check_device()


def test_gather():
    """Positions before, in and past a sequence, closed pages and open rows, an empty sequence."""
    kvh, hd = 3, 96
    c = Cache(3, 100, kvh, hd, seed=5)
    rng = np.random.default_rng(15)
    lens = [100, 33, 0]
    stands = [c.set(s, *rng.standard_normal((2, n, kvh, hd))) for s, n in enumerate(lens)]
    for t in ("f32", "bf16"):
        got = _gather(c, t, _i32([-3, 20, 0]), 104, _i32(lens))
        for j in range(2):
            for s, (n, first) in enumerate(zip(lens, (-3, 20, 0))):
                want = np.zeros((104, kvh, hd))
                for i in range(104):
                    if 0 <= first + i < n:
                        want[i] = stands[s][j][first + i]
                if t == "bf16":
                    want = U.bf16_round(want.astype(np.float32))
                assert np.array_equal(got[j][s], want.astype(np.float32))
    Q.check_device()


def _attend(cache, t, q, nh, kv_len, q_start, max_q, max_kv, scale=None, gate=None, ws=None):
    import torch
    rows, hd = q.shape[0], cache.hd
    out = torch.full((rows, nh * hd), float("nan"), dtype=q.dtype, device="cuda:0")
    n = Q.kv8_attend_workspace(nh, cache.kvh, hd, cache.n, rows, max_q, max_kv)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda:0") if ws is None else ws
    Q.kv8_attend(cache.view, _code(t), q.data_ptr(), q.shape[1], gate.data_ptr() if gate is not None else None,
                 gate.shape[1] if gate is not None else 0, out.data_ptr(), nh * hd, nh, hd ** -0.5 if scale is None else scale,
                 kv_len.data_ptr(), q_start.data_ptr() if q_start is not None else None, rows, max_q, max_kv, ws.data_ptr(),
                 ws.numel())
    return host(out.float())


def _filled(lens, max_tokens, kvh, hd, seed):
    c = Cache(len(lens), max_tokens, kvh, hd, seed=seed)
    rng = np.random.default_rng(seed + 100)
    stands = []
    for s, n in enumerate(lens):
        k, v = rng.standard_normal((2, n, kvh, hd))
        k *= np.exp(0.5 * rng.standard_normal((n // 32 + 1, 1, 1))).repeat(32, 0)[:n]  # scales of unlike sizes
        v *= np.exp(rng.standard_normal((n // 32 + 1, 1, 1))).repeat(32, 0)[:n]
        stands.append([z.transpose(1, 0, 2) for z in c.set(s, k, v)])
    return c, stands


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("nh,kvh,hd,rot", LAYOUTS + [(64, 8, 128, 0), (40, 2, 64, 0), (3, 3, 128, 0)])
def test_attend_single_tokens(nh, kvh, hd, rot, t):
    """One token of sequences of 1, 31, 32, 33, 64, 95, 200 and 1000 tokens, and an idle one (zeros)."""
    lens = [1, 31, 32, 33, 0, 64, 95, 200, 1000]
    c, stands = _filled(lens, 1000, kvh, hd, seed=hd + nh)
    rng = np.random.default_rng(hd)
    qd, q = _dev(rng.standard_normal((9, nh * hd)) * 1.5, t)
    gd, g = _dev(rng.standard_normal((9, nh * hd)), t)
    for gate in (False, True):
        got = _attend(c, t, qd, nh, _i32(lens), None, 1, 1000, gate=gd if gate else None)
        for s, n in enumerate(lens):
            want = U.attend(q[s].reshape(nh, hd), *stands[s], n - 1, hd ** -0.5, g[s].reshape(nh, hd) if gate else None)
            if n == 0:
                assert (got[s] == 0).all()
            else:
                assert rel_l2(got[s], want.ravel()) < TOL[t], (s, n)
    Q.check_device()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("nh,kvh,hd", [(28, 4, 128), (16, 4, 256), (14, 2, 64), (6, 3, 96), (8, 1, 32), (16, 2, 160)])
def test_attend_ragged_queries(nh, kvh, hd, t):
    """Prompts and chunks (rows that begin inside a page, fill pages and leave one open), a sequence without rows."""
    q_len, lens = [70, 5, 0, 33, 1, 129], [70, 100, 50, 64, 97, 300]
    c, stands = _filled(lens, 320, kvh, hd, seed=hd + 1)
    rng = np.random.default_rng(hd + 2)
    starts = np.concatenate([[0], np.cumsum(q_len)])
    qd, q = _dev(rng.standard_normal((starts[-1], nh * hd)) * 1.5, t)
    got = _attend(c, t, qd, nh, _i32(lens), _i32(starts), max(q_len), max(lens))
    for s in range(len(lens)):
        for i in range(q_len[s]):
            r = starts[s] + i
            want = U.attend(q[r].reshape(nh, hd), *stands[s], lens[s] - q_len[s] + i, hd ** -0.5)
            assert rel_l2(got[r], want.ravel()) < TOL[t], (s, i)
    Q.check_device()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("nh,kvh,hd", [(28, 4, 128), (14, 2, 64), (16, 2, 128), (3, 3, 64), (64, 2, 64), (8, 1, 256)])
@pytest.mark.parametrize("gate", [False, True])
def test_attend_prompts(nh, kvh, hd, t, gate):
    """Prompts and later chunks of hundreds of tokens beside single tokens and a sequence without rows: full tiles of
    keys, tiles that end inside one, an open block of 1 to 31 tokens or none, rows that end inside a tile."""
    q_len = [300, 1, 0, 257, 129, 32, 64]
    lens = [300, 1000, 64, 700, 129 + 96, 32, 1088]
    c, stands = _filled(lens, 1100, kvh, hd, seed=hd + 3)
    rng = np.random.default_rng(hd + 4)
    starts = np.concatenate([[0], np.cumsum(q_len)])
    qd, q = _dev(rng.standard_normal((starts[-1], nh * hd)) * 1.5, t)
    gd, g = _dev(rng.standard_normal((starts[-1], nh * hd)), t)
    got = _attend(c, t, qd, nh, _i32(lens), _i32(starts), max(q_len), max(lens), gate=gd if gate else None)
    for s in range(len(lens)):
        r = slice(starts[s], starts[s + 1])
        if q_len[s] == 0:
            continue
        want = U.attend_rows(q[r].reshape(-1, nh, hd), *stands[s], lens[s] - q_len[s], hd ** -0.5,
                             g[r].reshape(-1, nh, hd) if gate else None).reshape(-1, nh * hd)
        for i in range(q_len[s]):
            assert rel_l2(got[r][i], want[i]) < TOL[t], (s, i)
    Q.check_device()


@pytest.mark.parametrize("hd", [64, 128])
def test_attend_prompt_scores_of_every_size_and_signs(hd):
    """Scores of +-1e3, equal scores, tiny and huge queries, values whose scales lie 1e12 apart, a block of zeros, and a
    negative softmax scale, in a prompt."""
    nh, kvh, n = 8, 1, 300
    c = Cache(1, n, kvh, hd, seed=41)
    rng = np.random.default_rng(42)
    k, v = rng.standard_normal((2, n, kvh, hd))
    v[:64] *= 1e-6
    v[64:96] *= 1e6
    v[96:128] = 0
    k[128:160] = 0
    stands = [z.transpose(1, 0, 2) for z in c.set(0, k, v)]
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    q[:, 1] *= 100
    q[:, 2] = 0
    q[:, 3] *= 1e-30
    q[:, 4] = -q[:, 1]
    for scale in (hd ** -0.5, -hd ** -0.5):
        got = _attend(c, "f32", dev(q.reshape(n, -1)), nh, _i32([n]), _i32([0, n]), n, n, scale=scale).reshape(n, nh, hd)
        want = U.attend_rows(q, *stands, 0, scale)
        for h in range(nh):
            s = np.abs(stands[0][0] @ q[:, h].T.astype(np.float64)).max() * hd ** -0.5
            for i in range(n):
                assert rel_l2(got[i, h], want[i, h]) < 2e-6 + s * 2.0 ** -21, (h, i)
    Q.check_device()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_attend_prompt_nan_and_infinity(hd, t):
    """As for the few rows below: what is not finite reaches exactly the rows that see it, in a prompt."""
    nh, kvh = 4, 2
    lens, q_len = [207, 207, 207, 207], [200, 200, 200, 200]
    c, stands = _filled(lens, 224, kvh, hd, seed=43)
    c.ko[int(c.slot[0]), 0, :, 10, 3] = float("nan")   # token 202
    c.vo[int(c.slot[1]), 0, :, 10, 3] = float("-inf")  # token 202
    c.vs[int(c.table[2, 1])] = float("nan")            # tokens 32 .. 63
    c.ks[int(c.table[3, 5])] = float("nan")            # tokens 160 .. 191
    c.ko[int(c.slot[3]), 0, :, 15:] = float("nan")     # past the end
    c.vo[int(c.slot[3]), 0, :, 15:] = float("inf")
    rng = np.random.default_rng(44)
    starts = np.concatenate([[0], np.cumsum(q_len)])
    qd, q = _dev(rng.standard_normal((800, nh * hd)), t)
    got = _attend(c, t, qd, nh, _i32(lens), _i32(starts), 200, 207)
    for s, first_bad in enumerate([202, 202, 32, 160]):
        want = U.attend_rows(q[starts[s]:starts[s + 1]].reshape(-1, nh, hd), *stands[s], 7, hd ** -0.5).reshape(-1, nh * hd)
        for i in range(200):
            if 7 + i >= first_bad:
                assert np.isnan(got[starts[s] + i]).all(), (s, i)
            else:
                assert rel_l2(got[starts[s] + i], want[i]) < TOL[t], (s, i)


@pytest.mark.parametrize("nh,kvh,hd,n", [(64, 64, 32, 8200), (64, 8, 128, 8200), (16, 4, 256, 5000)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_attend_many_rows(nh, kvh, hd, n, t):
    """One call of more row groups than a grid dimension of 65535 holds, and prompts over thousands of keys (rows at
    both ends and at tile edges): K and V by ql_kv8_append, read back by ql_kv8_gather for the restatement."""
    import torch
    c = Cache(1, n, kvh, hd, seed=51)
    g = torch.Generator(device="cuda:0").manual_seed(52)
    dt = torch.float32 if t == "f32" else torch.bfloat16
    x = torch.randn(n, 2 * kvh * hd, generator=g, device="cuda:0").to(dt)
    _append(c, t, x, 0, None, _i32([n]), _i32([0, n]), n)
    k, v = (z[0].transpose(1, 0, 2).astype(np.float64) for z in _gather(c, "f32", None, n, _i32([n])))
    q = (torch.randn(n, nh * hd, generator=g, device="cuda:0") * 1.5).to(dt)
    got = _attend(c, t, q, nh, _i32([n]), _i32([0, n]), n, n)
    qh = host(q.float())
    for i in (0, 31, 32, 63, 64, 127, 1000, n // 2 + 1, n - 33, n - 2, n - 1):
        want = U.attend(qh[i].reshape(nh, hd), k, v, i, hd ** -0.5)
        assert rel_l2(got[i], want.ravel()) < TOL[t], i
    Q.check_device()


@pytest.mark.parametrize("n_seqs,kvh,max_kv", [(64, 8, 1 << 17), (2, 2, 1 << 20), (37, 6, 1 << 20)])
def test_attend_under_wide_bounds(n_seqs, kvh, max_kv):
    """Bounds far above the lengths, with few and many groups of rows: nothing is written behind the workspace, whose
    size the bounds do not change, and it is left zeroed where the next call counts."""
    import torch
    nh, hd = 2 * kvh, 128
    lens = [40 + 3 * s for s in range(n_seqs)]
    c, stands = _filled(lens, max(lens), kvh, hd, seed=53)
    q = torch.randn((n_seqs, nh * hd), device="cuda:0", generator=torch.Generator(device="cuda:0").manual_seed(54))
    n = Q.kv8_attend_workspace(nh, kvh, hd, n_seqs, n_seqs, 1, max_kv)
    assert n == Q.kv8_attend_workspace(nh, kvh, hd, 1, 1, 1, 64)
    room = torch.cat([torch.zeros(n, dtype=torch.uint8), torch.full((1 << 24,), 91, dtype=torch.uint8)]).to("cuda:0")
    for _ in range(2):
        got = _attend(c, "f32", q, nh, _i32(lens), None, 1, max_kv, ws=room[:n])
        for s in range(0, n_seqs, 7):
            want = U.attend(host(q)[s].reshape(nh, hd), *stands[s], lens[s] - 1, hd ** -0.5)
            assert rel_l2(got[s], want.ravel()) < TOL["f32"], s
    assert bool((room[n:] == 91).all())


@pytest.mark.parametrize("n_seqs", [2, 127, 128, 129])
@pytest.mark.parametrize("ragged", [False, True])
def test_attend_waves_of_unlike_lengths(n_seqs, ragged):
    """More CTAs than run at once, lengths in no order with many equal ones and idle sequences: every row is its own
    sequence's, whichever starts first."""
    import torch
    kvh, hd, nh = 16, 64, 32
    rng = np.random.default_rng(55)
    lens = [int(x) for x in rng.choice([0, 1, 33, 64, 64, 150, 300], n_seqs)]
    lens[-1] = 300
    q_len = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 6, n_seqs))] if ragged else [1] * n_seqs
    q_len[-1] = 5 if ragged else 1
    starts = np.concatenate([[0], np.cumsum(q_len)])
    c, stands = _filled(lens, 300, kvh, hd, seed=56)
    q = torch.randn((int(starts[-1]), nh * hd), device="cuda:0", generator=torch.Generator(device="cuda:0").manual_seed(57))
    got = _attend(c, "f32", q, nh, _i32(lens), _i32(starts) if ragged else None, 5 if ragged else 1, 300)
    for s in range(n_seqs):
        for i in range(q_len[s]):
            row = got[starts[s] + i]
            if lens[s] == 0:
                assert not row.any(), s
                continue
            want = U.attend(host(q)[starts[s] + i].reshape(nh, hd), *stands[s], lens[s] - q_len[s] + i, hd ** -0.5)
            assert rel_l2(row, want.ravel()) < TOL["f32"], (s, i)
    Q.check_device()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_attend_long_cache(t):
    """20011 tokens of one sequence: many key splits, merged in a fixed order (twice the same bits)."""
    import torch
    nh, kvh, hd, n = 14, 2, 128, 20011
    c, stands = _filled([n], n, kvh, hd, seed=21)
    qd, q = _dev(np.random.default_rng(22).standard_normal((1, nh * hd)) * 2, t)
    ws = torch.zeros(Q.kv8_attend_workspace(nh, kvh, hd, 1, 1, 1, 1 << 16), dtype=torch.uint8, device="cuda:0")
    got = [_attend(c, t, qd, nh, _i32([n]), None, 1, 1 << 16, ws=ws) for _ in range(3)]
    want = U.attend(q[0].reshape(nh, hd), *stands[0], n - 1, hd ** -0.5)
    assert rel_l2(got[0][0], want.ravel()) < TOL[t]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_attend_scores_of_every_size():
    """Scores of +-1e4 (one key takes all the weight), equal scores, queries of zeros and of 1e-30 and 1e30, values
    whose scales lie 1e12 apart."""
    nh, kvh, hd, n = 8, 1, 128, 200
    c = Cache(1, n, kvh, hd, seed=23)
    rng = np.random.default_rng(24)
    k, v = rng.standard_normal((2, n, kvh, hd))
    v[:64] *= 1e-6
    v[64:96] *= 1e6
    stands = [z.transpose(1, 0, 2) for z in c.set(0, k, v)]
    q = rng.standard_normal((nh, hd)).astype(np.float32)
    q[1] *= 1e3
    q[2] = 0
    q[3] *= 1e-30
    q[4] *= 1e30
    q[5] = -q[1]
    got = _attend(c, "f32", dev(q.reshape(1, -1)), nh, _i32([n]), None, 1, n)[0].reshape(nh, hd)
    want = U.attend(q, *stands, n - 1, hd ** -0.5)
    for h in range(nh):
        # a score of size S carries an error of 2^-22 S into the exponent
        s = np.abs(stands[0][0] @ q[h].astype(np.float64)).max() * hd ** -0.5
        assert rel_l2(got[h], want[h]) < 2e-6 + (0 if s > 1e6 else s * 2.0 ** -21), h


def test_attend_nan_and_infinity_reach_only_those_who_see_them():
    """NaN and infinity in open rows, a NaN scale of a closed page, and NaN beyond a sequence's end: rows before them
    are finite and right, rows that see them NaN, other sequences untouched."""
    import torch
    nh, kvh, hd = 4, 2, 64
    lens, q_len = [80, 80, 80, 80], [40, 40, 40, 40]
    c, stands = _filled(lens, 96, kvh, hd, seed=25)
    c.ko[int(c.slot[0]), 0, :, 10, 3] = float("nan")   # token 74 of sequence 0
    c.vo[int(c.slot[1]), 0, :, 10, 3] = float("-inf")  # token 74 of sequence 1
    c.vs[int(c.table[2, 1])] = float("nan")            # tokens 32 .. 63 of sequence 2
    c.ko[int(c.slot[3]), 0, :, 16:] = float("nan")     # past the end of sequence 3
    c.vo[int(c.slot[3]), 0, :, 16:] = float("inf")
    rng = np.random.default_rng(26)
    starts = np.concatenate([[0], np.cumsum(q_len)])
    q = rng.standard_normal((160, nh * hd)).astype(np.float32)
    got = _attend(c, "f32", dev(q), nh, _i32(lens), _i32(starts), 40, 80)
    first_bad = [74, 74, 32, 80]
    for s in range(4):
        for i in range(40):
            pos, r = 40 + i, starts[s] + i
            if pos >= first_bad[s]:
                assert np.isnan(got[r]).all(), (s, pos)
            else:
                assert rel_l2(got[r], U.attend(q[r].reshape(nh, hd), *stands[s], pos, hd ** -0.5).ravel()) < TOL["f32"]
    torch.cuda.synchronize()


def test_attend_strides():
    """Rows of q, gate and out inside wider rows, starting one element off."""
    import torch
    nh, kvh, hd = 6, 2, 64
    lens = [50, 33, 7]
    c, stands = _filled(lens, 64, kvh, hd, seed=27)
    for t, dt in (("f32", torch.float32), ("bf16", torch.bfloat16)):
        rng = np.random.default_rng(28)
        qd, q = _dev(rng.standard_normal((3, nh * hd + 9)), t)
        gd, g = _dev(rng.standard_normal((3, nh * hd + 4)), t)
        out = torch.zeros((3, nh * hd + 7), dtype=dt, device="cuda:0")
        ws = torch.zeros(Q.kv8_attend_workspace(nh, kvh, hd, 3, 3, 1, 64), dtype=torch.uint8, device="cuda:0")
        el = qd.element_size()
        Q.kv8_attend(c.view, _code(t), qd.data_ptr() + el, nh * hd + 9, gd.data_ptr() + el, nh * hd + 4, out.data_ptr() + el,
                     nh * hd + 7, nh, hd ** -0.5, _i32(lens).data_ptr(), None, 3, 1, 64, ws.data_ptr(), ws.numel())
        o = host(out.float())
        for s in range(3):
            want = U.attend(q[s, 1:1 + nh * hd].reshape(nh, hd), *stands[s], lens[s] - 1, hd ** -0.5,
                            g[s, 1:1 + nh * hd].reshape(nh, hd))
            assert rel_l2(o[s, 1:1 + nh * hd], want.ravel()) < TOL[t]
        assert (o[:, 0] == 0).all() and (o[:, 1 + nh * hd:] == 0).all()


def test_a_decode_step_replays_in_a_cuda_graph():
    """Append and attention captured once; lengths and inputs move on the device between replays, over a page's end."""
    import torch
    nh, kvh, hd, n0, steps = 14, 2, 64, 60, 8
    rng = np.random.default_rng(31)
    c, stands = _filled([n0, 10], 128, kvh, hd, seed=30)
    lens = torch.tensor([n0, 10], dtype=torch.int32, device="cuda:0")
    x = torch.zeros((2, (nh + 2 * kvh) * hd), device="cuda:0")
    qo, out = (torch.zeros((2, nh * hd), device="cuda:0") for _ in range(2))
    ws = torch.zeros(Q.kv8_attend_workspace(nh, kvh, hd, 2, 2, 1, 128), dtype=torch.uint8, device="cuda:0")

    def step():
        _append(c, "f32", x, nh, qo, lens, None, 1)
        Q.kv8_attend(c.view, Q.F32, qo.data_ptr(), nh * hd, None, 0, out.data_ptr(), nh * hd, nh, hd ** -0.5,
                     lens.data_ptr(), None, 2, 1, 128, ws.data_ptr(), ws.numel())
    try:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            Q.set_stream(s.cuda_stream)
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=s):
                step()
            k = [[a.transpose(1, 0, 2)[:0] for a in stands[i]] for i in range(2)]
            k = [[a.transpose(1, 0, 2) for a in stands[i]] for i in range(2)]
            raw = [[[], []] for _ in range(2)]
            for i in range(steps):
                new = rng.standard_normal((2, (nh + 2 * kvh) * hd)).astype(np.float32)
                x.copy_(torch.from_numpy(new))
                lens += 1
                g.replay()
                torch.cuda.synchronize()
                got = host(out)
                for q in range(2):
                    z = new[q].reshape(-1, hd)
                    for j in range(2):
                        k[q][j] = np.concatenate([k[q][j], z[nh + j * kvh:nh + (j + 1) * kvh][None].astype(np.float64)])
                        n = len(k[q][j])
                        if n % 32 == 0:  # the block closes: it stands quantised from now on
                            for h in range(kvh):
                                code, sc = U.quantize(k[q][j][n - 32:, h].astype(np.float32))
                                k[q][j][n - 32:, h] = (code - 128.0) * np.float64(np.float32(sc))
                    want = U.attend(z[:nh], *(a.transpose(1, 0, 2) for a in k[q]), len(k[q][0]) - 1, hd ** -0.5)
                    # (a byte at a tie may differ by one: 1 / 127 of a block's largest value, in one of its 2048 values)
                    assert rel_l2(got[q], want.ravel()) < 1e-4
        del g
    finally:
        Q.set_stream(torch.cuda.current_stream().cuda_stream)
    Q.check_device()


def test_what_lies_outside_the_cache_is_reported():
    """Page, slot, length and position out of range: nothing is accessed, ql_check_device says which."""
    import torch
    nh, kvh, hd = 2, 2, 64

    def run(change, expect):
        c, _ = _filled([40, 40], 64, kvh, hd, seed=33)
        kv, rope = _i32([41, 41]), dev(U.rope_table(64, hd))
        x = torch.randn((2, (nh + 2 * kvh) * hd), device="cuda:0")
        qo = torch.zeros((2, nh * hd), device="cuda:0")
        c, kv, rope = change(c, kv, rope)
        _append(c, "f32", x, nh, qo, kv, None, 1, rope=rope, rot=hd)
        _attend(c, "f32", qo, nh, kv, None, 1, 64)
        with pytest.raises(Q.QLError) as e:
            Q.check_device()
        assert e.value.status == Q.QL_EDEVICE and expect in str(e.value)

    def bad_page(c, kv, rope):
        c.td[1, 0] = c.pages
        return c, kv, rope

    def bad_slot(c, kv, rope):
        c.sd[0] = -1
        return c, kv, rope

    run(bad_page, "page")
    run(bad_slot, "slot")
    run(lambda c, kv, rope: (c, _i32([65, 41]), rope), "page")
    run(lambda c, kv, rope: (c, kv, rope[:40]), "position")
    for lens in ([41, 3], [1800, 200]):  # rows beyond max_q_len, in both forms of the kernel
        c, _ = _filled(lens, max(lens), kvh, hd, seed=36)
        q = torch.randn((sum(lens), nh * hd), device="cuda:0")
        _attend(c, "f32", q, nh, _i32(lens), _i32([0, lens[0], sum(lens)]), sum(lens) // 2, max(lens))
        with pytest.raises(Q.QLError, match="more rows"):
            Q.check_device()
    c, _ = _filled([10], 64, kvh, hd, seed=34)
    _append(c, "f32", torch.randn((20, 2 * kvh * hd), device="cuda:0"), 0, None, _i32([10]), _i32([0, 20]), 20)
    with pytest.raises(Q.QLError, match="more rows"):
        Q.check_device()


def test_refusals():
    import torch
    c, _ = _filled([40], 64, 2, 64, seed=35)
    x = torch.zeros((1, 4096), device="cuda:0")
    kv = _i32([41])
    p = x.data_ptr()
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda:0")

    def append(**k):
        a = dict(t=Q.F32, q=p, qs=256, k=p, ks=128, v=p, vs=128, o=p, os=256, nh=4, eps=1e-6, rope=None, rot=0, mp=0,
                 kv=kv.data_ptr(), st=None, rows=1, mq=1, cache=c.view)
        a.update(k)
        Q.kv8_append(a["cache"], a["t"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["o"], a["os"], a["nh"], None, None,
                     a["eps"], a["rope"], a["rot"], a["mp"], a["kv"], a["st"], a["rows"], a["mq"])

    def attend(**k):
        a = dict(t=Q.F32, q=p, qs=256, g=None, gs=0, o=p, os=256, nh=4, kv=kv.data_ptr(), st=None, rows=1, mq=1, mk=64,
                 ws=ws.data_ptr(), wb=ws.numel(), cache=c.view)
        a.update(k)
        Q.kv8_attend(a["cache"], a["t"], a["q"], a["qs"], a["g"], a["gs"], a["o"], a["os"], a["nh"], 0.125, a["kv"], a["st"],
                     a["rows"], a["mq"], a["mk"], a["ws"], a["wb"])

    import copy

    def view(**k):
        v = type(c.view)()
        for f, _ in c.view._fields_:
            setattr(v, f, k.get(f, getattr(c.view, f)))
        return v

    for call in (append, attend):
        for bad in (dict(t=1), dict(q=None), dict(qs=255), dict(o=None), dict(os=100), dict(kv=None), dict(rows=2),
                    dict(rows=-1), dict(mq=0), dict(q=p + 1), dict(cache=view(head_dim=80)), dict(cache=view(head_dim=288)),
                    dict(cache=view(kv_heads=0)), dict(cache=view(k_codes=None)), dict(cache=view(k_open=c.view.k_open + 4)),
                    dict(cache=view(max_pages=-1))):
            with pytest.raises(Q.QLError) as e:
                call(**bad)
            assert e.value.status == Q.QL_EINVAL, bad
    for bad in (dict(k=None), dict(vs=1), dict(rot=6), dict(rot=128), dict(rot=64), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(Q.QLError) as e:
            append(**bad)
        assert e.value.status == Q.QL_EINVAL, bad
    for bad in (dict(nh=3), dict(g=p, gs=1), dict(ws=None), dict(wb=16), dict(ws=ws.data_ptr() + 4), dict(mk=-1)):
        with pytest.raises(Q.QLError) as e:
            attend(**bad)
        assert e.value.status == Q.QL_EINVAL, bad
    with pytest.raises(Q.QLError):
        Q.kv8_gather(c.view, Q.F32, p + 4, None, None, 4, kv.data_ptr())
    with pytest.raises(Q.QLError):
        Q.kv8_gather(c.view, Q.F32, p, None, None, -1, kv.data_ptr())
    assert Q.kv8_attend_workspace(3, 2, 64, 1, 1, 1, 64) == 0
    # calls of no rows do nothing
    append(cache=view(n_seqs=0), rows=0)
    attend(cache=view(n_seqs=0), rows=0)
    Q.check_device()
