"""Low-rank adapters of many sequences beside a shared projection, against the products in 64 bits."""
import numpy as np
import pytest

import blog_b200 as Q

pytestmark = pytest.mark.gpu

TYPES = [Q.F16, Q.BF16, Q.F32]
U = 2.0 ** -24


def _torch(type_):
    import torch
    return {Q.F16: torch.float16, Q.BF16: torch.bfloat16, Q.F32: torch.float32}[type_]


class Case:
    """lens: rows of each sequence (None: one each, q_start NULL).  gap: rows before the first and behind the last one."""

    def __init__(self, type_, n_in, outs, adapter, lens=None, max_rank=16, ranks=None, n_adapters=None, gap=0, base="other",
                 x_pad=0, y_pad=0, lead=0, seed=0, without=(), garbage=float("nan"), scaled=True):
        import torch
        g = torch.Generator(device="cuda:0").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda:0")  # noqa: E731
        m = (max([i for i in adapter] + [0]) + 1) if n_adapters is None else n_adapters
        self.type, self.n_in, self.outs, self.max_rank, self.m = type_, n_in, outs, max_rank, m
        self.adapter, n = adapter, len(adapter)
        lens_ = [1] * n if lens is None else lens
        rows = sum(lens_) + (2 * gap if lens is not None else 0)
        starts = np.concatenate([[0], np.cumsum(lens_)]) + (gap if lens is not None else 0)
        self.rows, self.starts, self.base_kind = rows, starts, base
        self.q_start = None if lens is None else torch.tensor(starts, dtype=torch.int32, device="cuda:0")
        self.ad = torch.tensor(adapter, dtype=torch.int32, device="cuda:0")
        self.ranks = [max_rank] * m if ranks is None else ranks
        self.rank = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda:0")
        self.scale = (0.5 + torch.rand(m, generator=g, device="cuda:0")) if scaled else None
        dt = _torch(type_)
        self.a, self.b = [], []
        for p, o in enumerate(outs):
            a, b = (rn(m, max_rank, n_in) * n_in ** -0.5).to(dt), (rn(m, o, max_rank) * max_rank ** -0.5).to(dt)
            for i, r in enumerate(self.ranks):  # what is not in use may be anything
                if 0 <= r < max_rank:
                    a[i, r:] = garbage
                    b[i, :, r:] = garbage
            self.a.append(None if p in without else a)
            self.b.append(None if p in without else b)
        w = sum(outs)
        self.xs, self.ys = n_in + x_pad, w + y_pad
        self.xbuf = torch.full((lead + rows * self.xs + 32,), float("nan"), device="cuda:0")
        self.x = torch.as_strided(self.xbuf, (rows, n_in), (self.xs, 1), lead)
        self.x.copy_(rn(rows, n_in))
        self.ybuf = torch.full((lead + rows * self.ys + 32,), 7.0, device="cuda:0")
        self.y = torch.as_strided(self.ybuf, (rows, w), (self.ys, 1), lead)
        self.bbuf = torch.full((lead + rows * self.ys + 32,), float("nan"), device="cuda:0")
        self.base = torch.as_strided(self.bbuf, (rows, w), (self.ys, 1), lead)
        self.base.copy_(rn(rows, w))
        if base == "same":
            self.y.copy_(self.base)
        self.pool = Q.lora_pool(type_, [None if t is None else t.data_ptr() for t in self.a],
                                [None if t is None else t.data_ptr() for t in self.b], outs, n_in, m, max_rank,
                                None if self.rank is None else self.rank.data_ptr(),
                                None if self.scale is None else self.scale.data_ptr())

    def call(self):
        base = {"other": self.base.data_ptr(), "same": self.y.data_ptr(), "none": None}[self.base_kind]
        Q.lora_add(self.pool, self.x.data_ptr(), self.xs, base, self.ys, self.y.data_ptr(), self.ys, self.ad.data_ptr(),
                   len(self.adapter), None if self.q_start is None else self.q_start.data_ptr(), self.rows)

    def check(self):
        """Every row against 64 bits, and what is not a sequence's left alone."""
        import torch
        y0 = self.ybuf.clone()
        first = self.y.double().clone()
        Q.set_stream(None)
        self.call()
        Q.check_device()
        ref = first.clone()
        tol = torch.zeros_like(ref)
        for s, i in enumerate(self.adapter):
            lo, hi = int(self.starts[s]), int(self.starts[s + 1])
            b0 = 0.0 if self.base_kind == "none" else self.base[lo:hi].double()
            ref[lo:hi] = b0
            r = self.ranks[i] if 0 <= i < self.m else 0
            tol[lo:hi] = 0
            if r <= 0 or r > self.max_rank:
                continue
            x = self.x[lo:hi].double()
            col = 0
            k = 1.0 if self.scale is None else float(self.scale[i].double())
            for a, b, o in zip(self.a, self.b, self.outs):
                if a is not None:
                    A, B = a[i, :r].double(), b[i, :, :r].double()
                    h = k * (x @ A.T)
                    ref[lo:hi, col:col + o] += h @ B.T
                    # each product of x and A within 2^-21 (limbs: 2^-22 of x, for f32 weights 2^-22 of A and of both
                    # second limbs 2^-22 more, at most 3 x 2^-22) and its sums: 32 truncated additions (2 units each),
                    # then settled sums in fp32, fewer than 40 (1 unit): 104 units of 2^-24 of the sum of sizes; then
                    # h once more through limbs, the scale (1), and the second sum of up to 96 truncated additions
                    size = (k * x.abs() @ A.abs().T) @ B.abs().T
                    tol[lo:hi, col:col + o] += size * (3 * 2.0 ** -22 + 104 * U + 3 * 2.0 ** -22 + 192 * U)
                col += o
            tol[lo:hi] += ref[lo:hi].abs() * U
        err = (self.y.double() - ref).abs()
        assert bool((err <= tol).all()), float((err - tol).max())
        inside = torch.zeros_like(self.ybuf, dtype=torch.bool)
        rows = torch.as_strided(inside, self.y.shape, self.y.stride(), self.y.storage_offset())
        for s in range(len(self.adapter)):
            rows[int(self.starts[s]):int(self.starts[s + 1])] = True
        assert torch.equal(self.ybuf[~inside], y0[~inside])
        d, size = (self.y.double() - ref), ref - (0 if self.base_kind == "none" else self.base.double())
        return float(d.norm() / max(float(size[torch.isfinite(size)].norm()), 1e-30))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_in,outs", [(32, (1,)), (96, (17,)), (896, (896, 128, 128)), (3584, (3584, 512, 512)), (2048, (2816, 2815))])
def test_one_token(type_, n_in, outs):
    """And a few, of few adapters."""
    Case(type_, n_in, outs, [1]).check()
    Case(type_, n_in, outs, [0, 2, 1, 0, 2], seed=1).check()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rank", [1, 2, 3, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 128, 129, 250, 256])
def test_ranks(type_, rank):
    top = (rank + 7) // 8 * 8
    Case(type_, 160, (50, 33), [0, 1, 0], max_rank=top, ranks=[rank, max(1, rank // 2)], seed=rank).check()


@pytest.mark.parametrize("type_", TYPES)
def test_unlike_ranks_in_a_pool(type_):
    r = np.random.default_rng(3)
    adapter = [int(v) for v in r.integers(-1, 9, 70)]
    Case(type_, 512, (300, 70), adapter, max_rank=72, ranks=[0, 1, 72, 8, 33, 16, 5, 64, 40], n_adapters=9, seed=4).check()


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 33, 64, 65, 300, 511, 512, 513, 1025])
@pytest.mark.parametrize("kinds", [1, 3, 40])
def test_batches_of_tokens(n, kinds):
    r = np.random.default_rng(n)
    Case(Q.BF16, 256, (130, 64), [int(v) for v in r.integers(-1, kinds, n)], n_adapters=kinds, max_rank=16, seed=n).check()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens", [[1], [3], [8], [9], [40], [127], [128], [129], [500], [513], [700, 0, 1, 255], [0, 0, 5, 0, 64, 0],
                                  [4] * 33, [16, 17, 33, 64, 65, 128]])
def test_prompts(type_, lens):
    adapter = [i % 3 - (1 if i % 5 == 4 else 0) for i in range(len(lens))]
    Case(type_, 320, (200, 40, 24), adapter, lens=lens, n_adapters=3, max_rank=32, ranks=[32, 8, 19], gap=3, seed=sum(lens)).check()


@pytest.mark.parametrize("base", ["other", "same", "none"])
@pytest.mark.parametrize("lens", [None, [40, 90, 3]])
def test_base(base, lens):
    Case(Q.F16, 256, (100, 28), [0, -1, 1], lens=lens, base=base, gap=2).check()


@pytest.mark.parametrize("x_pad,y_pad,lead", [(4, 4, 0), (1, 1, 0), (0, 0, 1), (3, 5, 2), (0, 0, 4)])
@pytest.mark.parametrize("lens", [None, [70, 300, 130]])
def test_strides_and_starts(x_pad, y_pad, lead, lens):
    Case(Q.BF16, 288, (65, 64), [0, 1, 0], lens=lens, x_pad=x_pad, y_pad=y_pad, lead=lead, max_rank=24).check()


def test_projections_without_adapters():
    for without in ((1,), (0,), (0, 1, 2)):
        for base in ("other", "same", "none"):
            Case(Q.F16, 128, (64, 32, 40), [0, 1], without=without, base=base).check()


def test_no_adapters_at_all():
    for base in ("other", "same", "none"):
        Case(Q.F16, 128, (64,), [-1, -7, -1], n_adapters=0, base=base).check()
        Case(Q.F16, 128, (64,), [-1, -1], n_adapters=2, lens=[100, 30], base=base).check()


def test_shared_by_all_against_large_sums():
    """The largest inner sizes: cut-off sums would show here."""
    for type_ in TYPES:
        far = Case(type_, 18944, (3584,), [0, 1, 1], max_rank=64, seed=8).check()
        assert far < 1e-6, far
        far = Case(type_, 8192, (1024,), [0], lens=[300], max_rank=128, seed=9).check()
        assert far < 1e-6, far


def test_outside_the_pool():
    import torch
    c = Case(Q.F16, 128, (64,), [0, 5, 1, 2], n_adapters=3, ranks=[8, 17, 16])
    c.ranks = [8, 0, 16]  # 17 is above the pool's 16, 5 is no slot: as none
    Q.set_stream(None)
    c.call()
    with pytest.raises(Q.QLError) as e:
        Q.check_device()
    assert e.value.status == Q.QL_EDEVICE and "adapter" in str(e.value)
    assert torch.equal(c.y[1:3], c.base[1:3])
    c.ad[1] = -1
    c.rank[1] = 0
    c.adapter = [0, -1, 1, 2]
    c.check()


def test_offsets_past_32_bits():
    """A pool of more than 2^31 weights, and rows far apart."""
    import torch
    m, r, n_in = 36, 256, 262144
    a = torch.zeros(m, r, n_in, dtype=torch.float16, device="cuda:0")
    a[35, 3, n_in - 32:] = 1.0
    a[0, 3] = 5.0
    b = torch.zeros(m, 64, r, dtype=torch.float16, device="cuda:0")
    b[35, :, 3] = 2.0
    st = (1 << 30) + 64
    y = torch.zeros(2 * st + 64, device="cuda:0")
    x = torch.ones(3, n_in, device="cuda:0")
    ad = torch.tensor([35, -1, 35], dtype=torch.int32, device="cuda:0")
    pool = Q.lora_pool(Q.F16, [a.data_ptr()], [b.data_ptr()], [64], n_in, m, r)
    Q.set_stream(None)
    Q.lora_add(pool, x.data_ptr(), n_in, None, 0, y.data_ptr(), st, ad.data_ptr(), 3, None, 3)
    Q.check_device()
    rows = torch.as_strided(y, (3, 64), (st, 1))
    assert bool((rows[0] == 64).all()) and bool((rows[2] == 64).all()) and bool((rows[1] == 0).all())
    assert float(y.sum()) == 2 * 64 * 64


def test_rows_of_nan_stay_in_their_rows():
    for lens in (None, [200, 200]):
        c = Case(Q.BF16, 128, (64,), [0, 0], lens=lens)
        c.x[0, 5] = float("nan")
        c.x[c.rows - 1, 7] = float("inf")
        Q.set_stream(None)
        c.call()
        Q.check_device()
        good = c.y.isfinite().all(1)
        assert not bool(good[0]) and not bool(good[c.rows - 1]) and bool(good[1:c.rows - 1].all())


@pytest.mark.parametrize("lens", [None, [150, 40, 3]])
def test_replay_follows_the_device(lens):
    """A captured call takes adapters, ranks and row starts as they stand at the replay; repeated, the same bits."""
    import torch
    c = Case(Q.F16, 512, (96, 32), [0, 1, 2], lens=lens, ranks=[16, 8, 3], max_rank=16, garbage=0.5)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        c.call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.call()
        st.synchronize()
        c.ad.copy_(torch.tensor([2, -1, 1], dtype=torch.int32))
        c.rank.copy_(torch.tensor([1, 16, 5], dtype=torch.int32))
        if lens is not None:
            c.q_start.copy_(torch.tensor([0, 2, 100, 190], dtype=torch.int32))
        c.y.zero_()
        g.replay()
        st.synchronize()
        once = c.y.clone()
        c.y.zero_()
        g.replay()
        st.synchronize()
        assert torch.equal(once, c.y)
    Q.set_stream(None)
    c.adapter, c.ranks = [2, -1, 1], [1, 16, 5]
    if lens is not None:
        c.starts = [0, 2, 100, 190]
    c.y.zero_()
    c.check()
    assert torch.equal(once, c.y) and Q.last_launch_count() == 1


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_in,outs,max_rank,lens", [
    (32, (64,), 16, [128]), (64, (4,), 8, [130]), (96, (64, 64, 64), 64, [200, 70]), (896, (896, 128, 128), 64, [1000, 333]),
    (3584, (512,), 128, [513]), (1024, (260, 68), 96, [600, 64]), (512, (260, 68), 104, [300]), (2048, (1024,), 192, [257]),
    (8192, (8192, 1024, 1024), 64, [128]), (640, (128, 100, 36), 40, [90, 0, 51, 700, 128, 1]), (128, (64,), 256, [300]),
    (4128, (192, 64), 16, [5000])])
def test_long_prompts(type_, n_in, outs, max_rank, lens):
    """Tiles of 128 rows, their clusters, ranks side by side, and those that go one projection at a time."""
    adapter = [i % 2 for i in range(len(lens))]
    far = Case(type_, n_in, outs, adapter, lens=lens, max_rank=max_rank, ranks=[max_rank, max(1, max_rank - 11)], n_adapters=2,
               gap=5, seed=n_in).check()
    assert far < 1e-6, far


def test_long_prompts_some_without():
    for base in ("other", "same", "none"):
        for without in ((), (0,), (1,), (0, 2), (0, 1, 2)):
            Case(Q.BF16, 256, (132, 64, 200), [0, -1, 1], lens=[200, 150, 90], base=base, without=without, ranks=[16, 0], gap=1).check()
