"""The kernel that a call of adapters takes (ql_lora_add_form), and the tiles of 128 rows over all that can differ between two of
their calls: CTAs per tile, rows that lie together or do not, bases, strides, row starts, threads, replays."""
import threading

import numpy as np
import pytest

import blog_b200 as Q
from test_gpu_layer import QKV, H, Layer
from test_gpu_lora import TYPES, Case
from test_gpu_lora_slots import FAR

pytestmark = pytest.mark.gpu

TILES, ROWS = Q.LORA_FORM_TILES, Q.LORA_FORM_ROWS
WIDE = (1024, (1024, 132, 68))  # inputs, outputs: of few rows and of thousands in tiles


def _runs(rows, n=37):
    """Sequences of n rows: with two adapters in turn no tile's rows lie together."""
    return [n] * (rows // n) + [rows % n]


def _checked(c, form=TILES):
    far = c.check()
    assert Q.lora_add_form()[0] == form
    assert far < FAR, far
    return Q.lora_add_form()[1]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("joint", [True, False])
@pytest.mark.parametrize("base", ["other", "same", "none"])
def test_ctas_per_tile(type_, joint, base):
    """Every number of CTAs that share x's columns and the outputs, uneven shares among them."""
    seen = set()
    for rows in (1301, 2300, 2999, 4000, 5003, 6500, 14001):
        lens = [rows - 100, 100] if joint else _runs(rows)
        c = Case(type_, WIDE[0] - 32, WIDE[1], [i % 2 for i in range(len(lens))], lens=lens, max_rank=32, ranks=[32, 19], gap=2,
                 base=base, seed=rows)
        seen.add(_checked(c))
    assert {1, 2, 8} <= seen and len(seen) >= 5, seen


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens", [[1200, 1100], _runs(2300)])
@pytest.mark.parametrize("outs,rank", [((64,), 96), ((96, 32), 32), ((4, 4, 4), 32)])
def test_ctas_without_outputs(type_, lens, outs, rank):
    c = Case(type_, 1024, outs, [i % 2 for i in range(len(lens))], lens=lens, max_rank=rank, gap=1)
    assert _checked(c) > sum((o + 63) // 64 for o in outs)


@pytest.mark.parametrize("base", ["other", "same", "none"])
@pytest.mark.parametrize("x_pad,y_pad,lead,outs,form", [
    (0, 0, 0, (1024, 132, 68), TILES), (4, 8, 4, (1024, 132, 68), TILES), (0, 4, 0, (1024, 132, 68), TILES),
    (1, 0, 0, (1024, 132, 68), ROWS), (0, 2, 0, (1024, 132, 68), ROWS), (0, 0, 1, (1024, 132, 68), ROWS), (0, 0, 0, (1024, 130, 68), ROWS)])
def test_bases_and_strides(base, x_pad, y_pad, lead, outs, form):
    c = Case(Q.BF16, 1024, outs, [1, -1, 0], lens=[1160, 300, 840], max_rank=32, ranks=[16, 32], n_adapters=2, gap=1, base=base,
             x_pad=x_pad, y_pad=y_pad, lead=lead)
    _checked(c, form)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("starts", [[0, 1900, 1200, 2400], [-7, 600, 2000, 90000], [2400, 1600, 900, 0], [3, 3, 3, 3], [2400, 0, 0, 2401]])
def test_starts_out_of_order_stay_in_bounds(type_, starts):
    """Row starts that fall or pass the rows: every row has the result of one of the adapters, or is left as it was."""
    import torch
    Q.set_stream(None)
    c = Case(type_, 1024, (1024, 132), [0, 1, -1], lens=[1000, 1000, 400], max_rank=32)
    c.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
    c.y.fill_(7.0)
    c.call()
    torch.cuda.synchronize()
    assert Q.lora_add_form()[0] == TILES
    Q.check_device()
    x, y, base = c.x.double(), c.y.double(), c.base.double()
    options = [torch.full_like(base, 7.0), base]
    for i in (0, 1):
        options.append(base + torch.cat([(x @ a[i].double().T) @ b[i].double().T * c.scale[i].double() for a, b in zip(c.a, c.b)], 1))
    off = torch.stack([(y - o).abs().amax(1) for o in options]).amin(0)
    assert (off <= 1e-4).all() and (c.ybuf[c.rows * c.ys:] == 7.0).all()


@pytest.mark.parametrize("type_", TYPES)
def test_outside_the_pool(type_):
    """Slots that the pool does not have and ranks above its own: reported, and as none."""
    import torch
    lens = [900, 500, 700, 300]
    c = Case(type_, *WIDE, [0, 5, 1, 2], lens=lens, n_adapters=3, max_rank=32, ranks=[8, 33, 32])
    c.ranks = [8, 0, 32]
    Q.set_stream(None)
    c.call()
    assert Q.lora_add_form()[0] == TILES
    with pytest.raises(Q.QLError) as e:
        Q.check_device()
    assert e.value.status == Q.QL_EDEVICE and "adapter" in str(e.value)
    assert torch.equal(c.y[900:2100], c.base[900:2100])
    c.ad[1] = -1
    c.rank[1] = 0
    c.adapter = [0, -1, 1, 2]
    _checked(c)


def test_calls_of_several_threads():
    """Pools of unlike types and ranks, which take unlike amounts of shared memory, in both kernels; every thread is told of its
    own calls."""
    import torch
    Q.set_stream(None)
    cases = [(TILES, Case(t, *WIDE, [0, 1], lens=[1500, 800], max_rank=m, seed=m)) for t, m in
             ((Q.BF16, 16), (Q.BF16, 64), (Q.F16, 48), (Q.F32, 32), (Q.F32, 64))]
    cases += [(ROWS, Case(Q.BF16, 1024, (64,), [0, 1, 2], max_rank=m, seed=m)) for m in (8, 256)]
    failed = []

    def many(form, c):
        try:
            for _ in range(100):
                c.call()
                assert Q.lora_add_form()[0] == form
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=many, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for form, c in cases:
        _checked(c, form)


@pytest.mark.parametrize("type_", TYPES)
def test_replay_follows_the_device(type_):
    """Captured as two long prompts, replayed with other adapters, ranks and starts, rows that do not lie together among them."""
    import torch
    lens = [1500, 700] + [2] * 60
    c = Case(type_, *WIDE, [i % 3 for i in range(62)], lens=lens, ranks=[16, 32, 3], max_rank=32, garbage=0.5)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        c.call()
        assert Q.lora_add_form()[0] == TILES
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.call()
        st.synchronize()
        c.adapter, c.ranks = [(i * 7 + 1) % 4 - 1 for i in range(62)], [1, 16, 32]
        c.starts = [min(2300, 13 + 37 * i) for i in range(63)]
        c.ad.copy_(torch.tensor(c.adapter, dtype=torch.int32))
        c.rank.copy_(torch.tensor(c.ranks, dtype=torch.int32))
        c.q_start.copy_(torch.tensor(c.starts, dtype=torch.int32))
        c.y.zero_()
        g.replay()
        st.synchronize()
        once = c.y.clone()
    Q.set_stream(None)
    c.y.zero_()
    _checked(c)
    assert torch.equal(once, c.y)


def test_a_layer():
    """The layer of the other test with prompts long enough for tiles, also captured and replayed on other rows and adapters."""
    import torch
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        s = Layer([2000, 1100, 1], [3, 0, 1])
        s.run()
        assert Q.lora_add_form()[0] == TILES
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run()
        other = Layer([900, 1300, 901], [1, -1, 3], seed=5)
        for k in ("x", "res", "adapter", "start"):
            getattr(s, k).copy_(getattr(other, k))
        g.replay()
        st.synchronize()
        want, at = s.proj.double(), 0
        for m, i in zip(other.lens, (1, -1, 3)):
            if i >= 0:
                r = int(s.rank[i])
                for a, b, lo, hi in ((s.a[0], s.b[0], 0, QKV[0]), (s.a[2], s.b[2], QKV[0] + QKV[1], sum(QKV))):
                    want[at:at + m, lo:hi] += (s.y1[at:at + m].double() @ a[i, :r].double().T) @ b[i, :, :r].double().T * s.scale[i].double()
            at += m
        assert float((s.qkv.double() - want).norm() / (want - s.proj.double()).norm()) < 1e-6
        got = {k: getattr(s, k).clone() for k in ("h1", "y1", "xq", "proj", "qkv", "h2", "y2", "logits", "ids", "weights", "act", "out")}
        s.run()
        st.synchronize()
        for k, v in got.items():
            assert torch.equal(v, getattr(s, k)), k
    Q.set_stream(None)
    Q.check_device()
    assert H == s.x.shape[1]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_in,outs,max_rank,lens,n_adapters", [
    # prompts of the tests of thousands of rows, of values that are not finite, of slots in turn
    (32, (64,), 16, [6500], 2), (64, (4,), 8, [6003, 63], 2), (96, (64, 64, 64), 64, [3300, 2070], 2), (512, (260, 68), 104, [4500], 2),
    (640, (100, 36), 96, [1, 3000, 1900], 2), (608, (36, 4, 132), 24, [4010, 1290], 2), (288, (132, 64), 40, [1] * 6100, 2),
    (256, (128, 36, 8), 64, [6100], 2), (256, (128, 36, 8), 8, [3000, 2500], 2), (256, (128, 36, 8), 16, [1] * 6000, 2),
    (256, (128, 64), 8, [6000], 1), (1024, (4096, 1000, 36), 32, [127] * 24, 24), (1024, (5020,), 64, [127] * 24, 24),
    (1024, (28,) * 3, 32, [127] * 24, 24), (1024, (4096, 1000, 36), 32, [1000, 90, 700, 1100, 1, 129], 6)])
def test_sizes_meant_for_tiles_take_them(type_, n_in, outs, max_rank, lens, n_adapters):
    c = Case(type_, n_in, outs, [i % n_adapters for i in range(len(lens))], lens=lens, max_rank=max_rank, n_adapters=n_adapters)
    Q.set_stream(None)
    c.call()
    Q.check_device()
    fits = type_ != Q.F32 or max_rank <= 96  # (two limbs of f32 weights take twice the place)
    assert Q.lora_add_form()[0] == (TILES if fits else ROWS)


@pytest.mark.parametrize("n,lens,form", [(256, [40] * 300, TILES), (64, [1] * 4096, ROWS), (4, [1000] * 4, TILES)])
def test_many_adapters(n, lens, form):
    """Which kernel, where many tiles of a launch have no rows.  (12000 rows of 256 adapters on 3584 -> 3584 + 512 + 512 at rank 16:
    tiles of 128 rows 518 us, of 32 rows 771; 4096 tokens of 64 on 18944 -> 3584 at rank 64: 2512 and 1089.)"""
    n_in, outs, rank = (3584, (3584, 512, 512), 16) if n in (4, 256) else (18944, (3584,), 64)
    r = np.random.default_rng(n)
    c = Case(Q.BF16, n_in, outs, [int(v) for v in r.integers(0, n, len(lens))], lens=lens, n_adapters=n, max_rank=rank)
    Q.set_stream(None)
    c.call()
    Q.check_device()
    assert Q.lora_add_form()[0] == form
    if len(lens) <= 300:
        _checked(c, form)


def test_calls_that_launch_nothing():
    c = Case(Q.BF16, 64, (32,), [0, 1])
    Q.set_stream(None)
    c.call()
    assert Q.lora_add_form()[0] == ROWS and Q.lora_add_form()[1] >= 1
    c.rows = 0
    c.adapter = []
    c.call()
    assert Q.lora_add_form() == (0, 0)
    with pytest.raises(Q.QLError):
        Q.lora_add(c.pool, None, 64, None, 32, c.y.data_ptr(), 32, c.ad.data_ptr(), 2, None, 2)
    assert Q.lora_add_form() == (0, 0)
    assert np.isfinite(c.y.cpu().numpy()).all()
