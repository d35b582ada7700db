"""Low-rank adapters of long prompts (tiles of 128 rows of one adapter where these are the faster: always for the thousands of
rows of the later tests), against the products in 64 bits, and calls beside one another."""
import threading

import pytest

import blog_b200 as Q
from test_gpu_lora import TYPES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_in,outs,max_rank,lens", [
    (32, (64,), 16, [400]), (64, (4,), 8, [420, 63]), (96, (64, 64, 64), 64, [330, 70]), (512, (260, 68), 104, [500]),
    (2048, (1024,), 192, [457]), (128, (64,), 256, [600]), (8192, (8192, 1024, 1024), 64, [420]), (608, (36, 4, 132), 24, [401, 129])])
def test_sizes(type_, n_in, outs, max_rank, lens):
    adapter = [i % 2 for i in range(len(lens))]
    far = Case(type_, n_in, outs, adapter, lens=lens, max_rank=max_rank, ranks=[max_rank, max(1, max_rank - 5)], n_adapters=2,
               gap=3, seed=n_in + 1).check()
    assert far < 1e-6, far


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens", [[1] * 600, [100, 1, 0, 127, 3, 129, 40, 90, 2, 30], [512, 512, 1, 511], None])
def test_rows_that_do_not_lie_together(type_, lens):
    """An adapter's rows come from several sequences, or one of them is not among those beside it."""
    n = 610 if lens is None else len(lens)
    far = Case(type_, 288, (132, 64), [i % 2 - (i % 7 == 3) for i in range(n)], lens=lens, max_rank=40, ranks=[40, 17],
               n_adapters=2, gap=2).check()
    assert far < 1e-6, far


@pytest.mark.parametrize("base", ["other", "same", "none"])
@pytest.mark.parametrize("x_pad,y_pad,lead", [(0, 0, 0), (4, 8, 4), (1, 0, 0), (0, 2, 0), (0, 0, 1)])
def test_bases_and_strides(base, x_pad, y_pad, lead):
    Case(Q.BF16, 160, (96, 40, 4), [1, -1, 0], lens=[260, 100, 140], max_rank=16, ranks=[16, 9], n_adapters=2, gap=1, base=base,
         x_pad=x_pad, y_pad=y_pad, lead=lead).check()


@pytest.mark.parametrize("type_", TYPES)
def test_rows_of_nan_stay_in_their_rows(type_):
    import torch
    c = Case(type_, 256, (128, 64), [0, 1], lens=[300, 200], max_rank=32)
    Q.set_stream(None)
    c.call()
    torch.cuda.synchronize()
    want = c.y.clone()
    bad = [5, 130, 299, 300, 460]
    c.x[bad[0], 7], c.x[bad[1]], c.x[bad[2], 255], c.x[bad[3], 0], c.x[bad[4], 128] = (float("inf"), float("nan"), float("-inf"),
                                                                                    float("nan"), float("inf"))
    c.y.zero_()
    c.call()
    torch.cuda.synchronize()
    good = [i for i in range(c.rows) if i not in bad]
    assert torch.equal(c.y[good], want[good]) and not torch.isfinite(c.y[bad]).any()


def test_replay_follows_the_device():
    """Captured as two prompts, replayed as others: rows that lay together do not, adapters, ranks and starts are others."""
    import torch
    c = Case(Q.BF16, 512, (96, 32), [0, 1, 2, 0], lens=[300, 200, 10, 40], ranks=[16, 8, 3], max_rank=16, garbage=0.5)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        c.call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.call()
        st.synchronize()
        c.ad.copy_(torch.tensor([2, -1, 1, 2], dtype=torch.int32))
        c.rank.copy_(torch.tensor([1, 16, 5], dtype=torch.int32))
        c.q_start.copy_(torch.tensor([0, 2, 100, 290, 550], dtype=torch.int32))
        c.y.zero_()
        g.replay()
        st.synchronize()
        once = c.y.clone()
    Q.set_stream(None)
    c.adapter, c.ranks, c.starts = [2, -1, 1, 2], [1, 16, 5], [0, 2, 100, 290, 550]
    c.check()
    c.y.zero_()
    c.call()
    torch.cuda.synchronize()
    assert torch.equal(once, c.y)


def test_two_graphs_at_once():
    """Replayed on two streams beside each other, again and again: nothing is shared but what is read."""
    import torch
    cases = [Case(Q.BF16, 1024, (512, 128), [0, 1], lens=[700, 500], max_rank=32, seed=1),
             Case(Q.F16, 1024, (512, 128), [i % 3 for i in range(40)], max_rank=32, seed=2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in cases]
    for c, st in zip(cases, streams):
        with torch.cuda.stream(st):
            Q.set_stream(st.cuda_stream)
            c.call()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                c.call()
            graphs.append(g)
    torch.cuda.synchronize()
    Q.set_stream(None)
    want = [c.y.clone() for c in cases]
    for c in cases:
        c.y.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.y, w)
        c.check()


def test_calls_of_several_threads():
    """Pools of unlike ranks, which take unlike amounts of shared memory of one kernel."""
    import torch
    Q.set_stream(None)
    cases = [Case(Q.BF16, 256, (64,), [0, 1, 2], max_rank=m, seed=m) for m in (8, 256, 64)]
    cases += [Case(Q.BF16, 256, (64,), [0], lens=[400], max_rank=m, seed=m) for m in (16, 128)]
    failed = []

    def many(c):
        try:
            for _ in range(300):
                c.call()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=many, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for c in cases:
        c.check()


@pytest.mark.parametrize("starts", [[0, 300, 200, 420], [-7, 100, 400, 9000], [500, 400, 300, 0], [3, 3, 3, 3]])
def test_starts_out_of_order_stay_in_bounds(starts):
    """Row starts that fall or pass the rows: every row has the result of one of the adapters, or is left as it was."""
    import torch
    Q.set_stream(None)
    c = Case(Q.BF16, 128, (64,), [0, 1, -1], lens=[200, 200, 20], max_rank=16)
    c.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
    c.y.fill_(7.0)
    c.call()
    torch.cuda.synchronize()
    Q.check_device()
    x, y, base = c.x.double(), c.y.double(), c.base.double()
    options = [torch.full_like(base, 7.0), base]
    for i in (0, 1):
        options.append(base + (x @ c.a[0][i].double().T) @ c.b[0][i].double().T * c.scale[i].double())
    off = torch.stack([(y - o).abs().amax(1) for o in options]).amin(0)
    assert (off <= 1e-4).all() and (c.ybuf[c.rows * c.ys:] == 7.0).all()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_in,outs,max_rank,lens", [
    (32, (64,), 16, [6500]), (64, (4,), 8, [6003, 63]), (96, (64, 64, 64), 64, [3300, 2070]), (512, (260, 68), 104, [4500]),
    (640, (100, 36), 96, [1, 3000, 1900]), (608, (36, 4, 132), 24, [4010, 1290]), (1024, (1024,), 1, [5001]),
    (288, (132, 64), 40, [1] * 6100), (160, (68, 64), 192, [100, 1, 0, 127, 3, 129, 40, 90, 2, 3000, 2777])])
def test_thousands_of_rows(type_, n_in, outs, max_rank, lens):
    slots = (max_rank + 7) // 8 * 8
    adapter = [i % 2 - (i % 7 == 6) for i in range(len(lens))]
    far = Case(type_, n_in, outs, adapter, lens=lens, max_rank=slots, ranks=[max_rank, max(1, max_rank - 5)], n_adapters=2, gap=3,
               seed=n_in + 2).check()
    assert far < 1e-6, far


@pytest.mark.parametrize("base", ["other", "same", "none"])
@pytest.mark.parametrize("x_pad,y_pad,lead,without", [(0, 0, 0, (1,)), (4, 8, 4, ()), (1, 0, 0, ()), (0, 0, 1, (0,))])
def test_thousands_of_rows_bases_and_strides(base, x_pad, y_pad, lead, without):
    Case(Q.BF16, 160, (96, 40, 4), [1, -1, 0], lens=[2600, 1000, 2400], max_rank=16, ranks=[16, 9], n_adapters=2, gap=1, base=base,
         x_pad=x_pad, y_pad=y_pad, lead=lead, without=without).check()


@pytest.mark.parametrize("type_", TYPES)
def test_thousands_of_rows_some_of_nan(type_):
    import torch
    c = Case(type_, 256, (128, 64), [0, 1], lens=[3000, 2500], max_rank=64)
    Q.set_stream(None)
    c.call()
    torch.cuda.synchronize()
    want = c.y.clone()
    bad = [5, 130, 2999, 3000, 5460]
    for k, i in enumerate(bad):
        c.x[i, (k * 61) % 256] = (float("inf"), float("nan"), float("-inf"))[k % 3]
    c.y.zero_()
    c.call()
    torch.cuda.synchronize()
    good = [i for i in range(c.rows) if i not in bad]
    assert torch.equal(c.y[good], want[good]) and not torch.isfinite(c.y[bad]).any()


def test_thousands_of_rows_replayed():
    """Captured as two long prompts, replayed with other adapters, ranks and starts, scattered rows among them."""
    import torch
    lens = [2700, 2300] + [10] * 60
    c = Case(Q.BF16, 512, (96, 32), [i % 3 for i in range(62)], lens=lens, ranks=[16, 8, 3], max_rank=16, garbage=0.5)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        c.call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.call()
        st.synchronize()
        c.adapter, c.ranks = [(i * 7 + 1) % 4 - 1 for i in range(62)], [1, 16, 5]
        c.starts = [min(5600, 13 + 90 * i) for i in range(63)]
        c.ad.copy_(torch.tensor(c.adapter, dtype=torch.int32))
        c.rank.copy_(torch.tensor(c.ranks, dtype=torch.int32))
        c.q_start.copy_(torch.tensor(c.starts, dtype=torch.int32))
        c.y.zero_()
        g.replay()
        st.synchronize()
        once = c.y.clone()
    Q.set_stream(None)
    c.y.zero_()
    c.check()
    assert torch.equal(once, c.y)
