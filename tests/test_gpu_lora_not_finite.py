"""Adapters over rows that are not finite: NaN in that row's outputs, whatever the type, the rank and the kernel."""
import numpy as np
import pytest

import blog_b200 as Q
from test_gpu_lora import TYPES, Case

pytestmark = pytest.mark.gpu

# (a NaN whose bits beyond those of a limb are all that tells it from an infinity, among them)
BAD = np.array([0x7F800000, 0xFF800000, 0x7FC00000, 0x7F800001, 0xFF800001, 0x7FFFFFFF], np.uint32).view(np.int32)


def _check_rows(c, with_adapters):
    """Bad values in some rows: NaN in every output of a projection with adapters there, every other row as without them."""
    import torch
    Q.set_stream(None)
    c.call()
    Q.check_device()
    want = c.y.clone()
    rows = np.linspace(0, c.rows - 1, len(BAD)).astype(int)
    xi = c.xbuf.view(torch.int32)
    for k, i in enumerate(rows):
        xi[c.x.storage_offset() + int(i) * c.xs + (k * 37) % c.n_in] = int(BAD[k])
    c.call()
    Q.check_device()
    good = np.setdiff1d(np.arange(c.rows), rows)
    assert torch.equal(c.y[good], want[good])
    at = 0
    for o, there in zip(c.outs, with_adapters):
        got = c.y[rows][:, at:at + o]
        assert bool(torch.isnan(got).all()) if there else torch.equal(got, want[rows][:, at:at + o])
        at += o


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rank", [1, 8, 17, 64])
@pytest.mark.parametrize("n", [7, 100])
def test_few_rows(type_, rank, n):
    slots = (rank + 7) // 8 * 8
    c = Case(type_, 128, (64, 36, 8), [0] * n, max_rank=slots, ranks=[rank], without=(1,), scaled=False)
    c.a[0].abs_(), c.b[0].abs_()  # (terms of one sign: no inf - inf)
    _check_rows(c, (True, False, True))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rows", [5])
def test_h_beyond_the_range(type_, rows):
    """A finite row whose h is not."""
    import torch
    c = Case(type_, 64, (40,), [0] * rows, max_rank=8, ranks=[1])
    c.a[0].fill_(10.0), c.b[0].fill_(1.0)
    c.x[2].fill_(3e38)
    Q.set_stream(None)
    c.call()
    Q.check_device()
    assert bool(torch.isnan(c.y[2]).all()) and bool(c.y[[0, 1, 3, 4]].isfinite().all())


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rank", [1, 16, 40, 64])
@pytest.mark.parametrize("lens", [[6100], [3000, 2500], [1] * 6000])
def test_thousands_of_rows(type_, rank, lens):
    """Tiles of 128 rows: of rows that lie together and of rows that do not."""
    slots = (rank + 7) // 8 * 8
    c = Case(type_, 256, (128, 36, 8), [i % 2 for i in range(len(lens))], lens=lens, max_rank=slots, ranks=[rank] * 2, n_adapters=2,
             without=(1,), scaled=False)
    for t in (c.a[0], c.b[0], c.a[2], c.b[2]):
        t.abs_()
    _check_rows(c, (True, False, True))


@pytest.mark.parametrize("type_", TYPES)
def test_h_beyond_the_range_in_tiles(type_):
    import torch
    c = Case(type_, 256, (128, 64), [0], lens=[6000], max_rank=8, ranks=[1])
    for a, b in zip(c.a, c.b):
        a.fill_(10.0), b.fill_(1.0)
    bad = [7, 130, 5999]
    c.x[bad] = 3e38
    Q.set_stream(None)
    c.call()
    Q.check_device()
    assert bool(torch.isnan(c.y[bad]).all()) and int((~c.y.isfinite()).sum()) == 3 * 192
