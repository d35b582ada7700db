"""Every byte of the packed 8-bit rows that the norm writes: groups of four blocks whole, zeros behind the row."""
import numpy as np
import pytest

import blog_b200 as Q

pytestmark = pytest.mark.gpu


def _packed(type_, x, raw, eps=1e-6):
    """The norm's y and its packed rows, and those of ql_quantize_q8_1_mmq for that y, over buffers full of 0xA5."""
    import torch
    n, h = x.shape
    dt = torch.float32 if type_ == Q.F32 else torch.bfloat16
    tx = torch.from_numpy(x).cuda().to(dt)
    y = torch.empty(n, h, dtype=dt, device="cuda:0")
    size = n * Q.q8_1_mmq_row_bytes(h)
    got = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda:0")
    want = got.clone()
    Q.set_stream(None)
    Q.add_rms_norm(type_, tx.data_ptr(), h, None, 0, None, 0, None, eps, y.data_ptr(), h, got.data_ptr(), Q.Q8_MMQ, raw, n, h)
    Q.quantize_q8_1_mmq(y.float().data_ptr(), want.data_ptr(), h, n, raw)
    Q.check_device()
    assert bool((got[size:] == 0xA5).all())
    return got[:size].cpu().numpy(), want[:size].cpu().numpy()


def _rows(n, h):
    r = np.random.default_rng(h)
    x = (r.standard_normal((n, h)) * np.exp(r.standard_normal((n, h)))).astype(np.float32)
    if n > 2:  # rows that are not finite: NaN in the row, not behind it
        x[0, h // 2] = np.nan
        x[1, 0] = np.inf
        x[2] = 0
    return x


# (of blocks of 32: one to four in the last group; one, two, four and eight groups of values per thread)
@pytest.mark.parametrize("h", [1, 33, 64, 96, 127, 128, 352, 777, 1000, 2100, 4100, 8200, 8250, 16400, 16416, 32700])
@pytest.mark.parametrize("n", [1, 5, 700])
@pytest.mark.parametrize("raw", [False, True])
def test_all_bytes(h, n, raw):
    if n > 5 and h > 8250:
        n = 310
    got, want = _packed(Q.F32, _rows(n, h), raw)
    assert np.array_equal(got, want), np.argwhere(got != want)[:4]


@pytest.mark.parametrize("h", [96, 352, 777, 4100, 16416])
def test_bf16_rows_end_in_zeros(h):
    """(the norm's y before it is rounded to bf16 is not there to compare with)"""
    got, _ = _packed(Q.BF16, _rows(5, h), True)
    nb = (h + 31) // 32
    last = got.reshape(-1, 5, 144)[-1]
    for b in range(nb % 4 or 4, 4):
        assert not last[:, 4 * b:4 * b + 4].any() and not last[:, 16 + 32 * b:48 + 32 * b].any()


def test_rows_of_zeros_without_eps():
    """0 / 0 in the row; zeros behind it all the same."""
    x = np.zeros((3, 96), np.float32)
    got, want = _packed(Q.F32, x, True, eps=0.0)
    assert np.array_equal(got, want)
