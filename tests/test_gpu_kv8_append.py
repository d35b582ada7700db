"""ql_kv8_append where its blocks, lengths or arguments are out of the ordinary."""
import numpy as np
import pytest

import blog_b200 as Q
from gpu_util import dev, host
from test_gpu_kv8 import Cache, _append, _check_cache, _i32

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
