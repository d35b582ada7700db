"""The choice of experts where sums of two scores of a group pass fp32's range: biases of the type's lowest value, which close
experts to all but the last choice, and large ones."""
import numpy as np
import pytest

import blog_b200 as Q
from test_gpu_route import _check, _logits

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups", [2, 4, 8, 32])
@pytest.mark.parametrize("renorm", [False, True])
def test_biases_of_the_lowest_value(sigmoid, groups, renorm):
    """Groups of none but such experts are the last choice, not closed ones."""
    e = 64
    per = e // groups
    for open_groups in range(0, groups, max(1, groups // 4)):
        b = np.full(e, LOWEST, np.float32)
        for g in range(open_groups):  # (the open ones in the middle: those of the lowest value on both sides)
            at = (g + groups // 3) % groups
            b[at * per:(at + 1) * per] = 0.1 * g
        for best in (1, 2):
            for top in sorted({1, open_groups + 1, groups}):
                if 0 < top <= groups:
                    _check(_logits(33, e, groups + top), min(e, 12), sigmoid, bias=b, groups=groups, top=top, best=best, renorm=renorm)


def test_half_of_a_group_at_the_lowest_value():
    b = np.zeros(64, np.float32)
    b[::2] = LOWEST
    b[8:16] = LOWEST
    b[17:24] = LOWEST
    for top in (1, 4, 7, 8):
        _check(_logits(40, 64, 5), 8, True, bias=b, groups=8, top=top, best=2, renorm=True)


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_sums_of_two_beyond_the_range(sign, sigmoid):
    """Groups whose sums differ, but not in fp32."""
    level = np.float32([2.5e38, 3.1e38, 1.9e38, 3.3e38, 2.2e38, 1.8e38, 3.0e38, 2.0e38]) * sign
    b = np.repeat(level, 8)
    b[::8] *= np.float32(0.99)
    for top in (1, 3, 8):
        _check(_logits(40, 64, 6), 11, sigmoid, bias=b, groups=8, top=top, best=2)


def test_closed_groups_beside_them():
    b = np.full(48, LOWEST, np.float32)
    b[8:16] = -np.inf
    b[16:24] = 0.25
    b[24:31] = -np.inf
    b[40:48] = np.nan
    only = np.full(48, LOWEST, np.float32)  # the first group closed, no other bias than the lowest
    only[:8] = -np.inf
    for bias in (b, only):
        for top in (1, 2, 3, 5, 6):
            for best in (1, 2):
                for renorm in (False, True):
                    _check(_logits(40, 48, 7), 20, True, bias=bias, groups=6, top=top, best=best, renorm=renorm)
