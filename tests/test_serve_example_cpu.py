"""examples/serve_kv8.py refuses, before any work on a device, what its buffers do not hold."""
import os
import sys
import types

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("lens,steps", [((5, 3), 1), ((5, 3), 0), ((5, 3), -4), ((5, 60), 6), ((65, 1), 2), ((5,), 8),
                                        ((5, 3, 2), 8), ((5, 0), 8), ((), 8)])
def test_requests_that_do_not_fit(lens, steps):
    import serve_kv8 as S
    model = types.SimpleNamespace(n=2, max_tokens=64, V=8192)
    with pytest.raises(ValueError):
        S.generate(model, [[1] * n for n in lens], steps)


def test_requests_that_fit():
    import serve_kv8 as S
    S.check_request([60, 1], 5, 2, 64)  # the last token's key is not needed any more
    S.check_request([1, 1], 2, 2, 64)
