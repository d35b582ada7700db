"""The first call of a thread that has made no other use of the device: the same kernel and the same bits as on any other thread."""
import threading

import numpy as np
import pytest

import blog_b200 as Q
import oracle as O
from gpu_util import dev, make_weights
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


def _on_a_new_thread(call):
    import torch
    got = []

    def run():
        try:
            got.append(call())
        except BaseException as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    if isinstance(got[0], BaseException):
        raise got[0]
    return got[0]


def test_adapters_of_prompts():
    import torch
    Q.set_stream(None)
    c = Case(Q.BF16, 1024, (1024, 132, 68), [0, 1], lens=[1500, 800], max_rank=16)
    c.call()
    torch.cuda.synchronize()
    form, want = Q.lora_add_form(), c.y.clone()
    assert form[0] == Q.LORA_FORM_TILES
    c.y.zero_()
    torch.cuda.synchronize()

    def call():
        c.call()
        return Q.lora_add_form()

    assert _on_a_new_thread(call) == form
    assert torch.equal(c.y, want)


@pytest.mark.parametrize("t", [O.Q4_K, O.Q8_0, O.Q4_0])
@pytest.mark.parametrize("m", [1, 64])
def test_products(t, m):
    """Of weights that no call has seen before, and of such as one has."""
    import torch
    Q.set_stream(None)
    n, k = 512, 1024
    rb = O.row_bytes(t, k)
    w = make_weights(t, n, k, seed=t)
    x = dev(np.random.default_rng(t).standard_normal((m, k)).astype(np.float32))
    first, second = dev(w), dev(w)
    y = [torch.zeros(m, n, device="cuda:0") for _ in range(3)]
    Q.quant_matmul(t, first.data_ptr(), rb, x.data_ptr(), y[0].data_ptr(), n, k, m)
    torch.cuda.synchronize()
    launches = Q.last_launch_count()
    for wt, out in ((first, y[1]), (second, y[2])):
        def call():
            Q.quant_matmul(t, wt.data_ptr(), rb, x.data_ptr(), out.data_ptr(), n, k, m)
            return Q.last_launch_count()
        assert _on_a_new_thread(call) == launches
        assert torch.equal(out, y[0])
