"""Adapters of prompts whose tiles are not full and whose projections end inside 64 columns: results and copies take turns in
the same shared memory, many times per CTA.  Against the products in 64 bits, and the same bits again and again."""
import pytest

import blog_b200 as Q
from test_gpu_lora import TYPES, Case

pytestmark = pytest.mark.gpu

# Of h and of y: limbs, 3 x 2^-22 of a product (of unlike signs: of the sum's size), and at most 32 additions that are cut off
# (f16 weights: 4 blocks of 4 products with 2 limbs), each by 2 units in the last place of a sum so far, which is no larger than
# the result on average.  (f32 weights at rank 64: 24 and 24 of them, 1.07e-6 measured.)
FAR = 2 * (3 * 2.0 ** -22 + 32 * 2.0 ** -23)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("base", ["other", "same", "none"])
@pytest.mark.parametrize("outs", [(4096, 1000, 36), (5020,), (28,) * 3])
@pytest.mark.parametrize("lens", [[127] * 24, [1000, 90, 700, 1100, 1, 129]])
def test_slots_in_turn(type_, base, outs, lens):
    import torch
    c = Case(type_, 1024, outs, list(range(len(lens))), lens=lens, max_rank=64 if len(outs) == 1 else 32, gap=1, base=base,
             seed=len(lens))
    y0 = c.ybuf.clone()
    assert c.check() < FAR and Q.lora_add_form()[0] == Q.LORA_FORM_TILES
    want = c.ybuf.clone()
    for _ in range(5):
        c.ybuf.copy_(y0)
        c.call()
        torch.cuda.synchronize()
        assert torch.equal(c.ybuf, want)
