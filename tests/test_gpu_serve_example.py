"""examples/serve_kv8.py: prompts and a replayed graph of single tokens over the 8-bit cache, tokens under rules."""
import os
import sys

import pytest

import blog_b200 as Q

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_tokens_follow_the_rules_and_prompts_agree_with_single_tokens():
    """The last step's logits, from single tokens over the cache, against one prompt of the same text in a second
    model: the same tokens' keys stand in both, but a token that came as part of a prompt saw its block already
    quantised where a single token saw the exact rows, an error of at most 1 / 254 of a block's largest value per
    key and value; over two layers the logits agree to a few per cent."""
    import torch

    import serve_kv8 as S
    torch.cuda.init()
    Q.init(0)
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    g = torch.Generator().manual_seed(3)
    model = S.Decoder(layers=2, seqs=3, max_tokens=256)
    prompts = [torch.randint(0, model.V, (k,), generator=g).tolist() for k in (70, 33, 5)]
    steps = 40
    out, raw, _ = S.generate(model, prompts, steps)
    assert all(len(t) == steps for t in out)
    assert max(out[0]) < model.V // 2          # the mask
    assert 7 not in out[2]                     # the bias
    again = S.Decoder(layers=2, seqs=3, max_tokens=256)
    text = [p + t[:-1] for p, t in zip(prompts, out)]  # the last token came from these
    lens = [len(t) for t in text]
    starts = [0, lens[0], lens[0] + lens[1], sum(lens)]
    again.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
    logits = again.forward(torch.tensor([i for t in text for i in t], dtype=torch.int32, device="cuda:0"),
                           torch.tensor(starts, dtype=torch.int32, device="cuda:0"), max(lens),
                           last=torch.tensor([s - 1 for s in starts[1:]], device="cuda:0"))
    torch.cuda.synchronize()
    for i in range(3):
        err = float((logits[i] - raw[i]).norm() / logits[i].norm())
        assert err < 0.05, (i, err)
    Q.check_device()
