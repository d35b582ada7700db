"""Refusals of the 8-bit cache's and the logits rules' entries that come before any work on a device."""
import pytest

import blog_b200 as Q

P = 1 << 40  # never dereferenced: validation fails first


def _cache(**k):
    a = dict(k_codes=P, v_codes=P, k_scale=P, v_scale=P, k_open=P, v_open=P, page_table=P, slots=None, n_pages=8, n_slots=2,
             n_seqs=2, max_pages=4, kv_heads=2, head_dim=64)
    a.update(k)
    return Q.kv8_cache(**a)


def _refused(call, *args):
    with pytest.raises(Q.QLError) as e:
        call(*args)
    assert e.value.status == Q.QL_EINVAL, e.value


APPEND = dict(cache=None, t=Q.F32, q=P, qs=256, k=P, ks=128, v=P, vs=128, o=P, os=256, nh=4, gq=P, gk=P, eps=1e-6, rope=P,
              rot=64, mp=8, kv=P, st=P, rows=2, mq=2)
ATTEND = dict(cache=None, t=Q.F32, q=P, qs=256, g=P, gs=256, o=P, os=256, nh=4, scale=0.125, kv=P, st=P, rows=2, mq=2, mk=64,
              ws=P, wb=1 << 40)
GATHER = dict(cache=None, t=Q.F32, k=P, v=P, st=P, n=4, kv=P)
LOGITS = dict(x=P, xs=100, o=P, os=100, n=2, v=100, r=None, tok=P, w=P, wb=64)


@pytest.mark.parametrize("call,base,names", [(Q.kv8_append, APPEND, ("kv", "st", "gq", "gk", "rope")),
                                             (Q.kv8_attend, ATTEND, ("kv", "st")), (Q.kv8_gather, GATHER, ("kv", "st")),
                                             (Q.logits_apply, LOGITS, ("tok",))])
def test_misaligned_device_arrays(call, base, names):
    """32-bit arrays that the kernels read word by word."""
    for name in names:
        for off in (1, 2, 3):
            a = dict(base)
            if "cache" in a:
                a["cache"] = _cache()
            else:
                a["r"] = Q.logits_rules()
            a[name] = P + off
            _refused(call, *a.values())


def test_misaligned_rules():
    need = dict(history=P, history_len=P, history_stride=8, prompt_len=P, repetition=P, frequency=P, presence=P, bias_ids=P,
                bias_values=P, bias_start=P, mask=P, mask_stride=4, mask_rows=2, mask_row=P)
    for name in need:
        if name.endswith(("stride", "rows")):
            continue
        a = dict(LOGITS, r=Q.logits_rules(**dict(need, **{name: P + 2})))
        _refused(Q.logits_apply, *a.values())


def test_the_largest_numbers_of_rows():
    for rows in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30):
        _refused(Q.kv8_append, *dict(APPEND, cache=_cache(), rows=rows).values())
        _refused(Q.kv8_attend, *dict(ATTEND, cache=_cache(), rows=rows).values())


def test_workspace_of_bad_sizes():
    for a in ((3, 2, 64, 1, 1, 1, 64), (0, 1, 64, 1, 1, 1, 64), (4, 2, 80, 1, 1, 1, 64), (4, 2, 64, -1, 1, 1, 64)):
        assert Q.kv8_attend_workspace(*a) == 0
