"""Refusals of the norm's, the router's and the adapters' entries, before any work on a device."""
import pytest

import blog_b200 as Q

P = 1 << 40  # never dereferenced: validation fails first


def _refused(call, *args):
    with pytest.raises(Q.QLError) as e:
        call(*args)
    assert e.value.status == Q.QL_EINVAL, e.value


NORM = dict(t=Q.F32, x=P, xs=64, r=P + 4096, rs=64, s=P + 8192, ss=64, g=P, eps=1e-6, y=P + 16384, ys=64, q=P + 32768,
            layout=Q.Q8_ROWS, raw=0, rows=2, h=64)


@pytest.mark.parametrize("change", [dict(t=Q.F16), dict(t=Q.Q4_K), dict(rows=-1), dict(h=0), dict(h=-4), dict(h=32769), dict(eps=-1e-6),
                                    dict(eps=float("nan")), dict(layout=3), dict(layout=-1), dict(x=None), dict(xs=63),
                                    dict(rs=63), dict(ss=63), dict(ys=63), dict(x=P + 2), dict(r=P + 1), dict(s=P + 3),
                                    dict(y=P + 2), dict(g=P + 2), dict(q=P + 2), dict(q=None), dict(layout=Q.Q8_NONE),
                                    dict(s=P, ss=65), dict(y=P + 4096, ys=65), dict(y=P + 8192), dict(t=Q.BF16, x=P + 1)])
def test_norm(change):
    _refused(Q.add_rms_norm, *dict(NORM, **change).values())


def test_norm_of_no_rows():
    Q.add_rms_norm(*dict(NORM, rows=0, x=None, y=None).values())


ROUTE = dict(x=P, xs=64, i=P, w=P, n=2, e=64, k=4)
RULE = dict(score=Q.ROUTE_SOFTMAX, bias=P, n_groups=8, top_groups=2, group_best=2)


@pytest.mark.parametrize("change", [dict(x=None), dict(i=None), dict(w=None), dict(xs=63), dict(n=-1), dict(e=0), dict(e=1025, xs=1025),
                                    dict(k=0), dict(k=33), dict(k=65), dict(x=P + 2), dict(i=P + 1), dict(w=P + 3)])
def test_route(change):
    _refused(Q.moe_route, *dict(ROUTE, **change).values(), Q.moe_route_rule(**RULE))


@pytest.mark.parametrize("change", [dict(score=2), dict(score=-1), dict(bias=P + 2), dict(n_groups=0), dict(n_groups=7), dict(n_groups=64),
                                    dict(top_groups=0), dict(top_groups=9), dict(group_best=0), dict(group_best=3),
                                    dict(scale=float("inf")), dict(scale=float("nan"))])
def test_route_rule(change):
    _refused(Q.moe_route, *ROUTE.values(), Q.moe_route_rule(**dict(RULE, **change)))


def test_route_of_no_tokens():
    Q.moe_route(None, 64, None, None, 0, 64, 4, Q.moe_route_rule(**RULE))


LORA = dict(x=P, xs=64, base=P + 8192, bs=96, y=P + 65536, ys=96, ad=P, n=2, st=P, rows=5)
POOL = dict(t=Q.F16, a=[P, None], b=[P, None], out_dims=[64, 32], in_dim=64, n_adapters=4, max_rank=16, rank=P, scale=P)


@pytest.mark.parametrize("change", [dict(x=None), dict(y=None), dict(ad=None), dict(xs=63), dict(bs=95), dict(ys=95), dict(n=-1),
                                    dict(rows=-1), dict(st=None), dict(x=P + 2), dict(y=P + 65537), dict(base=P + 2), dict(ad=P + 1),
                                    dict(st=P + 2), dict(base=P + 65536, bs=97), dict(y=P)])
def test_lora(change):
    a = dict(LORA, **change)
    _refused(Q.lora_add, Q.lora_pool(**POOL), *a.values())


@pytest.mark.parametrize("change", [dict(t=Q.Q8_0), dict(t=5), dict(a=[], b=[], out_dims=[]), dict(a=[P, P]), dict(b=[P, P]),
                                    dict(a=[P + 8, None]), dict(b=[P + 4, None]), dict(out_dims=[64, 0]), dict(out_dims=[-1, 97]),
                                    dict(out_dims=[2 ** 31 - 1, 2 ** 31 - 1]), dict(in_dim=0), dict(in_dim=48), dict(in_dim=-32),
                                    dict(n_adapters=-1), dict(max_rank=0), dict(max_rank=12), dict(max_rank=264), dict(rank=P + 2),
                                    dict(scale=P + 1)])
def test_lora_pool(change):
    _refused(Q.lora_add, Q.lora_pool(**dict(POOL, **change)), *LORA.values())
    with pytest.raises(ValueError):
        Q.lora_pool(**dict(POOL, a=[P] * 4, b=[P] * 4, out_dims=[1] * 4))


def test_lora_of_no_rows():
    Q.lora_add(Q.lora_pool(**POOL), None, 64, None, 96, None, 96, None, 3, P, 0)
    Q.lora_add(Q.lora_pool(**POOL), None, 64, None, 96, None, 96, None, 0, P, 7)
    Q.lora_add(Q.lora_pool(**POOL), None, 64, None, 96, None, 96, None, 0, None, 0)
