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
