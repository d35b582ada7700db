"""A layer of many requests as a server runs it: residual and norm with 8-bit rows, the quantised projection on them, the
requests' adapters beside it, the next norm, the router's choice, the grouped experts.  Every stage against the definition on
what the stages before it left on the device, and the whole captured and replayed on other inputs and adapters."""
import numpy as np
import pytest

import blog_b200 as Q
import oracle as O
from gpu_util import dev, make_weights, rel_l2
from test_gpu_moe_grouped import oracle_down, oracle_swiglu
from test_gpu_norm import Y_TOL
from test_gpu_route import TOL as ROUTE_TOL, _reference as route_reference

pytestmark = pytest.mark.gpu

H, QKV, E, F, K = 1024, (1024, 256, 256), 32, 512, 4
N = sum(QKV)


class Layer:
    def __init__(self, lens, adapters, seed=0):
        import torch
        g = torch.Generator(device="cuda:0").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda:0")  # noqa: E731
        self.lens, self.rows, self.n = lens, sum(lens), len(lens)
        T = self.rows
        self.x, self.res = rn(T, H), rn(T, H) * 2
        self.h1, self.y1, self.h2, self.y2 = (torch.empty(T, H, device="cuda:0") for _ in range(4))
        self.xq = torch.zeros(T * Q.q8_1_row_bytes(H), dtype=torch.uint8, device="cuda:0")
        self.qkv, self.proj = torch.empty(T, N, device="cuda:0"), torch.empty(T, N, device="cuda:0")
        self.g1, self.g2 = 1 + 0.1 * rn(H), 1 + 0.1 * rn(H)
        self.w_qkv = make_weights(O.Q4_K, N, H, seed=11)
        self.wq = dev(self.w_qkv)
        # adapters on q and v, none on k
        self.rank = torch.tensor([16, 3, 0, 11], dtype=torch.int32, device="cuda:0")
        self.scale = 0.5 + torch.rand(4, generator=g, device="cuda:0")
        self.a = [(rn(4, 16, H) * H ** -0.5).half(), None, (rn(4, 16, H) * H ** -0.5).half()]
        self.b = [(rn(4, QKV[0], 16) * 0.25).half(), None, (rn(4, QKV[2], 16) * 0.25).half()]
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.pool = Q.lora_pool(Q.F16, [p(t) for t in self.a], [p(t) for t in self.b], QKV, H, 4, 16, p(self.rank), p(self.scale))
        self.adapter = torch.tensor(adapters, dtype=torch.int32, device="cuda:0")
        self.start = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda:0")
        self.w_r = make_weights(O.Q8_0, E, H, seed=12, std=0.05)
        self.wr = dev(self.w_r)
        self.logits, self.bias = torch.empty(T, E, device="cuda:0"), 0.05 * rn(E)
        self.ids, self.weights = torch.empty(T, K, dtype=torch.int32, device="cuda:0"), torch.empty(T, K, device="cuda:0")
        self.rule = Q.moe_route_rule(Q.ROUTE_SIGMOID, p(self.bias), n_groups=4, top_groups=2, group_best=2, renormalise=True, scale=2.5)
        self.w_g, self.w_u, self.w_d = (make_weights(t, E * r, k, seed=s) for t, r, k, s in
                                        ((O.Q4_K, F, H, 13), (O.Q4_K, F, H, 14), (O.Q8_0, H, F, 15)))
        self.wg, self.wu, self.wd = dev(self.w_g), dev(self.w_u), dev(self.w_d)
        self.act, self.out = torch.empty(T * K, F, device="cuda:0"), torch.empty(T, H, device="cuda:0")

    def run(self):
        p, T = lambda t: t.data_ptr(), self.rows  # noqa: E731
        Q.add_rms_norm(Q.F32, p(self.x), H, p(self.res), H, p(self.h1), H, p(self.g1), 1e-6, p(self.y1), H, p(self.xq), Q.Q8_ROWS,
                       False, T, H)
        Q.quant_matmul_q8_1(O.Q4_K, p(self.wq), O.row_bytes(O.Q4_K, H), p(self.xq), p(self.proj), N, H, T)
        Q.lora_add(self.pool, p(self.y1), H, p(self.proj), N, p(self.qkv), N, p(self.adapter), self.n, p(self.start), T)
        Q.add_rms_norm(Q.F32, p(self.qkv), N, p(self.h1), H, p(self.h2), H, p(self.g2), 1e-6, p(self.y2), H, None, Q.Q8_NONE, False,
                       T, H)
        Q.quant_matmul_ex(O.Q8_0, p(self.wr), O.row_bytes(O.Q8_0, H), p(self.y2), H, p(self.logits), E, E, H, T, path=Q.PATH_GEMV)
        Q.moe_route(p(self.logits), E, p(self.ids), p(self.weights), T, E, K, self.rule)
        rg, rd = O.row_bytes(O.Q4_K, H), O.row_bytes(O.Q8_0, F)
        Q.moe_swiglu_grouped(O.Q4_K, p(self.wg), p(self.wu), F * rg, F * rg, rg, rg, p(self.y2), H, p(self.ids), 0, E, p(self.act), T,
                             K, F, H)
        self.out.copy_(self.h2)
        Q.moe_down_grouped_accum_ordered(O.Q8_0, p(self.wd), H * rd, rd, p(self.act), p(self.ids), 0, E, p(self.weights), p(self.out),
                                         H, T, K, H, F)


def _norm(v, g):
    v = v.astype(np.float64)
    return v / np.sqrt((v ** 2).mean(1, keepdims=True) + 1e-6) * g.astype(np.float64)


@pytest.mark.parametrize("lens,adapters", [([1], [0]), ([1, 1, 1, 1, 1], [3, -1, 0, 1, 0]), ([5, 1, 30], [1, 0, 2]),
                                           ([300, 200], [0, 3])])
def test_a_layer(lens, adapters):
    import torch
    Q.set_stream(torch.cuda.current_stream().cuda_stream)
    s = Layer(lens, adapters)
    s.run()
    Q.check_device()
    n = {k: v.cpu().numpy() for k, v in vars(s).items() if isinstance(v, torch.Tensor)}
    T = s.rows
    assert np.array_equal(n["h1"], n["x"] + n["res"])
    ref = _norm(n["h1"], n["g1"])
    assert np.all(np.abs(n["y1"] - ref) <= Y_TOL * np.abs(ref))
    rows = n["xq"].reshape(T, -1)
    assert np.array_equal(rows, O.quantize_q8_1(n["y1"], False))
    some = range(0, T, max(1, T // 12))
    rb = O.row_bytes(O.Q4_K, H)
    assert rel_l2(n["proj"][list(some)], np.stack([O.gemv_q8_1(O.Q4_K, s.w_qkv, rb, rows[i], N, H) for i in some])) < 1e-5
    want, at = n["proj"].astype(np.float64), 0
    for m, i in zip(lens, adapters):
        if i >= 0:
            r = int(n["rank"][i])
            for a, b, lo, hi in ((s.a[0], s.b[0], 0, QKV[0]), (s.a[2], s.b[2], QKV[0] + QKV[1], N)):
                h = n["y1"][at:at + m].astype(np.float64) @ a[i, :r].double().cpu().numpy().T * float(n["scale"][i])
                want[at:at + m, lo:hi] += h @ b[i, :, :r].double().cpu().numpy().T
        at += m
    assert rel_l2(n["qkv"], want) < 1e-6
    assert np.array_equal(n["qkv"][:, QKV[0]:QKV[0] + QKV[1]], n["proj"][:, QKV[0]:QKV[0] + QKV[1]])  # no adapter there
    assert np.array_equal(n["h2"], n["qkv"][:, :H] + n["h1"])
    ref = _norm(n["h2"], n["g2"])
    assert np.all(np.abs(n["y2"] - ref) <= Y_TOL * np.abs(ref))
    idx, w, _ = route_reference(n["logits"], K, True, bias=n["bias"], groups=4, top=2, best=2, renorm=True, scale=2.5)
    assert np.array_equal(n["ids"], idx) and np.all(np.abs(n["weights"] - w) <= 2 * ROUTE_TOL * 2.5)
    rg, rd = O.row_bytes(O.Q4_K, H), O.row_bytes(O.Q8_0, F)
    pick = list(some)
    act = n["act"].reshape(T, K, F)
    assert rel_l2(act[pick], oracle_swiglu(O.Q4_K, s.w_g, s.w_u, F * rg, rg, n["y2"][pick], n["ids"][pick], 0, E, F, H)) < 1e-5
    down = oracle_down(O.Q8_0, s.w_d, H * rd, rd, act[pick].reshape(len(pick) * K, F), n["ids"][pick], 0, E, n["weights"][pick],
                       n["h2"][pick], H, F)
    assert rel_l2(n["out"][pick], down) < 1e-5


def test_a_layer_captured_and_replayed():
    """Other rows, residuals, adapters and row starts in the same buffers: the replay gives what fresh calls give."""
    import torch
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        Q.set_stream(st.cuda_stream)
        s = Layer([5, 1, 30], [1, 0, 2])
        s.run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run()
        other = Layer([12, 3, 21], [3, -1, 0], seed=5)
        for k in ("x", "res", "adapter", "start"):
            getattr(s, k).copy_(getattr(other, k))
        g.replay()
        st.synchronize()
        got = {k: getattr(s, k).clone() for k in ("h1", "y1", "xq", "proj", "qkv", "h2", "y2", "logits", "ids", "weights", "act", "out")}
        s.run()
        st.synchronize()
        for k, v in got.items():
            assert torch.equal(v, getattr(s, k)), k
    Q.set_stream(None)
    Q.check_device()
