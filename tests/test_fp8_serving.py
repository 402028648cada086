"""FP8 serving operators without a GPU: what the C ABI and the Python front end refuse, and the oracle's own checks."""

import math

import pytest
import torch

from oracle import fp8_serving as o

P = 1 << 20        # a pointer that no refused call follows
BF16, FP32, FP16 = 1, 0, 2


def _call(name, *args):
    from pypto_b200 import _lib
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.pto_last_error().decode()


def _norm(x=P, xdt=BF16, res=P, res_out=P, rdt=FP32, gamma=P, out=P, odt=BF16, q=None, s=None, rows=4, hidden=64, eps=1e-6):
    return _call("pto_add_rms_norm", x, xdt, res, res_out, rdt, gamma, out, odt, q, s, rows, hidden, eps, None)


def _linear(x=P, xs=P, w=P, ws=P, acc=None, out=P, odt=BF16, m=4, n=64, k=128):
    return _call("pto_linear_fp8", x, xs, w, ws, acc, out, odt, m, n, k, None, None)


def _route(logits=P, dt=FP32, bias=None, scoring=0, tokens=4, experts=64, ng=1, tg=1, gt=2, topk=4, idx=P, w=P):
    return _call("pto_moe_route", logits, dt, bias, scoring, tokens, experts, ng, tg, gt, topk, 1, 1.0, idx, w, None)


def _swiglu(x=P, dt=BF16, q=P, s=P, rows=4, inter=64):
    return _call("pto_swiglu_quantize", x, dt, q, s, rows, inter, None)


@pytest.mark.parametrize("call, kw, words", [
    (_norm, dict(hidden=0), "hidden"), (_norm, dict(hidden=49153), "hidden"), (_norm, dict(rows=-1), "rows"),
    (_norm, dict(rows=1 << 31), "rows"), (_norm, dict(xdt=FP16), "x must"), (_norm, dict(rdt=FP16), "residual"),
    (_norm, dict(odt=FP16), "out"), (_norm, dict(out=None), "neither"), (_norm, dict(q=P), "both"),
    (_norm, dict(s=P), "both"), (_norm, dict(eps=-1.0), "eps"), (_norm, dict(eps=math.nan), "eps"), (_norm, dict(x=None), "NULL"),
    (_norm, dict(x=8 * P, res_out=P + 64), "overlaps residual"), (_norm, dict(x=P + 1024 - 4, res_out=P, res=None), "overlaps x"),
    (_norm, dict(res=None), "overlaps x"), (_norm, dict(x=P + 1024, res_out=P + 4, res=None), "overlaps x"),
    (_linear, dict(n=0), "positive"), (_linear, dict(k=0), "positive"), (_linear, dict(m=-1), "positive"),
    (_linear, dict(m=(1 << 30) + 1), "2^30"), (_linear, dict(odt=FP16), "out"), (_linear, dict(x=None), "NULL"), (_linear, dict(ws=None), "NULL"),
    (_linear, dict(acc=P), "fp32 out"), (_linear, dict(acc=P + 4, odt=FP32), "overlaps acc"),
    (_linear, dict(acc=P - 1024 + 4), "overlaps acc"), (_linear, dict(acc=P + 512 - 4), "overlaps acc"),
    (_swiglu, dict(dt=FP16), "gate_up"), (_swiglu, dict(inter=0), "sizes"), (_swiglu, dict(rows=-1), "sizes"),
    (_swiglu, dict(q=None), "NULL"),
    (_route, dict(dt=FP16), "logits"), (_route, dict(scoring=2), "scoring"), (_route, dict(experts=1025), "experts"),
    (_route, dict(experts=0), "experts"), (_route, dict(tokens=(1 << 30) + 1), "tokens"), (_route, dict(ng=5, tg=2), "evenly"), (_route, dict(ng=4, tg=5), "topk_group"),
    (_route, dict(ng=4, tg=0), "topk_group"), (_route, dict(gt=3), "group_top"), (_route, dict(topk=0), "topk"),
    (_route, dict(topk=33), "topk"), (_route, dict(ng=32, tg=1, topk=3), "topk"), (_route, dict(idx=None), "NULL"),
])
def test_c_abi_refuses_before_any_launch(call, kw, words):
    status, message = call(**kw)
    assert status == 1 and words in message, (status, message)


def test_empty_calls_do_nothing():
    assert _norm(rows=0, x=None)[0] == 0
    assert _linear(m=0, x=None, out=None)[0] == 0
    assert _swiglu(rows=0, x=None, q=None, s=None)[0] == 0
    assert _route(tokens=0, logits=None, idx=None, w=None)[0] == 0


def test_python_front_end_refuses_cpu_tensors_and_bad_routings():
    from pypto_b200 import BackendUnavailable, ops
    x = torch.zeros(2, 128)
    with pytest.raises(BackendUnavailable):
        ops.add_rms_norm(x, x, None, 1e-6)
    with pytest.raises(BackendUnavailable):
        ops.swiglu_quantize(x)
    with pytest.raises(BackendUnavailable):
        ops.moe_route(x, 2)
    with pytest.raises(BackendUnavailable):
        ops.linear_fp8(x.to(ops.FP8), x[:, :1], x.to(ops.FP8), x[:1, :1])
    for bad in (dict(scoring="tanh"), dict(n_group=3), dict(n_group=4, topk_group=0), dict(group_top=0), dict(topk=0),
                dict(n_group=8, topk_group=1, topk=9), dict(experts=2000)):
        kw = dict(experts=64, topk=4, scoring="sigmoid", n_group=1, topk_group=1, group_top=2) | bad
        with pytest.raises(ValueError):
            ops.check_routing(**kw)


def test_layer_objects_check_their_arguments():
    from pypto_b200.layers import Fp8SwiGLUFFN, quantize_weight
    from pypto_b200.moe import MoELayer, Router
    g = torch.Generator().manual_seed(0)
    w = torch.randn(200, 300, generator=g)
    q, s = quantize_weight(w)
    assert q.shape == (300, 200) and s.shape == (3, 2) and q.is_contiguous()
    back = q.double() * s.double().repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :200]
    # half an e4m3 step of the value, or half the smallest step (2^-10) of the scale
    assert (back - w.t().double()).abs().le(2 ** -4 * w.t().double().abs() + 2.0 ** -10 * s.max().item() + 1e-6).all()
    with pytest.raises(ValueError):
        Fp8SwiGLUFFN((q, s), (q, s), torch.ones(200), 1e-6)
    down, down_s = quantize_weight(torch.randn(150, 200, generator=g))
    Fp8SwiGLUFFN((q, s), (down, down_s), torch.ones(200), 1e-6)
    for bad in ((down, down_s[:, :1]), (down.float(), down_s)):
        with pytest.raises(ValueError):
            Fp8SwiGLUFFN((q, s), bad, torch.ones(200), 1e-6)
    with pytest.raises(ValueError):
        MoELayer.from_packed(torch.zeros(6, 128, dtype=torch.bfloat16), torch.zeros(6), dict(w_gu=torch.zeros(6, 256, 128)), None,
                             topk=2, router=Router(n_group=4, topk_group=2))


def test_oracle_route_by_hand():
    # two groups of three; the second group's best two beat the first's although the best expert sits in the first
    bias = torch.tensor([0.9, -1.0, -1.0, 0.3, 0.35, -1.0])
    idx, w = o.route(torch.zeros(1, 6), 2, bias, n_group=2, topk_group=1, group_top=2)
    assert idx.tolist() == [[4, 3]] and w.tolist() == [[0.5, 0.5]]
    idx, _ = o.route(torch.zeros(1, 6), 2, bias, n_group=2, topk_group=1, group_top=1)
    assert idx.tolist() == [[0, 1]]
    idx, w = o.route(torch.zeros(1, 4), 3, torch.tensor([-math.inf, 0.0, -math.inf, -math.inf]))
    assert idx.tolist() == [[1, 0, 2]] and w.tolist() == [[1.0, 0.0, 0.0]]
    idx, w = o.route(torch.tensor([[1.0, 3.0, 2.0]]), 2, scoring="softmax", renormalize=False, route_scale=2.0)
    p = torch.softmax(torch.tensor([1.0, 3.0, 2.0], dtype=torch.float64), 0)
    assert idx.tolist() == [[1, 2]] and torch.allclose(w[0], 2 * p[[1, 2]])
