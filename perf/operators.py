"""Cases for the FP8 serving operators: residual + RMSNorm with an 8-bit output, the block-scaled FP8 linear
layer, SwiGLU with an 8-bit output, and expert routing with groups.

``run`` computes an operator either in elementary torch operations (``own`` false) or through the package's entry
points (``own`` true).  8-bit tensors are e4m3 with one fp32 scale per (row, 128 columns) or per 128 x 128 weight
block; they come back as the e4m3 values themselves, next to their scales.
"""

import math

import torch

own = False

BLK = 128
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
DT = {"bf16": torch.bfloat16, "fp32": torch.float32, "none": None}


def listed():
    return [
        # the norm between two blocks of a decoder layer, one token of one sequence: latency only
        dict(name="norm_token", op="norm", rows=1, hidden=4096, x="fp32", res="fp32", out="bf16", quant=False),
        # a decode batch entering a mixture-of-experts block: bf16 rows for the gate, e4m3 rows for the experts
        dict(name="norm_decode_moe", op="norm", rows=64, hidden=7168, x="bf16", res="fp32", out="bf16", quant=True),
        # a long prompt entering an FP8 projection: the bandwidth case
        dict(name="norm_prompt", op="norm", rows=8192, hidden=7168, x="bf16", res="bf16", out="none", quant=True),
        # one token through the gate/up projection of an FP8 feed-forward block: the weights are read once
        dict(name="linear_token", op="linear", m=1, n=4096, k=7168, acc=False, out="bf16"),
        # a decode batch through the gate/up projection of the decoder layer's feed-forward block (weights past L2)
        dict(name="linear_decode", op="linear", m=64, n=28672, k=4096, acc=False, out="bf16"),
        # a ragged piece of a prompt, the last K block cut short, added to the fp32 residual stream
        dict(name="linear_ragged", op="linear", m=777, n=1000, k=2000, acc=True, out="fp32"),
        # a long prompt through the same gate/up projection: the compute-bound case
        dict(name="linear_prompt", op="linear", m=8192, n=28672, k=4096, acc=False, out="bf16"),
        # activation of an expert-sized feed-forward block for a decode batch
        dict(name="swiglu_decode", op="swiglu", rows=64, inter=2048, x="bf16"),
        # activation of the decoder layer's feed-forward block for a long prompt
        dict(name="swiglu_prompt", op="swiglu", rows=8192, inter=14336, x="bf16"),
        # routing of one token, grouped sigmoid scores with a balance bias
        dict(name="route_token", op="route", tokens=1, experts=256, topk=8, groups=8, keep=4, best=2, scoring="sigmoid",
             bias=True, renorm=True, scale=2.5),
        # the same for a long prompt
        dict(name="route_prompt", op="route", tokens=16384, experts=256, topk=8, groups=8, keep=4, best=2,
             scoring="sigmoid", bias=True, renorm=True, scale=2.5),
        # softmax scores over a table that fills no power of two, no groups, weights as they come
        dict(name="route_softmax_odd", op="route", tokens=4099, experts=60, topk=6, groups=1, keep=1, best=1,
             scoring="softmax", bias=False, renorm=False, scale=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "swiglu", "route"])
    if op == "norm":
        hidden = _log(rng, 64, 16384)
        if rng.random() < 0.5:
            hidden = max(128, hidden // 128 * 128)
        rows = min(_log(rng, 1, 8192), max(1, 8192 * 7168 // (2 * hidden)))
        quant = rng.random() < 0.6
        out = rng.choice(["bf16", "fp32", "none"]) if quant else rng.choice(["bf16", "fp32"])
        return dict(op="norm", rows=rows, hidden=hidden, x=rng.choice(["bf16", "fp32"]), res=rng.choice(["bf16", "fp32"]),
                    out=out, quant=quant)
    if op == "linear":
        n = _log(rng, 32, 28672)
        k = max(16, _log(rng, 64, 14336) // 16 * 16)
        if rng.random() < 0.5:
            n, k = max(128, n // 128 * 128), max(128, k // 128 * 128)
        m = min(_log(rng, 1, 8192), max(1, 8192 * 28672 * 4096 // (n * k)))
        acc = rng.random() < 0.3
        return dict(op="linear", m=m, n=n, k=k, acc=acc, out="fp32" if acc else rng.choice(["bf16", "fp32"]))
    if op == "swiglu":
        inter = _log(rng, 64, 14336)
        if rng.random() < 0.5:
            inter = max(128, inter // 128 * 128)
        x = rng.choice(["bf16", "fp32"])
        rows = min(_log(rng, 1, 8192), max(1, 8192 * 14336 // (2 * inter)))
        return dict(op="swiglu", rows=rows, inter=inter, x=x)
    groups = rng.choice([1, 1, 2, 4, 8])
    per = max(2, _log(rng, 8, 512) // groups)
    keep = rng.randint(1, groups)
    topk = rng.randint(1, min(16, keep * per))
    return dict(op="route", tokens=_log(rng, 1, 16384) if groups * per <= 256 else _log(rng, 1, 8192), experts=groups * per,
                topk=topk, groups=groups, keep=keep, best=rng.choice([1, 2]), scoring=rng.choice(["sigmoid", "softmax"]),
                bias=rng.random() < 0.6, renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))


def _blocks(k):
    return (k + BLK - 1) // BLK


# ---------------------------------------------------------------- inputs

def _quantized_rows(x):
    """e4m3 rows with a scale per (row, 128 columns), as a producing layer hands them over."""
    m, k = x.shape
    pad = torch.nn.functional.pad(x, (0, _blocks(k) * BLK - k)).view(m, _blocks(k), BLK)
    s = pad.abs().amax(-1) / E4M3_MAX
    s = torch.where(s > 0, s, torch.ones_like(s))
    q = (pad / s.unsqueeze(-1)).view(m, -1)[:, :k]
    return q.to(E4M3).contiguous(), s.contiguous()


def _quantized_weight(n, k, g, dev):
    """e4m3 weight [n, k] with a scale per 128 x 128 block."""
    nb, kb = _blocks(n), _blocks(k)
    w = torch.zeros(nb * BLK, kb * BLK, device=dev)
    w[:n, :k].normal_(0.0, 0.02, generator=g)
    t = w.view(nb, BLK, kb, BLK)
    s = t.abs().amax((1, 3)) / E4M3_MAX
    s = torch.where(s > 0, s, torch.ones_like(s))
    t /= s.view(nb, 1, kb, 1)
    return w[:n, :k].to(E4M3).contiguous(), s.contiguous()


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    st = dict(case)
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        st["x"] = normal(rows, hidden).to(DT[case["x"]])
        st["res"] = (normal(rows, hidden) * 3.0).to(DT[case["res"]])
        st["res_out"] = torch.empty_like(st["res"])
        st["gamma"] = 1.0 + 0.1 * normal(hidden)
        st["eps"] = 1e-6
    elif case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st["a"], st["a_scale"] = _quantized_rows(normal(m, k) * torch.exp(normal(1, k)))
        st["w"], st["w_scale"] = _quantized_weight(n, k, g, dev)
        st["acc_in"] = normal(m, n) if case["acc"] else None
        st["y"] = torch.empty(m, n, dtype=DT[case["out"]], device=dev)
    elif case["op"] == "swiglu":
        st["gate_up"] = (normal(case["rows"], 2 * case["inter"]) * 1.5).to(DT[case["x"]])
    else:
        st["logits"] = normal(case["tokens"], case["experts"])
        st["bias_t"] = (torch.rand(case["experts"], generator=g, device=dev) * 0.2 - 0.1) if case["bias"] else None
    return st


# ---------------------------------------------------------------- one pass

def run(st):
    return (_own if own else _plain)[st["op"]](st)


def _own_norm(st):
    from pypto_b200 import ops
    if st["quant"]:
        r = ops.add_rms_norm_quantize(st["x"], st["res"], st["gamma"], st["eps"], DT[st["out"]], residual_out=st["res_out"])
        q, s, y = r if st["out"] != "none" else (*r, None)
        return {"residual": st["res_out"], "normed": y, "q": q, "scale": s}
    y = ops.add_rms_norm(st["x"], st["res"], st["gamma"], st["eps"], DT[st["out"]], residual_out=st["res_out"])
    return {"residual": st["res_out"], "normed": y, "q": None, "scale": None}


def _own_linear(st):
    from pypto_b200 import ops
    return ops.linear_fp8(st["a"], st["a_scale"], st["w"], st["w_scale"], acc=st["acc_in"], out=st["y"])


def _own_swiglu(st):
    from pypto_b200 import ops
    q, s = ops.swiglu_quantize(st["gate_up"])
    return {"q": q, "scale": s}


def _own_route(st):
    from pypto_b200 import ops
    idx, w = ops.moe_route(st["logits"], st["topk"], bias=st["bias_t"], scoring=st["scoring"], n_group=st["groups"],
                           topk_group=st["keep"], group_top=st["best"], renormalize=st["renorm"], route_scale=st["scale"])
    return {"idx": idx, "weights": w}


def _to_e4m3(y):
    m, k = y.shape
    pad = torch.nn.functional.pad(y, (0, _blocks(k) * BLK - k)).view(m, _blocks(k), BLK)
    amax = pad.abs().amax(-1)
    s = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    return (pad / s.unsqueeze(-1)).view(m, -1)[:, :k].to(E4M3).contiguous(), s


def _plain_norm(st):
    h = st["x"].float() + st["res"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + st["eps"]) * st["gamma"]
    q, s = _to_e4m3(y) if st["quant"] else (None, None)
    return {"residual": h.to(st["res"].dtype), "normed": None if st["out"] == "none" else y.to(DT[st["out"]]), "q": q,
            "scale": s}


def _plain_linear(st):
    m, n, k = st["m"], st["n"], st["k"]
    a = st["a"].float() * st["a_scale"].repeat_interleave(BLK, 1)[:, :k]
    w = st["w"].float() * st["w_scale"].repeat_interleave(BLK, 0)[:n].repeat_interleave(BLK, 1)[:, :k]
    y = a @ w.t()
    if st["acc_in"] is not None:
        y = y + st["acc_in"]
    return y.to(DT[st["out"]])


def _plain_swiglu(st):
    x = st["gate_up"].float()
    gate, up = x[:, : st["inter"]], x[:, st["inter"]:]
    q, s = _to_e4m3(gate / (1.0 + torch.exp(-gate)) * up)
    return {"q": q, "scale": s}


def _descending(v):
    return torch.sort(v, dim=-1, descending=True, stable=True)


def _plain_route(st):
    # 64 bits: choices next to a border must not depend on a rounding
    x = st["logits"].double()
    t, e = x.shape
    if st["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        p = torch.exp(x - x.amax(-1, keepdim=True))
        score = p / p.sum(-1, keepdim=True)
    key = score if st["bias_t"] is None else score + st["bias_t"].double()
    if st["keep"] < st["groups"]:
        by_group = key.view(t, st["groups"], -1)
        of_group = _descending(by_group)[0][..., : st["best"]].sum(-1)
        kept = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, _descending(of_group)[1][:, : st["keep"]], True)
        key = by_group.masked_fill(~kept.unsqueeze(-1), -math.inf).view(t, e)
    idx = _descending(key)[1][:, : st["topk"]]
    w = score.gather(1, idx)
    if st["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return {"idx": idx.to(torch.int32), "weights": (w * st["scale"]).float()}


_own = {"norm": _own_norm, "linear": _own_linear, "swiglu": _own_swiglu, "route": _own_route}
_plain = {"norm": _plain_norm, "linear": _plain_linear, "swiglu": _plain_swiglu, "route": _plain_route}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = {"bf16": 2, "fp32": 4, "none": 0}
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        b = n * (size[case["x"]] + 2 * size[case["res"]] + size[case["out"]]) + 4 * case["hidden"]
        if case["quant"]:
            b += n + 4 * case["rows"] * _blocks(case["hidden"])
        return {"bytes": b, "flops": 6 * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        b = (m + n) * k + 4 * _blocks(k) * (m + _blocks(n)) + m * n * size[case["out"]] + (4 * m * n if case["acc"] else 0)
        return {"bytes": b, "flops": 2 * m * n * k}
    if case["op"] == "swiglu":
        n = case["rows"] * case["inter"]
        return {"bytes": n * (2 * size[case["x"]] + 1) + 4 * case["rows"] * _blocks(case["inter"]), "flops": 8 * n}
    t, e = case["tokens"], case["experts"]
    return {"bytes": 4 * t * e + 8 * t * case["topk"] + (4 * e if case["bias"] else 0), "flops": 8 * t * e}


# ---------------------------------------------------------------- the definitions in 64 bits

def _group_scale(v):
    """v [rows, k] double -> (v / scale not rounded to 8 bits, scale): the value that a stored e4m3 number stands in
    for, and the scale."""
    m, k = v.shape
    col = torch.arange(k, device=v.device) // BLK
    top = torch.zeros(m, _blocks(k), dtype=torch.float64, device=v.device)
    top.scatter_reduce_(1, col.expand(m, k), v.abs(), "amax")
    s = torch.where(top == 0, 1.0, top / E4M3_MAX)
    return v / s[:, col], s


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        h = st["x"].double().add_(st["res"].double())
        ms = torch.linalg.vecdot(h, h) / case["hidden"]
        y = h / torch.sqrt(ms + st["eps"]).unsqueeze(1) * st["gamma"].double()
        q, s = _group_scale(y) if case["quant"] else (None, None)
        return {"residual": h, "normed": None if case["out"] == "none" else y, "q": q, "scale": s}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros(m, n, dtype=torch.float64, device=st["a"].device) if st["acc_in"] is None else st["acc_in"].double()
        feature = torch.arange(n, device=y.device) // BLK
        for b in range(_blocks(k)):      # the definition, one block of 128 channels after another
            cols = slice(b * BLK, min(k, (b + 1) * BLK))
            rows = st["a"][:, cols].double() * st["a_scale"][:, b: b + 1].double()
            y.addmm_(rows, (st["w"][:, cols].double() * st["w_scale"][:, b].double()[feature].unsqueeze(1)).T)
        return y
    if case["op"] == "swiglu":
        gate, up = st["gate_up"].double().split(case["inter"], dim=1)
        q, s = _group_scale(torch.special.expit(gate) * gate * up)
        return {"q": q, "scale": s}
    import numpy as np
    x = st["logits"].cpu().numpy().astype(np.float64)
    t, e = x.shape
    if case["scoring"] == "sigmoid":
        score = 0.5 * (1.0 + np.tanh(0.5 * x))
    else:
        score = np.exp(x - np.logaddexp.reduce(x, axis=1, keepdims=True))
    key = score.copy() if st["bias_t"] is None else score + st["bias_t"].cpu().numpy().astype(np.float64)
    per = e // case["groups"]
    best = np.sort(key.reshape(t, case["groups"], per), axis=2)[:, :, max(0, per - case["best"]):].sum(axis=2)
    for_out = np.argsort(-best, axis=1, kind="stable")[:, case["keep"]:]
    group = np.arange(e) // per
    dropped = np.zeros((t, case["groups"]), dtype=bool)
    np.put_along_axis(dropped, for_out, True, axis=1)
    key[dropped[:, group]] = -np.inf
    idx = np.argsort(-key, axis=1, kind="stable")[:, : case["topk"]]
    w = np.take_along_axis(score, idx, axis=1)
    if case["renorm"]:
        w = w / w.sum(axis=1, keepdims=True)
    return {"idx": idx.astype(np.int32), "weights": w * case["scale"]}
