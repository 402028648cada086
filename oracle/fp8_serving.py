"""Oracle of the FP8 serving operators, in 64 bits (test infrastructure, not product code).

PARITY UNPINNED: the reference has no FP8 row format with 128-wide fp32 scales, no dense product over it and no router.
This file is the only definition of

  add_rms_norm     h = x + residual; y = h / sqrt(mean(h^2) + eps) * gamma
  group_scale      max |y| / 448 over 128 columns, 1 where that is 0
  linear_fp8       (acc +) sum over K blocks of x_scale * w_scale * (sum of e4m3 products)
  swiglu           g * sigmoid(g) * u
  route            scores, keys, groups, top-k and weights, one row at a time in plain Python

and of the bounds that rounding in 32 bits can reach around them.
"""

from __future__ import annotations

import math

import torch

BLK = 128


def add_rms_norm(x, residual, gamma, eps):
    """(h, y) in 64 bits."""
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, y if gamma is None else y * gamma.double()


def group_scale(y):
    """[rows, k] -> scale of every (row, 128 columns)."""
    rows, k = y.shape
    pad = torch.zeros(rows, -(-k // BLK) * BLK, dtype=y.dtype, device=y.device)
    pad[:, :k] = y
    amax = pad.view(rows, -1, BLK).abs().amax(-1)
    return torch.where(amax > 0, amax / 448, torch.ones_like(amax))


def per_column(scale, k):
    """scale [rows, groups] -> [rows, k]."""
    return scale.repeat_interleave(BLK, 1)[:, :k]


def linear_fp8(x, x_scale, w, w_scale, acc=None):
    """(out, sum of the magnitudes of its terms) in 64 bits."""
    n, k = w.shape
    xd = x.double() * per_column(x_scale.double(), k)
    wd = w.double() * per_column(w_scale.double(), k).repeat_interleave(BLK, 0)[:n]
    y, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    return (y, mag) if acc is None else (y + acc.double(), mag + acc.double().abs())


def linear_fp8_bound(mag, k):
    """What fp32 arithmetic can be off by: a term of the sum goes through at most 128 additions inside its K block
    (products of e4m3 numbers are exact), a multiplication by the product of two scales (itself rounded), the additions
    of the K blocks, of up to 16 partial sums and of acc; a step of the tensor core's adder may drop the last bit
    (2^-23) where a rounding one is off by half of it."""
    return (BLK + -(-k // BLK) + 16 + 4) * 2.0 ** -23 * mag


def swiglu(gate_up):
    g, u = gate_up.double().chunk(2, dim=1)
    return g * torch.sigmoid(g) * u


def route_row(logits, topk, bias=None, scoring="sigmoid", n_group=1, topk_group=1, group_top=2, renormalize=True,
              route_scale=1.0):
    """One row of logits (a list of floats) -> (indices, weights).  64-bit arithmetic, ties to the lower id; an expert whose
    key is -inf or NaN is not available and adds nothing to its group."""
    e = len(logits)
    if scoring == "sigmoid":
        score = [v if math.isnan(v) else (1 / (1 + math.exp(-v)) if v > -700 else 0.0) for v in logits]
    else:
        top = max([v for v in logits if not math.isnan(v)], default=-math.inf)
        if math.isinf(top):
            p = [v if math.isnan(v) else (1.0 if top > 0 and v == top else 0.0) for v in logits]
        else:
            p = [v if math.isnan(v) else math.exp(v - top) for v in logits]
        total = math.fsum(v for v in p if not math.isnan(v))
        score = [v / total if total > 0 else v for v in p]
    key = [s + (0.0 if bias is None else bias[i]) for i, s in enumerate(score)]
    out = [math.isnan(v) or v == -math.inf for v in key]
    if topk_group < n_group:
        per = e // n_group
        of_group = []
        for g in range(n_group):
            have = sorted((key[i] for i in range(g * per, (g + 1) * per) if not out[i]), reverse=True)[:group_top]
            of_group.append(sum(have) if have else -math.inf)
        kept = sorted(range(n_group), key=lambda g: (-of_group[g], g))[:topk_group]
        out = [out[i] or i // per not in kept for i in range(e)]
    order = sorted(range(e), key=lambda i: (out[i], 0.0 if out[i] else -key[i], i))[:topk]
    w = [0.0 if out[i] else score[i] for i in order]
    if renormalize:
        total = sum(w)
        w = [v / total if total > 0 else 0.0 for v in w]
    return order, [v * route_scale for v in w]


def route(logits, topk, bias=None, **options):
    rows = [route_row(r, topk, None if bias is None else bias.double().tolist(), **options) for r in logits.double().tolist()]
    return (torch.tensor([r[0] for r in rows], dtype=torch.int32).reshape(len(rows), topk),
            torch.tensor([r[1] for r in rows], dtype=torch.float64).reshape(len(rows), topk))


def route_weight_bound(logits, topk):
    """Relative error that a weight may have from 32-bit scores: the exponential is within 2 ulp of its rounded argument
    (the argument of softmax, logit - max, is off by half an ulp of itself, which the exponential turns into that much
    relative error), then an addition, two divisions, the product with the route scale and the sums of the softmax (a
    tree of at most 32 terms a lane and five levels) and of the topk scores."""
    x = logits.double()
    x = x[torch.isfinite(x)]
    span = float(x.max() - x.min()) if x.numel() else 0.0
    return (span + 32 + 5 + topk + 12) * 2.0 ** -23
