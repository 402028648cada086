"""FP8 serving operators on the GPU against their definitions in 64 bits: residual + RMSNorm with FP8 rows, the
block-scaled FP8 linear layer, SwiGLU with FP8 rows, expert routing, and runs of them together."""

import math

import pytest
import torch

from oracle import fp8_serving as o

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, FP32: 2.0 ** -24}      # a rounding is off by at most this, relative to the value


def _ops():
    from pypto_b200 import ops
    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _fp8_rows(x):
    """FP8 rows with a scale per (row, 128 columns)."""
    s = o.group_scale(x.double()).float()
    return (x / o.per_column(s, x.shape[1])).to(_ops().FP8).contiguous(), s.contiguous()


def _fp8_weight(g, n, k):
    from pypto_b200.layers import quantize_weight
    return quantize_weight(_randn(g, k, n) * 0.02)


def _guarded(shape, dtype):
    """A tensor inside a larger allocation and a check that nothing around it was written."""
    n, pad = math.prod(shape), 256
    whole = torch.full((n + 2 * pad,), 7.0, device="cuda").to(dtype)
    def check():
        w = whole.float()
        assert (w[:pad] == 7).all() and (w[pad + n:] == 7).all(), "written outside the tensor"
    return whole[pad:pad + n].view(shape), check


# ---------------------------------------------------------------------------
# add_rms_norm
# ---------------------------------------------------------------------------

def _norm_bound(hidden):
    # squares are added hidden / 256 a thread and over 13 levels, the mean enters under a square root (half of its
    # error); rsqrtf is within 2 ulp (2^-22); the sum h, the mean, eps and two products round once each
    return (hidden / 512 + 7 + 4 + 5) * 2.0 ** -24


NORM_SIZES = [(1, 1), (1, 4096), (3, 7), (5, 130), (2, 1000), (64, 7168), (33, 2048), (7, 128), (4, 1032), (300, 640),
              (2, 16384), (3, 16392), (2, 20000), (1, 49152), (3, 5003), (2, 16383), (5, 2050), (2, 777), (4, 10222),
              (3, 1030), (2, 8189), (2, 12001), (1, 6142)]


@pytest.mark.parametrize("rows, hidden", NORM_SIZES)
@pytest.mark.parametrize("xdt, rdt, odt", [(BF16, FP32, BF16), (BF16, BF16, FP32), (FP32, FP32, FP32), (FP32, BF16, BF16)])
def test_add_rms_norm(rows, hidden, xdt, rdt, odt):
    g = _gen(rows * 31 + hidden)
    x, res = _randn(g, rows, hidden).to(xdt), (3 * _randn(g, rows, hidden)).to(rdt)
    gamma = 1 + 0.1 * _randn(g, hidden)
    h, y = o.add_rms_norm(x, res, gamma, 1e-6)
    before = res.clone()
    res_out, check = _guarded((rows, hidden), rdt)
    out = _ops().add_rms_norm(x, res, gamma, 1e-6, odt, residual_out=res_out)
    check()
    assert torch.equal(res, before)
    assert torch.equal(res_out, (x.float() + res.float()).to(rdt))
    bound = (_norm_bound(hidden) + HALF[odt]) * y.abs()
    assert out.dtype == odt and ((out.double() - y).abs() <= bound).all()
    # in place, and without gamma
    out2 = _ops().add_rms_norm(x, res, gamma, 1e-6, odt)
    assert torch.equal(res, res_out) and torch.equal(out2, out)
    _, y = o.add_rms_norm(x, None, None, 1e-5)
    out = _ops().add_rms_norm(x, None, None, 1e-5, odt)
    assert ((out.double() - y).abs() <= (_norm_bound(hidden) + HALF[odt]) * y.abs()).all()


def _check_fp8_rows_of(out32, q, scale):
    """q and scale are exactly the FP8 rows of the fp32 values."""
    y = out32.cpu()
    rows, k = y.shape
    amax = torch.zeros(rows, scale.shape[1] * 128)
    amax[:, :k] = y.abs()
    amax = amax.view(rows, -1, 128).amax(-1)
    s = torch.where(amax > 0, amax / torch.full_like(amax, 448.0), torch.ones_like(amax))
    assert torch.equal(scale.cpu(), s)
    exp = (y / o.per_column(s, k)).clamp(-448, 448).to(_ops().FP8)
    assert torch.equal(q.cpu().view(torch.uint8), exp.view(torch.uint8))


@pytest.mark.parametrize("rows, hidden", NORM_SIZES)
@pytest.mark.parametrize("xdt, rdt", [(BF16, FP32), (BF16, BF16), (FP32, FP32), (FP32, BF16)])
def test_add_rms_norm_quantize(rows, hidden, xdt, rdt):
    ops = _ops()
    g = _gen(rows * 17 + hidden)
    x, res = _randn(g, rows, hidden).to(xdt), (3 * _randn(g, rows, hidden)).to(rdt)
    gamma = 1 + 0.1 * _randn(g, hidden)
    if hidden >= 256:
        gamma[128:256] = 0          # a group of zeros: scale 1, codes 0
    q, scale, y = ops.add_rms_norm_quantize(x, res, gamma, 1e-6, FP32, residual_out=torch.empty_like(res))
    assert q.dtype == ops.FP8 and q.shape == x.shape and scale.shape == (rows, (hidden + 127) // 128)
    assert torch.equal(y, ops.add_rms_norm(x, res, gamma, 1e-6, FP32, residual_out=torch.empty_like(res)))
    _check_fp8_rows_of(y, q, scale)
    q2, scale2, y2 = ops.add_rms_norm_quantize(x, res, gamma, 1e-6, BF16, residual_out=torch.empty_like(res))
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale2, scale) and torch.equal(y2, y.to(BF16))
    summed = (x.float() + res.float()).to(rdt)
    q3, scale3 = ops.add_rms_norm_quantize(x, res, gamma, 1e-6)      # in place this time
    assert torch.equal(res, summed)
    assert torch.equal(q3.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale3, scale)


def test_add_rms_norm_odd_values_and_alignment():
    ops = _ops()
    g = _gen(5)
    x = _randn(g, 6, 512)
    x[1, 7] = math.inf
    x[2, 9] = math.nan
    x[3] = 0
    x[4] *= 1e-30
    x[5] *= 1e18
    y = ops.add_rms_norm(x, None, None, 1e-6, FP32)
    ref = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6))
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.isnan(y[2]).all()
    assert torch.allclose(y[[0, 3, 4, 5]], ref[[0, 3, 4, 5]], rtol=1e-5, atol=0)
    q, s = ops.add_rms_norm_quantize(x, None, None, 1e-6)
    assert (s[3] == 1).all() and (q[3].float() == 0).all()
    assert torch.isnan(q[2].float()).all() and torch.isnan(q[1, 7].float()) and (q[1, :7].float() == 0).all()
    # a view that starts in the middle of a 16-byte unit gives what an aligned copy gives
    for dt in (BF16, FP32):
        flat = _randn(g, 4 * 640 + 3).to(dt)
        view = flat[3:].view(4, 640)
        gamma = _randn(g, 641)[1:]
        a = ops.add_rms_norm_quantize(view, view, gamma, 1e-6, FP32, residual_out=torch.empty_like(view))
        b = ops.add_rms_norm_quantize(view.clone(), view.clone(), gamma.clone(), 1e-6, FP32)
        # the two kernels may add the squares in another order
        assert torch.allclose(a[2], b[2], rtol=2 * _norm_bound(640), atol=0)
        _check_fp8_rows_of(a[2], a[0], a[1])
        _check_fp8_rows_of(b[2], b[0], b[1])


@pytest.mark.parametrize("hidden", [256, 777, 1030, 7168, 20000])
@pytest.mark.parametrize("dt", [BF16, FP32])
def test_add_rms_norm_sum_written_over_x(hidden, dt):
    from pypto_b200 import _lib
    ops = _ops()
    g = _gen(hidden)
    x, res = _randn(g, 40, hidden).to(dt), _randn(g, 40, hidden).to(dt)
    total = torch.empty_like(x)
    want = ops.add_rms_norm(x, res, None, 1e-6, residual_out=total)
    over, keep = x.clone(), res.clone()
    assert torch.equal(ops.add_rms_norm(over, keep, None, 1e-6, residual_out=over), want)
    assert torch.equal(over, total) and torch.equal(keep, res)
    both = x.clone()                                            # x + x, in place
    twice = ops.add_rms_norm(x, x.clone(), None, 1e-6)
    assert torch.equal(ops.add_rms_norm(both, both, None, 1e-6), twice) and torch.equal(both, 2 * x)
    flat = torch.zeros(41 * hidden, dtype=dt, device="cuda")
    with pytest.raises(_lib.PtoError):
        ops.add_rms_norm(flat[:40 * hidden].view(40, hidden), None, None, 1e-6, residual_out=flat[hidden:].view(40, hidden))


def test_add_rms_norm_refusals():
    ops = _ops()
    x = torch.zeros(4, 256, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, torch.zeros(4, 128, device="cuda"), None, 1e-6)
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, x.float(), None, 1e-6, residual_out=x.clone())
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, x.half(), None, 1e-6)
    with pytest.raises(TypeError):
        ops.add_rms_norm(x.half(), x, None, 1e-6)
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, x, torch.ones(256, device="cuda", dtype=BF16), 1e-6)
    with pytest.raises(ValueError):
        ops.add_rms_norm(x.t(), x.t(), None, 1e-6)
    with pytest.raises(TypeError):
        ops.add_rms_norm(x, x, None, 1e-6, torch.float16)
    with pytest.raises(TypeError):
        ops.add_rms_norm(x, x, None, 1e-6, None)
    empty = ops.add_rms_norm_quantize(x[:0], x[:0], None, 1e-6, BF16)
    assert [t.shape[0] for t in empty] == [0, 0, 0]


# ---------------------------------------------------------------------------
# swiglu_quantize
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows, inter", [(1, 1), (1, 2048), (3, 100), (5, 136), (64, 2048), (7, 1288), (260, 384), (2, 14336), (9, 5), (3, 5003), (2, 2050), (33, 258)])
@pytest.mark.parametrize("dt", [BF16, FP32])
def test_swiglu_quantize(rows, inter, dt):
    ops = _ops()
    x = (1.5 * _randn(_gen(rows + inter), rows, 2 * inter)).to(dt)
    q, s = ops.swiglu_quantize(x)
    a = o.swiglu(x)
    assert q.dtype == ops.FP8 and q.shape == (rows, inter) and s.shape == (rows, (inter + 127) // 128)
    # __expf is within 2 + 1.173 |g| ulp, |g| < 9 here; the sum, the quotient (2 ulp if approximate) and two products
    rel = 20 * 2.0 ** -23
    es = o.group_scale(a)
    assert ((s.double() - es).abs() <= (rel + 2.0 ** -23) * es).all()
    step = 2.0 ** -4 * a.abs() + 2.0 ** -10 * o.per_column(es, inter)      # half a step; below 2^-6 the step is fixed
    assert ((q.double() * o.per_column(s.double(), inter) - a).abs() <= step * (1 + 2.0 ** -10) + rel * a.abs()).all()


def test_swiglu_quantize_odd_values():
    ops = _ops()
    x = torch.zeros(4, 512, device="cuda")
    x[0, :256], x[0, 256:] = -200.0, 3.0            # sigmoid underflows
    x[1, :256], x[1, 256:] = 200.0, 0.5
    x[2, 3], x[2, 259] = math.nan, 1.0
    q, s = ops.swiglu_quantize(x)
    assert (q[0].float() == 0).all() and (s[0] == 1).all()
    assert (q[1].float() * s[1, 0] - 100).abs().max() < 1e-3 and (s[3] == 1).all()
    assert torch.isnan(q[2, 3].float()) and (q[2, 4:].float() == 0).all()
    flat = _randn(_gen(3), 3 * 512 + 1).to(BF16)
    a, b = ops.swiglu_quantize(flat[1:].view(3, 512)), ops.swiglu_quantize(flat[1:].view(3, 512).clone())
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    for bad in (x[:, :511].contiguous(), x.half()):
        with pytest.raises(ValueError):
            ops.swiglu_quantize(bad)
    assert ops.swiglu_quantize(x[:0])[0].shape == (0, 256)


# ---------------------------------------------------------------------------
# linear_fp8
# ---------------------------------------------------------------------------

LINEAR_SIZES = [(1, 1, 16), (1, 128, 128), (1, 4096, 1024), (2, 130, 144), (8, 640, 2064), (17, 257, 2000), (31, 1000, 512),
                (64, 512, 512), (65, 384, 1040), (100, 2048, 7168), (128, 128, 14336), (200, 1000, 2000), (257, 512, 400),
                (300, 640, 4096), (4500, 3, 5), (513, 1152, 128), (777, 1000, 2000), (1024, 4096, 1024), (1500, 2200, 528),
                (2049, 1025, 384), (5, 7, 5), (130, 129, 17), (70, 200, 333),
                # the tile of 64 tokens, unsplit and split by eight; of 128, split by four and unsplit; pairs with few tokens
                (64, 28672, 256), (50, 4096, 7168), (128, 4096, 4096), (512, 4096, 2048), (256, 28672, 528), (150, 512, 512),
                (40, 520, 4112)]


@pytest.mark.parametrize("m, n, k", LINEAR_SIZES)
def test_linear_fp8(m, n, k):
    ops = _ops()
    g = _gen(m * 7 + n * 3 + k)
    x, xs = _fp8_rows(_randn(g, m, k) * torch.exp(_randn(g, 1, k)))
    w, ws = _fp8_weight(g, n, k)
    acc = _randn(g, m, n)
    y, mag = o.linear_fp8(x, xs, w, ws)
    bound = o.linear_fp8_bound(mag, k)
    out, check = _guarded((m, n), FP32)
    ops.linear_fp8(x, xs, w, ws, out=out)
    check()
    ops.check_device_status()
    assert ((out.double() - y).abs() <= bound).all(), ((out.double() - y).abs() / bound).max()
    got = ops.linear_fp8(x, xs, w, ws)
    assert got.dtype == BF16 and torch.equal(got, out.to(BF16))        # one rounding of the same sum
    assert torch.equal(ops.linear_fp8(x, xs, w, ws, out_dtype=FP32), out)      # equal calls give equal bits
    y, mag = o.linear_fp8(x, xs, w, ws, acc)
    out2, check = _guarded((m, n), BF16)
    ops.linear_fp8(x, xs, w, ws, acc=acc, out=out2)
    check()
    assert ((out2.double() - y).abs() <= o.linear_fp8_bound(mag, k) + HALF[BF16] * y.abs()).all()
    into = acc.clone()
    assert ops.linear_fp8(x, xs, w, ws, acc=into, out=into) is into     # the residual stream, in place
    assert ((into.double() - y).abs() <= o.linear_fp8_bound(mag, k)).all() and torch.equal(into.to(BF16), out2)


@pytest.mark.parametrize("m, n, k", [(1, 256, 512), (16, 384, 1280), (64, 512, 512), (130, 256, 640), (600, 1024, 1024),
                                     (1100, 2304, 768)])
def test_linear_fp8_known_answers(m, n, k):
    """Small whole numbers and power-of-two scales: every sum is exact in fp32."""
    ops = _ops()
    g = _gen(m + n + k)
    x = torch.randint(-3, 4, (m, k), generator=g, device="cuda").float().to(ops.FP8)
    w = torch.randint(-3, 4, (n, k), generator=g, device="cuda").float().to(ops.FP8)
    xs = torch.exp2(torch.randint(-1, 2, (m, k // 128), generator=g, device="cuda").float())
    ws = torch.exp2(torch.randint(-1, 2, (n // 128, k // 128), generator=g, device="cuda").float())
    y, _ = o.linear_fp8(x, xs, w, ws)
    assert torch.equal(ops.linear_fp8(x, xs, w, ws, out_dtype=FP32), y.float())


def test_linear_fp8_odd_values_alignment_and_refusals():
    from pypto_b200 import _lib
    ops = _ops()
    g = _gen(9)
    m, n, k = 40, 200, 256
    x, xs = _fp8_rows(_randn(g, m, k))
    w, ws = _fp8_weight(g, n, k)
    want = ops.linear_fp8(x, xs, w, ws, out_dtype=FP32)
    # a NaN or an infinity stays in its row
    xs2, x2 = xs.clone(), x.clone()
    xs2[3, 1] = math.inf
    x2.view(torch.uint8)[5, 17] = 0x7F
    got = ops.linear_fp8(x2, xs2, w, ws, out_dtype=FP32)
    assert torch.isnan(got[5]).all() and not torch.isfinite(got[3]).any()
    keep = [i for i in range(m) if i not in (3, 5)]
    assert torch.equal(got[keep], want[keep])
    # operands that no tensor map can describe: unaligned, or rows that are not whole 16-byte units
    flat = torch.empty(m * k + 1, dtype=torch.uint8, device="cuda")
    flat[1:] = x.view(torch.uint8).reshape(-1)
    y, mag = o.linear_fp8(x, xs, w, ws)
    got = ops.linear_fp8(flat[1:].view(ops.FP8).view(m, k), xs, w, ws, out_dtype=FP32)
    assert ((got.double() - y).abs() <= o.linear_fp8_bound(mag, k)).all()
    # scales and outputs at any 4-byte (2-byte) boundary
    sflat, oflat = torch.empty(xs.numel() + 1, device="cuda"), torch.empty(m * n + 1, dtype=BF16, device="cuda")
    sflat[1:] = xs.reshape(-1)
    wflat = torch.empty(ws.numel() + 1, device="cuda")
    wflat[1:] = ws.reshape(-1)
    got = ops.linear_fp8(x, sflat[1:].view(xs.shape), w, wflat[1:].view(ws.shape), out=oflat[1:].view(m, n))
    assert torch.equal(got, want.to(BF16))
    assert ops.linear_fp8(x[:0], xs[:0], w, ws).shape == (0, n)
    stream = torch.zeros(m + 1, n, device="cuda")               # the sum one row off its own place
    with pytest.raises(_lib.PtoError):
        ops.linear_fp8(x, xs, w, ws, acc=stream[:m], out=stream[1:])
    for args, kw, err in [((x, xs[:, :1].contiguous(), w, ws), {}, ValueError), ((x, xs, w, ws[:1].contiguous()), {}, ValueError),
                          ((x.view(torch.uint8), xs, w, ws), {}, TypeError), ((x, xs.double(), w, ws), {}, TypeError),
                          ((x[:, :128].contiguous(), xs[:, :1].contiguous(), w, ws), {}, ValueError),
                          ((x, xs, w, ws), dict(out=want.half()), ValueError), ((x, xs, w, ws), dict(out_dtype=torch.float16), TypeError),
                          ((x, xs, w, ws), dict(acc=want.to(BF16)), ValueError), ((x[:, ::2], xs, w, ws), {}, ValueError)]:
        with pytest.raises(err):
            ops.linear_fp8(*args, **kw)


# ---------------------------------------------------------------------------
# moe_route
# ---------------------------------------------------------------------------

def _check_route(logits, topk, bias=None, **kw):
    ops = _ops()
    dev = logits.cuda()
    idx, w = ops.moe_route(dev, topk, bias=None if bias is None else bias.cuda(), **kw)
    ei, ew = o.route(logits, topk, bias, **kw)
    assert idx.dtype == torch.int32 and torch.equal(idx.cpu(), ei), (idx.cpu() != ei).any(1).nonzero()[:5]
    bound = o.route_weight_bound(logits, topk) * ew
    assert ((w.cpu().double() - ew).abs() <= bound + 1e-40).all()
    return idx, w


ROUTES = [(1, 256, 8, 8, 4, 2), (300, 256, 8, 8, 4, 2), (77, 160, 6, 8, 3, 1), (65, 64, 6, 1, 1, 1), (9, 60, 6, 1, 1, 1), (50, 256, 8, 1, 1, 1),
          (5, 1, 1, 1, 1, 1), (7, 8, 8, 2, 2, 2), (33, 512, 32, 16, 9, 2), (11, 1024, 16, 4, 1, 2), (6, 900, 10, 30, 5, 1),
          (13, 96, 4, 48, 7, 2), (3, 31, 3, 31, 10, 2), (20, 128, 9, 4, 2, 1), (4, 512, 1, 1, 1, 1)]


@pytest.mark.parametrize("tokens, experts, topk, n_group, topk_group, group_top", ROUTES)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route(tokens, experts, topk, n_group, topk_group, group_top, scoring):
    g = torch.Generator().manual_seed(tokens + experts + topk)
    logits = 2 * torch.randn(tokens, experts, generator=g)
    bias = 0.2 * torch.rand(experts, generator=g) - 0.1
    kw = dict(scoring=scoring, n_group=n_group, topk_group=topk_group, group_top=group_top)
    _check_route(logits, topk, bias, **kw)
    _check_route(logits, topk, None, renormalize=False, route_scale=2.5, **kw)
    _check_route(logits.to(BF16), topk, bias, **kw)        # many equal logits


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route_ties_and_borders(scoring):
    """Choices that 32 bits cannot tell apart: equal keys, keys and group scores a few 2^-30 apart, saturated scores."""
    g = torch.Generator().manual_seed(3)
    same = torch.zeros(4, 64)
    kw = dict(scoring=scoring)
    _check_route(same, 8, **kw)
    _check_route(same, 8, n_group=8, topk_group=4, group_top=2, **kw)
    near = torch.randn(1, 256, generator=g).repeat(200, 1)
    near += 1e-7 * torch.randn(200, 256, generator=g)          # one or two ulp
    _check_route(near, 8, **kw)
    pairs = torch.randn(100, 128, generator=g).repeat_interleave(2, 1)
    pairs[:, 1::2] = torch.nextafter(pairs[:, ::2], torch.full_like(pairs[:, ::2], 9.0))
    _check_route(pairs, 8, **kw)
    _check_route(pairs, 8, n_group=8, topk_group=4, group_top=2, **kw)
    # equal keys made of different scores and biases: a bias that cancels the score's difference to the last bits
    logits = torch.randn(50, 32, generator=g)
    bias = (0.5 - torch.sigmoid(logits[0].double())).float()
    _check_route(logits[:1].repeat(3, 1), 6, bias, scoring="sigmoid")
    _check_route(logits[:1].repeat(3, 1), 6, bias, scoring="sigmoid", n_group=4, topk_group=2, group_top=2)
    wide = 60 * torch.randn(40, 96, generator=g)                # sigmoid saturates; softmax underflows
    _check_route(wide, 8, torch.zeros(96), **kw)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("depth", [79.0, 86.5, 95.0, 104.0, 300.0])
def test_route_weights_of_the_lowest_scores(scoring, depth):
    """Scores of e^-79 to e^-300 share the weight of a row in their own proportions."""
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(20, 64, generator=g) - depth
    bias = None
    if scoring == "softmax":                                    # one expert has the mass; the bias keeps it out
        logits[:, 63] = 0
        bias = torch.zeros(64)
        bias[63] = -math.inf
    for kw in (dict(), dict(n_group=8, topk_group=4, group_top=2)):
        _, w = _check_route(logits, 6, bias, scoring=scoring, **kw)
        assert ((w.double().sum(1) - 1).abs() <= 10 * 2.0 ** -23).all()
        _check_route(logits, 6, bias, scoring=scoring, renormalize=False, **kw)
    _check_route(logits[:, 40:].contiguous(), 6, None if bias is None else bias[40:], scoring=scoring)      # no more experts than lanes


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route_masks_and_odd_values(scoring):
    g = torch.Generator().manual_seed(4)
    inf = math.inf
    logits = torch.randn(30, 64, generator=g)
    bias = torch.zeros(64)
    bias[torch.randperm(64, generator=g)[:50]] = -inf           # 14 experts left
    for kw in (dict(), dict(n_group=8, topk_group=4, group_top=2), dict(n_group=8, topk_group=2, group_top=1)):
        idx, w = _check_route(logits, 8, bias, scoring=scoring, **kw)
        assert all(len(set(r)) == 8 for r in idx.cpu().tolist())
    _check_route(logits, 20, bias, scoring=scoring)             # more asked than there are: filled at weight 0
    idx, w = _check_route(logits, 4, torch.full((64,), -inf), scoring=scoring)
    assert idx.cpu().tolist() == [[0, 1, 2, 3]] * 30 and (w == 0).all()
    low = torch.finfo(FP32).min                                 # the other way to mask: availability by value
    masked = torch.where(torch.isinf(bias), torch.full_like(bias, low), bias)
    big = 1e6 * torch.where(torch.rand(64, generator=g) < 0.5, -1.0, 1.0)
    for b in (masked, big, big + 0.1 * torch.randn(64, generator=g)):
        for kw in (dict(), dict(n_group=8, topk_group=4, group_top=2), dict(n_group=8, topk_group=3, group_top=1),
                   dict(n_group=4, topk_group=3, group_top=2)):
            _check_route(logits, 8, b, scoring=scoring, **kw)
    odd = logits.clone()
    odd[0, 5] = math.nan
    odd[1] = math.nan
    odd[2, 7] = inf
    odd[3, 7] = odd[3, 9] = inf
    odd[4] = -inf
    odd[5, :60] = -inf
    odd[6, 3] = torch.finfo(FP32).max
    odd[7] = torch.finfo(FP32).min
    odd[8, ::2] = torch.finfo(FP32).min
    ops = _ops()
    for b in (None, 0.1 * torch.randn(64, generator=g)):
        for kw in (dict(), dict(n_group=8, topk_group=4, group_top=2)):
            idx, w = ops.moe_route(odd.cuda(), 6, bias=None if b is None else b.cuda(), scoring=scoring, **kw)
            ei, ew = o.route(odd, 6, b, scoring=scoring, **kw)
            assert torch.equal(idx.cpu(), ei)
            assert torch.allclose(w.cpu().double(), ew, rtol=1e-5, atol=1e-30)


def test_route_refusals_and_bounds():
    ops = _ops()
    logits = torch.randn(5, 64, device="cuda")
    for kw, err in [(dict(topk=0), ValueError), (dict(topk=65), ValueError), (dict(topk=4, scoring="relu"), ValueError),
                    (dict(topk=4, n_group=7), ValueError), (dict(topk=4, bias=torch.zeros(63, device="cuda")), ValueError),
                    (dict(topk=4, bias=torch.zeros(64, device="cuda", dtype=BF16)), ValueError)]:
        with pytest.raises(err):
            ops.moe_route(logits, **kw)
    with pytest.raises(TypeError):
        ops.moe_route(logits.half(), 4)
    with pytest.raises(ValueError):
        ops.moe_route(logits.t(), 4)
    assert ops.moe_route(logits[:0], 4)[0].shape == (0, 4)
    flat = torch.randn(1 + 6 * 64, device="cuda")
    a, b = ops.moe_route(flat[1:].view(6, 64), 5), ops.moe_route(flat[1:].view(6, 64).clone(), 5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def _ffn(g, hidden, inter):
    from pypto_b200.layers import Fp8SwiGLUFFN
    ws = [0.05 * _randn(g, *s) for s in ((hidden, inter), (hidden, inter), (inter, hidden))]
    return Fp8SwiGLUFFN.from_float(*ws, 1 + 0.1 * _randn(g, hidden), 1e-6), ws


@pytest.mark.parametrize("rows, hidden, inter", [(1, 512, 768), (33, 512, 640), (300, 384, 1008)])
def test_ffn_block(rows, hidden, inter):
    """The four launches of the FP8 feed-forward block: exactly its operators one after the other, and near the block in
    64 bits with unquantised weights."""
    ops = _ops()
    g = _gen(rows)
    ffn, (wg, wu, wd) = _ffn(g, hidden, inter)
    x, res = _randn(g, rows, hidden).to(BF16), _randn(g, rows, hidden)
    before, want = res.clone(), res.clone()
    q, s = ops.add_rms_norm_quantize(x, want, ffn.gamma, ffn.eps)
    q, s = ops.swiglu_quantize(ops.linear_fp8(q, s, ffn.w_gu, ffn.s_gu))
    want = ops.linear_fp8(q, s, ffn.w_d, ffn.s_d, acc=want, out_dtype=FP32)
    got = ffn(x, res)
    assert got is res and torch.equal(got, want)
    h, y = o.add_rms_norm(x, before, ffn.gamma, 1e-6)
    act = o.swiglu(torch.cat([y @ wg.double(), y @ wu.double()], 1))
    full = act @ wd.double()
    # four roundings to e4m3 (norm, weights, activation, weights), each 2^-4 / sqrt(3) of a value in the mean square at
    # the most, of independent signs in a product's terms: a twentieth each
    assert ((got.double() - h - full).norm() / full.norm()) < 4 * 0.05
    two = ffn(None, h.float())                                          # the sum already in the residual
    assert ((two.double() - h - full).norm() / full.norm()) < 4 * 0.05


def test_ffn_block_captured_and_replayed_beside_another():
    """Two graphs of the block and of a routing, replayed on two streams at once with changed inputs, give what eager
    calls give."""
    ops = _ops()
    g = _gen(1)
    ffn, _ = _ffn(g, 512, 768)
    logits_w = 0.05 * _randn(g, 512, 64)
    gate = ops.pack_weight(logits_w)
    bias = 0.1 * _randn(g, 64)

    def step(x, res):
        y = ffn(x, res)
        n = ops.add_rms_norm(y, None, ffn.gamma, 1e-6)
        return y, *ops.moe_route(ops.linear(n, gate), 8, bias=bias, n_group=8, topk_group=4)

    runs = []
    for rows in (3, 150):
        x, res = torch.zeros(rows, 512, dtype=BF16, device="cuda"), torch.zeros(rows, 512, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(x, res.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(x, res)
        runs.append((graph, side, x, res, out))
    for trial in range(3):
        wants = []
        for graph, side, x, res, out in runs:
            x.copy_(_randn(g, *x.shape))
            res.copy_(_randn(g, *res.shape))
            wants.append([t.clone() for t in step(x, res.clone())])
        torch.cuda.synchronize()
        for graph, side, *_ in runs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, side, x, res, out), want in zip(runs, wants):
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    ops.check_device_status()


def test_calls_on_two_streams_at_once():
    ops = _ops()
    g = _gen(2)
    jobs = []
    for m, n, k in ((4, 2048, 2048), (64, 1024, 4096), (1200, 2304, 512)):
        x, xs = _fp8_rows(_randn(g, m, k))
        jobs.append((x, xs, *_fp8_weight(g, n, k)))
    want = [ops.linear_fp8(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[] for _ in streams]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                for j in jobs:
                    got[i].append(ops.linear_fp8(*j))
    torch.cuda.synchronize()
    for i in range(3):
        for r, t in enumerate(got[i]):
            assert torch.equal(t, want[r % len(jobs)])


def _moe_weights(g, experts, hidden, inter):
    from pypto_b200 import ops
    def q(*shape):
        return (0.3 * _randn(g, *shape)).to(ops.FP8)
    def s(*shape):
        return 0.02 + 0.02 * torch.rand(*shape, generator=g, device="cuda")
    return dict(w_gu=q(experts, 2 * inter, hidden), s_gu=s(experts, 2 * inter // 128, hidden // 128),
                w_d=q(experts, hidden, inter), s_d=s(experts, hidden // 128, inter // 128))


def test_moe_layer_with_a_router():
    """The layer with grouped softmax routing gives what it gives when handed that routing, and a layer without a router
    routes as before."""
    from pypto_b200.moe import MoELayer, Router
    ops = _ops()
    g = _gen(8)
    experts, hidden, inter, tokens = 32, 256, 128, 70
    gate = (0.1 * _randn(g, experts, hidden)).to(BF16)
    bias = 0.1 * _randn(g, experts)
    w = _moe_weights(g, experts, hidden, inter)
    x = _randn(g, tokens, hidden).to(BF16)
    router = Router(scoring="softmax", n_group=8, topk_group=3, group_top=1, renormalize=False, route_scale=4.0)
    layer = MoELayer.from_packed(gate, bias, w, None, topk=6, router=router)
    y, idx, weights = layer.forward(x)
    ei, ew = ops.moe_route(ops.linear(x, gate), 6, bias=bias, scoring="softmax", n_group=8, topk_group=3, group_top=1,
                           renormalize=False, route_scale=4.0)
    ri, rw = layer.route(x)
    assert torch.equal(idx, ei) and torch.equal(weights, ew) and torch.equal(ri, ei) and torch.equal(rw, ew)
    assert layer.status()[0] == 0
    plain = MoELayer.from_packed(gate, bias, w, None, topk=6)
    y2, _, _ = plain.forward(x, routing=(ei, ew))
    assert torch.equal(y, y2)
    _, pi, pw = plain.forward(x)
    ti, tw = ops.moe_topk(ops.linear(x, gate), bias, 6, is_logits=True)
    assert torch.equal(pi, ti) and torch.equal(pw, tw)
    more = _randn(g, 3 * tokens, hidden).to(BF16)           # a larger call builds the layer object anew, router and all
    assert torch.equal(layer.forward(more)[1], layer.route(more)[0])
    layer.close()
    plain.close()


def test_registered_callables():
    """The operators as callables of a worker, in the tensors-then-scalars order of a compiled program."""
    import struct

    from pypto_b200 import _lib
    import ctypes as C
    ops = _ops()
    lib = _lib.load()
    g = _gen(6)
    handle = C.c_void_p()
    _lib.check(lib.pto_worker_create(0, C.byref(handle)))

    def run(name, tensors, scalars=()):
        cid = C.c_int32()
        _lib.check(lib.pto_register_callable(handle, name.encode(), C.byref(cid)))
        ts = (_lib.ChipTensor * len(tensors))()
        for d, t in zip(ts, tensors):
            d.addr, d.ndims, d.dtype = t.data_ptr(), t.dim(), ops.dtype_code(t.dtype)
            for i, n in enumerate(t.shape):
                d.shapes[i] = n
        sc = (C.c_uint64 * max(len(scalars), 1))(*scalars)
        args = _lib.TaskArgs(ts, len(tensors), sc, len(scalars))
        torch.cuda.synchronize()
        st = lib.pto_run(handle, cid, C.byref(args))
        _lib.check(lib.pto_synchronize(handle))
        _lib.check(lib.pto_unregister_callable(handle, cid))
        return st

    def bits(f):
        return struct.unpack("<I", struct.pack("<f", f))[0]

    x, res, gamma = _randn(g, 9, 384).to(BF16), _randn(g, 9, 384), _randn(g, 384)
    want_res = res.clone()
    wq, wsc = ops.add_rms_norm_quantize(x, want_res, gamma, 1e-6)
    mine = res.clone()
    q, s = torch.empty_like(wq), torch.empty_like(wsc)
    assert run("add_rms_norm", [x, mine, gamma, q, s], [bits(1e-6)]) == 0
    assert torch.equal(mine, want_res) and torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, wsc)
    out, again = torch.empty_like(x), res.clone()
    assert run("add_rms_norm", [x, again, gamma, out], [bits(1e-6)]) == 0
    assert torch.equal(out, ops.add_rms_norm(x, res.clone(), gamma, 1e-6))
    w, ws = _fp8_weight(g, 512, 384)
    y = torch.empty(9, 512, dtype=BF16, device="cuda")
    assert run("linear_fp8", [wq, wsc, w, ws, y]) == 0
    assert torch.equal(y, ops.linear_fp8(wq, wsc, w, ws))
    acc = _randn(g, 9, 512)
    y32 = torch.empty(9, 512, device="cuda")
    assert run("linear_fp8", [wq, wsc, w, ws, y32, acc]) == 0
    assert torch.equal(y32, ops.linear_fp8(wq, wsc, w, ws, acc=acc, out_dtype=FP32))
    q, s = torch.empty(9, 256, dtype=ops.FP8, device="cuda"), torch.empty(9, 2, device="cuda")
    assert run("swiglu_quantize", [y, q, s]) == 0
    eq, es = ops.swiglu_quantize(y)
    assert torch.equal(q.view(torch.uint8), eq.view(torch.uint8)) and torch.equal(s, es)
    logits, bias = _randn(g, 9, 64), _randn(g, 64)
    idx, wt = torch.empty(9, 6, dtype=torch.int32, device="cuda"), torch.empty(9, 6, device="cuda")
    assert run("moe_route", [logits, bias, idx, wt], [1, 8, 4, 2, 1, bits(2.0)]) == 0
    ei, ew = ops.moe_route(logits, 6, bias=bias, scoring="softmax", n_group=8, topk_group=4, route_scale=2.0)
    assert torch.equal(idx, ei) and torch.equal(wt, ew)
    assert run("moe_route", [logits, bias, idx, wt], [7, 8, 4, 2, 1, bits(2.0)]) == 1
    assert run("linear_fp8", [wq, wsc, w, ws[:1], y]) == 1
    assert run("add_rms_norm", [x, res, gamma], [bits(1e-6)]) == 1
    assert run("swiglu_quantize", [y, q]) == 1
    _lib.check(lib.pto_worker_destroy(handle))
