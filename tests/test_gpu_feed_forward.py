"""Root-mean-square norm, rows in 8 bits, 8-bit products and the gated linear map on the GPU, against their formulas in 64 bits.

Tolerances follow from the roundings.  u is what one rounding of the type may bring, relative to the value: 2^-8 for bf16, 2^-24
for f32.  A sum of n terms in f32 is off by at most n 2^-24 of the sum of the terms' magnitudes; sums that run over lanes and
parts count the longest chain of additions.  f32 products are six products of bf16 terms, so six times as many additions, and
2^-24 of each product's magnitude for the terms that are left out.  Codes in 8 bits are whole numbers and have to be the
formula's."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
F = 2.0 ** -24
UNIT = {torch.float32: F, torch.bfloat16: 2.0 ** -8}
ACTIVATIONS = ("silu", "gelu", "sigmoid", "relu")


@pytest.fixture(scope="module")
def ops():
    from pccnn_lib_amd import pccnn_lib_ops
    return pccnn_lib_ops


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float32)


def _within(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    excess = (got - want).abs() - bound
    assert float(excess.max() if excess.numel() else -1.0) <= 0.0, "%s: off by %g where %g is allowed" % (
        what, float((got - want).abs().flatten()[excess.argmax()]), float(bound.expand_as(want).flatten()[excess.argmax()]))


# --------------------------------------------------------------------------------------------- root-mean-square norm

def _chain(channels):
    """Additions behind one another in a row's sum: a lane's values and the lanes', or a thread's share of a long row."""
    return max(40, channels // 256 + 10)


def _norm_exact(s, gamma, eps, grads, total_grads):
    s, gamma, g = s.double(), gamma.double(), grads.double()
    rstd = 1.0 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    xhat, scaled = s * rstd, g * gamma
    dx = rstd * (scaled - xhat * (scaled * xhat).mean(1, keepdim=True))
    if total_grads is not None:
        dx = dx + total_grads.double()
    return xhat * gamma, dx, (g * xhat).sum(0), xhat, rstd


def _check_norm(ops, x, r, gamma, g, t, eps=1e-6):
    """x, r, g, t on the GPU (r and t may be None); against the formula of the same values."""
    dtype, weights, (rows, channels) = x.dtype, gamma.dtype, x.shape
    got = ops.rms_norm(x, gamma, r, eps, return_stats=True)
    out, rstd, total = got[0], got[-1], got[1] if r is not None else x
    assert len(got) == (3 if r is not None else 2) and out.dtype == dtype and rstd.dtype == torch.float32
    if r is not None:
        assert torch.equal(total, (x.float() + r.float()).to(dtype))
    d_feats, d_gamma = ops.rms_norm_grads(total, gamma, rstd, g, t)
    assert d_feats.dtype == dtype and d_gamma.dtype == weights
    w = gamma.cpu()
    y, dx, dg, xhat, exact_rstd = _norm_exact(total.cpu(), w, eps, g.cpu(), None if t is None else t.cpu())
    u, f = UNIT[dtype], F * (_chain(channels) / 2 + 8)
    _within(rstd, exact_rstd.squeeze(1), f * exact_rstd.squeeze(1), "rstd")
    _within(out, y, (u + f) * y.abs(), "out")
    scaled = (g.cpu().double() * w.double()).abs()
    size = exact_rstd * (scaled + xhat.abs() * (scaled * xhat.abs()).mean(1, keepdim=True))
    flow = 0.0 if t is None else t.cpu().double().abs()
    _within(d_feats, dx, u * dx.abs() + 4 * f * size + 2 * F * flow, "dx")
    # (a column's chain: a workgroup's rows behind one another, its wavefronts, the workgroups)
    _within(d_gamma, dg, UNIT[weights] * dg.abs() + F * (rows / 64 + 200 + _chain(channels)) * (g.cpu().double() * xhat).abs().sum(0),
            "dgamma")
    return out, total, rstd, d_feats, d_gamma


SHAPES = [(1, 1), (1, 64), (3, 7), (7, 33), (65, 64), (130, 96), (257, 130), (64, 512), (33, 986), (9, 1025), (17, 2048), (5, 2056),
          (3, 5001), (2, 8192), (2, 9001), (4099, 24), (0, 16)]


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels", SHAPES)
def test_norm_against_the_formula(ops, type, rows, channels):
    dtype, gen = TYPES[type], _gen(rows * 7 + channels)
    x, r, g, t = ((_normal(gen, rows, channels) * k).to(dtype).to(DEV) for k in (1.5, 0.7, 1.0, 1.0))
    gamma = 1.0 + 0.3 * _normal(gen, channels)
    for weights in {torch.float32, dtype}:
        w = gamma.to(weights).to(DEV)
        _check_norm(ops, x, None, w, g, None)
        _check_norm(ops, x, r, w, g, t)
        _check_norm(ops, x, r, w, g, None)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [96, 250, 1000, 2048])
def test_norm_of_views_by_every_load_width(ops, type, channels):
    dtype, gen = TYPES[type], _gen(channels)
    x, r, g, t = (_normal(gen, 33, channels + 8).to(dtype).to(DEV) for _ in range(4))
    gamma = (1.0 + 0.3 * _normal(gen, channels)).to(DEV)
    for lo in (0, 2, 3):
        _check_norm(ops, *(v[:, lo:lo + channels] for v in (x, r)), gamma, *(v[:, lo:lo + channels] for v in (g, t)))
    _check_norm(ops, x[::2, :channels], r[1::2, 1:1 + channels][:16].repeat(2, 1)[:17], gamma, g[:17, :channels], t[:17, 2:2 + channels])


def test_norm_parts_of_the_gradients_and_their_bits(ops):
    gen = _gen(4)
    for rows, channels in ((1, 8), (5000, 40), (700, 1100), (40, 9000)):
        x, g = (_normal(gen, rows, channels).to(DEV) for _ in range(2))
        gamma = (1.0 + 0.1 * _normal(gen, channels)).to(DEV)
        _, rstd = ops.rms_norm(x, gamma, return_stats=True)
        d_feats, d_gamma = ops.rms_norm_grads(x, gamma, rstd, g)
        only, nothing = ops.rms_norm_grads(x, gamma, rstd, g, grad_mask=ops.GRAD_FEATS)
        assert nothing is None and torch.equal(only, d_feats)
        nothing, only = ops.rms_norm_grads(x, gamma, rstd, g, grad_mask=ops.GRAD_WEIGHTS)
        assert nothing is None and torch.equal(only, d_gamma)


def test_norm_of_huge_tiny_and_empty_rows(ops):
    gen = _gen(9)
    for channels in (24, 700, 9100):
        x = _normal(gen, 6, channels)
        x[1] *= 1.0e30                                    # squares past the largest f32 value
        x[2] *= 1.0e-30                                   # squares below the smallest: eps decides
        x[3] = 0.0
        x[4, 1] = float("inf")
        x[5, 2] = float("nan")
        gamma = (1.0 + 0.2 * _normal(gen, channels)).to(DEV)
        out, rstd = ops.rms_norm(x.to(DEV), gamma, return_stats=True)
        y = _norm_exact(x, gamma.cpu(), 1e-6, torch.ones_like(x), None)[0]
        f = F * (_chain(channels) / 2 + 16)
        _within(out[:4], y[:4], f * y[:4].abs() + 1e-45, "out")
        want = x[4] * 0.0                                 # 1 / sqrt(inf)
        assert torch.equal(out[4].cpu().isnan(), want.isnan()) and float(out[4].cpu().nan_to_num().abs().max()) == 0.0
        assert bool(out[5].isnan().all())
        codes, scales = ops.rms_norm_8bit(x.to(DEV), gamma)
        assert bool(scales[4:].isnan().all()) and not bool(codes[3:].any())
        assert float(scales[3]) == 0.0 and bool(torch.isfinite(scales[:4]).all())
        assert torch.equal(codes[:3].cpu(), _codes(x[:3], gamma.cpu()))


# --------------------------------------------------------------------------------------------------- rows in 8 bits

def _codes(s, gamma=None):
    t = s.double() if gamma is None else s.double() * gamma.double()
    top = t.abs().amax(1, keepdim=True)
    return torch.round(t * 127.0 / torch.where(top > 0, top, torch.ones_like(top))).to(torch.int8)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels", SHAPES)
def test_rows_in_8_bits_are_the_nearest(ops, type, rows, channels):
    dtype, gen = TYPES[type], _gen(rows * 5 + channels)
    x, r = ((_normal(gen, rows, channels) * k).to(dtype) for k in (1.5, 0.7))
    gamma = 1.0 + 0.3 * _normal(gen, channels)
    codes, scales = ops.quantize_rows(x.to(DEV))
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32
    assert torch.equal(codes.cpu(), _codes(x))
    _within(scales, x.double().abs().amax(1) / 127.0, F * x.double().abs().amax(1) / 127.0, "scales")
    for weights in {torch.float32, dtype}:
        w = gamma.to(weights)
        for residual in (None, r):
            got = ops.rms_norm_8bit(x.to(DEV), w.to(DEV), None if residual is None else residual.to(DEV))
            s = x if residual is None else (x.float() + r.float()).to(dtype)
            if residual is not None:
                assert torch.equal(got[2].cpu(), s)
            assert len(got) == (2 if residual is None else 3) and torch.equal(got[0].cpu(), _codes(s, w))
            y = _norm_exact(s, w, 1e-6, torch.zeros_like(s), None)[0]
            want = y.abs().amax(1) / 127.0
            _within(got[1], want, F * (_chain(channels) / 2 + 9) * want, "scales")


def test_ties_between_two_codes_go_to_the_even_one(ops):
    # 127 t / a is half way between two integers where t = a (2 k + 1) / 254: half of the largest value is 63.5 -> 64, a tie for
    # any a; with a = 127 every half is one
    for dtype in TYPES.values():
        x = torch.zeros(3, 64)
        x[0, 0], x[0, 1], x[0, 2] = 3.140625, 1.5703125, -1.5703125
        x[1, :] = (torch.arange(64) - 32).float() + 0.5
        x[1, 0] = 127.0
        x[2, 0], x[2, 1] = -1.0e-30, 0.5e-30
        x = x.to(dtype)
        codes, _ = ops.quantize_rows(x.to(DEV))
        codes = codes.cpu()
        assert codes[0, :3].tolist() == [127, 64, -64] and codes[2, :2].tolist() == [-127, 64]
        assert codes[1, 1:].tolist() == torch.round(x[1, 1:].double()).to(torch.int8).tolist()
        scaled, _ = ops.rms_norm_8bit(x.to(DEV), torch.full((64,), 0.75, device=DEV))
        assert torch.equal(scaled.cpu(), codes)


# ---------------------------------------------------------------------------------------------------- 8-bit products

PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 1408, 512), (3, 17, 33), (16, 64, 20), (17, 100, 50), (33, 96, 70), (64, 130, 65), (65, 64, 64),
            (65, 48, 129), (128, 128, 128), (129, 127, 127), (257, 300, 40), (500, 16, 1000), (1000, 1111, 30), (0, 16, 16)]


def _random_codes(gen, rows, inner):
    return torch.randint(-128, 128, (rows, inner), generator=gen).to(torch.int8), torch.rand(rows, generator=gen) + 0.01


@pytest.mark.parametrize("rows,inner,outer", PRODUCTS)
def test_8bit_product_against_exact_sums(ops, rows, inner, outer):
    gen = _gen(rows + inner * 3 + outer)
    x, sx = _random_codes(gen, rows, inner)
    w, sw = _random_codes(gen, outer, inner)
    bias = _normal(gen, outer)
    value = (x.double() @ w.double().t()) * sx.double().unsqueeze(1) * sw.double()
    args = [v.to(DEV) for v in (x, sx, w, sw)]
    for dtype, u in UNIT.items():
        # sum, product of the scales, their product, the bias and the result are rounded once each
        _within(ops.linear_8bit(*args, dtype=dtype), value, (u + 4 * F) * value.abs(), "product")
        want = value + bias.double()
        _within(ops.linear_8bit(*args, bias.to(DEV), dtype), want, u * want.abs() + 4 * F * (value.abs() + want.abs()), "with bias")


def test_8bit_product_of_the_longest_sums(ops):
    # 131071 products of -128 and -128 are the largest sum that 32 bits hold; one product more is refused
    for rows in (1, 70):
        x = torch.full((rows, 131071), -128, dtype=torch.int8, device=DEV)
        w = torch.full((20, 131071), -128, dtype=torch.int8, device=DEV)
        ones = torch.ones(rows, device=DEV), torch.ones(20, device=DEV)
        out = ops.linear_8bit(x, ones[0], w, ones[1], dtype=torch.float32)
        assert bool((out == float(131071 * 16384)).all())
    big = torch.zeros((1, 131072), dtype=torch.int8, device=DEV)
    with pytest.raises(RuntimeError, match="131072 products"):
        ops.linear_8bit(big, ones[0][:1], big, ones[1][:1])


def test_8bit_product_of_codes_that_start_anywhere(ops):
    gen = _gen(3)
    for rows, inner, outer in ((5, 64, 48), (300, 64, 48), (300, 100, 200)):
        store = torch.zeros(rows * inner + 7, dtype=torch.int8, device=DEV)
        x, sx = _random_codes(gen, rows, inner)
        w, sw = (v.to(DEV) for v in _random_codes(gen, outer, inner))
        moved = store[7:].view(rows, inner)
        moved.copy_(x)
        want = ops.linear_8bit(x.to(DEV), sx.to(DEV), w, sw, dtype=torch.float32)
        assert torch.equal(ops.linear_8bit(moved, sx.to(DEV), w, sw, dtype=torch.float32), want)


# -------------------------------------------------------------------------------------------------- gated linear map

def _act(g, name):
    """Activation, slope, and the largest slope and curvature there are."""
    if name == "relu":
        live = (g > 0).double()
        return g * live, live, 1.0, 0.0
    if name == "gelu":
        phi = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi), 1.13, 0.8
    s = torch.sigmoid(g)
    if name == "sigmoid":
        return s, s * (1 - s), 0.25, 0.1
    return g * s, s * (1 + g * (1 - s)), 1.1, 0.5


def _gated_exact(x, gate, up, name, g=None):
    """Results in 64 bits, and from the roundings a bound on what each may be off."""
    dtype = x.dtype
    x, gate, up = x.double(), gate.double(), up.double()
    f32 = dtype == torch.float32
    u = UNIT[dtype]
    sums = lambda n: F * (6 * n + 1 if f32 else n + 1)                     # noqa: E731  of the terms' magnitudes
    G, U = x @ gate.t(), x @ up.t()
    eg, eu = (sums(x.shape[1]) * (x.abs() @ w.abs().t()) for w in (gate, up))
    act, slope, most, bend = _act(G, name)
    # exponentials and reciprocals: 2^-20 of the value; the normal distribution of bf16 results: 2e-7
    ea = most * eg + 2.0 ** -20 * act.abs() + 2e-7 * G.abs()
    es = bend * eg + 2.0 ** -20 * slope.abs() + 1e-6 * (1 + G.abs())
    if name == "relu":
        es = torch.where(G.abs() <= eg, torch.ones_like(es), torch.zeros_like(es))       # either side of the kink
    h = act * U
    eh = act.abs() * eu + ea * (U.abs() + eu)
    results = [(h, u * h.abs() + (1 + u) * eh + F * h.abs())]
    if g is None:
        return results
    g = g.double()
    dG, dU = g * U * slope, g * act
    edG = g.abs() * (slope.abs() * eu + es * (U.abs() + eu)) + 3 * F * dG.abs()
    edU = g.abs() * ea + 2 * F * dU.abs()
    kept = 2.0 ** -24 if f32 else 2.0 ** -8                                # the gradients of the projections as operands
    edG, edU = edG + kept * (dG.abs() + edG), edU + kept * (dU.abs() + edU)
    size = lambda a, b: a.abs() @ b.abs()                                  # noqa: E731
    dx = dG @ gate + dU @ up
    edx = edG @ gate.abs() + edU @ up.abs() + sums(2 * gate.shape[0]) * (size(dG, gate) + size(dU, up))
    results.append((dx, u * dx.abs() + (1 + u) * edx))
    for d, e in ((dG, edG), (dU, edU)):
        dw = d.t() @ x
        edw = e.t() @ x.abs() + sums(x.shape[0]) * size(d.t(), x)
        results.append((dw, u * dw.abs() + (1 + u) * edw))
    return results


def _check_gated(ops, x, gate, up, name, g=None):
    want = _gated_exact(x.cpu(), gate.cpu(), up.cpu(), name, None if g is None else g.cpu())
    got = [ops.gated_linear(x, gate, up, name)]
    if g is not None:
        got += list(ops.gated_linear_grads(x, gate, up, g, name))
    for a, (b, bound), what in zip(got, want, ("h", "dx", "dgate", "dup")):
        assert a.dtype == x.dtype
        _within(a, b, bound, "%s %s" % (name, what))
    return got


GATED = [(1, 1, 1), (1, 64, 128), (5, 24, 40), (17, 33, 7), (64, 96, 64), (65, 64, 64), (65, 32, 24), (129, 100, 65), (200, 128, 130),
         (300, 72, 200), (128, 512, 96), (1000, 20, 48), (70, 1000, 24), (2500, 8, 16)]


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels,hidden", GATED)
def test_gated_against_the_formula(ops, type, rows, channels, hidden):
    dtype, gen = TYPES[type], _gen(rows + 3 * channels + hidden)
    x, g = _normal(gen, rows, channels).to(dtype).to(DEV), _normal(gen, rows, hidden).to(dtype).to(DEV)
    gate, up = ((_normal(gen, hidden, channels) * (k / math.sqrt(channels))).to(dtype).to(DEV) for k in (1.5, 1.0))
    for name in ACTIVATIONS:
        _check_gated(ops, x, gate, up, name, g)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [9, 150])
def test_gated_of_views_that_start_anywhere(ops, type, rows):
    dtype, gen = TYPES[type], _gen(rows)
    x, g = _normal(gen, rows, 120).to(dtype).to(DEV), _normal(gen, rows, 120).to(dtype).to(DEV)
    fused = (_normal(gen, 130, 120) / 8).to(dtype).to(DEV)
    for lo, channels, hidden in ((0, 64, 64), (8, 64, 40), (4, 60, 36), (3, 61, 65)):
        gate, up = fused[:hidden, lo:lo + channels], fused[hidden:2 * hidden, lo:lo + channels]
        _check_gated(ops, x[:, lo:lo + channels], gate, up, "silu", g[:, lo:lo + hidden])
        _check_gated(ops, x[:, :channels], gate, up.contiguous(), "gelu", g[:, :hidden])
    _check_gated(ops, x[:1, :64].expand(rows, 64), fused[:40, :64], fused[40:80, :64], "silu", g[:, :40])


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_gated_f32_keeps_f32_accuracy(ops, rows):
    # 2^-24 and less is left out of each product; a product short of one of its six terms would be off by 2^-18
    gen = _gen(rows)
    x, gate, up, g = (_normal(gen, *s).to(DEV) for s in ((rows, 96), (80, 96), (80, 96), (rows, 80)))
    gate, up = gate / 10, up / 10
    want = _gated_exact(x.cpu(), gate.cpu(), up.cpu(), "silu", g.cpu())
    got = [ops.gated_linear(x, gate, up)] + list(ops.gated_linear_grads(x, gate, up, g))
    for a, (b, _) in zip(got, want):
        assert float((a.cpu().double() - b).norm() / b.norm()) < 2.0 ** -20


def test_gated_f32_of_values_near_the_largest(ops):
    # finite features and weights within 2^-9 of the largest f32 value keep their value (their bf16 part would round to infinity)
    for rows in (3, 90):
        x = torch.zeros(rows, 16, device=DEV)
        x[0, 0] = torch.finfo(torch.float32).max
        gate, up = torch.zeros(24, 16, device=DEV), torch.zeros(24, 16, device=DEV)
        gate[0, 0], up[0, 0] = 1.0, 2.0 ** -127          # the square of the value times 2^-127 is 2^129: infinity, as it must be
        assert float(ops.gated_linear(x, gate, up, "relu")[0, 0]) == float("inf")
        gate[0, 0], up[0, 0] = 2.0 ** -65, 2.0 ** -65
        out = ops.gated_linear(x, gate, up, "relu")
        want = (float(x[0, 0]) * 2.0 ** -65) ** 2
        assert abs(float(out[0, 0]) / want - 1) < 2.0 ** -20 and not bool(out[1:].any()) and not bool(out[:, 1:].any())


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_gated_parts_of_the_gradients_and_their_bits(ops, type):
    gen = _gen(12)
    for rows, channels, hidden in ((40, 24, 20), (3000, 72, 90)):
        x, gate, up, g = (_normal(gen, *s).to(TYPES[type]).to(DEV) for s in ((rows, channels), (hidden, channels), (hidden, channels),
                                                                           (rows, hidden)))
        whole = ops.gated_linear_grads(x, gate, up, g)
        again = ops.gated_linear_grads(x, gate, up, g)
        assert all(torch.equal(a, b) for a, b in zip(whole, again))
        feats, no_gate, no_up = ops.gated_linear_grads(x, gate, up, g, grad_mask=ops.GRAD_FEATS)
        assert no_gate is None and no_up is None and torch.equal(feats, whole[0])
        no_feats, d_gate, d_up = ops.gated_linear_grads(x, gate, up, g, grad_mask=ops.GRAD_WEIGHTS)
        assert no_feats is None and torch.equal(d_gate, whole[1]) and torch.equal(d_up, whole[2])


def test_gated_of_no_rows(ops):
    for dtype in TYPES.values():
        x, w, g = (torch.ones(s, dtype=dtype, device=DEV) for s in ((0, 24), (40, 24), (0, 40)))
        assert ops.gated_linear(x, w, w).shape == (0, 40)
        d_feats, d_gate, d_up = ops.gated_linear_grads(x, w, w, g)
        assert d_feats.shape == (0, 24) and not bool(d_gate.any()) and not bool(d_up.any()) and d_up.shape == (40, 24)


@pytest.mark.parametrize("rows,channels,hidden", GATED)
def test_gated_8bit_against_exact_sums(ops, rows, channels, hidden):
    gen = _gen(rows * 3 + channels + hidden)
    (x, sx), (gate, sg), (up, su) = (_random_codes(gen, n, channels) for n in (rows, hidden, hidden))
    sx, sg = sx / 64, sg / math.sqrt(channels) / 64
    G, U = ((x.double() @ w.double().t()) * sx.double().unsqueeze(1) * s.double() for w, s in ((gate, sg), (up, su)))
    args = [v.to(DEV) for v in (x, sx, gate, sg, up, su)]
    for name in ACTIVATIONS:
        act, _, most, _ = _act(G, name)
        h = act * U
        error = 4 * F * h.abs() + (most * 4 * F * G.abs() + 2.0 ** -20 * act.abs() + 2e-7 * G.abs()) * U.abs()
        for dtype, u in UNIT.items():
            _within(ops.gated_linear_8bit(*args, name, dtype), h, u * h.abs() + (1 + u) * error, name)
