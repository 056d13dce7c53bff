"""Layer norm, rotary positions and attention between levels on the GPU, against their formulas in 64 bits.

Tolerances follow from the roundings.  u is the relative error that one rounding of the type may bring: 2^-8 for bf16
(nearest even, 8 significant bits: half of a spacing of 2^-7), and for f32, whose sums run over at most a few thousand terms of 2^-24 each, 2^-16 of the
sum of the terms' magnitudes.  A bf16 attention rounds the probabilities, the score gradients and the results: the bound of
every element is formed in 64 bits from exactly these roundings (``_attention_exact``).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -16, torch.bfloat16: 2.0 ** -8}


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


# ------------------------------------------------------------------------------------------------------- layer norm

def _norm_exact(x, gamma, beta, eps, grads):
    x, gamma, beta, g = x.double(), gamma.double(), beta.double(), grads.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xhat = (x - mean) * rstd
    s = g * gamma
    dx = rstd * (s - s.mean(1, keepdim=True) - xhat * (s * xhat).mean(1, keepdim=True))
    return xhat * gamma + beta, dx, (g * xhat).sum(0), g.sum(0), xhat, rstd


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels", [(1, 1), (1, 64), (3, 7), (7, 33), (65, 64), (130, 96), (257, 130), (64, 512),
                                           (33, 986), (9, 1025), (17, 2048), (5, 2056), (3, 5001), (4099, 24), (0, 16)])
def test_norm_against_the_formula(ops, type, rows, channels):
    dtype = TYPES[type]
    gen = _gen(rows * 7 + channels)
    x = (_normal(gen, rows, channels) * 1.5 + 0.7).to(dtype)
    gamma, beta, g = 1.0 + 0.3 * _normal(gen, channels), 0.2 * _normal(gen, channels), _normal(gen, rows, channels).to(dtype)
    for weights in {torch.float32, dtype}:
        w, b = gamma.to(weights), beta.to(weights)
        out, stats = ops.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), 1e-5, return_stats=True)
        d_feats, d_gamma, d_beta = ops.layer_norm_grads(x.to(DEV), w.to(DEV), stats, g.to(DEV))
        assert out.dtype == dtype and d_feats.dtype == dtype and d_gamma.dtype == weights and d_beta.dtype == weights
        y, dx, dg, db, xhat, rstd = _norm_exact(x, w, b, 1e-5, g)
        u, uw, f = UNIT[dtype], UNIT[weights], UNIT[torch.float32]
        s = (g.double() * w.double()).abs()
        size = 1.0 + x.double().abs().amax(1, keepdim=True) * rstd if rows else 1.0        # of the terms of xhat
        _within(out, y, u * y.abs() + f * ((xhat * w.double()).abs() + b.double().abs() + size * w.double().abs()), "out")
        _within(d_feats, dx, u * dx.abs() + f * rstd * size * (s + s.mean(1, keepdim=True)
                                                               + (xhat.abs() * (s * xhat.abs()).mean(1, keepdim=True))), "dx")
        _within(d_gamma, dg, uw * dg.abs() + f * (g.double().abs() * (xhat.abs() + size)).sum(0), "dgamma")
        _within(d_beta, db, uw * db.abs() + f * g.double().abs().sum(0), "dbeta")


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels", [(128, 64), (129, 64), (256, 64), (257, 64), (32, 256), (33, 256), (64, 256), (65, 256),
                                           (16, 1024), (17, 1024), (8, 1021), (9, 1021)])
def test_norm_of_as_many_rows_as_one_workgroup_takes_and_one_more(ops, type, rows, channels):
    test_norm_against_the_formula(ops, type, rows, channels)
    gen = _gen(rows + channels)
    x, g = (_normal(gen, rows, channels).to(TYPES[type]).to(DEV) for _ in range(2))
    gamma, beta = torch.full((channels,), 1.25, device=DEV), torch.zeros(channels, device=DEV)
    _, stats = ops.layer_norm(x, gamma, beta, return_stats=True)
    d_feats, d_gamma, d_beta = ops.layer_norm_grads(x, gamma, stats, g)
    only, _, _ = ops.layer_norm_grads(x, gamma, stats, g, grad_mask=ops.GRAD_FEATS)
    _, dg, db = ops.layer_norm_grads(x, gamma, stats, g, grad_mask=ops.GRAD_WEIGHTS)
    assert torch.equal(only, d_feats) and torch.equal(dg, d_gamma) and torch.equal(db, d_beta)


def test_norm_of_a_views_rows_and_of_unaligned_rows(ops):
    gen = _gen(5)
    for type, dtype in TYPES.items():
        wide = (_normal(gen, 300, 200)).to(dtype).to(DEV)
        gamma, beta = torch.rand(96, generator=gen).to(DEV), torch.rand(96, generator=gen).to(DEV)
        g = _normal(gen, 300, 200).to(dtype).to(DEV)
        for lo in (0, 8, 3):                       # 16-byte rows, and rows that start anywhere
            x, dy = wide[:, lo:lo + 96], g[:, lo + 1:lo + 97]
            out, stats = ops.layer_norm(x, gamma, beta, return_stats=True)
            same, same_stats = ops.layer_norm(x.contiguous(), gamma, beta, return_stats=True)
            u = 4 * UNIT[dtype]
            assert torch.allclose(out.float(), same.float(), rtol=u, atol=u)
            got = ops.layer_norm_grads(x, gamma, stats, dy)
            want = ops.layer_norm_grads(x.contiguous(), gamma, same_stats, dy.contiguous())
            for a, b in zip(got, want):
                assert torch.allclose(a.float(), b.float(), rtol=u, atol=u * float(b.float().abs().max()))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [1000, 1024, 1026, 1536, 2048])
def test_norm_of_long_rows_by_every_load_width(ops, type, channels):
    # column slices: 16-byte loads, pairs of bf16 values, single values (which take the workgroup per row from 1025 on)
    dtype, gen = TYPES[type], _gen(channels)
    wide = [(_normal(gen, 33, channels + 8) * 1.5 + 0.7).to(dtype).to(DEV) for _ in range(2)]
    gamma, beta = 1.0 + 0.3 * _normal(gen, channels), 0.2 * _normal(gen, channels)
    for lo in (0, 2, 3):
        x, g = (t[:, lo:lo + channels] for t in wide)
        out, stats = ops.layer_norm(x, gamma.to(DEV), beta.to(DEV), 1e-5, return_stats=True)
        d_feats, d_gamma, d_beta = ops.layer_norm_grads(x, gamma.to(DEV), stats, g)
        y, dx, dg, db, xhat, rstd = _norm_exact(x.cpu(), gamma, beta, 1e-5, g.cpu())
        u, f, s = UNIT[dtype], UNIT[torch.float32], (g.cpu().double() * gamma.double()).abs()
        size = 1.0 + x.cpu().double().abs().amax(1, keepdim=True) * rstd
        _within(out, y, u * y.abs() + f * ((xhat * gamma.double()).abs() + beta.double().abs() + size * gamma.double().abs()), "out")
        _within(d_feats, dx, u * dx.abs() + f * rstd * size * (s + s.mean(1, keepdim=True)
                                                               + (xhat.abs() * (s * xhat.abs()).mean(1, keepdim=True))), "dx")
        _within(d_gamma, dg, f * dg.abs() + f * (g.cpu().double().abs() * (xhat.abs() + size)).sum(0), "dgamma")
        _within(d_beta, db, f * db.abs() + f * g.cpu().double().abs().sum(0), "dbeta")


def test_norm_statistics_survive_a_large_mean_and_constant_rows(ops):
    # the squares are taken of centred values: a mean of 10^4 leaves the variance of 1 intact
    gen = _gen(6)
    x = (_normal(gen, 64, 256) + 1.0e4)
    x[0] = 3.0
    ones, zeros = torch.ones(256, device=DEV), torch.zeros(256, device=DEV)
    out, stats = ops.layer_norm(x.to(DEV), ones, zeros, 1e-5, return_stats=True)
    want = _norm_exact(x, torch.ones(256), torch.zeros(256), 1e-5, x)
    # the mean is rounded to 2^-24 of 10^4 and its sum adds a few such errors
    assert float((out.cpu().double() - want[0])[1:].abs().max()) < 16 * 2.0 ** -24 * 1.0e4
    assert float(out[0].abs().max()) == 0.0 and bool(torch.isfinite(stats).all())


def test_norm_gradients_are_the_same_bits_on_every_run_and_match_differences(ops):
    gen = _gen(7)
    x, gamma, beta = _normal(gen, 5000, 96).to(DEV), _normal(gen, 96).to(DEV), _normal(gen, 96).to(DEV)
    g = _normal(gen, 5000, 96).to(DEV)
    out, stats = ops.layer_norm(x, gamma, beta, return_stats=True)
    first = ops.layer_norm_grads(x, gamma, stats, g)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.layer_norm_grads(x, gamma, stats, g)))
    only, none, none2 = ops.layer_norm_grads(x, gamma, stats, g, grad_mask=ops.GRAD_FEATS)
    assert torch.equal(only, first[0]) and none is None and none2 is None
    none, dg, db = ops.layer_norm_grads(x, gamma, stats, g, grad_mask=ops.GRAD_WEIGHTS)
    assert none is None and torch.equal(dg, first[1]) and torch.equal(db, first[2])
    loss = lambda x, w, b: float((ops.layer_norm(x, w, b).double() * g.double()).sum())
    h = 1e-2
    for i, base in enumerate((x, gamma, beta)):
        d = _normal(gen, *base.shape).to(DEV)
        args = [x, gamma, beta]
        up, down = list(args), list(args)
        up[i], down[i] = base + h * d, base - h * d
        slope = (loss(*up) - loss(*down)) / (2 * h)
        want = float((first[i].double() * d.double()).sum())
        # the third derivative's share is h^2 and the roundings' 2^-24 sqrt(count) / h
        assert abs(slope - want) < 5e-3 * float((first[i].double().norm() * d.double().norm())) / math.sqrt(96)


# ----------------------------------------------------------------------------------------------------------- rotary

def _rotary_exact(x, pts, freqs, axes, adjacent, sign=1.0):
    x, p = x.double().clone(), freqs.shape[0]
    angles = sign * pts.double()[:, axes.long()] * freqs.double()
    c, s = torch.cos(angles).unsqueeze(1), torch.sin(angles).unsqueeze(1)
    one, two = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if adjacent else (slice(0, p), slice(p, 2 * p))
    a, b = x[..., one].clone(), x[..., two].clone()
    x[..., one], x[..., two] = a * c - b * s, b * c + a * s
    return x


def _rotary_plan(gen, points, axes, pairs, reach=200.0):
    pts = torch.rand((points, axes), generator=gen) * reach - reach / 4
    of_axis = torch.tensor([p % axes for p in range(pairs)], dtype=torch.int32)
    freqs = torch.tensor([100.0 ** (-p / max(pairs, 1)) for p in range(pairs)], dtype=torch.float32)
    return pts, freqs, of_axis


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("points,heads,width,pairs,axes", [
    (1, 1, 2, 1, 1), (1, 8, 64, 32, 3), (77, 4, 32, 16, 3), (130, 3, 20, 10, 2), (65, 2, 33, 11, 3), (300, 1, 128, 64, 4),
    (51, 8, 48, 12, 6), (2049, 2, 24, 12, 3), (10, 1, 96, 0, 3), (0, 4, 32, 16, 3), (3, 1, 8192, 4096, 2)])
def test_rotary_against_the_formula(ops, type, adjacent, points, heads, width, pairs, axes):
    gen = _gen(points + width)
    x, g = _normal(gen, points, heads, width).to(TYPES[type]), _normal(gen, points, heads, width).to(TYPES[type])
    pts, freqs, of_axis = _rotary_plan(gen, points, axes, pairs)
    plan = [t.to(DEV) for t in (pts, freqs, of_axis)]
    out = ops.rotary(x.to(DEV), *plan, adjacent=adjacent)
    d_feats, d_pts = ops.rotary_grads(x.to(DEV), *plan, g.to(DEV), adjacent=adjacent,
                                      grad_mask=ops.GRAD_FEATS | ops.GRAD_PTS)
    u, f = UNIT[TYPES[type]], 2.0 ** -20
    want = _rotary_exact(x, pts, freqs, of_axis, adjacent)
    # cosine, sine and three operations in f32: a few 2^-24 of the pair's size (at most 8 here)
    _within(out, want, u * want.abs() + f * 8, "out")
    back = _rotary_exact(g, pts, freqs, of_axis, adjacent, -1.0)
    _within(d_feats, back, u * back.abs() + f * 8, "d_feats")
    if 2 * pairs < width and points:
        assert torch.equal(out[..., 2 * pairs:].cpu(), x[..., 2 * pairs:])
    p = pts.double().requires_grad_(True)
    angles = p[:, of_axis.long()] * freqs.double() if pairs else torch.zeros((points, 0), dtype=torch.float64)
    one, two = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b, ga, gb = (t.double() for t in (x[..., one], x[..., two], g[..., one], g[..., two]))
    c, s = torch.cos(angles).unsqueeze(1), torch.sin(angles).unsqueeze(1)
    loss = ((a * c - b * s) * ga + (b * c + a * s) * gb).sum()
    want = torch.autograd.grad(loss, p)[0] if pairs else torch.zeros_like(p)
    terms = ((a.abs() + b.abs()) * (ga.abs() + gb.abs())).sum((1, 2)).unsqueeze(1) if pairs else torch.zeros((points, 1))
    _within(d_pts, want.detach(), 2.0 ** -18 * terms.double() + 1e-30, "d_pts")


def test_rotary_keeps_its_accuracy_far_from_the_origin_and_takes_views(ops):
    gen = _gen(11)
    pts, freqs, of_axis = _rotary_plan(gen, 500, 3, 16, reach=1.0e6)
    x = _normal(gen, 500, 4, 32)
    plan = [t.to(DEV) for t in (pts, freqs, of_axis)]
    want = _rotary_exact(x, pts, freqs, of_axis, False)
    _within(ops.rotary(x.to(DEV), *plan), want, torch.full((1,), 2.0 ** -20 * 8, dtype=torch.float64), "far")
    packed = _normal(gen, 500, 2, 4, 33).to(DEV)                  # rows of 33 values: no 16-byte load fits
    got = ops.rotary(packed[:, 1, :, :32], *plan)
    want = _rotary_exact(packed[:, 1, :, :32].cpu(), pts, freqs, of_axis, False)
    _within(got, want, torch.full((1,), 2.0 ** -20 * 8, dtype=torch.float64), "view")
    heads_first = _normal(gen, 4, 500, 32).to(DEV)
    got = ops.rotary(heads_first.transpose(0, 1), *plan)
    assert torch.equal(got, ops.rotary(heads_first.transpose(0, 1).contiguous(), *plan))


def test_rotary_scores_depend_on_the_difference_of_positions(ops):
    # the reason for the operator: q(x) . k(y) is a function of x - y
    gen = _gen(12)
    pts, freqs, of_axis = _rotary_plan(gen, 64, 3, 16, reach=8.0)
    q, k = _normal(gen, 64, 1, 32).to(DEV), _normal(gen, 64, 1, 32).to(DEV)
    f, a = freqs.to(DEV), of_axis.to(DEV)
    def scores(shift):
        moved = (pts + torch.tensor(shift)).to(DEV)
        return ops.rotary(q, moved, f, a)[:, 0].double() @ ops.rotary(k, moved, f, a)[:, 0].double().t()
    # the shift is exact in f32 for these positions up to 2^-20 of them
    assert float((scores([0.0, 0.0, 0.0]) - scores([4.0, -2.0, 8.0])).abs().max()) < 64 * 2.0 ** -18


# -------------------------------------------------------------------------------------------------------- attention

def _starts(sizes):
    return torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32)


def _attention_exact(q, k, v, g, q_sizes, k_sizes, mask, scale):
    """Values in 64 bits and, beside each, the largest error that roundings of relative size u may bring (as a factor
    of u): probabilities, score gradients, D (from the rounded output) and results are rounded once each."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    group = q.shape[1] // k.shape[1]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
    e_out, e_dq, e_dk, e_dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
    qs, ks = _starts(q_sizes).tolist(), _starts(k_sizes).tolist()
    for c in range(len(q_sizes)):
        rows, cols = slice(qs[c], qs[c + 1]), torch.arange(ks[c], ks[c + 1])
        if mask is not None:
            cols = cols[mask[cols]]
        if len(cols) == 0 or qs[c] == qs[c + 1]:
            continue
        for h in range(q.shape[1]):
            hk = h // group
            Q, K, V, G = q[rows, h], k[cols, hk], v[cols, hk], g[rows, h]
            S = Q @ K.t() * scale
            lse[rows, h] = torch.logsumexp(S, 1)
            P = torch.softmax(S, 1)
            O = P @ V
            D = (G * O).sum(1, keepdim=True)
            dP = G @ V.t()
            dS = P * (dP - D)
            out[rows, h], dq[rows, h] = O, scale * dS @ K
            dk[cols, hk] += scale * dS.t() @ Q
            dv[cols, hk] += P.t() @ G
            e_O = P @ V.abs() + O.abs()
            e_S = dS.abs() + P * (G.abs() * e_O).sum(1, keepdim=True)
            e_out[rows, h] = e_O
            e_dq[rows, h] = scale * e_S @ K.abs() + (scale * dS @ K).abs()
            e_dk[cols, hk] += scale * e_S.t() @ Q.abs()
            e_dv[cols, hk] += P.t() @ G.abs()
    return (out, dq, dk, dv, lse), (e_out, e_dq, e_dk + dk.abs(), e_dv + dv.abs())


def _attention_check(ops, type, q_sizes, k_sizes, heads, key_heads, width, off=0.0, seed=0, views="dense", poison=True,
                     scale=None, spread=1.5):
    dtype, gen = TYPES[type], _gen(seed + 17 * width + heads)
    m, n = sum(q_sizes), sum(k_sizes)
    q, g = (_normal(gen, m, heads, width) * spread).to(dtype), _normal(gen, m, heads, width).to(dtype)
    k, v = _normal(gen, n, key_heads, width).to(dtype), _normal(gen, n, key_heads, width).to(dtype)
    mask = None
    if off > 0.0:
        mask = torch.rand((n,), generator=gen) >= off
    dev = [t.to(DEV) for t in (q, k, v, g)]
    if mask is not None and poison:                 # what a switched-off key holds must not matter
        bad = torch.tensor([math.inf, -math.inf, math.nan, torch.finfo(dtype).min])
        for t in (dev[1], dev[2]):
            t[~mask.to(DEV)] = bad[torch.arange(width) % 4].to(dtype).to(DEV)
    if views == "fused":                            # slices of one projection's result, as a network has them
        packed = torch.zeros((m, heads, 2 * width + 3), dtype=dtype, device=DEV)
        packed[..., 1:1 + width], packed[..., width + 3:] = dev[0], dev[3]
        dev[0], dev[3] = packed[..., 1:1 + width], packed[..., width + 3:]
        both = torch.zeros((n, 2, key_heads, width), dtype=dtype, device=DEV)
        both[:, 0], both[:, 1] = dev[1], dev[2]
        dev[1], dev[2] = both[:, 0], both[:, 1]
    elif views == "heads_first":
        dev = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in dev]
    plan = (_starts(q_sizes).to(DEV), _starts(k_sizes).to(DEV), max(q_sizes, default=0), max(k_sizes, default=0))
    key_mask = None if mask is None else mask.to(DEV)
    out, lse = ops.cross_attention(*dev[:3], *plan, key_mask=key_mask, scale=scale, return_lse=True)
    assert torch.equal(out, ops.cross_attention(*dev[:3], *plan, key_mask=key_mask, scale=scale))
    grads = ops.cross_attention_grads(*dev[:3], *plan, out, lse, dev[3], key_mask=key_mask, scale=scale)
    want, spread_of = _attention_exact(q, k, v, g, q_sizes, k_sizes, mask, width ** -0.5 if scale is None else scale)
    u = UNIT[dtype]
    for got, w, e, what in zip((out,) + tuple(grads), want, spread_of, ("out", "d_queries", "d_keys", "d_values")):
        # (bf16 results of f32 arithmetic: the f32 sums' own error on top; it is 2^-8 of u)
        _within(got, w, 1.02 * u * e + 1e-30, what)
    dead = torch.isinf(want[4])
    assert torch.equal(torch.isinf(lse.cpu()), dead) and bool((lse.cpu()[dead] < 0).all())
    if (~dead).any():
        assert float((lse.cpu().double() - want[4])[~dead].abs().max()) < 2.0 ** -16 * float(want[4][~dead].abs().max() + 8)
    if mask is not None and n:
        assert float(grads[1][~key_mask].abs().sum()) == 0.0 and float(grads[2][~key_mask].abs().sum()) == 0.0
    return dev, plan, key_mask, out, lse, grads


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("width", [8, 16, 20, 32, 33, 40, 64, 80, 96, 100, 128])
def test_attention_of_every_width(ops, type, width):
    _attention_check(ops, type, [70, 1, 33], [130, 65, 1], 2, 2, width)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("heads,key_heads", [(1, 1), (4, 1), (6, 2), (8, 8), (12, 4)])
def test_attention_of_shared_key_heads(ops, type, heads, key_heads):
    _attention_check(ops, type, [50, 129], [77, 200], heads, key_heads, 32, seed=3)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("q_sizes,k_sizes", [
    ([1], [1]), ([1], [63]), ([1], [64]), ([1], [65]), ([127], [128]), ([128], [127]), ([129], [129]), ([257], [31]),
    ([0, 5, 0], [7, 9, 0]), ([5, 0, 3], [0, 4, 0]), ([0], [12]), ([12], [0]), ([], []), ([3, 2, 1, 4], [1, 1, 70, 300]),
    ([2000], [3]), ([3], [2000])])
def test_attention_of_uneven_and_empty_clouds(ops, type, q_sizes, k_sizes):
    _attention_check(ops, type, q_sizes, k_sizes, 4, 2, 32, seed=5)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("off", [0.1, 0.9, 1.0])
@pytest.mark.parametrize("q_sizes,k_sizes", [([65, 40], [200, 64]), ([1, 1, 1], [900, 3, 1500]), ([300], [1])])
def test_attention_with_keys_switched_off(ops, type, off, q_sizes, k_sizes):
    _attention_check(ops, type, q_sizes, k_sizes, 4, 2, 64, off=off, seed=7)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("views", ["fused", "heads_first"])
@pytest.mark.parametrize("width", [32, 36])
def test_attention_of_views(ops, type, views, width):
    _attention_check(ops, type, [130, 17], [90, 160], 4, 2, width, seed=9, views=views)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("q_sizes,k_sizes,heads,key_heads,width", [
    ([1] * 3, [5000, 40, 3001], 8, 8, 64), ([1], [20011], 8, 2, 64), ([5, 1], [4097, 9000], 4, 1, 128),
    ([9001], [40], 2, 2, 32), ([6000, 3000], [7, 130], 4, 1, 64)])
def test_attention_split_over_the_long_side(ops, type, q_sizes, k_sizes, heads, key_heads, width):
    _attention_check(ops, type, q_sizes, k_sizes, heads, key_heads, width, seed=11)
    _attention_check(ops, type, q_sizes, k_sizes, heads, key_heads, width, seed=12, off=0.5)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("q_sizes,k_sizes,heads,key_heads,width,off", [
    ([1000, 900], [300, 41], 2, 2, 24, 0.3),       # several own tiles per cloud: f32 keys become planes of terms
    ([1000], [0], 2, 1, 32, 0.0), ([0], [1000], 2, 1, 32, 0.0),
    ([33, 20], [1000, 2000], 3, 1, 48, 0.2),       # groups of three: a tile's rows start inside a group (backward)
    ([40], [950], 6, 1, 64, 0.0), ([700, 2100], [950, 1000], 5, 1, 33, 0.1), ([900], [900], 2, 2, 128, 0.0),
    ([5, 0, 900], [1, 900, 900], 2, 2, 1, 0.0), ([7], [1000], 70, 1, 5, 0.0)])
def test_attention_of_many_own_tiles_and_odd_groups(ops, type, q_sizes, k_sizes, heads, key_heads, width, off):
    _attention_check(ops, type, q_sizes, k_sizes, heads, key_heads, width, off=off, seed=15)


def test_attention_of_more_clouds_than_a_wavefront_orders(ops):
    # up to 64 uneven clouds are worked on longest first, more in their own order; one head and eight (runs of tiles)
    gen = _gen(16)
    for clouds in (63, 64, 65, 130):
        q_sizes = torch.randint(0, 300, (clouds,), generator=gen).tolist()
        k_sizes = torch.randint(0, 200, (clouds,), generator=gen).tolist()
        for heads in (1, 8):
            _attention_check(ops, "bf16", q_sizes, k_sizes, heads, heads, 16, seed=clouds)


def test_the_operators_in_a_graph(ops):
    # captured once, replayed with eager work between the replays, on new inputs each time
    gen = _gen(17)
    x = _normal(gen, 700, 64).to(torch.bfloat16).to(DEV)
    gamma, beta = torch.rand(64, generator=gen).to(DEV), torch.rand(64, generator=gen).to(DEV)
    pts, freqs, of_axis = [t.to(DEV) for t in _rotary_plan(gen, 700, 3, 8)]
    starts, sizes = _starts([300, 400]).to(DEV), 400

    def block():
        y, stats = ops.layer_norm(x, gamma, beta, return_stats=True)
        q = ops.rotary(y.reshape(700, 4, 16), pts, freqs, of_axis)
        out, lse = ops.cross_attention(q, q, q, starts, starts, sizes, sizes, return_lse=True)
        grads = ops.cross_attention_grads(q, q, q, starts, starts, sizes, sizes, out, lse, q)
        back = ops.rotary_grads(q, pts, freqs, of_axis, grads[0])[0]
        return [y, q, out, lse, *grads, *ops.layer_norm_grads(x, gamma, stats, back.reshape(700, 64))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    for i in range(4):
        x.copy_(_normal(gen, 700, 64).to(torch.bfloat16).to(DEV))
        want = block()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), i


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_attention_of_sharp_and_flat_scores(ops, type):
    # scores up to hundreds: one key takes all, the running maximum moves from tile to tile; and all keys alike
    sharp = dict(spread=20.0, scale=0.5) if type == "bf16" else dict(spread=8.0)
    _attention_check(ops, type, [130], [700], 2, 2, 64, seed=13, **sharp)
    _attention_check(ops, type, [130], [700], 2, 2, 64, seed=14, scale=1e-6)


def test_attention_gradients_match_differences(ops):
    gen = _gen(21)
    q, k, v = (_normal(gen, s, 2, 32).to(DEV) for s in (90, 150, 150))
    g = _normal(gen, 90, 2, 32).to(DEV)
    plan = (_starts([40, 50]).to(DEV), _starts([100, 50]).to(DEV), 50, 100)
    mask = (torch.rand((150,), generator=gen) > 0.2).to(DEV)
    out, lse = ops.cross_attention(q, k, v, *plan, key_mask=mask, return_lse=True)
    grads = ops.cross_attention_grads(q, k, v, *plan, out, lse, g, key_mask=mask)
    loss = lambda *t: float((ops.cross_attention(*t, *plan, key_mask=mask).double() * g.double()).sum())
    h = 1e-2
    for i in range(3):
        d = _normal(gen, *(q, k, v)[i].shape).to(DEV)
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = up[i] + h * d, down[i] - h * d
        slope, want = (loss(*up) - loss(*down)) / (2 * h), float((grads[i].double() * d.double()).sum())
        # h^2 of the third derivative along d, and 2^-24 of the outputs over h
        assert abs(slope - want) < 2e-2 * float(grads[i].double().norm()), i


def test_attention_is_the_same_bits_on_every_run_and_stream(ops):
    dev, plan, key_mask, out, lse, grads = _attention_check(ops, "bf16", [300, 7], [900, 2500], 4, 2, 64, off=0.3, seed=23)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, lse2 = ops.cross_attention(*dev[:3], *plan, key_mask=key_mask, return_lse=True)
        grads2 = ops.cross_attention_grads(*dev[:3], *plan, again, lse2, dev[3], key_mask=key_mask)
    side.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert all(torch.equal(a, b) for a, b in zip(grads, grads2))
    only, none, none2 = ops.cross_attention_grads(*dev[:3], *plan, out, lse, dev[3], key_mask=key_mask,
                                                  grad_mask=ops.GRAD_QUERIES)
    assert torch.equal(only, grads[0]) and none is None and none2 is None
    none, dk, dv = ops.cross_attention_grads(*dev[:3], *plan, out, lse, dev[3], key_mask=key_mask, grad_mask=ops.GRAD_KEYS)
    assert none is None and torch.equal(dk, grads[1]) and torch.equal(dv, grads[2])


@pytest.mark.parametrize("width", [33, 64])
def test_attention_gradients_asked_for_alone_are_the_same_bits(ops, width):
    # the rows' statistics come from the queries' kernel when it runs, else from a kernel of their own
    for type in TYPES:
        dev, plan, key_mask, out, lse, grads = _attention_check(ops, type, [90, 300], [500, 77], 4, 2, width, off=0.1, seed=24)
        _, dk, dv = ops.cross_attention_grads(*dev[:3], *plan, out, lse, dev[3], key_mask=key_mask, grad_mask=ops.GRAD_KEYS)
        assert torch.equal(dk, grads[1]) and torch.equal(dv, grads[2])
        dq, _, _ = ops.cross_attention_grads(*dev[:3], *plan, out, lse, dev[3], key_mask=key_mask,
                                             grad_mask=ops.GRAD_QUERIES)
        assert torch.equal(dq, grads[0])


def test_attention_past_32_bit_offsets(ops):
    # keys whose last elements lie past 2^31 elements from the first (a view with wide rows): the last cloud's result is
    # that of the same keys stored densely
    rows, stride = 70000, 32768
    if torch.cuda.mem_get_info()[0] < 3 * rows * stride * 2:
        pytest.skip("needs 14 GB")
    gen = _gen(25)
    store = torch.zeros((rows, stride), dtype=torch.bfloat16, device=DEV)
    keys = store[:, :64].unflatten(1, (2, 32))
    keys[-300:] = _normal(gen, 300, 2, 32).to(torch.bfloat16).to(DEV)
    q = _normal(gen, 20, 2, 32).to(torch.bfloat16).to(DEV)
    starts = torch.tensor([0, 0, 20], dtype=torch.int32, device=DEV)
    key_starts = torch.tensor([0, rows - 300, rows], dtype=torch.int32, device=DEV)
    got = ops.cross_attention(q, keys, keys, starts, key_starts, 20, rows - 300)
    dense = keys[-300:].contiguous()
    want = ops.cross_attention(q, dense, dense, _starts([20]).to(DEV), _starts([300]).to(DEV), 20, 300)
    assert float((got.float() - want.float()).abs().max()) < 2 * 2.0 ** -8 * float(dense.float().abs().max())


def test_operators_refuse_what_they_cannot_take(ops):
    f32 = lambda *s: torch.zeros(s, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    bad = pytest.raises
    with bad(RuntimeError, match="dtype"):
        ops.layer_norm(f32(4, 8).half(), f32(8), f32(8))
    with bad(RuntimeError, match="channels"):
        ops.layer_norm(f32(4, 8), f32(7), f32(8))
    with bad(RuntimeError, match="dtype"):
        ops.layer_norm(f32(4, 8), f32(8), f32(8).bfloat16())
    with bad(RuntimeError, match="dense last dimension"):
        ops.layer_norm(f32(8, 4).t(), f32(8), f32(8))
    with bad(RuntimeError, match="eps"):
        ops.layer_norm(f32(4, 8), f32(8), f32(8), -1.0)
    with bad(RuntimeError, match="inconsistent shapes"):
        ops.layer_norm_grads(f32(4, 8), f32(8), f32(3, 2), f32(4, 8))
    with bad(RuntimeError, match="rows"):
        ops.rotary(f32(4, 2, 8), f32(3, 3), f32(4), i32(0, 1, 2, 0))
    with bad(RuntimeError, match="frequencies"):
        ops.rotary(f32(4, 2, 8), f32(4, 3), f32(5), i32(0, 1, 2, 0, 1))
    with bad(RuntimeError, match="positions"):
        ops.rotary(f32(4, 2, 8), f32(4, 7), f32(4), i32(0, 1, 2, 0))
    q, k, s = f32(4, 4, 16), f32(6, 2, 16), (i32(0, 4), i32(0, 6), 4, 6)
    with bad(RuntimeError, match="heads"):
        ops.cross_attention(q, f32(6, 3, 16), f32(6, 3, 16), *s)
    with bad(RuntimeError, match="expected"):
        ops.cross_attention(q, k, f32(6, 2, 12), *s)
    with bad(RuntimeError, match="head width 136"):
        ops.cross_attention(f32(4, 4, 136), f32(6, 2, 136), f32(6, 2, 136), *s)
    with bad(RuntimeError, match="starts"):
        ops.cross_attention(q, k, k, i32(0, 4), i32(0, 3, 6), 4, 6)
    with bad(RuntimeError, match="scale"):
        ops.cross_attention(q, k, k, *s, scale=-1.0)
    with bad(RuntimeError, match="key_mask"):
        ops.cross_attention(q, k, k, *s, key_mask=torch.ones(5, dtype=torch.bool, device=DEV))
    with bad(RuntimeError, match="dtype"):
        ops.cross_attention(q, k.bfloat16(), k.bfloat16(), *s)
    with bad(RuntimeError, match="keys"):
        ops.cross_attention(q, k, k, i32(0, 4), i32(0, 6), 4, 7)
    out, lse = ops.cross_attention(q, k, k, *s, return_lse=True)
    with bad(RuntimeError, match="inconsistent shapes"):
        ops.cross_attention_grads(q, k, k, *s, out, lse[:3].contiguous(), out)
