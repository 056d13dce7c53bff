"""The feed-forward operators at the ends of their values on the GPU: rows that no eps covers, products that leave f32, activations
far from zero.  Tolerances as in test_gpu_feed_forward.py; where results are far apart in size they are relative, value by value."""
import pytest
import torch

from . import test_gpu_feed_forward as base
from .test_gpu_feed_forward import DEV, F, TYPES, UNIT, _chain, _codes, _gen, _norm_exact, _normal, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pccnn_lib_amd import pccnn_lib_ops
    return pccnn_lib_ops


# ------------------------------------------------------------------------------------------------------- rows without eps

@pytest.mark.parametrize("eps", [0.0, 1e-60, 1e-42])                     # (the second is zero in f32)
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [24, 700, 9100])
def test_norm_of_tiny_rows_without_eps(ops, type, channels, eps):
    # squares of 1e-20 have a few bits in f32, those of 1e-25 none; 1e-39 has no 1 / rms in f32, but a norm
    dtype, gen = TYPES[type], _gen(channels)
    x, g = _normal(gen, 7, channels), _normal(gen, 7, channels).to(dtype)
    for row, size in enumerate((1.0, 1e-18, 1e-20, 1e-25, 1e-35, 1e-39, 1e30)):
        x[row] *= size
    x, w = x.to(dtype), (1.0 + 0.3 * _normal(gen, channels)).to(DEV)
    small = float(torch.tensor(eps, dtype=torch.float32))
    y, dx, _, xhat, exact = _norm_exact(x, w.cpu(), small, g, None)
    f = F * (_chain(channels) / 2 + 8)
    out, rstd = ops.rms_norm(x.to(DEV), w, eps=eps, return_stats=True)
    # (2^-149: results that are themselves below the smallest normal value)
    _within(out, y, (UNIT[dtype] + f) * y.abs() + (2.0 ** -134 if type == "bf16" else 2.0 ** -149), "out")
    inside = (exact.squeeze(1) < 3e38)
    _within(rstd[inside.to(DEV)], exact.squeeze(1)[inside], f * exact.squeeze(1)[inside] + 2.0 ** -149, "rstd")
    assert bool(rstd[~inside.to(DEV)].isinf().all())
    # the gradients of rows whose 1 / rms squared is far inside f32
    use = slice(0, 3)
    d_feats, _ = ops.rms_norm_grads(x[use].to(DEV), w, rstd[use], g[use].to(DEV))
    scaled = (g.double() * w.cpu().double()).abs()
    size = exact * (scaled + xhat.abs() * (scaled * xhat.abs()).mean(1, keepdim=True))
    _within(d_feats, dx[use], UNIT[dtype] * dx[use].abs() + 4 * f * size[use], "dx")
    codes, scales = ops.rms_norm_8bit(x.to(DEV), w, eps=eps)
    want = y.abs().amax(1) / 127.0
    assert torch.equal(codes.cpu(), _codes(x, w.cpu()))
    _within(scales, want, F * (_chain(channels) / 2 + 9) * want, "scales")


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [24, 700, 9100])
def test_rows_of_zeros_have_scale_zero_without_eps(ops, type, channels):
    gen = _gen(channels)
    x = _normal(gen, 5, channels).to(TYPES[type])
    x[0], x[3] = 0.0, -0.0
    gamma = torch.ones(channels, device=DEV)
    codes, scales = ops.rms_norm_8bit(x.to(DEV), gamma, eps=0.0)
    assert torch.equal(codes.cpu(), _codes(x)) and float(scales[0]) == float(scales[3]) == 0.0 and bool((scales[[1, 2, 4]] > 0).all())
    codes, scales, total = ops.rms_norm_8bit(x.to(DEV), gamma, (-x).to(DEV), eps=0.0)
    assert not bool(total.any()) and not bool(codes.any()) and not bool(scales.any())
    out, rstd = ops.rms_norm(x.to(DEV), gamma, eps=0.0, return_stats=True)
    assert bool(out[[0, 3]].isnan().all()) and bool(rstd[[0, 3]].isinf().all())           # 0 / 0, 1 / 0
    assert bool(torch.isfinite(out[[1, 2, 4]]).all())


@pytest.mark.parametrize("channels", [24, 700, 9100])
def test_norm_of_huge_rows_keeps_eps(ops, channels):
    # squares that leave f32 beside an eps that weighs as much as they do
    x = _normal(_gen(channels), 3, channels) * 1e19
    y, _, _, _, exact = _norm_exact(x, torch.ones(channels), 1e38, torch.ones_like(x), None)
    out, rstd = ops.rms_norm(x.to(DEV), torch.ones(channels, device=DEV), eps=1e38, return_stats=True)
    f = F * (_chain(channels) / 2 + 8)
    _within(rstd, exact.squeeze(1), f * exact.squeeze(1), "rstd")
    _within(out, y, 2 * f * y.abs(), "out")


# ------------------------------------------------------------------------------------------------ activations far from zero

def _one_hot(gates, dtype, rows):
    """Features and weights whose projections are `gates` (values of the type) for every row, and one: one channel each."""
    x = torch.zeros(rows, 8)
    x[:, 0] = x[:, 1] = 1.0
    gate, up = torch.zeros(len(gates), 8), torch.zeros(len(gates), 8)
    gate[:, 0], up[:, 1] = gates, 1.0
    return [t.to(dtype).to(DEV) for t in (x, gate, up)]


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_slopes_of_open_and_closed_gates(ops, type):
    # the gradients of the weights' first channel are sums over equal rows of the slope: of gates up to 80 each keeps its value,
    # on both sides of zero.  exp, reciprocal: 2^-20 as elsewhere and, of exp(-|g|), what a rounding of the exponent's argument brings
    dtype, rows = TYPES[type], 64
    gates = torch.tensor([s * v for v in (0.5, 4.0, 8.0, 12.0, 14.0, 17.0, 20.0, 40.0, 80.0) for s in (1.0, -1.0)], dtype=torch.float64)
    x, gate, up = _one_hot(gates, dtype, rows)
    g = torch.ones(rows, len(gates), dtype=dtype, device=DEV)
    error = 2.0 ** -20 + 2 * F * gates.abs()
    s, rest = torch.sigmoid(gates), torch.sigmoid(-gates)
    for name, act, slope, size in (("sigmoid", s, s * rest, s * rest),
                                   ("silu", gates * s, s * (1 + gates * rest), s * (1 + gates.abs() * rest))):
        d_gate, d_up = (d.cpu().double() for d in ops.gated_linear_grads(x, gate, up, g, name)[1:])
        # dG and dU are rounded as operands, and the sum as a result
        u = 2 * UNIT[dtype] + rows * F
        _within(d_gate[:, 0], rows * slope, rows * (u * slope.abs() + error * size), name + " slope")
        _within(d_up[:, 1], rows * act, rows * (u + error) * act.abs(), name)


def _act_64(g, name):
    """Activation, slope, and the magnitude that the slope's terms have, in 64 bits."""
    if name == "relu":
        return g.clamp(min=0), (g > 0).double(), (g > 0).double()
    if name == "gelu":
        phi, flow = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5), g * torch.exp(-0.5 * g * g) * (0.5 / torch.pi) ** 0.5
        return g * phi, phi + flow, phi + flow.abs()
    s, rest = torch.sigmoid(g), torch.sigmoid(-g)
    if name == "sigmoid":
        return s, s * rest, s * rest
    return g * s, s * (1 + g * rest), s * (1 + g.abs() * rest)


def _act_error(g, name, exact):
    """Of an activation relative to itself, of a slope relative to its terms.  f32 results: half a dozen operations of at most
    2^-23 each, and the arguments' roundings, which an exponential of -g^2 / 2 multiplies by g^2.  bf16 results: exponentials by
    their base-2 instruction, whose argument is rounded twice; the normal distribution to 2^-13.5."""
    if name == "relu":
        return torch.zeros_like(g)
    if name == "gelu":
        return (12 + 2 * g * g) * F + (0.0 if exact else 2.0 ** -13.5)
    return (12 + (0.0 if exact else 4 * g.abs())) * F


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid", "relu"])
def test_activations_keep_their_value_far_from_zero(ops, type, rows, name):
    dtype, exact = TYPES[type], type == "f32"
    far = 12.5 if name == "gelu" else 80.0                             # (Phi(-13) is below the smallest normal value)
    gates = torch.cat([torch.linspace(-far, far, 333), torch.linspace(-2.0, 2.0, 67)]).to(dtype)
    x, gate, up = _one_hot(gates.float(), dtype, rows)
    g = gates.double()
    act, slope, size = _act_64(g, name)
    error, u = _act_error(g, name, exact), UNIT[dtype]
    h = ops.gated_linear(x, gate, up, name)
    _within(h, act.expand(rows, -1), (u + error) * act.abs(), name)
    # one row: the gradients of the weights' channels are dG and dU, rounded as operands and as results
    upstream = torch.zeros(rows, len(gates), dtype=dtype, device=DEV)
    upstream[0] = 1.0
    d_gate, d_up = ops.gated_linear_grads(x, gate, up, upstream, name)[1:]
    twice = 2 * u * (1 + u)
    _within(d_gate[:, 0], slope, twice * slope.abs() + (1 + twice) * error * size, name + " slope")
    _within(d_up[:, 1], act, (twice + (1 + twice) * error) * act.abs(), name)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid", "relu"])
def test_activations_of_8bit_operands_keep_their_value_far_from_zero(ops, rows, name):
    codes = torch.arange(-127, 128).to(torch.int8)
    x, gate, up = (torch.zeros(n, 16, dtype=torch.int8) for n in (rows, len(codes), len(codes)))
    x[:, 0] = x[:, 1] = up[:, 1] = 1
    gate[:, 0] = codes
    scales = [torch.ones(rows), torch.full((len(codes),), 0.0977), torch.ones(len(codes))]           # gates up to 12.4
    g = codes.double() * scales[1].double()
    args = [t.to(DEV) for pair in zip((x, gate, up), scales) for t in pair]
    act, _, _ = _act_64(g, name)
    for dtype, u in UNIT.items():
        # (the scale's product rounds the gate once: as an argument's rounding)
        error = _act_error(g, name, dtype == torch.float32) + (0 if name == "relu" else (2 * g.abs() + 2 * g * g) * F) + F
        _within(ops.gated_linear_8bit(*args, name, dtype), act.expand(rows, -1), (u + error) * act.abs(), name)


# --------------------------------------------------------------------------------------------------- products that leave f32

def _gated_64(x, gate, up, name, g):
    """The formula in 64 bits, for sigmoid with its gradients.  (The slope is s(g) s(-g): s (1 - s) is zero from g = 37 on in 64
    bits too, and infinity times zero is not infinity.)"""
    x, gate, up, g = (t.cpu().double() for t in (x, gate, up, g))
    G, U = x @ gate.t(), x @ up.t()
    if name == "relu":
        return [torch.relu(G) * U]
    s = torch.sigmoid(G)
    dG, dU = g * U * s * torch.sigmoid(-G), g * s
    return [s * U, dG @ gate + dU @ up, dG.t() @ x, dU.t() @ x]


# Rows: without tiles (16, 32 and 64 of them); tiles of 64 x 64, with the weights' gradients and in parts; of 128 x 128; dx of 128 x 64
PAST = [(6, 40, 72), (20, 33, 17), (60, 40, 24), (300, 40, 72), (300, 72, 600), (20500, 40, 72), (10300, 200, 72)]


@pytest.mark.parametrize("rows,channels,hidden", PAST)
def test_gated_f32_of_finite_values_whose_products_leave_f32(ops, rows, channels, hidden):
    gen = _gen(rows + channels)
    x, gate, up, g = (_normal(gen, *s) for s in ((rows, channels), (hidden, channels), (hidden, channels), (rows, hidden)))
    gate, up = gate / channels ** 0.5, up / channels ** 0.5
    x[1, 3], gate[5, 3], gate[6, 3] = 2.5e25, 1e30, -1e30           # two projections of 2.5e55, whose sigmoid is one and zero
    x[:, 2], up[7, 2], g[2, 7] = 0.0, 1e30, 1e20                    # a term of 1e50 / 2 in dx
    x[4, 6], gate[9, 6], g[4, 9] = 1e25, 1.0, 1e20                  # a term of 1e45 in the gradient of up
    args = [t.to(DEV) for t in (x, gate, up)]
    got = [ops.gated_linear(*args, "sigmoid"), *ops.gated_linear_grads(*args, g.to(DEV), "sigmoid")]
    want = _gated_64(x, gate, up, "sigmoid", g)
    # the terms' magnitudes
    s, U = torch.sigmoid(x.double() @ gate.double().t()), (x.double() @ up.double().t()).abs()
    dG, dU = g.double().abs() * U * s * (1 - s), g.double().abs() * s
    U = x.double().abs() @ up.double().abs().t()
    sizes = [s * U, dG @ gate.double().abs() + dU @ up.double().abs(), dG.t() @ x.double().abs(), dU.t() @ x.double().abs()]
    left = 0
    for a, b, size, what in zip(got, want, sizes, ("h", "dx", "dgate", "dup")):
        a, inside = a.cpu(), b.abs() <= torch.finfo(torch.float32).max
        left += int((~inside).sum())
        assert torch.equal(a[~inside], b[~inside].float()), what
        _within(a[inside], b[inside], 2.0 ** -18 * size[inside] + 2.0 ** -100, what)
    assert left == 2                                                # dx[2, 2] and dup[9, 6]
    h, b = ops.gated_linear(*args, "relu").cpu(), _gated_64(x, gate, up, "relu", g)[0].float()
    assert float(b[1, 5].abs()) == float("inf")
    assert torch.equal(h[~torch.isfinite(b)], b[~torch.isfinite(b)]) and torch.equal(torch.isfinite(h), torch.isfinite(b))


@pytest.mark.parametrize("rows,channels,hidden", PAST)
def test_gated_f32_of_infinite_operands_is_what_f32_arithmetic_gives(ops, rows, channels, hidden):
    gen = _gen(rows + channels + 1)
    x, gate, up, g = (_normal(gen, *s) for s in ((rows, channels), (hidden, channels), (hidden, channels), (rows, hidden)))
    inf = float("inf")
    x[1, 3], x[rows - 1, 0], gate[5, 4], up[hidden - 1, channels - 1] = inf, -inf, -inf, inf
    gate[8, 3] = 0.0                                                # infinity times zero
    args = [t.to(DEV) for t in (x, gate, up)]
    h, d_feats = ops.gated_linear(*args, "sigmoid"), ops.gated_linear_grads(*args, g.to(DEV), "sigmoid")[0]
    want = [*_gated_64(x, gate, up, "sigmoid", g)[:2], _gated_64(x, gate, up, "relu", g)[0]]
    for a, b in zip((h, d_feats, ops.gated_linear(*args, "relu")), want):
        a, b = a.cpu(), b.float()
        assert bool(b.isnan().any()) and bool(b.isinf().any())
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[b.isinf()], b[b.isinf()])
        assert torch.equal(torch.isfinite(a), torch.isfinite(b))


# ------------------------------------------------------------------------------------------------------------ in the 2-norm

@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("rows,channels,hidden", [(40, 96, 80), (300, 96, 256), (5000, 128, 200)])
def test_results_and_gradients_in_the_2_norm(ops, type, name, rows, channels, hidden):
    # A rounding to bf16 is evenly spread over a step of 2^-7 of the value's power of two: 2^-7 / sqrt(12) of the value at most in the
    # root mean square.  Results have one, gradients another one of the gradients of the projections, independent of it.  f32: as
    # test_gated_f32_keeps_f32_accuracy has it.
    dtype, gen = TYPES[type], _gen(rows)
    x, gate, up, g = (_normal(gen, *s) for s in ((rows, channels), (hidden, channels), (hidden, channels), (rows, hidden)))
    x, gate, up, g = (t.to(dtype) for t in (x, 1.5 * gate / channels ** 0.5, up / channels ** 0.5, g))
    args = [t.to(DEV) for t in (x, gate, up)]
    got = [ops.gated_linear(*args, name), *ops.gated_linear_grads(*args, g.to(DEV), name)]
    x, gate, up, g = (t.double() for t in (x, gate, up, g))
    G, U = x @ gate.t(), x @ up.t()
    act, slope, _ = _act_64(G, name)
    dG, dU = g * U * slope, g * act
    want = [act * U, dG @ gate + dU @ up, dG.t() @ x, dU.t() @ x]
    one = 2.0 ** -20 if type == "f32" else 2.0 ** -7 / 12 ** 0.5
    for a, b, roundings, what in zip(got, want, (1, 2, 2, 2), ("h", "dx", "dgate", "dup")):
        off = float((a.cpu().double() - b).norm() / b.norm())
        assert off <= one * roundings ** 0.5, "%s: off by %g" % (what, off)


# ------------------------------------------------------------------------------------- few rows in 8 bits, by every load width

@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33])
@pytest.mark.parametrize("channels", [48, 512, 1040, 100, 1028, 33, 511, 513, 1031])
def test_gated_of_few_8bit_rows(ops, rows, channels):
    base.test_gated_8bit_against_exact_sums(ops, rows, channels, 40 + channels % 3)


# -------------------------------------------------------------------------------------- what a workspace held before a call

@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("rows,channels,hidden", [(5, 24, 40), (70, 61, 33), (300, 130, 65), (70, 24, 2056), (3000, 250, 264), (0, 24, 40)])
def test_what_a_workspace_held_has_no_effect(ops, type, rows, channels, hidden):
    import ctypes
    from pccnn_lib_amd import _lib
    lib, gen, dtype = _lib.load(), _gen(rows), (torch.float32, torch.bfloat16)[type]
    x, gate, up, g = (_normal(gen, *s).to(dtype).to(DEV) for s in ((rows, channels), (hidden, channels), (hidden, channels), (rows, hidden)))
    want = [ops.gated_linear(x, gate, up), *ops.gated_linear_grads(x, gate, up, g)]
    p = _lib.Gated()
    p.feats, p.gate, p.up = x.data_ptr(), gate.data_ptr(), up.data_ptr()
    p.feats_stride = p.gate_stride = p.up_stride = channels
    p.n, p.channels, p.hidden, p.type, p.activation = rows, channels, hidden, type, 0
    stream = torch.cuda.current_stream().cuda_stream
    gamma = torch.ones(channels, device=DEV)
    out, rstd = ops.rms_norm(x, gamma, return_stats=True)
    want += [ops.rms_norm_grads(x, gamma, rstd, x)[1]]
    codes, scales = ops.quantize_rows(x)
    weights, weight_scales = ops.quantize_rows(gate)
    want += [ops.linear_8bit(codes, scales, weights, weight_scales, dtype=dtype)]
    for fill in (0xFF, 0x7F):                                              # NaN, and the largest codes and values
        got = [torch.empty_like(t) for t in want]
        space = lambda size: torch.full((size,), fill, dtype=torch.uint8, device=DEV)  # noqa: E731
        work = space(lib.pccnn_gated_workspace_bytes(ctypes.byref(p), 0))
        assert lib.pccnn_gated_forward(ctypes.byref(p), got[0].data_ptr(), type, work.data_ptr(), work.numel(), stream) == 0
        back = space(lib.pccnn_gated_workspace_bytes(ctypes.byref(p), 1))
        assert lib.pccnn_gated_backward(ctypes.byref(p), g.data_ptr(), hidden, got[1].data_ptr(), got[2].data_ptr(), got[3].data_ptr(),
                                        back.data_ptr(), back.numel(), stream) == 0
        sums = space(lib.pccnn_rms_norm_workspace_bytes(rows, channels))
        assert lib.pccnn_rms_norm_backward(x.data_ptr(), type, channels, gamma.data_ptr(), 0, rstd.data_ptr(), x.data_ptr(), channels,
                                           None, 0, rows, channels, None, got[4].data_ptr(), sums.data_ptr(), sums.numel(), stream) == 0
        rows8 = space(lib.pccnn_linear_8bit_workspace_bytes(codes.data_ptr(), weights.data_ptr(), rows, channels, hidden))
        assert lib.pccnn_linear_8bit(codes.data_ptr(), scales.data_ptr(), weights.data_ptr(), weight_scales.data_ptr(), None, rows,
                                     channels, hidden, got[5].data_ptr(), type, rows8.data_ptr(), rows8.numel(), stream) == 0
        assert all(torch.equal(a, b) for a, b in zip(got, want))
