"""The feed-forward operators over their whole range on the GPU: every tile that a product may take, offsets past 32 bits, memory
beside results and workspaces, values that are not finite, calls side by side.  Tolerances as in test_gpu_feed_forward.py."""
import ctypes

import pytest
import torch

from .test_gpu_feed_forward import (ACTIVATIONS, DEV, F, TYPES, UNIT, _act, _check_gated, _check_norm, _codes, _gated_exact, _gen,
                                    _normal, _random_codes, _within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pccnn_lib_amd import pccnn_lib_ops
    return pccnn_lib_ops


@pytest.fixture(scope="module")
def lib():
    from pccnn_lib_amd import _lib
    return _lib.load()


# Rows, channels, hidden channels: tiles of 256 x 256 for the projections and for dx (both 225 of them), of 128 x 128, of 128 x 64
# (up to 64 channels), each with edges that end inside a tile; weights' gradients of 64, 128 and 256 channels a tile in many parts.
TILES = [(19169, 520, 264), (10300, 200, 72), (20500, 40, 24), (20501, 33, 61), (5001, 100, 300)]


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels,hidden", TILES)
def test_gated_by_every_tile(ops, type, rows, channels, hidden):
    dtype, gen = TYPES[type], _gen(rows)
    x, g = _normal(gen, rows, channels).to(dtype).to(DEV), _normal(gen, rows, hidden).to(dtype).to(DEV)
    gate, up = ((_normal(gen, hidden, channels) * (k / channels ** 0.5)).to(dtype).to(DEV) for k in (1.5, 1.0))
    _check_gated(ops, x, gate, up, "gelu" if channels % 3 else "silu", g)


# dx in parts of the hidden channels: two of unequal length, several, many, and one whose last 128 bytes are not full
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,channels,hidden", [(300, 72, 600), (300, 512, 1408), (1, 9, 4100), (65, 33, 2051)])
def test_gated_gradients_of_few_rows_and_many_hidden_channels(ops, type, rows, channels, hidden):
    dtype, gen = TYPES[type], _gen(rows + hidden)
    x, g = _normal(gen, rows, channels).to(dtype).to(DEV), _normal(gen, rows, hidden).to(dtype).to(DEV)
    gate, up = ((_normal(gen, hidden, channels) * (k / channels ** 0.5)).to(dtype).to(DEV) for k in (1.5, 1.0))
    got = _check_gated(ops, x, gate, up, "silu", g)
    assert torch.equal(got[1], ops.gated_linear_grads(x, gate, up, g, "silu", grad_mask=ops.GRAD_FEATS)[0])


@pytest.mark.parametrize("rows,channels,hidden", TILES)
def test_8bit_products_by_every_tile(ops, rows, channels, hidden):
    gen = _gen(rows + 1)
    (x, sx), (gate, sg), (up, su) = (_random_codes(gen, n, channels) for n in (rows, hidden, hidden))
    sx, sg = sx / 64, sg / channels ** 0.5 / 64
    bias = _normal(gen, hidden)
    G, U = ((x.double() @ w.double().t()) * sx.double().unsqueeze(1) * s.double() for w, s in ((gate, sg), (up, su)))
    args = [v.to(DEV) for v in (x, sx, gate, sg, up, su)]
    act, _, most, _ = _act(G, "silu")
    h = act * U
    error = 4 * F * h.abs() + (most * 4 * F * G.abs() + 2.0 ** -20 * act.abs()) * U.abs()
    want = U + bias.double()
    for dtype, u in UNIT.items():
        _within(ops.gated_linear_8bit(*args, "silu", dtype), h, u * h.abs() + (1 + u) * error, "gated")
        _within(ops.linear_8bit(args[0], args[1], args[4], args[5], bias.to(DEV), dtype), want,
                u * want.abs() + 4 * F * (U.abs() + want.abs()), "product")


# ------------------------------------------------------------------------------------------------ offsets past 32 bits

MANY = 17000000                                                      # rows of 128: 2.2e9 values


def test_norm_past_32_bit_offsets(ops):
    gen = _gen(1)
    x = torch.zeros((MANY, 128), dtype=torch.bfloat16, device=DEV)
    tail = _normal(gen, 100, 128).to(torch.bfloat16)
    x[-100:] = tail.to(DEV)
    gamma = (1.0 + 0.3 * _normal(gen, 128)).to(DEV)
    out, total, rstd = ops.rms_norm(x, gamma, x, return_stats=True)
    less = ops.rms_norm(x[-100:], gamma, x[-100:], return_stats=True)
    for whole, part in zip((out, total, rstd), less):
        assert torch.equal(whole[-100:], part) and not bool(out[:1000].any())
    d_feats, d_gamma = ops.rms_norm_grads(total, gamma, rstd, x)
    part_feats, part_gamma = ops.rms_norm_grads(less[1], gamma, less[2], x[-100:])
    assert torch.equal(d_feats[-100:], part_feats)
    # rows of zeros add nothing to gamma's gradient; the others are added in another order: a hundred terms, on both sides
    size = (x[-100:].double() * less[1].double() * less[2].double().unsqueeze(1)).abs().sum(0).cpu()
    _within(d_gamma, part_gamma.cpu(), 2 * 104 * F * size, "dgamma")
    del out, total, d_feats
    codes, scales = ops.quantize_rows(x)
    assert torch.equal(codes[-100:].cpu(), _codes(tail)) and not bool(codes[:1000].any()) and not bool(scales[:-100].any())


def test_8bit_product_past_32_bit_offsets(ops):
    gen = _gen(2)
    tail, st = _random_codes(gen, 100, 128)
    w, sw = (v.to(DEV) for v in _random_codes(gen, 130, 128))
    x = torch.zeros((MANY, 128), dtype=torch.int8, device=DEV)
    scales = torch.ones(MANY, device=DEV)
    x[-100:], scales[-100:] = tail.to(DEV), st.to(DEV)
    out = ops.linear_8bit(x, scales, w, sw)
    assert torch.equal(out[-100:], ops.linear_8bit(x[-100:], scales[-100:], w, sw)) and not bool(out[:1000].any())
    h = ops.gated_linear_8bit(x, scales, w, sw, w, sw)
    assert torch.equal(h[-100:], ops.gated_linear_8bit(x[-100:], scales[-100:], w, sw, w, sw)) and not bool(h[:1000].any())


def test_gated_past_32_bit_offsets(ops):
    gen = _gen(3)
    x = torch.zeros((MANY, 128), dtype=torch.bfloat16, device=DEV)
    g = torch.zeros((MANY, 136), dtype=torch.bfloat16, device=DEV)
    x[-100:], g[-100:] = _normal(gen, 100, 128).to(torch.bfloat16).to(DEV), _normal(gen, 100, 136).to(torch.bfloat16).to(DEV)
    gate, up = ((_normal(gen, 136, 128) / 11).to(torch.bfloat16).to(DEV) for _ in range(2))
    h = ops.gated_linear(x, gate, up)
    assert torch.equal(h[-100:], ops.gated_linear(x[-100:], gate, up)) and not bool(h[:1000].any())
    del h
    whole, part = ops.gated_linear_grads(x, gate, up, g), ops.gated_linear_grads(x[-100:], gate, up, g[-100:])
    assert torch.equal(whole[0][-100:], part[0]) and not bool(whole[0][:1000].any())
    # rows of zeros add nothing to the weights' gradients: those of the last rows, and no more error than theirs
    want = _gated_exact(x[-100:].cpu(), gate.cpu(), up.cpu(), "silu", g[-100:].cpu())
    for a, (b, bound), what in zip(whole[1:], want[2:], ("dgate", "dup")):
        _within(a, b, bound, what)


@pytest.mark.parametrize("rows,stride", [(2200, 1 << 20), (1100, 1 << 21)])
def test_rows_far_apart(ops, rows, stride):
    # 2^20 is the largest distance of rows that are operands as they are; beyond it they are laid out anew
    gen = _gen(rows)
    store = torch.empty((rows, stride), dtype=torch.bfloat16, device=DEV)
    x, g = _normal(gen, rows, 64).to(torch.bfloat16).to(DEV), _normal(gen, rows, 48).to(torch.bfloat16).to(DEV)
    store[:, 8:72], store[:, 128:176] = x, g
    gate, up = ((_normal(gen, 48, 64) / 8).to(torch.bfloat16).to(DEV) for _ in range(2))
    far, grads = store[:, 8:72], store[:, 128:176]
    assert torch.equal(ops.gated_linear(far, gate, up), ops.gated_linear(x, gate, up))
    for a, b in zip(ops.gated_linear_grads(far, gate, up, grads), ops.gated_linear_grads(x, gate, up, g)):
        assert torch.equal(a, b)
    gamma = torch.ones(64, device=DEV)
    out, rstd = ops.rms_norm(far, gamma, return_stats=True)
    assert torch.equal(out, ops.rms_norm(x, gamma))
    for a, b in zip(ops.rms_norm_grads(far, gamma, rstd, far), ops.rms_norm_grads(x, gamma, rstd, x)):
        assert torch.equal(a, b)
    assert torch.equal(ops.quantize_rows(far)[0], ops.quantize_rows(x)[0])


# --------------------------------------------------------------------------------- memory beside results and workspaces

class Guarded:
    """A tensor's memory between two guards of 64 KiB; `held` says that both are as they were."""

    def __init__(self, nbytes):
        self.size = 65536
        self.store = torch.full((nbytes + 2 * self.size,), 0xA5, dtype=torch.uint8, device=DEV)
        self.end = self.size + nbytes
        assert self.store.data_ptr() % 256 == 0
        self.p = self.store.data_ptr() + self.size

    def held(self):
        return bool((self.store[:self.size] == 0xA5).all()) and bool((self.store[self.end:] == 0xA5).all())


@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("rows,channels,hidden", [(5, 24, 40), (70, 61, 33), (300, 130, 65), (3000, 250, 264), (70, 24, 2056)])
def test_nothing_is_written_beside_results_and_workspaces(lib, type, rows, channels, hidden):
    from pccnn_lib_amd import _lib
    gen, dtype, bytes = _gen(rows), (torch.float32, torch.bfloat16)[type], (4, 2)[type]
    x, gate, up, g = (_normal(gen, *s).to(dtype).to(DEV) for s in ((rows, channels), (hidden, channels), (hidden, channels), (rows, hidden)))
    p = _lib.Gated()
    p.feats, p.gate, p.up = x.data_ptr(), gate.data_ptr(), up.data_ptr()
    p.feats_stride = p.gate_stride = p.up_stride = channels
    p.n, p.channels, p.hidden, p.type, p.activation = rows, channels, hidden, type, 0
    stream = torch.cuda.current_stream().cuda_stream
    size = lib.pccnn_gated_workspace_bytes(ctypes.byref(p), 0)
    work, out = Guarded(size), Guarded(rows * hidden * bytes)
    assert lib.pccnn_gated_forward(ctypes.byref(p), out.p, type, work.p, size, stream) == 0
    size = lib.pccnn_gated_workspace_bytes(ctypes.byref(p), 1)
    more = [Guarded(n) for n in (size, rows * channels * bytes, hidden * channels * bytes, hidden * channels * bytes)]
    assert lib.pccnn_gated_backward(ctypes.byref(p), g.data_ptr(), hidden, more[1].p, more[2].p, more[3].p, more[0].p, size, stream) == 0
    gamma, rstd = torch.ones(channels, device=DEV), Guarded(4 * rows)
    norm = [Guarded(rows * channels * bytes) for _ in range(3)]
    assert lib.pccnn_rms_norm_forward(x.data_ptr(), type, channels, x.data_ptr(), channels, gamma.data_ptr(), 0, 1e-6, rows, channels,
                                      norm[0].p, norm[1].p, rstd.p, stream) == 0
    size = lib.pccnn_rms_norm_workspace_bytes(rows, channels)
    sums, d_gamma = Guarded(size), Guarded(4 * channels)
    assert lib.pccnn_rms_norm_backward(norm[1].p, type, channels, gamma.data_ptr(), 0, rstd.p, x.data_ptr(), channels, None, 0, rows,
                                       channels, norm[2].p, d_gamma.p, sums.p, size, stream) == 0
    codes, scales = Guarded(rows * channels), Guarded(4 * rows)
    weights, weight_scales = Guarded(hidden * channels), Guarded(4 * hidden)
    assert lib.pccnn_quantize_rows(x.data_ptr(), type, channels, rows, channels, codes.p, scales.p, stream) == 0
    assert lib.pccnn_quantize_rows(gate.data_ptr(), type, channels, hidden, channels, weights.p, weight_scales.p, stream) == 0
    size = lib.pccnn_linear_8bit_workspace_bytes(codes.p, weights.p, rows, channels, hidden)
    space, product = Guarded(size), Guarded(rows * hidden * bytes)
    assert lib.pccnn_linear_8bit(codes.p, scales.p, weights.p, weight_scales.p, None, rows, channels, hidden, product.p, type, space.p,
                                 size, stream) == 0
    torch.cuda.synchronize()
    for memory in [work, out, rstd, sums, d_gamma, codes, scales, weights, weight_scales, space, product] + more + norm:
        assert memory.held()


# ------------------------------------------------------------------------------------------- values that are not finite

@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [20, 300, 20500])
def test_a_row_that_is_not_finite_stays_alone(ops, type, rows):
    dtype, gen = TYPES[type], _gen(rows)
    x, g = _normal(gen, rows, 40).to(dtype).to(DEV), _normal(gen, rows, 24).to(dtype).to(DEV)
    gate, up = ((_normal(gen, 24, 40) / 6).to(dtype).to(DEV) for _ in range(2))
    bad, bad_g = x.clone(), g.clone()
    bad[3, 5], bad[11, 39], bad_g[7, 1] = float("nan"), float("inf"), float("nan")
    fine = torch.ones(rows, dtype=torch.bool, device=DEV)
    fine[3] = fine[11] = False
    fine_g = fine.clone()
    fine_g[7] = False
    for name in ACTIVATIONS:
        h = ops.gated_linear(bad, gate, up, name)
        assert torch.equal(h[fine], ops.gated_linear(x, gate, up, name)[fine]) and bool(h[3].isnan().all())
        assert not bool(torch.isfinite(h[11]).all())
        d = ops.gated_linear_grads(bad, gate, up, bad_g, name)
        want = ops.gated_linear_grads(x, gate, up, g, name)
        assert torch.equal(d[0][fine_g], want[0][fine_g]) and bool(d[0][3].isnan().all()) and bool(d[0][7].isnan().all())
        assert not bool(torch.isfinite(d[1]).any()) and not bool(torch.isfinite(d[2]).any())
    codes, scales = ops.quantize_rows(bad)
    weights, weight_scales = ops.quantize_rows(gate)
    out = ops.linear_8bit(codes, scales, weights, weight_scales)
    hidden = ops.gated_linear_8bit(codes, scales, weights, weight_scales, weights, weight_scales)
    for result in (out, hidden):
        assert bool(torch.isfinite(result[fine]).all()) and bool(result[~fine].isnan().all())


# ------------------------------------------------------------------------------------------------------ side by side

def test_calls_on_two_streams_at_once(ops):
    gen = _gen(8)
    sets = []
    for rows in (4000, 4001):
        x, r, g = (_normal(gen, rows, 96).to(torch.bfloat16).to(DEV) for _ in range(3))
        gate, up = ((_normal(gen, 200, 96) / 10).to(torch.bfloat16).to(DEV) for _ in range(2))
        gamma = (1.0 + 0.1 * _normal(gen, 96)).to(DEV)
        sets.append((x, r, gamma, gate, up, g))

    def run(x, r, gamma, gate, up, g):
        normed, total, rstd = ops.rms_norm(x, gamma, r, return_stats=True)
        h = ops.gated_linear(normed, gate, up)
        grads = ops.gated_linear_grads(normed, gate, up, h)
        codes = ops.rms_norm_8bit(x, gamma, r)
        weights = ops.quantize_rows(gate)
        return [normed, total, rstd, h, *grads, *ops.rms_norm_grads(total, gamma, rstd, grads[0], g), *codes,
                ops.linear_8bit(codes[0], codes[1], *weights)]

    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(run(*s))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        for a, b in zip(results, want[i % 2]):
            assert torch.equal(a, b)


def test_the_same_tensor_in_every_place(ops):
    # features that are the residual too, gate that is up, gradients that are the features
    gen = _gen(5)
    for dtype in TYPES.values():
        x = _normal(gen, 77, 64).to(dtype).to(DEV)
        gamma = (1.0 + 0.1 * _normal(gen, 64)).to(DEV)
        _check_norm(ops, x, x, gamma, x, x)
        w = (_normal(gen, 64, 64) / 8).to(dtype).to(DEV)
        _check_gated(ops, x, w, w, "silu", x)
        _check_gated(ops, w, w, w, "gelu", w)
