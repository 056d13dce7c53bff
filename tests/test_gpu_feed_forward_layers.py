"""The layers of the feed-forward half of a block on the GPU: values and gradients against the formula in 64 bits, the whole block
with attention in front of it, its 8-bit form, HIP graphs, streams, both bindings and what is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# 2-norms, relative to the result's: f32 sums of some hundred terms; bf16 rounds the norm's result, the hidden features, what the
# linear maps give and their sum, one half step of 2^-8 each at most and the mean of one 2^-9.2: five of them and as many
# operands
CLOSE = {torch.float32: 2.0 ** -18, torch.bfloat16: 10 * 2.0 ** -9}


@pytest.fixture(scope="module")
def lib():
    import pccnn_lib_amd
    return pccnn_lib_amd


def _layer(lib, dtype, features=48, hidden=72, activation="silu", seed=0):
    torch.manual_seed(seed)
    layer = lib.pc.layers.GatedFeedForward(features, hidden, activation)
    with torch.no_grad():
        layer.norm_.gamma_.add_(0.2 * torch.randn_like(layer.norm_.gamma_))
    return layer.to(DEV).to(dtype)


def _formula(layer, x, update):
    """The block's formula in 64 bits, with the layer's parameters as leaves -> result, leaves by name."""
    leaves = {name: p.detach().double().requires_grad_(True) for name, p in layer.named_parameters()}
    s = x if update is None else x + update
    normed = s / torch.sqrt((s * s).mean(1, keepdim=True) + layer.norm_.eps_) * leaves["norm_.gamma_"]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid,
           "relu": torch.relu}[layer.activation_]
    hidden = act(normed @ leaves["gate_.weight"].t()) * (normed @ leaves["up_.weight"].t())
    return s + hidden @ leaves["down_.weight"].t() + leaves["down_.bias"], leaves


def _near(got, want, close):
    return float((got.detach().double() - want.detach()).norm()) <= close * float(want.detach().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 50, 300])
@pytest.mark.parametrize("with_update", [False, True])
def test_block_and_its_gradients_against_the_formula(lib, dtype, rows, with_update):
    layer = _layer(lib, dtype, seed=rows)
    x = torch.randn(rows, 48, device=DEV).to(dtype).requires_grad_(True)
    update = torch.randn(rows, 48, device=DEV).to(dtype).requires_grad_(True) if with_update else None
    upstream = torch.randn(rows, 48, device=DEV).to(dtype)
    out = layer(x, update)
    out.backward(upstream)
    ex = x.detach().double().requires_grad_(True)
    eu = None if update is None else update.detach().double().requires_grad_(True)
    want, leaves = _formula(layer, ex, eu)
    want.backward(upstream.double())
    assert out.dtype == dtype and _near(out, want, CLOSE[dtype])
    assert _near(x.grad, ex.grad, CLOSE[dtype]) and (update is None or torch.equal(update.grad, x.grad))
    for name, p in layer.named_parameters():
        assert p.grad.dtype == p.dtype and p.grad.shape == p.shape and _near(p.grad, leaves[name].grad, CLOSE[dtype]), name


def test_gradients_against_differences(lib):
    layer = _layer(lib, torch.float32, 12, 20, "gelu")
    x = torch.randn(70, 12, device=DEV)
    upstream = torch.randn(70, 12, device=DEV)
    leaf = x.clone().requires_grad_(True)
    layer(leaf).backward(upstream)
    loss = lambda v: float((layer(v).double() * upstream.double()).sum())  # noqa: E731
    step = 2.0 ** -6
    with torch.no_grad():
        for _ in range(5):
            way = torch.randn_like(x)
            slope = (loss(x + step * way) - loss(x - step * way)) / (2 * step)
            want = float((leaf.grad.double() * way.double()).sum())
            # third derivatives of O(1) times step^2 on 70 x 12 values, and f32 values of O(10^3) over the step
            assert abs(slope - want) <= 2.0 ** -10 * float(leaf.grad.norm() * way.norm())


def test_unused_results_and_frozen_parts(lib):
    ops = lib.pccnn_lib_ops
    x, r = (torch.randn(40, 24, device=DEV, requires_grad=True) for _ in range(2))
    gamma = torch.rand(24, device=DEV, requires_grad=True)
    _, total = lib.op_wrappers.ComputeRMSNorm.apply(x, gamma, r, 1e-6)
    total.sum().backward()                                      # the norm itself has no part in it
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(r.grad, x.grad) and gamma.grad is None
    x.grad = r.grad = None
    out, _ = lib.op_wrappers.ComputeRMSNorm.apply(x, gamma, r.detach(), 1e-6)
    out.sum().backward()                                        # (an expanded gradient)
    got, total, rstd = ops.rms_norm(x.detach(), gamma.detach(), r.detach(), 1e-6, return_stats=True)
    want = ops.rms_norm_grads(total, gamma.detach(), rstd, torch.ones_like(got))
    assert torch.equal(x.grad, want[0]) and torch.equal(gamma.grad, want[1]) and r.grad is None
    gate, up = (torch.randn(32, 24, device=DEV, requires_grad=True) for _ in range(2))
    lib.op_wrappers.ComputeGatedLinear.apply(x.detach(), gate, up.detach(), "silu").sum().backward()
    assert gate.grad is not None and up.grad is None
    with torch.no_grad():
        assert not lib.op_wrappers.ComputeGatedLinear.apply(x, gate, up, "silu").requires_grad
    tied = torch.randn(32, 24, device=DEV, requires_grad=True)   # one weight on both sides: both gradients add up
    lib.op_wrappers.ComputeGatedLinear.apply(x.detach(), tied, tied, "silu").sum().backward()
    d = ops.gated_linear_grads(x.detach(), tied.detach(), tied.detach(), torch.ones(40, 32, device=DEV))
    assert torch.allclose(tied.grad, d[1] + d[2], rtol=1e-6)


def test_attention_and_feed_forward_in_a_block(lib):
    # two levels of two clouds: attention, then the feed-forward half on what it adds, forward and backward
    torch.manual_seed(2)
    ids = lambda *counts: torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(counts)])  # noqa: E731
    coarse, fine = (lib.pc.Pointcloud(torch.rand(sum(c), 3), ids(*c), device=DEV) for c in ((30, 41), (200, 150)))
    attention = lib.pc.layers.CrossAttention(3, 32, 48, 4, p_unit=0.1).to(DEV)
    feed = _layer(lib, torch.float32)
    y, x = torch.randn(71, 32, device=DEV, requires_grad=True), torch.randn(350, 48, device=DEV, requires_grad=True)
    middle = attention(coarse, fine, y, x)
    out = feed(x, middle - x)
    out.sum().backward()
    want, _ = _formula(feed, x.detach().double(), (middle - x).detach().double())
    assert _near(out, want, CLOSE[torch.float32])
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in (*attention.parameters(), *feed.parameters(), x, y))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 64, 65, 400])
def test_8bit_block_is_its_steps_and_near_the_block(lib, dtype, rows):
    ops = lib.pccnn_lib_ops
    layer = _layer(lib, dtype, 64, 200, "gelu", seed=rows)
    small = lib.pc.layers.GatedFeedForward8Bit(layer)
    x, update = (torch.randn(rows, 64, device=DEV).to(dtype) for _ in range(2))
    with torch.no_grad():
        for u in (None, update):
            got = small(x, u)
            codes, scales, *rest = ops.rms_norm_8bit(x, layer.norm_.gamma_.reshape(-1).float(), u)
            total = rest[0] if rest else x
            weights = [ops.quantize_rows(w.weight) for w in (layer.gate_, layer.up_, layer.down_)]
            hidden = ops.gated_linear_8bit(codes, scales, *weights[0], *weights[1], "gelu", dtype)
            steps = total + ops.linear_8bit(*ops.quantize_rows(hidden), *weights[2], layer.down_.bias.float(), dtype)
            assert got.dtype == dtype and torch.equal(got, steps)
            # four roundings to 8 bits of up to a half of 1/127 of the row's largest, uncorrelated: a few percent of the update
            want = layer(x, u).double() - total.double()
            assert float((got.double() - total.double() - want).norm()) <= 0.1 * float(want.norm()) + CLOSE[dtype] * float(got.double().norm())


def test_8bit_block_refuses_gradients_and_keeps_its_scales(lib):
    layer = _layer(lib, torch.bfloat16)
    small = lib.pc.layers.GatedFeedForward8Bit(layer)
    x = torch.randn(5, 48, device=DEV)
    with pytest.raises(RuntimeError, match="no gradients"):
        small(x.clone().requires_grad_(True))
    want = small(x.bfloat16())
    before = {name: b.clone() for name, b in small.named_buffers()}
    small.to(torch.bfloat16)
    assert all(b.dtype == before[name].dtype and torch.equal(b, before[name]) for name, b in small.named_buffers())
    moved = small.cpu().to(DEV)
    assert torch.equal(moved(x.bfloat16()), want) and small(x).dtype == torch.float32
    copy = lib.pc.layers.GatedFeedForward8Bit(_layer(lib, torch.bfloat16, seed=9))
    copy.load_state_dict(moved.state_dict())
    assert torch.equal(copy(x.bfloat16()), want)


def test_run_in_a_graph_beside_eager_work(lib):
    # inference in both forms and a training step captured once, replayed on new values, with eager calls between the replays
    layer = _layer(lib, torch.bfloat16, 64, 176)
    small = lib.pc.layers.GatedFeedForward8Bit(layer)
    ops = lib.pccnn_lib_ops
    for rows in (3, 300):
        x, update, g = (torch.randn(rows, 64, device=DEV).bfloat16() for _ in range(3))
        gate, up, gamma = layer.gate_.weight.detach(), layer.up_.weight.detach(), layer.norm_.gamma_.detach().reshape(-1)
        hidden_g = torch.randn(rows, 176, device=DEV).bfloat16()

        def step():
            with torch.no_grad():
                served = small(x, update)
                normed, total, rstd = ops.rms_norm(x, gamma, update, return_stats=True)
                hidden = ops.gated_linear(normed, gate, up)
                grads = ops.gated_linear_grads(normed, gate, up, hidden_g)
                return [served, normed, total, hidden, *grads, *ops.rms_norm_grads(total, gamma, rstd, grads[0], g)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        for _ in range(4):
            for t in (x, update, g, hidden_g):
                t.copy_(torch.randn(t.shape, device=DEV))
            want = [t.clone() for t in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_calls_on_another_stream(lib):
    layer = _layer(lib, torch.float32, 64, 200)
    x = torch.randn(500, 64, device=DEV)
    with torch.no_grad():
        want = layer(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [layer(x) for _ in range(3)]
        here = layer(x)
        torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in (*got, here))


@pytest.mark.parametrize("which", ["compiled", "ctypes"])
def test_operators_refuse_what_does_not_belong_together(lib, which):
    ops = lib.pccnn_lib_ops
    before = ops.use_binding(which)
    try:
        x, w = torch.randn(6, 16, device=DEV), torch.randn(24, 16, device=DEV)
        gamma, h = torch.ones(16, device=DEV), torch.randn(6, 24, device=DEV)
        q, s = ops.quantize_rows(x)
        qw, sw = ops.quantize_rows(w)
        _, rstd = ops.rms_norm(x, gamma, return_stats=True)
        half = lambda t: t.half()  # noqa: E731
        for call, message in ((lambda: ops.rms_norm(half(x), gamma), "dtype"),
                              (lambda: ops.rms_norm(x, gamma[:8]), "8 values for 16"),
                              (lambda: ops.rms_norm(x, gamma.bfloat16()), "float32 or the features"),
                              (lambda: ops.rms_norm(x, gamma, x[:5]), "residual"),
                              (lambda: ops.rms_norm(x, gamma, x.bfloat16()), "dtype"),
                              (lambda: ops.rms_norm(x.t(), gamma[:6]), "dense last dimension"),
                              (lambda: ops.rms_norm(x, gamma, eps=-1.0), "eps"),
                              (lambda: ops.rms_norm_8bit(x, gamma, x[:, :8]), "residual"),
                              (lambda: ops.rms_norm_grads(x, gamma, rstd[:5], x), "inconsistent"),
                              (lambda: ops.rms_norm_grads(x, gamma, rstd, x, x[:5]), "inconsistent"),
                              (lambda: ops.rms_norm_grads(x, gamma, rstd, h), "inconsistent"),
                              (lambda: ops.quantize_rows(half(x)), "dtype"),
                              (lambda: ops.quantize_rows(x[:, :0]), "without channels"),
                              (lambda: ops.linear_8bit(x, s, qw, sw), "int8|Char"),
                              (lambda: ops.linear_8bit(q, s[:5], qw, sw), "5 scales for 6 rows"),
                              (lambda: ops.linear_8bit(q, s, qw[:, :8].contiguous(), sw), "expected"),
                              (lambda: ops.linear_8bit(q, s, qw.t(), sw), "contiguous"),
                              (lambda: ops.linear_8bit(q, s, qw, sw, gamma), "bias of 16"),
                              (lambda: ops.linear_8bit(q, s, qw, sw, None, torch.float16), "for the result"),
                              (lambda: ops.gated_linear(x, w, w[:20]), "expected"),
                              (lambda: ops.gated_linear(x, w, w, "tanh"), "activation"),
                              (lambda: ops.gated_linear(x, w.bfloat16(), w.bfloat16()), "dtype"),
                              (lambda: ops.gated_linear(x[:, :0], w[:, :0], w[:, :0]), "expected"),
                              (lambda: ops.gated_linear_grads(x, w, w, x), "in_grads"),
                              (lambda: ops.gated_linear_8bit(q, s, qw, sw, qw[:20], sw[:20]), "expected"),
                              (lambda: ops.gated_linear_8bit(q, s, qw, sw, qw, sw.cpu()), "GPU tensor|device"),
                              (lambda: ops.gated_linear_8bit(q, s, qw, sw, qw, sw, "silu", torch.int8), "for the result")):
            with pytest.raises(RuntimeError, match=message):
                call()
    finally:
        ops.use_binding(before)


def test_both_bindings_give_the_same_bits(lib):
    ops = lib.pccnn_lib_ops
    x, r, w = (torch.randn(s, device=DEV).bfloat16() for s in ((90, 40), (90, 40), (56, 40)))
    gamma, g = torch.rand(40, device=DEV), torch.randn(90, 56, device=DEV).bfloat16()
    results = []
    for which in ("compiled", "ctypes"):
        before = ops.use_binding(which)
        try:
            out, total, rstd = ops.rms_norm(x, gamma, r, return_stats=True)
            q, s, _ = ops.rms_norm_8bit(x, gamma, r)
            qw, sw = ops.quantize_rows(w)
            results.append([out, total, rstd, q, s, qw, sw, *ops.rms_norm_grads(total, gamma, rstd, out, r),
                            ops.linear_8bit(q, s, qw, sw, torch.ones(56, device=DEV)), ops.gated_linear(x, w, w, activation="relu"),
                            *ops.gated_linear_grads(x, w, w, g), ops.gated_linear_8bit(q, s, qw, sw, qw, sw, dtype=torch.float32)])
        finally:
            ops.use_binding(before)
    assert len(results[0]) == len(results[1]) and all(torch.equal(a, b) for a, b in zip(*results))
