"""The feed-forward half of a block under autocast on the GPU, where features and update come in two types and parameters are float32."""
import pytest
import torch

from .test_gpu_feed_forward_layers import CLOSE, DEV, _formula, _layer, _near

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    import pccnn_lib_amd
    return pccnn_lib_amd


@pytest.mark.parametrize("feats,update", [(F32, None), (BF16, None), (F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows", [7, 300])
def test_block_under_autocast_against_the_formula(lib, feats, update, rows):
    layer = _layer(lib, F32, seed=rows)
    x = torch.randn(rows, 48, device=DEV).to(feats).requires_grad_(True)
    u = None if update is None else torch.randn(rows, 48, device=DEV).to(update).requires_grad_(True)
    upstream = torch.randn(rows, 48, device=DEV)
    with torch.autocast("cuda", dtype=BF16):
        out = layer(x, u)
    assert out.dtype == (BF16 if feats == BF16 and update in (None, BF16) else F32)
    out.backward(upstream.to(out.dtype))
    ex = x.detach().double().requires_grad_(True)
    eu = None if u is None else u.detach().double().requires_grad_(True)
    want, leaves = _formula(layer, ex, eu)
    want.backward(upstream.to(out.dtype).double())
    # bf16 weights and hidden features: the bounds of the bf16 block, and a rounding of each of the four weights' types more
    close = CLOSE[BF16] * 1.5
    assert _near(out, want, close) and x.grad.dtype == feats and _near(x.grad, ex.grad, close)
    if u is not None:
        assert u.grad.dtype == update and _near(u.grad, eu.grad, close)
    for name, p in layer.named_parameters():
        assert p.grad.dtype == F32 and _near(p.grad, leaves[name].grad, close), name


def test_block_under_autocast_multiplies_in_bf16(lib):
    # the gated map's operands are the norm's result and the weights rounded to bf16, whatever the features' type
    layer = _layer(lib, F32, 64, 176)
    x = torch.randn(90, 64, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        got = layer(x)
    ops = lib.pccnn_lib_ops
    normed = ops.rms_norm(x, layer.norm_.gamma_.detach().reshape(-1)).to(BF16)
    hidden = ops.gated_linear(normed, layer.gate_.weight.detach().to(BF16), layer.up_.weight.detach().to(BF16))
    want = x + torch.nn.functional.linear(hidden, layer.down_.weight.detach().to(BF16), layer.down_.bias.detach().to(BF16))
    assert torch.equal(got, want)


def test_8bit_block_under_autocast(lib):
    layer = _layer(lib, F32, 64, 176)
    small = lib.pc.layers.GatedFeedForward8Bit(layer)
    x, u = torch.randn(90, 64, device=DEV), torch.randn(90, 64, device=DEV).to(BF16)
    with torch.no_grad():
        want = small(x, u.float())
        with torch.autocast("cuda", dtype=BF16):
            assert torch.equal(small(x, u), want) and small(u, x).dtype == F32 and small(u).dtype == BF16
        with pytest.raises(RuntimeError, match="dtype"):
            small(x, u)                                               # without autocast two types are a mistake


def test_block_after_attention_under_autocast(lib):
    # attention's result, features updated already, through the whole block, forward and backward
    torch.manual_seed(3)
    ids = lambda *counts: torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(counts)])  # noqa: E731
    coarse, fine = (lib.pc.Pointcloud(torch.rand(sum(c), 3), ids(*c), device=DEV) for c in ((30, 41), (200, 150)))
    attention = lib.pc.layers.CrossAttention(3, 32, 48, 4, p_unit=0.1).to(DEV)
    feed = _layer(lib, F32)
    y, x = torch.randn(71, 32, device=DEV, requires_grad=True), torch.randn(350, 48, device=DEV, requires_grad=True)
    project = torch.nn.Linear(48, 48).to(DEV)
    with torch.autocast("cuda", dtype=BF16):
        middle = attention(coarse, fine, y, x)
        out = feed(middle, project(middle))
        last = feed(project(out))                                     # bf16 features
    want, _ = _formula(feed, middle.detach().double(), project(middle.detach().to(BF16).float()).detach().double())
    assert _near(out, want, CLOSE[BF16] * 1.5) and last.dtype == BF16
    (out.sum() + last.float().sum()).backward()
    for p in (*attention.parameters(), *feed.parameters(), *project.parameters(), x, y):
        assert p.grad is not None and p.grad.dtype == F32 and bool(torch.isfinite(p.grad).all())
