"""The layers around layer norm, rotary positions and attention on the GPU: autograd wiring, the block of the three
against the same formula in 64 bits, batches in mixed order, training between two levels of a pooled cloud."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def lib():
    import pccnn_lib_amd
    return pccnn_lib_amd


def _clouds(lib, sizes, seed, shuffle=False):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(sizes)])
    if shuffle:
        ids = ids[torch.randperm(ids.shape[0], generator=gen)]
    return lib.pc.Pointcloud(torch.rand((ids.shape[0], 3), generator=gen).to(DEV), ids.to(DEV))


def _norm64(x, layer):
    mean = x.mean(1, keepdim=True)
    return (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + layer.eps_) * layer.gamma_.double() \
        + layer.betas_.double()


def _block64(layer, pc_in, pc_out, y, x, pts_in, pts_out, mask):
    """The block's formula in 64 bits, one cloud after the other (``pts_*`` double, so that they can carry gradients)."""
    heads, key_heads, width = layer.num_heads_, layer.num_key_heads_, layer.head_width_
    freqs, axes = layer.rotary_.plan(torch.device(DEV))

    def turn(f, pts):
        angles = (pts[:, axes.long()] * freqs.double()).unsqueeze(1)
        p = freqs.shape[0]
        a, b = f[..., :p], f[..., p:2 * p]
        return torch.cat([a * angles.cos() - b * angles.sin(), b * angles.cos() + a * angles.sin(), f[..., 2 * p:]], -1)

    w = lambda m: m.weight.double()
    q = turn((_norm64(x, layer.norm_out_) @ w(layer.proj_q_).t()).reshape(-1, heads, width), pts_out)
    kv = (_norm64(y, layer.norm_in_) @ w(layer.proj_kv_).t()).reshape(-1, 2, key_heads, width)
    k, v = turn(kv[:, 0], pts_in), kv[:, 1]
    out = torch.zeros_like(q)
    for c in range(max(pc_in.batch_size_host(), pc_out.batch_size_host())):
        rows = torch.nonzero(pc_out.batch_ids_ == c)[:, 0]
        keys = (pc_in.batch_ids_ == c) if mask is None else (pc_in.batch_ids_ == c) & mask
        keys = torch.nonzero(keys)[:, 0]
        if len(rows) == 0 or len(keys) == 0:
            continue
        for h in range(heads):
            g = h // (heads // key_heads)
            p = torch.softmax(q[rows, h] @ k[keys, g].t() / math.sqrt(width), 1)
            out = out.index_put((rows, torch.tensor(h, device=DEV)), p @ v[keys, g])
    return x + out.reshape(-1, heads * width) @ w(layer.proj_out_).t() + layer.proj_out_.bias.double()


@pytest.mark.parametrize("shuffle", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_block_and_all_its_gradients_against_the_formula(lib, shuffle, masked):
    torch.manual_seed(3)
    pc_in, pc_out = _clouds(lib, [150, 1, 77, 40], 1, shuffle), _clouds(lib, [60, 90, 33], 2, shuffle)
    layer = lib.pc.layers.CrossAttention(3, 20, 24, 6, p_head_width=16, p_num_key_heads=2, p_unit=0.25).to(DEV)
    gen = torch.Generator().manual_seed(4)
    x = torch.randn((183, 24), generator=gen).to(DEV).requires_grad_(True)
    y = torch.randn((268, 20), generator=gen).to(DEV).requires_grad_(True)
    grads = torch.randn((183, 24), generator=gen).to(DEV)
    mask = (torch.rand((268,), generator=gen) > 0.3).to(DEV) if masked else None
    for pc in (pc_in, pc_out):
        pc.pts_.requires_grad_(True)
    out = layer(pc_in, pc_out, y, x, p_key_mask=mask)
    leaves = [x, y, pc_in.pts_, pc_out.pts_] + list(layer.parameters())
    got = torch.autograd.grad(out, leaves, grads)
    x64, y64 = x.detach().double().requires_grad_(True), y.detach().double().requires_grad_(True)
    pin, pout = pc_in.pts_.detach().double().requires_grad_(True), pc_out.pts_.detach().double().requires_grad_(True)
    want_out = _block64(layer, pc_in, pc_out, y64, x64, pin, pout, mask)
    want = torch.autograd.grad(want_out, [x64, y64, pin, pout] + list(layer.parameters()), grads.double())
    # f32 throughout: 1e-5 of the largest value forward, 1e-4 backward, the project's bounds for whole layers
    assert float((out - want_out).abs().max() / want_out.abs().max()) < 1e-5
    for a, b in zip(got, want):
        assert a.shape == b.shape and float((a - b).abs().max() / b.abs().max()) < 1e-4


def test_functions_ask_for_the_gradients_that_are_wanted(lib):
    gen = torch.Generator().manual_seed(5)
    x, w, b = (torch.randn(s, generator=gen).to(DEV) for s in ((50, 32), (32,), (32,)))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    lib.ComputeLayerNorm.apply(*full, 1e-5).sum().backward()              # an expanded upstream gradient
    for i in range(3):
        one = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        lib.ComputeLayerNorm.apply(*one, 1e-5).sum().backward()
        assert torch.equal(one[i].grad, full[i].grad) and all(t.grad is None for j, t in enumerate(one) if j != i)
    q, k, v = (torch.randn((n, 2, 16), generator=gen).to(DEV) for n in (9, 30, 30))
    plan = (torch.tensor([0, 9], dtype=torch.int32, device=DEV), torch.tensor([0, 30], dtype=torch.int32, device=DEV), 9, 30,
            None, None)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    lib.ComputeCrossAttention.apply(*full, *plan).square().sum().backward()
    for i in range(3):
        one = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        lib.ComputeCrossAttention.apply(*one, *plan).square().sum().backward()
        assert torch.equal(one[i].grad, full[i].grad) and all(t.grad is None for j, t in enumerate(one) if j != i)
    with torch.no_grad():
        assert not lib.ComputeCrossAttention.apply(*full, *plan).requires_grad
    out = lib.ComputeLayerNorm.apply(x.clone().requires_grad_(True), w, b, 1e-5)
    first = torch.autograd.grad(out.square().sum(), out.grad_fn.next_functions[0][0].variable, create_graph=True)[0]
    with pytest.raises(RuntimeError):                                     # no second derivatives, and no wrong ones either
        first.sum().backward()


def test_both_bindings_give_the_same_bits(lib):
    ops = lib.pccnn_lib_ops
    gen = torch.Generator().manual_seed(6)
    x, w = torch.randn((70, 48), generator=gen).to(DEV), torch.randn((48,), generator=gen).to(DEV)
    heads = torch.randn((70, 3, 16), generator=gen).to(DEV).to(torch.bfloat16)
    pts = torch.rand((70, 3), generator=gen).to(DEV)
    freqs, axes = torch.ones(8, device=DEV), torch.zeros(8, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 30, 70], dtype=torch.int32, device=DEV)
    mask = torch.ones(70, dtype=torch.bool, device=DEV)
    results = []
    for which in ("compiled", "ctypes"):
        f = ops.BINDINGS[which]
        y, stats = f["layer_norm"](x, w, w, return_stats=True)
        out, lse = f["cross_attention"](heads, heads, heads, starts, starts, 40, 40, key_mask=mask, scale=0.3, return_lse=True)
        results.append([y, stats, *f["layer_norm_grads"](x, w, stats, x), f["rotary"](heads, pts, freqs, axes, adjacent=True),
                        *f["rotary_grads"](heads, pts, freqs, axes, heads, grad_mask=ops.GRAD_FEATS | ops.GRAD_PTS), out, lse,
                        *f["cross_attention_grads"](heads, heads, heads, starts, starts, 40, 40, out, lse, heads, key_mask=mask,
                                                    scale=0.3)])
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("type", [torch.float32, torch.bfloat16])
def test_training_between_the_levels_of_a_pooled_cloud(lib, type):
    # the fine points learn a function of the whole cloud's coarse points: the loss has to fall
    from pccnn_lib_amd import synthetic
    pts, ids = synthetic.primitives(5, 2, 2048)
    fine = lib.pc.Pointcloud(pts, ids, device=DEV)
    pooling = lib.pc.PointPooling(fine, 0.1)
    coarse = lib.pc.Pointcloud(pooling.pool_tensor(fine.pts_), pooling.pool_tensor(fine.batch_ids_))
    torch.manual_seed(0)
    layer = lib.pc.layers.CrossAttention(3, 16, 32, 4, p_unit=0.2).to(DEV).to(type)
    gen = torch.Generator().manual_seed(1)
    y = torch.randn((coarse.pts_.shape[0], 16), generator=gen).to(DEV).to(type)
    x = torch.randn((fine.pts_.shape[0], 32), generator=gen).to(DEV).to(type)
    ranges = (lib.pc.CloudRanges(coarse), lib.pc.CloudRanges(fine))
    target = fine.global_upsample(coarse.global_pooling(y.float()))[:, :8]
    optimiser = torch.optim.Adam(layer.parameters(), lr=5e-3)
    losses = []
    for _ in range(60):
        out = layer(coarse, fine, y, x, p_ranges=ranges)
        loss = ((out.float() - x.float())[:, :8] - target).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(float(loss))
    assert np.isfinite(losses).all() and losses[-1] < 0.5 * losses[0]


def test_one_token_per_cloud_as_it_is_served(lib):
    # a deployed head: no gradients, one query per cloud, the same answer as that query among others
    torch.manual_seed(2)
    points = _clouds(lib, [3000, 40, 5], 7)
    tokens = lib.pc.Pointcloud(torch.full((3, 3), 0.5, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV))
    twice = lib.pc.Pointcloud(torch.full((6, 3), 0.5, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV) // 2)
    layer = lib.pc.layers.CrossAttention(3, 16, 32, 4, p_num_key_heads=2).to(DEV)
    y, x = torch.randn((3045, 16), device=DEV), torch.randn((3, 32), device=DEV)
    with torch.no_grad():
        alone = layer(points, tokens, y, x)
        pair = layer(points, twice, y, x.repeat_interleave(2, 0))
    assert float((pair[::2] - alone).abs().max()) < 1e-5 * float(alone.abs().max())
    assert float((pair[1::2] - alone).abs().max()) < 1e-5 * float(alone.abs().max())


def test_serving_first_and_training_afterwards(lib):
    torch.manual_seed(4)
    pc_in, pc_out = _clouds(lib, [50, 20], 8, True), _clouds(lib, [9, 30], 9, True)
    served, trained = (lib.pc.layers.CrossAttention(3, 12, 16, 2).to(DEV) for _ in range(2))
    trained.load_state_dict(served.state_dict())
    y, x = torch.randn((70, 12), device=DEV), torch.randn((39, 16), device=DEV)
    with torch.inference_mode():
        ranges = (lib.pc.CloudRanges(pc_in), lib.pc.CloudRanges(pc_out))
        first = served(pc_in, pc_out, y, x, p_ranges=ranges)
    for layer, kept in ((served, ranges), (trained, None)):
        layer(pc_in, pc_out, y, x, p_ranges=kept).square().sum().backward()
    assert torch.equal(first, trained(pc_in, pc_out, y, x))
    for a, b in zip(served.parameters(), trained.parameters()):
        assert torch.equal(a.grad, b.grad)


def test_a_rotary_layers_first_call_in_a_graph(lib):
    layer = lib.pc.layers.RotaryPositions(3, 32).to(DEV)
    feats, pts = torch.randn((40, 2, 32), device=DEV), torch.rand((40, 3), device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(feats, pts)
    for _ in range(3):
        feats.copy_(torch.randn((40, 2, 32), device=DEV))
        want = layer(feats, pts)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_layer_saved_on_the_gpu_and_loaded_on_the_host_comes_back(lib, tmp_path):
    # (the file is this test's own; a whole module is pickled)
    layer = lib.pc.layers.RotaryPositions(3, 32).to(DEV)
    feats, pts = torch.randn((40, 2, 32), device=DEV), torch.rand((40, 3), device=DEV)
    want = layer(feats, pts)
    torch.save(layer, tmp_path / "layer.pt")
    loaded = torch.load(tmp_path / "layer.pt", map_location="cpu", weights_only=False)
    assert torch.equal(loaded(feats, pts), want) and torch.equal(loaded.to(DEV)(feats, pts), want)
