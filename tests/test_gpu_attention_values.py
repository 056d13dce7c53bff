"""Attention on the GPU where live features are not finite, and how exact f32 products are: against the formula in 64 bits."""
import math

import pytest
import torch

from tests import attention_f32

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from pccnn_lib_amd import pccnn_lib_ops
    return pccnn_lib_ops


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float32)


def _starts(*sizes):
    return torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("binding", ["compiled", "ctypes"])
def test_rows_without_a_cloud_are_refused(ops, binding):
    # nothing would write their results
    forward, backward = (ops.BINDINGS[binding][name] for name in ("cross_attention", "cross_attention_grads"))
    q, none, zero = torch.zeros((4, 2, 16), device=DEV), torch.zeros((0, 2, 16), device=DEV), _starts()
    lse = torch.zeros((4, 2), device=DEV)
    for queries, keys in ((q, q), (q, none), (none, q)):
        plan = (zero, zero, queries.shape[0], keys.shape[0])
        with pytest.raises(RuntimeError, match="no clouds"):
            forward(queries, keys, keys, *plan)
        with pytest.raises(RuntimeError, match="no clouds"):
            backward(queries, keys, keys, *plan, queries, lse[:queries.shape[0]], queries)
    assert forward(none, none, none, zero, zero, 0, 0).shape == (0, 2, 16)


# One cloud's queries and keys: the parts that few rows are cut into by the length of the other side.
LENGTHS = [(70, 50), (1, 90), (1, 1500), (2, 4096), (1, 200000), (1000, 40)]


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("queries,keys", LENGTHS)
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_a_query_that_is_not_finite_is_no_query_without_keys(ops, type, queries, keys, bad):
    # row 0 of the second cloud, head 1: every score is NaN (an infinity is one in f32, whose terms of it are; with both
    # signs of the key's features in bf16).  Its result, lse and gradient are NaN; so are, by the formula, the gradients of all
    # that this head's keys share with it; every other row and head is what it is without.
    gen = torch.Generator().manual_seed(queries * 7 + keys)
    dtype, sizes, key_sizes = TYPES[type], (3, queries), (5, keys)
    q, g = (_normal(gen, 3 + queries, 4, 32).to(dtype).to(DEV) for _ in range(2))
    k, v = (_normal(gen, 5 + keys, 2, 32).to(dtype).to(DEV) for _ in range(2))
    plan = (_starts(*sizes), _starts(*key_sizes), max(sizes), max(key_sizes))
    clean, clean_lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    clean_grads = ops.cross_attention_grads(q, k, v, *plan, clean, clean_lse, g)
    q[3, 1] = math.nan
    if bad == "inf":
        q[3, 1, ::2], q[3, 1, 1::2] = math.inf, -math.inf
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    grads = ops.cross_attention_grads(q, k, v, *plan, out, lse, g)
    hit = torch.zeros(out.shape[:2], dtype=torch.bool, device=DEV)
    hit[3, 1] = True
    for got, want in ((out, clean), (lse, clean_lse), (grads[0], clean_grads[0])):
        assert bool(torch.isnan(got[hit]).all())
        assert torch.equal(got[~hit], want[~hit])
    for got, want in zip(grads[1:], clean_grads[1:]):
        assert bool(torch.isnan(got[5:, 0]).all())
        assert torch.equal(got[:5], want[:5]) and torch.equal(got[5:, 1], want[5:, 1])


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("queries,keys", LENGTHS)
@pytest.mark.parametrize("alone", [False, True])
def test_a_live_key_that_is_nan_reaches_every_query_of_its_cloud(ops, type, queries, keys, alone):
    # the key is one among the live ones, or the only one that is not switched off
    gen = torch.Generator().manual_seed(queries * 5 + keys)
    dtype = TYPES[type]
    q, g = (_normal(gen, 3 + queries, 2, 32).to(dtype).to(DEV) for _ in range(2))
    k, v = (_normal(gen, 5 + keys, 2, 32).to(dtype).to(DEV) for _ in range(2))
    plan = (_starts(3, queries), _starts(5, keys), max(3, queries), max(5, keys))
    mask = torch.ones(5 + keys, dtype=torch.bool, device=DEV)
    if alone:
        mask[5:] = False
        mask[5 + keys // 2] = True
    clean, clean_lse = ops.cross_attention(q, k, v, *plan, key_mask=mask, return_lse=True)
    k[5 + keys // 2, 1] = math.nan
    out, lse = ops.cross_attention(q, k, v, *plan, key_mask=mask, return_lse=True)
    assert bool(torch.isnan(out[3:, 1]).all()) and bool(torch.isnan(lse[3:, 1]).all())
    assert torch.equal(out[:3], clean[:3]) and torch.equal(out[3:, 0], clean[3:, 0])
    assert torch.equal(lse[:3], clean_lse[:3]) and torch.equal(lse[3:, 0], clean_lse[3:, 0])
    d_queries, d_keys, d_values = ops.cross_attention_grads(q, k, v, *plan, out, lse, g, key_mask=mask)
    assert bool(torch.isnan(d_queries[3:, 1]).all()) and bool(torch.isfinite(d_queries[:3]).all())
    assert bool(torch.isfinite(d_queries[3:, 0]).all())
    assert bool(torch.isnan(d_keys[5:, 1][mask[5:]]).all()) and bool(torch.isnan(d_values[5:, 1][mask[5:]]).all())
    assert float(d_keys[~mask].abs().sum()) == 0.0 and float(d_values[~mask].abs().sum()) == 0.0


@pytest.mark.parametrize("queries,keys", LENGTHS)
def test_scores_that_are_all_minus_infinity_are_not_the_same_as_no_keys(ops, queries, keys):
    # bf16: every key scores minus infinity, the softmax is 0 / 0; with one key that does not, that key has it all
    gen = torch.Generator().manual_seed(3)
    q, v = torch.ones((queries, 1, 16), device=DEV).bfloat16(), _normal(gen, keys, 1, 16).bfloat16().to(DEV)
    k = torch.full((keys, 1, 16), -math.inf, device=DEV).bfloat16()
    plan = (_starts(queries), _starts(keys), queries, keys)
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())
    k[keys // 2] = 0.25
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    assert torch.equal(out, v[keys // 2:keys // 2 + 1].expand_as(out))
    assert float((lse - 1.0).abs().max()) < 1e-6                       # 16 x 0.25 / sqrt(16)
    none = torch.zeros(keys, dtype=torch.bool, device=DEV)
    out, lse = ops.cross_attention(q, k, v, *plan, key_mask=none, return_lse=True)
    assert float(out.abs().sum()) == 0.0 and bool((lse == -math.inf).all())


@pytest.mark.parametrize("queries,keys", [(1, 1), (3, 700), (1000, 40), (1, 20000)])
def test_f32_features_near_the_largest_value(ops, queries, keys):
    # values from 3.3962e38 on, whose nearest bf16 value is infinite: the key with all the weight hands them on
    row = torch.tensor([3.4e38, -3.4e38, 3.397e38, -3.3965e38, 3.39e38, 1.0, 0.0, -2.0] * 2, device=DEV)
    q, k, v = (torch.zeros((n, 1, 16), device=DEV) for n in (queries, keys, keys))
    q += 1.0
    k[keys // 2] = 8.0                                                  # a score of 32 among zeros
    v[keys // 2, 0] = row
    plan = (_starts(queries), _starts(keys), queries, keys)
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    want = row.double()
    # three terms hold 24 bits, then the products, sums and the division by the sum: a few 2^-24 of the value (the other keys
    # weigh 2^-46 each)
    assert bool(torch.isfinite(out).all())
    assert float(((out[:, 0].double() - want).abs() - 2.0 ** -21 * want.abs()).max()) <= 0.0
    # and as the one output gradient that is not zero: the value's gradient is P times it, P from an lse of 32 in f32 (2^-19)
    g = torch.zeros_like(q)
    g[0, 0] = row
    _, _, d_values = ops.cross_attention_grads(q, k, torch.zeros_like(v), *plan, torch.zeros_like(q), lse, g)
    assert bool(torch.isfinite(d_values).all())
    assert float(((d_values[keys // 2, 0].double() - want).abs() - 2.0 ** -16 * want.abs()).max()) <= 0.0


@pytest.mark.parametrize("queries,keys,heads,key_heads,width", [
    (64, 30, 2, 2, 32), (70, 30, 2, 2, 32), (1, 30, 2, 2, 64), (33, 300, 6, 2, 32), (5, 200, 4, 1, 128), (9001, 40, 2, 2, 32),
    (70, 30, 2, 2, 33)])
def test_a_key_that_scores_minus_infinity_has_no_gradient(ops, queries, keys, heads, key_heads, width):
    # bf16, queries all positive, one live key of minus infinities: probability zero, so its gradients are zero however many
    # rows the last tile of queries has, and every other key's are what they are with that key switched off
    gen = torch.Generator().manual_seed(queries + width)
    normal = lambda n, h: _normal(gen, n, h, width).bfloat16().to(DEV)
    q, g, k, v = normal(queries, heads).abs() + 0.01, normal(queries, heads), normal(keys, key_heads), normal(keys, key_heads)
    k[7] = -math.inf
    mask = torch.ones(keys, dtype=torch.bool, device=DEV)
    mask[7] = False
    plan = (_starts(queries), _starts(keys), queries, keys)
    want, want_lse = ops.cross_attention(q, k, v, *plan, key_mask=mask, return_lse=True)
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    got = ops.cross_attention_grads(q, k, v, *plan, out, lse, g, grad_mask=ops.GRAD_KEYS)[1:]
    for a, b in zip(got, ops.cross_attention_grads(q, k, v, *plan, out, lse, g, key_mask=mask, grad_mask=ops.GRAD_KEYS)[1:]):
        assert torch.equal(a, b) and float(a[7].abs().max()) == 0.0


@pytest.mark.parametrize("queries,keys,width,spread", attention_f32.CASES)
def test_f32_products_keep_f32_accuracy(ops, queries, keys, width, spread):
    # two heads of the second of two clouds, each against 64 bits; what the bounds tell apart: test_attention_f32.py
    heads = [attention_f32.inputs(queries, keys, width, spread, seed) for seed in range(2)]
    small = attention_f32.inputs(3, 5, width, spread)
    q, k, v, g = (torch.stack([torch.cat([small[i], head[i]]) for head in heads], 1).to(DEV) for i in range(4))
    plan = (_starts(3, queries), _starts(5, keys), max(3, queries), max(5, keys))
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    results = [out, lse] + list(ops.cross_attention_grads(q, k, v, *plan, out, lse, g))
    for h, head in enumerate(heads):
        got = [t[5 if t.shape[0] == 5 + keys and i > 2 else 3:, h] for i, t in enumerate(results)]
        for name, error in attention_f32.off(got, attention_f32.exact(*head)).items():
            assert error < attention_f32.MOST[name], (name, h, error)


@pytest.mark.parametrize("queries,keys", [(16, 20000), (40, 9000)])
def test_f32_products_keep_f32_accuracy_in_many_parts(ops, queries, keys):
    # few queries over many keys are split and joined; the sums are longer, of parts of at most some hundred keys
    q, k, v, g = (t.unsqueeze(1).to(DEV) for t in attention_f32.inputs(queries, keys, 64, 4.0))
    plan = (_starts(queries), _starts(keys), queries, keys)
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    results = [out, lse] + list(ops.cross_attention_grads(q, k, v, *plan, out, lse, g))
    want = attention_f32.exact(*(t[:, 0].cpu() for t in (q, k, v, g)))
    for name, error in attention_f32.off([t[:, 0] for t in results], want).items():
        assert error < attention_f32.MOST[name], (name, error)


@pytest.mark.parametrize("clouds,queries,keys,heads,key_heads,width,off", [
    (16, 1, 4096, 8, 8, 64, 0.0), (1, 1, 200000, 8, 2, 64, 0.0), (3, 8, 5000, 8, 2, 32, 0.2), (2, 32, 700, 16, 16, 128, 0.0),
    (4, 3, 900, 8, 1, 33, 0.5), (40, 1, 300, 8, 4, 96, 0.0)])
def test_a_few_bf16_queries_are_as_exact_as_their_results_type(ops, clouds, queries, keys, heads, key_heads, width, off):
    # up to 32 rows to a cloud and key head: the only rounding to bf16 is the result's own.  Probabilities of two terms are off
    # by 2^-17, which adds nothing to that in the 2-norm (rounded to one they would add as much again: 1.41 times)
    gen = torch.Generator().manual_seed(keys + width)
    normal = lambda n, h: _normal(gen, n, h, width).bfloat16()
    q, k, v = normal(clouds * queries, heads) * 1.5, normal(clouds * keys, key_heads), normal(clouds * keys, key_heads)
    live = torch.rand(clouds * keys, generator=gen) >= off
    plan = (_starts(*[queries] * clouds), _starts(*[keys] * clouds), queries, keys)
    out = ops.cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), *plan, key_mask=live.to(DEV) if off else None).double().cpu()
    shape = lambda t, n: t.double().reshape(clouds, n, -1, width).transpose(1, 2)
    q, k, v = shape(q, queries), shape(k, keys), shape(v, keys)
    k, v = (t.repeat_interleave(heads // key_heads, 1) for t in (k, v))
    scores = (q @ k.transpose(2, 3)) * width ** -0.5
    scores = scores.masked_fill(~live.reshape(clouds, 1, 1, keys), -math.inf)
    want = (torch.softmax(scores, 3) @ v).transpose(1, 2).reshape(out.shape)
    own = (want.bfloat16().double() - want).norm()
    assert float((out - want).norm() / own) < 1.05


@pytest.mark.parametrize("clouds,queries,keys,heads,key_heads,width,off", [
    (2, 2000, 2, 4, 4, 32, 0.0), (3, 700, 5, 8, 2, 64, 0.3), (2, 900, 17, 2, 2, 24, 0.0), (2, 1500, 33, 4, 4, 128, 0.2),
    (1, 2000, 64, 4, 2, 33, 0.0), (8, 40, 3, 4, 1, 96, 0.0)])
def test_bf16_gradients_of_few_keys(ops, clouds, queries, keys, heads, key_heads, width, off):
    # up to 64 keys to a cloud.  Score gradients and results are rounded to bf16 once each: sqrt(2) times the result's own
    # rounding in the 2-norm, 1.5 with what the sizes of few values scatter; D = dO . O of a rounded O would add up to twice
    # that again.  dq and dk are asked for together and alone, with the same bits.
    gen = torch.Generator().manual_seed(keys + width)
    normal = lambda n, h: _normal(gen, n, h, width).bfloat16()
    q, g = normal(clouds * queries, heads) * 1.5, normal(clouds * queries, heads)
    k, v = normal(clouds * keys, key_heads), normal(clouds * keys, key_heads)
    live = torch.rand(clouds * keys, generator=gen) >= off
    plan = (_starts(*[queries] * clouds), _starts(*[keys] * clouds), queries, keys)
    dev, mask = [t.to(DEV) for t in (q, k, v)], live.to(DEV) if off else None
    out, lse = ops.cross_attention(*dev, *plan, key_mask=mask, return_lse=True)
    grads = ops.cross_attention_grads(*dev, *plan, out, lse, g.to(DEV), key_mask=mask)
    dq, _, _ = ops.cross_attention_grads(*dev, *plan, out, lse, g.to(DEV), key_mask=mask, grad_mask=ops.GRAD_QUERIES)
    _, dk, dv = ops.cross_attention_grads(*dev, *plan, out, lse, g.to(DEV), key_mask=mask, grad_mask=ops.GRAD_KEYS)
    assert all(torch.equal(a, b) for a, b in zip(grads, (dq, dk, dv)))
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    shape = lambda t, n: t.reshape(clouds, n, -1, width).transpose(1, 2)
    x, y, z = (shape(t, n) for t, n in zip(leaves, (queries, keys, keys)))
    y, z = (t.repeat_interleave(heads // key_heads, 1) for t in (y, z))
    scores = (x @ y.transpose(2, 3)) * width ** -0.5
    scores = scores.masked_fill(~live.reshape(clouds, 1, 1, keys), -math.inf)
    probabilities = torch.softmax(scores, 3).nan_to_num(0.0)            # (a cloud without a live key)
    want = torch.autograd.grad((probabilities @ z).transpose(1, 2).reshape(g.shape), leaves, g.double())
    for name, a, b in zip(("d_queries", "d_keys", "d_values"), grads, want):
        own = (b.bfloat16().double() - b).norm()
        assert float((a.double().cpu() - b).norm() / own) < 1.5, name


def test_bf16_gradients_of_one_key(ops):
    # P is 1 and dP - D zero: what is left is the f32 rounding of the two
    gen = torch.Generator().manual_seed(2)
    q, k, v, g = (_normal(gen, n, 2, 32).bfloat16().to(DEV) for n in (500, 1, 1, 500))
    plan = (_starts(500), _starts(1), 500, 1)
    out, lse = ops.cross_attention(q, k, v, *plan, return_lse=True)
    d_queries, d_keys, _ = ops.cross_attention_grads(q, k, v, *plan, out, lse, g)
    size = (g.float().abs().amax() * v.float().abs().amax() * 32).item()
    assert float(d_queries.float().abs().max()) < 2.0 ** -20 * size * float(k.float().abs().max())
    assert float(d_keys.float().abs().max()) < 2.0 ** -20 * size * float(q.float().abs().sum(0).max())
