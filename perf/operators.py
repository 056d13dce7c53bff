"""What the speed of the attention operators is measured on: layer norm, rotary positions over several axes, and
attention from one level of a point cloud to another.

The three run one after the other in a block that carries features between levels (a decoder's fine points asking the
pooled ones, a few latent points asking a whole scene, one token per cloud asking all of it):

* ``norm``       layer norm of point features, inference or a training step (features', scale's and offset's gradients);
* ``rotary``     pairs of a head's features turned by angles that are positions times frequencies, inference or with the
                 gradient of the features;
* ``attention``  softmax attention of the queries of a cloud to the keys of the same cloud of another level, clouds of
                 uneven sizes stored one behind the other, several query heads to a key head, keys that are switched off;
                 inference or a training step (queries', keys' and values' gradients).

Point counts are those of the repository's benchmark and tests (16 x 4096, 8 x 8192, 8 x 100000, a scene of 10^6) and
sizes around them.
"""
import math

import torch

own = False

_DEVICE = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5


def _norm(name=None, rows=1024, channels=64, type="f32", weights="f32", mode="infer"):
    case = dict(kind="norm", rows=rows, channels=channels, type=type, weights=weights, mode=mode)
    if name:
        case["name"] = name
    return case


def _rotary(name=None, points=1024, heads=4, width=32, pairs=16, axes=3, adjacent=False, type="f32", mode="infer"):
    """``width``: features of a head; the first 2 * ``pairs`` of them are turned."""
    case = dict(kind="rotary", points=points, heads=heads, width=width, pairs=pairs, axes=axes, adjacent=adjacent,
                type=type, mode=mode)
    if name:
        case["name"] = name
    return case


def _attention(name=None, clouds=1, queries=1, keys=1024, ragged=False, heads=8, key_heads=8, width=64, off=0.0,
               type="bf16", mode="infer"):
    """``queries``, ``keys``: of every cloud, the largest when ``ragged``; ``off``: share of the keys switched off."""
    case = dict(kind="attention", clouds=clouds, queries=queries, keys=keys, ragged=ragged, heads=heads,
                key_heads=key_heads, width=width, off=off, type=type, mode=mode)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the latent tokens of one small batch, deployed: the smallest call
        _norm("norm_infer_8x96", rows=8, channels=96),
        # the features of the benchmark's object batch, a training step
        _norm("norm_train_16x4096x128", rows=65536, channels=128, mode="train"),
        # the finest level of the benchmark's encoder, bf16 features under fp32 weights
        _norm("norm_train_bf16_8x100000x64", rows=800000, channels=64, type="bf16", mode="train"),
        # a small batch's queries, deployed
        _rotary("rotary_infer_2x1024", points=2048, heads=4, width=32, pairs=16),
        # keys of four scenes in training, half of each head turned, odd point count
        _rotary("rotary_train_bf16_119997", points=119997, heads=8, width=64, pairs=32, type="bf16", mode="train"),
        # one token per cloud asks all points of its cloud (a deployed classifier's head)
        _attention("attention_token_16x4096", clouds=16, queries=1, keys=4096, heads=8, key_heads=8, width=64),
        # one token asks a whole scene, four query heads to a key head
        _attention("attention_token_scene_1000000", clouds=1, queries=1, keys=1000000, heads=8, key_heads=2, width=64),
        # a small deployed fp32 network, uneven clouds, narrow heads
        _attention("attention_infer_f32_5x777", clouds=5, queries=777, keys=1201, ragged=True, heads=4, key_heads=4,
                   width=24, type="f32"),
        # the way back up in fp32 training: all points ask the pooled ones, some of which are switched off
        _attention("attention_train_f32_16x4096", clouds=16, queries=4096, keys=600, heads=4, key_heads=4, width=32,
                   off=0.1, type="f32", mode="train"),
        # the same in bf16 training with uneven clouds
        _attention("attention_train_bf16_8x8192", clouds=8, queries=8192, keys=2047, ragged=True, heads=8, key_heads=8,
                   width=64, mode="train"),
        # latent points gather from the benchmark's encoder input, grouped heads, training
        _attention("attention_train_bf16_latents_8x100000", clouds=8, queries=256, keys=100000, heads=8, key_heads=2,
                   width=64, mode="train"),
        # a pooled level asks a room of the input level, deployed
        _attention("attention_infer_bf16_34123x100000", clouds=1, queries=34123, keys=100000, heads=4, key_heads=4,
                   width=128),
    ]


# what a drawn case may cost at most: the largest listed ones' arithmetic, bytes and scores (heads x pairs)
_MOST_FLOPS, _MOST_BYTES, _MOST_SCORES = 3.0e12, 4.8e8, 6.0e9


def _too_much(case):
    cost, train = work(case), case["mode"] == "train"
    if cost["bytes"] > _MOST_BYTES:
        return True
    scores = cost["flops"] / (2.0 * case["width"] * (7 if train else 2))
    return cost["flops"] > _MOST_FLOPS * (1.0 if case["type"] == "bf16" else 0.15) \
        or scores > _MOST_SCORES * (0.5 if train else 1.0)


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "rotary", "attention", "attention"])
    if kind == "norm":
        type = rng.choice(["f32", "bf16"])
        channels = rng.choice([_log_int(rng, 16, 1024), 8 * rng.randint(2, 64), 2 ** rng.randint(5, 10)])
        rows = _log_int(rng, 1, min(800000, (50000000 if type == "bf16" else 25000000) // channels))
        return _norm(None, rows, channels, type, rng.choice(["f32", type]), rng.choice(["infer", "train"]))
    type = rng.choice(["f32", "bf16"])
    width = rng.choice([16, 20, 24, 32, 32, 40, 48, 64, 64, 80, 96, 128])
    key_heads = rng.choice([1, 2, 4, 8])
    if kind == "rotary":
        axes = rng.randint(1, 4)
        pairs = max(axes, rng.choice([width // 2, width // 2, width // 4]))
        points = _log_int(rng, 1, (60000000 if type == "bf16" else 30000000) // (key_heads * width))
        return _rotary(None, points, key_heads, width, pairs, axes, rng.choice([True, False]), type,
                       rng.choice(["infer", "train"]))
    heads = key_heads * rng.choice([1, 1, 2, 4])
    clouds = rng.randint(1, 16)
    mode = rng.choice(["infer", "train"])
    shape = rng.choice(["token", "few", "down", "up", "even"])
    queries, keys = {"token": (1, _log_int(rng, 1, 1000000 // clouds)),
                     "few": (rng.randint(2, 64), _log_int(rng, 16, 400000 // clouds)),
                     "down": (_log_int(rng, 64, 1024), _log_int(rng, 1024, 100000 // clouds)),
                     "up": (_log_int(rng, 1024, 100000 // clouds), _log_int(rng, 1, 1024)),
                     "even": (_log_int(rng, 64, 40000 // clouds), _log_int(rng, 64, 40000 // clouds))}[shape]
    case = _attention(None, clouds, queries, keys, rng.choice([True, False]), heads, key_heads, width,
                      rng.choice([0.0, 0.0, 0.2, 0.6]), type, mode)
    while _too_much(case):
        case["queries"], case["keys"] = max(1, case["queries"] * 4 // 5), max(1, case["keys"] * 4 // 5)
    return case


# ------------------------------------------------------------------------------------------------------- preparation

def _sizes(case, largest, salt):
    """Rows of every cloud: all alike, or between nothing much and all of the stated number."""
    if not case["ragged"]:
        return [largest] * case["clouds"]
    steps = [((i * 7 + salt) % 11) / 10.0 for i in range(case["clouds"])]
    return [max(1, int(round(largest * (0.35 + 0.65 * s)))) for s in steps]


def _starts(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def _frequencies(pairs, axes):
    """Pairs dealt to the axes as evenly as they go, on each axis a geometric row of frequencies from 1 downwards."""
    of_axis, freqs = [], []
    for a in range(axes):
        count = pairs // axes + (1 if a < pairs % axes else 0)
        of_axis += [a] * count
        freqs += [100.0 ** (-j / count) for j in range(count)]
    return freqs, of_axis


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(int(seed) * 7919 + 13)
    type = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=_DEVICE, dtype=torch.float32)

    state = dict(case=case)
    if case["kind"] == "norm":
        rows, channels = case["rows"], case["channels"]
        weights = _TYPES[case["weights"]]
        # features behind a residual sum: uneven scales, a mean that is not zero
        state["feats"] = (normal(rows, channels) * 1.7 + normal(1, channels) * 0.5 + 0.3).to(type)
        state["gamma"] = (1.0 + 0.2 * normal(channels)).to(weights)
        state["beta"] = (0.1 * normal(channels)).to(weights)
        if case["mode"] == "train":
            state["in_grads"] = normal(rows, channels).to(type)
    elif case["kind"] == "rotary":
        points, heads, width = case["points"], case["heads"], case["width"]
        state["feats"] = normal(points, heads, width).to(type)
        # coordinates of a room of ten metres in units of a search radius of five centimetres
        state["pts"] = torch.rand((points, case["axes"]), generator=gen, device=_DEVICE) * 200.0
        freqs, of_axis = _frequencies(case["pairs"], case["axes"])
        state["freqs"] = torch.tensor(freqs, dtype=torch.float32, device=_DEVICE)
        state["axes"] = torch.tensor(of_axis, dtype=torch.int32, device=_DEVICE)
        if case["mode"] == "train":
            state["in_grads"] = normal(points, heads, width).to(type)
    else:
        heads, key_heads, width = case["heads"], case["key_heads"], case["width"]
        query_sizes, key_sizes = _sizes(case, case["queries"], 3), _sizes(case, case["keys"], 8)
        m, n = sum(query_sizes), sum(key_sizes)
        state["queries"] = (normal(m, heads, width) * 1.5).to(type)
        state["keys"] = normal(n, key_heads, width).to(type)
        state["values"] = normal(n, key_heads, width).to(type)
        state["query_sizes"], state["key_sizes"] = query_sizes, key_sizes
        state["query_starts"] = torch.tensor(_starts(query_sizes), dtype=torch.int32, device=_DEVICE)
        state["key_starts"] = torch.tensor(_starts(key_sizes), dtype=torch.int32, device=_DEVICE)
        state["key_mask"] = None
        if case["off"] > 0.0:
            state["key_mask"] = torch.rand((n,), generator=gen, device=_DEVICE) >= case["off"]
        if case["mode"] == "train":
            state["in_grads"] = normal(m, heads, width).to(type)
    return state


# ------------------------------------------------------------------------------------------------------ plain forms

def _plain_norm(state):
    feats, gamma, beta = state["feats"].float(), state["gamma"].float(), state["beta"].float()
    mean = feats.mean(dim=1, keepdim=True)
    centred = feats - mean
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + _EPS)
    normed = centred * rstd
    out = (normed * gamma + beta).to(state["feats"].dtype)
    if state["case"]["mode"] == "infer":
        return out
    grads = state["in_grads"].float()
    d_gamma, d_beta = (grads * normed).sum(dim=0), grads.sum(dim=0)
    scaled = grads * gamma
    d_feats = rstd * (scaled - scaled.mean(dim=1, keepdim=True) - normed * (scaled * normed).mean(dim=1, keepdim=True))
    return [out, d_feats.to(out.dtype), d_gamma.to(state["gamma"].dtype), d_beta.to(state["gamma"].dtype)]


def _turn(feats, cos, sin, pairs, adjacent):
    out = feats.float().clone()
    if adjacent:
        one, two = out[..., 0:2 * pairs:2].clone(), out[..., 1:2 * pairs:2].clone()
        out[..., 0:2 * pairs:2] = one * cos - two * sin
        out[..., 1:2 * pairs:2] = two * cos + one * sin
    else:
        one, two = out[..., :pairs].clone(), out[..., pairs:2 * pairs].clone()
        out[..., :pairs] = one * cos - two * sin
        out[..., pairs:2 * pairs] = two * cos + one * sin
    return out.to(feats.dtype)


def _plain_rotary(state):
    case = state["case"]
    angles = (state["pts"][:, state["axes"].long()] * state["freqs"]).unsqueeze(1)
    cos, sin = torch.cos(angles), torch.sin(angles)
    out = _turn(state["feats"], cos, sin, case["pairs"], case["adjacent"])
    if case["mode"] == "infer":
        return out
    return [out, _turn(state["in_grads"], cos, -sin, case["pairs"], case["adjacent"])]


_SCORES_AT_ONCE = 1 << 28


def _plain_attention(state):
    case = state["case"]
    heads, key_heads, width = case["heads"], case["key_heads"], case["width"]
    group, scale, type = heads // key_heads, 1.0 / math.sqrt(width), state["queries"].dtype
    train = case["mode"] == "train"
    out = torch.empty_like(state["queries"])
    d_queries, d_keys, d_values = (torch.empty_like(state[x]) if train else None for x in ("queries", "keys", "values"))
    q_end = k_end = 0
    for m, n in zip(state["query_sizes"], state["key_sizes"]):
        q0, q_end, k0, k_end = q_end, q_end + m, k_end, k_end + n
        keys = state["keys"][k0:k_end].float().transpose(0, 1).contiguous()              # [key heads, n, width]
        values = state["values"][k0:k_end].float().transpose(0, 1).contiguous()
        keys_t = keys.transpose(1, 2).contiguous()
        values_t = values.transpose(1, 2).contiguous() if train else None
        masked = None if state["key_mask"] is None else ~state["key_mask"][k0:k_end]
        dk = torch.zeros_like(keys) if train else None
        dv = torch.zeros_like(values) if train else None
        step = max(1, _SCORES_AT_ONCE // (heads * n))
        for lo in range(q0, q_end, step):
            hi = min(q_end, lo + step)
            rows = (hi - lo) * group

            def by_head(x):
                x = x[lo:hi].float().reshape(hi - lo, key_heads, group, width)
                return x.permute(1, 0, 2, 3).reshape(key_heads, rows, width).contiguous()

            def by_point(x):
                x = x.reshape(key_heads, hi - lo, group, width).permute(1, 0, 2, 3)
                return x.reshape(hi - lo, heads, width).to(type)

            queries = by_head(state["queries"])
            scores = torch.bmm(queries, keys_t) * scale
            if masked is not None:
                scores = scores.masked_fill(masked, -float("inf"))
            top = scores.amax(dim=2, keepdim=True)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            scores = torch.exp(scores - top)
            total = scores.sum(dim=2, keepdim=True)
            probs = scores / torch.where(total > 0, total, torch.ones_like(total))
            result = torch.bmm(probs, values)
            out[lo:hi] = by_point(result)
            if train:
                grads = by_head(state["in_grads"])
                dv += torch.bmm(probs.transpose(1, 2).contiguous(), grads)
                delta = (grads * result).sum(dim=2, keepdim=True)
                d_scores = probs * (torch.bmm(grads, values_t) - delta) * scale
                d_queries[lo:hi] = by_point(torch.bmm(d_scores, keys))
                dk += torch.bmm(d_scores.transpose(1, 2).contiguous(), queries)
        if train:
            d_keys[k0:k_end] = dk.transpose(0, 1).to(type)
            d_values[k0:k_end] = dv.transpose(0, 1).to(type)
    return [out, d_queries, d_keys, d_values] if train else out


# ----------------------------------------------------------------------------------------- the framework's operators

def _own(state):
    import pccnn_lib_amd.pccnn_lib_ops as ops
    case = state["case"]
    train = case["mode"] == "train"
    if case["kind"] == "norm":
        if not train:
            return ops.layer_norm(state["feats"], state["gamma"], state["beta"], _EPS)
        out, stats = ops.layer_norm(state["feats"], state["gamma"], state["beta"], _EPS, return_stats=True)
        return [out] + list(ops.layer_norm_grads(state["feats"], state["gamma"], stats, state["in_grads"]))
    if case["kind"] == "rotary":
        plan = (state["pts"], state["freqs"], state["axes"])
        out = ops.rotary(state["feats"], *plan, adjacent=case["adjacent"])
        if not train:
            return out
        d_feats, _ = ops.rotary_grads(state["feats"], *plan, state["in_grads"], adjacent=case["adjacent"],
                                      grad_mask=ops.GRAD_FEATS)
        return [out, d_feats]
    args = (state["queries"], state["keys"], state["values"], state["query_starts"], state["key_starts"],
            max(state["query_sizes"]), max(state["key_sizes"]))
    if not train:
        return ops.cross_attention(*args, key_mask=state["key_mask"])
    out, lse = ops.cross_attention(*args, key_mask=state["key_mask"], return_lse=True)
    return [out] + list(ops.cross_attention_grads(*args, out, lse, state["in_grads"], key_mask=state["key_mask"]))


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention}[state["case"]["kind"]](state)


def work(case):
    size = {"f32": 4, "bf16": 2}[case["type"]]
    train = case["mode"] == "train"
    if case["kind"] == "norm":
        cells, weight = case["rows"] * case["channels"], {"f32": 4, "bf16": 2}[case["weights"]]
        # features in, result out; training: gradient in, gradient out, gradients of both weights
        return {"bytes": cells * size * (4 if train else 2) + case["channels"] * weight * (4 if train else 2),
                "flops": cells * (22 if train else 8)}
    if case["kind"] == "rotary":
        cells = case["points"] * case["heads"] * case["width"]
        turned = case["points"] * case["heads"] * 2 * case["pairs"]
        return {"bytes": cells * size * (4 if train else 2) + case["points"] * case["axes"] * 4 + case["pairs"] * 8,
                "flops": turned * (6 if train else 3)}
    query_sizes, key_sizes = _sizes(case, case["queries"], 3), _sizes(case, case["keys"], 8)
    m, n = sum(query_sizes), sum(key_sizes)
    pairs = sum(a * b for a, b in zip(query_sizes, key_sizes)) * (1.0 - case["off"])
    products = 7 if train else 2                    # of 2 * width operations for every query head and pair
    cells_q, cells_k = m * case["heads"] * case["width"], n * case["key_heads"] * case["width"]
    moved = (cells_q * (4 if train else 2) + cells_k * (4 if train else 2)) * size + (n if case["off"] > 0.0 else 0)
    return {"bytes": moved, "flops": pairs * case["heads"] * case["width"] * 2 * products}


# --------------------------------------------------------------------------------------- the definitions, in 64 bits

def _exact_norm(state):
    train = state["case"]["mode"] == "train"
    leaves = [state[x].double().requires_grad_(train) for x in ("feats", "gamma", "beta")]
    feats, gamma, beta = leaves
    variance, mean = torch.var_mean(feats, dim=1, keepdim=True, correction=0)
    out = (feats - mean) / torch.sqrt(variance + _EPS) * gamma + beta
    if not train:
        return out
    return [out.detach()] + list(torch.autograd.grad(out, leaves, state["in_grads"].double()))


def _exact_turned(feats, state, sign):
    case, pairs = state["case"], state["case"]["pairs"]
    angles = state["pts"].double()[:, state["axes"].long()] * state["freqs"].double()
    turn = torch.polar(torch.ones_like(angles), sign * angles).unsqueeze(1)
    feats = feats.double()
    turned, rest = feats[..., :2 * pairs], feats[..., 2 * pairs:]
    if case["adjacent"]:
        turned = torch.view_as_real(torch.view_as_complex(turned.unflatten(-1, (pairs, 2)).contiguous()) * turn).flatten(-2)
    else:
        both = torch.complex(turned[..., :pairs].contiguous(), turned[..., pairs:].contiguous()) * turn
        turned = torch.cat([both.real, both.imag], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _exact_attention(state):
    case = state["case"]
    heads, key_heads, width = case["heads"], case["key_heads"], case["width"]
    train = case["mode"] == "train"
    names = ("queries", "keys", "values")
    out = torch.zeros(state["queries"].shape, dtype=torch.float64, device=_DEVICE)
    grads = [torch.zeros(state[x].shape, dtype=torch.float64, device=_DEVICE) for x in names] if train else []
    query_starts, key_starts = _starts(state["query_sizes"]), _starts(state["key_sizes"])
    for c in range(case["clouds"]):
        k_rows = slice(key_starts[c], key_starts[c + 1])
        step = max(1, (1 << 26) // max(1, state["key_sizes"][c]))
        live = None if state["key_mask"] is None else state["key_mask"][k_rows]
        for h in range(heads):
            hk = h // (heads // key_heads)
            for lo in range(query_starts[c], query_starts[c + 1], step):
                q_rows = slice(lo, min(lo + step, query_starts[c + 1]))
                leaves = [state["queries"][q_rows, h], state["keys"][k_rows, hk], state["values"][k_rows, hk]]
                q, k, v = leaves = [x.double().requires_grad_(train) for x in leaves]
                if live is not None:
                    if not bool(live.any()):
                        continue
                    k, v = k[live], v[live]
                part = torch.softmax(torch.mm(q, k.t()) / math.sqrt(width), dim=1).mm(v)
                out[q_rows, h] = part.detach()
                if train:
                    dq, dk, dv = torch.autograd.grad(part, leaves, state["in_grads"][q_rows, h].double())
                    grads[0][q_rows, h] = dq
                    grads[1][k_rows, hk] += dk
                    grads[2][k_rows, hk] += dv
    return [out] + grads if train else out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(state)
    if case["kind"] == "rotary":
        out = _exact_turned(state["feats"], state, 1.0)
        return out if case["mode"] == "infer" else [out, _exact_turned(state["in_grads"], state, -1.0)]
    return _exact_attention(state)
