"""f32 attention of one head in 64 bits, and the arithmetic of its kernels on the CPU with a choice of what a product leaves
out: what the accuracy that the GPU tests ask for is derived from (test_attention_f32.py)."""
import torch

# Queries, keys, width and spread of the queries.  From 896 rows (keys) of a cloud on, what they walk becomes planes of terms;
# fewer walk it through registers: both, in each direction.
CASES = [(queries, keys, width, spread) for queries, keys in ((100, 130), (1900, 120), (90, 1900), (1900, 1850))
         for width, spread in ((32, 1.5), (32, 4.0), (64, 4.0), (96, 1.5), (128, 4.0))]
NAMES = ("out", "lse", "d_queries", "d_keys", "d_values")
# The largest error of a result in the 2-norm, as a share of the result's.  Three bf16 terms to a value and six products to a
# product leave 2^-23 of each product out; a sum of n products adds sqrt(n) roundings of 2^-24 or less, n up to 750 here: 2^-20.
# The probabilities carry the scores' errors, absolute ones, and the gradients the differences of dP - D: with the spreads below
# the whole arithmetic with f32 sums in another order gives 2^-20.1 (out 2^-20.4, lse 2^-23.7), and a product that lacks a term
# of one of its factors 2^-18.8 or more (test_attention_f32.py shows both).
MOST = dict(out=2.0 ** -19.2, lse=2.0 ** -22.7, d_queries=2.0 ** -18.9, d_keys=2.0 ** -18.9, d_values=2.0 ** -19)


def inputs(queries, keys, width, spread, seed=0):
    """(queries, keys, values, gradient of the output) of one head."""
    gen = torch.Generator().manual_seed(queries + 3 * keys + width + 7 * seed)
    normal = lambda n: torch.randn((n, width), generator=gen)
    return normal(queries) * spread, normal(keys), normal(keys), normal(queries)


def exact(q, k, v, g):
    """(out, lse, d_queries, d_keys, d_values) in 64 bits."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    scale = q.shape[1] ** -0.5
    s = scale * q @ k.t()
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    out = p @ v
    ds = p * (g @ v.t() - (g * out).sum(1, keepdim=True))
    return out, lse, scale * ds @ k, scale * ds.t() @ q, p.t() @ g


def off(got, want):
    """Error of every result in the 2-norm, by name."""
    return {name: float((a.double().cpu() - b).norm() / b.norm()) for name, a, b in zip(NAMES, got, want)}


def terms(x, count):
    out, rest = [], x
    for _ in range(count):
        out.append(rest.to(torch.bfloat16).float())
        rest = rest - out[-1]
    return out


def product(a, b, kept):
    """a b^T of f32 sums, a and b as ``kept`` = (terms of a, terms of b): the products whose terms' indices add up to less than
    the larger count, smallest first."""
    x, y = terms(a, kept[0]), terms(b, kept[1])
    total = torch.zeros((a.shape[0], b.shape[0]))
    for order in range(max(kept) - 1, -1, -1):
        for i in range(order, -1, -1):
            if i < kept[0] and order - i < kept[1]:
                total = total + x[i] @ y[order - i].t()
    return total


FULL = (3, 3)


def emulated(q, k, v, g, scores=FULL, dots=FULL, forward=FULL, queries=FULL, keys=FULL, values=FULL):
    """The kernels' results; the terms that the products of S, dP, O, dq, dk and dv keep of either factor."""
    scale = q.shape[1] ** -0.5
    t = lambda x: x.t().contiguous()
    s = product(q, k, scores) * scale
    top = s.amax(1, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(1, keepdim=True)
    out, lse = product(p, t(v), forward) / total, top + torch.log(total)
    p = torch.exp(s - lse)
    ds = p * (product(g, v, dots) - (g * out).sum(1, keepdim=True))
    return (out, lse[:, 0], scale * product(ds, t(k), queries), scale * product(t(ds), t(q), keys),
            product(t(p), t(g), values))
