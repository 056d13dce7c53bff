"""The workspace that the attention entry points ask for is what their plans use: calls through the C ABI with exactly that many
bytes, guards behind them, over types, routes and gradient layouts."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
GUARD = 1 << 16
# Queries and keys of every cloud, clouds, query and key heads, width: few and many own tiles on either side (from 896 rows to a
# cloud on f32 is turned into planes), sides long enough to be cut into parts, odd widths and groups.
PROBLEMS = [(1, 5000, 1, 4, 2, 64), (40, 3000, 2, 4, 4, 32), (3000, 40, 2, 4, 4, 32), (1000, 1000, 1, 2, 2, 96),
            (2000, 100, 1, 3, 1, 33), (100, 2000, 1, 3, 1, 128), (300, 300, 3, 2, 1, 24), (5, 20000, 1, 8, 8, 16),
            (20000, 5, 1, 8, 8, 16), (895, 897, 1, 1, 1, 40), (897, 895, 1, 1, 1, 40)]


@pytest.fixture(scope="module")
def lib():
    from pccnn_lib_amd import _lib
    return _lib.load()


def _rows(count, heads, width, dtype, aligned):
    """[count, heads, width] of random values whose rows start at 16-byte multiples, or anywhere."""
    store = torch.randn((count, heads, (width + 7) // 8 * 8 + (0 if aligned else 1)), device=DEV).to(dtype)
    return store[..., 0 if aligned else 1:][..., :width]


def _call(run, nbytes):
    """``run`` with a workspace of exactly ``nbytes``; the bytes behind it stay as they are."""
    store = torch.full((nbytes + GUARD,), 0xA5, dtype=torch.uint8, device=DEV)
    status = run(ctypes.c_void_p(store.data_ptr()))
    torch.cuda.synchronize()
    assert bool((store[nbytes:] == 0xA5).all())
    return status


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("aligned,grads_aligned", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("problem", PROBLEMS)
def test_calls_do_with_the_workspace_they_ask_for(lib, problem, dtype, aligned, grads_aligned):
    from pccnn_lib_amd import _lib
    m, n, clouds, heads, key_heads, width = problem
    q, g = _rows(m * clouds, heads, width, dtype, aligned), _rows(m * clouds, heads, width, dtype, grads_aligned)
    k, v = (_rows(n * clouds, key_heads, width, dtype, aligned) for _ in range(2))
    starts = [torch.arange(clouds + 1, dtype=torch.int32, device=DEV) * count for count in (m, n)]
    p = _lib.Attention()
    p.queries, p.keys, p.values, p.query_starts, p.key_starts = (t.data_ptr() for t in (q, k, v, *starts))
    p.q_stride_n, p.k_stride_n, p.v_stride_n = (t.stride(0) for t in (q, k, v))
    p.q_stride_h, p.k_stride_h, p.v_stride_h = (t.stride(1) for t in (q, k, v))
    p.m, p.n, p.max_queries, p.max_keys = m * clouds, n * clouds, m, n
    p.type, p.clouds, p.heads, p.key_heads, p.width = int(dtype is torch.bfloat16), clouds, heads, key_heads, width
    p.scale = width ** -0.5
    problem, stream = ctypes.byref(p), torch.cuda.current_stream().cuda_stream
    new = lambda like: torch.full(like.shape, float("nan"), dtype=dtype, device=DEV)
    out, lse = new(q), torch.full((m * clouds, heads), float("nan"), device=DEV)
    nbytes = lib.pccnn_attention_workspace_bytes(problem, 0)
    assert _call(lambda ws: lib.pccnn_attention_forward(problem, out.data_ptr(), lse.data_ptr(), ws, nbytes, stream), nbytes) == 0
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    nbytes = lib.pccnn_attention_workspace_bytes(problem, 1)
    whole = []
    for want_queries, want_keys in ((True, True), (True, False), (False, True)):
        grads = [new(q) if want_queries else None] + [new(k) if want_keys else None for _ in range(2)]
        pointers = [None if t is None else t.data_ptr() for t in grads]
        assert _call(lambda ws: lib.pccnn_attention_backward(problem, out.data_ptr(), lse.data_ptr(), g.data_ptr(), g.stride(0),
                                                             g.stride(1), *pointers, ws, nbytes, stream), nbytes) == 0
        whole = whole or grads
        for a, b in zip(grads, whole):
            assert a is None or (bool(torch.isfinite(a).all()) and torch.equal(a, b))
