"""Host side of layer norm, rotary positions and attention between levels: what the C ABI refuses before any launch, the
plans the layers make, and that both bindings serve the operators.  No GPU."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import os
    from pccnn_lib_amd import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build(verbose=False)
    return _lib.load()


def test_layer_norm_entry_points_refuse_bad_arguments(lib):
    some = ctypes.c_void_p(16)
    forward = lambda type=0, stride=8, wtype=0, eps=1e-5, n=4, c=8, x=some: lib.pccnn_layer_norm_forward(
        x, type, stride, some, some, wtype, eps, n, c, some, None, None)
    assert forward(type=2) == -2 and b"element types 2" in lib.pccnn_last_error()
    assert forward(wtype=7) == -2
    assert forward(c=0) == -1 and forward(n=-1) == -1 and forward(stride=-8) == -1
    assert forward(eps=-1.0) == -1 and b"eps" in lib.pccnn_last_error()
    assert forward(x=None) == -1 and b"null" in lib.pccnn_last_error()
    assert forward(n=0, x=None) == 0
    backward = lambda dg=some, db=some, ws=None, nbytes=0: lib.pccnn_layer_norm_backward(
        some, 0, 8, some, 0, some, some, 8, 4, 8, some, dg, db, ws, nbytes, None)
    assert backward(db=None) == -1 and b"together" in lib.pccnn_last_error()
    assert backward() == -3 and b"workspace" in lib.pccnn_last_error()
    assert lib.pccnn_layer_norm_workspace_bytes(4, 8) >= 4 * 2 * 8 * 4


def test_rotary_entry_points_refuse_bad_arguments(lib):
    some = ctypes.c_void_p(16)
    turn = lambda type=0, n=4, heads=2, width=8, pairs=4, axes=3, x=some, sn=16: lib.pccnn_rotary(
        x, type, sn, 8, some, some, some, n, heads, width, pairs, axes, 0, 0, some, None)
    assert turn(type=3) == -2
    assert turn(pairs=5) == -1 and turn(heads=0) == -1 and turn(n=-1) == -1 and turn(sn=-1) == -1
    assert turn(axes=0) == -2 and turn(axes=7) == -2 and b"7 axes" in lib.pccnn_last_error()
    assert turn(width=20000, pairs=5000) == -2
    assert turn(x=None) == -1 and turn(n=0, x=None) == 0
    points = lambda axes=3, d=some: lib.pccnn_rotary_points_backward(some, 0, 16, 8, some, some, some, some, 16, 8, 4, 2, 8, 4,
                                                                     axes, 0, d, None)
    assert points(axes=9) == -2 and points(d=None) == -1


def test_attention_entry_points_refuse_bad_arguments(lib):
    from pccnn_lib_amd import _lib

    def problem(**changes):
        p = _lib.Attention()
        p.queries = p.keys = p.values = p.query_starts = p.key_starts = 16
        p.q_stride_n, p.k_stride_n, p.v_stride_n = 64, 32, 32
        p.q_stride_h = p.k_stride_h = p.v_stride_h = 16
        p.m, p.n, p.max_queries, p.max_keys = 10, 20, 10, 20
        p.type, p.clouds, p.heads, p.key_heads, p.width, p.scale = 0, 1, 4, 2, 16, 0.25
        for name, value in changes.items():
            setattr(p, name, value)
        return p

    def forward(out=16, **changes):
        return lib.pccnn_attention_forward(ctypes.byref(problem(**changes)), out, None, None, 0, None)
    assert lib.pccnn_attention_forward(None, 16, None, None, 0, None) == -1
    assert forward(type=5) == -2 and b"element type 5" in lib.pccnn_last_error()
    assert forward(heads=3) == -1 and forward(key_heads=0) == -1 and forward(width=0) == -1
    assert forward(width=129) == -2 and b"head width 129" in lib.pccnn_last_error()
    assert forward(max_keys=21) == -1 and forward(max_queries=-1) == -1 and forward(clouds=-1) == -1
    assert forward(m=1 << 31, max_queries=10) == -2 and forward(n=1 << 31, max_keys=10) == -2
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert forward(scale=scale) == -1 and b"scale" in lib.pccnn_last_error()
    assert forward(k_stride_n=-1) == -1 and forward(keys=None) == -1 and forward(query_starts=None) == -1
    assert forward(out=None) == -1 and b"null" in lib.pccnn_last_error()
    assert forward(out=20) == -1 and b"aligned" in lib.pccnn_last_error()
    assert forward(m=1 << 30, heads=8, key_heads=2) == -2
    assert forward(m=0, max_queries=0, out=None) == 0 and forward(clouds=0, out=None) == 0
    # one query over many keys is split over the keys, which takes a workspace
    long = dict(m=1, max_queries=1, n=1000000, max_keys=1000000, k_stride_n=32)
    assert forward(**long) == -3 and b"workspace" in lib.pccnn_last_error()
    assert lib.pccnn_attention_workspace_bytes(ctypes.byref(problem(**long)), 0) > 2 * 4 * 16 * 4

    def backward(dq=16, dk=16, dv=16, stride=64, **changes):
        return lib.pccnn_attention_backward(ctypes.byref(problem(**changes)), 16, 16, 16, stride, 16, dq, dk, dv, None, 0,
                                            None)
    assert backward(dv=None) == -1 and b"together" in lib.pccnn_last_error()
    assert backward(stride=-1) == -1
    assert backward() == -3 and backward(dq=None, dk=None, dv=None) == 0


def test_every_workspace_size_covers_every_plan_of_the_call(lib):
    # sizes are asked for before the gradient's layout is known: the answer has to do for aligned and unaligned rows
    from pccnn_lib_amd import _lib
    for m, n, clouds in ((1, 500000, 1), (100, 3, 5), (70000, 500, 7), (4096, 4096, 1)):
        p = _lib.Attention()
        p.queries = p.keys = p.values = p.query_starts = p.key_starts = 16
        p.q_stride_n = p.k_stride_n = p.v_stride_n = 64
        p.q_stride_h = p.k_stride_h = p.v_stride_h = 32
        p.m, p.n, p.max_queries, p.max_keys = m, n, -(-m // clouds), -(-n // clouds)
        p.type, p.clouds, p.heads, p.key_heads, p.width, p.scale = 1, clouds, 2, 2, 32, 0.2
        assert lib.pccnn_attention_workspace_bytes(ctypes.byref(p), 1) >= 2 * m * 2 * 4


def test_both_bindings_serve_the_operators_with_the_same_arguments():
    import inspect
    import re
    from pccnn_lib_amd import pccnn_lib_ops as ops
    assert ops.ADDED_NAMES == ("layer_norm", "layer_norm_grads", "rotary", "rotary_grads", "cross_attention",
                               "cross_attention_grads")
    before = ops.use_binding("compiled")
    try:
        for which in ("compiled", "ctypes"):
            ops.use_binding(which)
            z = torch.zeros(4, 8)
            for name, args in (("layer_norm", (z, z[0], z[0])), ("layer_norm_grads", (z, z[0], z, z)),
                               ("rotary", (z[None], z, z[0], z[0])), ("rotary_grads", (z[None], z, z[0], z[0], z[None])),
                               ("cross_attention", (z[None],) * 3 + (z[0], z[0], 1, 1)),
                               ("cross_attention_grads", (z[None],) * 3 + (z[0], z[0], 1, 1) + (z[None],) * 3)):
                assert getattr(ops, name) is ops.BINDINGS[which][name]
                with pytest.raises(RuntimeError, match="GPU tensor"):
                    getattr(ops, name)(*args)
        for name in ops.ADDED_NAMES:
            line = ops.BINDINGS["compiled"][name].__doc__.splitlines()[0]
            inner = line[line.index("(") + 1:line.rindex(")")]
            names = [p.split(":")[0].strip() for p in re.split(r",\s*(?![^\[]*\])", inner) if p]
            python = inspect.signature(ops.BINDINGS["ctypes"][name]).parameters
            assert names == list(python)
    finally:
        ops.use_binding(before)


def test_cloud_ranges_of_ordered_and_mixed_batches():
    import pccnn_lib_amd as lib
    pts = torch.rand(7, 3)
    mixed = lib.pc.CloudRanges(lib.pc.Pointcloud(pts, torch.tensor([1, 0, 0, 1, 3, 3, 0], dtype=torch.int32)), 6)
    assert mixed.starts_.dtype == torch.int32 and mixed.starts_.tolist() == [0, 3, 5, 5, 7, 7, 7]
    assert mixed.longest_ == 3 and mixed.order_.tolist() == [1, 2, 6, 0, 3, 4, 5]
    assert torch.equal(mixed.back(mixed.in_order(pts)), pts)
    ordered = lib.pc.CloudRanges(lib.pc.Pointcloud(pts, torch.tensor([0, 0, 1, 1, 1, 1, 2], dtype=torch.int32)))
    assert ordered.starts_.tolist() == [0, 2, 6, 7] and ordered.order_ is None and ordered.in_order(pts) is pts
    with pytest.raises(RuntimeError, match="2 clouds"):
        lib.pc.CloudRanges(lib.pc.Pointcloud(pts, torch.full((7,), 2, dtype=torch.int32)), 2)


def test_rotary_layer_deals_its_pairs_to_the_axes():
    import pccnn_lib_amd as lib
    layer = lib.pc.layers.RotaryPositions(3, 32, p_unit=0.5, p_base=100.0)
    freqs, axes = layer.plan(torch.device("cpu"))
    assert axes.tolist() == [0] * 6 + [1] * 5 + [2] * 5 and freqs.dtype == torch.float32
    assert abs(float(freqs[0]) - 2.0) < 1e-6 and abs(float(freqs[6 + 4]) - 2.0 * 100.0 ** -0.8) < 1e-6
    layer.to(torch.bfloat16)
    assert layer.plan(torch.device("cpu"))[0].dtype == torch.float32 and not list(layer.parameters())
    with pytest.raises(RuntimeError, match="pairs"):
        lib.pc.layers.RotaryPositions(3, 32, p_pairs=17)
    with pytest.raises(RuntimeError, match="key heads"):
        lib.pc.layers.CrossAttention(3, 8, 8, 4, p_num_key_heads=3)


def test_attention_layer_refuses_ranges_of_other_clouds():
    # before anything is computed, so no GPU is asked: ranges in the wrong order, of another batch, features of another level
    import pccnn_lib_amd as lib
    ids = lambda *counts: torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(counts)])
    coarse, fine = (lib.pc.Pointcloud(torch.rand(sum(c), 3), ids(*c)) for c in ((3, 4), (9, 8)))
    layer = lib.pc.layers.CrossAttention(3, 8, 8, 2)
    ranges = (lib.pc.CloudRanges(coarse), lib.pc.CloudRanges(fine))
    y, x = torch.zeros(7, 8), torch.zeros(17, 8)
    for args, message in (((coarse, fine, y, x, None, ranges[::-1]), "ranges of 17 points, p_pc_in of 7"),
                          ((coarse, fine, y, x, None, (ranges[0], ranges[0])), "ranges of 7 points, p_pc_out of 17"),
                          ((coarse, fine, x, x, None, ranges), "p_in_features of 17 rows"),
                          ((coarse, fine, y, y, None, ranges), "p_out_features of 7 rows"),
                          ((coarse, fine, x, y), "p_in_features of 17 rows")):
        with pytest.raises(RuntimeError, match=message):
            layer(*args)


def test_what_a_layer_keeps_from_serving_can_be_trained_with():
    import pccnn_lib_amd as lib
    pc = lib.pc.Pointcloud(torch.rand(5, 3), torch.tensor([1, 0, 0, 1, 2], dtype=torch.int32))
    with torch.inference_mode():
        layer = lib.pc.layers.RotaryPositions(3, 32)
        kept = list(layer.plan(torch.device("cpu")))
        ranges = lib.pc.CloudRanges(pc)
        kept += [ranges.starts_, ranges.order_, ranges.inverse_]
    assert not any(t.is_inference() for t in kept)
    rows = torch.rand(5, 4, requires_grad=True)
    ranges.back(ranges.in_order(rows)).sum().backward()               # (saves order_ and inverse_)
    assert torch.equal(rows.grad, torch.ones(5, 4))


def test_moving_a_rotary_layer_makes_its_plan_there():
    import pccnn_lib_amd as lib
    layer = torch.nn.Sequential(lib.pc.layers.RotaryPositions(3, 32))
    layer.to("meta")
    freqs, axes = layer[0].plans_[torch.device("meta")]
    assert freqs.dtype == torch.float32 and axes.dtype == torch.int32 and freqs.shape == axes.shape == (16,)
    layer.to(torch.bfloat16)
    assert all(plan[0].dtype == torch.float32 for plan in layer[0].plans_.values()) and not layer.state_dict()


def test_a_problem_that_is_refused_asks_for_no_workspace(lib):
    # the size is asked for before the call: a wrong length must end in the call's message, not in an allocation that fails
    from pccnn_lib_amd import _lib
    p = _lib.Attention()
    p.m, p.n, p.max_queries, p.max_keys = 10, 20, 10, 20
    p.type, p.clouds, p.heads, p.key_heads, p.width, p.scale = 0, 1, 4, 2, 16, 0.25
    good = [lib.pccnn_attention_workspace_bytes(ctypes.byref(p), backward) for backward in (0, 1)]
    assert good[0] >= 256 and good[1] >= 2 * 10 * 4 * 4
    for name, value in (("max_keys", 21), ("max_keys", 1 << 62), ("max_queries", 1 << 62), ("max_queries", -1), ("m", 1 << 40),
                        ("heads", 3), ("width", 129), ("scale", -1.0), ("k_stride_n", -1)):
        before = getattr(p, name)
        setattr(p, name, value)
        assert [lib.pccnn_attention_workspace_bytes(ctypes.byref(p), backward) for backward in (0, 1)] == [256, 256], name
        assert lib.pccnn_attention_forward(ctypes.byref(p), 16, None, None, 0, None) != 0
        setattr(p, name, before)
    assert good == [lib.pccnn_attention_workspace_bytes(ctypes.byref(p), backward) for backward in (0, 1)]


def test_planes_are_made_only_where_a_tiles_rows_are_within_32_bit_offsets(lib):
    # f32 queries enough for planes of the keys: 6 bytes per padded feature of both tensors, unless a tile of 64 keys spans 2^31
    # bytes of a plane (heads x padded width x 2 bytes a key)
    from pccnn_lib_amd import _lib

    def forward_bytes(heads, width, m=4000, n=64):
        p = _lib.Attention()
        p.m, p.n, p.max_queries, p.max_keys = m, n, m, n
        p.type, p.clouds, p.heads, p.key_heads, p.width, p.scale = 0, 1, heads, heads, width, 0.25
        return lib.pccnn_attention_workspace_bytes(ctypes.byref(p), 0)
    for width, padded in ((1, 32), (40, 64), (96, 96), (128, 128)):
        planes = lambda heads: 2 * 6 * 64 * heads * padded
        fits = (1 << 30) // (64 * padded) - 64
        assert planes(8) <= forward_bytes(8, width) < planes(8) + 1024
        assert planes(fits) <= forward_bytes(fits, width) < planes(fits) + 1024
        for heads in ((1 << 30) // (64 * padded), 1 << 19, 1 << 20):
            assert forward_bytes(heads, width) < 1024


def test_layer_norm_asks_for_the_sums_that_it_leaves(lib):
    # 1024 rows of 10^6 channels: few rows of sums, not as many as workgroups could leave of short ones (8 GB)
    size = lib.pccnn_layer_norm_workspace_bytes
    assert size(1 << 20, 1 << 20) <= 1 * 2 * (1 << 20) * 4 + 256
    assert 8 * 5000 * 51 <= size(100000, 5000) <= 8 * 5000 * 64
    assert 8 * 64 * 512 <= size(100000, 64) <= 8 * 64 * 1024 and size(3, 64) >= 8 * 64 * 3
