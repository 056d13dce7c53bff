"""Host side of the feed-forward operators: what the C ABI refuses before any launch, workspace sizes, both bindings, the layers'
plans.  No GPU."""
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


SOME = ctypes.c_void_p(16)


def test_rms_norm_entry_points_refuse_bad_arguments(lib):
    def forward(type=0, stride=8, residual=None, rstride=8, wtype=0, eps=1e-6, n=4, c=8, x=SOME, total=None, out=SOME):
        return lib.pccnn_rms_norm_forward(x, type, stride, residual, rstride, SOME, wtype, eps, n, c, out, total, None, None)
    assert forward(type=2) == -2 and b"element types 2" in lib.pccnn_last_error()
    assert forward(wtype=7) == -2
    assert forward(c=0) == -1 and forward(n=-1) == -1 and forward(stride=-8) == -1
    assert forward(eps=-1.0) == -1 and forward(eps=float("nan")) == -1 and b"eps" in lib.pccnn_last_error()
    assert forward(x=None) == -1 and forward(out=None) == -1 and b"null" in lib.pccnn_last_error()
    assert forward(residual=SOME) == -1 and b"together" in lib.pccnn_last_error()
    assert forward(total=SOME) == -1 and forward(residual=SOME, total=SOME, rstride=-1) == -1
    assert forward(n=0, x=None) == 0

    def codes(type=0, residual=None, n=4, c=8, x=SOME, codes=SOME, scales=SOME, total=None, eps=1e-6):
        return lib.pccnn_rms_norm_8bit(x, type, 8, residual, 8, SOME, 0, eps, n, c, codes, scales, total, None)
    assert codes(type=2) == -2 and codes(eps=-1.0) == -1 and codes(codes=None) == -1 and codes(scales=None) == -1
    assert codes(residual=SOME) == -1 and codes(codes=20) == -1 and b"aligned" in lib.pccnn_last_error()
    assert codes(n=0, x=None) == 0
    quantize = lambda type=0, n=4, c=8, stride=8, codes=SOME: lib.pccnn_quantize_rows(  # noqa: E731
        SOME, type, stride, n, c, codes, SOME, None)
    assert quantize(type=3) == -2 and quantize(c=0) == -1 and quantize(stride=-1) == -1 and quantize(codes=None) == -1
    assert quantize(n=0) == 0

    def backward(type=0, rstd=SOME, grads=SOME, total_grads=None, tstride=8, d_feats=SOME, d_gamma=SOME, n=4, ws=None, size=0):
        return lib.pccnn_rms_norm_backward(SOME, type, 8, SOME, 0, rstd, grads, 8, total_grads, tstride, n, 8, d_feats, d_gamma, ws,
                                           size, None)
    assert backward(type=2) == -2 and backward(rstd=None) == -1 and backward(grads=None) == -1
    assert backward(total_grads=SOME, tstride=-8) == -1
    assert backward() == -3 and b"workspace" in lib.pccnn_last_error()
    assert backward(d_feats=None, d_gamma=None) == 0 and backward(n=0, d_gamma=None) == 0
    assert lib.pccnn_rms_norm_workspace_bytes(4, 8) >= 4 * 8 * 4
    assert lib.pccnn_rms_norm_workspace_bytes(100000, 64) <= 512 * 64 * 4
    assert lib.pccnn_rms_norm_workspace_bytes(1 << 20, 1 << 20) <= 4 * (1 << 20) + 256


def test_linear_8bit_refuses_bad_arguments(lib):
    def call(n=4, inner=16, outer=8, type=0, x=SOME, s=SOME, w=SOME, ws=SOME, out=SOME, work=None, size=0):
        return lib.pccnn_linear_8bit(x, s, w, ws, None, n, inner, outer, out, type, work, size, None)
    assert call(type=2) == -2 and b"result type 2" in lib.pccnn_last_error()
    assert call(n=-1) == -1 and call(inner=0) == -1 and call(outer=0) == -1
    assert call(inner=131072) == -2 and b"131072 products" in lib.pccnn_last_error()
    assert call(outer=(1 << 20) + 1) == -2 and call(n=1 << 31) == -2
    assert call(x=None) == -1 and call(s=None) == -1 and call(w=None) == -1 and call(ws=None) == -1 and call(out=None) == -1
    assert call(out=24) == -1 and b"aligned" in lib.pccnn_last_error()
    assert call(n=0, x=None) == 0
    assert call(n=100, inner=17) == -3 and b"workspace" in lib.pccnn_last_error()
    size = lib.pccnn_linear_8bit_workspace_bytes
    assert size(SOME, SOME, 100, 32, 8) == 256 and size(SOME, SOME, 4, 17, 8) == 256
    assert size(SOME, SOME, 100, 17, 8) >= 108 * 32 and size(ctypes.c_void_p(17), SOME, 100, 32, 8) >= 100 * 32
    assert size(SOME, SOME, 100, 131072, 8) == size(SOME, SOME, -1, 1, 1) == 256


def _problem(**changes):
    from pccnn_lib_amd import _lib
    p = _lib.Gated()
    p.feats = p.gate = p.up = p.feats_scales = p.gate_scales = p.up_scales = 16
    p.feats_stride = p.gate_stride = p.up_stride = 32
    p.n, p.channels, p.hidden, p.type, p.activation = 100, 32, 48, 1, 0
    for name, value in changes.items():
        setattr(p, name, value)
    return p


def test_gated_entry_points_refuse_bad_arguments(lib):
    def forward(out=16, out_type=None, work=None, size=0, **changes):
        p = _problem(**changes)
        return lib.pccnn_gated_forward(ctypes.byref(p), out, p.type if out_type is None else out_type, work, size, None)
    assert lib.pccnn_gated_forward(None, 16, 0, None, 0, None) == -1
    assert forward(type=3) == -2 and b"element type 3" in lib.pccnn_last_error()
    assert forward(activation=4) == -2 and forward(activation=-1) == -2 and b"activation -1" in lib.pccnn_last_error()
    assert forward(n=-1) == -1 and forward(channels=0) == -1 and forward(hidden=0) == -1 and forward(gate_stride=-1) == -1
    assert forward(hidden=(1 << 20) + 1) == -2 and forward(n=1 << 31) == -2
    assert forward(type=2, channels=131072, out_type=0) == -2 and b"8-bit products" in lib.pccnn_last_error()
    assert forward(out_type=0) == -2 and forward(type=2, out_type=2) == -2 and b"result type 2" in lib.pccnn_last_error()
    assert forward(feats=None) == -1 and forward(up=None) == -1 and forward(out=None) == -1
    assert forward(type=2, out_type=0, gate_scales=None) == -1 and b"scales" in lib.pccnn_last_error()
    assert forward(out=24) == -1 and b"aligned" in lib.pccnn_last_error()
    assert forward(n=0, feats=None, out=None) == 0
    assert forward(type=0) == -3 and forward(channels=31) == -3 and forward(gate=18) == -3

    def backward(grads=16, stride=48, dx=16, dg=16, du=16, work=None, size=0, **changes):
        return lib.pccnn_gated_backward(ctypes.byref(_problem(**changes)), grads, stride, dx, dg, du, work, size, None)
    assert backward(type=2) == -2 and b"no gradients" in lib.pccnn_last_error()
    assert backward(du=None) == -1 and b"together" in lib.pccnn_last_error()
    assert backward(stride=-1) == -1 and backward(grads=None) == -1 and backward(dx=24) == -1 and backward(dg=20) == -1
    assert backward() == -3 and backward(dx=None, dg=None, du=None) == 0 and backward(n=0, dg=None, du=None) == 0


def test_gated_gradients_refuse_weights_of_more_values_than_a_launch_has(lib):
    def backward(channels, hidden):
        p = _problem(channels=channels, hidden=hidden, feats_stride=channels, gate_stride=channels, up_stride=channels)
        return lib.pccnn_gated_backward(ctypes.byref(p), 16, hidden, 16, 16, 16, None, 0, None)
    assert backward(1 << 16, 1 << 15) == -2 and b"65536 (2^31 - 1" in lib.pccnn_last_error()
    assert backward((1 << 16) - 1, 1 << 15) == -3


def test_products_refuse_more_workgroups_than_a_launch_has(lib):
    # 2^24 tiles of 128 rows, 256 threads each
    out = lib.pccnn_linear_8bit(SOME, SOME, SOME, SOME, None, (1 << 31) - 1, 16, 16, SOME, 0, None, 0, None)
    assert out == -2 and b"16777216 workgroups" in lib.pccnn_last_error()


def test_gated_workspace_covers_what_is_laid_out(lib):
    size = lambda backward=0, **changes: lib.pccnn_gated_workspace_bytes(ctypes.byref(_problem(**changes)), backward)  # noqa: E731
    assert size() == 256 and size(n=5, type=0) == 256
    assert size(type=0) >= 6 * 32 * (100 + 2 * 48) and size(channels=31) >= 2 * 32 * (100 + 2 * 48)
    assert size(feats=18) >= 2 * 32 * 100 and size(feats_stride=36) >= 2 * 32 * 100 and size(feats_stride=1 << 30) >= 2 * 32 * 100
    # gradients of the projections, turned weights, at least one part of the weights' gradients
    assert size(1) >= 2 * 100 * 2 * 48 + 2 * 32 * 2 * 48 + 4 * 2 * 48 * 32
    assert size(1, type=0) >= 6 * 32 * (100 + 2 * 48) + 6 * 100 * 2 * 48 + 6 * 32 * 2 * 48 + 4 * 2 * 48 * 32
    for bad in (dict(type=3), dict(n=-1), dict(hidden=1 << 21), dict(n=1 << 40), dict(activation=9)):
        assert size(**bad) == size(1, **bad) == 256


def test_both_bindings_serve_the_operators_with_the_same_arguments():
    import inspect
    import re
    from pccnn_lib_amd import pccnn_lib_ops as ops
    assert ops.FEED_FORWARD_NAMES == ("rms_norm", "rms_norm_grads", "rms_norm_8bit", "quantize_rows", "linear_8bit", "gated_linear",
                                      "gated_linear_grads", "gated_linear_8bit")
    before = ops.use_binding("compiled")
    try:
        for which in ("compiled", "ctypes"):
            ops.use_binding(which)
            z, q = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int8)
            for name, args in (("rms_norm", (z, z[0])), ("rms_norm_grads", (z, z[0], z[0], z)), ("rms_norm_8bit", (z, z[0])),
                               ("quantize_rows", (z,)), ("linear_8bit", (q, z[0], q, z[0])), ("gated_linear", (z, z, z)),
                               ("gated_linear_grads", (z, z, z, z)), ("gated_linear_8bit", (q, z[0], q, z[0], q, z[0]))):
                assert getattr(ops, name) is ops.BINDINGS[which][name]
                with pytest.raises(RuntimeError, match="GPU tensor"):
                    getattr(ops, name)(*args)
        for name in ops.FEED_FORWARD_NAMES:
            line = ops.BINDINGS["compiled"][name].__doc__.splitlines()[0]
            inner = line[line.index("(") + 1:line.rindex(")")]
            names = [p.split(":")[0].strip() for p in re.split(r",\s*(?![^\[]*\])", inner) if p]
            assert names == list(inspect.signature(ops.BINDINGS["ctypes"][name]).parameters)
    finally:
        ops.use_binding(before)


def test_feed_forward_layers_plan_their_sizes():
    import pccnn_lib_amd as lib
    layer = lib.pc.layers.GatedFeedForward(96)
    assert layer.hidden_ == 256 and layer.hidden_ % 8 == 0
    assert set(layer.state_dict()) == {"norm_.gamma_", "gate_.weight", "up_.weight", "down_.weight", "down_.bias"}
    assert tuple(layer.gate_.weight.shape) == (256, 96) and tuple(layer.norm_.gamma_.shape) == (1, 96)
    assert lib.pc.layers.GatedFeedForward(100).hidden_ == 272 and lib.pc.layers.GatedFeedForward(100, 33).hidden_ == 33
    with pytest.raises(RuntimeError, match="activation"):
        lib.pc.layers.GatedFeedForward(96, p_activation="tanh")
    with pytest.raises(RuntimeError, match="hidden"):
        lib.pc.layers.GatedFeedForward(96, 0)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lib.pc.layers.GatedFeedForward8Bit(layer)
