"""CPU: packing of 4-bit matrices, their rounding, and what the ops refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch


def test_layout_of_a_packed_matrix():
    """Against the layout as the library's header words it."""
    from asrback_amd.linear4 import pack4, unpack4

    g = torch.Generator().manual_seed(0)
    for outputs, inputs, group in ((1, 32, 32), (17, 160, 32), (40, 256, 128), (33, 192, 64)):
        values = torch.randint(0, 16, (outputs, inputs), generator=g, dtype=torch.uint8)
        scales = torch.rand(outputs, inputs // group, generator=g)
        zeros = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8)
        weight = pack4(values, scales, zeros)
        blocks_n, blocks_k = -(-outputs // 16), -(-inputs // 128)
        assert weight.packed.shape == (blocks_n, blocks_k, 64, 4) and weight.packed.dtype == torch.int32
        assert weight.scales.shape == (blocks_n, blocks_k, 4, 128 // group, 4)
        assert weight.zeros.shape == (blocks_n, blocks_k, 4, 128 // group, 2)
        order = (0, 2, 4, 6, 1, 3, 5, 7)
        for n, k in torch.stack((torch.randint(0, outputs, (60,), generator=g),
                                 torch.randint(0, inputs, (60,), generator=g)), 1).tolist():
            block, s, lane_group, j = k // 128, k % 128 // 32, k % 32 // 8, k % 8
            word = int(weight.packed[n // 16, block, 16 * lane_group + n % 16, s])
            assert word >> 4 * order.index(j) & 15 == int(values[n, k])
            at = n // 16, block, n % 16 // 4, k % 128 // group
            assert weight.scales[at][n % 4] == scales[n, k // group]
            assert int(weight.zeros[at][n % 4 // 2]) >> 4 * (n % 2) & 15 == int(zeros[n, k // group])
        whole = (values.float().view(outputs, -1, group) - zeros.float()[..., None]) * scales[..., None]
        assert torch.equal(unpack4(weight), whole.flatten(1))
        plain = pack4(values, scales)
        assert plain.zeros is None
        assert torch.equal(unpack4(plain), ((values.float().view(outputs, -1, group) - 8) * scales[..., None]).flatten(1))


def test_rounding():
    from asrback_amd.linear4 import quantize4, unpack4

    g = torch.Generator().manual_seed(1)
    w = torch.randn(20, 256, generator=g)
    w[3, :64] = 0.0
    w[4, 64:128] = w[4, 64:128].abs() + 5
    for dtype in (torch.float32, torch.bfloat16):
        matrix = w.to(dtype)
        for symmetric in (True, False):
            weight = quantize4(matrix, 64, symmetric)
            assert weight.scales.dtype == dtype
            back = unpack4(weight).view(20, 4, 64)
            steps = weight.scales.permute(0, 2, 4, 1, 3).reshape(32, 4)[:20].float()
            # Half a step; with a zero point, which is rounded to a step as well, one.
            # The scale, rounded to bf16 (2^-8), moves the ends by 7 or 15 of its own.
            slack = (0.5 if symmetric else 1.0) + (15 * 2**-8 if dtype == torch.bfloat16 else 1e-4)
            error = (back - matrix.float().view(20, 4, 64)).abs().amax(-1)
            assert (error <= steps * slack).all()
            assert not back[3, 0].any()


def test_refusals():
    from asrback_amd import _lib
    from asrback_amd.linear4 import Linear4, linear4, pack4, quantize4

    values = torch.zeros(8, 64, dtype=torch.uint8)
    scales = torch.ones(8, 2)
    for bad, kind, match in (
        ((values.int(), scales), ValueError, "uint8"),
        ((values[0], scales), ValueError, "uint8"),
        ((values, scales[:7]), ValueError, "scales"),
        ((values, torch.ones(8, 3)), ValueError, "scales"),
        ((values, torch.ones(8, 4)), ValueError, "group 16"),
        ((values, scales.half()), TypeError, "float32 or bfloat16"),
        ((values, scales, scales), ValueError, "zeros"),
        ((values + 16, scales), ValueError, "0 .. 15"),
        ((values, scales, torch.full((8, 2), 16, dtype=torch.uint8)), ValueError, "0 .. 15"),
    ):
        with pytest.raises(kind, match=match):
            pack4(*bad)
    with pytest.raises(ValueError, match="whole|multiple"):
        quantize4(torch.zeros(8, 100), 64)
    with pytest.raises(ValueError, match="group"):
        quantize4(torch.zeros(8, 96), 48)
    with pytest.raises(ValueError, match="matrix"):
        quantize4(torch.zeros(8, 64).half(), 64)
    for bad in (float("inf"), float("nan")):
        matrix = torch.zeros(8, 64)
        matrix[3, 5] = bad
        for symmetric in (True, False):
            with pytest.raises(ValueError, match="infinities"):
                quantize4(matrix, 64, symmetric)
    weight = pack4(values, scales)
    with pytest.raises(RuntimeError, match="GPU only"):
        linear4(torch.zeros(3, 64), weight)
    with pytest.raises(ValueError, match="x must be"):
        linear4(torch.zeros(3, 65), weight)
    with pytest.raises(TypeError, match="scales"):
        linear4(torch.zeros(3, 64, dtype=torch.bfloat16), weight)
    with pytest.raises(ValueError, match="bias"):
        linear4(torch.zeros(3, 64), weight, torch.zeros(9))
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        Linear4(weight).half()(torch.zeros(3, 64, dtype=torch.float16))
    layer = Linear4(weight)
    assert layer.weight4 == weight
    # Buffers that are not what the kernel would read.
    matrix = pack4(torch.zeros(40, 300 * 32, dtype=torch.uint8), torch.ones(40, 300))
    assert matrix.packed.shape[:2] == (3, 75)
    for name, bad in (("packed", layer.packed[:, :, :32].contiguous()), ("packed", layer.packed.float()),
                      ("scales", layer.scales[..., :2].contiguous()), ("zeros", torch.zeros(3, dtype=torch.uint8))):
        layer = Linear4(weight)
        setattr(layer, name, bad)
        with pytest.raises(ValueError, match="packed"):
            layer(torch.zeros(3, 64))
    wide = Linear4(matrix)
    wide.packed = wide.packed.to(memory_format=torch.channels_last)
    assert not wide.packed.is_contiguous()
    with pytest.raises(ValueError, match="packed"):
        wide(torch.zeros(3, 9600))

    lib = _lib.load()
    p = _lib.Linear4Params()
    p.rows, p.n, p.k, p.group, p.dtype = 3, 8, 64, 32, _lib.BF16
    assert lib.asrlayer_linear4(ctypes.byref(p), None) == _lib.ERR_INVALID
    assert b"non-NULL" in lib.asrattn_last_error()
    p.x = p.packed = p.scales = p.out = 4096
    p.x_row_stride = 60
    assert lib.asrlayer_linear4(ctypes.byref(p), None) == _lib.ERR_INVALID
    p.group = 16
    assert lib.asrlayer_linear4(ctypes.byref(p), None) == _lib.ERR_UNSUPPORTED
    p.group, p.k = 64, 96
    assert lib.asrlayer_linear4(ctypes.byref(p), None) == _lib.ERR_INVALID
    p.k, p.x_row_stride, p.rows = 128, 128, 65535 * 16 + 1
    assert lib.asrlayer_linear4(ctypes.byref(p), None) == _lib.ERR_UNSUPPORTED
    p.rows = 0
    assert lib.asrlayer_linear4(ctypes.byref(p), None) == _lib.OK


def test_tensors_that_change_after_a_weight_is_made(monkeypatch):
    """A weight keeps the memory that its tensors had: a call hands that to the kernel."""
    import copy
    import pickle

    from asrback_amd import linear4 as module
    from asrback_amd.linear4 import Weight4, linear4, pack4

    seen = []
    monkeypatch.setattr(module, "_product", lambda x, packed, scales, zeros, *args: seen.append((packed, scales, zeros)))
    values, zeros = torch.full((8, 64), 3, dtype=torch.uint8), torch.full((8, 2), 5, dtype=torch.uint8)
    for name in ("packed", "scales", "zeros"):
        for change in (lambda t: t.set_(torch.zeros(1, dtype=t.dtype)), lambda t: t.resize_(1),
                       lambda t: setattr(t, "data", torch.zeros(1, dtype=t.dtype))):
            weight = pack4(values, torch.ones(8, 2), zeros)
            held = [t.clone() for t in (weight.packed, weight.scales, weight.zeros)]
            change(getattr(weight, name))
            linear4(torch.zeros(3, 64), weight)
            assert all(torch.equal(a, b) for a, b in zip(seen.pop(), held))
    for weight in (pack4(values, torch.ones(8, 2), zeros), pack4(values, torch.ones(8, 2))):
        for twin in (copy.deepcopy(weight), pickle.loads(pickle.dumps(weight))):
            assert isinstance(twin, Weight4) and (twin.outputs, twin.inputs, twin.group) == (8, 64, 32)
            assert twin._held[0].data_ptr() == twin.packed.data_ptr() != weight.packed.data_ptr()
            assert (twin._held[2] is None) == (weight.zeros is None)


def test_scales_that_require_a_gradient():
    from asrback_amd.linear4 import Linear4, Weight4, linear4, pack4

    held = pack4(torch.zeros(8, 64, dtype=torch.uint8), torch.ones(8, 2))
    weight = Weight4(held.packed, held.scales.clone().requires_grad_(), None, 8, 64, 32)
    layer, x = Linear4(held), torch.zeros(3, 64)
    layer.scales = weight.scales
    for call in (lambda: linear4(x, weight), lambda: layer(x)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_quantize_linears_replaces_every_name():
    """A layer under two names of one parent, and under another parent, is rounded once
    and stays shared."""
    from asrback_amd.linear4 import Linear4, quantize_linears

    model, inner = torch.nn.Module(), torch.nn.Module()
    model.a = model.b = inner.c = torch.nn.Linear(64, 8)
    model.inner, model.none = inner, None
    model.register_module("absent", None)
    inner.other = torch.nn.Linear(64, 8, bias=False)
    inner.narrow = torch.nn.Linear(8, 4)
    assert quantize_linears(model, 32) == 2
    assert type(model.a) is Linear4 and model.a is model.b is inner.c
    assert type(inner.other) is Linear4 and type(inner.narrow) is torch.nn.Linear and model.absent is None


def test_quantize_linears_leaves_what_is_hooked():
    """Layers with hooks of any kind or a forward of their own go on running them."""
    from asrback_amd.linear4 import Linear4, quantize_linears

    model = torch.nn.Sequential(*(torch.nn.Linear(64, 64) for _ in range(8)))
    seen = []
    model[0].register_forward_hook(lambda m, x, y: seen.append("forward"))
    model[1].register_forward_pre_hook(lambda m, x: seen.append("pre"))
    model[2].register_full_backward_hook(lambda m, x, y: None)
    model[3].forward = lambda x: seen.append("own") or x
    model[4].register_state_dict_post_hook(lambda *a: None)
    torch.nn.utils.parametrizations.weight_norm(model[5])
    model[6].register_load_state_dict_post_hook(lambda *a: None)
    kept = list(model)[:7]
    assert quantize_linears(model, 64) == 1
    assert type(model[7]) is Linear4 and all(a is b for a, b in zip(model, kept))
    torch.nn.Sequential(*kept)(torch.zeros(2, 64))
    assert seen == ["forward", "pre", "own"]


def test_quantize_linears_replaces_all_or_none():
    """A matrix that cannot be rounded leaves the whole model as it was."""
    from asrback_amd.linear4 import quantize_linears

    for bad in (torch.nn.Linear(64, 8).half(), torch.nn.Linear(64, 8)):
        model = torch.nn.Sequential(torch.nn.Linear(64, 8), torch.nn.Sequential(bad))
        if bad.weight.dtype == torch.float32:
            with torch.no_grad():
                bad.weight[3, 5] = float("inf")
        with pytest.raises(ValueError):
            quantize_linears(model, 64)
        assert all(type(m) in (torch.nn.Linear, torch.nn.Sequential) for m in model.modules())
