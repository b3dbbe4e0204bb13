"""CPU: packing of 8-bit matrices, their rounding, and what the ops refuse."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad


def test_layout_of_a_packed_matrix():
    """Against the layout as the library's header words it."""
    from asrback_amd.linear8 import pack8, unpack8

    g = torch.Generator().manual_seed(0)
    for outputs, inputs in ((1, 1), (17, 160), (40, 256), (33, 65), (16, 64)):
        values = torch.randint(-127, 128, (outputs, inputs), generator=g, dtype=torch.int8)
        scales = torch.rand(outputs, generator=g)
        weight = pack8(values, scales)
        assert weight.packed.shape == (-(-outputs // 16), -(-inputs // 64), 4, 16, 16) and weight.packed.dtype == torch.int8
        whole = torch.zeros(weight.packed.shape[0] * 16, weight.packed.shape[1] * 64, dtype=torch.int8)
        for i, j, part, c in torch.cartesian_prod(*(torch.arange(n) for n in weight.packed.shape[:4])).tolist():
            whole[16 * i + c, 64 * j + 16 * part:64 * j + 16 * part + 16] = weight.packed[i, j, part, c]
        assert torch.equal(whole[:outputs, :inputs], values)
        assert not whole[outputs:].any() and not whole[:, inputs:].any()
        assert torch.equal(unpack8(weight), values.float() * scales[:, None])


def test_rounding():
    from asrback_amd.linear8 import quantize8, unpack8

    g = torch.Generator().manual_seed(1)
    w = torch.randn(20, 100, generator=g)
    w[3] = 0.0
    w[4] *= 1e-30
    w[5, 0] = 50
    for dtype in (torch.float32, torch.bfloat16):
        matrix = w.to(dtype)
        weight = quantize8(matrix)
        assert weight.scales.dtype == dtype
        error = (unpack8(weight).double() - matrix.double()).abs().amax(1)
        # Half a step; a scale rounded to bf16 moves the largest by up to 127 of its 2^-8.
        slack = 0.5 + 1e-4 + (127 * 2.0**-8 if dtype == torch.bfloat16 else 0)
        assert (error <= weight.scales.double() * slack).all()
        assert not unpack8(weight)[3].any()


def test_refusals():
    from asrback_amd import _lib
    from asrback_amd.linear8 import MAX_INPUTS, Linear8, Weight8, gated8, linear8, pack8, quantize8

    values, scales = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for bad, kind, match in (
        ((values.int(), scales), ValueError, "int8"),
        ((values[0], scales), ValueError, "int8"),
        ((values[:0], scales[:0]), ValueError, "at least one"),
        ((values[:, :0], scales), ValueError, "1 to"),
        ((torch.zeros(1, 1, dtype=torch.int8).expand(1, MAX_INPUTS + 1), scales[:1]), ValueError, "1 to"),
        ((values, scales[:7]), ValueError, "scales"),
        ((values, scales[:, None]), ValueError, "scales"),
        ((values, scales.half()), TypeError, "float32 or bfloat16"),
        ((values, scales.to("meta")), RuntimeError, "one device"),
        ((values - 128, scales), ValueError, "-127 .. 127"),
    ):
        with pytest.raises(kind, match=match):
            pack8(*bad)
    with pytest.raises(ValueError, match="matrix"):
        quantize8(torch.zeros(8, 64).half())
    with pytest.raises(ValueError, match="at least one"):
        quantize8(torch.zeros(0, 64))
    for bad in (float("inf"), float("nan")):
        matrix = torch.zeros(8, 64)
        matrix[3, 5] = bad
        with pytest.raises(ValueError, match="infinities"):
            quantize8(matrix)
    weight = pack8(values, scales)
    odd = pack8(values[:7], scales[:7])
    for f in (linear8, gated8):
        with pytest.raises(RuntimeError, match="GPU only"):
            f(torch.zeros(3, 64), weight)
        for x in (torch.zeros(3, 65), torch.zeros(())):
            with pytest.raises(ValueError, match="x must be"):
                f(x, weight)
        with pytest.raises(TypeError, match="scales"):
            f(torch.zeros(3, 64, dtype=torch.bfloat16), weight)
        for bias in (torch.zeros(9), torch.zeros(8, dtype=torch.bfloat16)):
            with pytest.raises(ValueError, match="bias"):
                f(torch.zeros(3, 64), weight, bias)
        with pytest.raises(RuntimeError, match="GPU only"):
            f(torch.zeros(3, 64, requires_grad=True), weight)
    with pytest.raises(ValueError, match="as many gates"):
        gated8(torch.zeros(3, 64), odd)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        Linear8(weight).half()(torch.zeros(3, 64, dtype=torch.float16))
    layer = Linear8(weight)
    assert layer.weight8 == weight and Linear8.from_linear(torch.nn.Linear(64, 8)).bias.shape == (8,)
    # Tensors that are not what the kernel would read.
    for name, bad in (("packed", layer.packed[:, :, :2].contiguous()), ("packed", layer.packed.float()),
                      ("scales", scales[:7]), ("scales", scales.expand(2, 8).t()[:, 0].as_strided((8,), (0,)))):
        layer = Linear8(weight)
        setattr(layer, name, bad)
        for call in (layer, layer.gated):
            with pytest.raises(ValueError, match="packed"):
                call(torch.zeros(3, 64))
    with pytest.raises(ValueError, match="packed"):
        Weight8(weight.packed, weight.scales, 17, 64)

    lib = _lib.load()
    p = _lib.Linear8Params()
    p.rows, p.n, p.k, p.x_row_stride, p.dtype = 40, 8, 64, 64, _lib.BF16

    def refused(code, word):
        assert lib.asrlayer_linear8(bytes(p), 0, 0, None) == code
        assert word in lib.asrattn_last_error()

    refused(_lib.ERR_INVALID, b"non-NULL")
    p.x = p.packed = p.scales = p.out = 4096
    refused(_lib.ERR_WORKSPACE, b"workspace bytes")
    need = lib.asrlayer_linear8_workspace_size(40, 8, 64, 0)
    assert 0 < need < 1 << 16 and lib.asrlayer_linear8_workspace_size(-1, 8, 64, 0) == (1 << 64) - 1
    assert lib.asrlayer_linear8_workspace_size(3, 8, 64, 0) == 0
    assert lib.asrlayer_linear8(bytes(p), 4096, need - 1, None) == _lib.ERR_WORKSPACE
    assert lib.asrlayer_linear8(bytes(p), 4096 + 16, need, None) == _lib.ERR_WORKSPACE
    p.packed = 4104
    refused(_lib.ERR_INVALID, b"aligned")
    for name, value, code in (("n", 0, _lib.ERR_INVALID), ("k", 0, _lib.ERR_INVALID), ("rows", -1, _lib.ERR_INVALID),
                              ("dtype", 7, _lib.ERR_INVALID), ("k", MAX_INPUTS + 1, _lib.ERR_UNSUPPORTED),
                              ("n", (1 << 28) + 1, _lib.ERR_UNSUPPORTED), ("rows", 65535 * 16 + 1, _lib.ERR_UNSUPPORTED)):
        held = getattr(p, name)
        setattr(p, name, value)
        assert lib.asrlayer_linear8(bytes(p), 0, 0, None) == code
        setattr(p, name, held)
    p.n, p.rows = 1 << 28, 65535 * 16
    refused(_lib.ERR_UNSUPPORTED, b"sums")
    p.n, p.gated = 7, 1
    refused(_lib.ERR_INVALID, b"gates")
    assert lib.asrlayer_linear8(None, 0, 0, None) == _lib.ERR_INVALID
    p.gated = p.rows = 0
    assert lib.asrlayer_linear8(bytes(p), 0, 0, None) == _lib.OK


def test_most_outputs_of_few_rows():
    """What a launch could not hold is refused before anything is launched."""
    from asrback_amd import _lib

    lib = _lib.load()
    p = _lib.Linear8Params()
    p.k, p.x_row_stride, p.dtype = 1, 1, _lib.BF16
    p.x = p.packed = p.scales = p.out = 4096
    for rows, n, gated, taken in ((1, (1 << 27) - 16, 0, True), (32, (1 << 27) - 15, 0, False), (1, 1 << 28, 0, False),
                                  (5, (1 << 28) - 32, 1, True), (5, (1 << 28) - 30, 1, False), (33, 1 << 28, 0, True)):
        p.rows, p.n, p.gated = rows, n, gated
        # (Enough of a workspace, but misaligned: what the sizes allow is refused for that.)
        code = lib.asrlayer_linear8(bytes(p), 4096 + 16, 1 << 40, None)
        assert code == (_lib.ERR_WORKSPACE if taken else _lib.ERR_UNSUPPORTED)
        assert (b"aligned" if taken else b"2^27 outputs") in lib.asrattn_last_error()


def test_tensors_that_change_after_a_weight_is_made(monkeypatch):
    """A weight keeps the memory that its tensors had: a call hands that to the kernel."""
    import copy
    import pickle

    from asrback_amd import linear8 as module
    from asrback_amd.linear8 import Weight8, gated8, linear8, pack8

    seen = []
    monkeypatch.setattr(module, "_product", lambda what, x, packed, scales, *args: seen.append((packed, scales)))
    for name in ("packed", "scales"):
        for change in (lambda t: t.set_(torch.zeros(1, dtype=t.dtype)), lambda t: t.resize_(1),
                       lambda t: setattr(t, "data", torch.zeros(1, dtype=t.dtype))):
            weight = pack8(torch.full((8, 64), 3, dtype=torch.int8), torch.ones(8))
            held = [t.clone() for t in (weight.packed, weight.scales)]
            change(getattr(weight, name))
            for f in (linear8, gated8):
                f(torch.zeros(3, 64), weight)
                assert all(torch.equal(a, b) for a, b in zip(seen.pop(), held))
    weight = pack8(torch.zeros(8, 64, dtype=torch.int8), torch.ones(8))
    for twin in (copy.deepcopy(weight), pickle.loads(pickle.dumps(weight))):
        assert isinstance(twin, Weight8) and (twin.outputs, twin.inputs) == (8, 64)
        assert all(a.data_ptr() == b.data_ptr() for a, b in zip(twin._held, (twin.packed, twin.scales)))
        assert twin.packed.data_ptr() != weight.packed.data_ptr()


def test_scales_that_require_a_gradient():
    from asrback_amd.linear8 import Linear8, Weight8, gated8, linear8, pack8

    held = pack8(torch.zeros(8, 64, dtype=torch.int8), torch.ones(8))
    weight = Weight8(held.packed, held.scales.clone().requires_grad_(), 8, 64)
    layer, x = Linear8(held), torch.zeros(3, 64)
    layer.scales = weight.scales
    for name, call in (("linear8", lambda: linear8(x, weight)), ("gated8", lambda: gated8(x, weight)),
                       ("linear8", lambda: layer(x)), ("gated8", lambda: layer.gated(x))):
        with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("gated", [False, True])
def test_out(gated):
    from asrback_amd.linear8 import gated8, linear8, pack8

    weight = pack8(torch.zeros(128 if gated else 64, 64, dtype=torch.int8), torch.ones(128 if gated else 64))
    arena = torch.zeros(16, 64)
    x, bias = arena[:4], arena[10:12].view(-1)[: weight.outputs]
    good = torch.zeros(4, 64)

    def call(out):
        return (gated8 if gated else linear8)(x, weight, bias, out=out)

    with pytest.raises(RuntimeError, match="GPU only"):
        call(good)
    for out in (x, arena[3:7], arena[8:12], weight.packed.view(-1).view(torch.float32)[:256].view(4, 64)):
        with pytest.raises(ValueError, match="shares memory"):
            call(out)
    for out in (good[:3], good.double(), good.t().contiguous().t(), torch.zeros(4, 128)[:, :64]):
        with pytest.raises(ValueError, match="contiguous"):
            call(out)
    with pytest.raises(RuntimeError, match="no gradient"):
        call(torch.zeros(4, 64, requires_grad=True))
    with torch.inference_mode():
        held = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="inference"):
        call(held)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        call(forward_ad.make_dual(good, good + 1))


def test_quantize_linears8():
    """Every place of a layer; hooked ones and wide ones stay; all or none."""
    from asrback_amd.linear8 import MAX_INPUTS, Linear8, quantize_linears8

    model, inner = torch.nn.Module(), torch.nn.Module()
    model.a = model.b = inner.c = torch.nn.Linear(60, 8)
    model.inner, model.none = inner, None
    inner.wide = torch.nn.Linear(MAX_INPUTS + 1, 1)
    inner.hooked = torch.nn.Linear(8, 8)
    seen = []
    inner.hooked.register_forward_hook(lambda m, x, y: seen.append("forward"))
    inner.own = torch.nn.Linear(8, 8)
    inner.own.forward = lambda x: x
    assert quantize_linears8(model) == 1
    assert type(model.a) is Linear8 and model.a is model.b is inner.c
    assert all(type(m) is torch.nn.Linear for m in (inner.wide, inner.hooked, inner.own))
    inner.hooked(torch.zeros(1, 8))
    assert seen == ["forward"] and quantize_linears8(model) == 0
    model = torch.nn.Sequential(torch.nn.Linear(64, 8), torch.nn.Linear(8, 8))
    with torch.no_grad():
        model[1].weight[3, 5] = float("inf")
    with pytest.raises(ValueError):
        quantize_linears8(model)
    assert all(type(m) in (torch.nn.Linear, torch.nn.Sequential) for m in model.modules())
    # State dicts carry the matrix.
    layer, other = (Linear8.from_linear(torch.nn.Linear(70, 9)) for _ in "ab")
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other.packed, layer.packed) and torch.equal(other.scales, layer.scales)
    assert "in_features=70, out_features=9" in repr(layer)
