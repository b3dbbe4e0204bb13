"""GPU: linear layers with 4-bit weights.

Integers and powers of two make every sum exact in float32, so those cases ask
for the exact result, rounded once.  Real values are held to what the kernel
rounds: the result once (2^-8 of it in bf16, 2^-24 in float32), and its float32
sums: per output at most 2^-24 c sum |x| |scale| times the values an operand and
its offset reach (bf16: 2 x 143, float32: 2 x 15), c the additions on a value's way
(twice the group's, in float32, whose x goes in three parts, four times; one a group,
the waves').
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def say(*args):
    print(*args, flush=True)


def quantized(outputs, inputs, group, zeros, dtype, g, powers=False):
    values = torch.randint(0, 16, (outputs, inputs), generator=g, dtype=torch.uint8)
    shape = (outputs, inputs // group)
    if powers:
        scales = 2.0 ** -torch.randint(0, 4, shape, generator=g).float()
    else:
        scales = torch.rand(shape, generator=g) * 0.02 + 0.01
    points = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8) if zeros else None
    return values, scales.to(dtype), points


def matrix(values, scales, points, group):
    spread = lambda t: t.double().repeat_interleave(group, 1)  # noqa: E731
    return (values.double() - (8.0 if points is None else spread(points))) * spread(scales)


SHAPES = [
    # rows, inputs, outputs, group
    (1, 32, 1, 32), (1, 2048, 2048, 128), (2, 64, 15, 64), (3, 384, 1536, 32), (5, 96, 17, 32), (7, 192, 33, 64),
    (16, 2048, 300, 128), (17, 1024, 40, 64), (31, 1280, 100, 32), (33, 640, 24, 128), (48, 6144, 64, 64),
    (64, 2048, 10000, 128), (65, 256, 31, 128), (130, 1152, 50, 32), (4, 16896, 40, 128), (1, 5120, 9, 32),
    (20, 4224, 21, 128), (300, 2048, 96, 64), (64, 6144, 2048, 64), (33, 2048, 4100, 32), (40, 1024, 9000, 32),
    (64, 4096, 2100, 128), (50, 3200, 2100, 32), (3, 4096, 4200, 64), (9, 2592, 4200, 32), (7, 2304, 4130, 128),
    (70, 1024, 11000, 64), (40, 2048, 16400, 64), (5, 10240, 70, 64),
    (3, 2304, 4300, 32), (20, 2688, 4200, 128), (36, 4352, 4300, 64), (5, 4224, 8400, 64), (35, 4352, 9000, 32),
    (5, 2432, 8300, 64), (3, 4096, 8300, 32), (30, 2688, 8250, 32), (2, 2816, 8400, 128), (2, 2048, 24700, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES)
def test_exact_on_integers(dtype, rows, inputs, outputs, group):
    from asrback_amd.linear4 import linear4, pack4, unpack4

    g = torch.Generator().manual_seed(rows * 7 + inputs)
    for zeros, bias in ((False, False), (True, True)):
        say("linear4", dtype, rows, inputs, outputs, group, zeros, bias)
        values, scales, points = quantized(outputs, inputs, group, zeros, dtype, g, powers=True)
        weight = pack4(values.cuda(), scales.cuda(), None if points is None else points.cuda())
        w = matrix(values, scales, points, group)
        assert torch.equal(unpack4(weight).cpu().double(), w)
        x = torch.randint(-4, 5, (rows, inputs), generator=g).to(dtype)
        b = torch.randint(-9, 10, (outputs,), generator=g).to(dtype) if bias else None
        out = linear4(x.cuda(), weight, None if b is None else b.cuda())
        ref = x.double() @ w.T
        if bias:
            ref = ref + b.double()
        assert torch.equal(out.cpu(), ref.to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES[1::3] + [(3, 2048, 151936, 128)])
def test_real_values(dtype, rows, inputs, outputs, group):
    from asrback_amd.linear4 import linear4, pack4

    g = torch.Generator().manual_seed(rows * 11 + inputs)
    zeros = rows % 2 == 1
    say("linear4 real", dtype, rows, inputs, outputs, group)
    values, scales, points = quantized(outputs, inputs, group, zeros, dtype, g)
    weight = pack4(values.cuda(), scales.cuda(), None if points is None else points.cuda())
    x = torch.randn(rows, inputs, generator=g).to(dtype)
    out = linear4(x.cuda(), weight).cpu().double()
    at = torch.arange(outputs)[:: max(1, outputs // 500)]
    points = None if points is None else points[at]
    ref = x.double() @ matrix(values[at], scales[at], points, group).T
    sums = x.double().abs() @ scales[at].double().repeat_interleave(group, 1).T
    reach, step, ways = (286, 2.0**-8, 2) if dtype == BF16 else (30, 2.0**-24, 4)
    bound = step * ref.abs() + 2.0**-24 * (ways * group + inputs // group + 32) * reach * sums
    assert ((out[:, at] - ref).abs() <= bound).all()
    # Far closer in the mean: the sums' errors do not add up.
    norm = float((out[:, at] - ref).norm() / ref.norm())
    assert norm < (2.0**-8 if dtype == BF16 else 2.0**-18), norm


def test_layouts_of_x_out_and_other_rows():
    """Leading dimensions, strided and misaligned rows, a given out, no rows; rows
    do not touch each other, NaN and infinities included."""
    from asrback_amd.linear4 import linear4, pack4

    g = torch.Generator().manual_seed(3)
    values, scales, points = quantized(70, 256, 64, True, BF16, g, powers=True)
    weight = pack4(values.cuda(), scales.cuda(), points.cuda())
    w = matrix(values, scales, points, 64)
    say("layouts")
    wide = torch.randint(-4, 5, (3, 5, 600), generator=g).to(BF16).cuda()
    for x in (wide[..., :256], wide[..., 8:264], wide[..., 3:259], wide[:, ::2, 256:512], wide[1, 1, :256],
              wide[:, :, :256].transpose(0, 1)):
        ref = (x.double().cpu() @ w.T).to(BF16)
        assert torch.equal(linear4(x, weight).cpu(), ref)
        out = torch.full(ref.shape, 7.0, dtype=BF16, device="cuda")
        assert linear4(x, weight, out=out) is out and torch.equal(out.cpu(), ref)
    assert linear4(wide[:0, :, :256], weight).shape == (0, 5, 70)
    say("rows apart")
    x = wide[0, :, :256].clone()
    x[1] = float("nan")
    x[3, 5] = float("inf")
    out = linear4(x, weight).cpu()
    keep = [0, 2, 4]
    assert torch.equal(out[keep], (x[keep].double().cpu() @ w.T).to(BF16))
    assert out[1].isnan().all() and not out[3].isfinite().any()


def test_out_apart_from_x():
    from asrback_amd.linear4 import linear4, quantize4

    g = torch.Generator().manual_seed(6)
    weight = quantize4(torch.randn(256, 256, generator=g).to("cuda", BF16), 64)
    arena = torch.randn(12, 256, generator=g).to("cuda", BF16)
    x = arena[:4]
    ref = linear4(x, weight)
    for out in (arena[:4], arena[3:7]):
        with pytest.raises(ValueError, match="shares memory"):
            linear4(x, weight, out=out)
    assert torch.equal(linear4(x, weight, out=arena[4:8]), ref)


def test_graph_replays_and_module():
    from asrback_amd.linear4 import Linear4, linear4, quantize4, quantize_linears, unpack4

    g = torch.Generator().manual_seed(4)
    model = torch.nn.Sequential(torch.nn.Linear(256, 130), torch.nn.Sequential(torch.nn.Linear(130, 8),
                                torch.nn.Linear(8, 128, bias=False)), torch.nn.Linear(128, 64, bias=False))
    model = model.to("cuda", BF16)
    first, last = model[0], model[2]
    with torch.no_grad():
        for symmetric in (True, False):
            for layer in (first, last):
                weight = quantize4(layer.weight, 64, symmetric)
                step = weight.scales.float().max()
                # Half a step of the group's scale, another half where the zero point is
                # rounded as well, and the scale's own rounding (2^-8) at the ends, 7 or
                # 15 steps out.
                assert float((unpack4(weight) - layer.weight.float()).abs().max()) <= float(step) * (0.5 + 7 * 2**-8 if symmetric else 1 + 15 * 2**-8)
    say("module")
    assert quantize_linears(model, 64) == 2
    assert type(model[0]) is Linear4 and type(model[2]) is Linear4 and type(model[1][0]) is torch.nn.Linear
    assert torch.equal(model[0].bias, first.bias)
    x = torch.randn(6, 256, generator=g).to("cuda", BF16)
    with torch.no_grad():
        got = model[0](x)
        want = (x.double().cpu() @ unpack4(model[0].weight4).double().cpu().T) + first.bias.double().cpu()
        assert float((got.double().cpu() - want).norm() / want.norm()) < 2.0**-8
    # State dicts and devices.
    other = Linear4(quantize4(torch.zeros(130, 256, dtype=BF16), 64), torch.zeros(130, dtype=BF16)).cuda()
    other.load_state_dict(model[0].state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), got)
    with pytest.raises(RuntimeError, match="no gradient"):
        model[0](x.requires_grad_())
    say("graph")
    static = torch.empty(6, 256, dtype=BF16, device="cuda")
    with torch.no_grad():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            model[0](static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model[0](static)
        for _ in range(4):
            static.copy_(torch.randn(6, 256, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, linear4(static, model[0].weight4, model[0].bias))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES)
def test_exact_on_the_largest_values(dtype, rows, inputs, outputs, group):
    """Rows of integers times 2^124, whose groups' sums pass the type's range before
    their scale brings them back, beside rows of ordinary and of tiny ones; and a
    value of 2^125 that a scale of zero takes out of a row.  Results are below 2^(126
    + 4 + 15 - 20), and sums of integers below 2^24 times a power of two: exact."""
    from asrback_amd.linear4 import linear4, pack4

    g = torch.Generator().manual_seed(rows * 5 + inputs)
    say("linear4 large", dtype, rows, inputs, outputs, group)
    values, scales, points = quantized(outputs, inputs, group, rows % 2 == 0, dtype, g, powers=True)
    scales *= 2.0**-20
    weight = pack4(values.cuda(), scales.cuda(), None if points is None else points.cuda())
    w = matrix(values, scales, points, group)
    powers = torch.tensor([124.0, 0.0, 112.0, -100.0, 64.0, 60.0])[torch.arange(rows) % 6]
    x = (torch.randint(-4, 5, (rows, inputs), generator=g) * 2.0**powers[:, None]).to(dtype)
    assert x.isfinite().all()
    assert torch.equal(linear4(x.cuda(), weight).cpu(), (x.double() @ w.T).to(dtype))
    # One large value in a group whose scales are zero.
    at = inputs // group // 2
    scales[:, at] = 0
    weight = pack4(values.cuda(), scales.cuda(), None if points is None else points.cuda())
    x = torch.randint(-4, 5, (rows, inputs), generator=g).to(dtype)
    x[::2, at * group + 3] = 2.0**125
    ref = (x.double() @ matrix(values, scales, points, group).T).to(dtype)
    assert torch.equal(linear4(x.cuda(), weight).cpu(), ref)


def test_results_past_the_range_are_infinite():
    from asrback_amd.linear4 import linear4, pack4

    say("linear4 overflow")
    for dtype in (BF16, F32):
        values = torch.full((2, 256), 8, dtype=torch.uint8)
        values[0, :64], values[1, 128:192] = 15, 1
        weight = pack4(values.cuda(), torch.ones(2, 2, dtype=dtype).cuda())
        x = torch.full((3, 256), 2.0**125, dtype=dtype)
        x[1] = 3.0
        out = linear4(x.cuda(), weight).cpu()
        inf = float("inf")
        assert out.tolist() == [[inf, -inf], [64 * 7 * 3.0, -64 * 7 * 3.0], [inf, -inf]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES[::5])
def test_smallest_values(dtype, rows, inputs, outputs, group):
    """Integers times powers of two down to 2^-118 are exact in bf16.  A float32 input
    goes in to 2^-121, which its weight's product and the sum for the zero point
    carry to at most 15 and 15 scales."""
    from asrback_amd.linear4 import linear4, pack4

    g = torch.Generator().manual_seed(rows * 3 + inputs)
    say("linear4 small", dtype, rows, inputs, outputs, group)
    values, scales, points = quantized(outputs, inputs, group, True, dtype, g, powers=True)
    weight = pack4(values.cuda(), scales.cuda(), points.cuda())
    w = matrix(values, scales, points, group)
    unit = 2.0 ** torch.tensor([-118.0, -100.0, -60.0])[torch.arange(rows) % 3, None]
    if dtype == BF16:
        x = (torch.randint(-4, 5, (rows, inputs), generator=g) * unit).to(dtype)
        assert torch.equal(linear4(x.cuda(), weight).cpu(), (x.double() @ w.T).to(dtype))
        return
    x = torch.randn(rows, inputs, generator=g) * unit
    out, ref = linear4(x.cuda(), weight).cpu().double(), x.double() @ w.T
    spread = scales.double().repeat_interleave(group, 1)
    bound = 2.0**-24 * ref.abs() + 2.0**-24 * (4 * group + inputs // group + 32) * 30 * (x.double().abs() @ spread.T)
    assert ((out - ref).abs() <= bound + 2.0**-121 * 30 * spread.sum(1)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_row_of_any_layout(dtype):
    """A single row of an odd row stride and rows at an odd offset, which torch calls
    contiguous."""
    from asrback_amd.linear4 import linear4, pack4

    g = torch.Generator().manual_seed(9)
    say("linear4 one row", dtype)
    values, scales, points = quantized(70, 256, 64, True, dtype, g, powers=True)
    weight = pack4(values.cuda(), scales.cuda(), points.cuda())
    buffer = torch.randint(-4, 5, (2000,), generator=g).to(dtype).cuda()
    for x in (buffer[:257].view(1, 257)[:, :256], buffer[3:259].view(1, 256), buffer[3:259], buffer[1:1025].view(2, 2, 256),
              buffer[:514].view(1, 2, 257)[:, :1, :256]):
        assert torch.equal(linear4(x, weight).cpu(), (x.double().cpu() @ matrix(values, scales, points, 64).T).to(dtype))


@pytest.mark.parametrize("rows,inputs,outputs,group", SHAPES[::4])
def test_inputs_with_a_mean(rows, inputs, outputs, group):
    """Where inputs share a sign, the offset that bf16 weights carry meets their whole
    sum: the same bound."""
    from asrback_amd.linear4 import linear4, pack4

    g = torch.Generator().manual_seed(rows * 13 + inputs)
    say("linear4 mean", rows, inputs, outputs, group)
    values, scales, points = quantized(outputs, inputs, group, False, BF16, g)
    weight = pack4(values.cuda(), scales.cuda())
    x = (torch.randn(rows, inputs, generator=g) + torch.tensor([1.0, -4.0])[torch.arange(rows) % 2, None]).to(BF16)
    ref = x.double() @ matrix(values, scales, points, group).T
    sums = x.double().abs() @ scales.double().repeat_interleave(group, 1).T
    # What is left of the result once it is taken off: the sums' own error.  A group's sums
    # reach some 143 * 128 (2^14.2), each addition off by half a step of 2^-24 of
    # that, a dozen of them as their root (2^1.8): 2^-9 of results of some 2^6.2.
    bias = -ref[0].to(BF16)
    left = linear4(x[:1].cuda(), weight, bias.cuda()).cpu().double() - (ref[:1] + bias.double())
    own = 2.0**-24 * (2 * group + inputs // group + 32) * 286 * sums
    assert (left.abs() <= 2.0**-8 * (ref[:1] + bias.double()).abs() + own[:1]).all()
    assert float(left.norm() / ref[0].norm()) < 2.0**-15
    out = linear4(x.cuda(), weight).cpu().double()
    assert ((out - ref).abs() <= 2.0**-8 * ref.abs() + own).all()
