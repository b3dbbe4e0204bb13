"""GPU: linear layers with 8-bit weights, and the gated block over them.

The rounding of the rows and the sums of the products are exact, so a float64
reference has the same whole numbers.  What the kernel rounds after them, relative to
the scaled product: its conversion to float32 and two scales, 2^-24 each; to the sum:
the bias, 2^-24, and the result, 2^-8 in bf16.  The gate's silu of g adds (2 |g| + 8)
2^-24 of itself (the exponent's product and constant, 2^-24 |g| each, the exponential
2^-23, the sum, the quotient and the two products), and carries g's own error times
its slope, at most 1.1; below -87 it is less than 1e-36 in magnitude.  All times 1.01 for
second-order terms.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
STEP = {F32: 2.0**-24, BF16: 2.0**-8}


def say(*args):
    print(*args, flush=True)


def rounded(x):
    """Whole numbers and float32 scales of rows, exact to the border."""
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float().double()
    q = torch.where(scale > 0, x.double() / scale.where(scale > 0, torch.ones_like(scale)), 0.0)
    return q.round().clamp(-127, 127), scale


def reference(x, values, scales, bias):
    """The sum and the bound of its error in float32."""
    q, scale = rounded(x)
    product = (q @ values.double().T) * scale * scales.double()
    y = product if bias is None else product + bias.double()
    return y, 2.0**-24 * (3 * product.abs() + (0 if bias is None else y.abs()))


def check(out, x, values, scales, bias, gated=False):
    y, error = reference(x, values, scales, bias)
    if gated:
        (g, u), (eg, eu) = y.chunk(2, -1), error.chunk(2, -1)
        s = g * torch.sigmoid(g)
        y = s * u
        error = u.abs() * (1.1 * eg + s.abs() * (2 * g.abs() + 8) * 2.0**-24 + 1e-36) + s.abs() * eu
    bound = 1.01 * (error + STEP[out.dtype] * y.abs()) + 1e-44
    out = out.cpu().double()
    worst = ((out - y).abs() / bound).max()
    assert worst <= 1, float(worst)


def matrix(outputs, inputs, dtype, g):
    values = torch.randint(-127, 128, (outputs, inputs), generator=g, dtype=torch.int8)
    return values, (torch.rand(outputs, generator=g) * 0.02 + 0.001).to(dtype)


SHAPES = [
    # rows, inputs, outputs
    (1, 1, 1), (1, 64, 16), (1, 2048, 2048), (2, 63, 15), (3, 384, 1536), (5, 65, 17), (7, 200, 34), (16, 2048, 300),
    (17, 1000, 40), (31, 1280, 100), (33, 640, 24), (48, 6144, 64), (64, 2048, 10000), (65, 257, 31), (100, 8192, 130),
    (130, 1152, 514), (200, 64, 1000), (255, 512, 256), (256, 1024, 1026), (257, 130, 700), (300, 2048, 96), (513, 1280, 258),
    (1, 20000, 50), (4, 2048, 30001), (1000, 512, 1536), (1537, 2048, 514), (2100, 100, 260), (40, 100001, 18),
    (12, 2049, 4096), (9, 4096, 2050), (129, 4096, 4100), (700, 1280, 5120), (1300, 193, 5007), (2600, 77, 9001),
    (3300, 100, 4096), (3231, 67, 4111),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,inputs,outputs", SHAPES)
def test_products(dtype, rows, inputs, outputs):
    from asrback_amd.linear8 import gated8, linear8, pack8, unpack8

    g = torch.Generator().manual_seed(rows * 7 + inputs)
    values, scales = matrix(outputs, inputs, dtype, g)
    weight = pack8(values.cuda(), scales.cuda())
    assert torch.equal(unpack8(weight).cpu(), values.float() * scales.float()[:, None])
    x = torch.randn(rows, inputs, generator=g).to(dtype)
    x[rows // 2] *= 1000
    for bias in (None, torch.randn(outputs, generator=g).to(dtype)):
        say("linear8", dtype, rows, inputs, outputs, bias is not None)
        out = linear8(x.cuda(), weight, None if bias is None else bias.cuda())
        check(out, x, values, scales, bias)
        if outputs % 2 == 0:
            small = x / (4 * math.sqrt(inputs))  # gates of some units
            out = gated8(small.cuda(), weight, None if bias is None else bias.cuda())
            assert out.shape == (rows, outputs // 2)
            check(out, small, values, scales, bias, gated=True)


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_borders_of_the_rounding(dtype, rows):
    """Ties, values next to them, subnormal and huge rows: against whole numbers of the
    identity matrix."""
    from asrback_amd.linear8 import linear8, pack8

    inputs = 256
    g = torch.Generator().manual_seed(rows)
    weight = pack8(torch.eye(inputs, dtype=torch.int8).cuda(), torch.ones(inputs, dtype=dtype).cuda())
    x = torch.empty(rows, inputs, dtype=F32)
    for r in range(rows):
        kind = r % 5
        if kind == 0:  # ties of a scale of one, and their neighbours
            row = torch.arange(inputs) % 254 - 126.5
            if r % 2:
                row = torch.nextafter(row, row + torch.randint(-1, 2, (inputs,), generator=g))
            row[0] = 127
        elif kind == 1:  # of other scales
            scale = torch.rand(1, generator=g) + 0.5
            row = (torch.arange(inputs) % 254 - 126.5) * scale
            row[3] = 127 * scale
        elif kind == 2:
            row = torch.randn(inputs, generator=g) * 2.0**-135
        elif kind == 3:
            row = torch.randn(inputs, generator=g) * 2.0**124
        else:
            row = torch.randn(inputs, generator=g) * 2.0**-147
        x[r] = row
    x = x.to(dtype)
    say("borders", dtype, rows)
    out = linear8(x.cuda(), weight).cpu()
    q, scale = rounded(x)
    # (the smallest rows' scale, below half of 2^-149, is 0)
    assert ((q.abs().amax(1) >= 100) | (scale[:, 0] == 0)).all() and torch.isfinite(x).all()
    # A product with one and a scale: rounded once to float32, once to the type.
    ref = (q.float() * scale.float()).to(dtype)
    assert torch.equal(out, ref)


def test_every_quotient_of_bf16_numbers():
    """Rows of each largest mantissa, of all mantissas at ten exponents: many lie within
    2^-24 of a border, and those of the largest 254 on one."""
    from asrback_amd.linear8 import linear8, pack8

    mantissas = torch.arange(128, 256).double()
    values = torch.cat([mantissas * 2.0**-j for j in range(1, 11)])
    rows = torch.cat([torch.cat((m[None], values, -values)) * 2.0 ** (int(m) % 5 - 2) for m in mantissas]).view(128, -1)
    x = rows.to(BF16)
    assert torch.equal(x.double(), rows)
    weight = pack8(torch.eye(x.shape[1], dtype=torch.int8).cuda(), torch.ones(x.shape[1], dtype=BF16).cuda())
    q, scale = rounded(x)
    for part in (x, x[:3]):  # rounded by a launch of its own and by the product
        say("quotients", len(part))
        out = linear8(part.cuda(), weight).cpu()
        assert torch.equal(out, (q[: len(part)].float() * scale[: len(part)].float()).to(BF16))


def test_layouts_of_x_out_and_other_rows():
    """Leading dimensions, strided and misaligned rows, a given out, no rows; rows do
    not touch each other, NaN and infinities included."""
    from asrback_amd.linear8 import gated8, linear8, pack8

    g = torch.Generator().manual_seed(3)
    for dtype in (BF16, F32):
        values, scales = matrix(70, 250, dtype, g)
        weight = pack8(values.cuda(), scales.cuda())
        say("layouts", dtype)
        wide = torch.randn(3, 5, 600, generator=g).to(dtype).cuda()
        whole = linear8(wide[..., :250].contiguous(), weight)
        assert whole.shape == (3, 5, 70)
        for x in (wide[..., :250], torch.cat((wide.new_zeros(3, 5, 1), wide), -1)[..., 1:251],
                  wide[..., :250].permute(2, 0, 1).contiguous().permute(1, 2, 0)):
            assert torch.equal(linear8(x, weight), whole)
        assert torch.equal(linear8(wide[1, 2, :250], weight), whole[1, 2])
        assert torch.equal(linear8(wide[:1, :1, :250].expand(3, 5, 250), weight), whole[:1, :1].expand(3, 5, 70))
        assert linear8(wide[:0, :, :250], weight).shape == (0, 5, 70)
        assert gated8(wide[:0, :, :250], weight).shape == (0, 5, 35)
        for f, width in ((linear8, 70), (gated8, 35)):
            held = torch.full((5, 5, width), 7.0, dtype=dtype, device="cuda")
            version = held._version
            out = f(wide[..., :250], weight, out=held[1:4])
            assert out.data_ptr() == held[1].data_ptr() and held._version > version
            assert torch.equal(out, f(wide[..., :250], weight)) and (held[0] == 7).all() and (held[4] == 7).all()
        for rows in (3, 16, 40, 300):
            x = torch.randn(rows, 250, generator=g).to(dtype).cuda()
            clean = linear8(x, weight)
            bad = x.clone()
            bad[1, 7], bad[rows - 1, 249] = math.nan, -math.inf
            bad[0] = 0
            out = linear8(bad, weight)
            assert torch.isnan(out[1]).all() and torch.isnan(out[rows - 1]).all() and not out[0].any()
            others = [r for r in range(rows) if r not in (0, 1, rows - 1)]
            assert torch.equal(out[others], clean[others])
            assert torch.isnan(gated8(bad, weight)[[1, rows - 1]]).all()


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_scales_far_apart(rows):
    """Nothing overflows or is lost on the way to a result within range."""
    from asrback_amd.linear8 import linear8, pack8

    g = torch.Generator().manual_seed(rows)
    values, _ = matrix(40, 2048, F32, g)
    for big, small in ((2.0**120, 2.0**-110), (2.0**-110, 2.0**100), (2.0**100, 2.0**-125), (2.0**-60, 2.0**-60)):
        for dtype in (F32, BF16):
            scales = (torch.rand(40, generator=g) * small + small).to(dtype)
            x = (torch.randn(rows, 2048, generator=g) * big).to(dtype)
            say("scales", rows, big, small, dtype)
            out = linear8(x.cuda(), pack8(values.cuda(), scales.cuda()))
            check(out, x, values, scales, None)


def test_largest_sums():
    """2^17 inputs of the largest values stay within 32 bits."""
    from asrback_amd.linear8 import MAX_INPUTS, linear8, pack8

    for rows in (1, 40):
        values = torch.full((33, MAX_INPUTS), 127, dtype=torch.int8)
        values[1::2] = -127
        x = torch.ones(rows, MAX_INPUTS)
        out = linear8(x.cuda(), pack8(values.cuda(), torch.ones(33).cuda())).cpu()
        assert torch.equal(out, out[:1].expand(rows, 33)) and torch.equal(out[:, 0], -out[:, 1])
        check(out, x, values, torch.ones(33), None)


def test_module_quantization_and_graph():
    """A module in place of nn.Linear, captured and replayed with the caller's own work
    between, and on another stream than the default."""
    from torch import nn

    from asrback_amd.linear8 import Linear8, quantize8, quantize_linears8, unpack8

    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(130, 260), nn.GELU(), nn.Linear(260, 50, bias=False)).to("cuda", BF16)
    weights = [unpack8(quantize8(m.weight)) for m in (model[0], model[2])]
    for w, m in zip(weights, (model[0], model[2])):
        # Half a step of 127 to the largest, and what the scale's own rounding moves.
        assert ((w - m.weight.float()).abs() <= w.abs().amax(1, keepdim=True) * (0.5 / 127 + 2.0**-8) * 1.01).all()
    assert quantize_linears8(model) == 2 and isinstance(model[0], Linear8)
    x = torch.randn(20, 130, device="cuda", dtype=BF16)
    with torch.no_grad():
        eager = model(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            on_side = model(x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(on_side, eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model(x)
        for seed in range(3):
            x.copy_(torch.randn(20, 130, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            assert torch.equal(out, model(x))
            torch.cuda.synchronize()


def test_most_rows():
    """As many rows as a call takes, some of them checked."""
    from asrback_amd.linear8 import gated8, linear8, pack8

    g = torch.Generator().manual_seed(8)
    rows, inputs, outputs = 65535 * 16, 64, 18
    values, scales = matrix(outputs, inputs, BF16, g)
    weight = pack8(values.cuda(), scales.cuda())
    x = torch.randn(rows, inputs, device="cuda").to(BF16)
    at = torch.tensor([0, 1, 4095, 300_007, 777_777, rows - 2, rows - 1], device="cuda")
    say("most rows")
    check(linear8(x, weight)[at], x[at].cpu(), values, scales, None)
    small = x / 32
    check(gated8(small, weight)[at], small[at].cpu(), values, scales, None, gated=True)
    with pytest.raises(RuntimeError, match="1048560 rows"):
        linear8(torch.zeros(rows + 1, 64, device="cuda", dtype=BF16), weight)


def test_most_outputs():
    """As many outputs as few rows' launch takes, some of them checked."""
    from asrback_amd.linear8 import linear8, pack8

    g = torch.Generator().manual_seed(9)
    outputs = (1 << 27) - 16
    values = torch.randint(-127, 128, (outputs, 1), device="cuda", dtype=torch.int8)
    scales = (torch.rand(outputs, device="cuda") * 0.02 + 0.001).to(BF16)
    x = torch.randn(1, 1, generator=g).to(BF16)
    say("most outputs")
    out = linear8(x.cuda(), pack8(values, scales))
    at = torch.tensor([0, 1, 15, 16, 9_999_999, 77_777_777, outputs - 17, outputs - 1], device="cuda")
    check(out[:, at], x, values[at].cpu(), scales[at].cpu(), None)


def check_here(out, x, values, scales, bias, gated=False):
    """:func:`check` where the tensors are, for many outputs.  Below 2^-126 the numbers of both
    types are evenly spaced, 2^-133 apart in bf16 (8 bits from 2^-126 down) and 2^-149 in
    float32, so a rounding there is off by up to half of that whatever the value: 2^-134
    (4.6e-41), and less than 1e-44."""
    y, error = reference(x, values, scales, bias)
    if gated:
        (g, u), (eg, eu) = y.chunk(2, -1), error.chunk(2, -1)
        s = g * torch.sigmoid(g)
        y = s * u
        error = u.abs() * (1.1 * eg + s.abs() * (2 * g.abs() + 8) * 2.0**-24 + 1e-36) + s.abs() * eu
    bound = 1.01 * (error + STEP[out.dtype] * y.abs()) + (1.01 * 2.0**-134 if out.dtype == BF16 else 1e-44)
    worst = ((out.double() - y).abs() / bound).max()
    assert worst <= 1, float(worst)


# Tiles of 64 x 128, of 128 x 128 and of 128 x 256 (gated: half as many outputs), the last
# two in more tiles than the card's 512 workgroups; an odd and an even number of blocks of
# 64 inputs, and widths that end inside a vector.
TILED = [
    # rows, inputs, outputs
    (1000, 512, 1541), (970, 700, 1536), (2600, 650, 9006), (2500, 1280, 9008), (3500, 700, 8450), (3457, 1024, 8706),
    (2600, 650, 6606), (2500, 1280, 6608), (5200, 330, 8450),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,inputs,outputs", TILED)
@pytest.mark.parametrize("gated", [False, True])
def test_deep_products_of_many_tiles(dtype, rows, inputs, outputs, gated):
    """Every output of tiles whose ring of stages turns over several times, from a tile into the
    next; then rows of far scales in some waves only, of NaN and of infinities."""
    from asrback_amd.linear8 import gated8, linear8, pack8

    g = torch.Generator().manual_seed(rows + inputs)
    if gated:
        outputs = outputs // 2 * 2
    call = gated8 if gated else linear8
    values, scales = (t.cuda() for t in matrix(outputs, inputs, dtype, g))
    bias = torch.randn(outputs, generator=g).to("cuda", dtype)
    x = torch.randn(rows, inputs, generator=g).to("cuda", dtype) / (4 * math.sqrt(inputs))
    say("tiled", dtype, rows, inputs, outputs, gated)
    weight = pack8(values, scales)
    check_here(call(x, weight, bias), x, values, scales, bias, gated)
    # Scales from 2^90 on are multiplied in another order; with an output's own far below, the
    # results are ordinary.
    far = torch.zeros(rows, dtype=torch.bool, device="cuda")
    far[:16] = far[rows // 2] = far[-1] = True
    small = (scales.float() * 2.0**-110).to(dtype)
    mixed = torch.where(far[:, None], x.float() * 2.0**115, x.float()).to(dtype)
    say("far rows")
    weight = pack8(values, small)
    out = call(mixed, weight)
    check_here(out, mixed, values, small, None, gated)
    at = torch.tensor([5, 40, rows // 3, rows - 1], device="cuda")
    bad = mixed.clone()
    bad[at, torch.tensor([0, 63, 64, inputs - 1], device="cuda")] = torch.tensor(
        [math.nan, math.inf, math.nan, -math.inf], device="cuda", dtype=dtype)
    say("rows without numbers")
    have = call(bad, weight)
    assert torch.isnan(have[at]).all()
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[at] = False
    assert torch.equal(have[others], out[others])
