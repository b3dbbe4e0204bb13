"""CPU: what the drafts' and 4-bit layers' ops refuse as ``out``."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad


def test_overlap():
    from asrback_amd.layers import overlap

    buffer = torch.zeros(4, 6, 5, 64)  # rows of five parts
    part = [buffer[:, :, i] for i in range(5)]
    assert overlap(part[1], part[1]) and overlap(buffer, part[2])
    assert not overlap(part[0], part[4]) and not overlap(part[4], part[0])
    assert not overlap(part[1], buffer[:, :, 2:4]) and overlap(buffer[:, :, 1:4], part[3])
    assert not overlap(buffer[0], buffer[1]) and overlap(buffer[:2], buffer[1])
    assert not overlap(buffer[:, :, 0, :32], buffer[:, :, 0, 32:])
    assert overlap(buffer[:, :, 0, :33], buffer[:, :, 0, 32:])
    assert not overlap(buffer[..., :1], torch.zeros(3)) and not overlap(buffer[:0], buffer)
    assert not overlap(buffer[::2, :, 0], buffer[1::2, :, 0]) and overlap(buffer[::2, :, 0], buffer[2:, :, 0])
    for a in (buffer[1:3, :, 1:3, 8:40], buffer[:, 2], buffer[0, 0]):
        for b in (buffer[2:, 1:4, 2, 30:], buffer[:, 2:, 3], buffer[:2, :, 4, 5], buffer[3], buffer[0, 0, 2]):
            held = torch.zeros(buffer.numel(), dtype=torch.int32)
            for t in (a, b):
                held.as_strided(t.shape, t.stride(), t.storage_offset()).add_(1)
            if (held > 1).any():
                assert overlap(a, b) and overlap(b, a)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_linear4_out():
    from asrback_amd.linear4 import linear4, pack4

    weight = pack4(torch.zeros(64, 64, dtype=torch.uint8), torch.ones(64, 2))
    arena = torch.zeros(12, 64)
    x, bias = arena[:4], arena[10]
    good = torch.zeros(4, 64)

    def call(out):
        return linear4(x, weight, bias, out=out)

    with pytest.raises(RuntimeError, match="GPU only"):
        call(good)
    for out in (x, arena[3:7], arena[8:]):
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


def test_tree_attention_out():
    from asrback_amd.drafts import tree_attention

    arena = torch.zeros(2, 3, 12, 64)  # q, drafted keys and values, out in one buffer
    q, kd, vd, out = arena[:, :, :4], arena[:, :, 4:6], arena[:, :, 6:8], arena[:, :, 8:]
    k, v = torch.zeros(2, 8, 2, 64), torch.zeros(2, 8, 2, 64)
    masks = torch.ones(2, 3, dtype=torch.int64)

    def call(out, **more):
        return tree_attention(q, k, v, kd, vd, masks, out=out, **more)

    for good in (out, q, torch.zeros(2, 3, 4, 64), torch.zeros(3, 2, 4, 64).transpose(0, 1),
                 torch.zeros(2, 3, 4, 128)[..., 32:96]):
        with pytest.raises(RuntimeError, match="GPU only"):
            call(good)
    for bad in (arena[:, :, 1:5], arena[:, :, 4:8], arena[:, :, 7:11], k.view(-1)[:1536].view(2, 3, 4, 64),
                v.view(-1)[512:2048].view(2, 3, 4, 64)):
        with pytest.raises(ValueError, match="shares memory"):
            call(bad)
    for bad in (torch.zeros(2, 3, 1, 64).expand(2, 3, 4, 64), torch.zeros(3, 4, 64).expand(2, 3, 4, 64),
                torch.zeros(4000).as_strided((2, 3, 4, 64), (768, 256, 32, 1))):
        with pytest.raises(ValueError, match="more than once"):
            call(bad)
    with pytest.raises(ValueError, match="unit last stride"):
        call(torch.zeros(2, 3, 64, 4).transpose(2, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        call(torch.zeros(2, 3, 4, 64, requires_grad=True))
    with torch.inference_mode():
        held = torch.zeros(2, 3, 4, 64)
    with pytest.raises(RuntimeError, match="inference"):
        call(held)
