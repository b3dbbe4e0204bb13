"""GPU: models with 4-bit layers (``quantize_linears``) against the same models
with those layers' rounded matrices unpacked into ``nn.Linear``."""

from __future__ import annotations

import copy

import pytest
import torch

from conftest import assert_close
from test_gpu_models import sensevoice_pair

pytestmark = pytest.mark.gpu


def say(*args):
    print(*args, flush=True)


def quantized_pair(model, group, symmetric=True):
    """The model with 4-bit layers, and with their matrices unpacked."""
    from asrback_amd.linear4 import Linear4, quantize_linears, unpack4

    four, plain = model, copy.deepcopy(model)
    count = quantize_linears(four, group, symmetric)
    assert count == sum(type(m) is Linear4 for m in four.modules()) > 0
    layers = dict(four.named_modules())
    with torch.no_grad():
        for name, layer in plain.named_modules():
            if isinstance(layers[name], Linear4):
                layer.weight.copy_(unpack4(layers[name].weight4))
    return four, plain


@pytest.mark.parametrize("symmetric", [True, False])
def test_sensevoice(device, symmetric):
    from oracle import sensevoice as osv

    say("4-bit sensevoice", symmetric)
    four, plain = quantized_pair(sensevoice_pair(device)[1], 64, symmetric)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 4 + 120, 560, generator=g).to(device)
    mask = osv.frame_mask(torch.tensor([80, 40, 120, 7]), 4, 120).to(device)
    with torch.inference_mode():
        out, expected = four(x, mask), plain(x, mask)
        assert_close((out * mask[..., None]).cpu(), (expected * mask[..., None]).cpu(), "module", 1e-4)
        assert_close(four(x[:1], None).cpu(), plain(x[:1], None).cpu(), "module", 1e-4)


def test_sensevoice_attention_bf16(device):
    """One attention module: its valid frames, and padded ones with linear_out's bias
    alone."""
    from asrback_amd import sensevoice as asv

    say("4-bit sensevoice, bf16")
    torch.manual_seed(3)
    four, plain = quantized_pair(asv.SANMAttention(512, 512, 4, 11).eval().to(device, torch.bfloat16), 128)
    x = torch.randn(3, 200, 512, generator=torch.Generator().manual_seed(9)).to(device, torch.bfloat16)
    lengths = torch.tensor([200, 31, 1])
    mask = (torch.arange(200) < lengths[:, None]).to(device)
    with torch.inference_mode():
        out, expected = four(x, mask, None), plain(x, mask, None)
    assert_close((out * mask[..., None]).float().cpu(), (expected * mask[..., None]).float().cpu(), "bf16")
    for b, n in enumerate(lengths.tolist()):
        assert torch.equal(out[b, n:], four.linear_out.bias.expand(200 - n, 512))
