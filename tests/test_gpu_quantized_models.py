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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whisper(device, dtype):
    """Encoder, prompt pass and steps; the layers leave the step's row kernels to plain
    layers."""
    import json

    from conftest import GOLDEN
    from oracle import whisper as ow
    from test_gpu_whisper import gpu_model

    say("4-bit whisper", dtype)
    fixture = json.loads((GOLDEN / "whisper_tiny_greedy.json").read_text())
    weights = ow.attention_heavy_weights(ow.WhisperForConditionalGeneration(fixture["config"]), fixture["seeds"]["weights"])
    four, plain = quantized_pair(gpu_model(fixture, weights, device, dtype), 128)
    # bf16: some ten roundings a layer (2^-8) in each of eight layers, as their square
    # root, on either side, and that of the unpacked matrices.
    bound = 1e-4 if dtype == torch.float32 else 2.0**-8 * (2 * 10 * 8) ** 0.5
    g = torch.Generator().manual_seed(2)
    mel = torch.randn(2, 80, 3000, generator=g).to(device, dtype)
    tokens = torch.randint(0, 50000, (2, 6), generator=g).to(device)
    positions = torch.arange(448, device=device)

    def close(a, b):
        assert a.shape == b.shape
        error = float((a.double() - b.double()).norm() / b.double().norm())
        assert error < bound, error

    with torch.inference_mode():
        encoded = [m.model.encoder(mel) for m in (four, plain)]
        close(*encoded)
        caches = []
        for m in (four, plain):
            caches.append(m.allocate_cache(2))
            m.set_encoder_output(caches[-1], encoded[1])
        close(*(m.decode(tokens[:, :4], positions[:4], c, length=4) for m, c in zip((four, plain), caches)))
        for i in (4, 5):
            at = torch.full((2,), i, device=device)
            close(*(m.decode(tokens[:, i:i + 1], at, c) for m, c in zip((four, plain), caches)))
