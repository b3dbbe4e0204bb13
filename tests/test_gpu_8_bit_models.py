"""GPU: models with 8-bit layers (``quantize_linears8``) and Qwen3-ASR's decoder over an
8-bit cache, against the same models on plain float64 layers, cache writes and
attention.

A rounding to 8 bits is off by half of a 127th of the row's largest number, which is
some four times the row's root mean square: by about 2^-7 of the row's norm, times
3^-1/2.  Both sides round rows that differ by the float32 work before them, and a number
on the border goes the other way by a whole step: at worst the two sides' roundings
are independent, 2^-7 of the norm between them a layer, growing as the square
root of the layers.  Where only the cache is rounded, a step's own key and value are the
ones that can differ.
"""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

from test_gpu_models import QWEN3, _qwen_decoder, qwen_pair, sensevoice_pair

pytestmark = pytest.mark.gpu


def say(*args):
    print(*args, flush=True)


def rounded(x):
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float().double()
    q = torch.where(scale > 0, x.double() / scale.where(scale > 0, torch.ones_like(scale)), 0.0)
    return q.round().clamp(-127, 127), scale


class Plain8(nn.Module):
    def __init__(self, layer):
        from asrback_amd.linear8 import unpack8

        super().__init__()
        self.in_features, self.out_features = layer.in_features, layer.out_features
        weight = layer.weight8
        self.weight = nn.Parameter(unpack8(weight).to(weight.scales.dtype))  # (models ask for its type)
        self.matrix, self.bias = unpack8(weight).double(), layer.bias

    def forward(self, x):
        q, scale = rounded(x)
        out = (q @ self.matrix.t()) * scale
        return (out if self.bias is None else out + self.bias.double()).to(x.dtype)


def with_plain_layers(model):
    """A copy with plain modules in place of the 8-bit layers, and how many there are."""
    from asrback_amd.linear8 import Linear8

    plain, count = copy.deepcopy(model), 0
    for parent in list(plain.modules()):
        for name, child in list(parent.named_children()):
            if isinstance(child, Linear8):
                setattr(parent, name, Plain8(child))
                count += 1
    assert count
    return plain, count


def difference(a, b):
    assert a.shape == b.shape and torch.isfinite(a).all()
    return float((a.double() - b.double()).norm() / b.double().norm())


def close(a, b, bound):
    error = difference(a, b)
    assert error < bound, error


def test_sensevoice(device):
    from asrback_amd.linear8 import quantize_linears8
    from oracle import sensevoice as osv

    say("8-bit sensevoice")
    eight = sensevoice_pair(device)[1]
    held = quantize_linears8(eight)
    plain, count = with_plain_layers(eight)
    assert count == held
    # The reference's own linear_out lies beside its attention kernel, as bias and matrix.
    for m in plain.modules():
        if hasattr(m, "linear_out"):
            m.forward = lambda x, mask, lengths, m=m: sanm(m, x, mask)

    def sanm(m, x, mask):
        b, n, _ = x.shape
        keep = torch.ones(b, n, dtype=torch.bool, device=device) if mask is None else mask
        q, k, v = m.linear_q_k_v(x).split(m.size, -1)
        memory = (v * keep[..., None]).transpose(1, 2)
        taps = m.fsmn_block.weight.shape[-1]
        left = (taps - 1) // 2
        memory = nn.functional.conv1d(nn.functional.pad(memory, (left, taps - 1 - left)), m.fsmn_block.weight, groups=m.size)
        memory = (memory.transpose(1, 2) + v) * keep[..., None]
        q, k, v = (t.view(b, n, m.heads, -1).transpose(1, 2).double() for t in (q, k, v))
        s = (q @ k.transpose(-1, -2).contiguous()) * (m.size // m.heads) ** -0.5
        w = torch.softmax(s.masked_fill(~keep[:, None, None], -torch.inf), -1)
        return m.linear_out((w @ v).transpose(1, 2).reshape(b, n, m.size).float()) + memory

    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 4 + 120, 560, generator=g).to(device)
    mask = osv.frame_mask(torch.tensor([80, 40, 120, 7]), 4, 120).to(device)
    bound = 2.0**-7 * count**0.5
    with torch.inference_mode():
        out, expected = eight(x, mask), plain(x, mask)
        close(out * mask[..., None], expected * mask[..., None], bound)
        close(eight(x[:1], None), plain(x[:1], None), bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whisper(device, dtype):
    """Encoder, prompt pass and steps."""
    import json

    from conftest import GOLDEN
    from oracle import whisper as ow
    from test_gpu_whisper import gpu_model

    from asrback_amd.linear8 import quantize_linears8

    say("8-bit whisper", dtype)
    fixture = json.loads((GOLDEN / "whisper_tiny_greedy.json").read_text())
    weights = ow.attention_heavy_weights(ow.WhisperForConditionalGeneration(fixture["config"]), fixture["seeds"]["weights"])
    eight = gpu_model(fixture, weights, device, dtype)
    held = quantize_linears8(eight)
    plain, count = with_plain_layers(eight)
    assert count == held
    # bf16: some ten more roundings of 2^-8 a layer, of about as many layers.
    bound = 2.0**-7 * count**0.5 * (1 if dtype == torch.float32 else 1.5)
    g = torch.Generator().manual_seed(2)
    mel = torch.randn(2, 80, 3000, generator=g).to(device, dtype)
    tokens = torch.randint(0, 50000, (2, 6), generator=g).to(device)
    positions = torch.arange(448, device=device)
    with torch.inference_mode():
        encoded = [m.model.encoder(mel) for m in (eight, plain)]
        close(*encoded, bound)
        caches = []
        for m in (eight, plain):
            caches.append(m.allocate_cache(2))
            m.set_encoder_output(caches[-1], encoded[1])
        close(*(m.decode(tokens[:, :4], positions[:4], c, length=4) for m, c in zip((eight, plain), caches)), bound)
        for i in (4, 5):
            at = torch.full((2,), i, device=device)
            close(*(m.decode(tokens[:, i:i + 1], at, c) for m, c in zip((eight, plain), caches)), bound)


# Plain forms of what the decoder calls.


def slots(cache, pages, row, count):
    """Entry and place in it of the row's first positions."""
    if pages is None:
        return [(row, j) for j in range(count)]
    size = cache.keys.shape[1]
    table = pages.block_table[row].tolist()
    return [(table[j // size], j % size) for j in range(count)]


def plain_write(cache, k, v, rows, positions, *, pages=None):
    rows = range(len(k)) if rows is None else rows.tolist()
    for held, scales, x in ((cache.keys, cache.key_scales, k), (cache.values, cache.value_scales, v)):
        q, scale = rounded(x)
        for t, (row, position) in enumerate(zip(rows, positions.tolist())):
            entry, at = slots(cache, pages, row, position + 1)[-1]
            if entry >= 0:
                held[entry, at] = q[t].to(torch.int8)
                scales[entry, :, at] = scale[t, :, 0].float()


def plain_write_rows(cache, q, k, v, rows, positions, *, q_norm, k_norm, q_eps, k_eps, cos, sin, pages=None, keys=False):
    def norm_rotate(x, weight, eps):
        x = x.double()
        y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()
        a, b = y.chunk(2, -1)
        return (y * cos.double()[:, None] + torch.cat((-b, a), -1) * sin.double()[:, None]).to(q.dtype)

    k = norm_rotate(k, k_norm, k_eps)
    plain_write(cache, k, v, rows, positions, pages=pages)
    return norm_rotate(q, q_norm, q_eps), k


def plain_read(cache, *, lengths, pages=None, dtype=torch.float64):
    batch, length = (cache.keys.shape[0], cache.keys.shape[1]) if pages is None else (len(pages.block_table), pages.max_len)
    out = [torch.zeros(batch, length, *cache.keys.shape[2:], dtype=dtype, device=cache.keys.device) for _ in "kv"]
    for b, n in enumerate(lengths.tolist()):
        for j, (entry, at) in enumerate(slots(cache, pages, b, min(n, length))):
            if entry >= 0:
                for x, held, scales in zip(out, (cache.keys, cache.values), (cache.key_scales, cache.value_scales)):
                    x[b, j] = (held[entry, at].double() * scales[entry, :, at, None].double()).to(dtype)
    return out


def plain_decode(q, cache, *, lengths, pages=None):
    k, v = plain_read(cache, lengths=lengths, pages=pages)
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[2]
    for b, n in enumerate(lengths.tolist()):
        kb, vb = (t[b, :n].transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
        w = torch.softmax((q[b].double()[:, None] * kb).sum(-1) * q.shape[-1] ** -0.5, -1)
        out[b] = (w[..., None] * vb).sum(1).to(q.dtype)
    return out


def plain_append(q, k, v, cache, positions, *, pages=None, **more):
    q, _ = plain_write_rows(cache, q, k, v, None, positions, pages=pages, **more)
    return plain_decode(q, cache, lengths=positions + 1, pages=pages)


@pytest.fixture
def plainly(monkeypatch):
    """A context in which the decoder calls the plain forms."""
    from asrback_amd import qwen3_asr as aq

    def context():
        patched = monkeypatch.context()
        m = patched.__enter__()
        for name, f in (("write8", plain_write), ("write_rows8", plain_write_rows), ("read8", plain_read),
                        ("decode8", plain_decode), ("decode_append8", plain_append)):
            m.setattr(aq, name, f)
        return patched

    class Context:
        def __enter__(self):
            self.patched = context()

        def __exit__(self, *args):
            self.patched.__exit__(*args)

    return Context


def caches(page, rows, device):
    from asrback_amd import qwen3_asr as aq

    if page is None:
        return aq.KVCache8.allocate(QWEN3, rows, 96, device)
    cache = aq.PagedKVCache8.allocate(QWEN3, rows, 3 * rows * 96 // page, page, device)
    for row in reversed(range(rows)):
        cache.assign(row, 96)
    return cache


def setting(device, dtype, layers8):
    from asrback_amd import qwen3_asr as aq
    from asrback_amd.linear8 import quantize_linears8

    text = qwen_pair(device)[1].to(dtype)
    layers = 4 * QWEN3["num_hidden_layers"]
    if layers8:
        assert quantize_linears8(text) == layers
    cos, sin = aq.rope_tables(QWEN3, 1024, device, dtype)
    g = torch.Generator().manual_seed(5)
    lengths = [37, 52, 1]
    ids = torch.randint(0, QWEN3["vocab_size"], (sum(lengths),), generator=g).to(device)
    rows = torch.repeat_interleave(torch.arange(3), torch.tensor(lengths)).to(device)
    positions = torch.cat([torch.arange(n) for n in lengths]).to(device)

    def prompt(model, cache):
        segments = aq.Segments.from_lengths(lengths, device)
        return model.prefill(model.embed_tokens(ids), cache, rows, positions, segments, cos[positions], sin[positions])

    # bf16: ten roundings of 2^-8 a layer of the model's two, on either side.
    bound = 2.0**-8 * (2 * 10 * QWEN3["num_hidden_layers"]) ** 0.5 if dtype == torch.bfloat16 else 2.0**-8
    if layers8:
        bound += 2.0**-7 * layers**0.5
    return text, prompt, cos, sin, torch.tensor(lengths, device=device), bound, g


@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("layers8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_and_steps(device, plainly, dtype, layers8, page):
    """Prompts into the cache and steps on from there, token by token on both sides."""
    say("8-bit steps", dtype, layers8, page)
    with torch.inference_mode():
        text, prompt, cos, sin, held, bound, g = setting(device, dtype, layers8)
        plain = with_plain_layers(text)[0] if layers8 else text
        mine, theirs = (caches(page, 3, device) for _ in "ab")
        out = prompt(text, mine)
        with plainly():
            expected = prompt(plain, theirs)
        close(out, expected, bound)
        # Hooked norms take the same sequence in parts.
        hooked = caches(page, 3, device)
        handles = [layer.self_attn.k_norm.register_forward_hook(lambda *args: None) for layer in text.layers]
        close(prompt(text, hooked), expected, bound)
        for handle in handles:
            handle.remove()
        for turn in range(5):
            tokens = torch.randint(0, QWEN3["vocab_size"], (3,), generator=g).to(device)
            out = text.step(tokens, held + turn, mine, cos, sin)
            close(text.step(tokens, held + turn, hooked, cos, sin), out, bound)
            with plainly():
                expected = plain.step(tokens, held + turn, theirs, cos, sin)
            close(out, expected, bound)
        for a, b in zip(mine.layers, theirs.layers):
            full = [plain_read(c, lengths=held + 5, pages=m.keys[0].pages) for c, m in ((a, mine), (b, theirs))]
            close(full[0][0], full[1][0], bound)
            close(full[0][1], full[1][1], bound)


@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafts(device, dtype, page):
    """A chain of drafts in one pass against single steps, which attend to the new tokens'
    rounded keys and values: 2^-7 a layer for each, about as for layers of 8 bits; and
    the accepted ones' way into the cache."""
    from asrback_amd import qwen3_asr as aq
    from asrback_amd.drafts import tree_masks

    say("8-bit drafts", dtype, page)
    with torch.inference_mode():
        text, prompt, cos, sin, held, bound, g = setting(device, dtype, False)
        bound += 2.0**-7 * (2 * QWEN3["num_hidden_layers"]) ** 0.5
        mine, theirs = (caches(page, 3, device) for _ in "ab")
        prompt(text, mine), prompt(text, theirs)
        width = 6
        tokens = torch.randint(0, QWEN3["vocab_size"], (3, width), generator=g).to(device)
        masks, depths = tree_masks(torch.arange(-1, width - 1, device=device).expand(3, width))
        drafts = aq.DraftCache.allocate(QWEN3, 3, width, device, dtype)
        before = [[t.clone() for t in layer.tensors] for layer in mine.layers]
        out = text.verify(tokens, held, mine, drafts, masks, depths, cos, sin)
        for layer, was in zip(mine.layers, before):
            assert all(torch.equal(a, b) for a, b in zip(layer.tensors, was))
        steps = torch.stack([text.step(tokens[:, i], held + i, theirs, cos, sin) for i in range(width)], 1)
        close(out, steps, bound)
        # Two rows take some of theirs, one none; what is behind stays as it was.
        path = torch.tensor([[0, 1, 2, 3, -1, -1], [0, 1, -1, 3, 4, 5], [0, 1, 2, 3, 4, 5]], device=device)
        count = torch.tensor([4, 2, 0], device=device)
        drafts.commit(mine, path, count, held)
        for index, (a, b, was) in enumerate(zip(mine.layers, theirs.layers, before)):
            pages = mine.keys[index].pages
            for tensors, drafted, step in zip(plain_read(a, lengths=held + width, pages=pages), (drafts.keys, drafts.values),
                                              plain_read(b, lengths=held + width, pages=theirs.keys[index].pages)):
                for row in range(3):
                    n, new = int(held[row]), int(count[row])
                    q, scale = rounded(drafted[index][row, :new])
                    assert torch.equal(tensors[row, n:n + new], q * scale)
                    assert not tensors[row, n + new:].any()
                    if new:
                        close(tensors[row, n:n + new], step[row, n:n + new], bound)


@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafts_see_the_cache_as_it_reads_back(device, dtype, page):
    """A pass over an 8-bit cache is one over a cache of the model's type that holds what
    reading the 8-bit one back gives, to the bit."""
    from asrback_amd import qwen3_asr as aq
    from asrback_amd.cache8 import read8
    from asrback_amd.drafts import tree_masks

    say("8-bit drafts read back", dtype, page)
    with torch.inference_mode():
        text, prompt, cos, sin, held, _, g = setting(device, dtype, False)
        mine = caches(page, 3, device)
        prompt(text, mine)
        plain = aq.KVCache.allocate(QWEN3, 3, mine.keys[0].shape[1], device, dtype)
        for index, layer in enumerate(mine.keys):
            plain.keys[index], plain.values[index] = read8(layer.cache, pages=layer.pages, dtype=dtype)
        width = 7
        tokens = torch.randint(0, QWEN3["vocab_size"], (3, width), generator=g).to(device)
        parents = torch.tensor([-1, 0, 0, 1, 1, 3, 2], device=device).expand(3, width)
        masks, depths = tree_masks(parents)
        out = [text.verify(tokens, held, cache, aq.DraftCache.allocate(QWEN3, 3, width, device, dtype), masks, depths, cos, sin)
               for cache in (mine, plain)]
        assert torch.equal(*out)


def drained(decoder, prompts, tokens):
    admitted = decoder.admit(prompts, tokens)
    results = {}
    while decoder.rows:
        decoder.advance()
        results |= decoder.finished_rows()
    return [results[s] for s in admitted]


@pytest.mark.parametrize("layers8", [False, True])
def test_decoder(device, layers8):
    """The whole decode loop: step by step, from graphs, from pages and by drafts."""
    from asrback_amd import qwen3_asr as aq
    from asrback_amd.linear8 import Linear8, quantize_linears8

    say("8-bit decoder", layers8)
    whole, prompts, _ = _qwen_decoder(device, False, [])
    text, head = whole.text, whole.lm_head
    if layers8:
        quantize_linears8(text)
        head = Linear8.from_linear(head)

    def decoder(**how):
        return aq.TextGreedyDecoder(text, head, QWEN3, 4, [], cache_bits=8, **how)

    eager = drained(decoder(graphs=False), prompts, 20)
    assert all(len(tokens) == 20 for tokens, _ in eager)
    for how in ({"graphs": True}, {"graphs": False, "page_size": 16, "num_pages": 14},
                {"graphs": True, "page_size": 64, "num_pages": 9}):
        made = decoder(**how)
        for _ in range(2):  # the same rows again
            assert drained(made, prompts, 20) == eager
        if "num_pages" in how:
            assert sorted(made.cache.free_pages) == list(range(how["num_pages"]))
            assert isinstance(made.cache, aq.PagedKVCache8)
    held = sum(t.numel() * t.element_size() for layer in made.cache.layers for t in layer.tensors)
    assert held == 9 * 64 * QWEN3["num_hidden_layers"] * 2 * QWEN3["num_key_value_heads"] * (QWEN3["head_dim"] + 4)
    # Drafted trees: the greedy tokens of the passes, whose first are the prompt's.
    for how in ({"graphs": False}, {"graphs": True, "draft_tokens": 5}, {"graphs": True, "draft_tokens": 5, "page_size": 16}):
        made = decoder(**how)
        admitted = made.admit(prompts, 20)
        passes, results = 0, {}
        while made.rows:
            drafted = torch.zeros(max(made.rows) + 1, 5, dtype=torch.int64)
            position = made.state.position.tolist()
            for slot, (tokens, _) in zip(admitted, eager):
                if slot in made.rows:
                    at = position[slot] - made.rows[slot]["prompt_length"] + 1
                    part = tokens[at:at + 4]
                    drafted[slot, 1:1 + len(part)] = torch.tensor(part)
            made.verify(drafted.to(device), torch.arange(-1, 4, device=device))
            results |= made.finished_rows()
            passes += 1
        assert 4 <= passes <= 19
        for slot, (tokens, _) in zip(admitted, eager):
            assert len(results[slot][0]) == 20 and results[slot][0][0] == tokens[0]
    with pytest.raises(ValueError, match="cache_bits"):
        aq.TextGreedyDecoder(text, head, QWEN3, 4, [], cache_bits=4)


def test_gated_block(device):
    """The feed-forward block: one product where the layer is its class's own, the two
    steps where it has a hook."""
    from asrback_amd import qwen3_asr as aq
    from asrback_amd.linear8 import quantize_linears8

    for dtype in (torch.float32, torch.bfloat16):
        torch.manual_seed(1)
        mlp = aq.TextMLP(QWEN3).to(device, dtype)
        assert quantize_linears8(mlp) == 2
        plain, _ = with_plain_layers(mlp)
        x = torch.randn(3, 7, QWEN3["hidden_size"], device=device, dtype=dtype)
        # The second layer's roundings; the block's own in bf16: three of 2^-8 (the plain
        # forms' gates, projections and activations).
        bound = 2.0**-7 + (2.0**-8 * 3 if dtype == torch.bfloat16 else 0)
        with torch.inference_mode():
            say("gated block", dtype)
            out = mlp(x)
            close(out, plain(x), bound)
            seen = []
            handle = mlp.gate_up_proj.register_forward_hook(lambda m, args, y: seen.append(y.shape))
            close(mlp(x), out, bound)
            assert seen == [(3, 7, 2 * QWEN3["intermediate_size"])]
            handle.remove()
            assert torch.equal(mlp(x), out)
