"""GPU: Qwen3-ASR's decoder on drafted trees (tree attention, greedy choice,
acceptance and commit together, with and without 4-bit weights): the tokens and
scores that single greedy steps give, in fewer passes.

Float32 models whose choices are far from ties, so the tokens have to be equal.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_models import QWEN3, _drain, _qwen_decoder

pytestmark = pytest.mark.gpu


def say(*args):
    print(*args, flush=True)


def drafts_for(decoder, known, width, g, right=0.8):
    """Random trees for every slot up to the last occupied one: each token hangs on
    an earlier one; where its branch has been right so far, it is the model's
    next token more often than not."""
    rows = max(decoder.rows) + 1
    tokens = torch.randint(0, QWEN3["vocab_size"], (rows, width), generator=g)
    parents = torch.full((rows, width), -2)
    state = decoder.state
    for slot in range(rows):
        if slot not in known:
            tokens[slot] = -1  # a free row's padding
            continue
        done = int(state.position[slot]) - decoder.rows[slot]["prompt_length"] + 1
        depth_right = {0: 0}  # tokens of a right branch, and how far they reach
        parents[slot, 0] = -1
        tokens[slot, 0] = -7  # not read
        for i in range(1, width):
            if float(torch.rand((), generator=g)) < 0.1:
                continue  # padding inside the tree
            parent = int(torch.randint(max(-1, i - 4), i, (1,), generator=g))
            parents[slot, i] = parent
            at = done + depth_right[parent] if parent in depth_right else len(known[slot])
            if at < len(known[slot]) and float(torch.rand((), generator=g)) < right:
                tokens[slot, i] = known[slot][at]
                depth_right[i] = depth_right[parent] + 1
    return tokens.to(decoder.device), parents.to(decoder.device)


def drain_by_drafts(decoder, known, width, g, results, right=0.8):
    passes = 0
    while decoder.rows:
        decoder.verify(*drafts_for(decoder, known, width, g, right))
        passes += 1
        for slot, outcome in decoder.finished_rows().items():
            results[slot] = outcome
            known.pop(slot)
    return passes


@pytest.mark.parametrize("width,graphs,cache", [
    (1, False, {}), (2, True, {"draft_tokens": 2}), (9, True, {"draft_tokens": 9}), (9, True, {"draft_tokens": 4}),
    (16, False, {"page_size": 16, "num_pages": 14}), (16, True, {"page_size": 16, "num_pages": 14, "draft_tokens": 16}),
    (64, True, {"page_size": 64, "draft_tokens": 64}), (33, False, {}),
])
def test_drafts_give_the_greedy_tokens(device, width, graphs, cache):
    say("verify", width, graphs, cache)
    decoder, prompts, expected = _qwen_decoder(device, graphs, [989], **cache)
    steps = {}
    slots = decoder.admit(prompts, 12)
    while decoder.rows:
        decoder.advance()
        steps |= decoder.finished_rows()
    want = [steps[s] for s in slots]
    assert [w[0] for w in want] == expected
    for right in (1.0, 0.7, 0.0):
        g = torch.Generator().manual_seed(width)
        slots = decoder.admit(prompts, 12)
        # The end of sequence is among the drafts, and tokens behind it.
        known = {s: [*e, 989, 5, 6][:15] for s, e in zip(slots, expected)}
        results = {}
        passes = drain_by_drafts(decoder, known, width, g, results, right)
        assert [results[s][0] for s in slots] == expected
        for s, w in zip(slots, want):
            assert results[s][1] == pytest.approx(w[1], abs=1e-4)
        if width >= 9 and right == 1.0:
            assert passes < 11  # what single steps take
        if right == 0.0:
            assert passes >= 10
    if cache.get("num_pages"):
        assert sorted(decoder.cache.free_pages) == list(range(14))


def test_drafts_and_steps_in_turn(device):
    """Rows admitted between passes, steps between trees."""
    say("verify, staggered")
    decoder, prompts, expected = _qwen_decoder(device, True, [], draft_tokens=5)
    g = torch.Generator().manual_seed(3)
    first = decoder.admit(prompts[:2], 12)
    known = dict(zip(first, expected))
    decoder.verify(*drafts_for(decoder, known, 5, g))
    decoder.advance()
    results = {s: r for s, r in decoder.finished_rows().items()}
    third = decoder.admit(prompts[2:], 12)
    known |= dict(zip(third, expected[2:]))
    for s in results:
        known.pop(s)
    decoder.verify(*drafts_for(decoder, known, 7, g))  # another size: eager
    results |= decoder.finished_rows()
    rest = {}
    _drain(decoder, rest)
    results = {s: r[0] for s, r in results.items()} | rest
    # A finished row's slot is taken over by the third window.
    got = [results.get(s) for s in first + third]
    assert got[2] == expected[2] and all(x in (e, expected[2]) for x, e in zip(got, expected))
    with pytest.raises(RuntimeError, match="no occupied"):
        decoder.verify(torch.zeros(1, 5, dtype=torch.int64, device=device), torch.zeros(5, dtype=torch.int64, device=device))
    decoder.admit(prompts[:2], 12)
    zeros = torch.zeros(2, 5, dtype=torch.int64, device=device)
    for bad, parents in ((zeros[:1], zeros[0]), (zeros.int(), zeros[0]), (zeros, zeros[:, :4]), (zeros, zeros[0].int()),
                         (zeros.new_zeros(2, 65), zeros.new_zeros(65)), (zeros[:, :0], zeros[0, :0])):
        with pytest.raises(ValueError):
            decoder.verify(bad, parents)


@pytest.mark.parametrize("symmetric", [True, False])
def test_drafts_through_4_bit_layers(device, symmetric):
    """The whole run of operators: drafted trees through 4-bit layers against the
    same layers' single steps, and the layers against their unpacked matrices."""
    from asrback_amd.linear4 import Linear4, quantize_linears, unpack4
    from asrback_amd.qwen3_asr import TextGreedyDecoder

    say("verify, 4 bits", symmetric)
    decoder, prompts, _ = _qwen_decoder(device, False, [])
    text = decoder.text
    assert quantize_linears(text, 32, symmetric) == 4 * QWEN3["num_hidden_layers"]
    head = Linear4.from_linear(decoder.lm_head, 32, symmetric)
    four = TextGreedyDecoder(text, head, QWEN3, 4, [], graphs=True, page_size=16, draft_tokens=8)
    slots = four.admit(prompts, 20)
    steps = {}
    while four.rows:
        four.advance()
        steps |= four.finished_rows()
    slots = four.admit(prompts, 20)
    known = {s: steps[s][0] for s in slots}
    results = {}
    passes = drain_by_drafts(four, dict(known), 8, torch.Generator().manual_seed(8), results, 0.9)
    assert passes < 19
    assert {s: r[0] for s, r in results.items()} == known
    # The same model with its rounded matrices unpacked into plain layers.
    for parent in list(text.modules()):
        for name, child in list(parent.named_children()):
            if type(child) is Linear4:
                plain = torch.nn.Linear(child.in_features, child.out_features, bias=False, device=device)
                plain.weight.data.copy_(unpack4(child.weight4))
                setattr(parent, name, plain)
    plain = torch.nn.Linear(head.in_features, head.out_features, bias=False, device=device)
    plain.weight.data.copy_(unpack4(head.weight4))
    whole = TextGreedyDecoder(text, plain, QWEN3, 4, [], graphs=False)
    slots = whole.admit(prompts, 20)
    results = {}
    _drain(whole, results)
    assert {s: results[s] for s in slots} == known


def test_bf16_verify_pass_matches_prefill(device):
    """One bf16 pass over trees of a wider model (16 query heads over 8 of 128)
    against the prompt pass over each branch: normwise 2^-5, three roundings of
    half a step (2^-8) in each of some ten layers' operations growing as their
    square root."""
    from asrback_amd import qwen3_asr as aq
    from asrback_amd.drafts import tree_masks

    config = {"hidden_size": 256, "head_dim": 128, "num_attention_heads": 16, "num_key_value_heads": 8,
              "rms_norm_eps": 1e-6, "rope_theta": 1e6, "num_hidden_layers": 2, "vocab_size": 500,
              "intermediate_size": 512}
    torch.manual_seed(0)
    text = aq.TextModel(config).to(device, torch.bfloat16)
    cos, sin = aq.rope_tables(config, 256, device, torch.bfloat16)
    lengths = [90, 33, 0]
    parents = [[-1, 0, 0, 1, 3, 2, 5, 5], [-1, 0, 1, 2, 3, 4, 5, 6], [-1, 0, 0, 0, 0, 1, 2, -2]]
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (n,), generator=g).to(device) for n in lengths]
    drafted = torch.randint(0, 500, (3, 8), generator=g).to(device)
    say("verify bf16")
    with torch.inference_mode():
        cache = aq.KVCache.allocate(config, 3, 256, device, torch.bfloat16)

        def prefill(row, tokens, into):
            positions = torch.arange(len(tokens), device=device)
            rows = torch.full_like(positions, row)
            return text.prefill(text.embed_tokens(tokens), into, rows, positions,
                                aq.Segments.from_lengths([len(tokens)], device), cos[positions], sin[positions])

        for row, prompt in enumerate(prompts):
            if len(prompt):
                prefill(row, prompt, cache)
        before = cache.keys.clone()
        drafts = aq.DraftCache.allocate(config, 3, 8, device, torch.bfloat16)
        masks, depths = tree_masks(torch.tensor(parents, device=device))
        hidden = text.verify(drafted, torch.tensor(lengths, device=device), cache, drafts, masks, depths, cos, sin)
        assert torch.equal(cache.keys, before)  # nothing is committed yet
        scratch = aq.KVCache.allocate(config, 3, 256, device, torch.bfloat16)
        for row in range(3):
            for t in range(8):
                branch, at = [], t
                while at >= 0:
                    branch.insert(0, at)
                    at = parents[row][at]
                if at < -1:
                    continue
                want = prefill(row, torch.cat((prompts[row], drafted[row, branch])), scratch)[-1]
                error = float((hidden[row, t].double() - want.double()).norm() / want.double().norm())
                assert error < 2.0**-5, (row, t, error)
        path = torch.tensor([[0, 2, 5, 7, -1, -1, -1, -1], [0, 1, -1, -1, -1, -1, -1, -1], [-1] * 8], device=device)
        count = torch.tensor([4, 2, 0], device=device)
        drafts.commit(cache, path, count, torch.tensor(lengths, device=device))
        changed = (cache.keys != before).flatten(3).any(-1).any(0)
        assert changed.nonzero().tolist() == [[0, 90], [0, 91], [0, 92], [0, 93], [1, 33], [1, 34]]
        assert torch.equal(cache.values[:, 0, 92], drafts.values[:, 0, 5])


def test_steps_after_rejected_drafts(device):
    """Passes that accept one token of a wide tree leave the next steps their count."""
    from asrback_amd.qwen3_asr import EOS_CHECK_INTERVAL

    say("steps after rejected drafts")
    decoder, prompts, expected = _qwen_decoder(device, True, [], draft_tokens=16)
    slots = decoder.admit(prompts, 12)
    width = torch.zeros(len(prompts), 16, dtype=torch.int64, device=device)
    wrong = width + torch.tensor([0] + [QWEN3["vocab_size"]] * 15, device=device)  # no token
    for taken in (1, 2):
        decoder.verify(wrong, torch.tensor([-1] + [0] * 15, device=device))
        assert decoder.finished_rows() == {}
        assert all(decoder.rows[s]["bound"] == decoder.rows[s]["prompt_length"] + taken for s in slots)
    assert decoder.advance() == EOS_CHECK_INTERVAL
    results = {}
    _drain(decoder, results)
    assert [results[s] for s in slots] == expected


def test_eager_passes_on_the_decoders_workspace(device):
    """Without graphs, trees of draft_tokens tokens take the decoder's workspace, at row
    counts between the buckets too."""
    say("eager, workspace")
    decoder, prompts, expected = _qwen_decoder(device, False, [], draft_tokens=16)
    slots = decoder.admit(prompts, 12)
    assert max(slots) + 1 == 3 not in decoder.buckets
    results = {}
    drain_by_drafts(decoder, dict(zip(slots, expected)), 16, torch.Generator().manual_seed(4), results)
    assert [results[s][0] for s in slots] == expected
