"""GPU: drafted trees -- masks, attention, acceptance, commit -- against plain
float64 on the CPU.

Attention's bound, per element, from what the kernel rounds.  With A = the
weights times |v| (the reference's weights), the output's absolute error is at
most

    2^-8 (A + |ref|)            bf16: each weight and the output once
    2^-24 A (2 (d + 8) S + n + 64)   float32 work: scores, exponentials, sums

times 1.01 for second-order terms, where S is the largest sum of |q| |k| scale over
a row's keys (a score's d products and sums are each off by 2^-24 of at most
S, its scaling, the maximum's subtraction and the exponential by 8 more; weights
and their sum both carry them), and n the row's keys (two sums).  float32 inputs
round the output to 2^-24 |ref|.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def say(*args):
    print(*args, flush=True)


def random_parents(tokens, g, padding=0):
    """Each token's parent is any earlier one, or (now and then) the context."""
    parents = [-1]
    for i in range(1, tokens):
        p = int(torch.randint(-1, i, (1,), generator=g))
        parents.append(p)
    for i in range(tokens - padding, tokens):
        parents[i] = -2
    return parents


def reference_masks(parents):
    masks = []
    for i, p in enumerate(parents):
        masks.append(0 if p < -1 else 1 << i | (masks[p] if 0 <= p < i else 0))
    return masks


def signed(masks):
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def reference(q, k, v, kd, vd, masks, lengths, scale):
    """Output, weights times |v|, and the largest |q| |k| scale sum and key count
    per row; k and v are lists of each row's (n, heads, d) cache."""
    q, kd, vd = (t.double().cpu() for t in (q, kd, vd))
    batch, tokens, heads, d = q.shape
    group = heads // kd.shape[2]
    out, absolute = torch.zeros_like(q), torch.zeros_like(q)
    slack = torch.zeros(batch, tokens, heads, 1, dtype=torch.float64)
    for b in range(batch):
        kb, vb = k[b].double().cpu(), v[b].double().cpu()
        for t in range(tokens):
            mask = masks[b][t]
            if mask == 0:
                continue
            seen = [i for i in range(tokens) if mask >> i & 1]
            kk, vv = torch.cat((kb, kd[b, seen])), torch.cat((vb, vd[b, seen]))
            if len(kk) == 0:
                continue
            for h in range(heads):
                s = kk[:, h // group] @ q[b, t, h] * scale
                w = torch.softmax(s, 0)
                out[b, t, h] = w @ vv[:, h // group]
                absolute[b, t, h] = w @ vv[:, h // group].abs()
                top = (kk[:, h // group].abs() @ q[b, t, h].abs()).max() * scale
                slack[b, t, h] = 2 * (d + 8) * top + len(kk) + 64
    return out, absolute, slack


def check(got, ref, absolute, slack, dtype, label):
    got = got.double().cpu()
    bound = 2.0**-24 * absolute * slack
    bound += 2.0**-8 * (absolute + ref.abs()) if dtype == BF16 else 2.0**-24 * ref.abs()
    bad = ~((got - ref).abs() <= 1.01 * bound + 1e-38)  # NaN is bad
    assert not bad.any(), f"{label}: {int(bad.sum())} of {bad.numel()} elements, worst {float(((got - ref).abs() / bound.clamp(min=1e-38)).max()):.3g} of the bound"


def make(dtype, batch, tokens, heads, kv_heads, d, length, page, g, layout="slab", spare=3):
    """Tensors, and each row's cache as the slab it stands for."""
    q = torch.randn(batch, tokens, heads, d, generator=g).to("cuda", dtype)
    kd, vd = (torch.randn(batch, tokens, kv_heads, d, generator=g).to("cuda", dtype) for _ in range(2))
    k, v = (torch.randn(batch, length, kv_heads, d, generator=g).to("cuda", dtype) for _ in range(2))
    if layout == "heads_first":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    if not page:
        return q, k, v, kd, vd, None, k, v
    from asrback_amd.attention import PageTable

    per = -(-length // page)
    order = torch.randperm(batch * per + spare, generator=g)[:batch * per].view(batch, per)
    pool_k, pool_v = (torch.full((batch * per + spare, page, kv_heads, d), float("nan"), device="cuda", dtype=dtype)
                      for _ in range(2))
    for pool, t in ((pool_k, k), (pool_v, v)):
        for b in range(batch):
            for i in range(per):
                part = t[b, i * page:(i + 1) * page]
                pool[order[b, i], :len(part)] = part
    return q, pool_k, pool_v, kd, vd, PageTable(order.int().cuda(), length), k, v


CASES = [
    # dtype, batch, tokens, heads, kv_heads, head_dim, length, lengths, page, layout
    (BF16, 1, 1, 1, 1, 64, 1, [1], 0, "slab"),
    (BF16, 2, 1, 16, 8, 128, 100, [0, 100], 0, "slab"),
    (F32, 2, 1, 6, 6, 64, 33, [0, 33], 0, "heads_first"),
    (BF16, 4, 7, 4, 2, 128, 70, [15, 16, 17, 70], 0, "slab"),
    (BF16, 3, 16, 6, 2, 128, 130, [31, 32, 33], 0, "heads_first"),
    (F32, 3, 9, 6, 2, 64, 130, [31, 47, 129], 0, "slab"),
    (F32, 2, 17, 4, 4, 128, 300, [300, 255], 0, "slab"),
    (BF16, 2, 33, 6, 2, 64, 513, [513, 1], 0, "slab"),
    (BF16, 1, 64, 8, 1, 128, 260, [259], 0, "slab"),
    (F32, 1, 64, 4, 1, 128, 260, [259], 0, "slab"),
    (BF16, 2, 64, 8, 4, 256, 200, [200, 77], 0, "slab"),
    (F32, 2, 20, 8, 4, 256, 90, [90, 77], 0, "slab"),
    (BF16, 3, 5, 4, 2, 256, 40, [0, 3, 40], 0, "slab"),
    # split keys: few rows over long caches
    (BF16, 1, 3, 2, 1, 128, 4096, [4095], 0, "slab"),
    (BF16, 1, 30, 2, 1, 128, 5000, [4001], 0, "slab"),
    (BF16, 2, 12, 8, 2, 64, 3000, [2999, 2], 0, "heads_first"),
    (F32, 1, 6, 3, 3, 64, 2100, [2100], 0, "slab"),
    (BF16, 1, 24, 2, 1, 256, 2000, [1999], 0, "slab"),
    # of up to four rows: of four waves
    (BF16, 1, 1, 16, 8, 128, 4096, [3001], 0, "slab"),
    (F32, 1, 2, 6, 6, 64, 2100, [2077], 0, "heads_first"),
    (BF16, 1, 4, 2, 2, 64, 3000, [2999], 64, "slab"),
    (BF16, 2, 1, 8, 2, 256, 1500, [1499, 0], 0, "slab"),
    # many rows over long caches: two row tiles a workgroup, several workgroups a kv head
    (BF16, 1, 61, 8, 1, 128, 20000, [17000], 0, "slab"),
    (BF16, 1, 64, 8, 1, 64, 20000, [19999], 64, "slab"),
    (F32, 1, 64, 8, 1, 64, 20000, [1234], 0, "heads_first"),
    # more workgroups than CUs: four waves each
    (BF16, 33, 2, 16, 8, 128, 96, [33, 96, 0, 1] * 8 + [17], 32, "slab"),
    (F32, 40, 1, 8, 8, 128, 64, [33, 64, 0, 1] * 10, 0, "slab"),
    (BF16, 70, 3, 8, 4, 256, 48, [33, 48, 0, 1, 20] * 14, 0, "slab"),
    (F32, 22, 17, 12, 4, 128, 64, [33, 64, 0, 1] * 5 + [5, 50], 0, "slab"),
    (F32, 17, 18, 16, 4, 256, 64, [33, 64, 0, 1] * 4 + [50], 0, "slab"),
    (BF16, 16, 40, 8, 4, 128, 1536, [33, 500, 0, 1] * 4, 0, "slab"),
    (BF16, 22, 40, 8, 4, 64, 1024, [33, 300, 0, 1] * 5 + [1024, 17], 64, "slab"),
    (BF16, 16, 40, 8, 4, 128, 1536, [33, 500, 0, 130] * 4, 128, "slab"),
    (F32, 22, 40, 8, 4, 64, 1024, [33, 300, 0, 1] * 5 + [200, 17], 0, "slab"),
    # pages: shorter than a tile, of one tile, longer; a last page in part
    (BF16, 3, 8, 4, 2, 128, 112, [111, 16, 0], 16, "slab"),
    (BF16, 2, 8, 4, 2, 128, 448, [447, 130], 64, "slab"),
    (F32, 2, 5, 4, 2, 64, 448, [447, 130], 16, "slab"),
    (BF16, 2, 40, 4, 2, 64, 1024, [1000, 513], 128, "slab"),
    (BF16, 1, 4, 4, 1, 256, 2048, [2041], 32, "slab"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:7]) + f"-p{c[8]}")
def test_tree_attention_matches_float64(case):
    from asrback_amd import drafts

    dtype, batch, tokens, heads, kv_heads, d, length, lengths, page, layout = case
    say("tree", case)
    g = torch.Generator().manual_seed(tokens * 1000 + length)
    q, k, v, kd, vd, pages, k_rows, v_rows = make(dtype, batch, tokens, heads, kv_heads, d, length, page, g, layout)
    parents = [random_parents(tokens, g, padding=(b % 2) * min(2, tokens - 1)) for b in range(batch)]
    masks = [reference_masks(p) for p in parents]
    device_masks, depths = drafts.tree_masks(torch.tensor(parents, device="cuda"))
    assert device_masks.tolist() == [signed(m) for m in masks]
    assert depths.tolist() == [[max(bin(m).count("1") - 1, 0) for m in row] for row in masks]
    out = drafts.tree_attention(q, k, v, kd, vd, device_masks, lengths=torch.tensor(lengths, device="cuda"), pages=pages)
    torch.cuda.synchronize()
    ref, absolute, slack = reference(q, [k_rows[b, :n] for b, n in enumerate(lengths)],
                                     [v_rows[b, :n] for b, n in enumerate(lengths)], kd, vd, masks, lengths, d**-0.5)
    check(out, ref, absolute, slack, dtype, str(case))
    # The same bits again: nothing depends on the order in which splits arrive.
    again = drafts.tree_attention(q, k, v, kd, vd, device_masks,
                                  lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32), pages=pages)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,page", [(64, 0), (128, 16), (128, 0), (256, 0)])
def test_masked_places_hold_anything(dtype, d, page):
    """NaN and infinities past a row's keys, in padded tokens and in drafted
    tokens that a row does not see leave its output alone; the rows that see them
    get what the formula gives."""
    from asrback_amd import drafts

    say("masked", dtype, d, page)
    g = torch.Generator().manual_seed(d + page)
    tokens, kv_heads, length, lengths = 37, 2, 96, [41, 96, 0]
    q, k, v, kd, vd, pages, _, _ = make(dtype, 3, tokens, 4, kv_heads, d, length, page, g)
    rows_k, rows_v = [], []
    for b, n in enumerate(lengths):
        for cache, rows in ((k, rows_k), (v, rows_v)):
            if page:
                at = torch.arange(length)
                where = pages.block_table.cpu()[b].long()[at // page], at % page
            else:
                where = torch.full((length,), b), torch.arange(length)
            where = tuple(x.cuda() for x in where)
            rows.append(cache[where][:n].clone())
            junk = torch.full_like(cache[where][n:], float("nan"))
            junk[::2] = float("inf")
            cache[tuple(x[n:] for x in where)] = junk
    # A chain 0..4, then leaves of token 4, the last three tokens padding.
    parents = [-1, 0, 1, 2, 3] + [4] * 29 + [-2] * 3
    masks = [reference_masks(parents)] * 3
    kd[:, 34:], vd[:, 34:], q[:, 34:] = float("nan"), float("-inf"), float("nan")
    vd[0, 7, 0, ::3] = float("inf")
    vd[0, 7, 0, 1] = float("nan")
    vd[1, 20, 1] = float("-inf")
    kd[1, 9] = float("nan")
    vd[2, 33, :, -1] = float("nan")
    device_masks = torch.tensor(signed(masks[0]), device="cuda")  # one tree in every row
    out = drafts.tree_attention(q, k, v, kd, vd, device_masks, lengths=torch.tensor(lengths, device="cuda"), pages=pages)
    torch.cuda.synchronize()
    ref, absolute, slack = reference(q, rows_k, rows_v, kd, vd, masks, lengths, d**-0.5)
    fine = ref.isfinite()
    got = out.double().cpu()
    assert torch.equal(got[~fine].nan_to_num(7.0), ref[~fine].nan_to_num(7.0))  # infinities' signs, NaN
    assert 0 < int((~fine).sum()) < fine.numel() // 10
    assert not got[:, 34:].any() and not got[:, 34:].isnan().any()
    zero = torch.zeros(())
    check(torch.where(fine, got, zero), torch.where(fine, ref, zero.double()),
          torch.where(fine, absolute, zero.double()), torch.where(slack.isfinite(), slack, zero.double()), dtype, "masked")


@pytest.mark.parametrize("dtype,batch,d,length", [(BF16, 24, 128, 1536), (BF16, 8, 64, 4096), (F32, 24, 64, 1536),
                                                  (BF16, 24, 256, 64), (F32, 24, 128, 64)])
def test_infinite_drafted_values_stay_with_their_rows(dtype, batch, d, length):
    """Launches of two row tiles and of four waves: infinities and NaN in two
    dimensions of a drafted value reach those dimensions of the rows that see it
    and change no other bit."""
    from asrback_amd import drafts

    say("infinite drafts", dtype, batch, d, length)
    g = torch.Generator().manual_seed(d + length)
    tokens, kv_heads = 33, 4
    q, k, v, kd, vd, _, _, _ = make(dtype, batch, tokens, 2 * kv_heads, kv_heads, d, length, 0, g)
    parents = torch.tensor([random_parents(tokens, g, padding=2) for _ in range(batch)])
    masks, _ = drafts.tree_masks(parents.cuda())
    lengths = torch.randint(0, 60, (batch,), generator=g).cuda()
    bad = (7, 20)
    vd[:, bad[0], :, 5] = 0.0
    vd[:, bad[1], :, d - 1] = 0.0
    clean = drafts.tree_attention(q, k, v, kd, vd, masks, lengths=lengths)
    vd[:, bad[0], :, 5] = float("inf")
    vd[:, bad[1], :, d - 1] = float("nan")
    out = drafts.tree_attention(q, k, v, kd, vd, masks, lengths=lengths)
    sees = [(masks >> j & 1).bool() for j in bad]
    assert sees[0].sum() > batch and sees[1].sum() > batch // 2
    assert not out[..., 5][sees[0]].isfinite().any() and out[..., d - 1][sees[1]].isnan().all()
    out[..., 5][sees[0]] = clean[..., 5][sees[0]]
    out[..., d - 1][sees[1]] = clean[..., d - 1][sees[1]]
    assert torch.equal(out, clean)


def test_missing_pages_and_counts_out_of_range():
    """Keys on no page or on one outside the pool are skipped; counts are clamped
    to the cache."""
    from asrback_amd import drafts
    from asrback_amd.attention import PageTable

    g = torch.Generator().manual_seed(5)
    q, k, v, kd, vd, pages, k_rows, v_rows = make(BF16, 3, 6, 4, 2, 128, 128, 16, g)
    table = pages.block_table.clone()
    table[0, 2], table[0, 5], table[1, 0] = -1, k.shape[0], 1 << 30
    gone = [(2, 5), (0,), ()]
    lengths = [100, 1 << 40, -7]
    used = [100, 128, 0]
    keep = [[j for j in range(n) if j // 16 not in skip] for n, skip in zip(used, gone)]
    masks = [reference_masks([-1, 0, 0, 1, 2, 2])] * 3
    say("missing pages")
    out = drafts.tree_attention(q, k, v, kd, vd, torch.tensor(masks, device="cuda"),
                                lengths=torch.tensor(lengths, device="cuda"), pages=PageTable(table, 128))
    ref, absolute, slack = reference(q, [k_rows[b, j] for b, j in enumerate(keep)],
                                     [v_rows[b, j] for b, j in enumerate(keep)], kd, vd, masks, used, 128**-0.5)
    check(out, ref, absolute, slack, BF16, "missing pages")
    # No lengths: the whole cache; mask bits past the tokens count for nothing.
    say("whole cache, stray bits")
    stray = torch.tensor(masks, device="cuda") | (1 << 50) | (1 << 6)
    out = drafts.tree_attention(q, k_rows, v_rows, kd, vd, stray)
    ref, absolute, slack = reference(q, list(k_rows), list(v_rows), kd, vd, masks, [128] * 3, 128**-0.5)
    check(out, ref, absolute, slack, BF16, "whole cache")
    # A cache of no positions at all.
    say("empty cache")
    empty = k_rows[:, :0]
    out = drafts.tree_attention(q, empty, empty, kd, vd, torch.tensor(masks, device="cuda"))
    ref, absolute, slack = reference(q, list(empty), list(empty), kd, vd, masks, [0] * 3, 128**-0.5)
    check(out, ref, absolute, slack, BF16, "empty cache")


def test_strides_offsets_past_32_bits_and_given_out():
    """A cache whose positions lie 80 KiB apart (its last past 5 GiB), queries out of
    a fused projection, an out whose rows are not 16-byte aligned."""
    from asrback_amd import drafts

    g = torch.Generator().manual_seed(6)
    length, apart = 66000, 40960
    base = torch.empty(length * apart, dtype=BF16, device="cuda")
    k = base.as_strided((1, length, 1, 64), (0, apart, 64, 1))
    v = base.as_strided((1, length, 1, 64), (0, apart, 64, 1), 128)
    k.copy_(torch.randn(1, length, 1, 64, generator=g))
    v.copy_(torch.randn(1, length, 1, 64, generator=g))
    fused = torch.randn(1, 5, 4, 3, 64, generator=g).to("cuda", BF16)
    q = fused[:, :, :, 1]
    kd, vd = (torch.randn(1, 5, 1, 64, generator=g).to("cuda", BF16) for _ in range(2))
    masks = [reference_masks([-1, 0, 0, 2, 1])]
    held = torch.zeros(1, 5, 4, 67, dtype=BF16, device="cuda")
    say("long strides")
    out = drafts.tree_attention(q, k, v, kd, vd, torch.tensor(masks, device="cuda"), out=held[..., 1:65],
                                lengths=torch.tensor([65999], device="cuda"))
    assert out.data_ptr() == held.data_ptr() + 2
    ref, absolute, slack = reference(q, [k[0, :65999]], [v[0, :65999]], kd, vd, masks, [65999], 0.125)
    check(out, ref, absolute, slack, BF16, "long strides")
    assert not held[..., 0].any() and not held[..., 65:].any()
    # Rows that share one key and value (stride 0).
    say("expanded")
    one_k, one_v = (t[:, :1].expand(1, 40, 1, 64) for t in (k, v))
    out = drafts.tree_attention(q, one_k, one_v, kd, vd, torch.tensor(masks, device="cuda"), scale=0.3,
                                lengths=torch.tensor([39], device="cuda"))
    ref, absolute, slack = reference(q, [one_k[0, :39]], [one_v[0, :39]], kd, vd, masks, [39], 0.3)
    check(out, ref, absolute, slack, BF16, "expanded")


def test_graphs_sharing_a_workspace_and_other_streams():
    """Two captured graphs on one workspace, replayed in turn with eager calls and
    changed inputs between, and a call on a side stream."""
    from asrback_amd import attention, drafts

    g = torch.Generator().manual_seed(7)
    shapes = [(BF16, 1, 9, 4, 2, 128, 3000, 0), (F32, 1, 5, 4, 4, 64, 2500, 0)]
    sets = []
    need = 0
    for dtype, batch, tokens, heads, kv, d, length, page in shapes:
        q, k, v, kd, vd, pages, _, _ = make(dtype, batch, tokens, heads, kv, d, length, page, g)
        masks, _ = drafts.tree_masks(torch.tensor(random_parents(tokens, g), device="cuda"))
        lengths = torch.tensor([length - 7], device="cuda")
        size = drafts.tree_workspace_size(batch, tokens, heads, kv, d, length, dtype)
        assert size > 0
        need = max(need, size)
        sets.append((q, k, v, kd, vd, masks, lengths))
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    graphs = []
    with attention.workspace(workspace):
        for s in sets:
            out = torch.empty_like(s[0])
            call = lambda s=s, out=out: drafts.tree_attention(*s[:6], lengths=s[6], out=out)  # noqa: E731
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
            graphs.append((graph, out, s))
    for turn in range(4):
        say("replay", turn)
        for graph, out, s in graphs:
            s[0].copy_(torch.randn(s[0].shape, generator=g))
            s[6].fill_(int(torch.randint(0, s[1].shape[1] + 1, (1,), generator=g)))
            graph.replay()
            eager = drafts.tree_attention(*s[:6], lengths=s[6])
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
    side = torch.cuda.Stream()
    s = sets[0]
    want = drafts.tree_attention(*s[:6], lengths=s[6])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = drafts.tree_attention(*s[:6], lengths=s[6])
    side.synchronize()
    assert torch.equal(got, want)
    # The workspace that a batch needs holds every smaller batch and tree.
    for batch in (1, 2, 3, 5, 9):
        for tokens in (1, 8, 33, 64):
            size = drafts.tree_workspace_size(batch, tokens, 8, 4, 128, 4096)
            if size:
                assert size >= drafts.tree_workspace_size(1, tokens, 8, 4, 128, 4096)
                assert size >= drafts.tree_workspace_size(batch, 1, 8, 4, 128, 4096)


def reference_walk(tokens, parents, choices, limit):
    path = []
    following = [0] if parents[0] >= -1 else []
    while following and len(path) < limit:
        now = following[0]
        path.append(now)
        following = [j for j in range(now + 1, len(tokens)) if parents[j] == now and tokens[j] == choices[now]]
    return path


def test_tree_masks_edges():
    from asrback_amd import drafts

    say("masks")
    masks = lambda parents: drafts.tree_masks(parents.cuda())[0].tolist()  # noqa: E731
    chain = torch.arange(-1, 63)
    assert masks(chain) == signed([(1 << (i + 1)) - 1 for i in range(64)])
    assert drafts.tree_masks(chain.cuda())[1].tolist() == list(range(64))
    assert masks(torch.tensor([-1])) == [1]
    # Parents that are no earlier token count as the context; children of padding
    # see themselves alone.
    odd = torch.tensor([[0, 0, 5, -2, 3, -9], [1 << 40, -1, 2, 1, 4, -1 << 40]])
    assert masks(odd) == [[1, 3, 4, 0, 16, 0], [1, 2, 4, 10, 16, 0]]
    assert drafts.tree_masks(odd.cuda())[1].tolist() == [[0, 1, 0, 0, 0, 0], [0, 0, 0, 1, 0, 0]]
    assert masks(odd.t().contiguous().t()) == masks(odd)
    assert drafts.tree_masks(odd[:0].cuda())[0].shape == (0, 6)


@pytest.mark.parametrize("batch,width,shared", [(1, 1, False), (3, 2, True), (40, 17, False), (25, 64, False), (7, 64, True)])
def test_accept_follows_the_choices(batch, width, shared):
    from asrback_amd import drafts

    g = torch.Generator().manual_seed(batch * 100 + width)
    say("accept", batch, width, shared)
    parents = [random_parents(width, g, padding=0 if shared else b % 3 if width > 3 else 0) for b in range(1 if shared else batch)]
    if not shared and batch > 2:
        parents[1] = [-2] * width
    rows = parents * batch if shared else parents
    # Few distinct tokens, so that siblings agree and branches run deep.
    tokens = torch.randint(0, 3, (batch, width), generator=g)
    choices = torch.randint(0, 3, (batch, width), generator=g)
    tokens[0] += 1 << 40  # beyond 32 bits
    choices[0] += 1 << 40
    if width > 1:
        tokens[0, 1], choices[0, 0] = 5, 5 + (1 << 40)  # equal in the low 32 bits alone
    limit = torch.randint(-1, width + 2, (batch,), generator=g)
    device_parents = torch.tensor(parents[0] if shared else parents, device="cuda")
    for lim in (None, limit):
        path, emitted, count = drafts.accept_drafts(tokens.cuda(), device_parents, choices.cuda(),
                                                    None if lim is None else lim.cuda())
        for b in range(batch):
            want = reference_walk(tokens[b].tolist(), rows[b], choices[b].tolist(), width if lim is None else int(lim[b]))
            assert count[b] == len(want)
            assert path[b].tolist() == want + [-1] * (width - len(want))
            assert emitted[b].tolist() == [int(choices[b, j]) for j in want] + [-1] * (width - len(want))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [0, 16, 64])
def test_commit_writes_the_accepted_positions_alone(dtype, page):
    from asrback_amd import drafts
    from asrback_amd.attention import PageTable

    g = torch.Generator().manual_seed(page)
    layers, batch, tokens, heads, d, length = 3, 5, 9, 2, 64, 128
    say("commit", dtype, page)
    lengths = [0, 15, 124, 130, -3]
    counts = [9, 4, 9, 2, 3]  # row 2 runs past the cache, rows 3 and 4 lie outside it
    path = torch.stack([torch.randperm(tokens, generator=g) for _ in range(batch)])
    path[1, 2] = tokens  # outside the tree
    path[1, 3] = -1
    kd, vd = (torch.randn(layers, batch, tokens, heads, d, generator=g).to("cuda", dtype) for _ in range(2))
    if page:
        per = length // page
        table = torch.randperm(batch * per, generator=g).view(batch, per).int()
        table[0, 0] = -1 if page == 16 else table[0, 0]
        shape = (layers, batch * per + 1, page, heads, d)
    else:
        table, shape = None, (layers, batch, length, heads, d)
    k, v = (torch.randn(shape, generator=g).to("cuda", dtype) for _ in range(2))
    want_k, want_v = k.clone(), v.clone()
    for b in range(batch):
        for i in range(counts[b]):
            at, node = lengths[b] + i, int(path[b, i])
            if lengths[b] < 0 or not 0 <= at < length or not 0 <= node < tokens:
                continue
            row = b
            if page:
                row, at = int(table[b, at // page]), at % page
                if row < 0:
                    continue
            want_k[:, row, at], want_v[:, row, at] = kd[:, b, node], vd[:, b, node]
    version = k._version
    drafts.commit_drafts(k, v, kd, vd, path.cuda(), torch.tensor(counts, device="cuda"),
                         torch.tensor(lengths, device="cuda"), pages=None if table is None else PageTable(table.cuda()))
    assert torch.equal(k, want_k) and torch.equal(v, want_v) and k._version > version
    # (batch, heads, length, head_dim) caches and other strides, int32 lengths.
    if not page:
        k2, v2 = (torch.randn(layers, batch, heads, length, d, generator=g).to("cuda", dtype).transpose(2, 3) for _ in range(2))
        want = k2.clone()
        drafts.commit_drafts(k2, v2, kd.transpose(2, 3).contiguous().transpose(2, 3), vd, path.cuda(),
                             torch.tensor([1] * batch, device="cuda"), torch.tensor([7] * batch, device="cuda").int())
        for b in range(batch):
            if 0 <= int(path[b, 0]) < tokens:
                want[:, b, 7] = kd[:, b, int(path[b, 0])]
        assert torch.equal(k2, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_contiguous_tensors_at_odd_offsets(dtype):
    """Queries and drafts that torch calls contiguous and vectors cannot read: at odd
    offsets, and single rows, tokens and heads of odd strides."""
    from asrback_amd import drafts

    say("odd offsets", dtype)
    g = torch.Generator().manual_seed(5)
    for batch, tokens, heads, kv_heads in ((2, 3, 4, 2), (1, 1, 4, 1), (1, 5, 1, 1)):
        q, k, v, kd, vd, _, _, _ = make(dtype, batch, tokens, heads, kv_heads, 64, 40, 0, g)
        masks, _ = drafts.tree_masks(torch.tensor([random_parents(tokens, g)] * batch).cuda())
        lengths = torch.tensor([33, 7][:batch]).cuda()
        ref = drafts.tree_attention(q, k, v, kd, vd, masks, lengths=lengths)

        def odd(t):
            moved = torch.empty(t.numel() + 3, dtype=dtype, device="cuda")[3:].view(t.shape).copy_(t)
            assert moved.is_contiguous() and moved.data_ptr() % 16
            return moved

        def wide(t):
            return torch.empty((*t.shape[:-1], 65), dtype=dtype, device="cuda")[..., :64].copy_(t)

        for change in (odd, wide):
            assert torch.equal(drafts.tree_attention(change(q), k, v, change(kd), change(vd), masks, lengths=lengths), ref)
            layers = torch.zeros(2, batch, 40, kv_heads, 64, dtype=dtype, device="cuda")
            caches = [layers.clone() for _ in range(4)]
            path = torch.zeros(batch, tokens, dtype=torch.int64, device="cuda")
            count = torch.ones(batch, dtype=torch.int64, device="cuda")
            both = [t.expand(2, *t.shape).contiguous() for t in (kd, vd)]
            drafts.commit_drafts(*caches[:2], *both, path, count, lengths)
            drafts.commit_drafts(*caches[2:], *(change(t) for t in both), path, count, lengths)
            assert caches[0].any() and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_out_is_written_in_place():
    """A given out counts as changed, may be the queries themselves and another part of
    the buffer that holds the inputs."""
    from asrback_amd import drafts
    from asrback_amd.linear4 import linear4, pack4

    say("out")
    g = torch.Generator().manual_seed(6)
    for dtype, length in ((BF16, 60), (F32, 60), (BF16, 4096)):
        q, k, v, kd, vd, _, _, _ = make(dtype, 1, 5, 8, 2, 64, length, 0, g)
        masks, _ = drafts.tree_masks(torch.tensor([-1, 0, 0, 2, 3]).cuda())
        ref = drafts.tree_attention(q, k, v, kd, vd, masks)
        arena = torch.cat((q, kd, vd, q), 2)
        q, kd, vd, out = arena[:, :, :8], arena[:, :, 8:10], arena[:, :, 10:12], arena[:, :, 12:]
        before = out._version
        assert drafts.tree_attention(q, k, v, kd, vd, masks, out=out) is out and out._version > before
        assert torch.equal(out, ref)
        assert torch.equal(drafts.tree_attention(q, k, v, kd, vd, masks, out=q), ref) and torch.equal(q, ref)
        with torch.inference_mode():
            held = torch.empty_like(out)
            assert torch.equal(drafts.tree_attention(q.copy_(ref), k, v, kd, vd, masks, out=held),
                               drafts.tree_attention(q, k, v, kd, vd, masks))
    weight = pack4(torch.randint(0, 16, (64, 64), generator=g, dtype=torch.uint8).cuda(), torch.ones(64, 1).cuda())
    x, out = torch.randn(3, 64, generator=g).cuda(), torch.empty(3, 64, device="cuda")
    before = out._version
    linear4(x, weight, out=out)
    assert out._version > before and torch.equal(out, linear4(x, weight))
    with torch.inference_mode():
        assert torch.equal(linear4(x, weight, out=torch.empty(3, 64, device="cuda")), out)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_same_bits_call_after_call(dtype, d):
    """Workgroups of one and two row tiles, of four and eight waves, split and whole,
    slab and pages, partly filled tiles."""
    from asrback_amd import drafts

    g = torch.Generator().manual_seed(d)
    for batch, tokens, heads, kv_heads, length, page in (
            (1, 1, 16, 8, 480, 0), (8, 16, 16, 8, 576, 64), (2, 64, 8, 4, 1216, 0), (1, 24, 16, 8, 8000, 0),
            (24, 33, 8, 4, 1536, 16), (70, 3, 8, 4, 48, 0), (5, 7, 6, 6, 448, 64), (16, 40, 8, 4, 1536, 0)):
        say("repeats", dtype, d, batch, tokens, heads, kv_heads, length, page)
        q, k, v, kd, vd, pages, _, _ = make(dtype, batch, tokens, heads, kv_heads, d, length, page, g)
        masks, _ = drafts.tree_masks(torch.tensor([random_parents(tokens, g) for _ in range(batch)]).cuda())
        lengths = torch.randint(0, length + 1, (batch,), generator=g).cuda()
        first = drafts.tree_attention(q, k, v, kd, vd, masks, lengths=lengths, pages=pages)
        differ = torch.zeros((), dtype=torch.int64, device="cuda")
        for _ in range(30):
            differ += (drafts.tree_attention(q, k, v, kd, vd, masks, lengths=lengths, pages=pages) != first).any()
        assert int(differ) == 0
