"""Operators of a decoder that verifies drafted tokens with 4-bit weights.

Each case is one pass through one operator with what a server has in hand at
that moment:

* ``tree``: attention of a tree of drafted tokens over a key/value cache (slab
  or pages), the tree as ancestor bit masks;
* ``commit``: the greedy choice's walk down the tree, then the accepted
  tokens' keys and values of every layer from the draft buffers into the cache;
* ``linear``: rows through a matrix of 4-bit weights with group scales.

``own`` False computes them in plain float32 torch, True on the package's
entry points; ``exact`` computes them in float64, apart from both.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # One window, one drafted token: a plain step through the same path (latency).
        {"name": "tree-1", "op": "tree", "dtype": "bf16", "rows": 1, "tokens": 1, "depth": 1, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "length": 1024, "low": 480, "high": 480, "page": 0, "ragged": False},
        # Qwen3-ASR's heads, a light load's windows verifying 16 tokens each, paged cache.
        {"name": "tree-paged-8", "op": "tree", "dtype": "bf16", "rows": 8, "tokens": 16, "depth": 6, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "length": 1024, "low": 400, "high": 560, "page": 64, "ragged": True},
        # Whisper-tiny's heads in float32, trees of seven tokens over its 448 positions.
        {"name": "tree-f32-4", "op": "tree", "dtype": "f32", "rows": 4, "tokens": 7, "depth": 4, "heads": 6, "kv_heads": 6,
         "head_dim": 64, "length": 448, "low": 17, "high": 440, "page": 0, "ragged": True},
        # Wide heads (8 over 4 of 256), the widest tree, full rows of a 1280-position cache.
        {"name": "tree-wide-2", "op": "tree", "dtype": "bf16", "rows": 2, "tokens": 64, "depth": 9, "heads": 8, "kv_heads": 4,
         "head_dim": 256, "length": 1280, "low": 1201, "high": 1216, "page": 0, "ragged": True},
        # A long recording: one row over 65536 positions.
        {"name": "tree-long-1", "op": "tree", "dtype": "bf16", "rows": 1, "tokens": 24, "depth": 8, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "length": 65536, "low": 65511, "high": 65511, "page": 0, "ragged": False},
        # After one window's pass: a chain of eight, all 28 layers of the slab.
        {"name": "commit-1", "op": "commit", "dtype": "bf16", "rows": 1, "tokens": 8, "depth": 8, "kv_heads": 8,
         "head_dim": 128, "layers": 28, "length": 1024, "low": 480, "high": 480, "page": 0, "ragged": False},
        # Sixteen windows' trees into a paged cache.
        {"name": "commit-paged-16", "op": "commit", "dtype": "bf16", "rows": 16, "tokens": 16, "depth": 6, "kv_heads": 8,
         "head_dim": 128, "layers": 7, "length": 1024, "low": 400, "high": 560, "page": 64, "ragged": True},
        # One token through a square projection (latency).
        {"name": "linear-1", "op": "linear", "dtype": "bf16", "rows": 1, "inputs": 2048, "outputs": 2048, "group": 128,
         "zeros": False, "bias": False},
        # A tree of 16 tokens through the gate and up projections.
        {"name": "linear-16", "op": "linear", "dtype": "bf16", "rows": 16, "inputs": 2048, "outputs": 12288, "group": 128,
         "zeros": False, "bias": False},
        # Four trees of 16 through a down projection with zero points and short groups.
        {"name": "linear-64", "op": "linear", "dtype": "bf16", "rows": 64, "inputs": 6144, "outputs": 2048, "group": 64,
         "zeros": True, "bias": False},
        # Four rows through the vocabulary's matrix, the largest there is.
        {"name": "linear-head-4", "op": "linear", "dtype": "bf16", "rows": 4, "inputs": 2048, "outputs": 151936, "group": 128,
         "zeros": False, "bias": False},
        # Whisper-tiny's first feed-forward matrix in float32, odd rows, bias.
        {"name": "linear-f32-5", "op": "linear", "dtype": "f32", "rows": 5, "inputs": 384, "outputs": 1536, "group": 32,
         "zeros": True, "bias": True},
    ]


def _log(rng: random.Random, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("tree", "tree", "commit", "linear", "linear"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "linear":
        group = rng.choice((32, 64, 128))
        inputs = max(1, _log(rng, 128, 8192) // group) * group
        rows = _log(rng, 1, 64)
        outputs = min(_log(rng, 16, 40000), 10**8 // inputs // max(1, rows // 16))
        return {"op": op, "dtype": dtype, "rows": rows, "inputs": inputs, "outputs": outputs, "group": group,
                "zeros": rng.random() < 0.5, "bias": rng.random() < 0.5}
    rows, tokens = _log(rng, 1, 64), _log(rng, 1, 64)
    kv_heads, head_dim = rng.choice(((8, 128), (4, 128), (2, 128), (6, 64), (12, 64), (20, 64), (4, 256), (1, 256)))
    page = rng.choice((0, 0, 16, 64, 128))
    per = 2 * kv_heads * head_dim * (2 if dtype == "bf16" else 4)  # bytes of a position
    case = {"op": op, "dtype": dtype, "rows": rows, "tokens": tokens, "depth": rng.randint(1, min(tokens, 12)),
            "kv_heads": kv_heads, "head_dim": head_dim}
    if op == "tree":
        group = rng.choice((1, 2, 3, 4, 8))
        case["heads"] = group * kv_heads
        most = 10**8 // per // max(1, tokens * group // 64)
    else:
        case["layers"] = rng.randint(1, 28)
        most = 10**8 // per // case["layers"]
    length = max(128, min(_log(rng, 128, 65536), most // rows) // 128 * 128)
    if length * rows > most:
        case["rows"] = rows = max(1, most // length)
    high = rng.randint(0, length - 64)
    case |= {"length": length, "low": rng.randint(0, high), "high": high, "page": page, "ragged": rng.random() < 0.7}
    return case


def _lengths(case: dict) -> list[int]:
    """Keys that each row holds in the cache."""
    rows, low, high = case["rows"], case["low"], case["high"]
    return [low + (high - low) * b // max(1, rows - 1) for b in range(rows)]


def _accepted(case: dict) -> list[int]:
    """Tokens that each row accepts (none of them: a finished row)."""
    depth, rows = case["depth"], case["rows"]
    return [0 if case["ragged"] and b % 5 == 4 else 1 + (5 * b + depth // 2) % depth for b in range(rows)]


def _trees(case: dict, rng: random.Random) -> tuple[list[list[int]], list[list[int]]]:
    """Each row's parents (-1: the context, -2: padding) and its longest branch."""
    parents, spines = [], []
    for b in range(case["rows"]):
        tokens, depth = case["tokens"], case["depth"]
        real = rng.randint(depth, tokens) if case["ragged"] and b % 2 else tokens
        spine = [0] + sorted(rng.sample(range(1, real), depth - 1))
        row = [-1 if i == 0 else rng.randrange(i) for i in range(real)]
        for i, j in zip(spine, spine[1:]):
            row[j] = i
        parents.append(row + [-2] * (tokens - real))
        spines.append(spine)
    return parents, spines


def _masks(parents: list[list[int]]) -> list[list[int]]:
    """Bit i of a token's mask: it sees drafted token i (as signed 64-bit values)."""
    out = []
    for row in parents:
        masks: list[int] = []
        for i, parent in enumerate(row):
            masks.append(0 if parent < -1 else 1 << i | (masks[parent] if parent >= 0 else 0))
        out.append([m - (1 << 64) if m >> 63 else m for m in masks])
    return out


def _table(case: dict, positions: list[int], rng: random.Random) -> tuple[torch.Tensor, int]:
    """Pages for these many positions a row, in any order, and the pool's size."""
    page = case["page"]
    needed = [-(-p // page) for p in positions]
    pool = sum(needed) + 3
    ids = rng.sample(range(pool), sum(needed))
    table = torch.full((case["rows"], case["length"] // page), -1, dtype=torch.int32)
    for b, count in enumerate(needed):
        table[b, :count] = torch.tensor([ids.pop() for _ in range(count)], dtype=torch.int32)
    return table, pool


def _inputs(case: dict, seed: int) -> dict:
    """A case's tensors, from its seed alone."""
    rng = random.Random(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] == "linear":
        rows, n, k, group = case["rows"], case["outputs"], case["inputs"], case["group"]
        return {
            "x": normal(rows, k),
            # Weights of deviation k^-1/2 in steps of about a seventh of their largest.
            "values": (torch.randn((n, k), generator=g, device="cuda") * 2.5 + 8).round_().clamp_(0, 15).to(torch.uint8),
            "scales": ((torch.rand((n, k // group), generator=g, device="cuda") + 0.5) * 0.4 * k**-0.5).to(dtype),
            "zeros": (torch.randint(5, 12, (n, k // group), generator=g, device="cuda", dtype=torch.uint8)
                      if case["zeros"] else None),
            "bias": normal(n) if case["bias"] else None,
        }
    rows, tokens, length, kv_heads, head_dim = (case[f] for f in ("rows", "tokens", "length", "kv_heads", "head_dim"))
    parents, spines = _trees(case, rng)
    lengths = _lengths(case)
    state = {"lengths": torch.tensor(lengths, device="cuda"), "table": None}
    if case["op"] == "tree":
        heads = case["heads"]
        lead, layers = [], 1
        state["masks"] = torch.tensor(_masks(parents), device="cuda")
        state["q"] = normal(rows, tokens, heads, head_dim)
        reach = lengths
    else:
        lead, layers = [case["layers"]], case["layers"]
        accepted = _accepted(case)
        reach = [n + a for n, a in zip(lengths, accepted)]
        # Children of one token differ; the choice follows the spine while
        # tokens are accepted and leaves the tree after them.
        drafted = [rng.sample(range(151936), tokens) for _ in range(rows)]
        choices = [[rng.randrange(151936, 160000) for _ in range(tokens)] for _ in range(rows)]
        for b, (spine, count) in enumerate(zip(spines, accepted)):
            for i, j in list(zip(spine, spine[1:]))[: max(0, count - 1)]:
                choices[b][i] = drafted[b][j]
        state |= {name: torch.tensor(x, device="cuda") for name, x in (
            ("tokens", drafted), ("parents", parents), ("choices", choices),
            ("limit", [tokens if a else 0 for a in accepted]))}
    if case["page"]:
        table, pool = _table(case, reach, rng)
        state["table"] = table.cuda()
        shape = (*lead, pool, case["page"], kv_heads, head_dim)
    else:
        shape = (*lead, rows, length, kv_heads, head_dim)
    state |= {"keys": normal(*shape), "values": normal(*shape),
              "draft_keys": normal(*lead, rows, tokens, kv_heads, head_dim),
              "draft_values": normal(*lead, rows, tokens, kv_heads, head_dim)}
    return state


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed) | {"case": case}
    if case["op"] == "linear":
        if own:
            from asrback_amd.linear4 import pack4

            # The matrix as a model holds it, laid out once.
            state["weight"] = pack4(state.pop("values"), state.pop("scales"), state.pop("zeros"))
        return state
    if own:
        from asrback_amd.attention import PageTable
        from asrback_amd.drafts import tree_workspace_size

        state["pages"] = None if state["table"] is None else PageTable(state["table"])
        if case["op"] == "tree":
            # A decoder's workspace, kept from step to step.
            need = tree_workspace_size(case["rows"], case["tokens"], case["heads"], case["kv_heads"], case["head_dim"],
                                       case["length"], DTYPES[case["dtype"]])
            state["workspace"] = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    return state


def run(state: dict):
    op = state["case"]["op"]
    if own:
        return {"tree": _own_tree, "commit": _own_commit, "linear": _own_linear}[op](state)
    return {"tree": _plain_tree, "commit": _plain_commit, "linear": _plain_linear}[op](state)


def _own_tree(s: dict) -> torch.Tensor:
    from asrback_amd.drafts import tree_attention

    return tree_attention(s["q"], s["keys"], s["values"], s["draft_keys"], s["draft_values"], s["masks"],
                          lengths=s["lengths"], pages=s["pages"], workspace=s["workspace"])


def _own_commit(s: dict):
    from asrback_amd.drafts import accept_drafts, commit_drafts

    path, emitted, count = accept_drafts(s["tokens"], s["parents"], s["choices"], s["limit"])
    commit_drafts(s["keys"], s["values"], s["draft_keys"], s["draft_values"], path, count, s["lengths"], pages=s["pages"])
    return path, emitted, count, s["keys"], s["values"]


def _own_linear(s: dict) -> torch.Tensor:
    from asrback_amd.linear4 import linear4

    return linear4(s["x"], s["weight"], s["bias"])


def _rows_of(pool: torch.Tensor, table: torch.Tensor | None, most: int) -> torch.Tensor:
    """Each row's first ``most`` positions of the cache, ``(rows, most, heads, head_dim)``."""
    if table is None:
        return pool[:, :most]
    page = pool.shape[1]
    pages = table[:, : -(-most // page)].long().clamp(min=0)
    return pool[pages].flatten(1, 2)[:, :most]


def _plain_tree(s: dict) -> torch.Tensor:
    q, masks, lengths = s["q"], s["masks"], s["lengths"]
    rows, tokens, heads, head_dim = q.shape
    most = max(_lengths(s["case"]))
    k = torch.cat((_rows_of(s["keys"], s["table"], most), s["draft_keys"]), 1).float()
    v = torch.cat((_rows_of(s["values"], s["table"], most), s["draft_values"]), 1).float()
    kv_heads = k.shape[2]
    real = masks != 0
    cached = torch.arange(most, device=q.device) < lengths[:, None]  # (rows, most)
    seen = torch.cat((cached[:, None, :] & real[:, :, None],
                      (masks[:, :, None] >> torch.arange(tokens, device=q.device)) & 1 == 1), -1)
    # (rows, kv_heads, group * tokens, keys)
    qh = q.float().view(rows, tokens, kv_heads, -1, head_dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    kh, vh = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    scores = torch.matmul(qh, kh) * head_dim**-0.5
    seen = seen[:, None, None].expand(-1, 1, heads // kv_heads, -1, -1).flatten(2, 3)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, vh) / torch.where(total == 0, 1.0, total)
    out = out.view(rows, kv_heads, -1, tokens, head_dim).permute(0, 3, 1, 2, 4)
    return out.reshape(q.shape).to(q.dtype)


def _plain_commit(s: dict):
    tokens, parents, choices, limit = s["tokens"], s["parents"], s["choices"], s["limit"]
    rows, width = tokens.shape
    node = torch.arange(width, device=tokens.device)
    path = torch.full_like(tokens, -1)
    now = torch.where((limit > 0) & (parents[:, 0] >= -1), 0, -1)
    for i in range(width):
        path[:, i] = now
        choice = choices.gather(1, now.clamp(min=0)[:, None])
        child = (parents == now[:, None]) & (tokens == choice) & (node > now[:, None])
        child &= (now >= 0)[:, None] & (i + 1 < limit)[:, None]
        now = torch.where(child.any(1), child.int().argmax(1), -1)
    held = path >= 0
    emitted = torch.where(held, choices.gather(1, path.clamp(min=0)), -1)
    count = held.sum(1)
    row, step = held.nonzero(as_tuple=True)
    source = path[row, step]
    position = s["lengths"][row] + step
    if s["table"] is not None:
        page = s["keys"].shape[2]
        row_to, position = s["table"][row, position // page].long(), position % page
    else:
        row_to = row
    s["keys"][:, row_to, position] = s["draft_keys"][:, row, source]
    s["values"][:, row_to, position] = s["draft_values"][:, row, source]
    return path, emitted, count, s["keys"], s["values"]


def _plain_linear(s: dict) -> torch.Tensor:
    x, values, scales, zeros, bias = s["x"], s["values"], s["scales"], s["zeros"], s["bias"]
    groups = values.float().view(values.shape[0], scales.shape[1], -1)
    groups -= 8.0 if zeros is None else zeros.float()[..., None]
    groups *= scales.float()[..., None]
    out = torch.matmul(x.float(), groups.flatten(1).T)
    if bias is not None:
        out += bias.float()
    return out.to(x.dtype)


def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["outputs"], case["inputs"]
        groups = n * (k // case["group"])
        # Zero points are four bits as well.
        return {"bytes": n * k // 2 + groups * size + (groups // 2 if case["zeros"] else 0) + size * rows * (k + n)
                + (size * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    position = 2 * case["kv_heads"] * case["head_dim"] * size
    if case["op"] == "tree":
        tokens, rows, heads = case["tokens"], case["rows"], case["heads"]
        keys = sum(_lengths(case))
        # The drafted keys' products, at most 64 keys a token, are left out.
        return {"bytes": (keys + rows * tokens) * position + 2 * rows * tokens * heads * case["head_dim"] * size
                + 8 * rows * (tokens + 1), "flops": 4 * keys * tokens * heads * case["head_dim"]}
    moved = 2 * sum(_accepted(case)) * case["layers"] * position
    return {"bytes": moved + 8 * case["rows"] * (5 * case["tokens"] + 3), "flops": 0}


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        scales = s["scales"].double().repeat_interleave(case["group"], 1)
        zeros = 8.0 if s["zeros"] is None else s["zeros"].double().repeat_interleave(case["group"], 1)
        parts = []
        for at in range(0, case["outputs"], 16384):
            stop = at + 16384
            w = (s["values"][at:stop].double() - (zeros if isinstance(zeros, float) else zeros[at:stop])) * scales[at:stop]
            parts.append(x @ w.T)
        out = torch.cat(parts, 1)
        return out if s["bias"] is None else out + s["bias"].double()
    lengths = _lengths(case)
    if case["op"] == "commit":
        parents, drafted, choices = (s[f].tolist() for f in ("parents", "tokens", "choices"))
        paths, emitted, counts = [], [], []
        for b in range(case["rows"]):
            path: list[int] = []
            following = [0] if parents[b][0] >= -1 else []
            while following and len(path) < s["limit"][b]:
                path.append(following[0])
                following = [j for j in range(path[-1] + 1, case["tokens"])
                             if parents[b][j] == path[-1] and drafted[b][j] == choices[b][path[-1]]]
            for i, node in enumerate(path):
                row, at = b, lengths[b] + i
                if case["page"]:
                    row, at = int(s["table"][b, at // case["page"]]), at % case["page"]
                s["keys"][:, row, at].copy_(s["draft_keys"][:, b, node])
                s["values"][:, row, at].copy_(s["draft_values"][:, b, node])
            pad = [-1] * (case["tokens"] - len(path))
            paths.append(path + pad)
            emitted.append([choices[b][node] for node in path] + pad)
            counts.append(len(path))
        as_long = (torch.tensor(x, device="cuda") for x in (paths, emitted, counts))
        return *as_long, s["keys"].double(), s["values"].double()
    group = case["heads"] // case["kv_heads"]
    masks = s["masks"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        if case["page"]:
            at = torch.arange(n, device="cuda")
            where = (s["table"][b].long()[at // case["page"]], at % case["page"])
        else:
            where = (b, slice(0, n))
        kb = torch.cat((s["keys"][where], s["draft_keys"][b])).double()
        vb = torch.cat((s["values"][where], s["draft_values"][b])).double()
        hidden = torch.ones((case["tokens"], n + case["tokens"]), dtype=torch.bool)
        for t, mask in enumerate(masks[b]):
            if mask:
                hidden[t, :n] = False
                for i in range(case["tokens"]):
                    hidden[t, n + i] = not mask >> i & 1
        hidden = hidden.cuda()
        empty = hidden.all(1)
        for h in range(case["heads"]):
            scores = s["q"][b, :, h].double() @ kb[:, h // group].T / math.sqrt(case["head_dim"])
            scores[hidden] = -math.inf
            scores[empty] = 0.0
            weights = torch.softmax(scores, -1)
            weights[empty] = 0.0
            out[b, :, h] = weights @ vb[:, h // group]
    return out
