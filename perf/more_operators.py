"""Operators of a model held and served in 8 bits.

Each case is one pass through one operator with what a server has in hand at
that moment:

* ``linear``: rows, rounded to 8 bits with a scale each, through a matrix of
  8-bit weights with a scale per output;
* ``gated``: both projections of a gated feed-forward block, the activation and
  the product, over such a matrix;
* ``write``: keys and values of new tokens, rounded to 8 bits with a scale per
  token and head, into a cache (slab or pages), and the cache read back;
* ``decode``: attention of one new token a row over such a cache.

``own`` False computes them in plain float32 torch (the rounding in float64,
where values lie next to a border), True on the package's entry points;
``exact`` computes them in float64, apart from both.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # One token through a square projection of Qwen3's decoder (latency).
        {"name": "linear-1", "op": "linear", "dtype": "bf16", "rows": 1, "inputs": 2048, "outputs": 2048, "bias": False},
        # Whisper-tiny's first feed-forward matrix in float32 over an odd number of rows.
        {"name": "linear-f32-7", "op": "linear", "dtype": "f32", "rows": 7, "inputs": 384, "outputs": 1536, "bias": True},
        # Four packed prompts of odd length through the fused projection of Qwen3's heads.
        {"name": "linear-prompt", "op": "linear", "dtype": "bf16", "rows": 1537, "inputs": 2048, "outputs": 4096,
         "bias": False},
        # Eight windows of 1500 frames through the first feed-forward matrix of Whisper turbo's encoder.
        {"name": "linear-frames", "op": "linear", "dtype": "bf16", "rows": 12000, "inputs": 1280, "outputs": 5120,
         "bias": True},
        # Sixteen rows' step through Qwen3's gate and up projections.
        {"name": "gated-16", "op": "gated", "dtype": "bf16", "rows": 16, "inputs": 2048, "hidden": 6144},
        # A full admission's prompts through them.
        {"name": "gated-prompt", "op": "gated", "dtype": "bf16", "rows": 4099, "inputs": 2048, "hidden": 6144},
        # One token of the smallest heads into one row of a short cache (latency).
        {"name": "write-1", "op": "write", "dtype": "f32", "rows": 1, "new": 1, "kv_heads": 6, "head_dim": 64,
         "length": 128, "low": 17, "high": 17, "page": 0},
        # Eight windows' prompts of Qwen3's heads into pages.
        {"name": "write-prompt-8", "op": "write", "dtype": "bf16", "rows": 8, "new": 430, "kv_heads": 8, "head_dim": 128,
         "length": 1024, "low": 401, "high": 430, "page": 64},
        # One window's step (latency).
        {"name": "decode-1", "op": "decode", "dtype": "bf16", "rows": 1, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "length": 1024, "low": 480, "high": 480, "page": 0, "window": 0},
        # Whisper-tiny's heads in float32 over the frames of windows of all lengths.
        {"name": "decode-f32-5", "op": "decode", "dtype": "f32", "rows": 5, "heads": 6, "kv_heads": 6, "head_dim": 64,
         "length": 1500, "low": 0, "high": 1500, "page": 0, "window": 0},
        # Qwen3-ASR's full batch over pages.
        {"name": "decode-64", "op": "decode", "dtype": "bf16", "rows": 64, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "length": 1024, "low": 400, "high": 560, "page": 64, "window": 0},
        # Two long recordings over 65536 positions.
        {"name": "decode-long", "op": "decode", "dtype": "bf16", "rows": 2, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "length": 65536, "low": 40001, "high": 65511, "page": 0, "window": 0},
    ]


def _log(rng: random.Random, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("linear", "linear", "gated", "write", "decode", "decode"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op in ("linear", "gated"):
        rows, inputs = _log(rng, 1, 12000), _log(rng, 64, 8192)
        if rng.random() < 0.7:  # most matrices are whole blocks
            inputs = (inputs + 63) // 64 * 64
        most = 7 * 10**10 // (rows * inputs)
        outputs = max(16, min(_log(rng, 16, 40000), most, 10**8 // inputs, 6 * 10**7 // rows))
        if op == "linear":
            return {"op": op, "dtype": dtype, "rows": rows, "inputs": inputs, "outputs": outputs,
                    "bias": rng.random() < 0.5}
        return {"op": op, "dtype": dtype, "rows": rows, "inputs": inputs, "hidden": max(8, outputs // 2)}
    kv_heads, head_dim = rng.choice(((8, 128), (4, 128), (2, 128), (6, 64), (12, 64), (20, 64), (4, 256), (1, 256)))
    page = rng.choice((0, 0, 16, 64, 128))
    rows = _log(rng, 1, 64)
    case = {"op": op, "dtype": dtype, "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim}
    most = (10**8 if op == "decode" else 4 * 10**7) // (2 * kv_heads * head_dim)
    length = max(128, min(_log(rng, 128, 65536), most // rows) // 128 * 128)
    case["rows"] = rows = max(1, min(rows, most // length))
    high = rng.randint(1, length)
    case |= {"length": length, "low": rng.randint(0, high), "high": high, "page": page}
    if op == "write":
        case["new"] = max(1, min(high, _log(rng, 1, 2 * high)))
    else:
        case["heads"] = rng.choice((1, 2, 3, 4, 8)) * kv_heads
        case["window"] = rng.choice((0, 0, 0, _log(rng, 1, length)))
    return case


def _lengths(case: dict) -> list[int]:
    """Keys that each row holds in the cache (after the call)."""
    rows, low, high = case["rows"], case["low"], case["high"]
    return [low + (high - low) * b // max(1, rows - 1) for b in range(rows)]


def _slots(case: dict) -> list[tuple[int, int]]:
    """Row and position of each token written: the last ``new`` of every row."""
    return [(b, at) for b, n in enumerate(_lengths(case)) for at in range(max(0, n - case["new"]), n)]


def _generator(seed: int) -> torch.Generator:
    return torch.Generator("cuda").manual_seed(seed)


def _held(shape: tuple[int, ...], scales: tuple[int, ...], g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """8-bit values as rounding leaves them of a row of normal ones (the largest at
    127) and their scales."""
    values = (torch.randn(shape, generator=g, device="cuda") * 45).round_().clamp_(-127, 127).to(torch.int8)
    values[..., 0] = 127
    return values, (torch.rand(scales, generator=g, device="cuda") + 0.5) * 0.02


def _inputs(case: dict, seed: int) -> dict:
    """A case's tensors, from its seed alone."""
    rng, g = random.Random(seed), _generator(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] in ("linear", "gated"):
        rows, k = case["rows"], case["inputs"]
        n = case["outputs"] if case["op"] == "linear" else 2 * case["hidden"]
        x = normal(rows, k)
        x[:, :: max(1, k // 5)] *= 6  # a few channels stand out
        # Weights of deviation k^-1/2, the largest of an output at about four of them.
        values = (torch.randn((n, k), generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)
        scales = ((torch.rand(n, generator=g, device="cuda") + 0.5) * k**-0.5 / 32).to(dtype)
        return {"x": x, "values": values, "scales": scales, "bias": normal(n) if case.get("bias") else None}
    rows, length, kv_heads, head_dim, page = (case[f] for f in ("rows", "length", "kv_heads", "head_dim", "page"))
    lengths = _lengths(case)
    state = {"lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "table": None}
    lead, span = rows, length
    if page:
        needed = [-(-n // page) for n in lengths]
        lead, span = sum(needed) + 3, page
        ids = rng.sample(range(lead), sum(needed))
        table = torch.full((rows, length // page), -1, dtype=torch.int32)
        for b, count in enumerate(needed):
            table[b, :count] = torch.tensor([ids.pop() for _ in range(count)], dtype=torch.int32)
        state["table"] = table.cuda()
    for name in ("key", "value"):
        state[name + "s"], state[name + "_scales"] = _held((lead, span, kv_heads, head_dim), (lead, kv_heads, span), g)
    if case["op"] == "decode":
        state["q"] = normal(rows, case["heads"], head_dim)
        return state
    slots = torch.tensor(_slots(case), device="cuda").view(-1, 2)
    state |= {"rows": slots[:, 0].contiguous(), "positions": slots[:, 1].contiguous(),
              "k": normal(len(slots), kv_heads, head_dim), "v": normal(len(slots), kv_heads, head_dim)}
    return state


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed) | {"case": case}
    if not own:
        return state
    if case["op"] in ("linear", "gated"):
        from asrback_amd.linear8 import pack8

        # The matrix as a model holds it, laid out once.
        state["weight"] = pack8(state.pop("values"), state.pop("scales"))
        return state
    from asrback_amd.attention import PageTable
    from asrback_amd.cache8 import Cache8, decode8_workspace_size

    state["pages"] = None if state["table"] is None else PageTable(state["table"])
    state["cache"] = Cache8(state["keys"], state["values"], state["key_scales"], state["value_scales"])
    if case["op"] == "decode":
        # A decoder's workspace, kept from step to step.
        need = decode8_workspace_size(case["rows"], case["heads"], case["kv_heads"], case["head_dim"], case["length"],
                                      DTYPES[case["dtype"]])
        state["workspace"] = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    return state


def run(state: dict):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "gated": _own_gated, "write": _own_write, "decode": _own_decode}[op](state)
    return {"linear": _plain_linear, "gated": _plain_gated, "write": _plain_write, "decode": _plain_decode}[op](state)


def _own_linear(s: dict) -> torch.Tensor:
    from asrback_amd.linear8 import linear8

    return linear8(s["x"], s["weight"], s["bias"])


def _own_gated(s: dict) -> torch.Tensor:
    from asrback_amd.linear8 import gated8

    return gated8(s["x"], s["weight"])


def _own_write(s: dict):
    from asrback_amd.cache8 import read8, write8

    write8(s["cache"], s["k"], s["v"], s["rows"], s["positions"], pages=s["pages"])
    return read8(s["cache"], lengths=s["lengths"], pages=s["pages"], dtype=s["k"].dtype)


def _own_decode(s: dict) -> torch.Tensor:
    from asrback_amd.cache8 import decode8

    return decode8(s["q"], s["cache"], lengths=s["lengths"], pages=s["pages"], window=s["case"]["window"] or None,
                   workspace=s["workspace"])


def _rounded(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows rounded to whole numbers -127 .. 127 (ties to even) and their float32
    scales, the largest magnitude's 127th part."""
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float()
    step = scale.double()
    values = torch.where(step > 0, x.double() / torch.where(step > 0, step, 1.0), 0.0).round().clamp(-127, 127)
    return values.float(), scale


def _product(s: dict) -> torch.Tensor:
    values, scale = _rounded(s["x"])
    out = torch.matmul(values, s["values"].float().T) * scale * s["scales"].float()
    return out if s["bias"] is None else out + s["bias"].float()


def _plain_linear(s: dict) -> torch.Tensor:
    return _product(s).to(s["x"].dtype)


def _plain_gated(s: dict) -> torch.Tensor:
    gate, up = _product(s).chunk(2, -1)
    return (gate / (1 + torch.exp(-gate)) * up).to(s["x"].dtype)


def _rows_of(pool: torch.Tensor, scales: torch.Tensor, table: torch.Tensor | None) -> torch.Tensor:
    """Every row's positions as the float32 values they stand for, ``(rows, length,
    heads, head_dim)``."""
    scales = scales.transpose(1, 2)
    if table is not None:
        pages = table.long().clamp(min=0)
        pool, scales = pool[pages].flatten(1, 2), scales[pages].flatten(1, 2)
    return pool.float() * scales[..., None]


def _plain_write(s: dict):
    row, position = s["rows"], s["positions"]
    if s["table"] is not None:
        page = s["case"]["page"]
        row, position = s["table"][row, position // page].long(), position % page
    for new, pool, scales in (("k", "keys", "key_scales"), ("v", "values", "value_scales")):
        values, scale = _rounded(s[new])
        s[pool][row, position] = values.to(torch.int8)
        s[scales][row, :, position] = scale[..., 0]
    held = torch.arange(s["case"]["length"], device="cuda") < s["lengths"][:, None]
    return tuple(torch.where(held[..., None, None], _rows_of(s[pool], s[scales], s["table"]), 0.0).to(s["k"].dtype)
                 for pool, scales in (("keys", "key_scales"), ("values", "value_scales")))


def _plain_decode(s: dict) -> torch.Tensor:
    q, lengths, window = s["q"], s["lengths"], s["case"]["window"]
    k = _rows_of(s["keys"], s["key_scales"], s["table"])
    v = _rows_of(s["values"], s["value_scales"], s["table"])
    rows, length, kv_heads, head_dim = k.shape
    at = torch.arange(length, device="cuda")
    seen = at < lengths[:, None]
    if window:
        seen &= at >= lengths[:, None] - window
    scores = torch.matmul(q.float().view(rows, kv_heads, -1, head_dim), k.permute(0, 2, 3, 1).contiguous())
    scores = (scores * head_dim**-0.5).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v.transpose(1, 2).contiguous()) / torch.where(total == 0, 1.0, total)
    return out.reshape(q.shape).to(q.dtype)


def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("linear", "gated"):
        rows, k = case["rows"], case["inputs"]
        n, out = (case["outputs"],) * 2 if case["op"] == "linear" else (2 * case["hidden"], case["hidden"])
        return {"bytes": n * k + size * (n + rows * (k + out) + (n if case.get("bias") else 0)), "flops": 2 * rows * n * k}
    values = 2 * case["kv_heads"] * case["head_dim"]  # of a position
    position = values + 8 * case["kv_heads"]
    lengths = _lengths(case)
    if case["op"] == "write":
        new = len(_slots(case))
        return {"bytes": new * (values * size + position + 16) + sum(lengths) * position
                + case["rows"] * case["length"] * values * size, "flops": 0}
    keys = sum(min(n, case["window"] or n) for n in lengths)
    row = case["heads"] * case["head_dim"]
    return {"bytes": keys * position + case["rows"] * (2 * row * size + 4), "flops": 4 * keys * row}


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    if case["op"] in ("linear", "gated"):
        x = s["x"].double()
        step = torch.abs(x).max(1, keepdim=True).values.div(127.0).float().double()
        q = torch.div(x, step.masked_fill(step == 0, 1.0)).round().clamp(-127, 127)
        parts = []
        for at in range(0, len(s["scales"]), 8192):
            w = s["values"][at : at + 8192].double() * s["scales"][at : at + 8192].double()[:, None]
            parts.append((q @ w.t().contiguous()) * step)
        out = torch.cat(parts, 1)
        if case["op"] == "gated":
            return torch.sigmoid(out[:, : case["hidden"]]) * out[:, : case["hidden"]] * out[:, case["hidden"] :]
        return out if s["bias"] is None else out + s["bias"].double()
    lengths, page = _lengths(case), case["page"]

    def where(b: int, first: int, last: int):
        at = torch.arange(first, last, device="cuda")
        if page:
            return s["table"][b].long()[at // page], at % page
        return torch.full_like(at, b), at

    def values_of(name: str, b: int, first: int, last: int) -> torch.Tensor:
        row, at = where(b, first, last)
        return s[name + "s"][row, at].double() * s[name + "_scales"].double()[row, :, at][..., None]

    if case["op"] == "write":
        out = []
        for name, new in (("key", s["k"].double()), ("value", s["v"].double())):
            whole = torch.zeros((case["rows"], case["length"], *new.shape[1:]), dtype=torch.float64, device="cuda")
            done = 0
            for b, n in enumerate(lengths):
                old = max(0, n - case["new"])
                whole[b, :old] = values_of(name, b, 0, old)
                x = new[done : done + n - old]
                done += n - old
                step = (x.abs().amax(-1, keepdim=True) / 127).float().double()
                whole[b, old:n] = torch.clamp(torch.round(x / torch.where(step == 0, 1.0, step)), -127, 127) * step
            out.append(whole)
        return tuple(out)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        first = max(0, n - case["window"]) if case["window"] else 0
        if first == n:
            continue
        k, v = values_of("key", b, first, n), values_of("value", b, first, n)
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            scores = s["q"][b, heads].double() @ k[:, h].t().contiguous() / math.sqrt(case["head_dim"])
            out[b, heads] = torch.softmax(scores, -1) @ v[:, h].contiguous()
    return out
