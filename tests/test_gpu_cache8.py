"""GPU: the 8-bit cache -- writes, reading back, attention -- against plain float64
on the CPU.

Writes round exactly, so their whole numbers and scales are the reference's.  Reading
back rounds a product to float32 and that to the type.  Attention's bound, per
element, with A = the weights times |v| and S the largest sum of |q| |k| scale over a
row's keys: the products are exact, a score's d additions are each off by 2^-24 of
at most S, its scales, the maximum's subtraction and the exponential by 8 more;
weights and their sum both carry them, and the weights' sums over n keys, twice:

    2^-24 A (2 (d + 8) S + 2 n + 64)   float32 work
    2^-16 A                            bf16: a weight times its scale, as two bf16
    2^-23 A                            float32: as three
    2^-8 |ref|, 2^-24 |ref|            the result

times 1.01 for second-order terms.  In bf16 the products are of the stored numbers plus
128, between 0 and 255, and the same sums of 128 are taken off again: both pass through
the float32 accumulator, so that an addition is off by 2^-24 of at most 255 in a stored
number's place, twice.  With B = the weights times the values' scales and Q the largest
sum of |q| times a key's scale and the scale, that adds

    2^-24 (n + 64) 510 B               to the output (n additions on a weight's way)
    2^-24 (d + 8) 510 Q                to a score: 2 A times it to the output
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def say(*args):
    print(*args, flush=True)


def rounded(x):
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float().double()
    q = torch.where(scale > 0, x.double() / scale.where(scale > 0, torch.ones_like(scale)), 0.0)
    return q.round().clamp(-127, 127).to(torch.int8), scale[..., 0].float()


def random_cache(batch, length, heads, head_dim, g, head_major=False):
    """A Cache8 on the GPU and its tensors on the CPU; with ``head_major`` of the other
    layout that strides allow."""
    from asrback_amd.cache8 import Cache8

    shape = (batch, heads, length, head_dim) if head_major else (batch, length, heads, head_dim)
    held = []
    for _ in "kv":
        t = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
        held.append(t.transpose(1, 2) if head_major else t)
    scales = [(torch.rand(batch, heads, length, generator=g) + 0.5) * 0.02 for _ in "kv"]
    device = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) if head_major else t.cuda() for t in held]
    return Cache8(*device, *(s.cuda() for s in scales)), (*held, *scales)


def paged(tensors, page, g, extra=3):
    """The same positions in pages of a pool in random order; the unowned slots hold the
    largest values and NaN scales."""
    from asrback_amd.attention import PageTable
    from asrback_amd.cache8 import Cache8

    k, v, ks, vs = tensors
    batch, length, heads, head_dim = k.shape
    per = -(-length // page)
    pool = batch * per + extra
    ids = torch.randperm(pool, generator=g)[: batch * per].view(batch, per)
    values = [torch.full((pool, page, heads, head_dim), 127, dtype=torch.int8) for _ in "kv"]
    scales = [torch.full((pool, heads, page), math.nan) for _ in "kv"]
    for b in range(batch):
        for i in range(per):
            n = min(page, length - i * page)
            for pool_t, t in zip(values, (k, v)):
                pool_t[ids[b, i], :n] = t[b, i * page : i * page + n]
            for pool_t, t in zip(scales, (ks, vs)):
                pool_t[ids[b, i], :, :n] = t[b, :, i * page : i * page + n]
    table = PageTable(ids.to(torch.int32).cuda(), length)
    return Cache8(*(t.cuda() for t in (*values, *scales))), table, ids


def reference(q, tensors, lengths, scale, window=None):
    """Output, weights times |v|, the largest |q| |k| scale sum per row and head, weights
    times v's scales, the largest |q| sum times a key's scale and the scale."""
    k, v, ks, vs = (t.double() for t in tensors)
    batch, heads, d = q.shape
    group = heads // k.shape[2]
    out = torch.zeros(batch, heads, d, dtype=torch.float64)
    weighted, largest = torch.zeros_like(out), torch.zeros(batch, heads, 1, dtype=torch.float64)
    units, queries = torch.zeros_like(largest), torch.zeros_like(largest)
    for b, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        if n <= first:
            continue
        kb = (k[b, first:n] * ks[b, :, first:n].T[..., None]).transpose(0, 1).repeat_interleave(group, 0)
        vb = (v[b, first:n] * vs[b, :, first:n].T[..., None]).transpose(0, 1).repeat_interleave(group, 0)
        qb = q[b].double()[:, None] * scale
        w = torch.softmax((qb * kb).sum(-1), -1)[:, None]
        out[b], weighted[b] = (w @ vb)[:, 0], (w @ vb.abs())[:, 0]
        largest[b] = (qb.abs() * kb.abs()).sum(-1).amax(-1, keepdim=True)
        units[b] = (w[:, 0] * vs[b, :, first:n].repeat_interleave(group, 0)).sum(-1, keepdim=True)
        queries[b] = qb.abs().sum(-1) * ks[b, :, first:n].repeat_interleave(group, 0).amax(-1, keepdim=True)
    return out, weighted, largest, units, queries


def check(out, q, tensors, lengths, scale=None, window=None, queries_off=0.0):
    """queries_off: how far the call's own queries are from q, of a head's largest."""
    d = q.shape[-1]
    ref, weighted, largest, units, queries = reference(q, tensors, lengths, d**-0.5 if scale is None else scale, window)
    n = torch.tensor([min(x, window or x) for x in lengths]).view(-1, 1, 1).double()
    step, parts = (2.0**-8, 2.0**-16) if q.dtype == BF16 else (2.0**-24, 2.0**-23)
    bound = 1.01 * (weighted * (2.0**-24 * (2 * (d + 8) * largest + 2 * n + 64) + parts) + step * ref.abs())
    bound += 1.01 * weighted * 2 * queries_off * q.double().abs().amax(-1, keepdim=True) * keys_sum(tensors, q, lengths, scale)
    if q.dtype == BF16:
        bound += 1.01 * 2.0**-24 * 510 * ((n + 64) * units + 2 * weighted * (d + 8) * queries)
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    worst = ((out - ref).abs() / bound.clamp(min=1e-40)).max()
    assert worst <= 1, float(worst)


def keys_sum(tensors, q, lengths, scale):
    """The largest sum of |k| times the scale over a row's keys, per query head."""
    k, _, ks, _ = (t.double() for t in tensors)
    group, d = q.shape[1] // k.shape[2], q.shape[2]
    sums = [((k[b, :n].abs().sum(-1) * ks[b, :, :n].T).amax(0) if n else k.new_zeros(k.shape[2])) for b, n in enumerate(lengths)]
    return torch.stack(sums).repeat_interleave(group, 1)[..., None] * (d**-0.5 if scale is None else scale)


def spread(lengths, dtype=torch.int32):
    return torch.tensor(lengths, dtype=dtype, device="cuda")


SHAPES = [
    # batch, heads, kv heads, head_dim, length
    (1, 1, 1, 64, 1), (1, 16, 8, 128, 480), (2, 4, 4, 64, 31), (3, 6, 6, 64, 33), (5, 6, 6, 64, 1500), (2, 8, 1, 256, 700),
    (4, 12, 4, 128, 65), (2, 16, 2, 128, 1000), (1, 17, 1, 64, 300), (2, 40, 1, 128, 200), (40, 16, 8, 128, 100),
    (3, 5, 1, 256, 260), (1, 8, 8, 64, 9001), (70, 4, 4, 256, 40), (2, 2, 1, 128, 20000),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,heads,kv,head_dim,length", SHAPES)
def test_attention(dtype, batch, heads, kv, head_dim, length):
    """Slabs of both layouts and pages, all lengths from none on, int32 and int64."""
    from asrback_amd.cache8 import decode8

    g = torch.Generator().manual_seed(batch * 1000 + length)
    q = torch.randn(batch, heads, head_dim, generator=g).to(dtype)
    lengths = [length] + [int(x) for x in torch.randint(0, length + 1, (batch - 1,), generator=g)]
    if batch > 2:
        lengths[1] = 0
    say("decode8", dtype, batch, heads, kv, head_dim, length)
    cache, tensors = random_cache(batch, length, kv, head_dim, g, head_major=batch % 2 == 0)
    out = decode8(q.cuda(), cache, lengths=spread(lengths))
    check(out, q, tensors, lengths)
    assert all(not out[b].any() for b, n in enumerate(lengths) if n == 0)
    if batch == 1:
        assert torch.equal(decode8(q.cuda(), cache), out)
    for page in (16, 64):
        pool, table, _ = paged(tensors, page, g)
        say("pages of", page)
        assert torch.equal(decode8(q.cuda(), pool, lengths=spread(lengths, torch.int64), pages=table), out)
    for window in (1, 30, length + 5):
        say("window", window)
        out = decode8(q.cuda(), cache, lengths=spread(lengths), window=window)
        check(out, q, tensors, lengths, window=window)
        assert torch.equal(decode8(q.cuda(), pool, lengths=spread(lengths), window=window, pages=table), out)


LONG = [
    # heads, kv heads, head_dim, room, lengths: splits by lengths, equal splits, none
    (4, 2, 128, 20000, (20000, 4097, 9031)), (16, 8, 128, 40032, (31999, 40032)), (6, 6, 64, 9000, (9000, 1, 0, 8801, 33)),
    (8, 1, 256, 6000, (5999, 6000, 4512)), (17, 1, 64, 12000, (11999, 7)), (16, 8, 128, 9001, (9001,)),
    (4, 4, 64, 1500, (1500, 700, 1499)), (2, 2, 128, 300, tuple(300 - 2 * b for b in range(140))),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv,head_dim,room,lengths", LONG)
@pytest.mark.parametrize("page", [0, 16])
def test_every_key_counts_once(dtype, heads, kv, head_dim, room, lengths, page):
    """Queries of zeros weigh every key 1, and keys have values at one dimension each: an output
    is the number of keys at its dimension over that of all.  Sums of whole numbers below 2^24
    are exact, so that only the quotient's two roundings are left, and a key (a tile) that is
    lost or taken twice stands out of the keys of its dimension."""
    from asrback_amd.attention import PageTable
    from asrback_amd.cache8 import Cache8, decode8

    g = torch.Generator().manual_seed(room)
    batch, scale = len(lengths), 0.25
    q = torch.zeros(batch, heads, head_dim, device="cuda", dtype=dtype)
    step = 2.0**-8 if dtype == BF16 else 2.0**-23
    at, table = torch.arange(room), None
    # By keys, and by tiles of 32.
    for dims in (at % head_dim, at // 32 % head_dim):
        values = torch.zeros(batch, room, kv, head_dim, dtype=torch.int8)
        values[:, at, :, dims] = 127
        tensors = [torch.randint(-127, 128, values.shape, generator=g, dtype=torch.int8), values,
                   *(torch.full((batch, kv, room), scale) for _ in "kv")]
        if page:
            cache, table, _ = paged(tensors, page, g)
            table = PageTable(table.block_table, room)
        else:
            cache = Cache8(*(t.cuda() for t in tensors))
        for window in (None, 1000, 4100):
            say("counts", dtype, heads, kv, head_dim, room, page, window)
            out = decode8(q, cache, lengths=spread(lengths), pages=table, window=window).cpu().double()
            for b, n in enumerate(lengths):
                first = max(0, n - window) if window else 0
                counts = torch.bincount(dims[first:n], minlength=head_dim).double()
                ref = counts * 127 * scale / max(1, n - first)
                assert ((out[b] - ref).abs() <= 1.01 * step * ref).all(), (b, n)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,room", [(128, 20000), (64, 40000), (256, 5000)])
def test_one_key_among_many(dtype, head_dim, room):
    """A key that dwarfs the others, at both ends of halves, tiles, turns of the waves and
    about everywhere else: its value comes out, whichever workgroup holds it."""
    from asrback_amd.cache8 import Cache8, decode8

    g = torch.Generator().manual_seed(head_dim)
    batch, kv = 2, 8
    near = [p + d for p in (0, 16, 32, 64, 128, 256, 512, 1024, 4096, room // 2 // 32 * 32) for d in (-1, 0, 1)]
    near += [*range(room // 40, room - 40, room // 40), room - 33, room - 32, room - 1]
    near = [p for p in near if 0 <= p < room]
    q = torch.zeros(batch, 2 * kv, head_dim)
    q[..., 0] = 1
    values = torch.randint(-127, 128, (batch, room, kv, head_dim), generator=g, dtype=torch.int8).cuda()
    ones = torch.ones(batch, kv, room, device="cuda")
    for first in range(0, len(near), kv):
        places = [near[(first + h) % len(near)] for h in range(kv)]
        keys = torch.zeros(batch, room, kv, head_dim, dtype=torch.int8, device="cuda")
        for h, p in enumerate(places):
            keys[:, p, h, 0] = 127
        lengths = [room, max(places) + 1]
        say("one key", dtype, head_dim, places)
        out = decode8(q.to("cuda", dtype), Cache8(keys, values, ones, ones / 8), lengths=spread(lengths), scale=1.0)
        # The others' weights are e^-127 each.
        ref = torch.stack([values[:, p, h].float() / 8 for h, p in enumerate(places)], 1).repeat_interleave(2, 1)
        assert torch.equal(out.float(), ref)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_places_hold_anything(dtype):
    """Positions past a row's keys and before its window hold NaN and infinite scales, and
    table entries outside the pool nothing."""
    from asrback_amd.attention import PageTable
    from asrback_amd.cache8 import Cache8, decode8

    g = torch.Generator().manual_seed(4)
    batch, heads, kv, d, length = 4, 8, 4, 128, 200
    q = torch.randn(batch, heads, d, generator=g).to(dtype)
    lengths, window = [0, 77, 128, 200], 50
    cache, tensors = random_cache(batch, length, kv, d, g)
    dirty = [t.clone() for t in cache.tensors]
    for b, n in enumerate(lengths):
        for t, bad in zip(dirty[2:], (math.nan, math.inf)):
            t[b, :, n:] = bad
            t[b, :, : max(0, n - window)] = -bad
    out = decode8(q.cuda(), Cache8(*dirty), lengths=spread(lengths), window=window)
    check(out, q, tensors, lengths, window=window)
    # Lengths outside the cache are clamped to it.
    ends = decode8(q.cuda(), cache, lengths=spread([-5, 200, 1 << 30, 0]))
    check(ends, q, tensors, [0, 200, 200, 0])
    pool, table, ids = paged(tensors, 16, g)
    broken = ids.clone()
    broken[1, 2], broken[2, 0], broken[3, 5] = -1, 99999, -7
    out = decode8(q.cuda(), pool, lengths=spread(lengths), pages=PageTable(broken.to(torch.int32).cuda(), length))
    for b, gone in ((1, 2), (2, 0), (3, 5)):
        kept = [j for j in range(lengths[b]) if j // 16 != gone]
        part = tuple(t[b : b + 1, kept] if i < 2 else t[b : b + 1][..., kept] for i, t in enumerate(tensors))
        check(out[b : b + 1], q[b : b + 1], part, [len(kept)])
    none = PageTable(torch.full((4, 13), -1, dtype=torch.int32, device="cuda"), length)
    assert not decode8(q.cuda(), pool, lengths=spread(lengths), pages=none).any()
    empty = Cache8(*(t[:0] for t in pool.tensors))
    assert not decode8(q.cuda(), empty, lengths=spread(lengths), pages=none).any()
    assert not decode8(q.cuda(), Cache8.allocate(4, 0, kv, d, "cuda")).any()
    assert decode8(q[:0].cuda(), Cache8.allocate(0, 8, kv, d, "cuda")).shape == (0, heads, d)
    # A scale of NaN at a key that is seen shows; so does a query that is not finite.
    seen = [t.clone() for t in cache.tensors]
    seen[2][3, 1, 10] = math.nan
    out = decode8(q.cuda(), Cache8(*seen))
    assert torch.isnan(out[3, 2:4]).all() and torch.isfinite(out[:3]).all() and torch.isfinite(out[3, 4:]).all()
    bad = q.clone()
    bad[1, 0, 5] = math.nan
    out = decode8(bad.cuda(), cache)
    assert torch.isnan(out[1, 0]).all() and torch.isfinite(out[1, 1:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_far_scores_and_values(dtype):
    """One key far above the others, a thousand equal ones, values of very different
    scales: no weight is lost."""
    from asrback_amd.cache8 import Cache8, decode8

    g = torch.Generator().manual_seed(9)
    batch, heads, kv, d, length = 3, 4, 2, 64, 1200
    q = torch.randn(batch, heads, d, generator=g).to(dtype)
    cache, tensors = random_cache(batch, length, kv, d, g)
    k, v, ks, vs = (t.clone() for t in tensors)
    ks[0, :, 700] *= 40
    ks[1] *= 1e-6
    vs[1, :, ::3] *= 1e12
    ks[2] *= 30
    for out_scale in (None, 1.0):
        cache = Cache8(*(t.cuda() for t in (k, v, ks, vs)))
        check(decode8(q.cuda(), cache, scale=out_scale), q, (k, v, ks, vs), [length] * batch, out_scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_and_scales_far_from_one(dtype):
    """Powers of two that take the products out of range, by themselves or together, where
    the scores are not: ordinary scores, and ones so far apart that one key is left."""
    from asrback_amd.cache8 import Cache8, decode8

    g = torch.Generator().manual_seed(19)
    batch, heads, kv, d, length = 2, 4, 2, 64, 300
    _, (k, v, ks, vs) = random_cache(batch, length, kv, d, g)
    plain = torch.randn(batch, heads, d, generator=g)
    for queries, keys in ((-60, 53), (-100, 93), (50, -57), (62, -69), (100, -107), (0, 90), (40, 60), (70, 30), (-30, -60)):
        q = (plain * 2.0**queries).to(dtype)
        tensors = k, v, ks * 2.0**keys, vs
        # One row's scale alone far off.
        tensors[2][1, 0, 5] *= 2.0**-40
        say("far", dtype, queries, keys)
        out = decode8(q.cuda(), Cache8(*(t.cuda() for t in tensors)), lengths=spread([length, 250]))
        check(out, q, tensors, [length, 250])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tiny_queries_beside_large_values(dtype):
    """Ordinary scores of tiny queries and huge keys, in tiles whose values' scales are large
    as well: those are converted, and the queries' power of two is far from 1."""
    from asrback_amd.cache8 import Cache8, decode8, decode_append8, write_rows8

    g = torch.Generator().manual_seed(23)
    batch, heads, kv, d, length = 2, 4, 2, 64, 300
    _, (k, v, ks, vs) = random_cache(batch, length, kv, d, g)
    plain, lengths = torch.randn(batch, heads, d, generator=g), [length, 250]
    rows = [torch.randn(batch, n, d, generator=g).to(dtype) for n in (heads, kv, kv)]
    norms = [(torch.rand(d, generator=g) + 0.5) for _ in "qk"]
    angles = torch.rand(batch, d // 2, generator=g).repeat(1, 2)
    for power in (20, 30, 40, 60, 100):
        q = (plain * 2.0**-power).to(dtype)
        tensors = k, v, ks * 2.0 ** (power - 7), vs.clone()
        tensors[3][:, :, 64:96] *= 2.0**20  # one tile's
        tensors[3][1, 1, 200] *= 2.0**20
        say("tiny queries", dtype, power)
        cache = Cache8(*(t.cuda() for t in tensors))
        check(decode8(q.cuda(), cache, lengths=spread(lengths)), q, tensors, lengths)
        # A step whose new key and value are such ones.
        new = {"q_norm": (norms[0] * 2.0**-power).to(dtype).cuda(), "k_norm": (norms[1] * 2.0 ** (power - 3)).to(dtype).cuda(),
               "q_eps": 1e-6, "k_eps": 1e-6, "cos": angles.cos().to(dtype).cuda(), "sin": angles.sin().to(dtype).cuda()}
        x = rows[0].cuda(), rows[1].cuda(), (rows[2] * 2.0**20).cuda()
        positions = torch.tensor([n - 1 for n in lengths], device="cuda")
        out = decode_append8(*x, cache, positions, **new)
        queries, _ = write_rows8(Cache8.allocate(batch, length, kv, d, "cuda"), *x, None, positions, **new)
        # (Queries rounded by another kernel: 2^-21 of their largest in float32.)
        check(out, queries.cpu(), [t.cpu() for t in cache.tensors], lengths, queries_off=0.0 if dtype == BF16 else 2.0**-21)


def test_windows_past_32_bits():
    from asrback_amd.cache8 import decode8

    g = torch.Generator().manual_seed(31)
    cache, _ = random_cache(2, 5000, 2, 64, g)
    q, lengths = torch.randn(2, 4, 64, generator=g).to("cuda", BF16), spread([5000, 321])
    say("windows")
    whole = decode8(q, cache, lengths=lengths)
    for window in (5000, 1 << 30, (1 << 31) - 1, 1 << 32, 1 << 80):
        assert torch.equal(decode8(q, cache, lengths=lengths, window=window), whole)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales_below_zero(dtype):
    """Another quantizer's scales may be negative, and large: of values, of keys that queries
    are small for."""
    from asrback_amd.cache8 import Cache8, decode8, read8

    g = torch.Generator().manual_seed(29)
    batch, heads, kv, d, length = 2, 4, 2, 128, 300
    _, (k, v, ks, vs) = random_cache(batch, length, kv, d, g)
    lengths = [length, 77]
    signs = [torch.randint(0, 2, ks.shape, generator=g) * 2.0 - 1 for _ in "kv"]
    for s in signs:
        s[..., :160] = -1  # whole tiles
    for power, values in ((0, 1.0), (0, 2.0**16), (90, 2.0**5), (-60, 2.0**-40)):
        tensors = k, v, signs[0] * ks * 2.0**power, signs[1] * vs * values
        q = (torch.randn(batch, heads, d, generator=g) * 2.0 ** (-power - 2)).to(dtype)
        say("negative", dtype, power, values)
        cache = Cache8(*(t.cuda() for t in tensors))
        # (The bound takes magnitudes: of scales with a sign, those of the numbers they scale.)
        flat = [k * signs[0].transpose(1, 2)[..., None].to(torch.int8), v * signs[1].transpose(1, 2)[..., None].to(torch.int8),
                tensors[2].abs(), tensors[3].abs()]
        check(decode8(q.cuda(), cache, lengths=spread(lengths)), q, flat, lengths)
        for out, t, s in zip(read8(cache, dtype=dtype), (k, v), tensors[2:]):
            assert torch.equal(out.cpu(), (t.float() * s.transpose(1, 2)[..., None]).to(dtype))


def test_long_cache_past_32_bits():
    """Positions whose offsets pass 2^31 and 2^32 bytes."""
    from asrback_amd.cache8 import Cache8, decode8, read8, write8

    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free memory")
    g = torch.Generator().manual_seed(2)
    length, kv, d = (1 << 22) + 40, 8, 128  # 4.3 GB each of keys and values
    say("long cache")
    cache = Cache8.allocate(1, length, kv, d, "cuda")
    at = [5, (1 << 21) + 3, (1 << 22) - 1, (1 << 22) + 39]
    k, v = (torch.randn(len(at), kv, d, generator=g).to(BF16) for _ in "kv")
    k *= 40  # above the zeros between them
    q = k[torch.arange(4) % 4][:1].reshape(1, kv, d).clone()
    write8(cache, k.cuda(), v.cuda(), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.tensor(at, device="cuda"))
    (qk, sk), (qv, sv) = rounded(k), rounded(v)
    assert torch.equal(cache.keys[0, at].cpu(), qk) and torch.equal(cache.key_scales[0, :, at].cpu().T, sk)
    assert torch.equal(cache.values[0, at].cpu(), qv)
    for seen, n in ((1, 6), (2, (1 << 21) + 4), (4, length)):
        out = decode8(q.cuda(), cache, lengths=spread([n]), window=n).cpu().double()
        s = (q.double()[0] * (qk[:seen].double() * sk[:seen, :, None].double())).sum(-1) * d**-0.5  # (seen, heads)
        e = torch.cat((s, torch.full((1, kv), 0.0, dtype=torch.float64)))
        top = e.amax(0)
        w = torch.exp(s - top)
        total = w.sum(0) + (n - seen) * torch.exp(-top)
        ref = (w[..., None] * qv[:seen].double() * sv[:seen, :, None].double()).sum(0) / total[:, None]
        # The first key dwarfs the others: its score is off by at most 2^-24 (2 d) of |q| |k|.
        assert ((out[0] - ref).abs() <= 2.0**-8 * ref.abs() + 2.0**-7 * ref.abs().amax()).all()
    two = Cache8(*(t[:, -64:] for t in cache.tensors[:2]), *(t[..., -64:] for t in cache.tensors[2:]))
    keys, _ = read8(two)
    assert torch.equal(keys[0, -1].cpu(), (qk[3].float() * sk[3, :, None]).to(BF16))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv,head_dim", [(6, 64), (8, 128), (1, 256), (5, 128)])
def test_write_and_read_back(dtype, kv, head_dim):
    """Slabs and pages, odd strides, slots outside the cache, positions left as they
    were; ties, rows of zeros, NaN and infinities."""
    from asrback_amd.attention import PageTable
    from asrback_amd.cache8 import Cache8, read8, write8

    g = torch.Generator().manual_seed(kv)
    batch, length, tokens = 3, 96, 50
    wide = torch.randn(tokens, 2 * kv + 1, head_dim, generator=g).to(dtype)
    wide[3] = 0
    wide[4, :, 0] = 127.0
    wide[4, :, 1:] = (torch.arange(head_dim - 1) % 254 - 126.5).to(dtype)
    wide[5, 0, 3], wide[6, 0, 4] = math.nan, math.inf
    k, v = wide[:, :kv], wide[:, kv : 2 * kv]
    slots = torch.randperm(batch * length, generator=g)[:tokens]
    rows, positions = slots // length, slots % length
    rows[7], rows[8], positions[9], positions[10] = -1, batch, -1, length
    cache, tensors = random_cache(batch, length, kv, head_dim, g)
    pool, table, ids = paged(tensors, 32, g)
    broken = ids.clone()
    broken[1, 1] = -1
    pool_before = [t.clone() for t in pool.tensors]
    table = PageTable(broken.to(torch.int32).cuda())
    say("write8", dtype, kv, head_dim)
    versions = [t._version for t in cache.tensors]
    write8(cache, k.cuda(), v.cuda(), rows.cuda(), positions.cuda())
    write8(pool, k.cuda(), v.cuda(), rows.cuda(), positions.cuda(), pages=table)
    assert all(t._version > old for t, old in zip(cache.tensors, versions))
    want = [t.clone() for t in tensors]
    for t in range(tokens):
        b, at = int(rows[t]), int(positions[t])
        if not (0 <= b < batch and 0 <= at < length):
            continue
        for x, values, scales in ((k, want[0], want[2]), (v, want[1], want[3])):
            finite = torch.isfinite(x[t]).all(-1)
            q, s = rounded(torch.where(finite[:, None], x[t], torch.zeros_like(x[t])))
            values[b, at] = torch.where(finite[:, None], q, cache.values[b, at].cpu() if x is v else cache.keys[b, at].cpu())
            scales[b, :, at] = torch.where(finite, s, math.nan)
    for have, t in zip(cache.tensors, want):
        assert torch.equal(have.cpu().nan_to_num(7.0) if t.is_floating_point() else have.cpu(),
                           t.nan_to_num(7.0) if t.is_floating_point() else t)
    # Pages: the same, but of the page that is not there.
    back, lengths = read8(cache, dtype=dtype), [96, 50, 0]
    held = read8(pool, pages=table, dtype=dtype)
    for a, b in zip(back, held):
        a = a.clone()
        a[1, 32:64] = 0
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    owned = set(int(x) for x in ids.flatten())
    for page in range(pool.keys.shape[0]):
        if page not in owned or page == int(ids[1, 1]):
            for a, b in zip(pool.tensors, pool_before):
                assert torch.equal(a[page].nan_to_num(7.0) if a.is_floating_point() else a[page],
                                   b[page].nan_to_num(7.0) if b.is_floating_point() else b[page])
    for out, values, scales in zip(back, want[:2], want[2:]):
        ref = (values.float() * scales.transpose(1, 2)[..., None]).to(dtype)
        assert torch.equal(out.cpu().nan_to_num(7.0), ref.nan_to_num(7.0))
    for kind in (torch.int32, torch.int64):
        part = read8(cache, lengths=spread(lengths, kind), dtype=dtype)
        for a, b in zip(back, part):
            for row, n in enumerate(lengths):
                assert torch.equal(a[row, :n].nan_to_num(7.0), b[row, :n].nan_to_num(7.0)) and not b[row, n:].any()
    # One token a row, and none.
    one = Cache8.allocate(4, 9, kv, head_dim, "cuda")
    write8(one, k[:4].cuda(), v[:4].cuda(), None, torch.tensor([0, 8, 3, 9], device="cuda"))
    assert torch.equal(one.keys[1, 8].cpu(), rounded(k[1])[0]) and not one.keys[3].any() and not one.keys[0, 1:].any()
    write8(one, k[:0].cuda(), v[:0].cuda(), None, torch.zeros(0, dtype=torch.int64, device="cuda"))
    empty = Cache8(*(t[:0] for t in pool.tensors))
    write8(empty, k.cuda(), v.cuda(), rows.cuda(), positions.cuda(), pages=table)
    assert not read8(empty, pages=table)[0].any()
    write8(Cache8.allocate(0, 9, kv, head_dim, "cuda"), k.cuda(), v.cuda(), rows.cuda(), positions.cuda())  # of no rows


def test_rows_of_a_decoder():
    """The norms and the rotation before the write are the prompt pass's: in bf16 to the
    bit; in float32 the rotation's sum may be contracted with either of its products, so
    that results differ by a rounding of each of two terms, 2^-24 of at most sqrt(2)
    times the row's largest, and of the norm's two products."""
    from asrback_amd.cache8 import Cache8, write8, write_rows8
    from asrback_amd.layers import prompt_rows
    from asrback_amd.qwen3_asr import RMSNorm, rope_tables

    for dtype in (BF16, F32):
        for head_dim, heads, kv in ((128, 16, 8), (64, 3, 3), (256, 8, 1)):
            torch.manual_seed(head_dim)
            tokens = 37
            config = {"head_dim": head_dim, "rope_theta": 1e6}
            cos, sin = rope_tables(config, tokens, "cuda", dtype)
            qkv = torch.randn(tokens, heads + 2 * kv, head_dim, device="cuda").to(dtype)
            q, k, v = qkv.split((heads, kv, kv), 1)
            norms = [RMSNorm(head_dim, eps).to("cuda", dtype) for eps in (1e-6, 1e-5)]
            for m in norms:
                m.weight.data.uniform_(0.5, 1.5)
            rows = torch.arange(tokens, device="cuda") % 2
            positions = torch.arange(tokens, device="cuda") // 2
            scratch = [torch.zeros(2, tokens, kv, head_dim, device="cuda", dtype=dtype) for _ in "kv"]
            with torch.no_grad():
                q_ref, k_ref, _ = prompt_rows(q, k, v, *scratch, rows, positions, *norms, cos, sin)
                want, have = (Cache8.allocate(2, tokens, kv, head_dim, "cuda") for _ in "ab")
                q_out, k_out = write_rows8(have, q, k, v, rows, positions, q_norm=norms[0].weight, k_norm=norms[1].weight,
                                           q_eps=norms[0].eps, k_eps=norms[1].eps, cos=cos, sin=sin, keys=True)
            say("write_rows8", dtype, head_dim)
            write8(want, k_out, v, rows, positions)
            for a, b in ((q_out, q_ref), (k_out, k_ref)):
                if dtype == BF16:
                    assert torch.equal(a, b)
                else:
                    assert ((a - b).abs() <= 2.0**-21 * b.abs().amax(-1, keepdim=True)).all()
            for a, b in zip(want.tensors, have.tensors):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv,head_dim,length,page,window", [
    (16, 8, 128, 1024, 0, None), (4, 2, 128, 200, 16, None), (3, 3, 64, 512, 0, None), (8, 1, 256, 640, 64, None),
    (40, 2, 64, 300, 0, 33), (16, 8, 128, 8192, 0, None), (4, 4, 256, 96, 32, 1), (34, 1, 128, 5000, 128, 700),
])
def test_steps_that_append(dtype, heads, kv, head_dim, length, page, window):
    """A step in one launch against its write and attention: positions at both ends of the
    cache, outside it, on no page and inside pages.  Both round the same rows; in float32
    the rotation's sum may be contracted differently (2^-21 of a row's largest, as in
    test_rows_of_a_decoder), so that scales and numbers at a border may differ."""
    from asrback_amd.attention import PageTable
    from asrback_amd.cache8 import Cache8, decode8, decode_append8, write_rows8
    from asrback_amd.qwen3_asr import rope_tables

    g = torch.Generator().manual_seed(heads * length)
    where = [0, length - 1, length // 2, 31, 32, -1, length, length + 700, -4, length // 3, 2**62]
    batch = len(where)
    _, tensors = random_cache(batch, length, kv, head_dim, g)
    tensors = list(tensors)
    for b, p in enumerate(where):  # what is not held yet may be anything
        if 0 <= p < length:
            tensors[2][b, :, p:] = math.nan
            tensors[3][b, :, p:] = math.inf
    pages = None
    if page:
        cache, pages, ids = paged(tensors, page, g)
        ids = ids.clone()
        ids[2, (length // 2) // page] = -1  # the new key's page
        ids[9, 0] = -1 if length // 3 >= page else ids[9, 0]
        pages = PageTable(ids.to(torch.int32).cuda(), length)
        both = [Cache8(*(t.clone() for t in cache.tensors)) for _ in "ab"]
    else:
        both = [Cache8(*(t.cuda() for t in tensors)) for _ in "ab"]
    q, k, v = (torch.randn(batch, n, head_dim, generator=g).to("cuda", dtype) for n in (heads, kv, kv))
    norms = [(torch.rand(head_dim, generator=g) + 0.5).to("cuda", dtype) for _ in "qk"]
    cos, sin = (t[:batch].flip(0) for t in rope_tables({"head_dim": head_dim, "rope_theta": 1e4}, batch, "cuda", dtype))
    more = {"q_norm": norms[0], "k_norm": norms[1], "q_eps": 1e-6, "k_eps": 1e-5, "cos": cos, "sin": sin}
    positions = torch.tensor(where, device="cuda")
    say("append", dtype, heads, kv, head_dim, length, page, window)
    # (The queries written over, and strided keys.)
    given = q.clone()
    strided = torch.stack((k, v), 2).flatten(1, 2)
    out = decode_append8(given, strided[:, ::2], strided[:, 1::2], both[1], positions, pages=pages, window=window,
                         out=given, **more)
    assert out is given
    queries, _ = write_rows8(both[0], q, k, v, None, positions, pages=pages, **more)
    counts = [min(max(p + 1, 0), length) for p in where]
    want = decode8(queries, both[0], lengths=spread(counts), pages=pages, window=window)
    for a, b in zip(*(c.tensors for c in both)):
        if dtype == BF16:
            assert torch.equal(a, b) if a.dtype == torch.int8 else torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))
        elif a.dtype == torch.int8:
            assert (a.int() - b.int()).abs().max() <= 1
        else:
            assert ((a - b).abs() <= 2.0**-21 * b.abs()).logical_or(a.isnan() & b.isnan()).logical_or(a == b).all()
    for b, n in enumerate(counts):
        if n == 0:
            assert not out[b].any()
    # Rows whose pages are all there, against float64 of the step's own cache.
    rows = [b for b in range(batch) if not page or b not in (2, 9)]
    if page:
        held = [t.cpu() for t in both[1].tensors]
        whole = [torch.stack([t[ids[b]].flatten(0, 1)[:length] for b in rows]) for t in held[:2]]
        whole += [torch.stack([t[ids[b]].transpose(0, 1).flatten(1)[:, :length] for b in rows]) for t in held[2:]]
    else:
        whole = [t.cpu()[rows] for t in both[1].tensors]
    check(out[rows], queries[rows].cpu(), whole, [counts[b] for b in rows], window=window,
          queries_off=0.0 if dtype == BF16 else 2.0**-21)
    # Rows with a page missing: the other call's answer, both within their bounds.
    for b in set(range(batch)) - set(rows):
        assert (out[b].double() - want[b].double()).abs().max() <= 2.0**-6 * want[b].double().abs().max()


def test_run_of_steps_in_a_graph_and_beside_another():
    """Write and attention as a decoder runs them, captured and replayed while positions
    move, two graphs sharing a workspace; an out given, q itself among them."""
    from asrback_amd.attention import workspace
    from asrback_amd.cache8 import Cache8, decode8, decode8_workspace_size, write8

    g = torch.Generator().manual_seed(1)
    batch, heads, kv, d, length = 2, 16, 8, 128, 600
    cache, _ = random_cache(batch, length, kv, d, g)
    other = Cache8(*(t.clone() for t in cache.tensors))
    buffer = torch.full((decode8_workspace_size(batch, heads, kv, d, length),), 255, dtype=torch.uint8, device="cuda")
    q = torch.randn(batch, heads, d, generator=g).to("cuda", BF16)
    new = [torch.randn(batch, kv, d, generator=g).to("cuda", BF16) for _ in "kv"]
    positions = torch.tensor([300, 511], device="cuda")

    def step(cache):
        write8(cache, *new, None, positions)
        return decode8(q, cache, lengths=positions + 1)

    graphs, outs = [], []
    with torch.no_grad(), workspace(buffer):
        step(cache), step(other)
        for held in (cache, cache):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(step(held))
            graphs.append(graph)
    for turn in range(4):
        q.copy_(torch.randn(batch, heads, d, generator=g))
        for t in new:
            t.copy_(torch.randn(batch, kv, d, generator=g))
        positions += 1
        with torch.no_grad():
            want = step(other)
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
        for a, b in zip(cache.tensors, other.tensors):
            assert torch.equal(a[..., :2], b[..., :2])
        torch.cuda.synchronize()
    want = decode8(q, cache)
    held = torch.zeros(batch, heads, 2 * d, device="cuda", dtype=BF16)
    out = decode8(q, cache, out=held[..., 1 : d + 1])
    assert torch.equal(out, want) and not held[..., 0].any() and not held[..., d + 1 :].any()
    same = q.clone()
    assert decode8(same, cache, out=same) is same and torch.equal(same, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = decode8(q, cache)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, want)


def test_appending_steps_in_graphs():
    """decode_append8 captured twice over one workspace, replayed while positions move past a
    page's end, eager calls between; and on two streams at once, each with memory of its
    own."""
    from asrback_amd.attention import PageTable, workspace
    from asrback_amd.cache8 import Cache8, decode_append8, decode8_workspace_size
    from asrback_amd.qwen3_asr import rope_tables

    g = torch.Generator().manual_seed(7)
    batch, heads, kv, d, page, length = 3, 16, 8, 128, 64, 1024
    _, tensors = random_cache(batch, length, kv, d, g)
    first, pages, _ = paged(tensors, page, g)
    caches = [Cache8(*(t.clone() for t in first.tensors)) for _ in range(3)]
    buffer = torch.full((decode8_workspace_size(batch, heads, kv, d, length),), 255, dtype=torch.uint8, device="cuda")
    q, k, v = (torch.randn(batch, n, d, generator=g).to("cuda", BF16) for n in (heads, kv, kv))
    norm = torch.ones(d, device="cuda", dtype=BF16)
    tables = rope_tables({"head_dim": d, "rope_theta": 1e6}, length, "cuda", BF16)
    positions = torch.tensor([300, 509, 1021], device="cuda")

    def step(cache):
        cos, sin = (t[positions.clamp(max=length - 1)] for t in tables)
        return decode_append8(q, k, v, cache, positions, q_norm=norm, k_norm=norm, q_eps=1e-6, k_eps=1e-6, cos=cos, sin=sin,
                              pages=PageTable(pages.block_table, length))

    def follow():
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        positions.add_(1)

    graphs, outs = [], []
    with torch.no_grad(), workspace(buffer):
        for cache in caches:
            step(cache)
        for cache in caches[:2]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(step(cache))
            graphs.append(graph)
    for turn in range(5):  # the last row's position leaves the cache
        follow()
        with torch.no_grad():
            want = step(caches[2])
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
        for cache in caches[:2]:
            for a, b in zip(cache.tensors, caches[2].tensors):
                assert torch.equal(a.nan_to_num(5.0) if a.is_floating_point() else a,
                                   b.nan_to_num(5.0) if a.is_floating_point() else b)
        torch.cuda.synchronize()
    follow()
    streams, got = [torch.cuda.Stream() for _ in "ab"], []
    with torch.no_grad():
        for _ in range(3):
            for stream, cache in zip(streams, caches):
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):
                    got.append(step(cache))
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        want = step(caches[2])
    assert all(torch.equal(out, want) for out in got)


def test_most_rows_and_a_far_position():
    """As many rows as a call takes, and a step at an offset past 2^32 bytes."""
    from asrback_amd.cache8 import Cache8, decode8, decode_append8, write_rows8

    g = torch.Generator(device="cuda").manual_seed(3)
    batch, length, d = 65535, 16, 64
    cache = Cache8.allocate(batch, length, 1, d, "cuda")
    for t in cache.tensors[:2]:
        t.random_(-127, 128, generator=g)
    for t in cache.tensors[2:]:
        t.uniform_(0.01, 0.02, generator=g)
    q, k, v = (torch.randn(batch, n, d, device="cuda", generator=g).to(BF16) for n in (2, 1, 1))
    table, norm = torch.ones(batch, d, device="cuda", dtype=BF16), torch.ones(d, device="cuda", dtype=BF16)
    more = {"q_norm": norm, "k_norm": norm, "q_eps": 1e-6, "k_eps": 1e-6}
    positions = torch.arange(batch, device="cuda") % length
    say("most rows")
    out = decode_append8(q, k, v, cache, positions, cos=table, sin=table, **more)
    for part in (slice(0, 400), slice(batch - 400, batch)):  # over 256 rows: unsplit as well
        held = Cache8(*(t[part].clone() for t in cache.tensors))
        queries, _ = write_rows8(held, q[part], k[part], v[part], None, positions[part], cos=table[part], sin=table[part], **more)
        check(out[part], queries.cpu(), [t.cpu() for t in held.tensors], (positions[part] + 1).tolist())
        assert all(torch.equal(a, b[part]) for a, b in zip(held.tensors, cache.tensors))
        assert torch.equal(decode8(queries, held, lengths=positions[part] + 1),
                           decode8(queries, cache_part(cache, part), lengths=positions[part] + 1))
    del cache
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free memory")
    length, kv, d = (1 << 22) + 40, 8, 128
    say("far position")
    cache = Cache8.allocate(1, length, kv, d, "cuda")
    q, k, v = (torch.randn(1, n, d, device="cuda", generator=g).to(BF16) for n in (16, kv, kv))
    table, norm = torch.ones(1, d, device="cuda", dtype=BF16), torch.ones(d, device="cuda", dtype=BF16)
    at = torch.tensor([length - 3], device="cuda")
    more |= {"q_norm": norm, "k_norm": norm, "cos": table, "sin": table}
    out = decode_append8(q, k, v, cache, at, window=40, **more)
    tail = Cache8(*(t[:, -64:].clone() for t in cache.tensors[:2]), *(t[..., -64:].clone() for t in cache.tensors[2:]))
    assert tail.keys[0, 61].any() and not tail.keys[0, :61].any() and not tail.keys[0, 62:].any()
    queries, _ = write_rows8(tail, q, k, v, None, at - length + 64, **more)
    assert all(torch.equal(a, b) for a, b in zip((tail.keys[0, 61], tail.key_scales[..., 61]),
                                                 (cache.keys[0, -3], cache.key_scales[..., -3])))
    check(out, queries.cpu(), [t.cpu() for t in tail.tensors], [62], window=40)


def cache_part(cache, part):
    from asrback_amd.cache8 import Cache8

    return Cache8(*(t[part] for t in cache.tensors))
