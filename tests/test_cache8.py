"""CPU: the 8-bit cache's structures, what its ops refuse, and the decoder's caches."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from conftest import ROOT

CONFIG = {"num_hidden_layers": 2, "num_key_value_heads": 2, "head_dim": 64}


@pytest.mark.parametrize("name,struct", [("Linear8Params", "asrlayer_linear8_params"), ("Write8Params", "asrlayer_write8_params"),
                                         ("Read8Params", "asrlayer_read8_params"), ("Decode8Params", "asrlayer_decode8_params"),
                                         ("Append8Params", "asrlayer_append8_params")])
def test_structs_match_the_header(name, struct, tmp_path):
    """The cache's fields come first, one by one."""
    from asrback_amd import _lib

    cls = getattr(_lib, name)
    inner = ["k", "v", "k_scales", "v_scales", *[f"{t}_{a}_stride" for t in "kv" for a in ("batch", "token", "head")],
             *[f"{t}_{a}_stride" for t in ("ks", "vs") for a in ("batch", "head")], "block_table", "bt_stride", "page_size",
             "num_pages", "batch", "heads_kv", "head_dim", "max_len"]
    fields = [f for f, _ in cls._fields_]
    if name != "Linear8Params":
        assert len(_lib._CACHE8) == len(inner)
        fields = [f"cache.{f}" for f in inner] + fields[len(inner):]
    if name == "Append8Params":  # the step's fields and its padding first
        step = len(_lib.Decode8Params._fields_)
        assert fields[step] == "padding" and ctypes.sizeof(_lib.Decode8Params) == cls.padding.offset + cls.padding.size
        fields = [f"step.{f}" for f in fields[:step]] + fields[step + 1:]
    lines = [f'printf("%zu\\n", sizeof({struct}));', *(f'printf("%zu\\n", offsetof({struct}, {f}));' for f in fields)]
    source = tmp_path / "layout.cpp"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "layers.hpp"\nint main() {\n'
                      + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["g++", f"-I{ROOT / 'include'}", f"-I{ROOT / 'asrback_amd' / 'csrc'}", str(source), "-o",
                    str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_ if f != "padding")]


def test_caches():
    from asrback_amd.cache8 import Cache8

    k, s = torch.zeros(2, 8, 3, 64, dtype=torch.int8), torch.zeros(2, 3, 8)
    Cache8(k, k, s, s)
    Cache8(torch.zeros(2, 3, 8, 64, dtype=torch.int8).transpose(1, 2), k, s, torch.zeros(3, 2, 16)[:, :, 4:12].transpose(0, 1))
    Cache8(k[:0], k[:0], s[:0], s[:0])
    for bad, kind, match in (
        ((k[0], k[0], s, s), ValueError, "share one"),
        ((k, k[:, :7], s, s), ValueError, "share one"),
        ((k[..., :48], k[..., :48], s, s), ValueError, "supported head dims"),
        ((k[:, :, :0], k[:, :, :0], s[:, :0], s[:, :0]), ValueError, "0 heads"),
        ((k.float(), k, s, s), TypeError, "int8"),
        ((k, k.view(torch.uint8), s, s), TypeError, "int8"),
        ((torch.zeros(2, 8, 3, 65, dtype=torch.int8)[..., :64], k, s, s), ValueError, "16-byte"),
        ((torch.zeros(2, 8, 64, 3, dtype=torch.int8).transpose(2, 3), k, s, s), ValueError, "16-byte"),
        ((k, torch.zeros(2 * 8 * 3 * 64 + 8, dtype=torch.int8)[8:].view(2, 8, 3, 64), s, s), ValueError, "16-byte"),
        ((k, k, s.double(), s), ValueError, "float32"),
        ((k, k, s, s[..., :7]), ValueError, "float32"),
        ((k, k, s, torch.zeros(2, 8, 3).transpose(1, 2)), ValueError, "unit last"),
        ((k, k.to("meta"), s, s), RuntimeError, "one device"),
    ):
        with pytest.raises((kind, ValueError) if kind is RuntimeError else kind, match=None if kind is RuntimeError else match):
            Cache8(*bad)


def test_tensors_that_change_after_a_cache_is_made():
    """A cache keeps the memory and the layout that its tensors had, so that no call reads past
    what a resized or re-set one has; a copy has its own."""
    import copy
    import pickle

    from asrback_amd.cache8 import Cache8, _cache_fields

    def small(i, dtype):
        return torch.zeros((1, 1, 3, 64) if i < 2 else (1, 3, 1), dtype=dtype)

    for i in range(4):
        for change in (lambda t: t.set_(small(i, t.dtype)), lambda t: setattr(t, "data", small(i, t.dtype)),
                       lambda t: t.resize_(small(i, t.dtype).shape), lambda t: t.resize_(16, *t.shape[1:]),
                       lambda t: t.transpose_(0, 1), lambda t: setattr(t, "data", t.data.double())):
            tensors = Cache8.allocate(2, 8, 3, 64).tensors
            cache, other = Cache8(*tensors), Cache8(*tensors)
            before = _cache_fields(cache, None, 2, -1)
            change(tensors[i])
            after, sizes = _cache_fields(cache, None, 2, -1), [t.untyped_storage().nbytes() for t in other._held]
            # (A storage that grows may move.)
            assert after[:4] == tuple(t.data_ptr() for t in other._held) and after[4:] == before[4:]
            assert all(n >= need for n, need in zip(sizes, (2 * 8 * 3 * 64, 2 * 8 * 3 * 64, 2 * 8 * 3 * 4, 2 * 8 * 3 * 4)))
    cache = Cache8.allocate(2, 8, 3, 64)
    for twin in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert all(a.data_ptr() == b.data_ptr() != c.data_ptr() for a, b, c in zip(twin._held, twin.tensors, cache.tensors))
    assert copy.copy(cache).keys is cache.keys
    for t in cache.tensors:
        t += 1
    assert all((t == 1).all() for t in cache._held)


def calls():
    """Name, call of one float tensor, that tensor."""
    from asrback_amd.cache8 import Cache8, decode8, decode_append8, read8, write8, write_rows8

    cache = Cache8.allocate(2, 8, 3, 64)
    k, positions, weight, table = torch.zeros(2, 3, 64), torch.zeros(2, dtype=torch.int64), torch.zeros(64), torch.zeros(2, 64)

    def rows(q, k=k, weight=weight, table=table):
        return write_rows8(cache, q, k, k, None, positions, q_norm=weight, k_norm=weight, q_eps=1e-6, k_eps=1e-6, cos=table,
                           sin=table)

    def append(q, k=k, weight=weight, table=table):
        return decode_append8(q, k, k, cache, positions, q_norm=weight, k_norm=weight, q_eps=1e-6, k_eps=1e-6, cos=table,
                              sin=table)

    def scaled(x, f):
        return f(Cache8(cache.keys, cache.values, cache.key_scales, x))

    s = torch.zeros(2, 3, 8)
    return [
        ("write8", lambda x: write8(cache, x, k, None, positions), k),
        ("write8", lambda x: write8(cache, k, x, None, positions), k),
        ("write8", lambda x: scaled(x, lambda c: write8(c, k, k, None, positions)), s),
        ("write_rows8", rows, torch.zeros(2, 6, 64)),
        ("write_rows8", lambda x: rows(torch.zeros(2, 6, 64), weight=x), weight),
        ("write_rows8", lambda x: rows(torch.zeros(2, 6, 64), table=x), table),
        ("read8", lambda x: scaled(x, read8), s),
        ("decode_append8", append, torch.zeros(2, 6, 64)),
        ("decode_append8", lambda x: append(torch.zeros(2, 6, 64), k=x), k),
        ("decode_append8", lambda x: append(torch.zeros(2, 6, 64), table=x), table),
        ("decode8", lambda x: decode8(x, cache), torch.zeros(2, 6, 64)),
        ("decode8", lambda x: scaled(x, lambda c: decode8(torch.zeros(2, 6, 64), c)), s),
    ]


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("index", range(12))
def test_unseen(index):
    """Forward mode, function transforms and tracers do not see what a kernel computes."""
    from torch.fx.experimental.proxy_tensor import make_fx

    name, call, x = calls()[index]
    with pytest.raises(RuntimeError, match="GPU only"):
        call(x)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} has no gradient"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
    with torch.no_grad():
        # (a fresh tensor: a cache's constructor asks for its address)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced|data.*pointer|storage"):
            make_fx(lambda x: call(x))(x)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_linear8_unseen():
    from torch.fx.experimental.proxy_tensor import make_fx

    from asrback_amd.linear8 import Linear8, gated8, linear8, pack8

    weight = pack8(torch.zeros(8, 64, dtype=torch.int8), torch.ones(8))
    x = torch.zeros(3, 64)
    for name, call, t in (("linear8", lambda t: linear8(t, weight), x), ("gated8", lambda t: gated8(t, weight), x),
                          ("linear8", Linear8(weight), x), ("gated8", Linear8(weight).gated, x),
                          ("linear8", lambda t: linear8(x, weight, t), torch.zeros(8))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call(t)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match=f"{name} has no gradient"):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match=f"{name} takes no part"):
            torch.func.jvp(call, (t,), (t,))
        with torch.no_grad():
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                torch.jit.trace(lambda t: call(t), (t,))
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                make_fx(lambda t: call(t))(t)


def test_scales_that_require_a_gradient():
    """No op drops the gradient of a cache's scales, or writes over such a leaf."""
    from asrback_amd.cache8 import Cache8, decode8, decode_append8, read8, write8, write_rows8

    k, q, positions = torch.zeros(2, 3, 64), torch.zeros(2, 6, 64), torch.zeros(2, dtype=torch.int64)
    norm, table = torch.zeros(64), torch.zeros(2, 64)
    more = {"q_norm": norm, "k_norm": norm, "q_eps": 1e-6, "k_eps": 1e-6, "cos": table, "sin": table}
    for field in ("key_scales", "value_scales"):
        cache = Cache8.allocate(2, 8, 3, 64)
        getattr(cache, field).requires_grad_()
        for name, call in (("write8", lambda: write8(cache, k, k, None, positions)), ("read8", lambda: read8(cache)),
                           ("write_rows8", lambda: write_rows8(cache, q, k, k, None, positions, **more)),
                           ("decode8", lambda: decode8(q, cache)),
                           ("decode_append8", lambda: decode_append8(q, k, k, cache, positions, **more))):
            with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
                call()
    # One that takes part in a graph without being a leaf.
    cache = Cache8(cache.keys, cache.values, torch.zeros(2, 3, 8, requires_grad=True) * 2, torch.zeros(2, 3, 8))
    with pytest.raises(RuntimeError, match="decode8 has no gradient"):
        decode8(q, cache)


def test_caches_that_hold_elements_twice():
    """Read, but not written: heads, rows and positions that share places."""
    from asrback_amd.cache8 import Cache8, decode8, decode_append8, read8, write8, write_rows8

    k, q, positions = torch.zeros(2, 3, 64), torch.zeros(2, 6, 64), torch.zeros(2, dtype=torch.int64)
    norm, table = torch.zeros(64), torch.zeros(2, 64)
    more = {"q_norm": norm, "k_norm": norm, "q_eps": 1e-6, "k_eps": 1e-6, "cos": table, "sin": table}
    whole = Cache8.allocate(2, 8, 3, 64).tensors
    for i, shared in ((0, torch.zeros(1, 8, 3, 64, dtype=torch.int8).expand(2, 8, 3, 64)),
                      (1, torch.zeros(2, 8, 1, 64, dtype=torch.int8).expand(2, 8, 3, 64)),
                      (1, torch.zeros(2 * 8 * 3 * 64, dtype=torch.int8).as_strided((2, 8, 3, 64), (1536, 16, 512, 1))),
                      (2, torch.zeros(2, 1, 8).expand(2, 3, 8)), (3, torch.zeros(2, 3, 1).expand(2, 3, 1))):
        if i == 3:  # one position: nothing is held twice
            cache = Cache8(*(t[:, :1] for t in whole[:2]), whole[2][..., :1], shared)
        else:
            cache = Cache8(*(shared if j == i else t for j, t in enumerate(whole)))
        word, kind = ("GPU only", RuntimeError) if i == 3 else ("more than once", ValueError)
        for call in (lambda: write8(cache, k, k, None, positions), lambda: write_rows8(cache, q, k, k, None, positions, **more),
                     lambda: decode_append8(q, k, k, cache, positions, **more)):
            with pytest.raises(kind, match=word):
                call()
        for call in (lambda: read8(cache), lambda: decode8(q, cache)):
            with pytest.raises(RuntimeError, match="GPU only"):
                call()
    # Keys that are the values, too, or reach into them; parts of the same pages are apart.
    flat, pool = torch.zeros(whole[0].numel() + 64, dtype=torch.int8), torch.zeros(2, 2, 8, 3, 64, dtype=torch.int8)
    scales = torch.zeros(2, 2, 3, 8)
    for tensors, taken in (((whole[0], whole[0], *whole[2:]), False), ((*whole[:2], whole[2], whole[2]), False),
                           ((flat[:-64].view(2, 8, 3, 64), flat[64:].view(2, 8, 3, 64), *whole[2:]), False),
                           ((pool[:, 0], pool[:, 1], scales[:, 0], scales[:, 1]), True)):
        with pytest.raises(RuntimeError if taken else ValueError, match="GPU only" if taken else "more than once"):
            write8(Cache8(*tensors), k, k, None, positions)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_refusals():
    from asrback_amd.cache8 import Cache8, decode8, decode8_workspace_size, decode_append8, read8, write8, write_rows8

    cache = Cache8.allocate(2, 8, 3, 64)
    k, positions = torch.zeros(2, 3, 64), torch.zeros(2, dtype=torch.int64)
    for args, kind, match in (
        ((k[0], k[0], None, positions), ValueError, "k and v"),
        ((k[:, :2], k[:, :2], None, positions), ValueError, "k and v"),
        ((k, k[:1], None, positions), ValueError, "k and v"),
        ((k, k, None, positions[:1]), ValueError, "positions"),
        ((k, k, None, positions.int()), ValueError, "positions"),
        ((k, k, positions.int(), positions), ValueError, "rows"),
        ((k, k, None, None), TypeError, "positions"),
        ((k.half(), k.half(), None, positions), TypeError, "float32 and bfloat16"),
        ((k, k.bfloat16(), None, positions), TypeError, "mixed"),
    ):
        with pytest.raises(kind, match=match):
            write8(cache, *args)
    q, norm, table = torch.zeros(2, 6, 64), torch.zeros(64), torch.zeros(2, 64)
    good = {"q_norm": norm, "k_norm": norm, "q_eps": 1e-6, "k_eps": 1e-6, "cos": table, "sin": table}
    for query, change, match in ((q, {"k_norm": norm[:32]}, "k_norm"), (q, {"cos": table[:1]}, "cos"),
                                 (q, {"sin": torch.zeros(2, 32)}, "sin"), (torch.zeros(3, 6, 64), {}, "cos|q must"),
                                 (torch.zeros(2, 6, 128), {}, "q_norm|q must")):
        with pytest.raises(ValueError, match=match):
            write_rows8(cache, query, k, k, None, positions, **(good | change))
    for args, change, match in (((q, k[:1], k, positions), {}, "k must"), ((q, k, k[:, :1], positions), {}, "v must"),
                                ((q, k, k, positions[:1]), {}, "positions"), ((q, k, k, positions.int()), {}, "positions"),
                                ((q, k, k, positions), {"k_norm": norm[:32]}, "k_norm"),
                                ((q, k, k, positions), {"cos": table[:1]}, "cos"), ((q[0], k, k, positions), {}, "must"),
                                ((q[:, :4], k, k, positions), {}, "multiple"), ((q, k, k, positions), {"window": 0}, "window")):
        with pytest.raises(ValueError, match=match):
            decode_append8(args[0], args[1], args[2], cache, args[3], **(good | change))
    with pytest.raises(TypeError, match="positions"):
        decode_append8(q, k, k, cache, None, **good)
    with pytest.raises(TypeError, match="mixed"):
        decode_append8(q, k.bfloat16(), k, cache, positions, **good)
    buffer = torch.zeros(2, 12, 64)
    with pytest.raises(ValueError, match="shares memory"):
        decode_append8(buffer[:, :6], buffer[:, 6:9], buffer[:, 9:], cache, positions, out=buffer[:, 5:11], **good)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        read8(cache, dtype=torch.float16)
    for bad in (positions[:1], positions.float()):
        with pytest.raises((ValueError, TypeError)):
            read8(cache, lengths=bad)
        with pytest.raises((ValueError, TypeError)):
            decode8(q, cache, lengths=bad)
    for query, more, kind, match in (
        (q[0], {}, ValueError, "q must"), (torch.zeros(2, 6, 128), {}, ValueError, "q must"),
        (torch.zeros(2, 4, 64), {}, ValueError, "multiple"), (torch.zeros(2, 0, 64), {}, ValueError, "multiple"),
        (q, {"window": 0}, ValueError, "window"), (q.half(), {}, TypeError, "float32 and bfloat16"),
        (q, {"out": q[:1]}, ValueError, "out must"), (q, {"out": q.bfloat16()}, ValueError, "out must"),
        (q, {"out": torch.zeros(2, 6, 128)[..., ::2]}, ValueError, "out must"),
    ):
        with pytest.raises(kind, match=match):
            decode8(query, cache, **more)
    arena = torch.zeros(2, 12, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        decode8(arena[:, :6], cache, out=arena[:, 6:])
    with pytest.raises(RuntimeError, match="GPU only"):
        decode8(arena[:, :6], cache, out=arena[:, :6])
    scales = torch.zeros(2, 3, 256)
    other = Cache8(torch.zeros(2, 256, 3, 64, dtype=torch.int8), torch.zeros(2, 256, 3, 64, dtype=torch.int8), scales, scales)
    for out in (arena[:, 3:9], scales.view(-1)[:768].view(2, 6, 64)):
        with pytest.raises(ValueError, match="shares memory"):
            decode8(arena[:, :6], other, out=out)
    assert decode8_workspace_size(1, 16, 8, 128, 4096) > 0
    assert decode8_workspace_size(64, 16, 8, 128, 4096) == 0 and decode8_workspace_size(0, 16, 8, 128, 4096) == 0
    for batch in range(1, 16):
        assert decode8_workspace_size(batch, 16, 8, 128, 4096) <= decode8_workspace_size(16, 16, 8, 128, 4096)
    for sizes in ((1, 16, 8, 96, 64), (1, 15, 8, 64, 64), (-1, 16, 8, 64, 64), (1, 16, 8, 64, -1), (65536, 16, 8, 64, 64)):
        with pytest.raises(ValueError):
            decode8_workspace_size(*sizes)
    with pytest.raises(TypeError):
        decode8_workspace_size(1, 16, 8, 64, 64, torch.float16)


def test_what_the_library_refuses():
    from asrback_amd import _lib

    lib = _lib.load()

    def cache(p):
        p.batch, p.heads_kv, p.head_dim, p.max_len, p.dtype = 2, 2, 64, 32, _lib.BF16
        p.cache_k = p.cache_v = p.k_scales = p.v_scales = 4096
        for name in ("ck_batch", "ck_token", "ck_head", "cv_batch", "cv_token", "cv_head"):
            setattr(p, f"{name}_stride", 4096)
        return p

    def write():
        p = cache(_lib.Write8Params())
        p.k = p.v = p.positions = 4096
        p.tokens = 1
        return p

    def read():
        p = cache(_lib.Read8Params())
        p.k_out = p.v_out = 4096
        return p

    def decode():
        p = cache(_lib.Decode8Params())
        p.q = p.out = 4096
        p.heads_q, p.scale = 4, 0.125
        return p

    def append():
        p = cache(_lib.Append8Params())
        p.q = p.out = p.k = p.v = p.positions = p.q_norm = p.k_norm = p.cos = p.sin = 4096
        p.heads_q, p.scale = 4, 0.125
        return p

    def run(p):
        if isinstance(p, _lib.Append8Params):
            return lib.asrlayer_append8(bytes(p), 0, 0, None)
        if isinstance(p, _lib.Write8Params):
            return lib.asrlayer_write8(bytes(p), None)
        if isinstance(p, _lib.Read8Params):
            return lib.asrlayer_read8(bytes(p), None)
        return lib.asrlayer_decode8(bytes(p), 0, 0, None)

    shared = [
        ({"dtype": 5}, _lib.ERR_INVALID, b"dtype"), ({"head_dim": 32}, _lib.ERR_UNSUPPORTED, b"head_dim"),
        ({"heads_kv": 0}, _lib.ERR_INVALID, b"heads_kv"), ({"batch": -1}, _lib.ERR_INVALID, b"batch"),
        ({"batch": 65536}, _lib.ERR_UNSUPPORTED, b"65535"), ({"max_len": (1 << 30) + 1}, _lib.ERR_UNSUPPORTED, b"2^30"),
        ({"cache_v": 0}, _lib.ERR_INVALID, b"non-NULL"), ({"ck_head_stride": 8}, _lib.ERR_INVALID, b"16"),
        ({"cache_k": 4104}, _lib.ERR_INVALID, b"16"), ({"cv_token_stride": 1 << 26}, _lib.ERR_UNSUPPORTED, b"64 MiB"),
        ({"block_table": 4096, "page_size": 24, "num_pages": 1, "bt_stride": 2}, _lib.ERR_UNSUPPORTED, b"power of two"),
        ({"block_table": 4096, "page_size": 8, "num_pages": 1, "bt_stride": 8}, _lib.ERR_UNSUPPORTED, b"power of two"),
        ({"block_table": 4096, "page_size": 16, "num_pages": 1, "bt_stride": 1}, _lib.ERR_INVALID, b"reach"),
        ({"block_table": 4096, "page_size": 16, "num_pages": -1, "bt_stride": 2}, _lib.ERR_INVALID, b"num_pages"),
    ]
    for make, own in (
        (write, [({"tokens": -1}, _lib.ERR_INVALID, b"tokens"), ({"tokens": 1 << 24}, _lib.ERR_UNSUPPORTED, b"2^23"),
                 ({"tokens": 1 << 23, "heads_q": 4096}, _lib.ERR_UNSUPPORTED, b"2^32"),
                 ({"positions": 0}, _lib.ERR_INVALID, b"positions"), ({"heads_q": 1}, _lib.ERR_INVALID, b"queries"),
                 ({"k_norm": 4096}, _lib.ERR_INVALID, b"pairs"), ({"sin": 4096}, _lib.ERR_INVALID, b"pairs"),
                 ({"k_token_stride": 4}, _lib.ERR_INVALID, b"16-byte"), ({"v": 4100}, _lib.ERR_INVALID, b"16-byte")]),
        (read, [({"v_out": 0}, _lib.ERR_INVALID, b"non-NULL"), ({"k_out": 4104}, _lib.ERR_INVALID, b"aligned"),
                ({"max_len": 1 << 30, "heads_kv": 4}, _lib.ERR_UNSUPPORTED, b"2^33")]),
        (append, [({"heads_q": 3}, _lib.ERR_INVALID, b"multiple"), ({"positions": 0}, _lib.ERR_INVALID, b"non-NULL"),
                  ({"cos": 0}, _lib.ERR_INVALID, b"non-NULL"), ({"k": 4100}, _lib.ERR_INVALID, b"16-byte"),
                  ({"v_head_stride": 4}, _lib.ERR_INVALID, b"16-byte"), ({"rope_stride": 4}, _lib.ERR_INVALID, b"16-byte"),
                  ({"max_len": 4096}, _lib.ERR_WORKSPACE, b"workspace")]),
        (decode, [({"heads_q": 3}, _lib.ERR_INVALID, b"multiple"), ({"heads_q": 8192}, _lib.ERR_UNSUPPORTED, b"4096"),
                  ({"window": -1}, _lib.ERR_INVALID, b"window"), ({"scale": float("nan")}, _lib.ERR_INVALID, b"scale"),
                  ({"q": 0}, _lib.ERR_INVALID, b"non-NULL"), ({"q_head_stride": 4}, _lib.ERR_INVALID, b"16-byte"),
                  ({"max_len": 4096}, _lib.ERR_WORKSPACE, b"workspace")]),
    ):
        for change, code, word in shared + own:
            p = make()
            for name, value in change.items():
                setattr(p, name, value)
            assert run(p) == code, (change, lib.asrattn_last_error())
            assert word in lib.asrattn_last_error(), (change, lib.asrattn_last_error())
    p = write()
    p.tokens = 0
    assert run(p) == _lib.OK
    p = decode()
    p.batch = 0
    assert run(p) == _lib.OK
    p = decode()
    p.max_len = 4096
    need = lib.asrlayer_decode8_workspace_size(bytes(p))
    assert 0 < need < 1 << 24
    assert lib.asrlayer_decode8(bytes(p), 4096 + 64, need, None) == _lib.ERR_WORKSPACE
    for f in (lambda: lib.asrlayer_write8(None, None), lambda: lib.asrlayer_read8(None, None),
              lambda: lib.asrlayer_decode8(None, 0, 0, None), lambda: lib.asrlayer_append8(None, 0, 0, None)):
        assert f() == _lib.ERR_INVALID
    assert lib.asrlayer_decode8_workspace_size(None) == (1 << 64) - 1


def test_decoder_caches():
    """Slab and pages, as the decoder narrows them and hands pages out."""
    from asrback_amd.qwen3_asr import CACHE_LENGTH, KVCache8, Layer8, PagedKVCache8, RowPages

    slab = KVCache8.allocate(CONFIG, 4, 96, "cpu")
    part = slab.narrow(3, 32)
    assert len(part.keys) == 2 and isinstance(part.keys[0], Layer8) and part.keys[1] is part.values[1]
    assert part.keys[0].shape == (3, 32, 2, 64) and part.keys[0].pages is None
    part.layers[1].value_scales[2, 1, 31] = 7
    assert slab.layers[1].value_scales[2, 1, 31] == 7
    assert slab.narrow(3, 32).layers[0].keys.data_ptr() == slab.layers[0].keys.data_ptr()
    paged = PagedKVCache8.allocate(CONFIG, 4, 6, 64, "cpu")
    assert isinstance(paged, RowPages) and "PagedKVCache8" in repr(paged) and paged.layers[0].keys.shape == (6, 64, 2, 64)
    pages = paged.assign(1, 65)
    assert len(pages) == 2 and paged.block_table[1, :3].tolist() == [*pages, -1]
    part = paged.narrow(2, 100)
    assert part.keys[0].shape == (2, CACHE_LENGTH, 2, 64) and part.keys[0].pages.block_table.shape[0] == 2
    with pytest.raises(RuntimeError, match="exhausted"):
        part.assign(0, 5 * 64)
    paged.release(1, pages)
    assert sorted(paged.free_pages) == list(range(6)) and (paged.block_table == -1).all()
    with pytest.raises(ValueError, match="divide"):
        PagedKVCache8.allocate(CONFIG, 4, 6, 48, "cpu")
    with pytest.raises(ValueError, match="head dims"):
        KVCache8.allocate(CONFIG | {"head_dim": 80}, 4, 96, "cpu")
