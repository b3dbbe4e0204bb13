"""CPU: what the drafted-tree ops refuse, and the layout of their parameter
structs."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from conftest import ROOT


def tensors(batch=2, tokens=3, heads=4, kv=2, d=64, length=8, dtype=torch.float32):
    return dict(q=torch.zeros(batch, tokens, heads, d, dtype=dtype), k=torch.zeros(batch, length, kv, d, dtype=dtype),
                v=torch.zeros(batch, length, kv, d, dtype=dtype), k_draft=torch.zeros(batch, tokens, kv, d, dtype=dtype),
                v_draft=torch.zeros(batch, tokens, kv, d, dtype=dtype),
                masks=torch.ones(batch, tokens, dtype=torch.int64))


def test_tree_attention_refuses():
    from asrback_amd.drafts import tree_attention

    good = tensors()
    with pytest.raises(RuntimeError, match="GPU only"):
        tree_attention(**good)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        tree_attention(**tensors(dtype=torch.float16))
    for name, bad, kind, match in (
        ("q", torch.zeros(2, 4, 64), ValueError, "4 dimensions"),
        ("q", torch.zeros(2, 3, 3, 64), ValueError, "multiple"),
        ("v", torch.zeros(2, 7, 2, 64), ValueError, "share one shape"),
        ("k", torch.zeros(2, 8, 2, 32), ValueError, "share one shape"),
        ("k_draft", torch.zeros(2, 2, 2, 64), ValueError, "k_draft"),
        ("v_draft", torch.zeros(2, 3, 1, 64), ValueError, "v_draft"),
        ("masks", torch.ones(2, 3, dtype=torch.int32), TypeError, "int64"),
        ("masks", torch.ones(2, 4, dtype=torch.int64), ValueError, "masks"),
        ("masks", torch.ones(1, 3, dtype=torch.int64), ValueError, "masks"),
    ):
        with pytest.raises(kind, match=match):
            tree_attention(**{**good, name: bad})
    with pytest.raises(ValueError, match="rows"):
        tree_attention(**{**good, "k": torch.zeros(3, 8, 2, 64), "v": torch.zeros(3, 8, 2, 64)})
    with pytest.raises(ValueError, match="1 to 64"):
        tree_attention(**tensors(tokens=65))
    with pytest.raises(ValueError, match="1 to 64"):
        tree_attention(**tensors(tokens=0))
    with pytest.raises(TypeError, match="lengths"):
        tree_attention(**good, lengths=torch.zeros(2))
    with pytest.raises(ValueError, match="lengths"):
        tree_attention(**good, lengths=torch.zeros(3, dtype=torch.int64))


def test_masks_accept_and_commit_refuse():
    from asrback_amd.drafts import accept_drafts, commit_drafts, tree_masks

    ints = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU only"):
        tree_masks(ints)
    with pytest.raises(TypeError, match="int64"):
        tree_masks(ints.int())
    with pytest.raises(ValueError, match="1 to 64"):
        tree_masks(torch.zeros(2, 65, dtype=torch.int64))
    with pytest.raises(ValueError, match="parents"):
        tree_masks(torch.zeros(2, 3, 4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU only"):
        accept_drafts(ints, ints, ints)
    with pytest.raises(ValueError, match="choices"):
        accept_drafts(ints, ints, ints[:1])
    with pytest.raises(ValueError, match="parents"):
        accept_drafts(ints, ints[:1], ints)
    with pytest.raises(TypeError, match="limit"):
        accept_drafts(ints, ints[0], ints, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="tokens"):
        accept_drafts(ints[0], ints[0], ints[0])

    cache, draft = torch.zeros(4, 2, 16, 2, 64), torch.zeros(4, 2, 3, 2, 64)
    count = torch.zeros(2, dtype=torch.int64)
    good = dict(keys=cache, values=cache.clone(), k_draft=draft, v_draft=draft, path=ints, count=count, lengths=count)
    with pytest.raises(RuntimeError, match="GPU only"):
        commit_drafts(**good)
    for name, bad, kind, match in (
        ("keys", cache[0], ValueError, "5 dimensions"),
        ("values", torch.zeros(4, 2, 15, 2, 64), ValueError, "share one shape"),
        ("v_draft", torch.zeros(4, 2, 4, 2, 64), ValueError, "differ"),
        ("path", ints[:, :2], ValueError, "path"),
        ("count", count.int(), TypeError, "count"),
        ("lengths", None, TypeError, "lengths"),
        ("lengths", torch.zeros(2), TypeError, "lengths"),
    ):
        with pytest.raises(kind, match=match):
            commit_drafts(**{**good, name: bad})
    with pytest.raises(ValueError, match="layers"):
        commit_drafts(**{**good, "keys": cache[:3], "values": cache[:3].clone()})


@pytest.fixture(scope="module")
def lib():
    from asrback_amd import _lib

    if not _lib.LIBRARY.is_file():
        from asrback_amd import build

        build.build()
    return _lib.load()


def test_workspace_size(lib):
    from asrback_amd.drafts import tree_workspace_size

    assert tree_workspace_size(64, 8, 16, 8, 128, 1024) == 0  # 512 units fill the GPU unsplit
    assert tree_workspace_size(0, 48, 16, 8, 128, 4096) >= 0
    one = tree_workspace_size(1, 8, 16, 8, 128, 4096)
    assert one >= 256 * 16 * 128 * 4 and one % 256 == 0
    for bad in (dict(head_dim=96), dict(tokens=65), dict(tokens=0), dict(heads_q=15)):
        sizes = dict(batch=1, tokens=8, heads_q=16, heads_kv=8, head_dim=128, max_len=64) | bad
        with pytest.raises(ValueError):
            tree_workspace_size(**sizes)
    with pytest.raises(TypeError):
        tree_workspace_size(1, 8, 16, 8, 128, 64, torch.float16)


def test_library_refuses(lib):
    """Checks before any device call (stand-in pointers, never dereferenced)."""
    from asrback_amd import _lib

    def tree(**more):
        p = _lib.TreeParams()
        p.batch, p.tokens, p.heads_q, p.heads_kv, p.head_dim, p.max_len_k = 1, 8, 4, 2, 128, 4096
        p.dtype, p.scale = _lib.BF16, 0.1
        for name in ("q", "k", "v", "k_draft", "v_draft", "out", "masks"):
            setattr(p, name, 4096)
        p.k_token_stride = p.v_token_stride = p.kd_token_stride = p.vd_token_stride = 256
        for name, value in more.items():
            setattr(p, name, value)
        return lib.asrlayer_tree(ctypes.byref(p), None, 0, None)

    assert tree() == _lib.ERR_WORKSPACE
    assert tree(batch=0) == _lib.OK
    assert tree(scale=float("nan")) == tree(heads_q=3) == tree(dtype=7) == tree(max_len_k=-1) == _lib.ERR_INVALID
    assert tree(head_dim=512) == tree(tokens=65) == tree(tokens=0) == tree(batch=70000) == _lib.ERR_UNSUPPORTED
    assert tree(masks=None) == tree(q=4100) == tree(k_token_stride=4) == _lib.ERR_INVALID
    assert tree(k_token_stride=1 << 26) == tree(vd_token_stride=-8) == _lib.ERR_UNSUPPORTED
    assert tree(batch=65535, heads_q=4096, heads_kv=64, tokens=64) == _lib.ERR_UNSUPPORTED  # 2^29 workgroups
    paged = dict(block_table=4096, bt_stride=64, page_size=64, num_pages=3)
    assert tree(**paged) == _lib.ERR_WORKSPACE
    assert tree(**paged | {"page_size": 8}) == tree(**paged | {"page_size": 48}) == _lib.ERR_UNSUPPORTED
    assert tree(**paged | {"bt_stride": 63}) == tree(**paged | {"k_page_stride": 4}) == _lib.ERR_INVALID
    assert lib.asrlayer_tree(None, None, 0, None) == lib.asrlayer_commit(None, None) == _lib.ERR_INVALID
    assert lib.asrlayer_tree_masks(None, 0, 1, 8, None, None, None) == _lib.ERR_INVALID
    assert lib.asrlayer_tree_masks(4096, 0, (1 << 25) + 1, 8, 4096, 4096, None) == _lib.ERR_INVALID
    assert lib.asrlayer_accept(4096, 4096, 0, 4096, None, (1 << 25) + 1, 8, 4096, 4096, 4096, None) == _lib.ERR_INVALID
    assert lib.asrlayer_tree_masks(4096, 0, 1, 65, 4096, 4096, None) == _lib.ERR_UNSUPPORTED
    assert lib.asrlayer_accept(4096, 4096, 0, 4096, None, -1, 8, 4096, 4096, 4096, None) == _lib.ERR_INVALID
    assert lib.asrlayer_accept(4096, 4096, 0, 4096, None, 0, 8, 4096, 4096, 4096, None) == _lib.OK
    c = _lib.CommitParams()
    c.layers, c.batch, c.tokens, c.heads_kv, c.head_dim, c.max_len_k, c.dtype = 2, 1, 8, 2, 64, 16, _lib.BF16
    assert lib.asrlayer_commit(ctypes.byref(c), None) == _lib.ERR_INVALID
    c.head_dim = 65
    assert lib.asrlayer_commit(ctypes.byref(c), None) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("name,struct", [("TreeParams", "asrlayer_tree_params"), ("CommitParams", "asrlayer_commit_params"),
                                         ("Linear4Params", "asrlayer_linear4_params")])
def test_structs_match_the_header(name, struct, tmp_path):
    from asrback_amd import _lib

    cls = getattr(_lib, name)
    lines = [f'printf("%zu\\n", sizeof({struct}));']
    lines += [f'printf("%zu\\n", offsetof({struct}, {f}));' for f, _ in cls._fields_]
    source = tmp_path / "layout.cpp"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "layers.hpp"\nint main() {\n'
                      + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["g++", f"-I{ROOT / 'include'}", f"-I{ROOT / 'asrback_amd' / 'csrc'}", str(source), "-o",
                    str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_)]


def test_decoder_workspace_holds_every_pass(lib):
    """Passes over fewer rows than a bucket's split their choice further."""
    from types import SimpleNamespace

    from asrback_amd.attention import choice_workspace_size, decode_workspace_size
    from asrback_amd.drafts import tree_workspace_size
    from asrback_amd.qwen3_asr import CACHE_LENGTH, TextGreedyDecoder

    for heads in (256, 8):
        decoder = SimpleNamespace(
            config={"num_attention_heads": heads, "num_key_value_heads": heads, "head_dim": 64}, buckets=[1, 2, 4, 8],
            lm_head=SimpleNamespace(weight=torch.empty(151936, 1)), kv_buckets=[CACHE_LENGTH], dtype=torch.float32,
            draft_tokens=16, max_batch_size=8)
        held = TextGreedyDecoder._workspace_bytes(decoder)
        for rows in range(1, 9):
            assert choice_workspace_size(rows * 16, 151936) <= held
            assert tree_workspace_size(rows, 16, heads, heads, 64, CACHE_LENGTH, torch.float32) <= held
        assert all(decode_workspace_size(b, heads, heads, 64, CACHE_LENGTH, torch.float32) <= held for b in (1, 2, 4, 8))
