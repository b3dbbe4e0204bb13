"""Drafted tokens on the HIP kernels of ``libasrattn.so``: verifying a tree of
them in one pass of a decoder and keeping what the model agrees with.

A drafted tree holds up to :data:`MAX_TOKENS` tokens a row.  Token 0 is the
row's newest token, the one a plain step would decode next (its key and value
are not in the cache yet); every other token names its parent, an earlier
token of the tree.  A pass over all of them costs little more than a plain
step, which is bound by reading the weights and the cache, and yields as many
tokens as the longest branch the model's own choices follow:

* :func:`tree_masks` turns parents into ancestor bit masks (once per tree);
* :func:`tree_attention` attends every drafted token over the cache, which all
  of them see, and its own ancestors, whose keys and values lie in draft
  buffers beside the cache;
* :func:`accept_drafts` walks each tree along the greedy choices;
* :func:`commit_drafts` writes the accepted tokens' keys and values of every
  layer from the draft buffers into the cache.

As in :mod:`asrback_amd.attention`, calls launch on the current HIP stream,
never synchronize, and can be captured into a graph; nothing here has a
gradient, and calls that would need one are refused.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch import Tensor

from . import _lib
from .attention import (
    _DTYPES, PageTable, _aligned, _check_device, _dtype_code, _paged, _ptr, _split_workspace, _stream,
)

# Tokens of a drafted tree, one bit each of an ancestor mask.
MAX_TOKENS = 64

_increment_version = torch.autograd.graph.increment_version


def _no_gradient(what: str, *tensors: Tensor) -> None:
    if any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad() or on detached tensors")


def _int64(t: Tensor, name: str, shape: tuple[int, ...]) -> Tensor:
    if t.dtype != torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    return t.contiguous()


def _per_tree(t: Tensor, name: str, batch: int, tokens: int) -> tuple[Tensor, int]:
    """``(tokens,)`` or ``(batch, tokens)`` int64 rows and their batch stride."""
    if t.dtype != torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.shape not in ((tokens,), (batch, tokens)):
        raise ValueError(f"{name} must be ({tokens},) or ({batch}, {tokens}), got {tuple(t.shape)}")
    if tokens > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t, 0 if t.dim() == 1 else t.stride(0)


def _tokens(tokens: int) -> None:
    if not 1 <= tokens <= MAX_TOKENS:
        raise ValueError(f"a tree has 1 to {MAX_TOKENS} drafted tokens, got {tokens}")


def _cuda(device: torch.device, what: str) -> None:
    if device.type != "cuda":
        raise RuntimeError(f"{what} runs on the GPU only; got tensors on {device}")


def _lengths(lengths: Tensor | None, batch: int) -> Tensor | None:
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"lengths must be int32 or int64, got {lengths.dtype}")
    if lengths.shape != (batch,):
        raise ValueError(f"lengths must be ({batch},), got {tuple(lengths.shape)}")
    return lengths.contiguous()


def tree_masks(parents: Tensor) -> tuple[Tensor, Tensor]:
    """Ancestor masks of drafted trees and their tokens' depths
    (``asrlayer_tree_masks``), int64 of the shape of ``parents``: bit ``i`` of a
    token's mask is set where ``i`` is the token or one of its ancestors, its
    depth is how many ancestors it has (its position behind the cache).

    ``parents`` int64 ``(tokens,)`` or ``(batch, tokens)``: each token's parent,
    an earlier token, or -1 where only the cache precedes it (so does a value
    from the token on); below -1 the token is padding, and its mask and depth 0."""
    if parents.dtype != torch.int64:
        raise TypeError(f"parents must be int64, got {parents.dtype}")
    if parents.dim() not in (1, 2):
        raise ValueError(f"parents must be (tokens,) or (batch, tokens), got {tuple(parents.shape)}")
    tokens = parents.shape[-1]
    _tokens(tokens)
    batch = parents.shape[0] if parents.dim() == 2 else 1
    parents, stride = _per_tree(parents, "parents", batch, tokens)
    device = _check_device(parents)
    _cuda(device, "tree_masks")
    masks = torch.empty(parents.shape, dtype=torch.int64, device=device)
    depths = torch.empty_like(masks)
    lib = _lib.load()
    _lib.check(lib.asrlayer_tree_masks(parents.data_ptr(), stride, batch, tokens, masks.data_ptr(), depths.data_ptr(),
                                       _stream(device)), "asrlayer_tree_masks")
    return masks, depths


@functools.lru_cache(maxsize=256)
def _tree_workspace(batch: int, tokens: int, heads_q: int, heads_kv: int, head_dim: int, max_len: int,
                    dtype: int) -> int:
    """``asrlayer_tree_workspace_size`` of these sizes (-1 for ones it does not
    take)."""
    params = _lib.TreeParams()
    params.batch, params.tokens, params.heads_q, params.heads_kv = batch, tokens, heads_q, heads_kv
    params.head_dim, params.max_len_k, params.dtype, params.scale = head_dim, max_len, dtype, 1.0
    need = _lib.load().asrlayer_tree_workspace_size(ctypes.byref(params))
    return -1 if need == ctypes.c_size_t(-1).value else need


def tree_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    k_draft: Tensor,
    v_draft: Tensor,
    masks: Tensor,
    *,
    lengths: Tensor | None = None,
    scale: float | None = None,
    out: Tensor | None = None,
    workspace: Tensor | None = None,
    pages: PageTable | None = None,
) -> Tensor:
    """Attention of drafted trees over a cache (``asrlayer_tree``).

    ``q`` ``(batch, tokens, heads_q, head_dim)``; ``k``/``v`` ``(batch, length,
    heads_kv, head_dim)``, any strides with a unit last one (pass
    ``cache.transpose(1, 2)`` for a ``(batch, heads, length, head_dim)``
    cache), or with ``pages`` the pools ``(num_pages, page_size, heads_kv,
    head_dim)``; ``k_draft``/``v_draft`` ``(batch, tokens, heads_kv,
    head_dim)``, the drafted tokens' own.  Token ``t`` of row ``b`` attends the
    cache's keys ``0 .. lengths[b] - 1`` (int32 or int64, default: all of
    them; outside the cache they are clamped to it) and the drafted keys whose
    bits are set in ``masks[b, t]`` (int64 ``(batch, tokens)``, or ``(tokens,)``
    for one tree in every row; :func:`tree_masks`).  A token with mask 0 is
    padding: it attends nothing and gets zeros.

    float32 or bfloat16, head_dim 64, 128 or 256, any number of query heads
    per kv head, up to :data:`MAX_TOKENS` tokens.  ``workspace``: the split
    partials' memory (:func:`tree_workspace_size`,
    :func:`asrback_amd.attention.workspace`).  Returns ``(batch, tokens,
    heads_q, head_dim)``."""
    q_shape, k_shape, draft_shape = q.shape, k.shape, k_draft.shape
    if not len(q_shape) == len(k_shape) == len(draft_shape) == 4:
        raise ValueError(f"q, k and k_draft must have 4 dimensions, got shapes {tuple(q_shape)}, {tuple(k_shape)}, "
                         f"{tuple(draft_shape)}")
    batch, tokens, heads_q, head_dim = q_shape
    length, heads_kv = k_shape[1:3]
    if v.shape != k_shape or k_shape[3] != head_dim:
        raise ValueError(f"k and v must share one shape with q's head_dim {head_dim}; got {tuple(k_shape)}, "
                         f"{tuple(v.shape)}")
    if pages is None and k_shape[0] != batch:
        raise ValueError(f"q has {batch} rows, the cache {k_shape[0]}")
    if heads_kv == 0 or heads_q % heads_kv or heads_q == 0:
        raise ValueError(f"{heads_q} query heads are not a positive multiple of {heads_kv} kv heads")
    if draft_shape != (batch, tokens, heads_kv, head_dim) or v_draft.shape != draft_shape:
        raise ValueError(f"k_draft and v_draft must be ({batch}, {tokens}, {heads_kv}, {head_dim}), got "
                         f"{tuple(draft_shape)}, {tuple(v_draft.shape)}")
    _tokens(tokens)
    masks, masks_stride = _per_tree(masks, "masks", batch, tokens)
    lengths = _lengths(lengths, batch)
    dtype = _dtype_code(q, k, v, k_draft, v_draft)
    if torch.is_grad_enabled():
        _no_gradient("tree_attention", q, k, v, k_draft, v_draft)
    q, k, v, k_draft, v_draft = _aligned(q), _aligned(k), _aligned(v), _aligned(k_draft), _aligned(v_draft)
    if out is None:
        out = torch.empty(q_shape, dtype=q.dtype, device=q.device)
    elif out.shape != q_shape or out.dtype != q.dtype or out.stride(-1) != 1:
        raise ValueError("out must match q's shape and dtype, with a unit last stride")
    k_strides, v_strides = k.stride()[:3], v.stride()[:3]
    if pages is None:
        device = _check_device(q, k, v, k_draft, v_draft, masks, lengths, out)
        paged = (None, 0, 0, 0, 0, 0)
    else:
        device = _check_device(q, k, v, k_draft, v_draft, masks, lengths, out, pages.block_table)
        pk, length = _paged(pages, k, v, batch)
        paged = (pk.block_table, pk.bt_stride, pk.k_page_stride, pk.v_page_stride, pk.page_size, pk.num_pages)
        k_strides, v_strides = (0, *k_strides[1:]), (0, *v_strides[1:])
    params = _lib.TreeParams(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), k_draft.data_ptr(), v_draft.data_ptr(), out.data_ptr(),
        *q.stride()[:3], *k_strides, *v_strides, *k_draft.stride()[:3], *v_draft.stride()[:3], *out.stride()[:3],
        masks.data_ptr(), masks_stride, None if lengths is None else lengths.data_ptr(), *paged,
        lengths is not None and lengths.dtype == torch.int64, batch, tokens, heads_q, heads_kv, head_dim, length, dtype,
        1.0 / math.sqrt(head_dim) if scale is None else scale)
    need = _tree_workspace(batch, tokens, heads_q, heads_kv, head_dim, length, dtype)
    # Sizes that the library does not take: the call says why.
    workspace = _split_workspace(max(need, 0), workspace, device)
    size = 0 if workspace is None else workspace.numel()
    status = _lib.load().asrlayer_tree(ctypes.byref(params), _ptr(workspace), size, _stream(device))
    if status:
        _lib.check(status, "asrlayer_tree")
    return out


def tree_workspace_size(batch: int, tokens: int, heads_q: int, heads_kv: int, head_dim: int, max_len: int,
                        dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes of split partials a :func:`tree_attention` call of these sizes
    needs (``asrlayer_tree_workspace_size``; 0 when it runs unsplit): where it
    is not 0, enough for every smaller batch and fewer tokens over the same
    cache.  Raises for sizes the library does not take."""
    if dtype not in _DTYPES:
        raise TypeError(f"attention supports float32 and bfloat16, got {dtype}")
    sizes = (batch, tokens, heads_q, heads_kv, head_dim, max_len, _DTYPES[dtype])
    need = _tree_workspace(*sizes)
    if need < 0:
        _tree_workspace.__wrapped__(*sizes)  # leaves its message
        raise ValueError(_lib.load().asrattn_last_error().decode("utf-8", "replace"))
    return need


def accept_drafts(tokens: Tensor, parents: Tensor, choices: Tensor,
                  limit: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """The walk of the model's choices down drafted trees
    (``asrlayer_accept``).

    ``tokens`` int64 ``(batch, width)`` are the drafted tokens, ``choices``
    int64 ``(batch, width)`` the token the model puts after each of them
    (:func:`~asrback_amd.attention.greedy_choice` of its logits), ``parents``
    as for :func:`tree_masks`.  Token 0 is accepted; after each accepted token
    comes the first one behind it whose parent it is and that equals its
    choice.  Returns int64 ``path`` ``(batch, width)``, the accepted tokens'
    indices, ``emitted`` ``(batch, width)``, the choice after each of them (the
    tokens this pass generated), both -1 past the walk's end, and ``count``
    ``(batch,)``, its length.  ``limit`` int64 ``(batch,)`` caps it; rows with
    a limit below 1, or whose token 0 is padding, accept nothing."""
    if tokens.dim() != 2:
        raise ValueError(f"tokens must be (batch, width), got {tuple(tokens.shape)}")
    shape = tokens.shape
    batch, width = shape
    _tokens(width)
    tokens, choices = _int64(tokens, "tokens", shape), _int64(choices, "choices", shape)
    parents, stride = _per_tree(parents, "parents", batch, width)
    if limit is not None:
        limit = _int64(limit, "limit", (batch,))
    device = _check_device(tokens, parents, choices, limit)
    _cuda(device, "accept_drafts")
    path, emitted = torch.empty((2, batch, width), dtype=torch.int64, device=device).unbind()
    count = torch.empty(batch, dtype=torch.int64, device=device)
    status = _lib.load().asrlayer_accept(
        tokens.data_ptr(), parents.data_ptr(), stride, choices.data_ptr(), _ptr(limit), batch, width, path.data_ptr(),
        emitted.data_ptr(), count.data_ptr(), _stream(device))
    if status:
        _lib.check(status, "asrlayer_accept")
    return path, emitted, count


def commit_drafts(
    keys: Tensor,
    values: Tensor,
    k_draft: Tensor,
    v_draft: Tensor,
    path: Tensor,
    count: Tensor,
    lengths: Tensor,
    *,
    pages: PageTable | None = None,
) -> None:
    """Write accepted drafts into the cache, every layer in one launch
    (``asrlayer_commit``): position ``lengths[b] + i`` of row ``b`` gets the key
    and value of drafted token ``path[b, i]``, for ``i < count[b]``.

    ``keys``/``values`` ``(layers, batch, length, heads_kv, head_dim)``, or with
    ``pages`` pools ``(layers, num_pages, page_size, heads_kv, head_dim)``, are
    written in place (any strides of whole 16-byte vectors, the last one unit);
    ``k_draft``/``v_draft`` ``(layers, batch, tokens, heads_kv, head_dim)`` must
    not share memory with them.  ``path`` int64 ``(batch, tokens)`` and
    ``count`` int64 ``(batch,)`` come from :func:`accept_drafts`; ``lengths``
    int32 or int64 ``(batch,)`` are the rows' keys before the call.  Positions
    outside the cache or on no page are left alone, as are path entries outside
    the tree."""
    cache_shape, draft_shape = keys.shape, k_draft.shape
    if len(cache_shape) != 5 or len(draft_shape) != 5:
        raise ValueError(f"keys and k_draft must have 5 dimensions, got shapes {tuple(cache_shape)}, {tuple(draft_shape)}")
    layers, batch, tokens, heads_kv, head_dim = draft_shape
    if v_draft.shape != draft_shape:
        raise ValueError(f"k_draft and v_draft shapes differ: {tuple(draft_shape)}, {tuple(v_draft.shape)}")
    if values.shape != cache_shape or cache_shape[0] != layers or cache_shape[3:] != (heads_kv, head_dim):
        raise ValueError(f"keys and values must share one shape with {layers} layers of ({heads_kv}, {head_dim}); got "
                         f"{tuple(cache_shape)}, {tuple(values.shape)}")
    if pages is None and cache_shape[1] != batch:
        raise ValueError(f"the drafts have {batch} rows, the cache {cache_shape[1]}")
    _tokens(tokens)
    path = _int64(path, "path", (batch, tokens))
    count = _int64(count, "count", (batch,))
    if lengths is None:
        raise TypeError("lengths must be a tensor")
    lengths = _lengths(lengths, batch)
    dtype = _dtype_code(keys, values, k_draft, v_draft)
    if torch.is_grad_enabled():
        _no_gradient("commit_drafts", keys, values, k_draft, v_draft)
    if not torch.is_inference_mode_enabled() and (keys.is_inference() or values.is_inference()):
        raise RuntimeError("inplace update to inference tensors outside InferenceMode is not allowed")
    if (_aligned(keys) is not keys or _aligned(values) is not values) and keys.numel():
        raise ValueError("keys and values need a unit last stride and 16-byte aligned rows (they are written in place)")
    k_draft, v_draft = _aligned(k_draft), _aligned(v_draft)
    length = cache_shape[2]
    if pages is None:
        device = _check_device(keys, values, k_draft, v_draft, path, count, lengths)
        paged = (None, 0, 0, 0)
    else:
        device = _check_device(keys, values, k_draft, v_draft, path, count, lengths, pages.block_table)
        if not layers:
            return
        pk, length = _paged(pages, keys[0], values[0], batch)
        paged = (pk.block_table, pk.bt_stride, pk.page_size, pk.num_pages)
    params = _lib.CommitParams(
        k_draft.data_ptr(), v_draft.data_ptr(), keys.data_ptr(), values.data_ptr(), *k_draft.stride()[:4],
        *v_draft.stride()[:4], *keys.stride()[:4], *values.stride()[:4], path.data_ptr(), count.data_ptr(),
        lengths.data_ptr(), *paged, lengths.dtype == torch.int64, layers, batch, tokens, heads_kv, head_dim, length, dtype)
    status = _lib.load().asrlayer_commit(ctypes.byref(params), _stream(device))
    if status:
        _lib.check(status, "asrlayer_commit")
    _increment_version((keys, values))
