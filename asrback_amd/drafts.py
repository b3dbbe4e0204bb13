"""Drafted tokens on the HIP kernels of ``libasrattn.so``: verifying a tree of
them in one pass of a decoder and keeping what the model agrees with.

A drafted tree holds up to :data:`MAX_TOKENS` tokens a row.  Token 0 is the
row's newest token, the one a plain step would decode next (its key and value
are not in the cache yet); every other token names its parent, an earlier
token of the tree.  A pass over all of them reads the weights and the cache once, as
a plain step does, and yields as many tokens as the longest branch the model's own
choices follow (28 layers of 2048 in bf16, one row: 2.3 ms a step, 2.7 ms a pass
over 4 or 16 tokens; 8 rows: 2.5 ms, 2.9 and 3.2):

* :func:`tree_masks` turns parents into ancestor bit masks (once per tree);
* :func:`tree_attention` attends every drafted token over the cache, which all
  of them see, and its own ancestors, whose keys and values lie in draft
  buffers beside the cache;
* :func:`accept_drafts` walks each tree along the greedy choices;
* :func:`commit_drafts` writes the accepted tokens' keys and values of every
  layer from the draft buffers into the cache.

As in :mod:`asrback_amd.attention`, calls launch on the current HIP stream,
never synchronize, and can be captured into a graph; nothing here has a
gradient, and calls that would need one, in forward mode too, or that a tracer
records are refused.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch import Tensor

from . import _lib
from .attention import (
    _DTYPES, PageTable, _aligned, _check_device, _dtype_code, _paged, _ptr, _split_workspace,
)
from .layers import check_out, refuse_unseen

# Tokens of a drafted tree, one bit each of an ancestor mask.
MAX_TOKENS = 64

_increment_version = torch.autograd.graph.increment_version
# The current stream's handle on a device.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _operands(what: str, tensors: tuple[Tensor, ...], written: tuple[Tensor, ...] = ()) -> tuple:
    """What a call passes of tensors of four or five axes that must share one
    supported type and the current GPU: their pointers, their strides (but the last) in a row, the
    dtype's code, the device's index, and the tensors themselves, those whose rows
    cannot be read with 16-byte vectors copied (of ``written`` ones refused)."""
    first = tensors[0]
    dtype, index = first.dtype, first.get_device()
    same, gradient, bits, ends, pointers, strides = True, False, 0, 0, [], []
    for t in tensors:
        if t.dtype is not dtype or t.get_device() != index:
            same = False
        if t.requires_grad:
            gradient = True
        pointer = t.data_ptr()
        pointers.append(pointer)
        ends |= pointer
        stride = t.stride()
        # A vector is a power of two of elements: one test for all strides.
        if len(stride) == 4:
            a, b, c, last = stride
            strides += (a, b, c)
            bits |= a | b | c
        else:
            a, b, c, d, last = stride
            strides += (a, b, c, d)
            bits |= a | b | c | d
        if last != 1:
            ends |= 1
    if not same or index < 0 or dtype not in _DTYPES or index != torch.cuda.current_device():
        _dtype_code(*tensors)  # these say what is wrong
        _check_device(*tensors)
    if gradient and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad() or on detached tensors")
    if ends & 15 or bits & (7 if dtype is torch.bfloat16 else 3):
        aligned = tuple(_aligned(t) for t in tensors)
        for t, held in zip(tensors, aligned):
            if t is not held and t.numel() and any(t is w for w in written):
                raise ValueError("keys and values need a unit last stride and 16-byte aligned rows (they are written in "
                                 "place)")
        tensors = aligned
        pointers = [t.data_ptr() for t in tensors]
        strides = [stride for t in tensors for stride in t.stride()[:-1]]
    return pointers, strides, _DTYPES[dtype], index, tensors


def _plain_operands(q: Tensor, k: Tensor, v: Tensor, k_draft: Tensor, v_draft: Tensor) -> tuple | None:
    """:func:`_operands` of tensors of four axes that the kernel takes as they are, in
    two thirds of its time; None where one is not."""
    dtype, index = q.dtype, q.get_device()
    if not (k.dtype is dtype and v.dtype is dtype and k_draft.dtype is dtype and v_draft.dtype is dtype
            and k.get_device() == index and v.get_device() == index and k_draft.get_device() == index
            and v_draft.get_device() == index) or dtype not in _DTYPES or index < 0 or index != torch.cuda.current_device():
        return None
    if q.requires_grad or k.requires_grad or v.requires_grad or k_draft.requires_grad or v_draft.requires_grad:
        return None
    a0, a1, a2, a = q.stride()
    b0, b1, b2, b = k.stride()
    c0, c1, c2, c = v.stride()
    d0, d1, d2, d = k_draft.stride()
    e0, e1, e2, e = v_draft.stride()
    pointers = (q.data_ptr(), k.data_ptr(), v.data_ptr(), k_draft.data_ptr(), v_draft.data_ptr())
    ends = pointers[0] | pointers[1] | pointers[2] | pointers[3] | pointers[4]
    bits = a0 | a1 | a2 | b0 | b1 | b2 | c0 | c1 | c2 | d0 | d1 | d2 | e0 | e1 | e2
    if not a == b == c == d == e == 1 or ends & 15 or bits & (7 if dtype is torch.bfloat16 else 3):
        return None
    return (pointers, [a0, a1, a2, b0, b1, b2, c0, c1, c2, d0, d1, d2, e0, e1, e2], _DTYPES[dtype], index,
            (q, k, v, k_draft, v_draft))


def _plain_caches(k_draft: Tensor, v_draft: Tensor, keys: Tensor, values: Tensor) -> tuple | None:
    """:func:`_plain_operands` of four tensors of five axes."""
    dtype, index = k_draft.dtype, k_draft.get_device()
    if not (v_draft.dtype is dtype and keys.dtype is dtype and values.dtype is dtype and v_draft.get_device() == index
            and keys.get_device() == index and values.get_device() == index) or dtype not in _DTYPES or index < 0 \
            or index != torch.cuda.current_device():
        return None
    if k_draft.requires_grad or v_draft.requires_grad or keys.requires_grad or values.requires_grad:
        return None
    a0, a1, a2, a3, a = k_draft.stride()
    b0, b1, b2, b3, b = v_draft.stride()
    c0, c1, c2, c3, c = keys.stride()
    d0, d1, d2, d3, d = values.stride()
    pointers = (k_draft.data_ptr(), v_draft.data_ptr(), keys.data_ptr(), values.data_ptr())
    bits = a0 | a1 | a2 | a3 | b0 | b1 | b2 | b3 | c0 | c1 | c2 | c3 | d0 | d1 | d2 | d3
    if (not a == b == c == d == 1 or (pointers[0] | pointers[1] | pointers[2] | pointers[3]) & 15
            or bits & (7 if dtype is torch.bfloat16 else 3)):
        return None
    return (pointers, (a0, a1, a2, a3, b0, b1, b2, b3, c0, c1, c2, c3, d0, d1, d2, d3), _DTYPES[dtype], index,
            (k_draft, v_draft, keys, values))


def _int64(t: Tensor, name: str, shape: tuple[int, ...]) -> Tensor:
    if t.dtype is not torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _per_tree(t: Tensor, name: str, batch: int, tokens: int) -> tuple[Tensor, int]:
    """``(tokens,)`` or ``(batch, tokens)`` int64 rows and their batch stride."""
    if t.dtype is not torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    strides = t.stride()
    if t.shape == (batch, tokens):
        if strides[1] == 1 or tokens == 1:
            return t, strides[0]
        return t.contiguous(), tokens
    if t.shape != (tokens,):
        raise ValueError(f"{name} must be ({tokens},) or ({batch}, {tokens}), got {tuple(t.shape)}")
    return t if strides[0] == 1 or tokens == 1 else t.contiguous(), 0


def _tokens(tokens: int) -> None:
    if not 1 <= tokens <= MAX_TOKENS:
        raise ValueError(f"a tree has 1 to {MAX_TOKENS} drafted tokens, got {tokens}")


def _cuda(what: str, *tensors: Tensor | None) -> int:
    """The index of the current GPU, which must hold the tensors."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            _check_device(*tensors)
    if index < 0:
        raise RuntimeError(f"{what} runs on the GPU only; got tensors on {tensors[0].device}")
    if index != torch.cuda.current_device():
        _check_device(*tensors)
    return index


def _on(index: int, *tensors: Tensor | None) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"tensors on different devices: cuda:{index} and {t.device}")


def _lengths(lengths: Tensor | None, batch: int) -> Tensor | None:
    if lengths is None:
        return None
    if lengths.dtype is not torch.int64 and lengths.dtype is not torch.int32:
        raise TypeError(f"lengths must be int32 or int64, got {lengths.dtype}")
    if lengths.shape != (batch,):
        raise ValueError(f"lengths must be ({batch},), got {tuple(lengths.shape)}")
    return lengths if lengths.stride() == (1,) else lengths.contiguous()


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
    refuse_unseen("tree_masks", parents)
    index = _cuda("tree_masks", parents)
    masks = torch.empty_like(parents, memory_format=torch.contiguous_format)
    depths = torch.empty_like(masks)
    lib = _lib.load()
    _lib.check(lib.asrlayer_tree_masks(parents.data_ptr(), stride, batch, tokens, masks.data_ptr(), depths.data_ptr(),
                                       _raw_stream(index)), "asrlayer_tree_masks")
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
    per kv head, up to :data:`MAX_TOKENS` tokens.  ``out`` is written in place; it
    may be ``q`` itself and shares memory with no other input.  ``workspace``: the split
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
    refuse_unseen("tree_attention", q, k, v, k_draft, v_draft)
    given = out is not None
    if given:
        if out.shape != q_shape or out.dtype != q.dtype or out.stride(-1) != 1:
            raise ValueError("out must match q's shape and dtype, with a unit last stride")
        # A row's queries are read before any of its outputs is written.
        in_place = out.data_ptr() == q.data_ptr() and out.stride() == q.stride()
        check_out("tree_attention", out, None if in_place else q, k, v, k_draft, v_draft, masks, lengths)
    pointers, strides, dtype, index, held = (_plain_operands(q, k, v, k_draft, v_draft)
                                             or _operands("tree_attention", (q, k, v, k_draft, v_draft)))
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if pages is None:
        _on(index, masks, lengths, out)
        paged = (0, 0, 0, 0, 0, 0)
    else:
        _on(index, masks, lengths, out, pages.block_table)
        pk, length = _paged(pages, held[1], held[2], batch)
        paged = (pk.block_table, pk.bt_stride, pk.k_page_stride, pk.v_page_stride, pk.page_size, pk.num_pages)
        strides[3] = strides[6] = 0  # the pools' first axis is no row
    params = _lib.pack_tree(
        *pointers, out.data_ptr(), *strides, *out.stride()[:3], masks.data_ptr(), masks_stride,
        0 if lengths is None else lengths.data_ptr(), *paged, lengths is not None and lengths.dtype is torch.int64, batch,
        tokens, heads_q, heads_kv, head_dim, length, dtype, head_dim**-0.5 if scale is None else scale)
    need = _tree_workspace(batch, tokens, heads_q, heads_kv, head_dim, length, dtype)
    size = 0
    if need > 0:
        workspace = _split_workspace(need, workspace, out.device)
    if workspace is not None:
        size, workspace = workspace.numel(), workspace.data_ptr()
    # Sizes that the library does not take (need -1): the call says why.
    status = _lib.load().asrlayer_tree(params, workspace, size, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_tree")
    if given:
        _increment_version(out)
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
    refuse_unseen("accept_drafts", tokens, parents, choices, limit)
    index = tokens.get_device()
    if (tokens.dtype is choices.dtype is parents.dtype is torch.int64 and choices.shape == parents.shape == shape
            and tokens.is_contiguous() and choices.is_contiguous() and parents.is_contiguous()
            and index == choices.get_device() == parents.get_device() >= 0
            and (limit is None or (limit.dtype is torch.int64 and limit.shape == (batch,) and limit.is_contiguous()
                                   and limit.get_device() == index))
            and index == torch.cuda.current_device()):
        stride = width
    else:
        tokens, choices = _int64(tokens, "tokens", shape), _int64(choices, "choices", shape)
        parents, stride = _per_tree(parents, "parents", batch, width)
        if limit is not None:
            limit = _int64(limit, "limit", (batch,))
        index = _cuda("accept_drafts", tokens, parents, choices, limit)
    path, emitted = torch.empty_like(tokens), torch.empty_like(tokens)
    count = tokens.new_empty(batch) if limit is None else torch.empty_like(limit)
    status = _lib.load().asrlayer_accept(
        tokens.data_ptr(), parents.data_ptr(), stride, choices.data_ptr(), _ptr(limit), batch, width, path.data_ptr(),
        emitted.data_ptr(), count.data_ptr(), _raw_stream(index))
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
    refuse_unseen("commit_drafts", keys, values, k_draft, v_draft)
    pointers, strides, dtype, index, held = (
        _plain_caches(k_draft, v_draft, keys, values)
        or _operands("commit_drafts", (k_draft, v_draft, keys, values), (keys, values)))
    if not torch.is_inference_mode_enabled() and (keys.is_inference() or values.is_inference()):
        raise RuntimeError("inplace update to inference tensors outside InferenceMode is not allowed")
    length = cache_shape[2]
    if pages is None:
        _on(index, path, count, lengths)
        paged = (0, 0, 0, 0)
    else:
        _on(index, path, count, lengths, pages.block_table)
        if not layers:
            return
        pk, length = _paged(pages, keys[0], values[0], batch)
        paged = (pk.block_table, pk.bt_stride, pk.page_size, pk.num_pages)
    params = _lib.pack_commit(
        *pointers, *strides, path.data_ptr(), count.data_ptr(), lengths.data_ptr(), *paged,
        lengths.dtype is torch.int64, layers, batch, tokens, heads_kv, head_dim, length, dtype)
    status = _lib.load().asrlayer_commit(params, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_commit")
    del held  # copies live until the launch
    _increment_version((keys, values))
