"""A key/value cache of 8-bit values on the HIP kernels of ``libasrattn.so``.

A decoder step is bound by reading the cache; with 8 bits a value (and a float32 scale
per position and kv head) there is half as much of it to read as in bfloat16, and
twice as many positions fit.  :class:`Cache8` is one layer's cache, a slab or a page
pool; :func:`write8` rounds new tokens' keys and values into it, :func:`decode8` is
the attention of one query a row over it, :func:`decode_append8` both for a
decoder's step, and :func:`read8` gives it back in a float
type, for what attends over it in another way.

As in :mod:`asrback_amd.attention`, calls launch on the current HIP stream, never
synchronize, and can be captured into a graph; nothing here has a gradient, and calls
that would need one, in forward mode too, or that a tracer records are refused.
"""

from __future__ import annotations

import functools
import itertools
from dataclasses import dataclass

import torch
from torch import Tensor

from . import _lib
from .attention import _DTYPES, PageTable, _aligned, _check_device, _split_workspace
from .drafts import _lengths, _on
from .layers import _increment_version, check_out, overlap, refuse_gradient, refuse_unseen, repeats

HEAD_DIMS = (64, 128, 256)
# The current stream's handle on a device; the current device (once a tensor is on one).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


@dataclass(frozen=True)
class Cache8:
    """One layer's 8-bit keys and values: position ``j`` of row ``b`` holds the key
    ``key_scales[b, h, j] * keys[b, j, h]`` of kv head ``h``, and its value likewise.

    ``keys``/``values`` int8 ``(batch, length, heads_kv, head_dim)``, any strides of
    whole 16-byte vectors with a unit last one; the scales float32 ``(batch, heads_kv,
    length)`` with a unit last stride.  With a :class:`~asrback_amd.attention.PageTable`
    at a call they are pools, ``(num_pages, page_size, heads_kv, head_dim)`` and
    ``(num_pages, heads_kv, page_size)``.  Tensors that hold an element more than once, as
    expanded ones do, or share memory can be read but not written.  As a view of them
    would, it keeps the memory and the layout that they have when it is made: a tensor
    that is resized or set to another memory afterwards does not change it."""

    keys: Tensor
    values: Tensor
    key_scales: Tensor
    value_scales: Tensor

    def __post_init__(self) -> None:
        shape = self.keys.shape
        if len(shape) != 4 or self.values.shape != shape:
            raise ValueError(f"keys and values must share one (batch, length, heads_kv, head_dim) shape; got "
                             f"{tuple(shape)}, {tuple(self.values.shape)}")
        batch, length, heads, head_dim = shape
        if head_dim not in HEAD_DIMS or heads < 1:
            raise ValueError(f"{heads} heads of {head_dim} (supported head dims: {', '.join(map(str, HEAD_DIMS))})")
        for name in ("keys", "values"):
            t = getattr(self, name)
            *strides, last = t.stride()
            if t.dtype != torch.int8:
                raise TypeError(f"{name} must be int8, got {t.dtype}")
            if t.numel() and (last != 1 or t.data_ptr() % 16 or any(s % 16 for s in strides)):
                raise ValueError(f"{name} needs a unit last stride and 16-byte aligned rows (it is written in place)")
        for name in ("key_scales", "value_scales"):
            t = getattr(self, name)
            if t.dtype != torch.float32 or t.shape != (batch, heads, length):
                raise ValueError(f"{name} must be float32 ({batch}, {heads}, {length}), got {t.dtype} {tuple(t.shape)}")
            if t.stride(2) != 1 and length > 1:
                raise ValueError(f"{name} needs a unit last stride")
        if any(t.device != self.keys.device for t in self.tensors):
            raise RuntimeError("a cache's tensors must be on one device")
        # What the kernels read and write: views of the cache's own, which nothing done to the
        # tensors given can resize (detach() makes them in a third of view()'s time).
        object.__setattr__(self, "_held", tuple(t.detach() for t in self.tensors))
        # What a call needs to know of them besides their addresses (asking anew is a
        # third of its time): sizes, the strides as the kernels take them, and whether they
        # are inference tensors.
        object.__setattr__(self, "_sizes", (batch, length, heads, head_dim))
        strides = (*self.keys.stride()[:3], *self.values.stride()[:3], *self.key_scales.stride()[:2],
                   *self.value_scales.stride()[:2])
        object.__setattr__(self, "_strides", strides)
        object.__setattr__(self, "_inference", any(t.is_inference() for t in self.tensors))

    @functools.cached_property
    def _repeats(self) -> bool:
        apart = len({t.untyped_storage().data_ptr() for t in self._held}) == len(self._held)
        return any(repeats(t) for t in self._held) or \
            not apart and any(overlap(*pair) for pair in itertools.combinations(self._held, 2))

    def __reduce__(self):
        return type(self), self.tensors  # (a copy holds views of its own)

    @property
    def tensors(self) -> tuple[Tensor, Tensor, Tensor, Tensor]:
        return self.keys, self.values, self.key_scales, self.value_scales

    @classmethod
    def allocate(cls, batch: int, length: int, heads_kv: int, head_dim: int, device=None) -> Cache8:
        """An empty cache (zeros), or with pages a pool of ``batch`` pages of ``length``
        positions."""
        keys, values = (torch.zeros((batch, length, heads_kv, head_dim), dtype=torch.int8, device=device) for _ in "kv")
        scales = [torch.zeros((batch, heads_kv, length), dtype=torch.float32, device=device) for _ in "kv"]
        return cls(keys, values, *scales)


def _cache_fields(cache: Cache8, pages: PageTable | None, batch: int, index: int) -> tuple:
    """The fields of ``asrlayer_cache8`` over ``batch`` rows, on GPU ``index``."""
    k, v, key_scales, value_scales = cache._held
    lead, length, heads, head_dim = cache._sizes
    if k.get_device() != index:
        _on(index, k)
    if pages is None:
        if lead != batch:
            raise ValueError(f"{batch} rows, the cache has {lead}")
        paged = (0, 0, 0, 0)
    else:
        table = pages.block_table
        if table.shape[0] < batch:
            raise ValueError(f"block_table has {table.shape[0]} rows for {batch} sequences")
        if table.get_device() != index:
            _on(index, table)
        reach, page_size = table.shape[1] * length, length
        length = reach if pages.max_len is None else pages.max_len
        if not 0 <= length <= reach:
            raise ValueError(f"max_len {length} outside the table's reach {reach}")
        # (a table that reaches nothing is no table)
        paged = (table.data_ptr(), table.stride(0), page_size, lead) if length else (0, 0, 0, 0)
    return (k.data_ptr(), v.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), *cache._strides, *paged, batch, heads,
            head_dim, length)


def _ready(what: str, first: Tensor, *others: Tensor | None) -> int:
    """The index of the current GPU, which must hold these float tensors of one
    supported type, none of which may need a gradient."""
    index, dtype, grad = first.get_device(), first.dtype, torch.is_grad_enabled()
    if dtype not in _DTYPES:
        raise TypeError(f"{what} supports float32 and bfloat16, got {dtype}")
    elsewhere = index >= 0 and index != _current_device()
    for t in (first, *others):
        if t is None:
            continue
        if t.dtype is not dtype:
            raise TypeError(f"mixed dtypes: {dtype} and {t.dtype}")
        if t.get_device() != index:
            elsewhere = True
        if grad and t.requires_grad and index >= 0:
            raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad() or on detached tensors")
    if index < 0:
        raise RuntimeError(f"{what} runs on the GPU only; got tensors on {first.device}")
    if elsewhere:
        _check_device(first, *others)  # says what is wrong
    return index


def _check_written(what: str, cache: Cache8) -> None:
    if cache._repeats:
        raise ValueError(f"{what} cannot write a cache that holds elements more than once")
    if cache._inference and not torch.is_inference_mode_enabled():
        raise RuntimeError("inplace update to inference tensors outside InferenceMode is not allowed")


def _index(t: Tensor | None, name: str, tokens: int) -> Tensor | None:
    if t is None:
        return None
    if t.dtype != torch.int64 or t.shape != (tokens,):
        raise ValueError(f"{name} must be int64 ({tokens},), got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def write8(cache: Cache8, k: Tensor, v: Tensor, rows: Tensor | None, positions: Tensor, *,
           pages: PageTable | None = None) -> None:
    """Round new tokens' keys and values ``k``/``v`` ``(tokens, heads_kv, head_dim)``
    (float32 or bfloat16) into ``cache`` (``asrlayer_write8``): token ``t`` goes to
    position ``positions[t]`` of row ``rows[t]`` (int64; None: row ``t``).  Slots
    outside the cache or on no page are left alone; of two tokens for one slot
    neither is sure to be held whole.  Each key and value becomes whole numbers -127 ..
    127 (of the exact quotient, ties to even) times a float32 scale, its largest
    magnitude's 127th part; one with an infinity or a NaN gets the scale NaN."""
    _write("write8", cache, k, v, rows, positions, pages)


def write_rows8(cache: Cache8, q: Tensor, k: Tensor, v: Tensor, rows: Tensor | None, positions: Tensor, *,
                q_norm: Tensor, k_norm: Tensor, q_eps: float, k_eps: float, cos: Tensor, sin: Tensor,
                pages: PageTable | None = None, keys: bool = False) -> tuple[Tensor, Tensor | None]:
    """:func:`write8` of a decoder's projections, in one pass with what comes before: the
    per-head norms and the rotation of ``q`` ``(tokens, heads_q, head_dim)`` and ``k``
    (as :func:`asrback_amd.layers.prompt_rows` computes them; weights ``(head_dim,)``,
    tables ``(tokens, head_dim)``).  Returns the queries and, with ``keys``, the
    keys as they were before their rounding."""
    tokens, heads_q, head_dim = q.shape
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t.shape != (head_dim,):
            raise ValueError(f"{name} must be ({head_dim},), got {tuple(t.shape)}")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.shape != (tokens, head_dim):
            raise ValueError(f"{name} must be ({tokens}, {head_dim}), got {tuple(t.shape)}")
    return _write("write_rows8", cache, k, v, rows, positions, pages, q, (q_norm, k_norm, q_eps, k_eps, cos, sin), keys)


def _write(what: str, cache: Cache8, k: Tensor, v: Tensor, rows: Tensor | None, positions: Tensor,
           pages: PageTable | None, q: Tensor | None = None, prologue: tuple | None = None, keys: bool = False):
    lead, _, heads, head_dim = cache._sizes
    shape = k.shape
    if len(shape) != 3 or shape != (shape[0], heads, head_dim) or v.shape != shape:
        raise ValueError(f"k and v must be (tokens, {heads}, {head_dim}); got {tuple(shape)}, {tuple(v.shape)}")
    tokens = shape[0]
    if q is not None and (q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != head_dim):
        raise ValueError(f"q must be ({tokens}, heads, {head_dim}), got {tuple(q.shape)}")
    rows, positions = _index(rows, "rows", tokens), _index(positions, "positions", tokens)
    if positions is None:
        raise TypeError("positions must be a tensor")
    weights = () if prologue is None else (*prologue[:2], *prologue[4:])
    refuse_unseen(what, k, v, q, *weights, *cache.tensors)
    refuse_gradient(what, cache.key_scales, cache.value_scales)
    _check_written(what, cache)
    index = _ready(what, k, v, q, *weights)
    _on(index, rows, positions)
    batch = lead if pages is None else pages.block_table.shape[0]
    if rows is None and tokens > batch:
        raise ValueError(f"{tokens} tokens without rows for a cache of {batch}")
    k, v = _aligned(k), _aligned(v)
    fields = _cache_fields(cache, pages, batch, index)
    q_out = k_out = None
    q_fields, outs, norms, eps, heads_q = (0, 0, 0), (0, 0), (0, 0, 0, 0, 0), (0.0, 0.0), 0
    if q is not None:
        q = _aligned(q)
        q_norm, k_norm, q_eps, k_eps, cos, sin = prologue
        q_norm, k_norm, cos, sin = (_aligned(t if t.is_contiguous() else t.contiguous()) for t in (q_norm, k_norm, cos, sin))
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if keys else None
        heads_q = q.shape[1]
        q_fields, outs = (q.data_ptr(), *q.stride()[:2]), (q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr())
        norms, eps = (q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.stride(0)), (q_eps, k_eps)
    params = _lib.pack_write8(
        *fields, q_fields[0], k.data_ptr(), v.data_ptr(), *outs, *q_fields[1:], *k.stride()[:2], *v.stride()[:2],
        0 if rows is None else rows.data_ptr(), positions.data_ptr(), *norms, tokens, *eps, heads_q, _DTYPES[k.dtype])
    status = _lib.load().asrlayer_write8(params, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_write8")
    _increment_version(cache._held)
    return q_out, k_out


def read8(cache: Cache8, *, lengths: Tensor | None = None, pages: PageTable | None = None,
          dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
    """The keys and values that ``cache`` stands for, ``(batch, length, heads_kv,
    head_dim)`` in ``dtype`` (float32 or bfloat16; ``asrlayer_read8``): zeros from
    position ``lengths[b]`` (int32 or int64, default: none) of row ``b`` on, and where
    there is no page."""
    if dtype not in _DTYPES:
        raise TypeError(f"read8 gives float32 and bfloat16, not {dtype}")
    lead, _, heads, head_dim = cache._sizes
    batch = lead if pages is None else pages.block_table.shape[0]
    lengths = _lengths(lengths, batch)
    refuse_unseen("read8", *cache.tensors)
    refuse_gradient("read8", cache.key_scales, cache.value_scales)
    keys = cache._held[0]
    index = keys.get_device()
    if index < 0:
        raise RuntimeError(f"read8 runs on the GPU only; got tensors on {keys.device}")
    if index != _current_device():
        _check_device(keys)
    _on(index, lengths)
    fields = _cache_fields(cache, pages, batch, index)
    k_out = torch.empty((batch, fields[-1], heads, head_dim), dtype=dtype, device=keys.device)
    v_out = torch.empty_like(k_out)
    params = _lib.pack_read8(*fields, k_out.data_ptr(), v_out.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
                             lengths is not None and lengths.dtype is torch.int64, _DTYPES[dtype])
    status = _lib.load().asrlayer_read8(params, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_read8")
    return k_out, v_out


@functools.lru_cache(maxsize=256)
def _workspace(batch: int, heads_q: int, heads_kv: int, head_dim: int, max_len: int, window: int, dtype: int) -> int:
    """``asrlayer_decode8_workspace_size`` of these sizes (-1 for ones it does not
    take)."""
    params = _lib.Decode8Params()
    params.batch, params.heads_q, params.heads_kv, params.head_dim = batch, heads_q, heads_kv, head_dim
    params.max_len, params.window, params.dtype, params.scale = max_len, window, dtype, 1.0
    need = _lib.load().asrlayer_decode8_workspace_size(bytes(params))
    return -1 if need == (1 << 64) - 1 else need


def decode8_workspace_size(batch: int, heads_q: int, heads_kv: int, head_dim: int, max_len: int,
                           dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes of split partials a :func:`decode8` call of these sizes needs
    (``asrlayer_decode8_workspace_size``; 0 when it runs unsplit), with any window:
    where it is not 0, enough for every smaller batch over the same cache.  Raises for
    sizes the library does not take."""
    if dtype not in _DTYPES:
        raise TypeError(f"attention supports float32 and bfloat16, got {dtype}")
    sizes = (batch, heads_q, heads_kv, head_dim, max_len, 0, _DTYPES[dtype])
    need = _workspace(*sizes)
    if need < 0:
        _workspace.__wrapped__(*sizes)  # leaves its message
        raise ValueError(_lib.load().asrattn_last_error().decode("utf-8", "replace"))
    return need


def decode8(q: Tensor, cache: Cache8, *, lengths: Tensor | None = None, scale: float | None = None,
            out: Tensor | None = None, workspace: Tensor | None = None, pages: PageTable | None = None,
            window: int | None = None) -> Tensor:
    """One query per row over an 8-bit cache (``asrlayer_decode8``): ``q`` ``(batch,
    heads_q, head_dim)`` float32 or bfloat16 attends positions ``0 .. lengths[b] - 1``
    of row ``b`` (int32 or int64, default: all of them; outside the cache they are
    clamped to it), with ``window`` the last ``window`` of them.  Rows with none get
    zeros.  Any number of query heads per kv head.  Products are of the stored numbers
    and exact, sums float32.  ``out`` is written in place; it may be ``q`` itself.
    ``workspace``: the split partials' memory (:func:`decode8_workspace_size`,
    :func:`asrback_amd.attention.workspace`).  Returns ``(batch, heads_q, head_dim)``."""
    return _decode("decode8", q, cache, lengths, scale, out, workspace, pages, window)


def decode_append8(q: Tensor, k: Tensor, v: Tensor, cache: Cache8, positions: Tensor, *, q_norm: Tensor, k_norm: Tensor,
                   q_eps: float, k_eps: float, cos: Tensor, sin: Tensor, scale: float | None = None,
                   out: Tensor | None = None, workspace: Tensor | None = None, pages: PageTable | None = None,
                   window: int | None = None) -> Tensor:
    """A decoder step in one launch (``asrlayer_append8``): :func:`write_rows8` of one token a
    row, ``k``/``v`` ``(batch, heads_kv, head_dim)`` at ``positions`` (int64), and
    :func:`decode8` of the queries ``q`` ``(batch, heads_q, head_dim)`` over positions ``0 ..
    positions[b]`` (the whole cache where that is past its end, without the new key,
    which is dropped there as it is where there is no page; none below 0).  Returns
    ``(batch, heads_q, head_dim)``."""
    batch, heads, head_dim = q.shape[0], *cache._sizes[2:]
    for name, t in (("k", k), ("v", v)):
        if t.shape != (batch, heads, head_dim):
            raise ValueError(f"{name} must be ({batch}, {heads}, {head_dim}), got {tuple(t.shape)}")
    for name, t, shape in (("q_norm", q_norm, (head_dim,)), ("k_norm", k_norm, (head_dim,)),
                           ("cos", cos, (batch, head_dim)), ("sin", sin, (batch, head_dim))):
        if t.shape != shape:
            raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    positions = _index(positions, "positions", batch)
    if positions is None:
        raise TypeError("positions must be a tensor")
    return _decode("decode_append8", q, cache, None, scale, out, workspace, pages, window,
                   (k, v, q_norm, k_norm, cos, sin), positions, q_eps, k_eps)


def _decode(what: str, q: Tensor, cache: Cache8, lengths: Tensor | None, scale: float | None, out: Tensor | None,
            workspace: Tensor | None, pages: PageTable | None, window: int | None, new: tuple = (),
            positions: Tensor | None = None, q_eps: float = 0.0, k_eps: float = 0.0) -> Tensor:
    shape = q.shape
    _, _, heads_kv, head_dim = cache._sizes
    if len(shape) != 3 or shape[2] != head_dim:
        raise ValueError(f"q must be (batch, heads, {head_dim}), got {tuple(shape)}")
    batch, heads_q, _ = shape
    if heads_q == 0 or heads_q % heads_kv:
        raise ValueError(f"{heads_q} query heads are not a positive multiple of {heads_kv} kv heads")
    if window is not None and window < 1:
        raise ValueError(f"a window holds at least one position, got {window}")
    lengths = _lengths(lengths, batch)
    refuse_unseen(what, q, *new, *cache.tensors)
    refuse_gradient(what, cache.key_scales, cache.value_scales)
    given = out is not None
    if given:
        if out.shape != shape or out.dtype != q.dtype or out.stride(-1) != 1:
            raise ValueError("out must match q's shape and dtype, with a unit last stride")
        # A row's queries are read before any of its outputs is written.
        in_place = out.data_ptr() == q.data_ptr() and out.stride() == q.stride()
        check_out(what, out, None if in_place else q, *new, *cache._held, lengths, positions)
    if new:
        _check_written(what, cache)
    index = _ready(what, q, *new)
    q = _aligned(q)
    _on(index, lengths, out, positions)
    fields = _cache_fields(cache, pages, batch, index)
    if not given:
        out = q.new_empty(shape)
    # (A cache has at most 2^30 positions.)
    code, span = _DTYPES[q.dtype], min(window or 0, 1 << 30)
    step = (*fields, q.data_ptr(), out.data_ptr(), *q.stride()[:2], *out.stride()[:2],
            0 if lengths is None else lengths.data_ptr(), lengths is not None and lengths.dtype is torch.int64, heads_q, span,
            code, head_dim**-0.5 if scale is None else scale)
    need = _workspace(batch, heads_q, heads_kv, head_dim, fields[-1], span, code)
    size = 0
    if need > 0:
        workspace = _split_workspace(need, workspace, out.device)
    if workspace is not None:
        size, workspace = workspace.numel(), workspace.data_ptr()
    # Sizes that the library does not take (need -1): the call says why.
    lib = _lib.load()
    if not new:
        status = lib.asrlayer_decode8(_lib.pack_decode8(*step), workspace, size, _raw_stream(index))
    else:
        k, v = _aligned(new[0]), _aligned(new[1])
        q_norm, k_norm, cos, sin = (_aligned(t if t.is_contiguous() else t.contiguous()) for t in new[2:])
        status = lib.asrlayer_append8(
            _lib.pack_append8(*step, 0, k.data_ptr(), v.data_ptr(), *k.stride()[:2], *v.stride()[:2], positions.data_ptr(),
                              q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.stride(0), q_eps, k_eps),
            workspace, size, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_append8" if new else "asrlayer_decode8")
    if new:
        _increment_version(cache._held)
    if given:
        _increment_version(out)
    return out
