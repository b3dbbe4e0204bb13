"""Linear layers with 8-bit weights on the HIP kernels of ``libasrattn.so``.

The matrix holds whole numbers -127 .. 127 and a scale per output, and a call rounds
its rows to such numbers with a scale each, so that the product is one of whole
numbers, at twice the rate of bfloat16 and half of its bytes: for prompts, encoder
frames and large batches as well as for a step's few rows, where the 4-bit layers
(:mod:`asrback_amd.linear4`) read half as much again.  :func:`quantize8` rounds a
matrix, :func:`pack8` takes one quantized elsewhere, both laid out once as the kernel
reads it (:class:`Weight8`); :func:`linear8` is the product, :func:`gated8` the
projections, activation and product of a gated feed-forward block over it,
:class:`Linear8` the module in place of ``nn.Linear``, and :func:`quantize_linears8`
puts it under a model.

Calls launch on the current HIP stream, never synchronize (the matrix is checked when
it is packed) and can be captured into a graph; there is no gradient, and calls that
would need one, in forward mode too, or that a tracer records are refused.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch
from torch import Tensor, nn

from . import _lib
from .attention import _DTYPES, _check_device
from .layers import _increment_version, check_out, computes, refuse_gradient, refuse_unseen
from .linear4 import _as_built

_BLOCK_N, _BLOCK_K = 16, 64
# Inputs of a row: the sum of their products stays within 32 bits.
MAX_INPUTS = 1 << 17
# The current stream's handle on a device; the current device (once a tensor is on one).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


@dataclass(frozen=True)
class Weight8:
    """A matrix ``(outputs, inputs)`` of 8-bit values with a scale per output, in
    the kernel's layout (``asrlayer_linear8_params``).  Made by :func:`pack8` or
    :func:`quantize8`.  As a view of them would, it keeps the memory and the layout that
    its tensors have when it is made."""

    packed: Tensor
    scales: Tensor
    outputs: int
    inputs: int

    def __post_init__(self) -> None:
        _check_layout(self.packed, self.scales, self.outputs, self.inputs)
        # What the kernel reads: views of its own, which nothing done to the tensors given
        # can resize.
        object.__setattr__(self, "_held", (self.packed.view(self.packed.shape), self.scales.view(self.scales.shape)))

    def __reduce__(self):
        return type(self), (self.packed, self.scales, self.outputs, self.inputs)  # (a copy holds views of its own)


def _check_layout(packed: Tensor, scales: Tensor, outputs: int, inputs: int) -> None:
    """The tensors are as large as the kernel reads them, and in its order: once for a
    :class:`Weight8`, at each call of a module, whose buffers can be replaced."""
    blocks = -(-outputs // _BLOCK_N) * -(-inputs // _BLOCK_K)
    if not (packed.numel() == blocks * 1024 and packed.dtype is torch.int8 and packed.is_contiguous()
            and scales.shape == (outputs,) and scales.is_contiguous()):
        raise ValueError(f"packed and scales are not a packed ({outputs}, {inputs}) matrix")


def pack8(values: Tensor, scales: Tensor) -> Weight8:
    """Lay out a quantized matrix: weight ``(n, k)`` is ``scales[n] * values[n, k]``
    with ``values`` int8 ``(outputs, inputs)`` in -127 .. 127 and ``scales`` float32
    or bfloat16 ``(outputs,)`` (the type of the rows the matrix will take)."""
    if values.dim() != 2 or values.dtype != torch.int8:
        raise ValueError(f"values must be int8 (outputs, inputs), got {values.dtype} {tuple(values.shape)}")
    outputs, inputs = values.shape
    if outputs < 1 or not 1 <= inputs <= MAX_INPUTS:
        raise ValueError(f"a matrix has at least one output and 1 to {MAX_INPUTS} inputs, got {tuple(values.shape)}")
    if scales.shape != (outputs,):
        raise ValueError(f"scales must be ({outputs},), got {tuple(scales.shape)}")
    if scales.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"scales must be float32 or bfloat16, got {scales.dtype}")
    if scales.device != values.device:
        raise RuntimeError("values and scales must be on one device")
    if int(values.min()) < -127:
        raise ValueError("values must lie in -127 .. 127")
    blocks_n, blocks_k = -(-outputs // _BLOCK_N), -(-inputs // _BLOCK_K)
    packed = torch.empty((blocks_n, blocks_k, 4, _BLOCK_N, 16), dtype=torch.int8, device=values.device)
    step = max(1, (1 << 26) // (blocks_k * _BLOCK_K * _BLOCK_N))  # bounds the temporaries
    for first in range(0, blocks_n, step):
        last = min(first + step, blocks_n)
        part = values[first * _BLOCK_N:last * _BLOCK_N]
        block = part.new_zeros(((last - first) * _BLOCK_N, blocks_k * _BLOCK_K))
        block[: part.shape[0], :inputs] = part
        packed[first:last] = block.view(-1, _BLOCK_N, blocks_k, 4, 16).permute(0, 2, 3, 1, 4)
    return Weight8(packed, scales.detach().contiguous(), outputs, inputs)


def unpack8(weight: Weight8) -> Tensor:
    """The matrix a :class:`Weight8` stands for, float32 ``(outputs, inputs)``."""
    blocks_n, blocks_k = weight.packed.shape[:2]
    values = weight.packed.permute(0, 3, 1, 2, 4).reshape(blocks_n * _BLOCK_N, blocks_k * _BLOCK_K)
    return values[: weight.outputs, : weight.inputs].float() * weight.scales.float()[:, None]


@torch.no_grad()
def quantize8(weight: Tensor) -> Weight8:
    """Round a float32 or bfloat16 matrix ``(outputs, inputs)`` to 8 bits: an
    output's scale puts its largest magnitude at 127 and is kept in the matrix's
    type, and the values are rounded for the scale as kept."""
    if weight.dim() != 2 or weight.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"a float32 or bfloat16 matrix, got {weight.dtype} {tuple(weight.shape)}")
    if not weight.numel():
        raise ValueError(f"a matrix has at least one output and input, got {tuple(weight.shape)}")
    w = weight.detach().float()
    scales = (w.abs().amax(1) / 127).to(weight.dtype)
    if not torch.isfinite(scales).all():
        raise ValueError("the matrix holds infinities or NaN")
    step = scales.float()[:, None]
    values = torch.where(step > 0, w / step, 0.0).round_().clamp_(-127, 127).to(torch.int8)
    return pack8(values, scales)


def linear8(x: Tensor, weight: Weight8, bias: Tensor | None = None, *, out: Tensor | None = None) -> Tensor:
    """``x @ w.T + bias`` for the matrix ``w`` that ``weight`` stands for, over rows
    rounded to 8 bits (``asrlayer_linear8``): ``x`` ``(..., inputs)`` float32 or
    bfloat16, the type of the weight's scales, ``bias`` ``(outputs,)`` of the same type.
    Each row is rounded to whole numbers -127 .. 127 (of the exact quotient, ties to
    even) times a float32 scale, its largest magnitude's 127th part; the sum of the
    products is exact, what follows float32, rounded once.  A row with an infinity or
    a NaN comes out as NaN.  ``out`` is written in place and must not share
    memory with ``x`` or ``bias``.  Returns ``(..., outputs)``."""
    refuse_gradient("linear8", weight.scales)
    return _product("linear8", x, *weight._held, weight.outputs, weight.inputs, bias, out, False)


def gated8(x: Tensor, weight: Weight8, bias: Tensor | None = None, *, out: Tensor | None = None) -> Tensor:
    """``silu(y[..., :n]) * y[..., n:]`` for ``y = linear8(x, weight, bias)`` with
    ``2 n`` outputs, the gates before the projections, in one product
    (``asrlayer_linear8``): float32 until the one rounding at the end.  Arguments as
    for :func:`linear8`.  Returns ``(..., n)``."""
    refuse_gradient("gated8", weight.scales)
    return _product("gated8", x, *weight._held, weight.outputs, weight.inputs, bias, out, True)


@functools.lru_cache(maxsize=1024)
def _workspace(rows: int, outputs: int, inputs: int, gated: bool) -> int:
    return _lib.load().asrlayer_linear8_workspace_size(rows, outputs, inputs, gated)


def _product(what: str, x: Tensor, packed: Tensor, scales: Tensor, outputs: int, inputs: int, bias: Tensor | None,
             out: Tensor | None, gated: bool) -> Tensor:
    shape = x.shape
    if not shape or shape[-1] != inputs:
        raise ValueError(f"x must be (..., {inputs}), got {tuple(shape)}")
    dtype, index = x.dtype, x.get_device()
    if gated and outputs % 2:
        raise ValueError(f"a gated matrix has as many gates as projections, got {outputs} outputs")
    if dtype is not scales.dtype:
        raise TypeError(f"x is {dtype}, the weight's scales {scales.dtype}")
    if dtype not in _DTYPES:
        raise TypeError(f"{what} supports float32 and bfloat16, got {dtype}")
    if bias is not None and (bias.shape != (outputs,) or bias.dtype is not dtype):
        raise ValueError(f"bias must be {dtype} ({outputs},), got {bias.dtype} {tuple(bias.shape)}")
    refuse_unseen(what, x, scales, bias)
    width = outputs // 2 if gated else outputs
    given = out is not None
    if given:
        if out.shape != (*shape[:-1], width) or out.dtype is not dtype or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {(*shape[:-1], width)} tensor of x's dtype")
        check_out(what, out, x, bias, packed, scales)
    if index < 0:
        raise RuntimeError(f"{what} runs on the GPU only; got a tensor on {x.device}")
    refuse_gradient(what, x, bias)
    if (index != _current_device() or packed.get_device() != index or scales.get_device() != index
            or (bias is not None and bias.get_device() != index) or (given and out.get_device() != index)):
        _check_device(x, packed, scales, bias, out)  # says what is wrong
    if not given:
        out = x.new_empty((*shape[:-1], width))
    rows = x if len(shape) == 2 else x.reshape(-1, inputs)
    if rows.stride(1) != 1 and inputs > 1:
        rows = rows.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    count = rows.shape[0]
    # Rounded rows, 16 to a block, and their scales, where a launch of its own rounds them.
    size = _workspace(count, outputs, inputs, gated)
    held = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    params = _lib.pack_linear8(
        rows.data_ptr(), rows.stride(0), packed.data_ptr(), scales.data_ptr(), 0 if bias is None else bias.data_ptr(),
        out.data_ptr(), width, count, outputs, inputs, gated, _DTYPES[dtype])
    status = _lib.load().asrlayer_linear8(params, held.data_ptr() if size else None, size, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_linear8")
    if given:
        _increment_version(out)
    return out


@computes
class Linear8(nn.Module):
    """``nn.Linear`` with 8-bit weights (:func:`linear8`); made by
    :meth:`from_linear` or from a :class:`Weight8`.  The matrix lies in
    buffers, so ``.to(device)`` and state dicts carry it, and ``.to(dtype)``
    rounds its scales and bias."""

    def __init__(self, weight: Weight8, bias: Tensor | None = None) -> None:
        super().__init__()
        self.in_features, self.out_features = weight.inputs, weight.outputs
        self.register_buffer("packed", weight.packed)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach())

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> Linear8:
        return cls(quantize8(linear.weight), linear.bias)

    @property
    def weight8(self) -> Weight8:
        return Weight8(self.packed, self.scales, self.out_features, self.in_features)

    def forward(self, x: Tensor) -> Tensor:
        _check_layout(self.packed, self.scales, self.out_features, self.in_features)
        refuse_gradient("linear8", self.scales)
        return _product("linear8", x, self.packed, self.scales, self.out_features, self.in_features, self.bias, None, False)

    def gated(self, x: Tensor) -> Tensor:
        """:func:`gated8` over this layer's matrix and bias."""
        _check_layout(self.packed, self.scales, self.out_features, self.in_features)
        refuse_gradient("gated8", self.scales)
        return _product("gated8", x, self.packed, self.scales, self.out_features, self.in_features, self.bias, None, True)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def quantize_linears8(module: nn.Module) -> int:
    """Replace every ``nn.Linear`` under ``module`` (not ``module`` itself) by a
    :class:`Linear8` of its rounded weights, in place; returns how many.  A layer that
    appears in several places is rounded once and stays shared; one that carries
    hooks or a forward of its own stays as it is.

    Prompts and steps gain where their layers are calls, as Qwen3's are.  An encoder of
    inputs of 768 to 1280 gains 3 to 12% (four Whisper layers of 1280 in bf16: 2.43 ms
    for 2.51 over 8 x 1500 frames, 0.57 for 0.64 over 1500): the rounding of its rows
    takes most of what the products save.  Kernels that read a layer's matrix in place
    of its call run for ``nn.Linear`` only, so that a Whisper decoder's step, whose layers
    take six launches, goes op by op and is slower (12 layers of 768 in bf16: 810 us for
    394 at one row, 1026 for 774 at 16; 4 layers of 1280: 300 for 159 and 445 for 417; 12
    of 768 in float32 801 for 456 and 1224 for 903): quantize the encoder alone there."""
    places = [(parent, name, child) for parent in module.modules()
              # (named_children leaves out a child's second name)
              for name, child in parent._modules.items()
              if child is not None and _as_built(child) and child.weight.numel() and child.in_features <= MAX_INPUTS]
    # All are rounded before the first is replaced: one that cannot be leaves the model
    # as it is.
    made = {child: Linear8.from_linear(child) for child in dict.fromkeys(c for _, _, c in places)}
    for parent, name, child in places:
        setattr(parent, name, made[child])
    return len(made)
