"""Linear layers with 4-bit weights on the HIP kernels of ``libasrattn.so``.

A decoder step of few rows is bound by reading the weights; with 4 bits each
(and a scale for every 32, 64 or 128 inputs of an output) there is a quarter
of them to read.  :func:`quantize4` rounds a matrix, :func:`pack4` takes one
quantized elsewhere, both laid out once as the kernel reads it
(:class:`Weight4`); :func:`linear4` is the product, :class:`Linear4` the module
in place of ``nn.Linear``, and :func:`quantize_linears` puts it under a model.

Calls launch on the current HIP stream, never synchronize (the matrix is
checked when it is packed) and can be captured into a graph; there is no
gradient, and calls that would need one, in forward mode too, or that a tracer
records are refused.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor, nn

from . import _lib
from .attention import _DTYPES, _aligned, _check_device
from .layers import _FORWARDS, _increment_version, check_out, refuse_gradient, refuse_unseen

GROUPS = (32, 64, 128)
_BLOCK_N, _BLOCK_K = 16, 128
# Inputs of a dword's nibbles, from the low one up (csrc/layers.hpp).
_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)
# The current stream's handle on a device.
_raw_stream = torch._C._cuda_getCurrentRawStream


@dataclass(frozen=True)
class Weight4:
    """A matrix ``(outputs, inputs)`` of 4-bit values with a scale (and a zero
    point) per ``group`` inputs of an output, in the kernel's layout
    (``asrlayer_linear4_params``).  Made by :func:`pack4` or
    :func:`quantize4`.  As a view of them would, it keeps the memory and the layout
    that its tensors have when it is made."""

    packed: Tensor
    scales: Tensor
    zeros: Tensor | None
    outputs: int
    inputs: int
    group: int

    def __post_init__(self) -> None:
        _check_layout(self.packed, self.scales, self.zeros, self.outputs, self.inputs, self.group)
        # What the kernel reads: views of its own, which nothing done to the tensors given
        # can resize.
        held = tuple(None if t is None else t.view(t.shape) for t in (self.packed, self.scales, self.zeros))
        object.__setattr__(self, "_held", held)

    def __reduce__(self):
        # (a copy holds views of its own)
        return type(self), (self.packed, self.scales, self.zeros, self.outputs, self.inputs, self.group)


def _check_layout(packed: Tensor, scales: Tensor, zeros: Tensor | None, outputs: int, inputs: int, group: int) -> None:
    """The tensors are as large as the kernel reads them, and in its order: once for a
    :class:`Weight4`, at each call of a module, whose buffers can be replaced and
    take the strides of another memory format."""
    _check_group(group, inputs)
    blocks = -(-outputs // _BLOCK_N) * -(-inputs // _BLOCK_K)
    groups = blocks * (_BLOCK_K // group)
    if not (packed.numel() == blocks * 256 and packed.dtype is torch.int32 and packed.is_contiguous()
            and scales.numel() == groups * 16 and scales.is_contiguous()
            and (zeros is None or (zeros.numel() == groups * 8 and zeros.dtype is torch.uint8 and zeros.is_contiguous()))):
        raise ValueError(f"packed, scales and zeros are not a packed ({outputs}, {inputs}) matrix with groups of {group}")


def _check_group(group: int, inputs: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"group {group} (supported: {', '.join(map(str, GROUPS))})")
    if inputs < 1 or inputs % group:
        raise ValueError(f"{inputs} inputs are not a positive multiple of the group of {group}")


def pack4(values: Tensor, scales: Tensor, zeros: Tensor | None = None) -> Weight4:
    """Lay out a quantized matrix: weight ``(n, k)`` is ``scales[n, k // group]
    * (values[n, k] - zeros[n, k // group])`` with ``values`` uint8 ``(outputs,
    inputs)`` in 0 .. 15, ``scales`` float32 or bfloat16 ``(outputs, inputs /
    group)`` (the type of the rows the matrix will take) and ``zeros`` uint8 of
    the same shape in 0 .. 15, or None for 8 everywhere."""
    if values.dim() != 2 or values.dtype != torch.uint8:
        raise ValueError(f"values must be uint8 (outputs, inputs), got {values.dtype} {tuple(values.shape)}")
    outputs, inputs = values.shape
    if outputs < 1 or scales.dim() != 2 or scales.shape[0] != outputs or scales.shape[1] < 1 or inputs % scales.shape[1]:
        raise ValueError(f"scales must be ({outputs}, inputs / group), got {tuple(scales.shape)}")
    if scales.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"scales must be float32 or bfloat16, got {scales.dtype}")
    group = inputs // scales.shape[1]
    _check_group(group, inputs)
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError(f"zeros must be uint8 {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
    for name, t in (("values", values), ("zeros", zeros)):
        if t is not None and int(t.max()) > 15:
            raise ValueError(f"{name} must lie in 0 .. 15")
    device = values.device
    if scales.device != device or (zeros is not None and zeros.device != device):
        raise RuntimeError("values, scales and zeros must be on one device")
    blocks_n, blocks_k = -(-outputs // _BLOCK_N), -(-inputs // _BLOCK_K)
    groups = blocks_k * _BLOCK_K // group
    packed = torch.empty((blocks_n, blocks_k, 64, 4), dtype=torch.int32, device=device)
    step = max(1, (1 << 26) // (blocks_k * _BLOCK_K * _BLOCK_N))  # bounds the temporaries
    for first in range(0, blocks_n, step):
        last = min(first + step, blocks_n)
        part = values[first * _BLOCK_N:last * _BLOCK_N]
        block = part.new_zeros(((last - first) * _BLOCK_N, blocks_k * _BLOCK_K))
        block[: part.shape[0], :inputs] = part
        # (block_n, i, block_k, s, g, j) -> (block_n, block_k, g, i, s, j)
        lanes = block.view(-1, _BLOCK_N, blocks_k, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
        pairs = [lanes[..., _ORDER[2 * i]] | lanes[..., _ORDER[2 * i + 1]] << 4 for i in range(4)]
        packed[first:last] = torch.stack(pairs, -1).contiguous().view(torch.int32).view(-1, blocks_k, 64, 4)

    def spread(t: Tensor) -> Tensor:
        """``(outputs, groups)`` as ``(block_n, block_k, 4, groups of a block, 4)``."""
        whole = t.new_zeros((blocks_n * _BLOCK_N, groups))
        whole[:outputs, : t.shape[1]] = t
        return whole.view(blocks_n, 4, 4, blocks_k, -1).permute(0, 3, 1, 4, 2).contiguous()

    if zeros is not None:
        nibbles = spread(zeros)
        zeros = nibbles[..., 0::2] | nibbles[..., 1::2] << 4
    return Weight4(packed, spread(scales.detach()), zeros, outputs, inputs, group)


def unpack4(weight: Weight4) -> Tensor:
    """The matrix a :class:`Weight4` stands for, float32 ``(outputs, inputs)``."""
    blocks_n, blocks_k = weight.packed.shape[:2]
    nibbles = torch.stack([weight.packed >> (4 * i) & 15 for i in range(8)], -1)  # (.., 64, 4, nibble)
    values = torch.empty_like(nibbles)
    values[..., list(_ORDER)] = nibbles
    values = values.view(blocks_n, blocks_k, 4, _BLOCK_N, 4, 8).permute(0, 3, 1, 4, 2, 5)
    values = values.reshape(blocks_n * _BLOCK_N, -1, weight.group).float()

    def gather(t: Tensor) -> Tensor:
        return t.permute(0, 2, 4, 1, 3).reshape(blocks_n * _BLOCK_N, -1, 1).float()

    zeros = 8.0
    if weight.zeros is not None:
        zeros = gather(torch.stack((weight.zeros & 15, weight.zeros >> 4), -1).flatten(-2))
    whole = ((values - zeros) * gather(weight.scales)).flatten(1)
    return whole[: weight.outputs, : weight.inputs].contiguous()


@torch.no_grad()
def quantize4(weight: Tensor, group: int = 128, symmetric: bool = True) -> Weight4:
    """Round a float32 or bfloat16 matrix ``(outputs, inputs)`` to 4 bits.
    ``symmetric``: values -8 .. 7 times a scale that puts the group's largest
    magnitude at 7; otherwise 0 .. 15 around a zero point, the group's smallest
    and largest weight (and 0) at the ends.  Scales are kept in the matrix's
    type, and the values are rounded for the scale as kept."""
    if weight.dim() != 2 or weight.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"a float32 or bfloat16 matrix, got {weight.dtype} {tuple(weight.shape)}")
    outputs, inputs = weight.shape
    _check_group(group, inputs)
    w = weight.detach().float().reshape(outputs, inputs // group, group)
    if symmetric:
        scales = (w.abs().amax(-1) / 7).to(weight.dtype)
        zeros, offset = None, 8.0
    else:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scales = ((high - low) / 15).to(weight.dtype)
        step = scales.float()
        offset = torch.where(step > 0, -low / step, 0.0).round_().clamp_(0, 15)
        zeros, offset = offset.to(torch.uint8), offset[..., None]
    if not torch.isfinite(scales).all():
        raise ValueError("the matrix holds infinities, NaN or values too large for a scale")
    step = scales.float()[..., None]
    values = torch.where(step > 0, w / step, 0.0).round_().add_(offset).clamp_(0, 15).to(torch.uint8)
    return pack4(values.view(outputs, inputs), scales, zeros)


def linear4(x: Tensor, weight: Weight4, bias: Tensor | None = None, *, out: Tensor | None = None) -> Tensor:
    """``x @ w.T + bias`` for the matrix ``w`` that ``weight`` stands for
    (``asrlayer_linear4``): ``x`` ``(..., inputs)`` float32 or bfloat16, the
    type of the weight's scales, ``bias`` ``(outputs,)`` of the same type.
    Sums are float32, of any finite row within range where their scale brings them
    there, and rounded once; a row with an infinity or a NaN comes out without a
    finite value.  Built for the few rows of a decoder step or a
    drafted tree (up to 32 are read against the weights in one pass); more rows
    are right, the weights being read again for each 32.  ``out`` is written in
    place and must not share memory with ``x`` or ``bias``.  Returns ``(..., outputs)``."""
    refuse_gradient("linear4", weight.scales)
    return _product(x, *weight._held, weight.outputs, weight.inputs, weight.group, bias, out)


def _product(x: Tensor, packed: Tensor, scales: Tensor, zeros: Tensor | None, outputs: int, inputs: int, group: int,
             bias: Tensor | None, out: Tensor | None) -> Tensor:
    shape = x.shape
    if not shape or shape[-1] != inputs:
        raise ValueError(f"x must be (..., {inputs}), got {tuple(shape)}")
    dtype, index = x.dtype, x.get_device()
    if dtype is not scales.dtype:
        raise TypeError(f"x is {dtype}, the weight's scales {scales.dtype}")
    if dtype not in _DTYPES:
        raise TypeError(f"linear4 supports float32 and bfloat16, got {dtype}")
    if bias is not None and (bias.shape != (outputs,) or bias.dtype is not dtype):
        raise ValueError(f"bias must be {dtype} ({outputs},), got {bias.dtype} {tuple(bias.shape)}")
    refuse_unseen("linear4", x, scales, bias)
    given = out is not None
    if given:
        if out.shape != (*shape[:-1], outputs) or out.dtype is not dtype or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {(*shape[:-1], outputs)} tensor of x's dtype")
        check_out("linear4", out, x, bias)
    if index < 0:
        raise RuntimeError(f"linear4 runs on the GPU only; got a tensor on {x.device}")
    refuse_gradient("linear4", x, bias)
    if not given:
        out = x.new_empty((*shape[:-1], outputs))
    rows = _aligned(x if len(shape) == 2 else x.reshape(-1, inputs))
    others = (packed, scales, zeros, bias, out)
    if index != torch.cuda.current_device() or any(t is not None and t.get_device() != index for t in others):
        _check_device(x, *others)  # says what is wrong
    if bias is not None:
        bias = bias.contiguous()
    params = _lib.pack_linear4(
        rows.data_ptr(), rows.stride(0), packed.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(),
        0 if bias is None else bias.data_ptr(), out.data_ptr(), outputs, rows.shape[0], outputs, inputs, group,
        _DTYPES[dtype])
    status = _lib.load().asrlayer_linear4(params, _raw_stream(index))
    if status:
        _lib.check(status, "asrlayer_linear4")
    if given:
        _increment_version(out)
    return out


class Linear4(nn.Module):
    """``nn.Linear`` with 4-bit weights (:func:`linear4`); made by
    :meth:`from_linear` or from a :class:`Weight4`.  The matrix lies in
    buffers, so ``.to(device)`` and state dicts carry it, and ``.to(dtype)``
    rounds its scales and bias."""

    def __init__(self, weight: Weight4, bias: Tensor | None = None) -> None:
        super().__init__()
        self.in_features, self.out_features, self.group = weight.inputs, weight.outputs, weight.group
        self.register_buffer("packed", weight.packed)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.register_buffer("bias", None if bias is None else bias.detach())

    @classmethod
    def from_linear(cls, linear: nn.Linear, group: int = 128, symmetric: bool = True) -> Linear4:
        return cls(quantize4(linear.weight, group, symmetric), linear.bias)

    @property
    def weight4(self) -> Weight4:
        return Weight4(self.packed, self.scales, self.zeros, self.out_features, self.in_features, self.group)

    def forward(self, x: Tensor) -> Tensor:
        _check_layout(self.packed, self.scales, self.zeros, self.out_features, self.in_features, self.group)
        refuse_gradient("linear4", self.scales)
        return _product(x, self.packed, self.scales, self.zeros, self.out_features, self.in_features, self.group, self.bias,
                        None)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, group={self.group}, "
                f"zeros={self.zeros is not None}, bias={self.bias is not None}")


def _as_built(layer: nn.Module) -> bool:
    """Whether ``layer`` is an ``nn.Linear`` and nothing else: no hooks, no forward of its
    own."""
    own = layer.__dict__
    return (type(layer) is nn.Linear and "forward" not in own and nn.Linear.forward is _FORWARDS[nn.Linear]
            and not any(hooks for name, hooks in own.items() if name.endswith("_hooks")))


def quantize_linears(module: nn.Module, group: int = 128, symmetric: bool = True) -> int:
    """Replace every ``nn.Linear`` under ``module`` (not ``module`` itself) whose
    inputs are whole groups by a :class:`Linear4` of its rounded weights, in
    place; returns how many.  A layer that appears in several places is rounded
    once and stays shared; one that carries hooks or a forward of its own stays as
    it is.

    Steps of few rows gain where their layers are calls, as Qwen3's are.  Kernels that
    read a layer's matrix in place of its call run for ``nn.Linear`` only: a
    Whisper decoder's step, whose layers take six launches, goes op by op with 4-bit
    ones (a step of 6 layers of 768 in bf16: 412 us for 244 at one row, 463 for 443 at
    16; 8 layers of 1280: 625 for 395 and 770 for 1017, in float32 821 for 1077 and
    1144 for 1303), and a batch of encoder frames reads the weights again for each
    32 of them."""
    places = [(parent, name, child) for parent in module.modules()
              # (named_children leaves out a child's second name)
              for name, child in parent._modules.items()
              if child is not None and _as_built(child) and child.in_features % group == 0]
    # All are rounded before the first is replaced: one that cannot be leaves the model
    # as it is.
    made = {child: Linear4.from_linear(child, group, symmetric) for child in dict.fromkeys(c for _, _, c in places)}
    for parent, name, child in places:
        setattr(parent, name, made[child])
    return len(made)
