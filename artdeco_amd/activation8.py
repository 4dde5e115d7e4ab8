"""An MLP's activation whose backward pass reads its input from 8 bits (csrc/activation8.hip), and the MLP that keeps nothing else.

A float16 MLP layer keeps fc1's output for the activation's gradient and the activation's output for fc2's weight gradient: 4 bytes a
hidden value.  Here the forward pass leaves one code a value, 32 consecutive values sharing a power of two (33/32 byte a value), and the
backward pass takes both from it.  int8 holds a value to 1/254 .. 1/127 of its block's largest, e4m3 to 1/16 of itself, at best to 2^-18
of its block's largest (smaller ones are held as 0).  Forward results are those of the values as they are, worked out in 32 bits and rounded
once; gradients are those of the held values."""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F

from artdeco_amd import _lib

_DTYPES = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}
_KINDS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}
_FORMATS = {"int8": 0, "e4m3": 1}


class Packed8(NamedTuple):
    """A tensor in 8 bits: `codes` (uint8, its values in order, then room up to a multiple of 32) and `units` (uint8, one for 32 values,
    unit 2^(units - 127)); the tensor's shape and type, and the format."""
    codes: torch.Tensor
    units: torch.Tensor
    shape: tuple
    dtype: torch.dtype
    format: str


def _rows_width(what, shape, gated):
    if not shape or (gated and shape[-1] % 2):
        raise _lib.AdkError(f"{what}: x [..., width]{', width even (gate and up halves),' if gated else ''} is required; got {tuple(shape)}")
    width = shape[-1] // 2 if gated else shape[-1]
    return math.prod(shape[:-1]), width


def _names(what, kind, format):
    if kind not in _KINDS:
        raise _lib.AdkError(f"{what}: kind is gelu, gelu_tanh or silu; got {kind!r}")
    if format not in _FORMATS:
        raise _lib.AdkError(f"{what}: format is int8 or e4m3; got {format!r}")


def _forward(x, kind, gated, format, keep):
    """-> (act(x), x as Packed8 or None without `keep`)."""
    _names("activation8", kind, format)
    if x.dtype not in _DTYPES or not x.is_contiguous():
        raise _lib.AdkError(f"activation8: a contiguous float16, bfloat16 or float32 tensor is required; got {x.dtype}, strides {x.stride()}")
    rows, width = _rows_width("activation8", x.shape, gated)
    if not x.is_cuda:
        _lib.require_cuda(x)
    shape, dtype, device = x.shape, x.dtype, x.device
    blocks = -(-x.numel() // 32)
    y = torch.empty((*shape[:-1], width), dtype=dtype, device=device)
    codes = torch.empty(32 * blocks, dtype=torch.uint8, device=device) if keep else None
    units = torch.empty(blocks, dtype=torch.uint8, device=device) if keep else None
    _lib.launch(_lib.load().adk_activation8_fwd, "adk_activation8_fwd", device, x.data_ptr(), _DTYPES[dtype], rows, width, _KINDS[kind], gated, _FORMATS[format],
                y.data_ptr(), _lib.ptr(codes), _lib.ptr(units))
    return y, Packed8(codes, units, shape, dtype, format) if keep else None


def activation8_forward(x, *, kind="gelu", gated=False, format="int8"):
    """-> (act(x), or act(gate) * up for x's halves, in x's type; x as Packed8), outside autograd.  x contiguous, float16, bfloat16 or
    float32, fewer than 2^35 values.  Infinities are held as the format's largest value in their block, NaN as NaN."""
    return _forward(x, kind, gated, format, True)


def activation8_backward(grad, packed, *, kind="gelu", gated=False, again=True):
    """The gradient of activation8_forward's result from its Packed8 -> (dx, the activation of the held values or None without `again`).
    grad of the result's shape and type."""
    _names("activation8_backward", kind, packed.format)
    codes, units, pshape, dtype, format = packed
    rows, width = _rows_width("activation8_backward", pshape, gated)
    shape, device = (*pshape[:-1], width), grad.device
    if grad.shape != shape or grad.dtype != dtype:
        raise _lib.AdkError(f"activation8_backward: grad {shape} {dtype} is required; got {tuple(grad.shape)} {grad.dtype}")
    blocks = -(-rows * width * (2 if gated else 1) // 32)
    if (codes.dtype != torch.uint8 or units.dtype != torch.uint8 or codes.numel() < 32 * blocks or units.numel() < blocks or not codes.is_contiguous()
            or not units.is_contiguous() or codes.device != device or units.device != device or codes.data_ptr() & 7 or dtype not in _DTYPES):
        raise _lib.AdkError("activation8_backward: packed is not what activation8_forward returned, on grad's device")
    if not grad.is_cuda:
        _lib.require_cuda(grad)
    grad = grad.contiguous()
    dx = torch.empty(pshape, dtype=dtype, device=device)
    y = torch.empty(shape, dtype=dtype, device=device) if again else None
    _lib.launch(_lib.load().adk_activation8_bwd, "adk_activation8_bwd", device, grad.data_ptr(), codes.data_ptr(), units.data_ptr(), _DTYPES[dtype], rows, width,
                _KINDS[kind], gated, _FORMATS[format], dx.data_ptr(), _lib.ptr(y))
    return dx, y


class _Activation8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, gated, format):
        y, packed = activation8_forward(x, kind=kind, gated=gated, format=format)
        ctx.save_for_backward(packed.codes, packed.units)
        ctx.how = (packed.shape, packed.dtype, format, kind, gated)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        shape, dtype, format, kind, gated = ctx.how
        dx, _ = activation8_backward(grad, Packed8(*ctx.saved_tensors, shape, dtype, format), kind=kind, gated=gated, again=False)
        return dx, None, None, None


def activation8(x, *, kind="gelu", gated=False, format="int8") -> torch.Tensor:
    """activation8_forward's result as part of autograd, which keeps x in 8 bits (nothing where no gradient is recorded)."""
    if not _lib.differentiated(x):
        return _forward(x, kind, gated, format, False)[0]
    return _Activation8.apply(x, kind, gated, format)


class _Mlp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, kind, gated, format):
        y, packed = activation8_forward(F.linear(x, w1, b1), kind=kind, gated=gated, format=format)
        ctx.save_for_backward(x, w1, w2, packed.codes, packed.units)
        ctx.how = (packed.shape, packed.dtype, format, kind, gated)
        return F.linear(y, w2, b2)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w1, w2, codes, units = ctx.saved_tensors
        shape, dtype, format, kind, gated = ctx.how
        nx, nw1, nb1, nw2, nb2 = ctx.needs_input_grad[:5]
        g2 = grad.reshape(-1, grad.shape[-1])
        dx = dw1 = db1 = dw2 = None
        with torch.autocast(grad.device.type, enabled=False):  # all of one type: the products are to stay in it
            if nx or nw1 or nb1 or nw2:
                dh, y = activation8_backward(torch.mm(g2, w2).view(*shape[:-1], w2.shape[1]), Packed8(codes, units, shape, dtype, format), kind=kind, gated=gated, again=nw2)
                dh = dh.view(-1, dh.shape[-1])
                dx = torch.mm(dh, w1).view(x.shape) if nx else None
                dw1 = torch.mm(dh.t(), x.reshape(-1, x.shape[-1])) if nw1 else None
                db1 = dh.sum(0) if nb1 else None
                dw2 = torch.mm(g2.t(), y.view(-1, y.shape[-1])) if nw2 else None
            return dx, dw1, db1, dw2, g2.sum(0) if nb2 else None, None, None, None


def mlp8(x, w1, b1, w2, b2, *, kind="gelu", gated=False, format="int8") -> torch.Tensor:
    """act(x w1^T + b1) w2^T + b2 (gated: w1's outputs are gate and up halves), keeping x and 8 bits a hidden value for the backward pass.
    x, weights and biases (or None) of one type; under autocast of any, and taken in autocast's, as linear layers are.  The four products of the
    gradient are the library's."""
    given, device = (x, w1, b1, w2, b2), x.device.type
    if torch.is_autocast_enabled(device):
        dtype = torch.get_autocast_dtype(device)
        given = tuple(t.to(dtype) if t is not None and t.dtype in _DTYPES else t for t in given)
    if any(t is not None and t.dtype != given[0].dtype for t in given):
        raise _lib.AdkError(f"mlp8: x, weights and biases are of one type; got {', '.join('none' if t is None else str(t.dtype) for t in given)}")
    with torch.autocast(device, enabled=False):
        if not _lib.differentiated(*(t for t in given if t is not None)):
            return F.linear(_forward(F.linear(*given[:3]), kind, gated, format, False)[0], *given[3:])
        return _Mlp8.apply(*given, kind, gated, format)
