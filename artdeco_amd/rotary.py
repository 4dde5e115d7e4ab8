"""Rotary positions beside `curope.rope_2d` (csrc/rotary.hip): any number of axes, a part of the head, both layouts, long contexts,
out of place or in place, and differentiable.

Channels [2 P a, 2 P (a + 1)) of a head, P = len(frequencies), turn by positions[..., a]: pair (u, v) by the angle positions *
frequencies[m] becomes factor * (u cos - v sin, v cos + u sin).  `curope.rope_2d` (croco/models/curope/kernels.cu:17-108) is
rotary_ with two axes, layout "half" and frequencies base^(-m / P).  The angle is formed in 64 bits, so positions of a million keep
their turn."""
from __future__ import annotations

import math
from array import array

import torch

from artdeco_amd import _lib

_DTYPES = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}
_LAYOUTS = {"half": 1, "interleaved": 0}


def rotary_frequencies(rotary_dim, *, axes=1, base=10000.0, scaling="none", scale_factor=1.0, trained_length=None, fast=32.0, slow=1.0, device=None):
    """-> (frequencies float64 [rotary_dim / (2 axes)], factor): base^(-m / P) for pair m of P, fitted to contexts scale_factor times the
    trained length.

    scaling "none"; "linear": every frequency / scale_factor; "ntk": base * scale_factor^(2P / (2P - 2)), which leaves the first pair as
    it is and divides the last by scale_factor; "by_parts": pairs that turn more than `fast` times within trained_length stay, those
    below `slow` turns are divided by scale_factor, the ones between are mixed along the logarithm of their turns, and cosine and
    sine get the factor 0.1 ln(scale_factor) + 1."""
    if rotary_dim < 2 or axes < 1 or rotary_dim % (2 * axes):
        raise _lib.AdkError(f"rotary_frequencies: rotary_dim is a multiple of 2 * axes; got {rotary_dim} and {axes} axes")
    if not base > 0 or not scale_factor > 0:
        raise _lib.AdkError("rotary_frequencies: base and scale_factor are positive")
    pairs = rotary_dim // (2 * axes)
    if scaling == "ntk":
        base = base * scale_factor ** (2 * pairs / max(1, 2 * pairs - 2))
    f = torch.pow(torch.tensor(float(base), dtype=torch.float64), -torch.arange(pairs, dtype=torch.float64) / pairs)
    factor = 1.0
    if scaling == "linear":
        f = f / scale_factor
    elif scaling == "by_parts":
        if not trained_length or not fast > slow > 0:
            raise _lib.AdkError("rotary_frequencies: by_parts needs trained_length and fast > slow > 0")
        turns = trained_length * f / (2 * math.pi)
        keep = ((turns.log() - math.log(slow)) / (math.log(fast) - math.log(slow))).clamp(0.0, 1.0)
        f = f * keep + f / scale_factor * (1 - keep)
        factor = 0.1 * math.log(scale_factor) + 1.0 if scale_factor > 1 else 1.0
    elif scaling not in ("none", "ntk"):
        raise _lib.AdkError(f"rotary_frequencies: scaling is none, linear, ntk or by_parts; got {scaling!r}")
    return f.to(device), factor


def _turn(x, y, positions, frequencies, factor, layout, heads, transpose):
    """The kernel's call: y may be x."""
    if x.dim() != 4:
        raise _lib.AdkError(f"rotary: x [B,N,H,D] is required; got {tuple(x.shape)}")
    B, N, H, D = x.shape
    if x.dtype not in _DTYPES:
        raise _lib.AdkError(f"rotary: float16, bfloat16 and float32 are supported; got {x.dtype}")
    if D > 1 and x.stride(3) != 1:
        raise _lib.AdkError("rotary: x needs a dense last dimension")
    if y is x and any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
        raise _lib.AdkError("rotary_: x has elements that share their place")
    if layout not in _LAYOUTS:
        raise _lib.AdkError(f"rotary: layout is half or interleaved; got {layout!r}")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or not frequencies.is_contiguous() or frequencies.numel() == 0:
        raise _lib.AdkError("rotary: frequencies is a contiguous float64 vector, one entry a pair")
    if positions.dtype != torch.int64:
        raise _lib.AdkError(f"rotary: positions are int64; got {positions.dtype}")
    if positions.dim() == 3:
        p = positions
    elif positions.dim() in (1, 2):
        p = positions.unsqueeze(-1)
    else:
        raise _lib.AdkError("rotary: positions [N], [B,N] or [B,N,axes]")
    axes = p.shape[-1]
    if tuple(p.shape[-3:-1]) not in ((B, N), (1, N), (N,)) or axes < 1:
        raise _lib.AdkError(f"rotary: positions of shape {tuple(positions.shape)} do not fit x {tuple(x.shape)}")
    if 2 * axes * frequencies.numel() > D:
        raise _lib.AdkError(f"rotary: {axes} axes of {frequencies.numel()} pairs do not fit heads of {D}")
    heads = H if heads is None else heads
    if not 0 <= heads <= H:
        raise _lib.AdkError(f"rotary: {heads} of {H} heads to turn")
    device = x.device
    if device != positions.device or device != frequencies.device:
        raise _lib.AdkError("rotary: all tensors are on one device")
    _lib.require_cuda(x)
    pb, pn, pa = p.stride()[-3:] if p.dim() == 3 else (0, *p.stride())
    if p.dim() == 3 and p.shape[0] == 1:
        pb = 0
    held = array("q", (*_strides(x), *_strides(y), pb, pn, pa))  # alive until the call returns
    lib = _lib.load()
    with _lib.on_device(device):
        rc = lib.adk_rotary(x.data_ptr(), y.data_ptr(), positions.data_ptr(), frequencies.data_ptr(), _DTYPES[x.dtype], B, N, H, D, heads, frequencies.numel(),
                            axes, _LAYOUTS[layout], transpose, factor, held.buffer_info()[0], _lib.stream_of(x))
    _lib.check(rc, "adk_rotary")
    return y


def _strides(t):
    """Element strides of (batch, token, head); a dimension of one element has none that matters."""
    a, b, c = t.shape[:3]
    x, y, z, _ = t.stride()
    return (x if a > 1 else 0, y if b > 1 else 0, z if c > 1 else 0)


def _recorded(x):
    return torch.is_grad_enabled() and x.requires_grad


def _new(x, positions, frequencies, factor, layout, heads, transpose):
    if x.dim() != 4 or x.dtype not in _DTYPES:
        raise _lib.AdkError(f"rotary: x [B,N,H,D] is required, float16, bfloat16 and float32 are supported; got {tuple(x.shape)} {x.dtype}")
    return _turn(x, torch.empty(x.shape, dtype=x.dtype, device=x.device), positions, frequencies, factor, layout, heads, transpose)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, frequencies, factor, layout, heads, transpose, inplace):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (factor, layout, heads, transpose)
        if inplace:
            ctx.mark_dirty(x)
            return _turn(x, x, positions, frequencies, factor, layout, heads, transpose)
        return _new(x, positions, frequencies, factor, layout, heads, transpose)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        positions, frequencies = ctx.saved_tensors
        factor, layout, heads, transpose = ctx.how
        if grad.shape[-1] > 1 and grad.stride(-1) != 1:
            grad = grad.contiguous()
        grad = _new(grad, positions, frequencies, factor, layout, heads, not transpose)
        return (grad,) + (None,) * 7


def rotary(x, positions, frequencies, *, factor=1.0, layout="half", heads=None) -> torch.Tensor:
    """x [B,N,H,D] (float16, bfloat16 or float32, dense last dimension) with the first `heads` heads (all if None) turned, as a new
    contiguous tensor; the other channels and heads are copied.  positions int64 [N], [B,N] or [B,N,axes].  Differentiable."""
    if not _recorded(x):
        return _new(x, positions, frequencies, factor, layout, heads, False)
    return _Rotary.apply(x, positions, frequencies, factor, layout, heads, False, False)


def rotary_(x, positions, frequencies, *, factor=1.0, layout="half", heads=None) -> torch.Tensor:
    """rotary in place: what is not turned is not touched.  -> x."""
    return _Rotary.apply(x, positions, frequencies, factor, layout, heads, False, True)


def rotary_transpose(x, positions, frequencies, *, factor=1.0, layout="half", heads=None) -> torch.Tensor:
    """The transpose of rotary, which is the gradient's form: the same pairs turned back, times factor."""
    if not _recorded(x):
        return _new(x, positions, frequencies, factor, layout, heads, True)
    return _Rotary.apply(x, positions, frequencies, factor, layout, heads, True, False)
