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
    """The kernel's call: y is x (in place), or None for a new tensor.  -> y."""
    try:
        B, N, H, D = shape = x.shape
    except ValueError:
        raise _lib.AdkError(f"rotary: x [B,N,H,D] is required; got {tuple(x.shape)}") from None
    dtype, device = x.dtype, x.device
    xb, xn, xh, xd = x.stride()
    if (B | N | H | D) >> 31:
        raise _lib.AdkError(f"rotary: batch, tokens, heads and channels are counted in 31 bits; got {tuple(shape)}")
    if dtype not in _DTYPES:
        raise _lib.AdkError(f"rotary: float16, bfloat16 and float32 are supported; got {dtype}")
    if xd != 1 and D > 1:
        raise _lib.AdkError("rotary: x needs a dense last dimension")
    if layout not in _LAYOUTS:
        raise _lib.AdkError(f"rotary: layout is half or interleaved; got {layout!r}")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or not frequencies.is_contiguous():
        raise _lib.AdkError("rotary: frequencies is a contiguous float64 vector, one entry a pair")
    if positions.dtype != torch.int64:
        raise _lib.AdkError(f"rotary: positions are int64; got {positions.dtype}")
    pshape, pstride = positions.shape, positions.stride()
    if len(pshape) == 3:
        (pB, pN, axes), (pb, pn, pa) = pshape, pstride
    elif len(pshape) == 2:
        (pB, pN), (pb, pn), axes, pa = pshape, pstride, 1, 0
    elif len(pshape) == 1:
        pB, pN, axes, pb, pn, pa = 1, pshape[0], 1, 0, pstride[0], 0
    else:
        raise _lib.AdkError("rotary: positions [N], [B,N] or [B,N,axes]")
    if pN != N or (pB != B and pB != 1) or axes < 1:
        raise _lib.AdkError(f"rotary: positions of shape {tuple(pshape)} do not fit x {tuple(shape)}")
    if pB == 1:
        pb = 0
    pairs = frequencies.shape[0]
    if pairs < 1 or 2 * axes * pairs > D:
        raise _lib.AdkError(f"rotary: {axes} axes of {pairs} pairs do not fit heads of {D}")
    if heads is None:
        heads = H
    elif not 0 <= heads <= H:
        raise _lib.AdkError(f"rotary: {heads} of {H} heads to turn")
    if device != positions.device or device != frequencies.device:
        raise _lib.AdkError("rotary: all tensors are on one device")
    if y is not None and ((xb == 0 and B > 1) or (xn == 0 and N > 1) or (xh == 0 and H > 1)):
        raise _lib.AdkError("rotary_: x has elements that share their place")
    if not x.is_cuda:
        _lib.require_cuda(x)
    # a dimension of one element has no stride that matters
    xb, xn, xh = xb if B > 1 else 0, xn if N > 1 else 0, xh if H > 1 else 0
    if y is None:
        y = torch.empty(shape, dtype=dtype, device=device)
        held = array("q", (xb, xn, xh, N * H * D, H * D, D, pb, pn, pa))  # alive until the call returns
    else:
        held = array("q", (xb, xn, xh, xb, xn, xh, pb, pn, pa))
    _lib.launch(_lib.load().adk_rotary, "adk_rotary", device, x.data_ptr(), y.data_ptr(), positions.data_ptr(), frequencies.data_ptr(), _DTYPES[dtype], B, N, H, D,
                heads, pairs, axes, _LAYOUTS[layout], transpose, factor, held.buffer_info()[0])
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, frequencies, factor, layout, heads, transpose, inplace):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (factor, layout, heads, transpose)
        if inplace:
            ctx.mark_dirty(x)
            return _turn(x, x, positions, frequencies, factor, layout, heads, transpose)
        return _turn(x, None, positions, frequencies, factor, layout, heads, transpose)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        positions, frequencies = ctx.saved_tensors
        factor, layout, heads, transpose = ctx.how
        if grad.shape[-1] > 1 and grad.stride(-1) != 1:
            grad = grad.contiguous()
        grad = _turn(grad, None, positions, frequencies, factor, layout, heads, not transpose)
        return (grad,) + (None,) * 7


def rotary(x, positions, frequencies, *, factor=1.0, layout="half", heads=None) -> torch.Tensor:
    """x [B,N,H,D] (float16, bfloat16 or float32, dense last dimension) with the first `heads` heads (all if None) turned, as a new
    contiguous tensor; the other channels and heads are copied.  positions int64 [N], [B,N] or [B,N,axes].  Differentiable
    (in reverse mode; forward-mode differentiation raises torch's error, as in rotary_ and rotary_transpose)."""
    if not _lib.differentiated(x):
        return _turn(x, None, positions, frequencies, factor, layout, heads, False)
    return _Rotary.apply(x, positions, frequencies, factor, layout, heads, False, False)


def rotary_(x, positions, frequencies, *, factor=1.0, layout="half", heads=None) -> torch.Tensor:
    """rotary in place: what is not turned is not touched.  -> x."""
    if torch.is_grad_enabled() and x.requires_grad:
        # what torch refuses as well, but only when x has been turned
        if x.is_leaf or (x._is_view() and x._base.is_leaf):
            raise _lib.AdkError("rotary_: x is a leaf that requires a gradient, or a view of one: turn it out of place, with rotary")
        if x._is_view() and torch._C._autograd._get_creation_meta(x) != torch._C._autograd.CreationMeta.DEFAULT:
            raise _lib.AdkError("rotary_: x is a view that autograd does not follow in place (one of a split's, or made without grad mode): turn it out of "
                                "place, with rotary")
    return _Rotary.apply(x, positions, frequencies, factor, layout, heads, False, True)


def rotary_transpose(x, positions, frequencies, *, factor=1.0, layout="half", heads=None) -> torch.Tensor:
    """The transpose of rotary, which is the gradient's form: the same pairs turned back, times factor."""
    if not _lib.differentiated(x):
        return _turn(x, None, positions, frequencies, factor, layout, heads, True)
    return _Rotary.apply(x, positions, frequencies, factor, layout, heads, True, False)
