"""softmax(q k^T / sqrt(D)) v for the MASt3R blocks on the hand-written gfx950 kernel (csrc/attention.hip).

Arithmetic of croco/models/blocks.py:105-109 / :150-155 (the reference materialises the N x N matrix in fp32/TF32; here the
operands are fp16 and scores, softmax and accumulation fp32 -- the model's "TF32-class" mode).  Returns the result already in
the [B, N, H*D] layout blocks.py:109 produces with `.transpose(1, 2).reshape(B, N, C)`."""
from __future__ import annotations

import ctypes
import math
from array import array

import torch

from artdeco_amd import _lib


def supported(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> bool:
    """fp16 CUDA tensors [B,H,N,64] whose last dim is dense and whose other strides / base addresses allow 128-bit loads."""
    for t in (q, k, v):
        if not (t.is_cuda and t.dtype == torch.float16 and t.dim() == 4 and t.shape[-1] == 64 and t.stride(3) == 1):
            return False
        if any(s % 8 for s in t.stride()[:3]) or t.data_ptr() % 16:
            return False
    return q.shape[:2] == k.shape[:2] == v.shape[:2] and k.shape[2] == v.shape[2] and q.shape[2] > 0 and k.shape[2] > 0


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """q [B,H,Nq,64], k / v [B,H,Nk,64] (any views accepted by `supported`) -> [B, Nq, H*64] float16."""
    if not supported(q, k, v):
        raise _lib.AdkError("adk_attention_fwd_f16: float16 CUDA tensors [B,H,N,64] with a dense last dim, strides that are "
                            "multiples of 8 elements and 16-byte aligned storage are required")
    B, H, Nq, D = q.shape
    Nk = k.shape[2]
    out = torch.empty(B, Nq, H * D, dtype=torch.float16, device=q.device)
    lib = _lib.load()
    i3 = ctypes.c_int64 * 3
    with torch.cuda.device(q.device):
        rc = lib.adk_attention_fwd_f16(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, Nq, Nk,
                                       i3(*q.stride()[:3]), i3(*k.stride()[:3]), i3(*v.stride()[:3]),
                                       float(scale if scale is not None else 1.0 / math.sqrt(D)), _lib.stream_of(q))
    _lib.check(rc, "adk_attention_fwd_f16")
    return out


# ---------------------------------------------------------------------------------------------------------------------------
# Attention with its gradient (csrc/attend.hip): what training the blocks, or answering token by token, needs beside the kernel
# above.  fp16 or bf16, head sizes 8 .. 128 (multiples of 8), several query heads to a key head, causal order, a length for each
# sequence, a free boolean mask.
#
# Where both do (fp16, head size 64, no gradient): `attention` is a little faster for one image's tokens, which is what the frontend asks for (768
# tokens x 16 heads 10.4 against 10.9 us; 192 x 12 4.9, 5.4) and keeps its bits; attend_forward from two images on (2 x 768: 14.2 against 19.1; 8192
# tokens x 16 heads: 356, 564).
#
# What is held in fewer than 32 bits: probabilities, rounded to the operands' type for the products with v and dout; dS, for those with k and q; delta
# is taken of the rounded out.  Each is a rounding of half a step (fp16 2^-11, bf16 2^-8) of its term; fp16 holds them in powers of two that keep them
# off both ends of its range.
_DTYPES = {torch.float16: 0, torch.bfloat16: 2}


def _strides(t: torch.Tensor):
    """Element strides of the first three dimensions; a dimension of one element has none that matters."""
    a, b, c = t.shape[:3]
    x, y, z = t.stride()[:3]
    return (x if a > 1 else 0, y if b > 1 else 0, z if c > 1 else 0)


def _prepare(what, q, k, v, scale, mask, key_lengths):
    """-> (scale, mask broadcast to [B, H, Nq, Nk] or None, the strides of q, k, v and the mask); raises AdkError for what the kernels do
    not take.  The usual call passes one test; _refuse says what is wrong with another."""
    try:
        B, H, Nq, D = q.shape
        Bk, Hk, Nk, Dk = kshape = k.shape
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        plain = (Bk == B and Dk == D and v.shape == kshape and Hk > 0 and H > 0 and H % Hk == 0 and not D & 7 and 8 <= D <= 128 and q.dtype in _DTYPES
                 and q.dtype == k.dtype == v.dtype and q.device == k.device == v.device and qs[3] == ks[3] == vs[3] == 1
                 and not (qs[0] | qs[1] | qs[2] | ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & 7 and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15)
    except ValueError:
        plain = False
    if not plain or (qs[2] | ks[2] | vs[2]) >> 24:  # (a single token far from the next is no matter)
        _refuse(what, q, k, v)
        B, H, Nq, D = q.shape
        Nk = k.shape[2]
        qs, ks, vs = _strides(q), _strides(k), _strides(v)
    if (B | H | Nq | Nk) >> 31:
        raise _lib.AdkError(f"{what}: batch, heads and tokens are counted in 31 bits; got q {tuple(q.shape)}, k {tuple(k.shape)}")
    if scale is None:
        scale = D ** -0.5
    elif not 0.0 < scale < 1e37:
        raise _lib.AdkError(f"{what}: scale is a positive number below 1e37; got {scale}")
    if key_lengths is not None and (key_lengths.dtype != torch.int32 or key_lengths.shape != (B,) or not key_lengths.is_contiguous() or key_lengths.device != q.device):
        raise _lib.AdkError(f"{what}: key_lengths is a contiguous int32 tensor of the batch's size on q's device")
    if mask is None:
        ms = (0, 0, 0, 0)
    else:
        if mask.dtype != torch.bool or mask.device != q.device:
            raise _lib.AdkError(f"{what}: mask is a boolean tensor on q's device, True where a query sees a key (biases that are added to the scores are not "
                                "supported)")
        try:
            mask = mask.broadcast_to(B, H, Nq, Nk)
        except RuntimeError:
            raise _lib.AdkError(f"{what}: mask of shape {tuple(mask.shape)} does not broadcast to {(B, H, Nq, Nk)}") from None
        ms = [0 if n == 1 else s for n, s in zip(mask.shape, mask.stride())]
    if not q.is_cuda:
        _lib.require_cuda(q)
    return scale, mask, (*qs[:3], *ks[:3], *vs[:3], *ms)


def _refuse(what, q, k, v):
    if not (q.dim() == k.dim() == v.dim() == 4):
        raise _lib.AdkError(f"{what}: q [B,H,Nq,D], k and v [B,Hk,Nk,D] are required")
    B, H, Nq, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D or k.shape[1] == 0 or H == 0 or H % k.shape[1]:
        raise _lib.AdkError(f"{what}: k and v [B,Hk,Nk,D] of q's batch and head size, Hk dividing q's {H} heads, are required; got q {tuple(q.shape)}, "
                            f"k {tuple(k.shape)}, v {tuple(v.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise _lib.AdkError(f"{what}: q, k and v are float16 or bfloat16, all of one type; got {q.dtype}, {k.dtype}, {v.dtype}")
    if D % 8 or not 8 <= D <= 128:
        raise _lib.AdkError(f"{what}: head sizes 8 to 128, multiples of 8, are supported; got {D}")
    if not q.device == k.device == v.device:
        raise _lib.AdkError(f"{what}: all tensors are on one device; got {q.device}, {k.device}, {v.device}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        a, b, c = _strides(t)
        if t.numel() and (t.stride(3) != 1 or (a | b | c) & 7 or t.data_ptr() & 15):
            raise _lib.AdkError(f"{what}: {name} needs a dense last dimension, strides that are multiples of 8 elements and 16-byte aligned storage")


def _workspace(nbytes, what, device):
    if nbytes <= 0:
        _lib.check(nbytes, what)
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def attend_forward(q, k, v, *, scale=None, causal=False, mask=None, key_lengths=None):
    """softmax(scale q k^T) v over the keys that each query sees -> (out [B,Nq,H*D] in q's type, lse [B,H,Nq] float32), outside
    autograd.  q [B,H,Nq,D], k / v [B,Hk,Nk,D], any views with a dense last dimension; query head h reads key head h * Hk // H.

    scale        positive, 1/sqrt(D) if None.
    causal       query i sees keys j <= i + Nk - Nq (the last query sees every key).
    key_lengths  int32 [B]: sequence b has keys below key_lengths[b] (clamped to 0 .. Nk).  What lies behind is never read.
    mask         bool, broadcastable to [B,H,Nq,Nk], True where a query sees a key; what it hides from a query has to hold finite
                 numbers (for fp16 gradients, v of not much more than the others' size), unless the mask is the same for all queries and heads.
    All three hold together.  A query that sees no key gives zeros and lse = -inf; the queries of a padded sequence are all computed."""
    scale, mask, strides = _prepare("attend_forward", q, k, v, scale, mask, key_lengths)
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1], k.shape[2]
    dtype, device = q.dtype, q.device
    held = array("q", strides)  # alive until the call returns
    out = torch.empty((B, Nq, H * D), dtype=dtype, device=device)
    lse = torch.empty((B, H, Nq), dtype=torch.float32, device=device)
    lib = _lib.load()
    ws, nbytes = _workspace(lib.adk_attend_fwd_workspace_bytes(B, H, Hk, Nq, Nk, D), "adk_attend_fwd", device)
    _lib.launch(lib.adk_attend_fwd, "adk_attend_fwd", device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _lib.ptr(key_lengths),
                _lib.ptr(mask), _DTYPES[dtype], B, H, Hk, Nq, Nk, D, held.buffer_info()[0], scale, causal, _lib.ptr(ws), nbytes)
    return out, lse


def _backward_into(grad_out, q, k, v, out, lse, scale, causal, mask, key_lengths, strides, dq, dk, dv):
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1], k.shape[2]
    a, b, c = grad_out.stride()
    g = (a if B > 1 else 0, D if H > 1 else 0, b if Nq > 1 else 0)
    if (c != 1 or (g[0] | g[2]) & 7 or grad_out.data_ptr() & 15) and grad_out.numel():  # an expanded gradient, of a sum for instance
        grad_out = grad_out.contiguous()
        grad_out = grad_out.clone() if grad_out.data_ptr() & 15 else grad_out
        g = (Nq * H * D, D, H * D)
    device = q.device
    lib = _lib.load()
    held = array("q", (*strides, *g, *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3]))
    nbytes = lib.adk_attend_bwd_workspace_bytes(B, H, Hk, Nq, Nk, D)
    if mask is not None and nbytes > 0:
        nbytes += lib.adk_attend_mask_bytes(B, H, Nq, Nk, held.buffer_info()[0] + 72)  # strides: the mask's come after q's, k's and v's
    ws, nbytes = _workspace(nbytes, "adk_attend_bwd", device)
    _lib.launch(lib.adk_attend_bwd, "adk_attend_bwd", device, grad_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                _lib.ptr(key_lengths), _lib.ptr(mask), _DTYPES[q.dtype], B, H, Hk, Nq, Nk, D, held.buffer_info()[0], scale, causal, dq.data_ptr(), dk.data_ptr(),
                dv.data_ptr(), _lib.ptr(ws), nbytes)


def attend_backward(grad_out, q, k, v, out, lse, *, scale=None, causal=False, mask=None, key_lengths=None):
    """The gradient of attend_forward's out, called with the same arguments and what it returned -> (dq, dk, dv) in the shapes and
    the type of q, k and v ([B,N,heads,D] in memory).  grad_out [B,Nq,H*D].  The heads that share a key head are summed in 32 bits, in a
    fixed order; keys behind a sequence's length get zeros."""
    scale, mask, strides = _prepare("attend_backward", q, k, v, scale, mask, key_lengths)
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1], k.shape[2]
    dtype, device, shape = q.dtype, q.device, (B, Nq, H * D)
    if not (grad_out.shape == shape and out.shape == shape and lse.shape == (B, H, Nq) and grad_out.dtype == out.dtype == dtype and lse.dtype == torch.float32
            and grad_out.device == out.device == lse.device == device):
        raise _lib.AdkError(f"attend_backward: grad_out and out {shape} {dtype} and lse {(B, H, Nq)} float32 on {device} are required; got {tuple(grad_out.shape)} "
                            f"{grad_out.dtype}, {tuple(out.shape)} {out.dtype}, {tuple(lse.shape)} {lse.dtype}")
    out, lse = out.contiguous(), lse.contiguous()
    if out.data_ptr() & 15:
        out = out.clone()
    like = ((Nq * H * D, D, H * D, 1), (Nk * Hk * D, D, Hk * D, 1))
    dq = torch.empty_strided((B, H, Nq, D), like[0], dtype=dtype, device=device)
    dk = torch.empty_strided((B, Hk, Nk, D), like[1], dtype=dtype, device=device)
    dv = torch.empty_strided((B, Hk, Nk, D), like[1], dtype=dtype, device=device)
    _backward_into(grad_out, q, k, v, out, lse, scale, causal, mask, key_lengths, strides, dq, dk, dv)
    return dq, dk, dv


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, mask, key_lengths):
        out, lse = attend_forward(q, k, v, scale=scale, causal=causal, mask=mask, key_lengths=key_lengths)
        ctx.save_for_backward(q, k, v, out, lse, mask, key_lengths)
        ctx.how = (scale, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, mask, key_lengths = ctx.saved_tensors
        scale, causal = ctx.how
        dq, dk, dv = attend_backward(grad_out, q, k, v, out, lse, scale=scale, causal=causal, mask=mask, key_lengths=key_lengths)
        return dq, dk, dv, None, None, None, None


def attend(q, k, v, *, scale=None, causal=False, mask=None, key_lengths=None) -> torch.Tensor:
    """attend_forward's out as part of autograd: differentiable once with respect to q, k and v, in reverse mode (forward-mode
    differentiation raises torch's error).  -> [B,Nq,H*D].

    A training step that is captured into a graph is captured whole, while no graph of the same leaves recorded outside it is alive
    (autograd would wait for the stream that one was recorded on, which ends the capture); attend_forward and attend_backward have no
    such tie."""
    if not _lib.differentiated(q, k, v):
        return attend_forward(q, k, v, scale=scale, causal=causal, mask=mask, key_lengths=key_lengths)[0]
    return _Attend.apply(q, k, v, scale, causal, mask, key_lengths)


def _packed_views(qkv, heads, kv_heads):
    t = qkv.transpose(1, 2)
    return t[:, :heads], t[:, heads:heads + kv_heads], t[:, heads + kv_heads:]


class _AttendPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, kv_heads, scale, causal, mask, key_lengths):
        q, k, v = _packed_views(qkv, heads, kv_heads)
        out, lse = attend_forward(q, k, v, scale=scale, causal=causal, mask=mask, key_lengths=key_lengths)
        ctx.save_for_backward(qkv, out, lse, mask, key_lengths)
        ctx.how = (heads, kv_heads, scale, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        qkv, out, lse, mask, key_lengths = ctx.saved_tensors
        heads, kv_heads, scale, causal = ctx.how
        q, k, v = _packed_views(qkv, heads, kv_heads)
        scale, mask, strides = _prepare("attend_packed", q, k, v, scale, mask, key_lengths)
        grad = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _backward_into(grad_out, q, k, v, out, lse, scale, causal, mask, key_lengths, strides, *_packed_views(grad, heads, kv_heads))
        return grad, None, None, None, None, None, None


def attend_packed(qkv, heads, kv_heads=None, *, scale=None, causal=False, mask=None, key_lengths=None) -> torch.Tensor:
    """attend on the heads of one projection, qkv [B,N,heads + 2 kv_heads,D] (q's heads, then k's, then v's): the gradient arrives in
    one tensor of that shape, where three views of qkv would each be padded to it and added up.  -> [B,N,heads*D]."""
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.dim() != 4 or heads < 1 or kv_heads < 1 or qkv.shape[2] != heads + 2 * kv_heads:
        raise _lib.AdkError(f"attend_packed: qkv [B,N,heads + 2 kv_heads,D] is required; got {tuple(qkv.shape)} for {heads} and {kv_heads} heads")
    if not _lib.differentiated(qkv):
        return attend_forward(*_packed_views(qkv, heads, kv_heads), scale=scale, causal=causal, mask=mask, key_lengths=key_lengths)[0]
    return _AttendPacked.apply(qkv, heads, kv_heads, scale, causal, mask, key_lengths)
