"""attend / attend_forward / attend_backward / attend_packed (csrc/attend.hip) against the formulas in 64 bits.

Tolerances, elementwise, u = half a step of the type (fp16 2^-11, bf16 2^-8), all sums over the visible keys:
  out   every probability is rounded once (u each: u P|v|), the result once (u |o|), 32-bit work below 2e-5 P|v|;
        fp16 probabilities below its normal range are off by at most 2^-25 of the row's largest
  dV    the same with P^T |dO|
  dS    rounded once (u |dS|); delta is taken of the rounded out: P_ij (|dO_i| . (tolerance of out)); 32-bit work below 3e-5 of
        P (|dO| . |v| + |dO| . P|v|); fp16 holds dS in units of the largest |dO|: below its normal range 2^-24 of that
  dQ, dK  scale * (tolerance of dS) |K|, |Q|, and the result's rounding."""
import math

import pytest
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def formulas(q, k, v, do, scale, causal, mask, lengths, u, fp16):
    """-> {name: (value, tolerance)} in float64 on the CPU; q [B,H,Nq,D], k / v [B,Hk,Nk,D], do [B,Nq,H*D]."""
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1:3]
    G = H // Hk
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    see = torch.ones(B, H, Nq, Nk, dtype=torch.bool)
    j = torch.arange(Nk)
    if causal:
        see &= j[None] <= torch.arange(Nq)[:, None] + (Nk - Nq)
    if lengths is not None:
        see &= (j[None] < lengths.cpu()[:, None])[:, None, None]
        gone = (j[None] >= lengths.cpu()[:, None])[:, None, :, None]
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    if mask is not None:
        see &= mask.cpu()
        gone = ~mask.cpu().broadcast_to(B, H, Nq, Nk).any(2).view(B, Hk, G, Nk).any(2)[..., None]  # seen by nobody: its numbers do not matter
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ kk.transpose(2, 3) * scale).masked_fill(~see, -math.inf)
    some = see.any(-1)
    lse = torch.where(some, torch.logsumexp(s, -1), -math.inf) if Nk else torch.full((B, H, Nq), -math.inf, dtype=torch.float64)
    p = torch.where(see, torch.exp(s - torch.where(some, lse, 0.0)[..., None]), 0.0)
    o = p @ vv
    pv = p @ vv.abs()
    size = (q.abs() @ kk.abs().transpose(2, 3) * scale)
    tiny = 2.0 ** -25 if fp16 else 0.0
    tol_o = u * pv + u * o.abs() + 2e-5 * pv + tiny * vv.abs().sum(2, keepdim=True) + 2.0 ** -24 * fp16 + 1e-12
    flat = lambda t: t.transpose(1, 2).reshape(B, Nq, H * D)  # noqa: E731
    got = {"out": (flat(o), flat(tol_o)), "lse": (lse, 2.0 ** -20 * (size.amax(-1) if Nk else torch.zeros_like(lse)) + 1e-6 * lse.abs().nan_to_num(posinf=0.0) + 1e-6)}
    if do is None:
        return got
    g = do.double().cpu().view(B, Nq, H, D).transpose(1, 2)
    pt = p.transpose(2, 3)
    dv, gabs = pt @ g, g.abs()
    dp = g @ vv.transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = u * ds.abs() + p * ((gabs * tol_o).sum(-1, keepdim=True) + 3e-5 * (gabs @ vv.abs().transpose(2, 3) + (gabs * pv).sum(-1, keepdim=True)))
    off = off + torch.where(see, 2.0 ** -24 * float(gabs.max()) if fp16 and gabs.numel() else 0.0, 0.0)
    dq, dk = scale * (ds @ kk), scale * (ds.transpose(2, 3) @ q)
    low = 2.0 ** -24 * fp16 + 1e-12  # the gradient's own smallest step
    heads = lambda t: t.view(B, Hk, G, Nk, D).sum(2)  # noqa: E731
    tol_v = heads((u + 3e-5) * (pt @ gabs) + tiny * gabs.sum(2, keepdim=True))
    got["dq"] = (dq, scale * (off @ kk.abs()) + u * dq.abs() + low)
    got["dk"] = (heads(dk), heads(scale * (off.transpose(2, 3) @ q.abs())) + u * heads(dk).abs() + low)
    got["dv"] = (heads(dv), tol_v + u * heads(dv).abs() + low)
    return got


def check(got, want):
    for name, (value, tol) in want.items():
        t = got[name].double().cpu()
        assert t.shape == value.shape, name
        fine = torch.isfinite(value)
        assert torch.equal(t[~fine], value[~fine]), name
        bad = (t - value).abs() - tol
        assert bool((bad[fine] <= 0).all()), (name, float(bad[fine].max()), float((((t - value).abs() / tol)[fine]).max()))


def inputs(B, H, Hk, Nq, Nk, D, dtype, dev, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(B, Nq, H, D, generator=g) * size for _ in range(2))
    k = torch.randn(B, Nk, Hk, D, generator=g) * size
    # a swapped key order, a transposed tile or a wrong channel shows in v
    v = torch.randn(B, Nk, Hk, D, generator=g) + 0.01 * torch.arange(Nk)[None, :, None, None] % 1.7 + 0.02 * torch.arange(D)
    q, k, v = (t.to(dtype).to(dev).transpose(1, 2) for t in (q, k, v))
    return q, k, v, do.reshape(B, Nq, H * D).to(dtype).to(dev)


def both(q, k, v, do, scale=None, causal=False, mask=None, lengths=None):
    from artdeco_amd import attention as att
    how = dict(scale=scale, causal=causal, mask=mask, key_lengths=lengths)
    out, lse = att.attend_forward(q, k, v, **how)
    dq, dk, dv = att.attend_backward(do, q, k, v, out, lse, **how)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def run(q, k, v, do, **how):
    s = how.pop("scale", None)
    got = both(q, k, v, do, scale=s, **how)
    fp16 = q.dtype == torch.float16
    check(got, formulas(q, k, v, do, s or q.shape[-1] ** -0.5, how.get("causal", False), how.get("mask"), how.get("lengths"), U[q.dtype], fp16))
    return got


SIZES = [  # B, H, Hk, Nq, Nk, D
    (1, 1, 1, 1, 1, 8), (2, 3, 3, 7, 1, 64), (1, 2, 1, 1, 130, 128), (1, 8, 1, 1, 1000, 128), (2, 6, 2, 33, 65, 40), (1, 2, 2, 64, 64, 64), (1, 4, 2, 129, 127, 72),
    (2, 16, 16, 200, 200, 64), (1, 3, 1, 97, 300, 128), (1, 1, 1, 513, 257, 96), (3, 2, 1, 300, 64, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_gradients(size, causal, dtype, dev):
    run(*inputs(*size, dtype, dev, seed=sum(size)), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batch_never_reads_behind_the_lengths(D, causal, dtype, dev):
    """Lengths 0, 1, a tile, inside a tile, all; NaN behind them; lengths outside 0 .. Nk are clamped."""
    B, H, Hk, Nq, Nk = 6, 4, 2, 70, 200
    q, k, v, do = inputs(B, H, Hk, Nq, Nk, D, dtype, dev, seed=3)
    lengths = torch.tensor([0, 1, 64, 131, 999, -5], dtype=torch.int32, device=dev)
    for b, n in enumerate([0, 1, 64, 131, 200, 0]):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
    got = both(q, k, v, do, causal=causal, lengths=lengths)
    want = formulas(q.cpu(), k.cpu(), v.cpu(), do, D ** -0.5, causal, None, lengths.clamp(0, Nk), U[dtype], dtype == torch.float16)
    check(got, want)
    assert float(got["dk"][1, :, 1:].abs().max()) == 0 and float(got["dv"][0].abs().max()) == 0 and float(got["out"][5].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 4, 77, 150), (2, 1, 77, 150), (1, 4, 1, 150), (1, 1, 77, 1), (77, 150)])
def test_free_masks_with_rows_that_see_nothing(shape, dtype, dev):
    q, k, v, do = inputs(2, 4, 2, 77, 150, 64, dtype, dev, seed=5)
    g = torch.Generator().manual_seed(1)
    mask = torch.rand(shape, generator=g) < 0.6
    if shape[-2] > 1:
        mask[..., ::5, :] = False
    run(q, k, v, do, mask=mask.to(dev))
    run(q, k, v, do, mask=mask.to(dev), causal=True, lengths=torch.tensor([150, 40], dtype=torch.int32, device=dev))
    # a mask read through strides: every second byte of a wider one
    wide = torch.zeros(*shape[:-1], 2 * shape[-1], dtype=torch.bool)
    wide[..., ::2] = mask
    run(q, k, v, do, mask=wide.to(dev)[..., ::2])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["batch", "heads", "queries alone", "transposed"])
@pytest.mark.parametrize("size", [(2, 2, 1, 100, 333, 64), (1, 32, 32, 300, 1133, 64), (3, 8, 4, 270, 523, 96), (2, 24, 24, 300, 1133, 96), (1, 12, 12, 290, 777, 128),
                                  (2, 24, 24, 301, 1134, 128)], ids=str)
def test_masks_in_small_and_large_calls(size, kind, dev):
    """More keys than queries, so that a causal call begins inside a word of the mask's bits; from a few workgroups to several for each CU."""
    B, H, Hk, Nq, Nk, D = size
    q, k, v, do = inputs(*size, torch.bfloat16, dev, seed=7)
    g = torch.Generator().manual_seed(2)
    shape = {"batch": (B, 1, Nq, Nk), "heads": (1, H, Nq, Nk), "queries alone": (B, 1, Nq, 1), "transposed": (B, 1, Nk, Nq)}[kind]
    mask = (torch.rand(shape, generator=g) < 0.7).to(dev)
    mask = mask.transpose(2, 3) if kind == "transposed" else mask
    run(q, k, v, do, mask=mask, causal=kind != "heads")


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["whole", "causal", "lengths and mask"])
@pytest.mark.parametrize("size", [(1, 8, 1, 2100, 7, 64), (2, 4, 2, 16, 4100, 96), (1, 16, 2, 900, 150, 128), (1, 1, 1, 2001, 1999, 40), (2, 20, 20, 128, 2100, 128),
                                  (1, 12, 12, 1, 3000, 64), (1, 2, 1, 4000, 1, 8)], ids=str)
def test_few_keys_or_few_queries_beside_many(size, how, dev):
    """Walks that are cut into parts and joined: of the keys' owners, of the rows', of both."""
    B, H, Hk, Nq, Nk, D = size
    q, k, v, do = inputs(*size, torch.bfloat16 if D > 64 else torch.float16, dev, seed=11)
    mask = lengths = None
    if how == "lengths and mask":
        g = torch.Generator().manual_seed(4)
        mask = (torch.rand(1, 1, Nq, Nk, generator=g) < 0.8).to(dev)
        lengths = torch.tensor([Nk // 3, Nk][:B], dtype=torch.int32, device=dev)
    first = run(q, k, v, do, causal=how == "causal", mask=mask, lengths=lengths)
    again = both(q, k, v, do, causal=how == "causal", mask=mask, lengths=lengths)
    assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_mask_over_keys_alone_hides_what_is_not_finite(bad, dev):
    q, k, v, do = inputs(2, 4, 2, 50, 100, 64, torch.bfloat16, dev, seed=8)
    mask = torch.ones(2, 1, 1, 100, dtype=torch.bool, device=dev)
    mask[0, :, :, 30:41] = False
    mask[1, :, :, 99:] = False
    k[0, :, 30:41] = bad
    v[0, :, 30:41] = bad
    v[1, :, 99:] = -bad
    run(q, k, v, do, mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sharp_scores_and_scale(dtype, dev):
    run(*inputs(1, 2, 2, 130, 300, 64, dtype, dev, seed=9, size=4.0), scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** 13])
def test_fp16_gradients_of_small_and_of_scaled_losses(size, dev):
    """dS of a gradient of 6e-5 would fall below fp16's normal range, of 8000 leave it: the tolerance stays relative to the gradient's size."""
    q, k, v, do = inputs(1, 2, 1, 100, 260, 64, torch.float16, dev, seed=10)
    do = (do.float().clamp(-3, 3) * size).half()
    v = v * 0.25
    run(q, k, v, do)


@pytest.mark.gpu
def test_no_keys_and_no_queries(dev):
    from artdeco_amd import attention as att
    for Nq, Nk, B in ((5, 0, 2), (0, 5, 2), (0, 0, 2), (5, 5, 0)):
        for dtype in (torch.float16, torch.bfloat16):
            q, k, v, do = inputs(B, 4, 2, Nq, Nk, 64, dtype, dev, seed=1)
            got = both(q, k, v, do)
            assert got["out"].shape == (B, Nq, 256) and got["dk"].shape == (B, 2, Nk, 64)
            if Nk == 0 or B == 0:
                assert not got["out"].any() and not got["dq"].any() and bool((got["lse"] == -math.inf).all())
            if Nq == 0:
                assert not got["dk"].any() and not got["dv"].any()
    q = torch.zeros(2, 4, 5, 64, device=dev, dtype=torch.float16, requires_grad=True)
    k = torch.zeros(2, 4, 0, 64, device=dev, dtype=torch.float16, requires_grad=True)
    att.attend(q, k, k).sum().backward()
    assert not q.grad.any() and k.grad.shape == k.shape


@pytest.mark.gpu
def test_few_rows_over_many_keys_split_and_join(dev):
    """Single tokens over long caches: the keys are cut into parts, of which a short sequence leaves most empty."""
    for H, Hk, Nk, D in ((8, 2, 4099, 128), (3, 3, 2000, 64)):
        q, k, v, do = inputs(4, H, Hk, 1, Nk, D, torch.bfloat16, dev, seed=Nk)
        run(q, k, v, do, lengths=torch.tensor([Nk, 1, 0, 700], dtype=torch.int32, device=dev))
    q, k, v, do = inputs(1, 2, 1, 40, 3000, 64, torch.float16, dev, seed=4)
    run(q, k, v, do, causal=True)


@pytest.mark.gpu
def test_layouts_and_strides(dev):
    """Head-major, token-major, views of one projection, a batch stride of zero: the same numbers."""
    B, H, N, D = 2, 4, 90, 64
    q, k, v, do = inputs(B, H, H, N, N, D, torch.float16, dev, seed=12)
    want = both(q, k, v, do)
    other = both(q.contiguous(), k.contiguous(), v.contiguous(), do)
    packed = torch.stack([t.transpose(1, 2) for t in (q, k, v)], 2)
    views = both(*(packed[:, :, i].transpose(1, 2) for i in range(3)), do)
    padded = torch.zeros(B, N, H * D + 8, device=dev, dtype=do.dtype)
    padded[..., :H * D] = do
    for got in (other, views, both(q, k, v, padded[..., :H * D])):
        for name in want:
            assert torch.equal(got[name], want[name]), name
    one_k, one_v = k[:1].expand(B, H, N, D), v[:1].expand(B, H, N, D)
    run(q, one_k, one_v, do)


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """A cache whose tokens lie 2 MiB apart: 8 GiB from the first key to the last, queries likewise; and one whose mask does."""
    room = torch.empty(4200 * 2 ** 20 // 2 * 2, dtype=torch.bfloat16, device=dev)
    q, k, v, do = inputs(1, 4, 2, 3000, 4100, 64, torch.bfloat16, dev, seed=33)
    far_k, far_v = (room[o:].as_strided((1, 2, 4100, 64), (8, 64, 2 ** 20, 1)) for o in (0, 256))
    far_q = room[512:].as_strided((1, 4, 3000, 64), (8, 64, 2 ** 20, 1))
    for a, b in ((far_k, k), (far_v, v), (far_q, q)):
        a.copy_(b)
    want = both(q, k, v, do, causal=True)
    got = both(far_q, far_k, far_v, do, causal=True)
    assert all(torch.equal(got[n], want[n]) for n in want)
    mask = torch.rand(1, 1, 3000, 4100, device=dev) < 0.7
    far_mask = room.view(torch.bool).as_strided((1, 1, 3000, 4100), (1, 1, 2 ** 21 + 2 ** 19, 1))
    far_mask.copy_(mask)
    want, got = both(q, k, v, do, mask=mask), both(q, k, v, do, mask=far_mask)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.gpu
def test_attend_in_autograd(dev):
    """The differentiable forms give attend_backward's gradients: leaves, an expanded incoming gradient, one packed projection, a broadcast
    key tensor whose gradient is summed; twice the same bits; no second derivative."""
    from artdeco_amd import attention as att
    B, H, Hk, N, D = 2, 6, 2, 130, 64
    q, k, v, do = inputs(B, H, Hk, N, N, D, torch.bfloat16, dev, seed=21)
    want = both(q, k, v, do, causal=True)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    out = att.attend(*leaves, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    assert torch.equal(out, want["out"]) and all(torch.equal(g, want[n]) for g, n in zip(grads, ("dq", "dk", "dv")))
    qkv = torch.cat([t.transpose(1, 2) for t in (q, k, v)], 2).contiguous().requires_grad_(True)
    packed = att.attend_packed(qkv, H, Hk, causal=True)
    g, = torch.autograd.grad(packed, qkv, do)
    assert torch.equal(packed, want["out"])
    assert torch.equal(g, torch.cat([want[n].transpose(1, 2) for n in ("dq", "dk", "dv")], 2))
    ones = torch.ones_like(do)
    a = torch.autograd.grad(att.attend(*leaves).sum(), leaves)
    b = both(q, k, v, ones)
    assert all(torch.equal(x, b[n]) for x, n in zip(a, ("dq", "dk", "dv")))
    shared = k[:, :1].detach().clone().requires_grad_(True)
    gk, = torch.autograd.grad(att.attend(q, shared.expand(B, Hk, N, D), v), shared, do)
    full = both(q, shared.detach().expand(B, Hk, N, D), v, do)["dk"]
    assert torch.equal(gk, full.sum(1, keepdim=True))
    with pytest.raises(RuntimeError):
        x = att.attend(*leaves)
        y, = torch.autograd.grad(x.float().square().sum(), leaves[0], create_graph=True)
        torch.autograd.grad(y.float().sum(), leaves[0])


@pytest.mark.gpu
def test_gradient_against_differences(dev):
    """The slope along a direction against the 64-bit loss's difference quotient at the same (rounded) points."""
    q, k, v, do = inputs(1, 4, 2, 20, 30, 32, torch.float16, dev, seed=30)
    got = both(q, k, v, do, causal=True)
    loss = lambda q, k, v: float((formulas(q, k, v, None, 32 ** -0.5, True, None, None, 0.0, True)["out"][0] * do.double().cpu()).sum())  # noqa: E731
    g = torch.Generator().manual_seed(2)
    for i, name in enumerate(("dq", "dk", "dv")):
        at = [t.double().cpu() for t in (q, k, v)]
        way = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * way, at[i] - 1e-5 * way
        slope = (loss(*up) - loss(*down)) / 2e-5
        want = formulas(q, k, v, do, 32 ** -0.5, True, None, None, U[torch.float16], True)[name]
        assert abs(slope - float((got[name].double().cpu() * way).sum())) <= float((want[1] * way.abs()).sum()) + 1e-6 * abs(slope) + 1e-6


@pytest.mark.gpu
def test_streams_and_captured_graphs(dev):
    """On another stream, two calls at once, and captured: replayed with new contents between the eager work, each replay equal to the eager result."""
    sizes = [(1, 8, 2, 1, 3000, 128), (2, 4, 4, 150, 150, 64)]
    cases = [inputs(*s, torch.bfloat16, dev, seed=40 + i) for i, s in enumerate(sizes)]
    want = [both(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got.append(both(*c))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[n], w[n]) for n in w)
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(*c))
        graphs.append(graph)
    for turn in range(4):
        for c, s in zip(cases, sizes):
            for t, n in zip(c, inputs(*s, torch.bfloat16, dev, seed=60 + turn)):
                t.copy_(n)
        want = [both(*c) for c in cases]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(outs, want):
            assert all(torch.equal(g[n], w[n]) for n in w), turn


def test_refusals():
    """Checked before anything reaches the GPU: CPU tensors show each."""
    from artdeco_amd import _lib, attention as att
    ok = dict(dtype=torch.float16)
    q, k = torch.zeros(2, 4, 8, 64, **ok), torch.zeros(2, 2, 8, 64, **ok)

    def no(text, *a, **kw):
        with pytest.raises(_lib.AdkError, match=text):
            att.attend_forward(*a, **kw)
    no("CPU tensor", q, k, k)
    no("required", q[0], k, k)
    no("required", q, k[:, :0], k[:, :0])
    no("required", q, torch.zeros(2, 3, 8, 64, **ok), torch.zeros(2, 3, 8, 64, **ok))
    no("required", q, k, k[:, :, :7])
    no("one type", q.float(), k.float(), k.float())
    no("one type", q, k.bfloat16(), k)
    no("head sizes", q[..., :4], k[..., :4], k[..., :4])
    big = torch.zeros(1, 1, 4, 136, **ok)
    no("head sizes", big, big, big)
    no("dense last", torch.zeros(2, 4, 8, 128, **ok)[..., ::2], k, k)
    no("multiples of 8", torch.zeros(2, 4, 8, 65, **ok)[..., :64], k, k)
    no("scale", q, k, k, scale=0.0)
    no("scale", q, k, k, scale=math.inf)
    no("key_lengths", q, k, k, key_lengths=torch.zeros(2, dtype=torch.int64))
    no("key_lengths", q, k, k, key_lengths=torch.zeros(3, dtype=torch.int32))
    no("boolean", q, k, k, mask=torch.zeros(8, 8))
    no("boolean", q, k, k, mask=torch.full((8, 8), torch.finfo(torch.float16).min, dtype=torch.float16))
    no("broadcast", q, k, k, mask=torch.ones(7, 8, dtype=torch.bool))
    with pytest.raises(_lib.AdkError, match="attend_packed"):
        att.attend_packed(torch.zeros(2, 8, 7, 64, **ok), 4, 2)
    out, lse = torch.zeros(2, 8, 256, **ok), torch.zeros(2, 4, 8)
    for bad in ((out[:, :7], out, lse), (out, out.float(), lse), (out, out, lse.double())):
        with pytest.raises(_lib.AdkError):
            att.attend_backward(bad[0], q, k, k, bad[1], bad[2])


def test_c_entry_refuses_before_any_launch(lib):
    import ctypes
    fine = (ctypes.c_int64 * 25)(*[8] * 25)
    odd = (ctypes.c_int64 * 25)(8, 4, *[8] * 23)
    P = ctypes.c_void_p(1 << 20)
    fwd = lambda q=P, D=64, H=4, Hk=2, Nq=4, dtype=0, s=fine, scale=1.0, out=P, ws=None, n=0: lib.adk_attend_fwd(  # noqa: E731
        q, P, P, out, P, None, None, dtype, 1, H, Hk, Nq, 4096, D, s, scale, 0, ws, n, None)
    assert fwd(D=60) == -3 and fwd(D=256) == -3 and fwd(dtype=1) == -3
    wide = (ctypes.c_int64 * 25)(8, 8, 1 << 24, *[8] * 22)
    assert fwd(s=wide) == -3 and fwd(scale=1e38) == -1
    assert fwd(H=3) == -1 and fwd(scale=0.0) == -1 and fwd(scale=float("nan")) == -1 and fwd(q=None) == -1 and fwd(s=odd) == -1 and fwd(out=None) == -1
    assert fwd(q=ctypes.c_void_p((1 << 20) + 8)) == -1
    assert fwd() == -2 and fwd(ws=P, n=64) == -2
    assert fwd(Nq=0) == 0
    assert lib.adk_attend_fwd_workspace_bytes(1, 4, 2, 4, 4096, 64) > 0 and lib.adk_attend_fwd_workspace_bytes(1, 4, 3, 4, 4, 64) == -1
    assert lib.adk_attend_bwd_workspace_bytes(2, 4, 2, 8, 8, 64) == 4 * (64 + 4)
    per_head, for_keys = (ctypes.c_int64 * 4)(0, 33 * 65, 65, 1), (ctypes.c_int64 * 4)(65, 0, 0, 1)
    assert lib.adk_attend_mask_bytes(2, 4, 33, 65, per_head) == 4 * 4 * (3 * 33 + 2 * 65) and lib.adk_attend_mask_bytes(2, 4, 33, 65, for_keys) == 4 * 2 * (3 + 65)
    assert lib.adk_attend_mask_bytes(2, 4, 0, 65, per_head) == 0 and lib.adk_attend_mask_bytes(2, 4, 33, 65, None) == -1
    masked = (P, P, P, P, P, P, None, P, 0, 1, 4, 2, 4, 4, 64, fine, 1.0, 0, P, P, P, P)  # a workspace without room for the mask's bits
    assert lib.adk_attend_bwd(*masked, lib.adk_attend_bwd_workspace_bytes(1, 4, 2, 4, 4, 64), None) == -2
    assert lib.adk_attend_bwd(P, P, P, P, P, P, None, None, 0, 1, 4, 2, 4, 4, 64, fine, 1.0, 0, P, P, P, None, 0, None) == -2


def test_the_formulas_are_torchs():
    """The checker itself against torch's attention and its gradient, in 64 bits."""
    q, k, v, do = inputs(2, 4, 2, 9, 12, 16, torch.float64, "cpu", seed=2)
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    see = torch.arange(12)[None] <= torch.arange(9)[:, None] + 3
    ref = torch.nn.functional.scaled_dot_product_attention(q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1), attn_mask=see)
    grads = torch.autograd.grad(ref, (q, k, v), do.view(2, 9, 4, 16).transpose(1, 2))
    got = formulas(q.detach(), k.detach(), v.detach(), do, 0.25, True, None, None, 0.0, False)
    assert torch.allclose(got["out"][0], ref.transpose(1, 2).reshape(2, 9, 64))
    assert all(torch.allclose(got[n][0], g) for n, g in zip(("dq", "dk", "dv"), grads))
