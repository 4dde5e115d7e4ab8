"""The fp16 gradients of attend over fp16's range: what a row or a key gets is held to its own size, whatever the sizes of V, of the gradients
of other rows and of other sequences.

Errors are measured in the 2-norm over a row's (or a key's) channels, against the formulas in 64 bits.  Tolerance, u = 2^-11 half a step:
  dS    each of the terms of dQ_i = scale sum_j dS_ij k_j is rounded on its own, by at most u |dS_ij| in fp16's normal range and by 2^-25 of the
        unit's step below it; roundings of different terms do not know of each other, so their squares add.  The unit brings 2 |dO| |v| to
        2^15, with at most 2.5 places lost to whole exponents: 2^-25 / 2^12.5, below 2^-37 of |dO| |v|, the row's |dO| for dQ, the key head's
        largest for dK, the key head's largest |v|
  delta is taken of the rounded out (probabilities and result, u each, their squares add; 2^-25 below the normal range): an error that a
        row's terms share
  32 bits  2^-19 of the probabilities, 2^-21 of the products, shared by a row's terms
  dV    as dQ, of P^T dO, P held to u or 2^-39
  and u of the result, or 2^-25."""
import math

import pytest
import torch

U = 2.0 ** -11


def norm_tolerances(q, k, v, do, lengths=None, mask=None):
    """q, do [B,H,Nq,D], k / v [B,Hk,Nk,D] -> {name: (value, tolerance of the 2-norm over D)}, float64 on the CPU."""
    B, H, Nq, D = q.shape
    Hk, Nk = k.shape[1:3]
    G, scale = H // Hk, D ** -0.5
    q, k, v, g = (t.double().cpu() for t in (q, k, v, do))
    see = torch.ones(B, 1, 1, Nk, dtype=torch.bool)
    if lengths is not None:
        see = see & (torch.arange(Nk)[None] < lengths.cpu()[:, None])[:, None, None]
    if mask is not None:
        see = see & mask.cpu()
    gone = ~see[:, :, 0, :, None].expand(B, 1, Nk, 1)
    k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    p = torch.softmax((q @ kk.transpose(2, 3) * scale).masked_fill(~see, -math.inf), -1)
    o, dp = p @ vv, g @ vv.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    squares = lambda a, b: (a * a) @ (b * b)  # noqa: E731
    tol_o = (U * U * (squares(p, vv) + o * o)).sqrt() + 2.0 ** -25
    shared = ((g * tol_o) ** 2).sum(-1, keepdim=True).sqrt() + 2.0 ** -21 * g.norm(dim=-1, keepdim=True) * vv.norm(dim=-1).amax(-1)[..., None, None]
    grad, value = g.norm(dim=-1), v.norm(dim=-1).amax(-1).repeat_interleave(G, 1)          # [B,H,Nq], [B,H]
    heads = lambda t: t.view(B, Hk, G, *t.shape[2:]).sum(2)  # noqa: E731
    top = grad.view(B, Hk, -1).amax(-1).repeat_interleave(G, 1)
    off = lambda floor: U * U * ds * ds + torch.where(see, floor * floor, 0.0)  # noqa: E731
    dq, dk, dv = scale * (ds @ kk), scale * heads(ds.transpose(2, 3) @ q), heads(p.transpose(2, 3) @ g)
    eq = scale * ((off(2.0 ** -37 * (grad * value[..., None])[..., None]) @ kk ** 2).sum(-1).sqrt() + shared[..., 0] * (p @ kk).norm(dim=-1)
                  + 2.0 ** -19 * (ds.abs() @ kk.abs()).norm(dim=-1))
    ek = scale * (heads(off(2.0 ** -37 * (top * value)[..., None, None]).transpose(2, 3) @ q ** 2).sum(-1).sqrt()
                  + heads((p * shared).transpose(2, 3) @ q.abs() + 2.0 ** -19 * ds.abs().transpose(2, 3) @ q.abs()).norm(dim=-1))
    held = U * U * p * p + torch.where(see, 2.0 ** -78, 0.0)
    ev = heads(held.transpose(2, 3) @ g ** 2).sum(-1).sqrt() + 2.0 ** -19 * heads(p.transpose(2, 3) @ g.abs()).norm(dim=-1)
    own = lambda t: U * t.norm(dim=-1) + 2.0 ** -25 * D ** 0.5  # noqa: E731
    return {"dq": (dq, eq + own(dq)), "dk": (dk, ek + own(dk)), "dv": (dv, ev + own(dv))}


def gradients(q, k, v, do, **how):
    from artdeco_amd import attention as att
    B, H, Nq, D = q.shape
    flat = do.transpose(1, 2).reshape(B, Nq, H * D)
    out, lse = att.attend_forward(q, k, v, **how)
    return dict(zip(("dq", "dk", "dv"), att.attend_backward(flat, q, k, v, out, lse, **how)))


def check(got, want, names=("dq", "dk", "dv"), shows=None):
    """shows: the tolerance that a typical row (or key) may have at most, relative to what it holds (the test is worth nothing above)."""
    for name in names:
        value, tol = want[name]
        off = (got[name].double().cpu() - value).norm(dim=-1)
        assert bool((off <= tol).all()), (name, float((off / tol).max()), float((off / value.norm(dim=-1)).median()))
        if shows:
            assert float((tol / value.norm(dim=-1)).median()) <= shows, name


def tensors(B, H, Hk, Nq, Nk, D, dev, seed):
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(B, H, Nq, D, generator=g) for _ in range(2))
    k, v = (torch.randn(B, Hk, Nk, D, generator=g) for _ in range(2))
    return [t.half().to(dev) for t in (q, k, v, do)]


@pytest.mark.gpu
@pytest.mark.parametrize("Nk,size", [(8192, 0.01), (768, 0.001), (768, 1.0), (300, 2000.0)])
def test_sizes_of_v(Nk, size, dev):
    """Values far from 1: dS = P (dO v - delta) goes with them."""
    q, k, v, do = tensors(1, 2, 1, 70, Nk, 64, dev, seed=1)
    v = v * size
    check(gradients(q, k, v, do), norm_tolerances(q, k, v, do), names=("dq", "dk"), shows=4e-3)


@pytest.mark.gpu
def test_values_along_the_gradient(dev):
    """Two keys whose values of 1024 run along and against the gradient, D 128: dP is 128 x 1024 times |dO|, the true dS about 6."""
    g = torch.Generator().manual_seed(2)
    way = torch.where(torch.rand(128, generator=g) < 0.5, -1.0, 1.0)
    q, k, v, do = tensors(1, 1, 1, 40, 2, 128, dev, seed=3)
    v = torch.stack([1024 * way, -1024 * way])[None, None].half().to(dev)
    do = (1e-4 * way * (1 + torch.rand(1, 1, 40, 1, generator=g))).half().to(dev)
    check(gradients(q, k, v, do), norm_tolerances(q, k, v, do), shows=4e-3)


@pytest.mark.gpu
def test_hidden_and_padded_values_do_not_count(dev):
    """What a mask over keys hides, and what lies behind a length, leaves the others' gradients as they are: large numbers, infinities, NaN."""
    q, k, v, do = tensors(2, 4, 2, 50, 700, 64, dev, seed=4)
    v = v * 0.001
    lengths = torch.tensor([700, 300], dtype=torch.int32, device=dev)
    mask = torch.ones(2, 1, 1, 700, dtype=torch.bool, device=dev)
    mask[0, :, :, 100:110] = False
    for bad in (6e4, math.inf, math.nan):
        v[0, :, 100:110] = bad
        v[1, :, 300:] = bad
        check(gradients(q, k, v, do, mask=mask, key_lengths=lengths), norm_tolerances(q, k, v, do, lengths, mask), names=("dq", "dk"), shows=4e-3)


@pytest.mark.gpu
def test_a_gradient_that_is_not_finite_stays_in_its_row(dev):
    q, k, v, do = tensors(1, 2, 1, 90, 2000, 64, dev, seed=5)
    do = do * 1e-3
    want = norm_tolerances(q, k, v, do)
    others = torch.arange(90) != 17
    for bad in (math.inf, math.nan):
        do[0, 1, 17, 3] = bad
        got = gradients(q, k, v, do)
        assert bool(torch.isnan(got["dq"][0, 1, 17]).all())
        value, tol = want["dq"]
        off = (got["dq"].double().cpu() - value).norm(dim=-1)[:, :, others]
        assert bool((off <= tol[:, :, others]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("Nk", [1031, 8192])
def test_rows_of_unequal_gradients(Nk, dev):
    """Rows, heads and sequences whose gradients differ by 1e-4, 37 rows a head, so that no 16 rows end with one: each row's dQ to its own size,
    dK to its key head's."""
    q, k, v, do = tensors(3, 4, 2, 37, Nk, 64, dev, seed=6)
    size = torch.ones(3, 4, 37, 1)
    size[:, :, 1::2] = 1e-2
    size[:, :, 2::3] = 1e-4
    size[1] *= 1e-3
    size[:, 3] *= 1e-1
    do = (do.cpu() * size).half().to(dev)
    got = gradients(q, k, v, do)
    check(got, norm_tolerances(q, k, v, do))
    value, tol = norm_tolerances(q, k, v, do)["dq"]
    large = value.norm(dim=-1) > 1e-4  # the rest is near the end of fp16's range as a result
    assert float((tol / value.norm(dim=-1))[large].median()) <= 4e-3


@pytest.mark.gpu
def test_a_sequence_beside_one_of_large_gradients(dev):
    """The same bits alone and in the batch (calls this small are cut alike)."""
    q, k, v, do = tensors(2, 4, 2, 37, 400, 64, dev, seed=7)
    do[0] *= 1e-3
    do[1] *= 1e3
    both = gradients(q, k, v, do)
    alone = gradients(*(t[:1] for t in (q, k, v, do)))
    assert all(torch.equal(both[n][:1], alone[n]) for n in both)


@pytest.mark.gpu
@pytest.mark.parametrize("Nk", [1031, 8192])
def test_a_row_of_a_huge_gradient_beside_others(Nk, dev):
    """One row's gradient is 3e5 times the others': their dQ keeps the accuracy that it has without that row."""
    q, k, v, do = tensors(1, 2, 1, 70, Nk, 64, dev, seed=9)
    do *= 0.05
    do[0, 1, 33] = (do[0, 1, 33].float() * 3e5).half()
    check(gradients(q, k, v, do), norm_tolerances(q, k, v, do), names=("dq",), shows=4e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("Nk", [40000, 300001])
def test_probabilities_of_many_keys(Nk, dev):
    """An even softmax over so many keys that each probability lies below fp16's normal range."""
    q, k, v, do = tensors(1, 1, 1, 40, Nk, 64, dev, seed=8)
    do = do * 1000
    check(gradients(q, k, v, do), norm_tolerances(q, k, v, do), names=("dv",), shows=2e-3)
