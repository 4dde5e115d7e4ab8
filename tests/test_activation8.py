"""activation8 / mlp8 (csrc/activation8.hip): codes and units exactly as defined, values and gradients against the formulas in 64 bits.

Tolerance: half a step of the type on the result plus, for the 32-bit function values (erf, exponential, reciprocal: each within 2^-21
of the function or, for erf, of 1), 2^-20 of the factors' size."""
import math

import pytest
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def codes_of(x, fmt):
    """-> (the values that the codes stand for, units' exponents), by the definition, float64."""
    flat = torch.nn.functional.pad(x.double().cpu().reshape(-1), (0, -x.numel() % 32)).view(-1, 32)
    size = flat.abs()
    top = torch.where(torch.isfinite(size), size, 0.0).amax(1)
    most = 127.0 if fmt == "int8" else 448.0
    e = torch.full(top.shape, -126.0, dtype=torch.float64)
    for n in range(-126, 128):
        e = torch.where(top > most * 2.0 ** n, torch.tensor(float(n + 1), dtype=torch.float64), e)
    w = flat / torch.exp2(e)[:, None]
    w = torch.where(torch.isinf(w), torch.sign(w) * most, w)
    if fmt == "int8":
        r = torch.round(w)
    else:
        step = torch.exp2(torch.floor(torch.log2(w.abs().clamp(min=2.0 ** -6))) - 3)
        r = torch.round(w / step) * step
    return (r * torch.exp2(e)[:, None]).reshape(-1)[:x.numel()].view(x.shape), e


def decode(packed):
    n = 1
    for s in packed.shape:
        n *= s
    c, u = packed.codes.cpu(), packed.units.cpu()
    if packed.format == "int8":
        v = c.view(torch.int8).double()
        v = torch.where(v == -128, math.nan, v)
    else:
        v = c.view(torch.float8_e4m3fn).double()
    return (v.view(-1, 32) * torch.exp2(u.double() - 127)[:, None]).view(-1)[:n].view(packed.shape)


def act(x, kind):
    f = {"gelu": torch.nn.functional.gelu, "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"), "silu": torch.nn.functional.silu}[kind]
    return f(x)


def slope(z, kind):
    z = z.clone().requires_grad_(True)
    g, = torch.autograd.grad(act(z, kind).sum(), z)
    return g


def close(got, want, size, dtype):
    tol = U[dtype] * want.abs() + 2.0 ** -20 * size + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    assert bool(((got.double().cpu() - want).abs() <= tol).all()), float(((got.double().cpu() - want).abs() - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("kind,gated", [("gelu", False), ("gelu_tanh", False), ("silu", False), ("silu", True), ("gelu", True)])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (5, 33), (3, 7, 40), (257, 1000), (64, 4096)], ids=str)
def test_forward_codes_and_backward(shape, kind, gated, fmt, dtype, dev):
    from artdeco_amd import activation8 as a8
    g = torch.Generator().manual_seed(sum(shape))
    W = shape[-1]
    x = torch.randn(*shape[:-1], W * (2 if gated else 1), generator=g) * torch.exp2(torch.randint(-6, 4, (*shape[:-1], 1), generator=g).float())
    x = x.to(dtype).to(dev)
    grad = torch.randn(shape, generator=g).to(dtype).to(dev)
    y, packed = a8.activation8_forward(x, kind=kind, gated=gated, format=fmt)
    held, e = codes_of(x, fmt)
    assert torch.equal(packed.units.cpu().double(), e + 127) and torch.equal(decode(packed), held)
    dx, again = a8.activation8_backward(grad, packed, kind=kind, gated=gated)
    assert a8.activation8_backward(grad, packed, kind=kind, gated=gated, again=False)[1] is None
    xd, gd = x.double().cpu(), grad.double().cpu()
    if gated:
        close(y, act(xd[..., :W], kind) * xd[..., W:], (xd[..., :W] * xd[..., W:]).abs(), dtype)
        z, up = held[..., :W], held[..., W:]
        close(again, act(z, kind) * up, (z * up).abs(), dtype)
        close(dx[..., :W], gd * up * slope(z, kind), (gd * up).abs() * (1 + z.abs()), dtype)
        close(dx[..., W:], gd * act(z, kind), (gd * z).abs(), dtype)
    else:
        close(y, act(xd, kind), xd.abs(), dtype)
        close(again, act(held, kind), held.abs(), dtype)
        close(dx, gd * slope(held, kind), gd.abs() * (1 + held.abs()), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_zeros_tiny_huge_and_not_finite(fmt, dev):
    from artdeco_amd import activation8 as a8
    x = torch.zeros(9, 32)
    x[1] = torch.linspace(-1e-38, 1e-38, 32)
    x[2] = torch.linspace(-3e38, 3e38, 32)
    x[3, 3], x[3, 4], x[3, 5] = math.inf, -math.inf, 2.0
    x[4, 0], x[4, 1] = math.nan, 1.0
    x[5, 0], x[5, 1], x[5, 2] = 448.0, 127.0, 126.5                              # the formats' largest, a tie
    x[6, 0], x[6, 1:9] = 448.0, torch.tensor([17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 17.001, 18.999])  # ties to even, the smallest steps
    x[7, 0], x[7, 1] = 127.0, 2.5
    x[8, 0] = float(torch.nextafter(torch.tensor(448.0), torch.tensor(500.0)))
    y, packed = a8.activation8_forward(x.to(dev), kind="silu", format=fmt)
    held, e = codes_of(x, fmt)
    got = decode(packed)
    assert torch.equal(packed.units.cpu().double(), e + 127)
    assert bool(torch.isnan(got[4, 0])) and float(got[4, 1]) == 1.0
    torch.testing.assert_close(got, held, rtol=0, atol=0, equal_nan=True)        # the second row's steps overflow: infinities and NaN too
    dx, again = a8.activation8_backward(torch.ones(9, 32, device=dev), packed, kind="silu")
    assert bool(torch.isfinite(dx[3]).all()) and bool(torch.isnan(dx[4, 0])) and float(dx[0, 0]) == 0.5 and float(again[0, 0]) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_whose_squares_are_infinite(kind, dtype, dev):
    """Far out the slope is 1 or 0; each value in a block of its own unit."""
    from artdeco_amd import activation8 as a8
    x = torch.zeros(8, 32)
    x[:, 0] = torch.tensor([1e19, -1e19, 2e19, -2e19, 1e25, -1e25, 1e37, -1e37])
    y, packed = a8.activation8_forward(x.to(dtype).to(dev), kind=kind)
    dx, again = a8.activation8_backward(torch.ones(8, 32, dtype=dtype, device=dev), packed, kind=kind)
    z = decode(packed)
    close(dx, slope(z, kind), torch.ones_like(z), dtype)
    close(again, act(z, kind), z.abs(), dtype)
    close(y, act(x.to(dtype).double(), kind), x.double().abs(), dtype)


@pytest.mark.gpu
def test_rows_of_odd_width_at_odd_addresses(dev):
    """A contiguous tensor whose storage starts between 16-byte lines."""
    from artdeco_amd import activation8 as a8
    g = torch.Generator().manual_seed(3)
    room = torch.randn(7 * 26 + 3, generator=g).to(torch.bfloat16).to(dev)
    x = room[3:].view(7, 26)
    want = a8.activation8_forward(x.clone(), gated=True, format="e4m3")
    got = a8.activation8_forward(x, gated=True, format="e4m3")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].codes[:182], want[1].codes[:182])
    grad = torch.randn(7 * 13 + 1, generator=g).to(torch.bfloat16).to(dev)[1:].view(7, 13)
    for a, b in zip(a8.activation8_backward(grad, got[1], gated=True), a8.activation8_backward(grad.clone(), want[1], gated=True)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_in_autograd_and_empty(dev):
    from artdeco_amd import activation8 as a8
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 50, generator=g).to(dev).requires_grad_(True)
    grad = torch.randn(3, 25, generator=g).to(dev)
    gx, = torch.autograd.grad(a8.activation8(x, kind="gelu_tanh", gated=True, format="e4m3"), x, grad)
    _, packed = a8.activation8_forward(x.detach(), kind="gelu_tanh", gated=True, format="e4m3")
    assert torch.equal(gx, a8.activation8_backward(grad, packed, kind="gelu_tanh", gated=True)[0])
    gx, = torch.autograd.grad(a8.activation8(x).sum(), x)
    assert gx.shape == x.shape
    y, packed = a8.activation8_forward(x.detach()[:0])
    assert y.shape == (0, 50) and a8.activation8_backward(y, packed)[0].shape == (0, 50)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_mlp8(gated, dev):
    """Output as the plain layers give it; gradients those of the layers with the hidden values replaced by the held ones, in 64 bits.
    float32 products of at most 96 terms: within 96 * 2^-23 of the terms' sizes, twice through two layers."""
    from artdeco_amd import activation8 as a8
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 9, 32, generator=g).to(dev)
    w1, b1 = torch.randn(96 * (2 if gated else 1), 32, generator=g).to(dev) * 0.2, torch.randn(96 * (2 if gated else 1), generator=g).to(dev)
    w2, b2 = torch.randn(24, 96, generator=g).to(dev) * 0.2, torch.randn(24, generator=g).to(dev)
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    out = a8.mlp8(*leaves, kind="silu", gated=gated)
    grad = torch.randn(2, 9, 24, generator=g).to(dev)
    got = torch.autograd.grad(out, leaves, grad)
    h = torch.nn.functional.linear(x, w1, b1).detach()
    held = decode(a8.activation8_forward(h, kind="silu", gated=gated)[1])
    d = [t.detach().double().cpu() for t in (x, w1, b1, w2, b2)]
    z = held.requires_grad_(True)
    f = lambda t: act(t[..., :96], "silu") * t[..., 96:] if gated else act(t, "silu")  # noqa: E731
    w2d = d[3].clone().requires_grad_(True)
    gd = grad.double().cpu()
    dz, dw2 = torch.autograd.grad(f(z) @ w2d.t(), (z, w2d), gd)
    want = (dz @ d[1], dz.flatten(0, 1).t() @ d[0].flatten(0, 1), dz.flatten(0, 1).sum(0), dw2, gd.flatten(0, 1).sum(0))
    ref = f(torch.nn.functional.linear(d[0], d[1], d[2])) @ d[3].t() + d[4]
    for a, b in zip((out, *got), (ref, *want)):
        assert a.shape == b.shape and float((a.detach().double().cpu() - b).abs().max()) <= 2 * 96 * 2.0 ** -23 * float(b.abs().max()) * 4
    none = a8.mlp8(x, w1, None, w2, None, kind="silu", gated=gated)
    assert len(torch.autograd.grad(none, (x, w1, w2), grad)) == 3


@pytest.mark.gpu
def test_captured_graph(dev):
    from artdeco_amd import activation8 as a8
    x = torch.randn(40, 100, device=dev).half()
    grad = torch.randn(40, 100, device=dev).half()

    def once():
        y, p = a8.activation8_forward(x)
        return (y, p.codes[:4000], p.units, *a8.activation8_backward(grad, p))
    once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for turn in range(3):
        x.copy_(torch.randn(40, 100, device=dev))
        want = once()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_refusals(lib):
    from artdeco_amd import _lib, activation8 as a8
    x = torch.zeros(4, 6)

    def no(text, *a, **kw):
        with pytest.raises(_lib.AdkError, match=text):
            a8.activation8_forward(*a, **kw)
    no("CPU tensor", x)
    no("kind", x, kind="relu")
    no("format", x, format="e5m2")
    no("contiguous", x.t())
    no("contiguous", x.double())
    no("width", torch.zeros(4, 5), gated=True)
    no("width", torch.zeros(()))
    p = a8.Packed8(torch.zeros(32, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), (4, 6), torch.float32, "int8")

    def back(text, grad, packed, **kw):
        with pytest.raises(_lib.AdkError, match=text):
            a8.activation8_backward(grad, packed, **kw)
    back("CPU tensor", x, p)
    back("grad", x[:3], p)
    back("grad", x.half(), p)
    back("grad", x, p, gated=True)
    back("format", x, p._replace(format="int4"))
    back("not what", x, p._replace(codes=torch.zeros(24, dtype=torch.uint8)))
    back("not what", x, p._replace(units=torch.zeros(1)))
    N = None
    assert lib.adk_activation8_fwd(N, 3, 1, 1, 0, 0, 0, N, N, N, N) == -3 and lib.adk_activation8_fwd(N, 0, 1, 1, 3, 0, 0, N, N, N, N) == -3
    assert lib.adk_activation8_fwd(N, 0, -1, 1, 0, 0, 0, N, N, N, N) == -1 and lib.adk_activation8_fwd(N, 0, 1, 1, 0, 0, 0, N, N, N, N) == -1
    assert lib.adk_activation8_fwd(N, 0, 0, 1, 0, 0, 0, N, N, N, N) == 0
    assert lib.adk_activation8_bwd(N, N, N, 0, 1, 1, 0, 0, 2, N, N, N) == -3 and lib.adk_activation8_bwd(N, N, N, 0, 1, 1, 0, 0, 0, N, N, N) == -1
