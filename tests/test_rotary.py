"""rotary / rotary_ / rotary_transpose / rotary_frequencies (csrc/rotary.hip) against complex multiplication in 64 bits.

Tolerance: half a step of the type on the result, plus 2^-21 (|u| + |v|) factor for cosine, sine and the two products in 32 bits (each
below 2^-23), plus the type's smallest step."""
import math

import pytest
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def formula(x, positions, f, factor, layout, heads, sign):
    x = x.double().cpu()
    B, N, H, D = x.shape
    p = positions.cpu()
    p = p if p.dim() == 3 else p[..., None]
    p = p.broadcast_to(B, N, p.shape[-1])
    A, P = p.shape[-1], len(f)
    heads = H if heads is None else heads
    y, size = x.clone(), torch.zeros_like(x)
    for a in range(A):
        seg = slice(2 * P * a, 2 * P * (a + 1))
        z = x[:, :, :heads, seg]
        u, v = (z[..., :P], z[..., P:]) if layout == "half" else (z[..., ::2], z[..., 1::2])
        angle = sign * p[:, :, None, a, None].double() * f.cpu()
        c = torch.complex(u, v) * torch.polar(torch.full_like(angle, factor), angle)
        m = (u.abs() + v.abs()) * factor
        both = (torch.cat([c.real, c.imag], -1), torch.cat([m, m], -1)) if layout == "half" else (torch.stack([c.real, c.imag], -1).flatten(-2), torch.stack([m, m], -1).flatten(-2))
        y[:, :, :heads, seg], size[:, :, :heads, seg] = both
    return y, size


def check(got, x, positions, f, factor, layout, heads, sign):
    want, size = formula(x, positions, f, factor, layout, heads, sign)
    tol = U[x.dtype] * want.abs() + 2.0 ** -21 * size + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    tol = torch.where(size > 0, tol, 0.0)  # what is not turned is copied
    assert got.dtype == x.dtype and bool(((got.double().cpu() - want).abs() <= tol).all()), float(((got.double().cpu() - want).abs() - tol).max())


CASES = [  # B, N, H, D, rotary_dim, axes, heads
    (1, 1, 1, 2, 2, 1, None), (2, 5, 3, 20, 12, 1, 2), (1, 768, 48, 64, 64, 2, 32), (3, 33, 6, 128, 64, 1, 5), (2, 17, 4, 96, 96, 3, None), (8, 1, 40, 128, 128, 1, 33),
    (1, 3001, 2, 256, 192, 1, 1), (2, 9, 5, 72, 72, 1, 0), (1, 4, 200, 128, 16, 1, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_turns_and_turns_back(case, layout, dtype, dev):
    from artdeco_amd import rotary as ro
    B, N, H, D, R, A, heads = case
    g = torch.Generator().manual_seed(N + D)
    x = torch.randn(B, N, H, D, generator=g).to(dtype).to(dev)
    pos = torch.randint(-50, 1000000, (B, N, A), generator=g).to(dev)
    f, factor = ro.rotary_frequencies(R, axes=A, scaling="by_parts", scale_factor=4.0, trained_length=2048, device=dev)
    how = dict(factor=factor, layout=layout, heads=heads)
    keep = x.clone()
    check(ro.rotary(x, pos, f, **how), x, pos, f, factor, layout, heads, 1)
    check(ro.rotary_transpose(x, pos, f, **how), x, pos, f, factor, layout, heads, -1)
    assert torch.equal(x, keep)
    y = x.clone()
    version = y._version
    assert ro.rotary_(y, pos, f, **how) is y and torch.equal(y, ro.rotary(x, pos, f, **how)) and y._version > version


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_positions_and_alignment(layout, dev):
    """Views with odd strides and bases, head-major tensors, positions shared by a batch or the axes apart in memory: what a contiguous call gives."""
    from artdeco_amd import rotary as ro
    B, N, H, D = 2, 11, 4, 64
    g = torch.Generator().manual_seed(0)
    x = torch.randn(B, N, H, D, generator=g).half().to(dev)
    pos = torch.randint(0, 5000, (B, N), generator=g).to(dev)
    f, _ = ro.rotary_frequencies(32, device=dev)
    want = ro.rotary(x, pos, f, layout=layout)
    wide = torch.zeros(B, N, H, D + 3, dtype=x.dtype, device=dev)
    wide[..., 1:D + 1] = x
    head_major = x.transpose(1, 2).contiguous().transpose(1, 2)
    for v in (wide[..., 1:D + 1], head_major):
        assert torch.equal(ro.rotary(v, pos, f, layout=layout), want)
        ro.rotary_(v, pos, f, layout=layout)
        assert torch.equal(v, want)
    assert not wide[..., 0].any() and not wide[..., D + 1:].any()
    assert torch.equal(ro.rotary(x, pos[0], f, layout=layout), ro.rotary(x, pos[:1].expand(B, N), f, layout=layout))
    apart = torch.stack([pos, pos + 1]).permute(1, 2, 0)
    assert torch.equal(ro.rotary(x, apart, f[:16], layout=layout), ro.rotary(x, apart.contiguous(), f[:16], layout=layout))
    assert ro.rotary(x[:, :0], pos[:, :0], f).shape == (B, 0, H, D)


@pytest.mark.gpu
def test_is_rope_2d_with_two_axes(dev):
    """The model's in-place rotation: angles there are 32-bit, positions below 32, so the two agree to a few 32-bit steps."""
    import curope
    from artdeco_amd import rotary as ro
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 768, 16, 64, generator=g).to(dev)
    pos = torch.randint(0, 32, (1, 768, 2), generator=g).to(dev)
    f, _ = ro.rotary_frequencies(64, axes=2, base=100.0, device=dev)
    want = x.clone()
    curope.rope_2d(want, pos, 100.0, 1.0)
    # an angle below 32 is off by 2^-24 of itself for each of its three roundings (power, division, product)
    assert float((ro.rotary(x, pos, f) - want).abs().max()) <= 4 * 32 * 2.0 ** -24 * float(x.abs().max()) * 2


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
def test_gradient(inplace, dev):
    from artdeco_amd import rotary as ro
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 7, 5, 32, generator=g).to(dev).requires_grad_(True)
    pos = torch.randint(0, 100, (2, 7), generator=g).to(dev)
    f, _ = ro.rotary_frequencies(16, device=dev)
    go = torch.randn(2, 7, 5, 32, generator=g).to(dev)
    turn = ro.rotary_ if inplace else ro.rotary
    y = turn(x * 1.0, pos, f, factor=1.5, heads=3)
    gx, = torch.autograd.grad(y, x, go)
    assert torch.equal(gx, ro.rotary_transpose(go, pos, f, factor=1.5, heads=3))
    # <rotary(x), go> is linear in x: its slope along any direction is <direction, gradient>
    way = torch.randn(2, 7, 5, 32, generator=g).to(dev)
    slope = float((formula(way.detach(), pos, f, 1.5, "half", 3, 1)[0] * go.double().cpu()).sum())
    assert abs(slope - float((gx.double() * way.double()).sum())) <= 2.0 ** -20 * float((gx.double() * way.double()).abs().sum())
    gx, = torch.autograd.grad(turn(x * 1.0, pos, f).sum(), x)                # an expanded gradient
    assert torch.equal(gx, ro.rotary_transpose(torch.ones_like(go), pos, f))
    if inplace:                                                              # on a view of a projection, whose base autograd follows
        base = x * 1.0
        ro.rotary_(base.view(2, 7, 5, 32), pos, f)
        gx, = torch.autograd.grad(base, x, go)
        assert torch.equal(gx, ro.rotary_transpose(go, pos, f))


@pytest.mark.gpu
def test_stream_and_captured_graph(dev):
    from artdeco_amd import rotary as ro
    x = torch.randn(4, 33, 6, 64, device=dev).half()
    pos = torch.arange(33, device=dev) + 70000
    f, _ = ro.rotary_frequencies(64, device=dev)
    want = ro.rotary(x, pos, f)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ro.rotary(x, pos, f)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ro.rotary(x, pos, f)
    for turn in range(3):
        x.copy_(torch.randn(4, 33, 6, 64, device=dev))
        pos.add_(1)
        want = ro.rotary(x, pos, f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), turn


def test_frequencies():
    from artdeco_amd import _lib, rotary as ro
    f, factor = ro.rotary_frequencies(8, base=10000.0)
    assert factor == 1.0 and f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    lin, _ = ro.rotary_frequencies(8, scaling="linear", scale_factor=4.0)
    assert torch.allclose(lin, f / 4)
    ntk, _ = ro.rotary_frequencies(8, scaling="ntk", scale_factor=4.0)
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4)
    parts, factor = ro.rotary_frequencies(128, scaling="by_parts", scale_factor=8.0, trained_length=8192)
    plain, _ = ro.rotary_frequencies(128)
    turns = 8192 * plain / (2 * math.pi)
    assert torch.equal(parts[turns > 32], plain[turns > 32]) and torch.allclose(parts[turns < 1], plain[turns < 1] / 8)
    assert bool((parts <= plain).all()) and bool((parts[1:] < parts[:-1]).all()) and math.isclose(factor, 0.1 * math.log(8.0) + 1)
    assert ro.rotary_frequencies(60, axes=3)[0].numel() == 10
    for kw in (dict(rotary_dim=7), dict(rotary_dim=8, axes=3), dict(rotary_dim=8, base=0), dict(rotary_dim=8, scaling="by_parts"), dict(rotary_dim=8, scaling="other")):
        with pytest.raises(_lib.AdkError):
            ro.rotary_frequencies(**kw)


def test_refusals(lib):
    from artdeco_amd import _lib, rotary as ro
    x, pos = torch.zeros(2, 4, 3, 16), torch.zeros(2, 4, dtype=torch.int64)
    f, _ = ro.rotary_frequencies(16)

    def no(text, *a, **kw):
        with pytest.raises(_lib.AdkError, match=text):
            ro.rotary(*a, **kw)
    no("CPU tensor", x, pos, f)
    no("required", x[0], pos, f)
    no("supported", x.double(), pos, f)
    no("dense", torch.zeros(2, 4, 3, 32)[..., ::2], pos, f)
    no("layout", x, pos, f, layout="quarter")
    no("float64", x, pos, f.float())
    no("int64", x, pos.int(), f)
    no("do not fit", x, pos[:, :3], f)
    no("do not fit", x, torch.zeros(2, 4, 2, dtype=torch.int64), f)
    no("to turn", x, pos, f, heads=4)
    with pytest.raises(_lib.AdkError, match="share"):
        ro.rotary_(torch.zeros(1, 4, 3, 16).expand(2, 4, 3, 16), pos, f)
    with pytest.raises(_lib.AdkError, match="leaf"):
        ro.rotary_(torch.zeros(2, 4, 3, 16, requires_grad=True), pos, f)
    N = None
    assert lib.adk_rotary(N, N, N, N, 0, 1, 1, 1, 16, 1, 9, 1, 1, 0, 1.0, N, N) == -1      # 18 channels of 16
    assert lib.adk_rotary(N, N, N, N, 3, 1, 1, 1, 16, 1, 8, 1, 1, 0, 1.0, N, N) == -3
    assert lib.adk_rotary(N, N, N, N, 0, 1, 1, 1, 16, 1, 8, 1, 1, 0, 1.0, N, N) == -1
    assert lib.adk_rotary(N, N, N, N, 0, 0, 1, 1, 16, 1, 8, 1, 1, 0, 1.0, N, N) == 0
