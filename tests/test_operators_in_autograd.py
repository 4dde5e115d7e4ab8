"""attend, rotary, activation8 and the model's blocks as autograd and callers meet them: what is decided on the host, before any launch, with the
launches replaced by a record of them."""
import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    """CPU tensors pass for the GPU's; what would be launched is listed as (entry, arguments), and computes nothing."""
    from artdeco_amd import _lib
    made = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(_lib, "launch", lambda fn, what, device, *args: made.append((what, args)))
    return made


def test_forward_mode_differentiation_is_refused(launches):
    """A dual tensor requires no gradient; passing it by would give a result without a tangent, a constant."""
    import torch.autograd.forward_ad as ad
    from artdeco_amd import activation8 as a8, attention as att, rotary as ro
    f, _ = ro.rotary_frequencies(8)
    x, pos, q = torch.randn(1, 4, 3, 8), torch.arange(4), torch.randn(1, 2, 4, 8).half()
    with ad.dual_level():
        dx, dq = ad.make_dual(x, torch.ones_like(x)), ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: ro.rotary(dx, pos, f), lambda: ro.rotary_transpose(dx, pos, f), lambda: ro.rotary_(dx * 1, pos, f), lambda: att.attend(dq, q, q),
                     lambda: att.attend(q, q, dq), lambda: att.attend_packed(dx.half(), 1), lambda: a8.activation8(dx)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        assert ad.unpack_dual(ro.rotary(x, pos, f)).tangent is None and ad.unpack_dual(att.attend(q, q, q)).tangent is None
    with pytest.raises(Exception, match="jvp|setup_context"):
        torch.func.jvp(lambda t: ro.rotary(t, pos, f), (x,), (x,))
    assert not ro.rotary(x, pos, f).requires_grad and not att.attend(q, q, q).requires_grad
    assert ro.rotary(x.requires_grad_(True), pos, f).requires_grad
    with torch.no_grad():
        assert not ro.rotary(x, pos, f).requires_grad


class Adapted(torch.nn.Linear):
    """A Linear with something beside it, as adapters have it."""
    def __init__(self, inner):
        super().__init__(inner.in_features, inner.out_features)
        self.load_state_dict(inner.state_dict())
        self.called = 0

    def forward(self, x):
        self.called += 1
        return super().forward(x)


@pytest.mark.parametrize("layer", ["fc1", "fc2", "act"])
def test_an_mlp_that_keeps_8_bits_calls_what_hangs_on_its_layers(layer, launches, monkeypatch):
    """Hooks of each kind, an adapter in a layer's place, a forward of its own; without them the layers are one operator."""
    from artdeco_amd import mast3r_model as mm
    monkeypatch.setattr(mm, "_trains", lambda module, x: True)
    x = torch.randn(2, 3, 8, requires_grad=True)

    def fresh():
        mlp = mm.Mlp(8, 16)
        mlp.kept8 = "int8"
        return mlp, getattr(mlp, layer)
    forwards = lambda: [n for n, _ in launches].count("adk_activation8_fwd")  # noqa: E731
    mlp, _ = fresh()
    assert type(mlp(x).grad_fn).__name__ == "_Mlp8Backward" and forwards() == 1
    seen = []
    for hang in (lambda m: m.register_forward_hook(lambda *a: seen.append(1)), lambda m: m.register_forward_pre_hook(lambda *a: seen.append(1)),
                 lambda m: m.register_full_backward_hook(lambda *a: seen.append(1)), lambda m: m.register_full_backward_pre_hook(lambda *a: seen.append(1))):
        mlp, m = fresh()
        seen.clear()
        launches.clear()
        hang(m)
        mlp(x).sum().backward()
        assert seen == [1] and forwards() == (0 if layer == "act" else 1)
    mlp, m = fresh()
    m.forward = lambda t, f=m.forward: (seen.append(2), f(t))[1]
    mlp(x).sum().backward()
    assert seen[-1] == 2
    if layer != "act":
        mlp, m = fresh()
        setattr(mlp, layer, Adapted(m))
        mlp(x).sum().backward()
        assert getattr(mlp, layer).called == 1 and getattr(mlp, layer).weight.grad is not None
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, *a: seen.append(type(m).__name__))
    try:
        seen.clear()
        fresh()[0](x)
        assert {"Linear", "GELU"} <= set(seen)
    finally:
        handle.remove()


def test_mlp8_takes_autocasts_type_and_refuses_a_mixture(launches):
    from artdeco_amd import _lib, activation8 as a8
    x, w1, b1, w2, b2 = (torch.randn(s, requires_grad=True) for s in ((2, 8), (16, 8), (16,), (4, 16), (4,)))
    with torch.autocast("cpu", dtype=torch.bfloat16):
        out = a8.mlp8(x, w1, b1.bfloat16(), w2, b2)
    assert out.dtype == torch.bfloat16
    assert all(g.dtype == torch.float32 for g in torch.autograd.grad(out, (x, w1, w2, b2), torch.ones_like(out)))
    out = a8.mlp8(x, w1, b1, w2, b2)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert all(g.dtype == torch.float32 for g in torch.autograd.grad(out, (x, w1, b1, w2, b2), torch.ones_like(out)))
    for bad in ((x.half(), w1, b1, w2, b2), (x, w1, b1, w2.double(), b2), (x, w1, b1, w2, b2.half())):
        with pytest.raises(_lib.AdkError, match="of one type"):
            a8.mlp8(*bad)


def test_nothing_is_kept_where_no_gradient_is_recorded(launches):
    from artdeco_amd import activation8 as a8
    x, w = torch.randn(4, 8), torch.randn(8, 8)
    kept = lambda: [args[-2:] for _, args in launches][-1]  # noqa: E731  (codes, units)
    with torch.no_grad():
        a8.activation8(x.clone().requires_grad_(True))
        assert kept() == (None, None)
    a8.mlp8(x, w, None, w, None)
    assert kept() == (None, None)
    a8.activation8(x.clone().requires_grad_(True))
    assert None not in kept()
    a8.mlp8(x, w, None, w.clone().requires_grad_(True), None)
    assert None not in kept()
    a8.activation8_forward(x)
    assert None not in kept()


def test_the_activations_c_entry_keeps_both_codes_and_units_or_neither(lib):
    P, N = 1 << 20, None
    assert lib.adk_activation8_fwd(P, 0, 1, 1, 0, 0, 0, P, P, N, N) == -1 and lib.adk_activation8_fwd(P, 0, 1, 1, 0, 0, 0, P, N, P, N) == -1


def test_rotary_in_place_refuses_before_it_turns(launches):
    """Views that autograd does not follow in place: the refusal leaves them as they are."""
    from artdeco_amd import _lib, rotary as ro
    f, _ = ro.rotary_frequencies(8)
    pos, leaf = torch.arange(4), torch.randn(1, 4, 16, requires_grad=True)
    whole = (leaf * 1).view(1, 4, 2, 8)
    with torch.no_grad():
        unrecorded = (leaf * 1).requires_grad_(True).view(1, 4, 2, 8)
    for x in (leaf.view(1, 4, 2, 8), whole.split(1, 2)[0], whole.chunk(2, 2)[1], unrecorded):
        with pytest.raises(_lib.AdkError, match="out of place|out of"):
            ro.rotary_(x, pos, f)
    assert not launches
    for x in (whole, whole[:, :, :1], leaf.detach().view(1, 4, 2, 8), leaf.detach().view(1, 4, 2, 8).split(1, 2)[0]):
        ro.rotary_(x, pos, f)
    with torch.no_grad():
        ro.rotary_(leaf.view(1, 4, 2, 8), pos, f)
    assert len(launches) == 5


def test_a_single_token_has_no_token_stride(monkeypatch):
    """One position of a sequence-major cache of a large batch: its token stride is past the kernels' 2^24 elements and used by nothing."""
    import ctypes
    from artdeco_amd import _lib, attention as att
    strides = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(_lib, "launch", lambda fn, what, device, *args: strides.append(list((ctypes.c_int64 * 13).from_address(args[14]))))
    far = torch.empty(2 * 4 * 64, dtype=torch.float16).as_strided((2, 4, 1, 64), (256, 64, 1 << 24, 1))
    att.attend_forward(far, far, far)
    att.attend_forward(torch.empty(2, 4, 1, 64, dtype=torch.float16), far, far)
    assert [s[2::3][:3] for s in strides] == [[0, 0, 0]] * 2


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 1])
def test_sizes_past_31_bits_are_refused(n, launches):
    """They would reach the library cut to 32 bits: 2^32 + 1 tokens as one."""
    from artdeco_amd import _lib, attention as att, rotary as ro
    one = torch.zeros(1, 1, 1, 8, dtype=torch.float16)
    f, _ = ro.rotary_frequencies(2)
    for q, k in ((one.expand(1, 1, n, 8), one), (one, one.expand(1, 1, n, 8)), (one.expand(n, 1, 1, 8), one.expand(n, 1, 1, 8)), (one.expand(1, n, 1, 8), one)):
        with pytest.raises(_lib.AdkError, match="31 bits"):
            att.attend_forward(q, k, k)
    for shape in ((1, n, 1, 2), (n, 1, 1, 2), (1, 1, n, 2)):
        with pytest.raises(_lib.AdkError, match="31 bits"):
            ro.rotary(one[..., :2].expand(shape), torch.zeros(1, dtype=torch.int64).expand(shape[1]), f)
    assert not launches


def test_c_entries_refuse_launches_that_the_grid_does_not_hold(lib):
    """2^24 workgroups of 256 threads are 2^32 threads: refused before a launch (of several, the first would be missing)."""
    import ctypes
    P, N = 1 << 20, None
    assert lib.adk_activation8_fwd(P, 0, 1 << 20, 1 << 16, 0, 0, 0, P, P, P, N) == -3
    assert lib.adk_activation8_bwd(P, P, P, 0, 1 << 20, 1 << 16, 0, 0, 0, P, N, N) == -3
    odd = (ctypes.c_int64 * 9)(256 << 26, 257, 257, 256 << 26, 257, 257, 0, 1, 0)
    assert lib.adk_rotary(P, P, P, P, 0, 1, 1 << 26, 1, 256, 1, 128, 1, 1, 0, 1.0, odd, N) == -3
    strides = (ctypes.c_int64 * 25)(*[8] * 9, 0, 0, 1, 0, *[8] * 12)
    for dtype, mask, rows in ((0, N, 1 << 28), (2, N, 1 << 28), (2, P, (1 << 28) - 64)):
        assert lib.adk_attend_bwd(P, P, P, P, P, P, N, mask, dtype, 1, 1, 1, rows, 1, 8, strides, 1.0, 0, P, P, P, P, 1 << 60, N) == -3, (dtype, mask, rows)
