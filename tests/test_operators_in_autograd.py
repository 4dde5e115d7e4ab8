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
