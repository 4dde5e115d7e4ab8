"""The blocks of the MASt3R trunk set up for fine-tuning (to_training_dtype): rotary positions, attention with its gradient and the MLP with
its 8-bit checkpoint as they run together.

Tolerance of a block against the same block in 64 bits, in relative 2-norm: an activation or gradient on its way through a block is rounded
to the operands' type about a dozen times (projection, rotation, probabilities, attention, projection, two MLP layers, and back), each
by at most u of its norm, and no step of a freshly initialised block doubles what came before: 24 u.  Hidden values kept as int8 move
GELU's slope (|gelu''| < 0.8) by at most 0.8 of half a unit, a unit being at most 2/127 of the block's largest, about 4 standard
deviations against a slope of about 0.6: below 0.05 in all."""
import pytest
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def positions(B, h, w):
    ys, xs = torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij")
    return torch.stack([ys.reshape(-1), xs.reshape(-1)], -1)[None].expand(B, -1, 2).contiguous()


def far(a, b):
    return float((a.detach().double().cpu() - b).norm() / b.norm())


def narrowed(block, dtype):
    from artdeco_amd import mast3r_model as mm
    for m in block.modules():
        if isinstance(m, torch.nn.Linear):
            m.to(dtype)
        if isinstance(m, (mm.Attention, mm.CrossAttention, mm.Mlp)):
            m.trains = True
    return block


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kept8", [None, "int8"])
def test_a_block_and_its_gradients(dtype, kept8, dev):
    from functools import partial
    from artdeco_amd import mast3r_model as mm
    torch.manual_seed(0)
    rope, norm = mm.RoPE2D(100.0), partial(torch.nn.LayerNorm, eps=1e-6)
    dec = mm.DecoderBlock(192, 3, 4, norm, rope)
    ref = mm.DecoderBlock(192, 3, 4, norm, rope).double()
    with torch.no_grad():
        for a, b in zip(dec.parameters(), ref.parameters()):
            a.copy_(a.to(dtype))                      # both start from the same representable weights
            b.copy_(a.double())
    narrowed(dec.to(dev), dtype)
    dec.mlp.kept8 = kept8
    x, y, go = torch.randn(2, 35, 192), torch.randn(2, 35, 192), torch.randn(2, 35, 192)
    pos = positions(2, 5, 7)
    gx, gy = x.to(dev).requires_grad_(True), y.to(dev).requires_grad_(True)
    out, _ = dec(gx, gy, pos.to(dev), pos.flip(1).to(dev).contiguous())
    grads = torch.autograd.grad(out, [gx, gy, *dec.parameters()], go.to(dev))
    rx, ry = x.double().requires_grad_(True), y.double().requires_grad_(True)
    rout, _ = ref(rx, ry, pos, pos.flip(1))
    want = torch.autograd.grad(rout, [rx, ry, *ref.parameters()], go.double())
    tol = 24 * U[dtype] + (0.05 if kept8 else 0.0)
    assert far(out, rout.detach()) <= 24 * U[dtype]
    names = ["x", "y"] + [n for n, _ in ref.named_parameters()]
    for name, a, b in zip(names, grads, want):
        if "projk.bias" in name or "qkv.bias" in name:  # a bias that all keys share shifts every score of a row alike: its slope is rounding alone
            a, b = a[..., -192:] if "qkv" in name else a * 0, b[..., -192:] if "qkv" in name else b * 0 + 1e-30
            if "projk" in name:
                continue
        assert far(a, b) <= tol, (name, far(a, b), tol)


@pytest.mark.gpu
def test_the_model_trains_through_the_kernels(dev):
    """Every trunk parameter gets a finite gradient, every attention and MLP goes through the kernels, a step changes the result, inference
    afterwards is the inference path's."""
    from artdeco_amd import activation8 as a8, attention as att
    from artdeco_amd.mast3r_model import AsymmetricMASt3R
    torch.manual_seed(0)
    net = AsymmetricMASt3R(img_size=(64, 64), enc_embed_dim=128, enc_depth=2, enc_num_heads=2, dec_embed_dim=64, dec_depth=4, dec_num_heads=1).to(dev)
    net.to_training_dtype(torch.bfloat16, kept8="int8")
    views = [{"img": torch.rand(1, 3, 48, 64, device=dev) * 2 - 1, "true_shape": torch.tensor([[48, 64]])} for _ in range(2)]
    calls = {"attend": 0, "mlp": 0}
    forward, kept = att.attend_forward, a8.activation8_forward
    att.attend_forward = lambda *a, **kw: (calls.__setitem__("attend", calls["attend"] + 1), forward(*a, **kw))[1]
    a8.activation8_forward = lambda *a, **kw: (calls.__setitem__("mlp", calls["mlp"] + 1), kept(*a, **kw))[1]
    try:
        r1, r2 = net.training_forward(*views)
    finally:
        att.attend_forward, a8.activation8_forward = forward, kept
    assert calls == {"attend": 2 * 2 + 4 * 2 * 2, "mlp": 2 * 2 + 4 * 2}
    loss = r1["pts3d"].square().mean() + r2["pts3d_in_other_view"].square().mean() + r1["desc"].square().mean() + r2["desc"].sum() * 0.01
    loss.backward()
    for n, p in net.named_parameters():
        if n.startswith(("enc_", "dec_", "decoder_embed", "patch_embed")):
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
    f1, pos, _ = net._encode_image(views[0]["img"])
    with torch.no_grad():
        for p in net.parameters():
            if p.grad is not None:
                p.sub_(1e-2 * p.grad)
    assert not torch.equal(net._encode_image(views[0]["img"])[0], f1)
    assert not net(*views)[0]["pts3d"].requires_grad
    with torch.no_grad():
        a = net._encode_image(views[0]["img"])[0]
        net.to_inference_dtype(torch.bfloat16, fp32_stream=True)
        assert not any(getattr(m, "trains", False) for m in net.modules())
        assert torch.equal(net._encode_image(views[0]["img"])[0], a)


@pytest.mark.gpu
def test_a_training_step_captured_and_replayed(dev):
    """rotary_, attend_packed and mlp8 with their backward passes in one graph, replayed with new inputs between eager work."""
    from artdeco_amd import activation8 as a8, attention as att, rotary as ro
    torch.manual_seed(1)
    H, D, N = 4, 64, 70
    C = H * D
    w = [(torch.randn(s, device=dev) * 0.05).bfloat16() for s in ((3 * C, C), (C, C), (2 * C, C), (C, 2 * C))]
    x, go, pos = torch.randn(1, N, C, device=dev).bfloat16(), torch.randn(1, N, C, device=dev).bfloat16(), torch.arange(N, device=dev)
    f, _ = ro.rotary_frequencies(D, device=dev)

    def step():
        ws = [t.detach().requires_grad_(True) for t in w]
        qkv = ro.rotary_(torch.nn.functional.linear(x, ws[0]).view(1, N, 3 * H, D), pos, f, heads=2 * H)
        h = torch.nn.functional.linear(att.attend_packed(qkv, H, causal=True), ws[1])
        return torch.autograd.grad(a8.mlp8(h, ws[2], None, ws[3], None, format="e4m3"), ws, go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        x.copy_(torch.randn(1, N, C, device=dev))
        go.copy_(torch.randn(1, N, C, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        held = [g.clone() for g in got]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), turn


def test_setting_up_and_back():
    from artdeco_amd.mast3r_model import AsymmetricMASt3R
    net = AsymmetricMASt3R(img_size=(32, 32), enc_embed_dim=64, enc_depth=1, enc_num_heads=1, dec_embed_dim=64, dec_depth=4, dec_num_heads=1)
    with pytest.raises(ValueError):
        net.to_training_dtype(torch.float32)
    with pytest.raises(ValueError):
        net.to_training_dtype(torch.bfloat16, kept8="int4")
    net.to_training_dtype(torch.bfloat16, kept8="e4m3")
    assert net.enc_blocks[0].attn.trains and net.dec_blocks[0].mlp.kept8 == "e4m3" and net.downstream_head1.head_local_features.kept8 is None
    assert net.enc_blocks[0].attn.qkv.weight.dtype == torch.bfloat16 and net.enc_norm.weight.dtype == torch.float32
    x, pos = torch.randn(1, 4, 64), positions(1, 2, 2)
    assert net.enc_blocks[0](x, pos).shape == (1, 4, 64)     # on the CPU: torch's operators, as before
    net.to_inference_dtype(torch.float32)
    assert not net.enc_blocks[0].attn.trains and net.enc_blocks[0].mlp.kept8 is None
