"""The operators for fine-tuning in the forms that training programs call them: autocast, frozen parameters, adapters, masks on packed
projections, validation between steps.

Tolerances: where two ways make the same launches on the same operands the bits are the same; otherwise as said at each test."""
import pytest
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def mlp_leaves(dev, dtype=torch.float32, gated=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    W = 96 * (2 if gated else 1)
    make = lambda *s, size=1.0: (torch.randn(*s, generator=g) * size).to(dtype).to(dev).requires_grad_(True)  # noqa: E731
    return [make(2, 9, 32), make(W, 32, size=0.2), make(W), make(24, 96, size=0.2), make(24)], (torch.randn(2, 9, 24, generator=g)).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_mlp8_under_autocast(dtype, dev):
    """float32 leaves, and leaves of several types: the call and the gradients of the same operands cast by hand; backward inside the region
    too, also for a call that was made outside it."""
    from artdeco_amd import activation8 as a8
    leaves, grad = mlp_leaves(dev)
    cast = [t.detach().to(dtype).requires_grad_(True) for t in leaves]
    out = a8.mlp8(*cast)
    want = torch.autograd.grad(out, cast, grad.to(dtype))
    mixed = [leaves[0].detach().to(dtype).requires_grad_(True)] + leaves[1:]
    for operands in (leaves, mixed):
        with torch.autocast("cuda", dtype=dtype):
            got = a8.mlp8(*operands)
            assert got.dtype == dtype and torch.equal(got, out)
            inside = torch.autograd.grad(got, operands, grad.to(dtype), retain_graph=True)
        for grads in (inside, torch.autograd.grad(got, operands, grad.to(dtype))):
            assert all(torch.equal(a, b.to(a.dtype)) and a.dtype == t.dtype for a, b, t in zip(grads, want, operands))
    plain = a8.mlp8(*leaves)
    first = torch.autograd.grad(plain, leaves, grad, retain_graph=True)
    with torch.autocast("cuda", dtype=dtype):
        again = torch.autograd.grad(plain, leaves, grad)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,gated", [((1, 1), False), ((3, 7, 41), False), ((5, 26), True), ((257, 1000), True)], ids=str)
def test_values_without_a_checkpoint(shape, gated, dtype, dev):
    """The same bits as with one."""
    from artdeco_amd import activation8 as a8
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).to(dtype).to(dev)
    for kind in ("gelu", "gelu_tanh", "silu"):
        want, _ = a8.activation8_forward(x, kind=kind, gated=gated)
        assert torch.equal(a8.activation8(x, kind=kind, gated=gated), want)
    leaves, _ = mlp_leaves(dev, dtype, gated)
    with torch.no_grad():
        got = a8.mlp8(*leaves, gated=gated)
    assert torch.equal(got, a8.mlp8(*leaves, gated=gated).detach()) and not got.requires_grad


def small_model(dev):
    from artdeco_amd.mast3r_model import AsymmetricMASt3R
    torch.manual_seed(0)
    net = AsymmetricMASt3R(img_size=(64, 64), enc_embed_dim=128, enc_depth=2, enc_num_heads=2, dec_embed_dim=64, dec_depth=4, dec_num_heads=1).to(dev)
    g = torch.Generator().manual_seed(1)
    return net, [{"img": (torch.rand(1, 3, 48, 64, generator=g) * 2 - 1).to(dev), "true_shape": torch.tensor([[48, 64]])} for _ in range(2)]


@pytest.mark.gpu
def test_validation_between_steps_is_the_inference_path(dev, monkeypatch):
    """forward() of a model set up for training: the fused norms, the second stream and the trunk's bits of one set up for inference (the heads
    are library convolutions, whose results differ by a step from call to call of one and the same model)."""
    from artdeco_amd import fused_norm
    net, views = small_model(dev)
    tokens, heads = [], net.both_heads
    monkeypatch.setattr(net, "both_heads", lambda dec1, dec2, *a: (tokens.append([*dec1, *dec2]), heads(dec1, dec2, *a))[1])
    norms, add_layernorm = [], fused_norm.add_layernorm
    monkeypatch.setattr(fused_norm, "add_layernorm", lambda *a, **kw: (norms.append(1), add_layernorm(*a, **kw))[1])
    net.to_inference_dtype(torch.float16, fp32_stream=True)
    net(*views)
    count = len(norms)
    net.to_training_dtype(torch.float16, kept8="int8")
    norms.clear()
    net(*views)
    assert count > 0 and len(norms) == count and net._side_stream(views[0]["img"]) is None
    with torch.no_grad():
        assert net._side_stream(views[0]["img"]) is not None
    assert len(tokens[0]) == 10 and all(torch.equal(a, b) for a, b in zip(*tokens))
    norms.clear()
    r1, r2 = net.training_forward(*views)
    assert not norms and r1["pts3d"].requires_grad and r2["desc"].requires_grad


@pytest.mark.gpu
def test_validation_sees_the_weights_of_a_replayed_step(dev, monkeypatch):
    """A captured step changes weights without touching their version counters: forward() between replays and after the training."""
    net, views = small_model(dev)
    net.to_training_dtype(torch.float16)
    tokens, heads = [], net.both_heads
    monkeypatch.setattr(net, "both_heads", lambda dec1, dec2, *a: (tokens.append([*dec1, *dec2]), heads(dec1, dec2, *a))[1])
    net(*views)
    weights = [blk.cross_attn.projk.weight for blk in (*net.dec_blocks, *net.dec_blocks2)]
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        for w in weights:
            w.mul_(-1.5)
    for turn in ("between", "between", "after", "after one without validation"):
        if turn == "after one without validation":
            net.to_training_dtype(torch.float16)
        graph.replay()
        if turn != "between":
            net.to_inference_dtype(torch.float16, fp32_stream=True)
        net(*views)
        with torch.no_grad():
            for blk in (*net.dec_blocks, *net.dec_blocks2):
                blk.cross_attn.projk.weight.mul_(1.0)      # seen by its version counter
        net(*views)
        assert all(torch.equal(a, b) for a, b in zip(tokens[-2], tokens[-1])) and not torch.equal(tokens[0][-1], tokens[-1][-1]), turn


@pytest.mark.gpu
def test_a_model_set_up_for_inference_does_not_pretend_to_train(dev):
    """Its kernels pass autograd by: the rotation would be missing from the gradients, or everything before the attention."""
    net, views = small_model(dev)
    for set_up in (lambda: None, lambda: net.to_inference_dtype(torch.float16, fp32_stream=True), lambda: (net.to_training_dtype(torch.float16), net.to_inference_dtype(torch.float16))):
        set_up()
        with pytest.raises(RuntimeError, match="to_training_dtype"):
            net.training_forward(*views)
        with torch.no_grad():
            assert not net.training_forward(*views)[0]["pts3d"].requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 4, 2, 77, 150, 64), (1, 24, 24, 300, 1133, 96), (8, 8, 2, 1, 700, 128)], ids=str)
def test_masks_of_any_bytes(size, dev):
    """A boolean view of bytes other than 0 and 1 shows what the same mask of 0 and 1 shows, side by side in memory and apart."""
    from artdeco_amd import attention as att
    B, H, Hk, Nq, Nk, D = size
    g = torch.Generator().manual_seed(3)
    q, do = (torch.randn(B, H, Nq, D, generator=g).bfloat16().to(dev) for _ in range(2))
    k, v = (torch.randn(B, Hk, Nk, D, generator=g).bfloat16().to(dev) for _ in range(2))
    flat = do.transpose(1, 2).reshape(B, Nq, H * D)
    values = torch.tensor([0, 255, 2, 0, 128, 1, 0, 254], dtype=torch.uint8)
    for shape in ((B, 1, Nq, Nk), (B, 1, 1, Nk), (1, 1, Nk, Nq)):
        raw = values[torch.randint(0, 8, shape, generator=g)].to(dev)
        raw = raw.transpose(2, 3) if shape[2] == Nk else raw
        results = []
        for mask in (raw != 0, raw.view(torch.bool)):
            out, lse = att.attend_forward(q, k, v, mask=mask)
            results.append((out, lse, *att.attend_backward(flat, q, k, v, out, lse, mask=mask)))
        assert all(torch.equal(a, b) for a, b in zip(*results)), shape


@pytest.mark.parametrize("first", [dict(dtype=torch.bfloat16), dict(dtype=torch.float16, fp32_stream=True, heads=True)], ids=["trunk", "heads"])
def test_training_after_a_narrower_inference(first):
    """Norms and heads are fp32 again, whatever to_inference_dtype() had narrowed."""
    from artdeco_amd.mast3r_model import AsymmetricMASt3R
    net = AsymmetricMASt3R(img_size=(32, 32), enc_embed_dim=64, enc_depth=1, enc_num_heads=1, dec_embed_dim=64, dec_depth=4, dec_num_heads=1)
    net.to_inference_dtype(**first)
    net.to_training_dtype(torch.bfloat16)
    for name, p in net.named_parameters():
        trunk = name.startswith(("enc_blocks", "dec_blocks", "patch_embed", "decoder_embed")) and "norm" not in name
        assert p.dtype == (torch.bfloat16 if trunk else torch.float32), name
    view = {"img": torch.rand(1, 3, 32, 32)}
    assert net.training_forward(view, view)[0]["pts3d"].requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
def test_mlp8_of_some_gradients(gated, dtype, dev):
    """Frozen parameters and inputs, every combination of two kinds: the gradients that are asked for are those of the full call; without biases,
    those of biases of zero."""
    from artdeco_amd import activation8 as a8
    leaves, grad = mlp_leaves(dev, dtype, gated)
    grad = grad.to(dtype)
    full = torch.autograd.grad(a8.mlp8(*leaves, kind="silu", gated=gated), leaves, grad)
    for asked in ([0], [1], [2], [3], [4], [0, 3], [1, 2], [3, 4], [0, 1, 2], [1, 2, 3, 4]):
        some = [t.detach().requires_grad_(i in asked) for i, t in enumerate(leaves)]
        got = torch.autograd.grad(a8.mlp8(*some, kind="silu", gated=gated), [some[i] for i in asked], grad)
        assert all(torch.equal(g, full[i]) for g, i in zip(got, asked)), asked
    x, w1, b1, w2, b2 = leaves
    zeros = [torch.zeros_like(b1).requires_grad_(True), torch.zeros_like(b2).requires_grad_(True)]
    bare, filled = a8.mlp8(x, w1, None, w2, None, gated=gated), a8.mlp8(x, w1, zeros[0], w2, zeros[1], gated=gated)
    assert torch.equal(bare, filled)
    for a, b in zip(torch.autograd.grad(bare, (x, w1, w2), grad), torch.autograd.grad(filled, (x, w1, w2), grad)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,D", [(6, 2, 64), (4, 1, 40), (3, 3, 128)])
def test_attend_packed_with_masks_and_lengths(heads, kv_heads, D, dtype, dev):
    """One projection's heads, fewer of keys than of queries: the bits of attend_forward and attend_backward on its three views, whatever hides."""
    from artdeco_amd import attention as att
    B, N = 3, 77
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(B, N, heads + 2 * kv_heads, D, generator=g).to(dtype).to(dev).requires_grad_(True)
    do = torch.randn(B, N, heads * D, generator=g).to(dtype).to(dev)
    lengths = torch.tensor([N, 0, 31], dtype=torch.int32, device=dev)
    free = (torch.rand(B, heads, N, N, generator=g) < 0.6).to(dev)
    wide = torch.zeros(B, 1, N, 2 * N, dtype=torch.bool, device=dev)
    wide[..., ::2] = free[:, :1]
    for mask in (None, free, free[:, :1], free[:1, :1, :1], wide[..., ::2]):
        for how in (dict(mask=mask), dict(mask=mask, key_lengths=lengths), dict(mask=mask, key_lengths=lengths, causal=True, scale=0.3)):
            out = att.attend_packed(qkv, heads, kv_heads, **how)
            got, = torch.autograd.grad(out, qkv, do)
            t = qkv.detach().transpose(1, 2)
            q, k, v = t[:, :heads], t[:, heads:heads + kv_heads], t[:, heads + kv_heads:]
            o, lse = att.attend_forward(q, k, v, **how)
            want = torch.cat([s.transpose(1, 2) for s in att.attend_backward(do, q, k, v, o, lse, **how)], 2)
            assert torch.equal(out, o) and torch.equal(got, want), how.keys()
