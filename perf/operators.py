"""The transformer-training operators as they are measured: rotary positions, attention with its gradient, and activations whose
backward pass reads an 8-bit checkpoint.

`own` selects the side: False computes the plain form (elementary torch operations in 32 bits, rounded once at the end), True makes
the calls a program makes of artdeco_amd.  Both take what prepare() returns."""
import math

import torch

own = False

_DTYPE = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}


def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


# ------------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token of each of 8 sequences, deep inside a long context: q, k and v heads of one projection, q and k turned
        {"name": "rotary_token", "op": "rotary", "batch": 8, "tokens": 1, "heads": 48, "turned": 40, "dim": 128, "rotary_dim": 128, "axes": 1,
         "layout": "half", "scaling": "by_parts", "span": 1000000, "transpose": False, "type": "bfloat16"},
        # the encoder's packed projection of 4 views, 24 x 32 patches each: two axes, as the model rotates
        {"name": "rotary_views", "op": "rotary", "batch": 4, "tokens": 768, "heads": 48, "turned": 32, "dim": 64, "rotary_dim": 64, "axes": 2,
         "layout": "half", "scaling": "none", "span": 32, "transpose": False, "type": "float16"},
        # gradient of one long sequence, half of every head turned in interleaved pairs, positions interpolated; an odd length
        {"name": "rotary_long_gradient", "op": "rotary", "batch": 1, "tokens": 32749, "heads": 32, "turned": 32, "dim": 128, "rotary_dim": 64,
         "axes": 1, "layout": "interleaved", "scaling": "linear", "span": 131072, "transpose": True, "type": "bfloat16"},
        # answering token by token: one query of each of 16 sequences against caches of different fill, 4 query heads to a key head
        {"name": "attend_token", "op": "attend", "batch": 16, "heads": 32, "kv_heads": 8, "queries": 1, "keys": 8192, "dim": 128, "causal": False,
         "lengths": True, "mask": False, "train": False, "type": "bfloat16"},
        # one image pair through an encoder block
        {"name": "attend_pair", "op": "attend", "batch": 2, "heads": 16, "kv_heads": 16, "queries": 768, "keys": 768, "dim": 64, "causal": False,
         "lengths": False, "mask": False, "train": False, "type": "float16"},
        # a long prompt read at once
        {"name": "attend_prompt", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "queries": 8192, "keys": 8192, "dim": 128, "causal": True,
         "lengths": False, "mask": False, "train": False, "type": "bfloat16"},
        # one training step through the decoder's cross attention at a tenth of its tokens: launches count
        {"name": "attend_train_small", "op": "attend", "batch": 1, "heads": 12, "kv_heads": 12, "queries": 77, "keys": 130, "dim": 64, "causal": False,
         "lengths": False, "mask": False, "train": True, "type": "float16"},
        # a training batch of padded sets of tokens with a free mask, a head size between the tiles', odd lengths
        {"name": "attend_train_masked", "op": "attend", "batch": 4, "heads": 12, "kv_heads": 4, "queries": 517, "keys": 1031, "dim": 80, "causal": False,
         "lengths": True, "mask": True, "train": True, "type": "bfloat16"},
        # the encoder's training batch: 8 images of 768 tokens
        {"name": "attend_train_views", "op": "attend", "batch": 8, "heads": 16, "kv_heads": 16, "queries": 768, "keys": 768, "dim": 64, "causal": False,
         "lengths": False, "mask": False, "train": True, "type": "float16"},
        # a long causal sequence, 4 query heads to a key head: the largest
        {"name": "attend_train_long", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "queries": 8192, "keys": 8192, "dim": 128, "causal": True,
         "lengths": False, "mask": False, "train": True, "type": "bfloat16"},
        # the encoder's MLP activation of one image, forward and backward through its 8-bit checkpoint
        {"name": "activation8_image", "op": "activation8", "rows": 768, "width": 4096, "kind": "gelu", "gated": False, "format": "int8", "type": "float16"},
        # a gated MLP's activation over a long batch, an odd width
        {"name": "activation8_gated", "op": "activation8", "rows": 16384, "width": 5461, "kind": "silu", "gated": True, "format": "e4m3", "type": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attend", "attend", "activation8"])
    if op == "rotary":
        dim = 8 * rng.randint(4, 32)
        axes = rng.choice([1, 1, 2, 3])
        rotary_dim = 2 * axes * max(1, (dim // rng.choice([1, 1, 2, 4])) // (2 * axes))
        heads = rng.randint(1, 64)
        tokens = _log(rng, 1, 32768)
        batch = _log(rng, 1, max(1, min(16, 134000000 // (heads * dim * tokens))))
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "turned": rng.randint(1, heads), "dim": dim, "rotary_dim": rotary_dim, "axes": axes,
                "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "ntk", "by_parts"]), "span": _log(rng, 32, 1000000),
                "transpose": rng.random() < 0.5, "type": rng.choice(["float16", "bfloat16", "float32"])}
    if op == "attend":
        kv_heads, group = rng.randint(1, 16), rng.choice([1, 1, 2, 4, 8])
        dim = rng.choice([32, 48, 64, 64, 80, 96, 112, 128, 128])
        causal, train = rng.random() < 0.4, rng.random() < 0.5
        keys = _log(rng, 1, 8192)
        queries = keys if causal and rng.random() < 0.7 else 1 if not train and rng.random() < 0.3 else _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(16, 1000000000 // (kv_heads * group * queries * keys))))
        return {"op": op, "batch": batch, "heads": kv_heads * group, "kv_heads": kv_heads, "queries": queries, "keys": keys, "dim": dim, "causal": causal,
                "lengths": rng.random() < 0.4, "mask": rng.random() < 0.25 and batch * queries * keys < 300000000, "train": train,
                "type": rng.choice(["float16", "bfloat16"])}
    rows, gated = _log(rng, 1, 16384), rng.random() < 0.5
    return {"op": op, "rows": rows, "width": _log(rng, 1, 5400), "kind": rng.choice(["gelu", "gelu_tanh", "silu"]), "gated": gated,
            "format": rng.choice(["int8", "e4m3"]), "type": rng.choice(["float16", "bfloat16", "float32"])}


def _fills(case):
    """How many keys each sequence of a padded batch has: spread over the whole length, the first full, the last of several empty."""
    B, N = case["batch"], case["keys"]
    return [N if b == 0 else 0 if b == B - 1 and B > 2 else int(N * ((b * 0.6180339887498949) % 1.0)) for b in range(B)]


def _visible(case):
    """Pairs of a query and a key that it sees, over the batch, for one head (a free mask counts as seen: its tiles are computed)."""
    total = 0
    for n in (_fills(case) if case["lengths"] else [case["keys"]] * case["batch"]):
        if not case["causal"]:
            total += case["queries"] * n
            continue
        first = case["keys"] - case["queries"] + 1  # keys that query 0 sees, before the fill cuts them
        lo = max(0, -first)                         # queries before this one see nothing
        full = min(case["queries"], max(lo, n - first + 1))
        total += sum((first + lo, first + full - 1)) * (full - lo) // 2 if full > lo else 0
        total += (case["queries"] - full) * n
    return total


def work(case):
    es = _BYTES[case["type"]]
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"]
        turned = n * case["turned"] * case["rotary_dim"]
        return {"bytes": 2 * n * case["heads"] * case["dim"] * es + 8 * n * case["axes"], "flops": 3 * turned}
    if case["op"] == "attend":
        B, H, D = case["batch"], case["heads"], case["dim"]
        q = B * H * case["queries"] * D * es
        kv = 2 * case["kv_heads"] * D * es * (sum(_fills(case)) if case["lengths"] else B * case["keys"])
        kv_out = 2 * case["kv_heads"] * D * es * B * case["keys"]
        lse = 4 * B * H * case["queries"]
        m = B * case["queries"] * case["keys"] if case["mask"] else 0
        pairs = H * _visible(case)
        if not case["train"]:
            return {"bytes": 2 * q + kv + lse + m, "flops": 4 * D * pairs}
        return {"bytes": 4 * q + kv + kv_out + lse + m, "flops": 14 * D * pairs}
    n = case["rows"] * case["width"]
    wide = n * (2 if case["gated"] else 1)
    return {"bytes": (2 * wide + 3 * n) * es + 2 * (wide + -(-wide // 32)), "flops": 60 * n}


# ------------------------------------------------------------------------------------------------------------------ the inputs
def _scaling(case):
    """The factor and the trained length that go with a kind of scaling: contexts eight times the trained 8192."""
    return {"none": {}, "linear": {"factor": 8.0}, "ntk": {"factor": 8.0}, "by_parts": {"factor": 8.0, "trained_length": 8192}}[case["scaling"]]


def _frequencies(case, dev):
    """Angle per position of each pair of one axis, in 64 bits, and the factor on cosine and sine."""
    pairs = case["rotary_dim"] // (2 * case["axes"])
    base, extra = 10000.0, _scaling(case)
    at = torch.arange(pairs, dtype=torch.float64, device=dev) / pairs
    if case["scaling"] == "ntk":
        width = 2 * pairs
        base = base * extra["factor"] ** (width / max(1, width - 2))
    inv = torch.pow(torch.tensor(base, dtype=torch.float64, device=dev), -at)
    if case["scaling"] == "linear":
        inv = inv / extra["factor"]
    if case["scaling"] != "by_parts":
        return inv, 1.0
    # pairs that turn more than 32 times within the trained length stay, those below one turn are interpolated, a ramp between
    turns = extra["trained_length"] * inv / (2 * math.pi)
    keep = ((turns.log() - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0.0, 1.0)
    return inv * keep + inv / extra["factor"] * (1 - keep), 0.1 * math.log(extra["factor"]) + 1.0


def prepare(case, seed):
    dev, dt = _device(), _DTYPE[case["type"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "rotary":
        B, N = case["batch"], case["tokens"]
        x = torch.randn(B, N, case["heads"], case["dim"], generator=g, device=dev).to(dt)
        positions = torch.randint(0, case["span"], (B, N, case["axes"]), generator=g, device=dev)
        inv, factor = _frequencies(case, dev)                   # a model keeps these, as it keeps its weights
        return {"case": case, "x": x, "positions": positions, "inv": inv, "factor": factor}
    if case["op"] == "attend":
        B, H, K, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        nq, nk = case["queries"], case["keys"]
        # token-major, as the projections leave them: [B, N, heads, D] seen as [B, heads, N, D]
        q, k, v = (torch.randn(B, n, h, D, generator=g, device=dev).to(dt).transpose(1, 2) for n, h in ((nq, H), (nk, K), (nk, K)))
        grad = torch.randn(B, nq, H * D, generator=g, device=dev).to(dt) if case["train"] else None
        lengths = torch.tensor(_fills(case), dtype=torch.int32, device=dev) if case["lengths"] else None
        mask = None
        if case["mask"]:  # four fifths seen, and every eighth query sees nothing
            mask = torch.rand(B, 1, nq, nk, generator=g, device=dev) < 0.8
            mask[..., 0] = True
            mask[:, :, 7::8] = False
        return {"case": case, "q": q, "k": k, "v": v, "grad": grad, "lengths": lengths, "mask": mask}
    shape = (case["rows"], case["width"] * (2 if case["gated"] else 1))
    x = (torch.randn(shape, generator=g, device=dev) * 2.0).to(dt)
    grad = torch.randn(case["rows"], case["width"], generator=g, device=dev).to(dt)
    return {"case": case, "x": x, "grad": grad}


# ----------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "rotary":
        return _plain_rotary(s, case)
    if case["op"] == "attend":
        return _plain_attend(s, case)
    return _plain_activation(s, case)


def _run_own(s, case):
    if case["op"] == "rotary":
        from artdeco_amd import rotary
        turn = rotary.rotary_transpose if case["transpose"] else rotary.rotary
        return turn(s["x"], s["positions"], s["inv"], factor=s["factor"], layout=case["layout"], heads=case["turned"])
    if case["op"] == "attend":
        from artdeco_amd import attention
        how = {"causal": case["causal"], "key_lengths": s["lengths"], "mask": s["mask"]}
        out, lse = attention.attend_forward(s["q"], s["k"], s["v"], **how)
        if not case["train"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = attention.attend_backward(s["grad"], s["q"], s["k"], s["v"], out, lse, **how)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    from artdeco_amd import activation8
    y, packed = activation8.activation8_forward(s["x"], kind=case["kind"], gated=case["gated"], format=case["format"])
    # the backward pass also gives the activation again, from the checkpoint: the next layer's weight gradient reads it
    dx, again = activation8.activation8_backward(s["grad"], packed, kind=case["kind"], gated=case["gated"])
    return {"y": y, "dx": dx, "again": again}


# --------------------------------------------------------------------------------------------------------------- plain forms
def _plain_rotary(s, case):
    x, A = s["x"], case["axes"]
    pairs, T, R = case["rotary_dim"] // (2 * A), case["turned"], case["rotary_dim"]
    inv, factor = s["inv"], s["factor"]
    angle = s["positions"].double()[..., None] * inv            # [B, N, A, pairs]: far positions lose their turn in 32 bits
    c, sn = (angle.cos() * factor).float()[:, :, None], (angle.sin() * factor).float()[:, :, None]
    if case["transpose"]:
        sn = -sn
    f = x[:, :, :T, :R].float()
    if case["layout"] == "half":
        f = f.reshape(*f.shape[:3], A, 2, pairs)
        u, v = f[..., 0, :], f[..., 1, :]
        turned = torch.stack([u * c - v * sn, v * c + u * sn], dim=-2)
    else:
        f = f.reshape(*f.shape[:3], A, pairs, 2)
        u, v = f[..., 0], f[..., 1]
        turned = torch.stack([u * c - v * sn, v * c + u * sn], dim=-1)
    y = x.clone()
    y[:, :, :T, :R] = turned.reshape(*turned.shape[:3], R).to(x.dtype)
    return y


def _seen(s, case, rows, dev):
    """Which keys each query of `rows` (their numbers) sees, as [B, 1, rows, keys]; None where all of them."""
    seen = None
    at = torch.arange(case["keys"], device=dev)
    if case["causal"]:
        seen = (at[None, :] <= rows[:, None] + (case["keys"] - case["queries"]))[None, None]
    if s["lengths"] is not None:
        fill = at[None, None, None, :] < s["lengths"][:, None, None, None]
        seen = fill if seen is None else seen & fill
    if s["mask"] is not None:
        seen = s["mask"] if seen is None else seen & s["mask"]
    return seen


def _plain_attend(s, case):
    B, H, K, D, nq, nk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "queries", "keys"))
    G, scale = H // K, 1.0 / math.sqrt(D)
    q, k, v = s["q"].float().reshape(B, K, G * nq, D), s["k"].float().contiguous(), s["v"].float().contiguous()
    if s["lengths"] is not None:  # what lies behind a sequence's end is not its own, whatever it holds
        mine = (torch.arange(nk, device=k.device)[None] < s["lengths"][:, None])[:, None, :, None]
        k, v = torch.where(mine, k, 0.0), torch.where(mine, v, 0.0)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    seen = _seen(s, case, torch.arange(nq, device=q.device), q.device)
    if seen is not None:
        score = torch.where(seen[:, :, None], score.view(B, K, G, nq, nk), -math.inf).view(B, K, G * nq, nk)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).view(B, H, nq)                    # a query that sees nothing: -inf, and zeros below
    p = torch.where(total > 0, p / total, 0.0)
    o = torch.matmul(p, v)
    out = o.view(B, H, nq, D).transpose(1, 2).reshape(B, nq, H * D).to(s["q"].dtype)
    if not case["train"]:
        return {"out": out, "lse": lse}
    do = s["grad"].float().view(B, nq, H, D).transpose(1, 2).reshape(B, K, G * nq, D)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k).view(B, H, nq, D)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dt = s["q"].dtype
    return {"out": out, "lse": lse, "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}


def _plain_kept(x, fmt):
    """x as the 8-bit checkpoint holds it, in x's shape: blocks of 32 consecutive values share the smallest power of two under which
    their largest fits the format."""
    n = x.numel()
    f = torch.nn.functional.pad(x.reshape(-1).float(), (0, -n % 32)).view(-1, 32)
    top = f.abs().amax(1, keepdim=True)
    m, e = torch.frexp(top)                                     # top = m 2^e, 1/2 <= m < 1
    room, most = (7, 127.0 / 128.0) if fmt == "int8" else (9, 448.0 / 512.0)
    e = (e - room + (m > most).to(e.dtype)).clamp(min=-126)
    unit = torch.ldexp(torch.ones_like(top), e)
    f = f / unit
    if fmt == "int8":
        f = torch.round(f)
    else:                                                       # three bits behind the leading one, and steps of 2^-9 below 2^-6
        step = torch.ldexp(torch.ones_like(f), torch.frexp(f)[1].clamp(min=-5) - 4)
        f = torch.round(f / step) * step
    return (f * unit).view(-1)[:n].view(x.shape)


def _plain_value(x, kind):
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_slope(x, kind):
    if kind == "silu":
        t = 1 / (1 + torch.exp(-x))
        return t * (1 + x * (1 - t))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)


def _plain_activation(s, case):
    x, grad, w = s["x"].float(), s["grad"].float(), case["width"]
    kept = _plain_kept(s["x"], case["format"])
    dt = s["x"].dtype
    if not case["gated"]:
        return {"y": _plain_value(x, case["kind"]).to(dt), "dx": (grad * _plain_slope(kept, case["kind"])).to(dt), "again": _plain_value(kept, case["kind"]).to(dt)}
    y = _plain_value(x[:, :w], case["kind"]) * x[:, w:]
    value = _plain_value(kept[:, :w], case["kind"])
    da = grad * kept[:, w:] * _plain_slope(kept[:, :w], case["kind"])
    return {"y": y.to(dt), "dx": torch.cat([da, grad * value], dim=1).to(dt), "again": (value * kept[:, w:]).to(dt)}


# ------------------------------------------------------------------------------------------------------- the definitions, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s, case)
    if case["op"] == "attend":
        return _exact_attend(s, case)
    return _exact_activation(s, case)


def _exact_rotary(s, case):
    """Every pair as a complex number, multiplied by the angle's."""
    x, A, R, T = s["x"].double(), case["axes"], case["rotary_dim"], case["turned"]
    pairs = R // (2 * A)
    inv, factor = s["inv"], s["factor"]
    angle = (s["positions"].double()[:, :, None, :, None] * inv) * (-1.0 if case["transpose"] else 1.0)
    turn = torch.polar(torch.full_like(angle, factor), angle)   # [B, N, 1, A, pairs]
    first = torch.arange(R, device=x.device).view(A, 2, pairs)[:, 0] if case["layout"] == "half" else torch.arange(0, R, 2, device=x.device).view(A, pairs)
    second = first + (pairs if case["layout"] == "half" else 1)
    z = torch.complex(x[:, :, :T][..., first], x[:, :, :T][..., second]) * turn
    y = x.clone()
    head = y[:, :, :T]
    head[..., first.reshape(-1)] = z.real.reshape(*z.shape[:3], -1)
    head[..., second.reshape(-1)] = z.imag.reshape(*z.shape[:3], -1)
    return y


def _exact_attend(s, case):
    """Softmax, weighted sum and the chain rule head by head, a slice of queries at a time."""
    B, H, K, D, nq, nk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "queries", "keys"))
    if B * H * nq * nk > 4e9:
        return None
    dev, scale = s["q"].device, D ** -0.5
    out = torch.zeros(B, nq, H, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, H, nq), -math.inf, dtype=torch.float64, device=dev)
    dq = torch.zeros(B, H, nq, D, dtype=torch.float64, device=dev)
    dk = torch.zeros(B, K, nk, D, dtype=torch.float64, device=dev)
    dv = torch.zeros_like(dk)
    fills = s["lengths"].tolist() if s["lengths"] is not None else [nk] * B
    step = max(1, min(nq, 60000000 // max(1, nk)))
    for b in range(B):
        n = fills[b]
        if n == 0:
            continue
        for h in range(H):
            k, v = s["k"][b, h * K // H, :n].double(), s["v"][b, h * K // H, :n].double()
            for i in range(0, nq, step):
                rows = torch.arange(i, min(nq, i + step), device=dev)
                q = s["q"][b, h, rows].double()
                a = (q @ k.t().contiguous()) * scale
                hidden = torch.zeros(len(rows), n, dtype=torch.bool, device=dev)
                if case["causal"]:
                    hidden |= torch.arange(n, device=dev)[None] > rows[:, None] + (nk - nq)
                if s["mask"] is not None:
                    hidden |= ~s["mask"][b, 0, rows][:, :n]
                a = a.masked_fill(hidden, -math.inf)
                some = ~hidden.all(1)
                part = torch.where(some, torch.logsumexp(a, 1), -math.inf)
                lse[b, h, rows] = part
                p = torch.where(some[:, None], torch.softmax(a, 1), 0.0)
                out[b, rows, h] = p @ v
                if case["train"]:
                    g = s["grad"].view(B, nq, H, D)[b, rows, h].double()
                    slope = g @ v.t().contiguous()
                    slope = p * (slope - (p * slope).sum(1, keepdim=True)) * scale
                    dq[b, h, rows] = slope @ k
                    dk[b, h * K // H, :n] += slope.t().contiguous() @ q
                    dv[b, h * K // H, :n] += p.t().contiguous() @ g
    got = {"out": out.view(B, nq, H * D), "lse": lse}
    return {**got, "dq": dq, "dk": dk, "dv": dv} if case["train"] else got


def _exact_activation(s, case):
    """The formats as lists of the values that they hold: the nearest one, the one with an even code where two are as near."""
    x, w = s["x"].double(), case["width"]
    if case["format"] == "int8":
        values = torch.arange(0, 128, dtype=torch.float64, device=x.device)
    else:
        values = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1],
                              dtype=torch.float64, device=x.device)
    flat = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % 32)).view(-1, 32)
    top = flat.abs().amax(1, keepdim=True)
    power = torch.where(top > 0, torch.log2(torch.where(top > 0, top, 1.0) / values[-1]).ceil(), -126.0).clamp(min=-126)
    power = torch.where(top > values[-1] * torch.exp2(power), power + 1, power)             # the logarithm's own rounding
    power = torch.where(top <= values[-1] * torch.exp2(power - 1), power - 1, power).clamp(min=-126)
    size = flat.abs() / torch.exp2(power)
    between = (values[1:] + values[:-1]) / 2
    below = torch.searchsorted(between, size)                    # a midpoint itself goes to the lower code
    code = below + ((below % 2 == 1) & (below < len(between)) & (size == between[below.clamp(max=len(between) - 1)])).long()
    kept = (values[code] * flat.sign() * torch.exp2(power)).reshape(-1)[:x.numel()].view(x.shape)
    z = kept.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        act = {"gelu": torch.nn.functional.gelu, "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"), "silu": torch.nn.functional.silu}[case["kind"]]
        of = lambda t: act(t[:, :w]) * t[:, w:] if case["gated"] else act(t)  # noqa: E731
        again = of(z)
        dx, = torch.autograd.grad(again, z, s["grad"].double())
    return {"y": of(x), "dx": dx, "again": again.detach()}
