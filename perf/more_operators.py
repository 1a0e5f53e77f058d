"""What a training step does beside its products and attention cores, as measurable cases.

  layer_norm     LayerNorm and RMS norm over rows of any width, forward and
                 backward with the parameters' gradients
  rotary         rotary positions of query and key heads, forward and backward
  gradient_norm  the norm of many gradients, and the factor that clips it
  adamw          an AdamW step over many tensors, its moments in 32 bits or in 8

``run`` computes them in elementary torch operations, or, where ``own`` is
true, through the framework's entry points.

Moments in 8 bits: blocks of 256 elements of a tensor with one fp32 scale each.
The first moment is an e4m3 code, rounded to nearest, times max |m| / 448.  Of
the second its root is, times max sqrt(v) / 448, and the code is one of the
two neighbours a <= sqrt(v) / scale < b: b where v / scale^2 - a^2 exceeds u (b^2 - a^2), so
that the mean of the squares is v.  u = (draw + 1/2) / 65536; the draws are 16 bits
of Philox4x32-10 with the seed as its key and the counter (element >> 3, tensor, step, 0).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
LOW = 0xFFFFFFFF
BLOCK = 256          # elements that share a scale of 8-bit moments
ALIGN = 64           # tensors of a flat buffer begin at multiples of this
LR, BETAS, ADAM_EPS, DECAY = 3e-4, (0.9, 0.999), 1e-8, 0.05
# Elements of the largest listed case of the norms and of the positions, and values of the largest parameter set.
LARGEST_ROWS = 288 * 544 * 1024
LARGEST_SET = 12 * 12 * 1024 * 1024


def _norm(rows, channels, *, name=None, x="bf16", y=None, params="fp32", rms=False, heads=0, train=True):
    case = dict(op="layer_norm", rows=rows, channels=channels, x=x, y=y or x, params=params, rms=rms, heads=heads,
                train=train)
    return dict(case, name=name) if name else case


def _rotary(batch, tokens, heads, head_dim, *, name=None, dtype="bf16", dim=None, window=0, interleaved=False,
            scaling="none", first=0, spread=1, row_heads=0, train=False):
    case = dict(op="rotary", batch=batch, tokens=tokens, heads=heads, head_dim=head_dim, dtype=dtype, dim=dim or head_dim,
                window=window, interleaved=interleaved, scaling=scaling, first=first, spread=spread,
                row_heads=row_heads or heads, train=train)
    return dict(case, name=name) if name else case


def _set(op, channels, blocks, *, name=None, window=8, heads=8, grads="fp32", params="fp32", bits=32, clip=True, step=1000):
    case = dict(op=op, channels=channels, blocks=blocks, window=window, heads=heads, grads=grads)
    if op == "adamw":
        case.update(params=params, bits=bits, clip=clip, step=step)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token in inference: the shortest call.
        _norm(1, 1024, name="norm_one_token", train=False),
        # Patch merging behind a 288x544 grid of 1024 channels: four neighbours' channels normed as one row.
        _norm(144 * 272, 4096, name="norm_c4096_train"),
        # The fp32 stream of the 512x1024 grid under bf16 autocast, normed into the next product's bf16 input.
        _norm(512 * 1024, 192, name="norm_c192_autocast_train", x="fp32", y="bf16"),
        # Query and key norms: rows are the 8 + 8 heads of 64 of a packed q|k|v, parameters in the activations' type.
        _norm(128 * 256 * 16, 64, name="norm_heads_rms_train", params="bf16", rms=True, heads=24),
        # One token of a decoding step far into a long context: 8 + 8 heads of 128.
        _rotary(1, 1, 16, 128, name="rotary_one_token", first=123456),
        # Query and key heads of 1024-token windows (288x544 grid, 8 heads of 128), positions by row and column, training.
        _rotary(153, 1024, 16, 128, name="rotary_windows_train", window=32, train=True),
        # A long scaled context, neighbours as pairs, half of each head rotated, inside a packed q|k|v.
        _rotary(1, 131072, 10, 64, name="rotary_long_partial", dim=32, interleaved=True, scaling="yarn", spread=7,
                row_heads=12),
        # The gradients of one small block: 17 tensors, most of them a few kilobytes.
        _set("gradient_norm", 96, 1, name="gradient_norm_c96", window=7, heads=3),
        # The bf16 gradients of 12 blocks of the pretrain width.
        _set("gradient_norm", 1024, 12, name="gradient_norm_c1024_bf16", grads="bf16"),
        # One small fp32 block: the shortest optimizer step.
        _set("adamw", 96, 1, name="adamw_c96", window=7, heads=3, clip=False, step=1),
        # 12 blocks of the pretrain width: fp32 parameters and moments, gradients clipped.
        _set("adamw", 1024, 12, name="adamw_c1024"),
        # The same with moments in 8 bits.
        _set("adamw", 1024, 12, name="adamw_c1024_8bit", bits=8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "rotary", "rotary", "gradient_norm", "adamw", "adamw"])
    if op == "layer_norm":
        x = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        y = rng.choice([x, x, "bf16" if x == "fp32" else "fp32"])
        most = LARGEST_ROWS // (4 if "fp32" in (x, y) else 2)
        channels = _log(rng, 16, 16384)
        if rng.random() < 0.6:
            channels = max(8, channels // 8 * 8)
        heads = 0
        rows = _log(rng, 1, min(1 << 20, most // channels))
        if rng.random() < 0.25:
            channels = rng.choice([32, 64, 80, 128])
            heads = rng.choice([9, 12, 24])
            rows = heads // 3 * 2 * _log(rng, 1, min(1 << 16, most // channels // heads))
        return _norm(rows, channels, x=x, y=y, params=rng.choice(["fp32", x]), rms=rng.random() < 0.4, heads=heads,
                     train=rng.random() < 0.7)
    if op == "rotary":
        head_dim = rng.choice([32, 64, 80, 96, 128, 256])
        dim = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4 * 2 - 4])
        heads = rng.choice([1, 2, 6, 10, 16, 40])
        options = dict(dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), interleaved=rng.random() < 0.5,
                       row_heads=heads + rng.choice([0, 0, heads // 2, 1]), train=rng.random() < 0.5)
        if rng.random() < 0.4:
            window = rng.choice([7, 8, 16, 32])
            batch = _log(rng, 1, min(4096, LARGEST_ROWS // 4 // (window * window * heads * head_dim)))
            return _rotary(batch, window * window, heads, head_dim, dim=dim // 4 * 4, window=window, **options)
        batch = rng.choice([1, 1, 3, 32])
        tokens = _log(rng, 1, min(1 << 17, LARGEST_ROWS // 4 // (batch * heads * head_dim)))
        return _rotary(batch, tokens, heads, head_dim, dim=dim, scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                       first=rng.choice([0, 0, _log(rng, 1, 1 << 20)]), spread=rng.choice([1, 1, 5]), **options)
    channels = _log(rng, 12, 1024)
    if rng.random() < 0.6:
        channels = max(8, channels // 8 * 8)
    blocks = _log(rng, 1, max(1, min(24, LARGEST_SET // (13 * channels * channels))))
    options = dict(window=rng.choice([7, 8]), heads=rng.choice([3, 6, 8]))
    if op == "gradient_norm":
        return _set(op, channels, blocks, grads=rng.choice(["fp32", "bf16", "fp16"]), **options)
    params = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    return _set(op, channels, blocks, params=params, grads=rng.choice([params, "fp32"]), bits=rng.choice([32, 8]),
                clip=rng.random() < 0.5, step=_log(rng, 1, 100000), **options)


def _shapes(case):
    """The parameters of Swin blocks: norms, bias table, q, k, v, proj, fc1, fc2."""
    C, table = case["channels"], (2 * case["window"] - 1) ** 2
    linear = [(C, C), (C,)]
    block = [(C,), (C,), (table, case["heads"])] + linear * 4 + [(C,), (C,), (4 * C, C), (4 * C,), (C, 4 * C), (C,)]
    return block * case["blocks"]


def _places(shapes, align):
    """Where each tensor begins in a flat buffer, and the buffer's length."""
    at, end = [], 0
    for s in shapes:
        at.append(end)
        end += -(-math.prod(s) // align) * align
    return at, end


def _views(flat, shapes, at):
    return [flat[a:a + math.prod(s)].view(s) for s, a in zip(shapes, at)]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype="fp32", scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device=DEVICE).mul_(scale).add_(mean).to(DTYPES[dtype])

    return {"layer_norm": _prepare_norm, "rotary": _prepare_rotary, "gradient_norm": _prepare_set,
            "adamw": _prepare_set}[case["op"]](case, gen, normal)


def _prepare_norm(case, gen, normal):
    R, C = case["rows"], case["channels"]
    # A residual stream deep in a network: a mean that is not zero, some channels far larger than the others.
    width = case["heads"] * C if case["heads"] else C
    heads = case["heads"] // 3 * 2
    x = normal(R // heads if heads else R, width, scale=2.0, mean=0.3)
    x[:, ::61] *= 8.0
    x = x.to(DTYPES[case["x"]])
    if heads:  # the query and key heads of a packed q|k|v
        x = x.view(-1, case["heads"], C)[:, :heads]
    state = {"case": case, "x": x, "weight": normal(C, dtype=case["params"], scale=0.2, mean=1.0)}
    if not case["rms"]:
        state["bias"] = normal(C, dtype=case["params"], scale=0.1)
    if case["train"]:
        state["dy"] = normal(*x.shape, dtype=case["y"])
        for name in _leaves(state):
            state[name].requires_grad_(True)
    if own:
        from terra_amd import kernels

        state["norm"] = kernels.Norm(state["weight"], state.get("bias"), EPS, rms=case["rms"])
    return state


def _leaves(state):
    return [n for n in ("x", "weight", "bias") if n in state]


SCALING = {"none": {}, "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=8.0),
           "yarn": dict(scaling="yarn", factor=16.0, original_length=8192)}


def _prepare_rotary(case, gen, normal):
    B, N, H, D, w = case["batch"], case["tokens"], case["heads"], case["head_dim"], case["window"]
    x = normal(B, N, case["row_heads"] * D, dtype=case["dtype"]).view(B, N, case["row_heads"], D)[:, :, :H]
    at = torch.arange(N, device=DEVICE)
    # Windows share the positions of their tokens; sequences have their own, in packed order or with gaps.
    if w:
        positions = torch.stack((at // w, at % w), -1)
    else:
        positions = case["first"] + at * case["spread"] + torch.arange(B, device=DEVICE)[:, None] * 17
    state = {"case": case, "x": x, "positions": positions}
    if case["train"]:
        state["dy"] = normal(B, N, H, D, dtype=case["dtype"])
        x.requires_grad_(True)
    if own:
        from terra_amd import kernels

        state["rotary"] = kernels.Rotary(case["dim"], axes=2 if w else 1, interleaved=case["interleaved"], device=DEVICE,
                                         **SCALING[case["scaling"]])
    return state


def _prepare_set(case, gen, normal):
    shapes = _shapes(case)
    at, total = _places(shapes, ALIGN)
    state = {"case": case, "shapes": shapes}
    # Gradients differ by tensor by orders of magnitude; the gaps between the tensors hold zeros.
    scale = 10.0 ** (torch.rand(len(shapes), generator=gen, device=DEVICE) * 3 - 5)
    sizes = [math.prod(s) for s in shapes]
    spans = [n for a, b, s in zip(at, at[1:] + [total], sizes) for n in (s, b - a - s)]
    level = torch.stack((scale, torch.zeros_like(scale)), -1).view(-1).repeat_interleave(torch.tensor(spans, device=DEVICE))
    state["grads_flat"] = (normal(total) * level).to(DTYPES[case["grads"]])
    state["grads"] = _views(state["grads_flat"], shapes, at)
    if case["op"] == "gradient_norm":
        return state
    state["params_flat"] = (normal(total, scale=0.02) * (level > 0)).to(DTYPES[case["params"]])
    state["params"] = _views(state["params_flat"], shapes, at)
    m = normal(total, scale=0.3) * level
    v = (normal(total).square() * 0.5 + 0.5) * level.square()
    if case["step"] == 1:
        m.zero_(), v.zero_()
    del level
    if case["bits"] == 32:
        state["exp_avg_flat"], state["exp_avg_sq_flat"] = m, v
        firsts, seconds, scales = _views(m, shapes, at), _views(v, shapes, at), [None] * len(shapes)
    else:
        state["seed"] = torch.randint(0, 1 << 62, (1,), generator=gen, device=DEVICE)
        blocks = [(2, -(-math.prod(s) // BLOCK)) for s in shapes]
        scales_at, scales_total = _places(blocks, 1)
        state["scales_flat"] = torch.zeros(scales_total, device=DEVICE)
        scales = _views(state["scales_flat"], blocks, scales_at)
        for name, values in (("exp_avg_flat", m), ("exp_avg_sq_flat", v.sqrt_())):
            state[name] = torch.zeros(total, device=DEVICE, dtype=torch.float8_e4m3fn)
            for s, a, sc in zip(shapes, at, scales):
                rows = _blocks(values[a:a + math.prod(s)])
                one = rows.abs().amax(1) / 448
                sc[0 if name == "exp_avg_flat" else 1] = one
                codes = (rows / one.clamp_min(1e-38)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                state[name].view(torch.uint8)[a:a + math.prod(s)] = codes.view(torch.uint8).view(-1)[:math.prod(s)]
        firsts, seconds = _views(state["exp_avg_flat"], shapes, at), _views(state["exp_avg_sq_flat"], shapes, at)
    state["moments"] = list(zip(firsts, seconds, scales))
    if own:
        from terra_amd import kernels

        state["moments"] = [kernels.Moments(*t) for t in state["moments"]]
    return state


def _blocks(flat):
    """[blocks, 256] of a flat tensor, padded with zeros."""
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_norm, "rotary": _own_rotary, "gradient_norm": _own_gradient_norm,
                "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"layer_norm": _plain_norm, "rotary": _plain_rotary, "gradient_norm": _plain_gradient_norm,
                "adamw": _plain_adamw}[op](state)


# ---- the framework's entry points -------------------------------------------


def _own_norm(state):
    from terra_amd import autograd

    case = state["case"]
    y = autograd.layer_norm(state["x"], state["norm"], out_dtype=DTYPES[case["y"]])
    out = {"y": y.detach()}
    if case["train"]:
        names = _leaves(state)
        out.update(("d" + n, g) for n, g in zip(names, torch.autograd.grad(y, [state[n] for n in names], state["dy"])))
    return out


def _own_rotary(state):
    from terra_amd import autograd

    y = autograd.rotary(state["x"], state["rotary"], state["positions"])
    out = {"y": y.detach()}
    if state["case"]["train"]:
        out["dx"], = torch.autograd.grad(y, state["x"], state["dy"])
    return out


def _own_gradient_norm(state):
    from terra_amd import kernels

    n = kernels.gradient_norm(state["grads"], max_norm=1.0)
    return {"norm": n.norm, "factor": n.factor}


def _own_adamw(state):
    from terra_amd import kernels

    case = state["case"]
    n = kernels.gradient_norm(state["grads"], max_norm=1.0) if case["clip"] else None
    kernels.adamw_step(state["params"], state["grads"], state["moments"], case["step"], lr=LR, betas=BETAS, eps=ADAM_EPS,
                       weight_decay=DECAY, grad_factor=None if n is None else n.factor, seed=state.get("seed"))
    return _updated(state)


def _updated(state):
    return {k: state[k + "_flat"] for k in ("params", "exp_avg", "exp_avg_sq", "scales") if k + "_flat" in state}


# ---- the plain form ----------------------------------------------------------


def _plain_norm(state):
    case = state["case"]
    x, w = state["x"].float(), state["weight"].float()
    if not case["rms"]:
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    hat = x * r
    y = hat * w
    if "bias" in state:
        y = y + state["bias"].float()
    out = {"y": y.to(DTYPES[case["y"]])}
    if case["train"]:
        dy = state["dy"].float()
        g = dy * w
        d = g - hat * (g * hat).mean(-1, keepdim=True)
        if not case["rms"]:
            d = d - g.mean(-1, keepdim=True)
        out["dx"] = (d * r).to(DTYPES[case["x"]])
        over = tuple(range(dy.dim() - 1))
        out["dweight"] = (dy * hat).sum(over, dtype=torch.float64).to(DTYPES[case["params"]])
        if "bias" in state:
            out["dbias"] = dy.sum(over, dtype=torch.float64).to(DTYPES[case["params"]])
    return out


def _frequencies(case):
    """Angles a position of the pairs of one axis, and the amplitude."""
    pairs = case["dim"] // 2 // (2 if case["window"] else 1)
    s = SCALING[case["scaling"]]
    base, factor = 10000.0, s.get("factor", 1.0)
    if case["scaling"] == "ntk" and pairs > 1:
        base *= factor ** (pairs / (pairs - 1))
    f = base ** (-torch.arange(pairs, device=DEVICE, dtype=torch.float64) / pairs)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "yarn":  # pairs that turn more than 32 times within the original length keep their angle
        turns = s["original_length"] * f / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return f, 1.0


def _plain_rotary(state):
    case = state["case"]
    f, a = _frequencies(case)
    at = state["positions"].double()
    angles = (at[..., None] * f).flatten(-2) if case["window"] else at[..., None] * f
    c, s = (angles.cos() * a).float()[..., None, :], (angles.sin() * a).float()[..., None, :]
    out = {"y": _turned(state["x"], c, s, case)}
    if case["train"]:
        out["dx"] = _turned(state["dy"], c, -s, case)
    return out


def _turned(x, c, s, case):
    d = case["dim"]
    v = x.float()
    y = v.clone()
    if case["interleaved"]:
        a, b = v[..., 0:d:2], v[..., 1:d:2]
        y[..., 0:d:2], y[..., 1:d:2] = a * c - b * s, a * s + b * c
    else:
        a, b = v[..., :d // 2], v[..., d // 2:d]
        y[..., :d // 2], y[..., d // 2:d] = a * c - b * s, a * s + b * c
    return y.to(x.dtype)


def _plain_gradient_norm(state):
    total = torch.zeros((), dtype=torch.float64, device=DEVICE)
    for g in state["grads"]:
        total = total + g.float().square().sum(dtype=torch.float64)
    n = total.sqrt()
    return {"norm": n.float(), "factor": (1.0 / (n + 1e-6)).clamp_max(1.0).float()}


def _plain_adamw(state):
    case = state["case"]
    factor = _plain_gradient_norm(state)["factor"] if case["clip"] else 1.0
    b1, b2 = BETAS
    c1, c2 = 1 - b1 ** case["step"], 1 - b2 ** case["step"]
    for i, (p, g, (first, second, scales)) in enumerate(zip(state["params"], state["grads"], state["moments"])):
        if scales is None:
            g = g.float() * factor
            m = first.mul_(b1).add_(g, alpha=1 - b1)
            v = second.mul_(b2).add_(g * g, alpha=1 - b2)
        else:
            # In 64 bits: a value next to a border between two codes has to take the same one every time.
            g = _blocks(g.double().view(-1)) * factor
            m = _blocks(first.float().view(-1)).double() * scales[0].double()[:, None] * b1 + g * (1 - b1)
            v = (_blocks(second.float().view(-1)).double() * scales[1].double()[:, None]).square() * b2 + g * g * (1 - b2)
            _store(m, v, first, second, scales, state["seed"], i, case["step"])
            m, v = (t.view(-1)[:p.numel()].view(p.shape).float() for t in (m, v))
        q = p.float() * (1 - LR * DECAY)
        p.copy_(q - (LR / c1) * m / ((v / c2).sqrt() + ADAM_EPS))
    return _updated(state)


def _store(m, v, first, second, scales, seed, tensor, step):
    """The moments of one tensor as codes and scales."""
    n = first.numel()
    largest, root = m.abs().amax(1), v.amax(1).sqrt()
    scales[0], scales[1] = (largest / 448).float(), (root / 448).float()
    inv = [torch.where(s > 0, 1 / s.double(), torch.zeros((), dtype=torch.float64, device=DEVICE))[:, None] for s in scales]
    y = m * inv[0]
    grid = _grid(y.abs())
    codes = (torch.round(y / grid) * grid).clamp(-448, 448)
    _put(first, codes, n)
    w = v * inv[1] * inv[1]
    r = w.sqrt()
    grid = _grid(r)
    low = (torch.floor(r / grid) * grid).clamp_max(448)
    high = low + grid
    draws = _draws(seed, v.numel(), tensor, step).view_as(v)
    up = (w - low * low > (draws + 0.5) / 65536 * (high * high - low * low)) & (low < 448)
    r = torch.where(up, high, low)
    _put(second, torch.where(w > 0, r.clamp_min(2.0 ** -9), r), n)


def _grid(y):
    """The step of e4m3 at y: 2^-3 of the power of two below, from 2^-6 down 2^-9."""
    _, e = torch.frexp(y)
    return torch.ldexp(torch.ones_like(y), e.clamp(-5, 9) - 4)


def _put(codes, values, n):
    # Every value is one of e4m3's, so the casts do not round.
    codes.view(torch.uint8).view(-1)[:] = values.view(-1)[:n].float().to(torch.float8_e4m3fn).view(torch.uint8)


def _draws(seed, n, tensor, step):
    c0 = torch.arange(-(-n // 8), device=DEVICE)
    c1, c2, c3 = torch.full_like(c0, tensor), torch.full_like(c0, step), torch.zeros_like(c0)
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        # int64 products wrap; their 64 bits are the unsigned product's.
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack((c0, c1, c2, c3), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).view(-1)[:n]


# ---- the definition in 64 bits -----------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"layer_norm": _exact_norm, "rotary": _exact_rotary, "gradient_norm": _exact_gradient_norm,
            "adamw": _exact_adamw}[case["op"]](case, state)


def _exact_norm(case, state):
    names, C = _leaves(state), case["channels"]
    v = {n: state[n].detach().double().requires_grad_(case["train"]) for n in names}
    with torch.enable_grad():
        if case["rms"]:
            y = v["x"] / (v["x"].pow(2).mean(-1, keepdim=True) + EPS).sqrt() * v["weight"]
        else:
            y = torch.nn.functional.layer_norm(v["x"], (C,), v["weight"], v["bias"], EPS)
    out = {"y": y.detach()}
    if case["train"]:
        out.update(("d" + n, g) for n, g in zip(names, torch.autograd.grad(y, [v[n] for n in names], state["dy"].double())))
    return out


def _exact_rotary(case, state):
    """Each pair as a complex number, turned by a unit one."""
    d = case["dim"]
    axes = 2 if case["window"] else 1
    pairs = d // 2 // axes
    s = SCALING[case["scaling"]]
    amplitude, rates = 1.0, []
    for i in range(pairs):
        rate = 10000.0 ** (-i / pairs)
        if case["scaling"] == "linear":
            rate /= s["factor"]
        elif case["scaling"] == "ntk" and pairs > 1:
            rate *= s["factor"] ** (-i / (pairs - 1))
        elif case["scaling"] == "yarn":
            keep = min(max((s["original_length"] * rate / math.tau - 1) / (32 - 1), 0.0), 1.0)
            rate = rate / s["factor"] + keep * (rate - rate / s["factor"])
            amplitude = 1 + math.log(s["factor"]) / 10
        rates.append(rate)
    at = state["positions"].to(torch.float64).unsqueeze(-1)
    angles = (at * torch.tensor(rates, dtype=torch.float64, device=DEVICE)).reshape(*state["positions"].shape[:2 - (axes == 2)], d // 2)
    turn = torch.polar(torch.full_like(angles, amplitude), angles).unsqueeze(-2)

    def turned(t, by):
        t = t.detach().double()
        inner = t[..., :d].unflatten(-1, (d // 2, 2)) if case["interleaved"] else t[..., :d].unflatten(-1, (2, d // 2)).mT
        z = torch.view_as_real(torch.view_as_complex(inner.contiguous()) * by)
        return torch.cat(((z if case["interleaved"] else z.mT).flatten(-2), t[..., d:]), -1)

    out = {"y": turned(state["x"], turn)}
    if case["train"]:
        out["dx"] = turned(state["dy"], turn.conj())
    return out


def _exact_gradient_norm(case, state):
    n = torch.linalg.vector_norm(state["grads_flat"], dtype=torch.float64)
    return {"norm": n, "factor": torch.clamp(1 / (n + 1e-6), max=1.0)}


def _exact_adamw(case, state):
    clip = _exact_gradient_norm(case, state)["factor"] if case["clip"] else 1.0
    if case["bits"] == 8:
        return _exact_adamw_8bit(case, state, clip)
    (b1, b2), t = BETAS, case["step"]
    p, g = state["params_flat"].double(), state["grads_flat"].double() * clip
    m = state["exp_avg_flat"].double()
    m = m + (1 - b1) * (g - m)
    v = state["exp_avg_sq_flat"].double()
    v = v + (1 - b2) * (g * g - v)
    new = p - LR * (DECAY * p + m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + ADAM_EPS))
    return {"params": new, "exp_avg": m, "exp_avg_sq": v}


def _exact_adamw_8bit(case, state, clip):
    """Parameters and scales; the codes are rounded values, which the scales and the definition's draws fix."""
    (b1, b2), t = BETAS, case["step"]
    params, scales = state["params_flat"].double(), state["scales_flat"].double()
    at, _ = _places(state["shapes"], ALIGN)
    begin = 0
    for s, a, g in zip(state["shapes"], at, state["grads"]):
        n = math.prod(s)
        blocks = -(-n // BLOCK)
        own_scales = scales[begin:begin + 2 * blocks].view(2, blocks)
        block_of = torch.arange(n, device=DEVICE) // BLOCK
        g = g.reshape(-1).double() * clip
        m = state["exp_avg_flat"][a:a + n].double() * own_scales[0][block_of]
        r = state["exp_avg_sq_flat"][a:a + n].double() * own_scales[1][block_of]
        m, v = b1 * m + (1 - b1) * g, b2 * r * r + (1 - b2) * g * g
        p = params[a:a + n]
        params[a:a + n] = p - LR * DECAY * p - LR * m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + ADAM_EPS)
        largest = torch.zeros(2, blocks, dtype=torch.float64, device=DEVICE)
        largest.scatter_reduce_(1, block_of.expand(2, n), torch.stack((m.abs(), v.sqrt())), "amax")
        own_scales.copy_(largest / 448)
        begin += 2 * blocks
    return {"params": params, "exp_avg": None, "exp_avg_sq": None, "scales": scales}


def work(case):
    size = lambda t: DTYPES[t].itemsize  # noqa: E731
    if case["op"] == "layer_norm":
        n = case["rows"] * case["channels"]
        params = case["channels"] * size(case["params"]) * (1 if case["rms"] else 2)
        moved, ops = n * (size(case["x"]) + size(case["y"])) + params, 8
        if case["train"]:
            # The pass's gradient arrives after its output is written, so x is read again.
            moved, ops = moved + n * (2 * size(case["x"]) + size(case["y"])) + params, 22
        return {"bytes": moved, "flops": n * ops}
    if case["op"] == "rotary":
        tokens, passes = case["batch"] * case["tokens"], 2 if case["train"] else 1
        n = tokens * case["heads"] * case["head_dim"]
        positions = (case["tokens"] * 2 if case["window"] else tokens) * 8
        return {"bytes": passes * (2 * n * size(case["dtype"]) + positions),
                "flops": passes * 3 * tokens * case["heads"] * case["dim"]}
    n = sum(math.prod(s) for s in _shapes(case))
    if case["op"] == "gradient_norm":
        return {"bytes": n * size(case["grads"]), "flops": 2 * n}
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    # Clipping needs the norm of all gradients before the first of them is used.
    moved = n * (2 * size(case["params"]) + size(case["grads"]) * (2 if case["clip"] else 1) + moments)
    return {"bytes": int(moved), "flops": n * (16 if case["clip"] else 14)}
