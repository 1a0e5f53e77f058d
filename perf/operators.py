"""The operators of a regularised block tail, as measurable cases.

Three operators that training a Swin block with regularisation runs beside its
attention and its GEMMs:

  dropout        y = keep * s * x, forward and backward, the mask drawn from a
                 counter-based generator and never stored
  gelu_dropout   a = keep * s * GELU(h) between fc1 and fc2, its backward and
                 fc1's bias gradient
  residual_norm  the end of a half-block: the branch's post-norm, dropout, gate,
                 the scaled residual, and the norm that the next half-block
                 begins with; the branch in row order or in window order

``run`` computes them in elementary torch operations, or, where ``own`` is
true, through the framework's entry points.

The mask: Philox4x32-10 with the 64-bit seed as its key and the counter
(column >> 3, row low, row high, stream); the four words are eight 16-bit draws
for the eight columns of a chunk, low half first.  An element is dropped where
its draw is below round(p * 65536) = t; the others are scaled by 65536 / (65536 - t).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
LOW = 0xFFFFFFFF
# Elements of the largest listed case: no drawn case has more.
LARGEST = 156672 * 1024


def _dropout(rows, channels, *, name=None, dtype="bf16", p=0.1, train=False):
    case = dict(op="dropout", rows=rows, channels=channels, dtype=dtype, p=p, train=train)
    return dict(case, name=name) if name else case


def _gelu(rows, channels, *, name=None, dtype="bf16", p=0.1, train=True):
    case = dict(op="gelu_dropout", rows=rows, channels=channels, dtype=dtype, p=p, train=train)
    return dict(case, name=name) if name else case


def _tail(rows, channels, *, name=None, batch=1, branch="bf16", stream="bf16", post="layer", next="layer", gate="channel",
          alpha=1.0, p=0.0, train=False, window=0, height=0, width=0, pad_bottom=0):
    case = dict(op="residual_norm", batch=batch, rows=rows, channels=channels, branch=branch, stream=stream, post=post,
                next=next, gate=gate, alpha=alpha, p=p, train=train, window=window, height=height, width=width,
                pad_bottom=pad_bottom)
    return dict(case, name=name) if name else case


def listed():
    return [
        # Dropout of the tokens of one small fp32 image (56x56, C = 96): the shortest call, bound by its launch.
        _dropout(56 * 56, 96, name="dropout_fp32_c96", dtype="fp32"),
        # Dropout of the embedded 512x1024 grid before the first block, both directions.
        _dropout(512 * 1024, 192, name="dropout_c192_train", p=0.05, train=True),
        # The hidden layer of a small batch of 112x112 grids (4 x 128 features) in training.
        _gelu(4 * 112 * 112, 512, name="gelu_c128_train"),
        # The same for the 512x1024 grid at C = 192.
        _gelu(512 * 1024, 768, name="gelu_c192_train"),
        # A ragged hidden layer in fp16: an odd number of rows, features that are no whole 16-byte chunks.
        _gelu(2001, 770, name="gelu_fp16_ragged_train", dtype="fp16", p=0.25),
        # One token in inference: the fewest rows there are.
        _tail(1, 1024, name="tail_one_token"),
        # The fp32 block of the small image in training.
        _tail(56 * 56, 96, name="tail_fp32_c96_train", branch="fp32", stream="fp32", p=0.1, train=True),
        # Inference of a wide block on a 128x256 grid: post-norm, layer scale, residual and the next norm.
        _tail(128 * 256, 768, name="tail_c768"),
        # The attention half of the 512x1024 grid under bf16 autocast: the bf16 proj output in window order (8x8
        # windows, shift 4), the fp32 stream, layer scale and dropout, the MLP half's norm.
        _tail(512 * 1024, 192, name="tail_windows_c192_train", stream="fp32", post="none", p=0.1, train=True, window=8,
              height=512, width=1024),
        # The widest pretrain grid (288x544 tokens, C = 1024), everything on.
        _tail(288 * 544, 1024, name="tail_c1024_train", p=0.1, train=True),
        # Three samples of an odd number of odd rows, a gate of each sample's own, RMS norms, fp16.
        _tail(2001, 385, name="tail_fp16_sample_gate_train", batch=3, branch="fp16", stream="fp16", post="rms",
              next="rms", gate="sample", alpha=0.75, p=0.15, train=True),
        # Rows of 4096 channels in inference: a row that no one wave holds.
        _tail(8192, 4096, name="tail_c4096", post="rms", next="rms", gate="none"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["dropout", "gelu_dropout", "residual_norm", "residual_norm"])
    p = round(rng.uniform(0.02, 0.5), 3)
    train = rng.random() < 0.7
    if op != "residual_norm":
        channels = _log(rng, 16, 4096)
        if rng.random() < 0.7:
            channels = max(8, channels // 8 * 8)
        rows = _log(rng, 1, min(1 << 19, LARGEST // 2 // channels))
        make = _dropout if op == "dropout" else _gelu
        return make(rows, channels, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), p=p, train=train)
    branch, stream = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
    norms = dict(post=rng.choice(["none", "layer", "rms"]), next=rng.choice(["none", "layer", "rms"]),
                 alpha=rng.choice([1.0, 1.0, 0.75]), p=rng.choice([0.0, p]), train=train, branch=branch, stream=stream)
    most = LARGEST // (2 if branch == "fp32" or stream == "fp32" else 1) // 2
    if rng.random() < 0.4:
        window, channels = rng.choice([(7, 96), (7, 128), (8, 192), (8, 384), (8, 768), (8, 1024)])
        pad = rng.choice([0, 0, window])
        height, width = window * rng.randint(2, 24), window * rng.randint(1, 48)
        return _tail(height * width, channels, batch=rng.randint(1, 3), window=window, height=height, width=width,
                     pad_bottom=pad, gate=rng.choice(["none", "channel", "sample"]), **norms)
    channels = _log(rng, 16, 8192)
    if rng.random() < 0.7:
        channels = max(8, channels // 8 * 8)
    batch = rng.choice([1, 1, 2, 5])
    rows = _log(rng, 1, min(1 << 18, most // channels // batch))
    return _tail(rows, channels, batch=batch, gate=rng.choice(["none", "channel", "sample"]), **norms)


def _frame(case):
    """Rows of h in window order (the padded frame's tokens), or the stream's own."""
    if case["window"]:
        return case["batch"] * (case["height"] + case["pad_bottom"]) * case["width"]
    return case["batch"] * case["rows"]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype="fp32", scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device=DEVICE).mul_(scale).add_(mean).to(DTYPES[dtype])

    state = {"case": case, "seed": torch.randint(0, 1 << 62, (1,), generator=gen, device=DEVICE)}
    rows, C, train = case["rows"], case["channels"], case["train"]
    if case["op"] != "residual_norm":
        state["x"] = normal(rows, C, dtype=case["dtype"], scale=1.5)
        if train:
            state["dy"] = normal(rows, C, dtype=case["dtype"])
        return state
    B, branch, stream = case["batch"], case["branch"], case["stream"]
    if case["window"]:
        ws = case["window"]
        grid = (B, case["height"], case["width"], C)
        state["h"] = normal(_frame(case) // ws ** 2, ws * ws, C, dtype=branch, scale=0.8, mean=0.1)
    else:
        grid = (B, rows, C)
        state["h"] = normal(*grid, dtype=branch, scale=0.8, mean=0.1)
    # A residual stream deep in a network: a mean that is not zero, some channels far larger than the others.
    x = torch.randn(grid, generator=gen, device=DEVICE).mul_(2.0).add_(0.3)
    x[..., ::61] *= 8.0
    state["x"] = x.to(DTYPES[stream])
    for which in ("post", "next"):
        if case[which] != "none":
            state[which + "_weight"] = normal(C, scale=0.2, mean=1.0)
        if case[which] == "layer":
            state[which + "_bias"] = normal(C, scale=0.1)
    if case["gate"] == "channel":
        state["gate"] = normal(C, scale=0.2, mean=0.3)
    elif case["gate"] == "sample":  # from a conditioning network, in the activations' type
        state["gate"] = normal(B, C, dtype=branch, scale=0.5)
    if train:
        state["dy"] = normal(*grid, dtype=stream)
        if case["next"] != "none":
            state["dz"] = normal(*grid, dtype=branch)
        for name in _leaves(state):
            state[name].requires_grad_(True)
    return state


def _leaves(state):
    return [n for n in ("h", "x", "post_weight", "post_bias", "gate", "next_weight", "next_bias") if n in state]


def run(state):
    case = state["case"]
    if own:
        return {"dropout": _own_dropout, "gelu_dropout": _own_gelu, "residual_norm": _own_tail}[case["op"]](state)
    with torch.no_grad():
        return {"dropout": _plain_dropout, "gelu_dropout": _plain_gelu, "residual_norm": _plain_tail}[case["op"]](state)


# ---- the framework's entry points -------------------------------------------


def _own_dropout(state):
    from terra_amd import kernels

    case = state["case"]
    out = {"y": kernels.dropout(state["x"], case["p"], state["seed"], stream=1)}
    if case["train"]:  # the gradient's kernel is the same one
        out["dx"] = kernels.dropout(state["dy"], case["p"], state["seed"], stream=1)
    return out


def _own_gelu(state):
    from terra_amd import kernels

    case = state["case"]
    out = {"a": kernels.gelu_dropout(state["x"], case["p"], state["seed"], stream=2)}
    if case["train"]:
        out["dh"], out["db"] = kernels.gelu_dropout_backward(state["dy"], state["x"], case["p"], state["seed"], stream=2,
                                                             column_sums=True)
    return out


def _own_tail(state):
    from terra_amd import autograd, kernels

    case = state["case"]
    norms = {}
    for which in ("post", "next"):
        if case[which] != "none":
            norms[which + "_norm"] = kernels.Norm(state[which + "_weight"], state.get(which + "_bias"), EPS,
                                                  rms=case[which] == "rms")
    geom = None
    if case["window"]:
        ws = case["window"]
        geom = kernels.WindowGeometry(case["batch"], case["height"], case["width"], case["channels"], ws, ws // 2, ws // 2,
                                      (0, case["pad_bottom"], 0, 0))
    out = autograd.residual_norm(state["h"], state["x"], gate=state.get("gate"), geom=geom, residual_scale=case["alpha"],
                                 p=case["p"], seed=state["seed"], stream=3, **norms)
    outs = dict(zip(("y", "z"), out)) if case["next"] != "none" else {"y": out}
    if case["train"]:
        names = _leaves(state)
        grads = torch.autograd.grad(list(outs.values()), [state[n] for n in names],
                                    [state["d" + k] for k in outs])
        outs.update(("d" + n, g) for n, g in zip(names, grads))
        outs["y"] = outs["y"].detach()
        if "z" in outs:
            outs["z"] = outs["z"].detach()
    return outs


# ---- the plain form ----------------------------------------------------------


def _keep(state, rows, stream):
    """The kept elements' mask [rows, C] and their scale."""
    case = state["case"]
    C = case["channels"]
    t = int(math.floor(case["p"] * 65536 + 0.5))
    if t == 0:
        return None, 1.0
    chunks = (C + 7) // 8
    row = torch.arange(rows, device=DEVICE).view(-1, 1)
    c0 = torch.arange(chunks, device=DEVICE).view(1, -1).expand(rows, chunks)
    c1, c2 = (row & LOW).expand(rows, chunks), (row >> 32).expand(rows, chunks)
    c3 = torch.full_like(c1, stream)
    k0, k1 = state["seed"] & LOW, (state["seed"] >> 32) & LOW
    for _ in range(10):
        # int64 products wrap; their 64 bits are the unsigned product's.
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack((c0, c1, c2, c3), -1)
    draws = torch.stack((words & 0xFFFF, words >> 16), -1).view(rows, chunks * 8)[:, :C]
    return draws >= t, 65536 / (65536 - t) if t < 65536 else 0.0


def _dropped(x, keep, scale):
    return x if keep is None else torch.where(keep, x * scale, torch.zeros((), device=DEVICE))


def _plain_dropout(state):
    case = state["case"]
    keep, scale = _keep(state, case["rows"], 1)
    dt = DTYPES[case["dtype"]]
    out = {"y": _dropped(state["x"].float(), keep, scale).to(dt)}
    if case["train"]:
        out["dx"] = _dropped(state["dy"].float(), keep, scale).to(dt)
    return out


def _plain_gelu(state):
    case = state["case"]
    keep, scale = _keep(state, case["rows"], 2)
    dt = DTYPES[case["dtype"]]
    h = state["x"].float()
    cdf = 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5)))
    out = {"a": _dropped(h * cdf, keep, scale).to(dt)}
    if case["train"]:
        slope = cdf + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2.0 * math.pi))
        dh = _dropped(state["dy"].float() * slope, keep, scale)
        out["dh"], out["db"] = dh.to(dt), dh.sum(0, dtype=torch.float64).float()
    return out


def _to_grid(h, case):
    """Window order -> the grid's rows [B, H * W, C] (reverse, roll back, crop)."""
    B, ws, C = case["batch"], case["window"], case["channels"]
    Hp, W = case["height"] + case["pad_bottom"], case["width"]
    g = h.view(B, Hp // ws, W // ws, ws, ws, C).permute(0, 1, 3, 2, 4, 5).reshape(B, Hp, W, C)
    g = torch.roll(g, (ws // 2, ws // 2), (1, 2))
    return g[:, :case["height"]].reshape(B, -1, C)


def _to_windows(g, case):
    """The adjoint: the grid's rows -> window order, zero where the frame is padding."""
    B, ws, C = case["batch"], case["window"], case["channels"]
    Hp, W = case["height"] + case["pad_bottom"], case["width"]
    full = torch.zeros(B, Hp, W, C, dtype=g.dtype, device=DEVICE)
    full[:, :case["height"]] = g.view(B, case["height"], W, C)
    full = torch.roll(full, (-(ws // 2), -(ws // 2)), (1, 2))
    return full.view(B, Hp // ws, ws, W // ws, ws, C).permute(0, 1, 3, 2, 4, 5).reshape(-1, ws * ws, C)


def _normed(v, kind):
    """(v - mean) * r and r over the last dimension; RMS norms take no mean off."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * r, r


def _norm_grad(g, hat, r, kind):
    """The gradient through _normed for the gradient g of its result."""
    d = g - hat * (g * hat).mean(-1, keepdim=True)
    return r * (d - g.mean(-1, keepdim=True) if kind == "layer" else d)


def _plain_tail(state):
    case = state["case"]
    B, C, post, nxt = case["batch"], case["channels"], case["post"], case["next"]
    R = case["rows"]
    branch, stream = DTYPES[case["branch"]], DTYPES[case["stream"]]
    h = state["h"].float()
    h = _to_grid(h, case) if case["window"] else h
    x = state["x"].float().view(B, R, C)
    gate = state["gate"].float().view(-1, 1, C) if "gate" in state else None
    keep, scale = _keep(state, B * R, 3)
    keep = None if keep is None else keep.view(B, R, C)
    n = h
    if post != "none":
        hat1, r1 = _normed(h, post)
        n = hat1 * state["post_weight"]
        if "post_bias" in state:
            n = n + state["post_bias"]
    m = _dropped(n, keep, scale)
    y = case["alpha"] * x + (m if gate is None else gate * m)
    shape = state["x"].shape
    out = {"y": y.to(stream).view(shape)}
    if nxt != "none":
        hat2, r2 = _normed(y, nxt)
        z = hat2 * state["next_weight"]
        if "next_bias" in state:
            z = z + state["next_bias"]
        out["z"] = z.to(branch).view(shape)
    if not case["train"]:
        return out
    total = lambda t: t.sum((0, 1), dtype=torch.float64).float()  # noqa: E731
    d = state["dy"].float().view(B, R, C)
    if nxt != "none":
        dz = state["dz"].float().view(B, R, C)
        out["dnext_weight"] = total(dz * hat2)
        if "next_bias" in state:
            out["dnext_bias"] = total(dz)
        d = d + _norm_grad(dz * state["next_weight"], hat2, r2, nxt)
    out["dx"] = (case["alpha"] * d).to(stream).view(shape)
    if gate is not None:
        dg = d * m
        out["dgate"] = total(dg) if case["gate"] == "channel" else dg.sum(1, dtype=torch.float64).to(branch)
    dn = _dropped(d if gate is None else d * gate, keep, scale)
    if post != "none":
        out["dpost_weight"] = total(dn * hat1)
        if "post_bias" in state:
            out["dpost_bias"] = total(dn)
        dn = _norm_grad(dn * state["post_weight"], hat1, r1, post)
    dn = dn.to(branch)
    out["dh"] = _to_windows(dn, case) if case["window"] else dn
    return out


# ---- the definition in 64 bits -----------------------------------------------


def _philox_chunk(seed, row, chunk, stream):
    """Philox4x32-10 of counters (chunk, row low, row high, stream): the high halves of the products are put together
    from 16-bit limbs."""
    def product(m, v):
        high = m * (v >> 16)             # < 2^48
        low = m * (v & 0xFFFF)
        return (high + (low >> 16)) >> 16, (((high & 0xFFFF) << 16) + low) & LOW

    key = (seed & LOW, (seed >> 32) & LOW)
    v = [chunk + 0 * row, (row & LOW) + 0 * chunk, (row >> 32) + 0 * chunk, stream + 0 * (row + chunk)]
    for i in range(10):
        ka, kb = (key[0] + i * 0x9E3779B9) & LOW, (key[1] + i * 0xBB67AE85) & LOW
        hi0, lo0 = product(0xD2511F53, v[0])
        hi1, lo1 = product(0xCD9E8D57, v[2])
        v = [hi1 ^ v[1] ^ ka, lo1, hi0 ^ v[3] ^ kb, lo0]
    return v


def _factor(state, rows, stream):
    """What dropout multiplies each element of [rows, C] by, in 64 bits; None without dropout."""
    case = state["case"]
    C, t = case["channels"], int(round(case["p"] * 65536))
    if t == 0:
        return None
    factor = torch.empty(rows, C, dtype=torch.float64, device=DEVICE)
    one = 65536.0 / (65536.0 - t)
    words = _philox_chunk(int(state["seed"]), torch.arange(rows, device=DEVICE)[:, None],
                          torch.arange((C + 7) // 8, device=DEVICE)[None, :], stream)
    for j in range(8):
        cols = len(range(j, C, 8))
        bits = (words[j // 2] >> (16 if j % 2 else 0)) % 65536
        factor[:, j::8] = one * (bits >= t)[:, :cols]
    return factor


def exact(case, seed):
    state = prepare(case, seed)
    return {"dropout": _exact_dropout, "gelu_dropout": _exact_gelu, "residual_norm": _exact_tail}[case["op"]](case, state)


def _times(v, factor):
    return v if factor is None else v * factor


def _exact_dropout(case, state):
    f = _factor(state, case["rows"], 1)
    out = {"y": _times(state["x"].double(), f)}
    if case["train"]:
        out["dx"] = _times(state["dy"].double(), f)
    return out


def _exact_gelu(case, state):
    f = _factor(state, case["rows"], 2)
    h = state["x"].double().requires_grad_(case["train"])
    with torch.enable_grad():
        a = _times(0.5 * h * torch.erfc(-h / math.sqrt(2.0)), f)
    if not case["train"]:
        return {"a": a}
    dh, = torch.autograd.grad(a, h, state["dy"].double())
    return {"a": a.detach(), "dh": dh, "db": dh.sum(0)}


def _norm64(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        return torch.nn.functional.layer_norm(v, v.shape[-1:], weight, bias, EPS)
    return v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight


def _source_rows(case):
    """For each row of the stream its row of h: token ids put through pad, roll and partition, and inverted."""
    B, H, W, ws = case["batch"], case["height"], case["width"], case["window"]
    ids = torch.full((B, H + case["pad_bottom"], W), -1, device=DEVICE)
    ids[:, :H] = torch.arange(B * H * W, device=DEVICE).view(B, H, W)
    ids = ids.roll((-(ws // 2), -(ws // 2)), (1, 2))
    order = torch.cat([ids[b, i:i + ws].unfold(1, ws, ws).permute(1, 0, 2).reshape(-1)
                       for b in range(B) for i in range(0, ids.shape[1], ws)])
    at = torch.empty(B * H * W, dtype=torch.int64, device=DEVICE)
    held = order >= 0
    at[order[held]] = torch.arange(order.numel(), device=DEVICE)[held]
    return at


def _exact_tail(case, state):
    names = _leaves(state)
    C = case["channels"]
    v = {n: state[n].detach().double().requires_grad_(case["train"]) for n in names}
    f = _factor(state, case["batch"] * case["rows"], 3)
    with torch.enable_grad():
        h = v["h"].reshape(-1, C)
        if case["window"]:
            h = h[_source_rows(case)]
        m = _times(_norm64(h, case["post"], v.get("post_weight"), v.get("post_bias")), f)
        m = m.view(case["batch"], -1, C)
        if "gate" in v:
            m = m * (v["gate"] if case["gate"] == "channel" else v["gate"][:, None])
        y = v["x"] * case["alpha"] + m.view(v["x"].shape)
        out = {"y": y}
        if case["next"] != "none":
            out["z"] = _norm64(y, case["next"], v.get("next_weight"), v.get("next_bias"))
    if not case["train"]:
        return out
    grads = torch.autograd.grad(list(out.values()), [v[n] for n in names], [state["d" + k].double() for k in out])
    out = {k: t.detach() for k, t in out.items()}
    out.update(("d" + n, g) for n, g in zip(names, grads))
    return out


def work(case):
    C, train = case["channels"], case["train"]
    if case["op"] != "residual_norm":
        n, e = case["rows"] * C, DTYPES[case["dtype"]].itemsize
        passes = 2 if not train else 4
        gelu = case["op"] == "gelu_dropout"
        return {"bytes": n * e * passes + (4 * C if gelu and train else 0), "flops": n * ((12 if gelu else 1) * passes // 2)}
    rows = case["batch"] * case["rows"]
    h, x = DTYPES[case["branch"]].itemsize, DTYPES[case["stream"]].itemsize
    n, frame = rows * C, _frame(case) * C
    nxt = case["next"] != "none"
    params = C * 4 * ((case["post"] != "none") + (case["post"] == "layer") + nxt + (case["next"] == "layer")
                      + (case["gate"] == "channel"))
    if case["gate"] == "sample":
        params += case["batch"] * C * h
    ops = 4 + (8 if case["post"] != "none" else 0) + (8 if nxt else 0)
    # Padding rows of a window-order branch are never read.
    moved = n * (h + x) + n * x + (n * h if nxt else 0) + params
    if train:
        moved += n * x + (n * h if nxt else 0) + n * x + frame * h + params
        ops *= 3
    return {"bytes": moved, "flops": n * ops}
