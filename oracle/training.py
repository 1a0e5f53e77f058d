"""CPU restatement, in 64 bits, of the operators of a training step beside its
products and attention cores: norms over rows, rotary positions, the norm of the
gradients and the AdamW step (test infrastructure only)."""
from __future__ import annotations

import math

import torch

LOW = 0xFFFFFFFF


# ---- norms over rows -------------------------------------------------------------


def layer_norm(x, weight=None, bias=None, eps=1e-5, rms=False):
    """(y, xh, mean, r) of the rows of x [..., C] in 64 bits."""
    x = x.double()
    mean = torch.zeros_like(x[..., :1]) if rms else x.mean(-1, keepdim=True)
    r = 1.0 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * r
    y = xh if weight is None else xh * weight.double()
    return y if bias is None else y + bias.double(), xh, mean, r


def layer_norm_backward(dy, x, weight=None, eps=1e-5, rms=False):
    """(dx, dweight, dbias) in 64 bits."""
    _, xh, _, r = layer_norm(x, eps=eps, rms=rms)
    dy = dy.double()
    g = dy if weight is None else dy * weight.double()
    dx = g - xh * (g * xh).mean(-1, keepdim=True)
    if not rms:
        dx = dx - g.mean(-1, keepdim=True)
    over_rows = lambda t: t.reshape(-1, t.shape[-1]).sum(0)  # noqa: E731
    return r * dx, over_rows(dy * xh), over_rows(dy)


# ---- rotary positions ------------------------------------------------------------


def rates(dim, base=10000.0, axes=1, scaling=None, factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0):
    """(angles a position of an axis's pairs, amplitude), pair by pair."""
    n = dim // 2 // axes
    out, amplitude = [], 1.0
    for i in range(n):
        if scaling == "ntk" and n > 1:
            f = (base * factor ** (n / (n - 1))) ** (-i / n)
        else:
            f = base ** (-i / n)
        if scaling == "linear":
            f /= factor
        if scaling == "yarn":
            turns = original_length * f / (2 * math.pi)
            keep = min(max((turns - beta_slow) / (beta_fast - beta_slow), 0.0), 1.0)
            f = f * keep + f / factor * (1 - keep)
            amplitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), amplitude


def rotary(x, positions, rate, dim, axes=1, interleaved=False, amplitude=1.0, inverse=False):
    """x [..., heads, head_dim] with the first dim elements of each head turned, in 64 bits; the turns'
    product with a position in 64 bits, brought to one turn exactly."""
    x = x.double()
    turns = rate / (2 * math.pi)
    at = positions.double().unsqueeze(-1)                   # [.., 1] or [.., axes, 1]
    t = (at * turns).flatten(-2) if axes > 1 else at * turns  # [.., dim / 2]
    angle = (t - torch.round(t)) * (2 * math.pi)
    c, s = amplitude * angle.cos().unsqueeze(-2), amplitude * angle.sin().unsqueeze(-2)
    if inverse:
        s = -s
    y = x.clone()
    first, second = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    u, v = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * c - v * s, u * s + v * c
    return y


# ---- the update of the parameters ------------------------------------------------


def gradient_norm(grads, max_norm=None):
    """(norm, factor) in 64 bits."""
    n = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    return n, 1.0 if max_norm is None else min(1.0, max_norm / (n + 1e-6))


def moments(g, m, v, beta1, beta2):
    return beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g


def updated(p, m, v, step, lr, beta1, beta2, eps, decay):
    """(the parameter after the step, what was taken off beside the decay)."""
    d = lr / (1 - beta1 ** step) * m / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return p.double() * (1 - lr * decay) - d, d


def e4m3_values():
    """The values of the codes 0 .. 126 of e4m3, from its definition: 3 bits of
    fraction, an exponent with bias 7, subnormals below 2^-6."""
    return torch.tensor([(c & 7) * 2.0 ** -9 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)],
                        dtype=torch.float64)


def nearest_code(y):
    """(code of the nearest e4m3 value, ties to the even code, saturated; the distance of |y| from the
    border it lies next to, relative to that)."""
    values = e4m3_values()
    borders = (values[1:] + values[:-1]) / 2
    a = y.abs()
    c = torch.bucketize(a, borders)              # a on a border: the lower code
    tie = (c < 126) & (a == borders[c.clamp(max=125)]) & (c % 2 == 1)
    c = (c + tie).clamp(max=126)
    near = torch.minimum((a - borders[(c - 1).clamp(0, 125)]).abs(), (a - borders[c.clamp(0, 125)]).abs())
    return torch.where(torch.signbit(y), c + 128, c).to(torch.uint8), near / a.clamp_min(2.0 ** -10)


def root_code(w, draw):
    """(code of the root of w by its draw, how far the draw's threshold is from deciding otherwise)."""
    values = e4m3_values()
    squares = values.square()
    c = (torch.searchsorted(squares, w, right=True) - 1).clamp(0, 126)
    low, high = squares[c], squares[(c + 1).clamp(max=126)]
    part = torch.where(high > low, (w - low) / (high - low).clamp_min(1e-300), torch.zeros_like(w))
    u = (draw.double() + 0.5) / 65536
    out = torch.where(part > u, c + 1, c)
    return torch.where(w > 0, out.clamp(min=1), torch.zeros_like(out)).to(torch.uint8), (part - u).abs()


def draws(seed, count, tensor, step, stream=0):
    """16-bit draws of elements 0 .. count - 1: Philox4x32-10, counter (element >> 3, tensor, step, stream)."""
    c = [torch.arange(-(-count // 8)), *(torch.full((-(-count // 8),), v) for v in (tensor, step & LOW, stream))]
    k0, k1 = seed & LOW, (seed >> 32) & LOW

    def product(m, v):  # (high, low) of a 32x32 -> 64-bit product, by 16-bit limbs
        high, low = m * (v >> 16), m * (v & 0xFFFF)
        return (high + (low >> 16)) >> 16, (((high & 0xFFFF) << 16) + low) & LOW

    for _ in range(10):
        ha, la = product(0xD2511F53, c[0])
        hb, lb = product(0xCD9E8D57, c[2])
        c = [hb ^ c[1] ^ k0, lb, ha ^ c[3] ^ k1, la]
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack(c, 1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).view(-1)[:count]


# ---- a block with rotary positions -------------------------------------------------


def swin_block_rotary(x, H, W, window, shift, heads, params, rate, dim, interleaved=False, amplitude=1.0, use_attn_mask=True):
    """SequentialSwinTransformer.forward (models/transformer.py:138-298) with rotary
    positions by a token's row and column in its window, in 64 bits; params as
    swin_oracle.swin_block_attention's, those that need a gradient in the graph."""
    from . import swin_oracle as so

    B, _, C = x.shape
    p = {k: v.double() for k, v in params.items() if v.is_floating_point()}
    y = layer_norm(x, p["norm1.weight"], p["norm1.bias"])[0].view(B, H, W, C)
    win = so.partition_frame(y, window, shift, shift)
    at = torch.arange(window * window)
    positions = torch.stack((at // window, at % window), -1)

    def projected(name):
        t = win @ p[f"attn.{name}_linear.weight"].T + p[f"attn.{name}_linear.bias"]
        if name == "v":
            return t
        t = t.unflatten(-1, (heads, C // heads))
        return rotary(t, positions, rate, dim, 2, interleaved, amplitude).flatten(-2)

    mask = so.shift_mask(H, W, window, shift) if shift > 0 and use_attn_mask else None
    o = so.window_attention_core(projected("q"), projected("k"), projected("v"), heads, (C // heads) ** -0.5,
                                 p.get("attn.relative_position_bias_table"), (window, window), mask, compute_dtype=torch.float64)
    o = o @ p["attn.proj.weight"].T + p["attn.proj.bias"]
    return so.reverse_frame(o, B, H, W, window, shift, shift, residual=x.double()).view(B, H * W, C)


def mlp(x, params):
    """SequentialMlp.forward (models/mlp.py:152-172) in 64 bits, in the graph."""
    p = {k: v.double() for k, v in params.items()}
    h = layer_norm(x, p["norm2.weight"], p["norm2.bias"])[0] @ p["fc1.weight"].T + p["fc1.bias"]
    return torch.nn.functional.gelu(h) @ p["fc2.weight"].T + p["fc2.bias"] + x
