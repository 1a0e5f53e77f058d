"""CPU restatement, in 64 bits, of the regularised training operators:
counter-based dropout, GELU followed by dropout, and the end of a half-block
(post-norm, dropout, gate, scaled residual, next norm), with gradients by
torch autograd over float64 tensors.  Test infrastructure only."""
from __future__ import annotations

import math
from typing import Optional

import numpy as np
import torch

LOW = np.uint64(0xFFFFFFFF)
S32 = np.uint64(32)


def philox4x32_10(counter, key):
    """Philox4x32-10 of four counter words and two key words (arrays of
    uint64 below 2^32, broadcast together); the four result words."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    c = list(np.broadcast_arrays(*c))
    k = [np.uint64(v) for v in key]
    with np.errstate(over="ignore"):
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> S32) ^ c[1] ^ k[0], b & LOW, (a >> S32) ^ c[3] ^ k[1], a & LOW]
            k = [(k[0] + np.uint64(0x9E3779B9)) & LOW, (k[1] + np.uint64(0xBB67AE85)) & LOW]
    return c


def threshold(p: float) -> int:
    return int(math.floor(p * 65536 + 0.5))


def keep_mask(seed: int, rows: int, columns: int, p: float, stream: int = 0, first_row: int = 0) -> torch.Tensor:
    """The kept elements of [rows, columns]."""
    seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    row = np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None]
    chunk = np.arange((columns + 7) // 8, dtype=np.uint64)[None, :]
    words = philox4x32_10((chunk, row & LOW, row >> S32, np.uint64(stream)), (seed & 0xFFFFFFFF, seed >> 32))
    draws = np.empty((rows, chunk.shape[1], 8), dtype=np.uint64)
    for j in range(8):
        draws[:, :, j] = (words[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF)
    return torch.from_numpy((draws.reshape(rows, -1)[:, :columns] >= threshold(p)).copy())


def keep_scale(p: float) -> float:
    t = threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def dropout(x: torch.Tensor, p: float, seed: int, stream: int = 0) -> torch.Tensor:
    """x [..., C] in float64; dropped elements are 0 whatever they were."""
    if threshold(p) == 0:
        return x
    C = x.shape[-1]
    keep = keep_mask(seed, x.numel() // C, C, p, stream).view(x.shape)
    return torch.where(keep, x * keep_scale(p), torch.zeros((), dtype=x.dtype))


def gelu(h: torch.Tensor) -> torch.Tensor:
    return 0.5 * h * torch.erfc(-h / math.sqrt(2.0))


def norm(v: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float, rms: bool):
    d = v if rms else v - v.mean(-1, keepdim=True)
    v = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    v = v if weight is None else v * weight
    return v if bias is None else v + bias


def window_sources(geom) -> torch.Tensor:
    """For each grid token its row of the window tensor, -1 where no emitted,
    valid window holds it: every window token walked one by one."""
    at = torch.full((geom.batch * geom.height * geom.width,), -1, dtype=torch.int64)
    Hp, Wp, ws = geom.frame_h, geom.frame_w, geom.window
    row = 0
    for b in range(geom.batch):
        for w in range(geom.windows_per_image):
            wr, wc = divmod(w, geom.cols)
            valid = geom.valid is None or geom.valid[0] <= w < geom.valid[1]
            for t in range(ws * ws):
                i = ((wr + geom.win_row_begin) * ws + t // ws + geom.shift_h) % Hp - geom.pad[0]
                j = (wc * ws + t % ws + geom.shift_w) % Wp - geom.pad[2]
                if valid and 0 <= i < geom.height and 0 <= j < geom.width:
                    at[(b * geom.height + i) * geom.width + j] = row
                row += 1
    return at


def residual_norm(h, x, post=None, gate=None, nxt=None, geom=None, residual_scale=1.0, p=0.0, seed=0, stream=0):
    """(y, z): float64 tensors, z None without ``nxt``.  post, nxt: (weight,
    bias, eps, rms) or None; gate [C] or [B, C]."""
    C = x.shape[-1]
    n = h.reshape(-1, C)
    have = None
    if geom is not None:
        src = window_sources(geom)
        have = (src >= 0)[:, None]
        n = n[src.clamp(min=0)]
    if post is not None:
        n = norm(n, *post)
    if have is not None:
        n = torch.where(have, n, torch.zeros((), dtype=n.dtype))
    m = dropout(n, p, seed, stream)
    if gate is not None:
        m = (m.view(gate.shape[0], -1, C) * gate[:, None]).view(-1, C) if gate.dim() == 2 else m * gate
    y = residual_scale * x + m.view(x.shape)
    return y, None if nxt is None else norm(y, *nxt)
