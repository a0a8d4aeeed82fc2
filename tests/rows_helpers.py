"""Layer norm and dropout in 64 bits on the CPU, with the magnitudes their error bounds count (tests/memory_helpers.py)."""
from __future__ import annotations

import numpy as np
import torch


def layer_norm(x, w, b, eps, g=None):
    """x [rows, D] in float64, w, b float64 [D] or None -> (y, its magnitude), and with g the gradients of x, w, b, each with its
    magnitude.  A mean of D numbers is off by D u of the mean magnitude A, so a centred number's terms are |x - m| + A."""
    D = x.shape[1]
    m = x.mean(1, keepdim=True)
    off, A = x - m, x.abs().mean(1, keepdim=True)
    r = (off.square().mean(1, keepdim=True) + eps).rsqrt()
    w1 = torch.ones(D, dtype=torch.float64) if w is None else w
    b1 = torch.zeros(D, dtype=torch.float64) if b is None else b
    xh, xm = off * r, (off.abs() + A) * r
    y = [(xh * w1 + b1, xm * w1.abs() + b1.abs())]
    if g is None:
        return y
    u, um = g * w1, (g * w1).abs()
    gx = r * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    mag = r * (um + um.mean(1, keepdim=True) + xm * (um * xm).mean(1, keepdim=True))
    return y + [(gx, mag), ((g * xh).sum(0), (g.abs() * xm).sum(0)), (g.sum(0), g.abs().sum(0))]


def philox(block, offset: int, seed: int):
    """Philox4x32 of 10 rounds of the counters (block, offset) [n] and the key seed -> uint32 [n, 4]."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    block = np.asarray(block, np.uint64)
    c = [block & low, block >> u(32), np.full(len(block), offset & 0xFFFFFFFF, u), np.full(len(block), offset >> 32, u)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [b >> u(32) ^ c[1] ^ u(k[0]), b & low, a >> u(32) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1).astype(np.uint32)


def dropout(x, share, counter):
    """x (any shape, on the CPU) with the share dropped, in x's type: the product in float32, rounded once."""
    seed, offset = (int(v) % (1 << 64) for v in counter)
    t = round(share * 65536)
    draws = philox(np.arange(-(-x.numel() // 8)), offset, seed).astype("<u4").reshape(-1).view("<u2")[:x.numel()]
    kept = torch.from_numpy(draws.astype(np.int32) >= t).view(x.shape)
    f = torch.tensor(65536 / (65536 - t) if t < 65536 else 0.0, dtype=torch.float64).float()
    return torch.where(kept, (x.float() * f).to(x.dtype), torch.zeros((), dtype=x.dtype))
