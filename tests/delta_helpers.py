"""The gated delta rule in 64 bits on the CPU, moment by moment, and the error bounds its tests use."""
from __future__ import annotations

import math

import torch

from memory_helpers import ROUND, U


def delta(q, k, v, log_decay, beta, state, scale, starts=None, go=None, gs=None):
    """q [N, T, H, K] (starts: [M, H, K]), k, v with as many heads or fewer, log_decay, beta [N, T, H], in float64 -> (o, end
    states), and the gradients of q, k, v, log_decay, beta, state where go is given."""
    H = q.shape[-2]
    share = H // k.shape[-2]
    given = (q, k, v, log_decay, beta)
    if starts is None:
        N, T = q.shape[:2]
        spans = [(n * T, (n + 1) * T) for n in range(N)]
        q, k, v, log_decay, beta = (x.reshape(-1, *x.shape[2:]) for x in given)
        go = None if go is None else go.reshape(-1, *go.shape[2:])
    else:
        spans = list(zip(starts[:-1], starts[1:]))
        N = len(spans)
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    K, V = q.shape[2], v.shape[2]
    state = torch.zeros(N, H, K, V, dtype=torch.float64) if state is None else state
    o = torch.zeros(q.shape[0], H, V, dtype=torch.float64)
    end = state.clone()
    dq, dk, dv, dl, db = (torch.zeros_like(x) for x in (q, k, v, log_decay, beta))
    ds = torch.zeros_like(state)
    outer = lambda x, y: x[:, :, None] * y[:, None, :]                    # noqa: E731
    for n, (b, e) in enumerate(spans):
        s, kept = state[n].clone(), []
        for t in range(b, e):
            a = torch.exp(log_decay[t])[:, None, None] * s
            err = v[t] - (k[t][:, :, None] * a).sum(1)
            kept.append((a, err))
            s = a + outer(k[t], beta[t][:, None] * err)
            o[t] = scale * (q[t][:, :, None] * s).sum(1)
            if go is not None:
                dq[t] = scale * (s * go[t][:, None, :]).sum(2)
        end[n] = s
        if go is None:
            continue
        g = gs[n].clone() if gs is not None else torch.zeros_like(s)
        for t in range(e - 1, b - 1, -1):
            a, err = kept[t - b]
            g = g + scale * outer(q[t], go[t])
            du = (g * k[t][:, :, None]).sum(1)
            dv[t] = beta[t][:, None] * du
            db[t] = (du * err).sum(1)
            dk[t] = (g * (beta[t][:, None] * err)[:, None, :]).sum(2) - (a * dv[t][:, None, :]).sum(2)
            g = g - outer(k[t], dv[t])
            dl[t] = (g * a).sum((1, 2))
            g = torch.exp(log_decay[t])[:, None, None] * g
        ds[n] = g
    out = o.reshape(*given[0].shape[:-1], V), end
    if go is None:
        return out
    shared = lambda x, like: x.unflatten(1, (-1, share)).sum(2).reshape(like.shape)               # noqa: E731
    return (*out, dq.reshape(given[0].shape), shared(dk, given[1]), shared(dv, given[2]), dl.reshape(given[3].shape),
            db.reshape(given[4].shape), ds)


def near(got, want, K, V, T, dtype, what):
    """Against `want` in 64 bits, with keys of length 1 at most and rates in (0, 1): every moment's update then shrinks what an
    earlier one was off by, so errors do not grow, they add.  Signs are either way, so n roundings of u add like sqrt(n) u: K + V terms
    of a product, 64 of a chunk, and one per moment; 32 for how much larger than a sum its terms may be.  In 16 bits a product of
    two numbers that are not inputs is off by 2^-17 of its terms in addition (two bfloat16 terms each).  Measured by the
    largest number of the whole, plus the rounding of each number to its type."""
    got64 = got.detach().cpu().double()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    assert torch.isfinite(got64).all(), what
    if not want.numel():
        return
    tol = 32 * U * math.sqrt(K + V + 64 + T) + (0 if dtype == torch.float32 else 32 * 2.0 ** -17)
    off = (got64 - want).abs() - ROUND[got.dtype] * want.abs()
    assert float(off.max()) <= tol * float(want.abs().max()) + 1e-30, (
        f"{what}: off by {float(off.max()):.3g}, {tol:.3g} of the largest, {float(want.abs().max()):.3g}, allowed")
