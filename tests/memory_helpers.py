"""The memory operators in 64 bits on the CPU, moment by moment, and the error bounds their tests use.

u = 2^-24 is float32's unit rounding.  A sum of n float32 terms is off by at most about n u times the sum of the terms'
magnitudes, however it is ordered; the bounds below are such counts times the operator applied to magnitudes, plus the
output's own rounding."""
from __future__ import annotations

import torch

U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def turned(x, cs, interleaved, back=False):
    """x [.., H, D] turned by cs [.., 1, R/2, 2] (back: by the negative angles)."""
    R = 2 * cs.shape[-2]
    c, s = cs[..., 0], (-1 if back else 1) * cs[..., 1]
    y = x.clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def turned_magnitude(x, cs, interleaved):
    """The sum of the magnitudes of each turned value's terms."""
    R = 2 * cs.shape[-2]
    x, c, s = x.abs(), cs[..., 0].abs(), cs[..., 1].abs()
    y = x.clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., a] = x[..., a] * c + x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def attention(q, k, v, log_decay, state, scale, starts=None, go=None, gs=None):
    """q [N, T, H, K] (starts: [M, H, K]), k, v with as many heads or fewer, in float64 -> (o, end states), and the
    gradients of q, k, v, state where go is given."""
    H = q.shape[-2]
    share = H // k.shape[-2]
    shape = {n: x.shape for n, x in (("q", q), ("k", k), ("v", v))}
    if starts is None:
        N, T = q.shape[:2]
        spans = [(n * T, (n + 1) * T) for n in range(N)]
        q, k, v = (x.reshape(-1, *x.shape[2:]) for x in (q, k, v))
        go = None if go is None else go.reshape(-1, *go.shape[2:])
    else:
        spans = list(zip(starts[:-1], starts[1:]))
        N = len(spans)
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    K, V = q.shape[2], v.shape[2]
    l = torch.exp(log_decay.double())[:, None, None]
    state = torch.zeros(N, H, K, V, dtype=torch.float64) if state is None else state
    o = torch.zeros(q.shape[0], H, V, dtype=torch.float64)
    end = state.clone()
    dq, dk, dv, ds = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(state)
    for n, (b, e) in enumerate(spans):
        s = state[n].clone()
        for t in range(b, e):
            s = l * s + k[t][:, :, None] * v[t][:, None, :]
            o[t] = scale * (q[t][:, :, None] * s).sum(1)
            if go is not None:
                dq[t] = scale * (s * go[t][:, None, :]).sum(2)
        end[n] = s
        if go is None:
            continue
        g = gs[n].clone() if gs is not None else torch.zeros_like(s)
        for t in range(e - 1, b - 1, -1):
            g = g + scale * q[t][:, :, None] * go[t][:, None, :]
            dk[t] = (g * v[t][:, None, :]).sum(2)
            dv[t] = (g * k[t][:, :, None]).sum(1)
            g = l * g
        ds[n] = g
    out = o.reshape(*shape["q"][:-1], V), end
    if go is None:
        return out
    return (*out, dq.reshape(shape["q"]), dk.unflatten(1, (-1, share)).sum(2).reshape(shape["k"]),
            dv.unflatten(1, (-1, share)).sum(2).reshape(shape["v"]), ds)


def risen(starts, moments):
    """Starts that do not fall, with the same stretches as `starts` where the library gives each moment to one of them: a search
    in rows of 8 bounds, in each up to the first bound past the moment."""
    b, n_seq = [min(max(x, 0), moments) for x in starts], len(starts) - 1
    out = [b[0]]
    for n in range(n_seq):
        lo, low, high = 0, 0, moments
        for step in (4096, 512, 64, 8, 1):
            passed = (n - lo) // step + 1
            low = max(low, *(b[lo + i * step] for i in range(passed)), 0)
            if passed < 8 and lo + passed * step <= n_seq:
                high = min(high, b[lo + passed * step])
            lo += (passed - 1) * step
        assert high <= low or low == out[-1]       # (stretches follow each other)
        out.append(max(high, out[-1]) if high > low else out[-1])
    return out


def within(got, want, magnitude, count, what, extra=0.0):
    """|got - want| at most (count u + extra) magnitude plus the rounding of got's type (and of its smallest numbers)."""
    got64 = got.detach().cpu().double()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    small = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}[got.dtype]
    off = (got64 - want).abs()
    bound = (count * U + extra) * magnitude * (1 + ROUND[got.dtype]) + ROUND[got.dtype] * want.abs() + small
    assert torch.isfinite(got64).all() and (off <= bound).all(), (
        f"{what}: off by {float((off / bound.clamp_min(1e-300)).max()):.3g} of what rounding explains, "
        f"{float(off.max()):.3g} at most")
