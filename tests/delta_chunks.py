"""The gated delta rule in chunks, in float32 on the CPU, with its gradients: how near 64 bits the kernels' sums come in plain float32.
Written from the formulas at the head of csrc/memory_delta.hip: with G the sums of a chunk's log decays, D_ij = exp(G_i - G_j) for
j <= i, E = exp(G), F = exp(G_end - G), S the state before the chunk and X the gradient of the one after it, g that of o:
  T = (I + strict lower(K K^T D) beta)^-1,  P = c lower(Q K^T D) beta,  e = T (v - E K S),  o = c E Q S + P e,  S' = E_end S + K^T (F beta e);
  y = T^T (P^T g + beta F K X),  X' = E_end X + Q^T (c E g) - K^T (E y),  H = c lower(g e^T) D,  Z = -strict lower(y e^T) D,
  gq = c E g S^T + H beta K,  r = -E y S^T + Z beta K,  w = F e X^T + Z^T K + H^T Q,  gk = r + beta w,  gv = y,  gbeta = k . w,
  gG = q . gq + k . r - beta gbeta, at the chunk's end E_end <S, X> + sum of F beta k . (X e) besides."""
from __future__ import annotations

import torch


def kept(x, bits):
    """x with the first `bits` bits of each number, 8 a term as the kernels' sums have them (24: all of a float32)."""
    if bits >= 24:
        return x
    out = torch.zeros_like(x)
    for _ in range(bits // 8):
        out = out + (x - out).bfloat16().to(x.dtype)
    return out


def chunked(q, k, v, log_decay, beta, state, scale, go, gs, chunk, dtype=torch.float32, bits=24):
    """Stretches alike, [N, T, H, ..], as many key as query heads -> (o, end states, the gradients of q, k, v, log_decay, beta,
    state), in `dtype`; bits: of a product's operands."""
    t = lambda x: x.transpose(-1, -2)                         # noqa: E731
    mul = lambda x, y: kept(x, bits) @ kept(y, bits)          # noqa: E731
    q, k, v, go = (x.to(dtype).transpose(1, 2) for x in (q, k, v, go))
    g, b = log_decay.double().transpose(1, 2), beta.to(dtype).transpose(1, 2)[..., None]
    S, X, c = state.to(dtype), gs.to(dtype), scale
    starts = range(0, q.shape[2], chunk)
    held, outs = [], []
    for i in starts:
        Q, K, V, B, go_i = (x[:, :, i:i + chunk] for x in (q, k, v, b, go))
        G = g[:, :, i:i + chunk].cumsum(-1)                   # (in 64 bits)
        low = torch.ones(G.shape[-1], G.shape[-1]).tril().bool()
        D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, -float("inf"))).to(dtype)
        E, F, end = (torch.exp(x)[..., None].to(dtype) for x in (G, G[..., -1:] - G, G[..., -1:]))
        eye = torch.eye(G.shape[-1], dtype=dtype)
        N = (mul(K, t(K)) * D).tril(-1) * t(B)
        T = torch.linalg.solve_triangular(N + eye, eye.expand_as(N), upper=False)
        P = c * mul(Q, t(K)) * D * t(B)
        e = mul(T, V - E * mul(K, S))
        outs.append(c * E * mul(Q, S) + mul(P, e))
        held.append((Q, K, B, go_i, D, E, F, end, T, P, e, S))
        S = end * S + mul(t(K), F * B * e)
    grads = []
    for Q, K, B, go_i, D, E, F, end, T, P, e, S0 in reversed(held):
        y = mul(t(T), mul(t(P), go_i) + B * F * mul(K, X))
        H, Z = c * mul(go_i, t(e)).tril() * D, -mul(y, t(e)).tril(-1) * D
        gq = c * E * mul(go_i, t(S0)) + mul(H, B * K)
        r = -E * mul(y, t(S0)) + mul(Z, B * K)
        from_end = F * mul(e, t(X))
        w = from_end + mul(t(Z), K) + mul(t(H), Q)
        gb = (K * w).sum(-1)
        gG = (Q * gq).sum(-1) + (K * r).sum(-1) - B[..., 0] * gb
        at_end = end[..., 0] * (S0 * X).sum((-1, -2))[..., None] + (B[..., 0] * (K * from_end).sum(-1)).sum(-1, keepdim=True)
        grads.append((gq, r + B * w, y, gG.flip(-1).cumsum(-1).flip(-1) + at_end, gb))
        X = end * X + mul(t(Q), c * E * go_i) - mul(t(K), E * y)
    whole = [torch.cat(x, 2).transpose(1, 2) for x in zip(*reversed(grads))]
    return (torch.cat(outs, 2).transpose(1, 2), S, *whole, X)


def off_by_head(got, want, heads_at):
    """For each head (dimension `heads_at`), the 2-norm of what `got` is off by."""
    d = (got.detach().cpu().double() - want).movedim(heads_at, 0).flatten(1)
    return d.norm(dim=1)
