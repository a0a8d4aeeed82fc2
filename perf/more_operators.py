"""More operators of the memory over decisions whose speed is tracked, through the package's public entry points: a memory
that corrects itself, and what its teaching puts around it.

A case names an operator:
  delta      the gated delta rule over whole stretches of moments (flyguy_amd.memory_hip.delta_attention): each moment the
             state decays, and what it holds under the moment's key is moved towards the moment's value
  delta_step the same for one new moment of each car, on the cars' states (delta_step)
  layer_norm rows of numbers (the network's firing) centred, divided by their deviation, scaled and shifted
             (flyguy_amd.rows_hip.layer_norm)
  dropout    numbers dropped by a counter-based generator, the mask made again for the gradient (rows_hip.dropout)
and its sizes.  delta, delta_step: seqs stretches (cars) of moments moments each, q_heads query heads (each with a state, a
decay and a rate of its own each moment) and k_heads key / value heads (query heads share them in consecutive groups), dim
values of a query or key, v_dim of a value.  layer_norm, dropout: rows x width numbers.  dtype "float32", "bfloat16" or
"float16" of the inputs and outputs; gates, weights and states are float32.  grad: the pass is the forward and the gradients
of everything that learns.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the package's kernels.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
CHUNK = 64                               # moments per chunk of the plain form


def listed() -> list[dict]:
    return [
        # one car's new moment: the smallest call, its latency counts
        {"name": "delta_step_one", "op": "delta_step", "seqs": 1, "q_heads": 8, "k_heads": 8, "dim": 64, "v_dim": 64,
         "dtype": "float32"},
        # a few hundred environments acting at once: bound by reading and writing their states
        {"name": "delta_step_acting", "op": "delta_step", "seqs": 416, "q_heads": 8, "k_heads": 8, "dim": 128, "v_dim": 128,
         "dtype": "bfloat16"},
        # one whole recording read in before play goes on: few long sequences
        {"name": "delta_game", "op": "delta", "seqs": 1, "moments": 32768, "q_heads": 8, "k_heads": 8, "dim": 128,
         "v_dim": 128, "ragged": False, "dtype": "bfloat16", "grad": False},
        # packed recordings of different lengths, each going on from a state of its own
        {"name": "delta_ragged", "op": "delta", "seqs": 37, "moments": 1531, "q_heads": 4, "k_heads": 4, "dim": 64,
         "v_dim": 128, "ragged": True, "dtype": "bfloat16", "grad": False},
        # a learner's minibatch in float32, as the rest of the package learns
        {"name": "delta_learn", "op": "delta", "seqs": 16, "moments": 512, "q_heads": 8, "k_heads": 8, "dim": 64,
         "v_dim": 64, "ragged": False, "dtype": "float32", "grad": True},
        # odd sizes: heads of 40 and 56 values, query heads that share keys, binary16 as the recordings hold their values
        {"name": "delta_shared", "op": "delta", "seqs": 2, "moments": 1001, "q_heads": 6, "k_heads": 2, "dim": 40,
         "v_dim": 56, "ragged": True, "dtype": "float16", "grad": True},
        # the largest learning step
        {"name": "delta_large", "op": "delta", "seqs": 8, "moments": 4096, "q_heads": 16, "k_heads": 16, "dim": 128,
         "v_dim": 128, "ragged": False, "dtype": "bfloat16", "grad": True},
        # the firing of the benchmark network's 1,332 descending neurons, of a few hundred environments acting at once
        {"name": "layer_norm_acting", "op": "layer_norm", "rows": 416, "width": 1332, "dtype": "float32", "shift": True,
         "grad": False},
        # the same of a learner's minibatch: 16 stretches of 256 moments
        {"name": "layer_norm_learn", "op": "layer_norm", "rows": 4096, "width": 1332, "dtype": "float32", "shift": True,
         "grad": True},
        # many wide rows in 16 bits: bound by memory
        {"name": "layer_norm_large", "op": "layer_norm", "rows": 32768, "width": 4096, "dtype": "bfloat16", "shift": False,
         "grad": True},
        # what a learner's minibatch reads out of 8 heads of 64 values
        {"name": "dropout_learn", "op": "dropout", "rows": 4096, "width": 512, "share": 0.1, "dtype": "float32", "grad": True},
        # the largest learning step's read-out, 16 heads of 128
        {"name": "dropout_large", "op": "dropout", "rows": 32768, "width": 2048, "share": 0.25, "dtype": "bfloat16",
         "grad": True},
    ]


def draw(rng: random.Random) -> dict:
    """A case of the same ranges, none of the listed ones and none that costs more than the largest of them."""
    known = [{k: v for k, v in c.items() if k != "name"} for c in listed()]
    most = max(_cost(c) for c in known)
    c = _draw(rng)
    while c in known or _cost(c) > most:
        c = _draw(rng)
    return c


def _cost(case: dict) -> float:
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _draw(rng: random.Random) -> dict:
    def log_int(lo, hi):                        # (each whole number's share of the logarithm, the ends in full)
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))

    op = rng.choice(["delta", "delta", "delta", "delta_step", "layer_norm", "dropout"])
    c = {"op": op, "dtype": rng.choice(["float32", "bfloat16", "bfloat16", "float16"])}
    if op in ("layer_norm", "dropout"):
        c["width"] = rng.choice([1332, 64 * rng.randint(1, 64), log_int(1, 8192), log_int(1, 8192)])
        c["rows"] = log_int(1, max(1, min(1 << 16, (1 << 27) // c["width"])))
        c["grad"] = rng.random() < 0.6
        if op == "layer_norm":
            c["shift"] = rng.random() < 0.5
        else:
            c["share"] = rng.choice([0.05, 0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)])
        return c
    k_heads, share = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4])
    c.update(q_heads=k_heads * share, k_heads=k_heads, dim=rng.choice([64, 128, 8 * rng.randint(2, 16)]))
    c["v_dim"] = rng.choice([c["dim"], 64, 128, 8 * rng.randint(2, 16)])
    c["seqs"] = log_int(1, 512 if op == "delta_step" else 64)
    if op == "delta":
        c["moments"] = log_int(1, 32768 // c["seqs"])
        c.update(ragged=rng.random() < 0.4, grad=rng.random() < 0.6)
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case: dict) -> list[int]:
    """The stretches' lengths: all the same, or anything from 1 to twice the middle one (the same for every seed: a program
    that packs recordings has them before anything else)."""
    n = case["moments"]
    if not case["ragged"]:
        return [n] * case["seqs"]
    r = random.Random(n)
    return [r.randint(1, max(1, 2 * n - 1)) for _ in range(case["seqs"])]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = getattr(torch, case["dtype"])

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    st = {"op": case["op"], "grad": case.get("grad", False)}
    if case["op"] in ("layer_norm", "dropout"):
        shape = case["rows"], case["width"]
        if case["op"] == "layer_norm":
            # firing: nothing below 0, rows and columns of different sizes
            st["x"] = (normal(*shape).clamp_min(0) * (0.2 + normal(shape[1]).square()) + 0.1).to(dt)
            st["weight"], st["bias"] = 1 + 0.1 * normal(shape[1]), 0.1 * normal(shape[1]) if case["shift"] else None
            learn = ("x", "weight", "bias")
        else:
            st["x"], st["share"] = normal(*shape, dtype=dt), case["share"]
            st["counter"] = torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 63), seed + 7], device=DEV)
            learn = ("x",)
        if st["grad"]:
            st["gy"] = normal(*shape, dtype=dt)
            st.update({k: st[k].requires_grad_() for k in learn if st[k] is not None})
        return st
    N, Hq, Hk, K, V = case["seqs"], case["q_heads"], case["k_heads"], case["dim"], case["v_dim"]
    lengths = [1] * N if case["op"] == "delta_step" else _lengths(case)
    total = sum(lengths)
    # keys of length 1, alike from moment to moment (a game changes slowly); queries normed; values as a projection gives them
    k = normal(1, Hk, K) + 1.5 * normal(total, Hk, K)
    st["k"] = (k / k.square().sum(-1, keepdim=True).sqrt()).to(dt)
    q = normal(total, Hq, K)
    st["q"] = (q / q.square().mean(-1, keepdim=True).sqrt()).to(dt)
    st["v"] = normal(total, Hk * (K + V), dtype=dt)[:, Hk * K:].unflatten(-1, (Hk, V))
    # each head's memory: from 8 moments to about 2,000 where nothing is asked, more or less by the moment; rates in (0, 1)
    decay = -(2.0 ** -torch.linspace(3, 11, Hq, device=DEV))
    st["log_decay"] = decay * torch.nn.functional.softplus(normal(total, Hq)) / math.log(2)
    st["beta"] = torch.sigmoid(normal(total, Hq))
    st["state"] = normal(N, Hq, K, V)
    st["scale"] = K ** -0.5
    if case["op"] == "delta_step":
        st["next"] = torch.empty_like(st["state"])
        return st
    st["starts"], st["lengths"] = None, lengths
    named = ("q", "k", "v", "log_decay", "beta")
    if case["ragged"]:
        st["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=DEV)
    else:
        st.update({n: st[n].unflatten(0, (N, -1)) for n in named})
    if st["grad"]:
        st["go"] = normal(*st["q"].shape[:-1], V, dtype=dt)
        st["gs"] = normal(N, Hq, K, V)
        st.update({n: st[n].detach().requires_grad_() for n in (*named, "state")})
    return st


# ------------------------------------------------------------------------------------------------ a pass
def run(st: dict):
    if own:
        return _own(st)
    return {"delta": _plain_delta, "delta_step": _plain_step, "layer_norm": _plain_norm, "dropout": _plain_dropout}[st["op"]](st)


_LEAVES = ("q", "k", "v", "log_decay", "beta", "state")


def _own(st: dict):
    from flyguy_amd import memory_hip as m, rows_hip as r
    if st["op"] == "delta_step":
        o = m.delta_step(st["q"], st["k"], st["v"], st["log_decay"], st["beta"], st["state"], into=st["next"],
                         scale=st["scale"])
        return o, st["next"]
    if st["op"] == "delta":
        out = m.delta_attention(*(st[n] for n in _LEAVES), st["starts"], scale=st["scale"])
        leaves, grads = [st[n] for n in _LEAVES], ("go", "gs")
    elif st["op"] == "layer_norm":
        out = (r.layer_norm(st["x"], st["weight"], st["bias"], eps=EPS),)
        leaves, grads = [x for x in (st["x"], st["weight"], st["bias"]) if x is not None], ("gy",)
    else:
        out = (r.dropout(st["x"], st["share"], st["counter"]),)
        leaves, grads = [st["x"]], ("gy",)
    if not st["grad"]:
        return out
    return (*(x.detach() for x in out), *torch.autograd.grad(out, leaves, [st[k] for k in grads]))


@torch.no_grad()
def _plain_norm(st):
    x, w, b = st["x"].float(), st["weight"], st["bias"]
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * r
    y = (xh * w if b is None else xh * w + b).to(st["x"].dtype)
    if not st["grad"]:
        return (y,)
    g = st["gy"].float()
    u = g * w
    gx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
    return (y, gx.to(y.dtype), (g * xh).sum(0), *(() if b is None else (g.sum(0),)))


def _halves(counter: torch.Tensor, blocks: int) -> torch.Tensor:
    """The generator's 16-bit numbers, 8 a block [blocks, 8]: Philox4x32 of 10 rounds (Salmon et al., 2011), key = the seed
    (counter[0]), counter = (block, counter[1]), both low word first; a word's low half first."""
    low = 0xFFFFFFFF
    b = torch.arange(blocks, device=counter.device)
    c0, c1 = b & low, b >> 32
    c2, c3 = (counter[1] & low).expand(blocks), (counter[1] >> 32 & low).expand(blocks)
    k0, k1 = counter[0] & low, counter[0] >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57             # (64 bits, whose top one is a bit like the others)
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).flatten(-2)


@torch.no_grad()
def _plain_dropout(st):
    x = st["x"]
    t = round(st["share"] * 65536)
    keep = (_halves(st["counter"], -(-x.numel() // 8)).flatten()[:x.numel()] >= t).view(x.shape)
    f = 65536 / (65536 - t)
    return tuple(torch.where(keep, z.float() * f, 0.0).to(z.dtype) for z in ((x, st["gy"]) if st["grad"] else (x,)))


@torch.no_grad()
def _plain_step(st):
    share = st["q"].shape[1] // st["k"].shape[1]
    k, v = (st[x].float().repeat_interleave(share, 1) for x in ("k", "v"))
    s = torch.exp(st["log_decay"])[..., None, None] * st["state"]
    u = st["beta"][..., None] * (v - (k[..., None, :] @ s).squeeze(-2))
    s = s + k[..., :, None] * u[..., None, :]
    return (st["scale"] * (st["q"].float()[..., None, :] @ s).squeeze(-2)).to(st["q"].dtype), s


def _inverse(n):
    """(I + n)^-1 of strictly lower triangular n [.., C, C], C a power of two: blocks of twice the size from those on the
    diagonal, (a 0; b d)^-1 = (a^-1 0; -d^-1 b a^-1 d^-1)."""
    C = n.shape[-1]
    inv = torch.ones(*n.shape[:-2], C, 1, 1, device=n.device)                                     # [.., blocks, size, size]
    size = 1
    while size < C:
        pairs = torch.arange(C // (2 * size), device=n.device)
        blocks = n.unflatten(-1, (-1, size)).unflatten(-3, (-1, size))                            # [.., rb, size, cb, size]
        b = blocks.movedim(-2, -3)[..., 2 * pairs + 1, 2 * pairs, :, :]
        a, d = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        low = torch.cat([-(d @ b) @ a, d], -1)
        inv = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), low], -2)
        size *= 2
    return inv.squeeze(-3)


def _plain_delta(st):
    """In chunks: with G the log decays summed up inside a chunk, D_ij = exp(G_i - G_j) for j <= i, S the state before it,
    e = (I + lower(K K^T D) B)^-1 (V - exp(G) K S) what the state is wrong by at each moment, u = B e:
    o = c (exp(G) Q S + lower(Q K^T D) u), S' = exp(G_end) S + (exp(G_end - G) K)^T u."""
    c, dt = st["scale"], st["q"].dtype
    lengths, N, T = st["lengths"], st["state"].shape[0], max(st["lengths"])
    share = st["q"].shape[-2] // st["k"].shape[-2]
    T += -T % CHUNK
    there = torch.arange(T, device=DEV) < torch.tensor(lengths, device=DEV)[:, None]              # [N, T]

    def laid(name):                                           # [N, H, chunks, CHUNK, .], zeros past a stretch's end
        x = st[name].float()
        x = x[..., None] if name in ("log_decay", "beta") else x
        if st["starts"] is None:
            x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, T - x.shape[1]))
        else:
            at = (st["starts"][:-1, None].long() + torch.arange(T, device=DEV)) * there
            x = x[at] * there[..., None, None]
        if name in ("k", "v") and share > 1:
            x = x.repeat_interleave(share, 2)
        return x.transpose(1, 2).unflatten(2, (-1, CHUNK))

    def forward():
        q, k, v, g, beta = (laid(n) for n in _LEAVES[:5])
        s = st["state"]
        G = g.squeeze(-1).cumsum(-1)
        apart = G[..., :, None] - G[..., None, :]
        low = torch.ones(CHUNK, CHUNK, device=DEV).tril().bool()
        D = torch.where(low, torch.exp(torch.where(low, apart, 0.0)), 0.0)
        kt = k.transpose(-1, -2)
        inv = _inverse(((k @ kt) * D).tril(-1) * beta.transpose(-1, -2))
        own, read = inv @ v, inv @ (torch.exp(G)[..., None] * k)
        weights = (q @ kt) * D
        end = G[..., -1:]
        write = (torch.exp(end - G)[..., None] * k).transpose(-1, -2)
        keep, q = torch.exp(end)[..., None], torch.exp(G)[..., None] * q
        out = []
        for i in range(T // CHUNK):
            u = beta[:, :, i] * (own[:, :, i] - read[:, :, i] @ s)
            out.append(c * (q[:, :, i] @ s + weights[:, :, i] @ u))
            s = keep[:, :, i] * s + write[:, :, i] @ u
        o = torch.cat(out, 2).transpose(1, 2)                 # [N, T, H, V]
        return (o[:, :lengths[0]] if st["starts"] is None else o[there]).to(dt), s

    if not st["grad"]:
        with torch.no_grad():
            return forward()
    with torch.enable_grad():
        out = forward()
    return (*(x.detach() for x in out), *torch.autograd.grad(out, [st[n] for n in _LEAVES], [st["go"], st["gs"]]))


# ------------------------------------------------------------------------------------------------ what a pass has to do
def work(case: dict) -> dict:
    """Each input read once and each output written once, and the recurrent form's operations (a state is read under the
    key, added to and read under the query once a moment; for the gradients once more, and seven such products)."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] in ("layer_norm", "dropout"):
        values = case["rows"] * case["width"]
        of_row = 4 * case["width"] * (1 + case.get("shift", False)) if case["op"] == "layer_norm" else 0
        # gradients: gy read and gx written, x read once for both where the norm needs it
        return {"bytes": values * size * (4 if case["grad"] else 2) + of_row * (2 if case["grad"] else 1),
                "flops": values * ((8 if case["op"] == "layer_norm" else 1) * (2 if case["grad"] else 1))}
    N, Hq, Hk, K, V = case["seqs"], case["q_heads"], case["k_heads"], case["dim"], case["v_dim"]
    state = 4 * N * Hq * K * V
    moments = N if case["op"] == "delta_step" else sum(_lengths(case))
    ins = moments * ((Hq * K + Hk * (K + V)) * size + 8 * Hq)
    out = moments * Hq * V * size
    flops = moments * Hq * 6 * K * V
    if case.get("grad"):
        # q, k, v, gates, the output's and the state's gradients read; the output, the state and all gradients written
        return {"bytes": 2 * ins + 2 * out + 4 * state, "flops": flops * 20 / 6}
    return {"bytes": ins + out + 2 * state, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    """The definitions in 64 bits: the delta rule moment by moment, its gradients moment by moment backwards."""
    st = {k: (v.detach() if isinstance(v, torch.Tensor) else v) for k, v in prepare(case, seed).items()}
    st = {k: (v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in st.items()}
    if st["op"] == "layer_norm":
        x, n = st["x"], case["width"]
        off = x - x.sum(1, keepdim=True) / n
        dev = (off.square().sum(1, keepdim=True) / n + EPS).sqrt()
        y = off / dev * st["weight"]
        y = y if st["bias"] is None else y + st["bias"]
        if not st["grad"]:
            return (y,)
        u = st["gy"] * st["weight"]
        gx = (u - u.sum(1, keepdim=True) / n) / dev - off * (u * off).sum(1, keepdim=True) / (n * dev ** 3)
        return (y, gx, (st["gy"] * off / dev).sum(0), *(() if st["bias"] is None else (st["gy"].sum(0),)))
    if st["op"] == "dropout":
        return _exact_dropout(st)
    q, k, v, s = st["q"], st["k"], st["v"], st["state"].clone()
    share, c = q.shape[-2] // k.shape[-2], st["scale"]
    if st["op"] == "delta_step":
        k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
        s = torch.exp(st["log_decay"])[..., None, None] * s
        e = v - (k[..., :, None] * s).sum(-2)
        s = s + k[..., :, None] * (st["beta"][..., None] * e)[..., None, :]
        return c * (q[..., :, None] * s).sum(-2), s
    lengths = case["seqs"] * [case["moments"]] if st["starts"] is None else _lengths(case)
    N, T, BLOCK = len(lengths), max(lengths), 64
    if T * s.numel() * (4 if st["grad"] else 1) > 2.5e11 or T > 70000:
        return None
    first = np.concatenate([[0], np.cumsum(lengths)[:-1]])
    flat = {n: (st[n] if st["starts"] is not None else st[n].flatten(0, 1)) for n in (*_LEAVES[:5], "go") if n in st}
    for n in ("k", "v"):
        flat[n] = flat[n].repeat_interleave(share, 1)
    at = torch.from_numpy(first).to(DEV)[:, None] + torch.arange(T, device=DEV)
    there = torch.arange(T, device=DEV) < torch.tensor(lengths, device=DEV)[:, None]
    at = at * there

    def moment(name, t):                                      # zeros past a stretch's end: the state stays as it is
        x = flat[name][at[:, t]]
        return x * there[:, t].view(-1, *[1] * (x.dim() - 1))

    def forward(s, t):                                        # -> the state decayed, what it is wrong by, the new state
        a = torch.exp(moment("log_decay", t))[..., None, None] * s
        k = moment("k", t)
        e = moment("v", t) - (k[..., None, :] @ a).squeeze(-2)
        return a, e, a + k[..., :, None] * (moment("beta", t)[..., None] * e)[..., None, :]

    H, K, V = s.shape[1:]
    o = torch.zeros(flat["q"].shape[0], H, V, dtype=torch.float64, device=DEV)
    kept = []
    for t in range(T):
        if st["grad"] and t % BLOCK == 0:
            kept.append(s)
        s = forward(s, t)[2]
        o[at[there[:, t], t]] = c * (moment("q", t)[..., None, :] @ s).squeeze(-2)[there[:, t]]
    like = lambda x, n: x.reshape(*st[n].shape)               # noqa: E731
    o_shape = (*st["q"].shape[:-1], V)
    if not st["grad"]:
        return o.reshape(o_shape), s
    end, d = s, st["gs"].clone()
    dq, dk, dv = (torch.zeros_like(flat[n]) for n in ("q", "k", "v"))
    dg, db = (torch.zeros_like(flat[n]) for n in ("log_decay", "beta"))
    for b in range(len(kept) - 1, -1, -1):
        s, states = kept[b], []
        for t in range(b * BLOCK, min(T, (b + 1) * BLOCK)):
            a, e, s2 = forward(s, t)
            states.append((s, a, e, s2))
            s = s2
        for t in range(min(T, (b + 1) * BLOCK) - 1, b * BLOCK - 1, -1):
            s, a, e, s2 = states.pop()
            here, rows = there[:, t], at[there[:, t], t]
            go, k, beta = moment("go", t), moment("k", t), moment("beta", t)[..., None]
            d = d + c * moment("q", t)[..., :, None] * go[..., None, :]
            du = (k[..., None, :] @ d).squeeze(-2)
            de = beta * du
            dq[rows] = c * (s2 @ go[..., None]).squeeze(-1)[here]
            db[rows] = (du * e).sum(-1)[here]
            dv[rows] = de[here]
            dk[rows] = ((d @ (beta * e)[..., None]) - a @ de[..., None]).squeeze(-1)[here]
            d = d - k[..., :, None] * de[..., None, :]
            dg[rows] = (d * a).sum((-1, -2))[here]
            d = torch.exp(moment("log_decay", t))[..., None, None] * d
    shared = lambda x, n: like(x.unflatten(1, (-1, share)).sum(2), n)                             # noqa: E731
    return (o.reshape(o_shape), end, like(dq, "q"), shared(dk, "k"), shared(dv, "v"), like(dg, "log_decay"),
            like(db, "beta"), d)


def _exact_dropout(st):
    seed, offset = (int(x) % (1 << 64) for x in st["counter"])
    n, t = st["x"].numel(), round(st["share"] * 65536)
    block = np.arange(-(-n // 8), dtype=np.uint64)
    word, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [block & word, block >> s, np.uint64(offset & 0xFFFFFFFF), np.uint64(offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [b >> s ^ c[1] ^ np.uint64(key[0]), b & word, a >> s ^ c[3] ^ np.uint64(key[1]), a & word]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    words = np.stack([np.broadcast_to(x, block.shape) for x in c], -1).astype("<u4")
    kept = torch.from_numpy(words.reshape(-1).view("<u2").astype(np.int32)[:n] >= t).to(DEV).view(st["x"].shape)
    f = 65536 / (65536 - t)
    return tuple(kept * z * f for z in ((st["x"], st["gy"]) if st["grad"] else (st["x"],)))
