"""The operators of the memory over decisions whose speed is tracked: what programs have this package do with a stream of
moments (a recorded game, many cars acting at once), through the package's public entry points.

A case names an operator:
  rotary     queries and keys rotated by their positions (flyguy_amd.memory_hip.rotary)
  norm       each head's queries and keys normed, then rotated, in one pass (norm_rotary)
  attention  linear attention with a decay for each head over whole stretches of moments (decay_attention)
  step       the same for one new moment of each car, on the cars' states (decay_step)
and its sizes: seqs stretches (cars) of moments moments each, q_heads query heads and k_heads key / value heads (query
heads share them in consecutive groups), dim values of a query or key, v_dim of a value, dtype "float32", "bfloat16" or
"float16" of queries, keys, values and outputs.  grad: the pass is the forward and the gradients of everything that
learns.  Queries, keys and values are views of one projection's output, as a layer has them.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the package's kernels.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
CHUNK = 64                               # moments per chunk of the plain form


def listed() -> list[dict]:
    return [
        # one car's new moment: the smallest call, its latency counts
        {"name": "rotary_one", "op": "rotary", "seqs": 1, "moments": 1, "q_heads": 8, "k_heads": 8, "dim": 64, "rotated": 64,
         "interleaved": False, "scaling": 1.0, "dtype": "float32", "grad": False},
        # two whole recorded games, longer than what was taught: interleaved pairs of half of each head, a stretched table,
        # query heads that share keys; forward and gradients
        {"name": "rotary_games", "op": "rotary", "seqs": 2, "moments": 16384, "q_heads": 16, "k_heads": 4, "dim": 128,
         "rotated": 64, "interleaved": True, "scaling": 4.0, "dtype": "bfloat16", "grad": True},
        # a few hundred environments acting at once, each at a position of its own
        {"name": "norm_acting", "op": "norm", "seqs": 416, "moments": 1, "q_heads": 8, "k_heads": 8, "dim": 64, "rotated": 64,
         "interleaved": False, "scaling": 1.0, "dtype": "bfloat16", "grad": False},
        # a learner's minibatch of stretches
        {"name": "norm_learn", "op": "norm", "seqs": 8, "moments": 2048, "q_heads": 16, "k_heads": 16, "dim": 128,
         "rotated": 128, "interleaved": False, "scaling": 1.0, "dtype": "bfloat16", "grad": True},
        # odd sizes: a ragged length, heads of 80 values of which 32 turn, float32 as the rest of the package
        {"name": "norm_odd", "op": "norm", "seqs": 3, "moments": 1021, "q_heads": 6, "k_heads": 2, "dim": 80, "rotated": 32,
         "interleaved": False, "scaling": 1.0, "dtype": "float32", "grad": True},
        # one car's new moment
        {"name": "step_one", "op": "step", "seqs": 1, "q_heads": 8, "k_heads": 8, "dim": 64, "v_dim": 64,
         "dtype": "float32"},
        # a few hundred environments acting at once: bound by reading and writing their states
        {"name": "step_acting", "op": "step", "seqs": 416, "q_heads": 8, "k_heads": 8, "dim": 128, "v_dim": 128,
         "dtype": "bfloat16"},
        # one whole recording read in before play goes on: few long sequences
        {"name": "attention_game", "op": "attention", "seqs": 1, "moments": 32768, "q_heads": 8, "k_heads": 8, "dim": 128,
         "v_dim": 128, "ragged": False, "dtype": "bfloat16", "grad": False},
        # packed recordings of different lengths, each going on from a state of its own
        {"name": "attention_ragged", "op": "attention", "seqs": 37, "moments": 1531, "q_heads": 4, "k_heads": 4, "dim": 64,
         "v_dim": 128, "ragged": True, "dtype": "bfloat16", "grad": False},
        # a learner's minibatch in float32, as the rest of the package learns
        {"name": "attention_learn", "op": "attention", "seqs": 16, "moments": 512, "q_heads": 8, "k_heads": 8, "dim": 64,
         "v_dim": 64, "ragged": False, "dtype": "float32", "grad": True},
        # odd sizes: heads of 40 and 56 values, query heads that share keys, binary16 as the recordings hold their values
        {"name": "attention_shared", "op": "attention", "seqs": 2, "moments": 1001, "q_heads": 6, "k_heads": 2, "dim": 40,
         "v_dim": 56, "ragged": True, "dtype": "float16", "grad": True},
        # the largest learning step
        {"name": "attention_large", "op": "attention", "seqs": 8, "moments": 4096, "q_heads": 16, "k_heads": 16, "dim": 128,
         "v_dim": 128, "ragged": False, "dtype": "bfloat16", "grad": True},
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

    op = rng.choice(["rotary", "norm", "step", "attention", "attention"])
    k_heads, share = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4])
    c = {"op": op, "q_heads": k_heads * share, "k_heads": k_heads, "dim": rng.choice([64, 128, 8 * rng.randint(2, 16)]),
         "dtype": rng.choice(["float32", "bfloat16", "bfloat16", "float16"])}
    if op in ("rotary", "norm"):
        c["seqs"] = log_int(1, 512)
        c["moments"] = 1 if rng.random() < 0.2 else log_int(1, max(2, 32768 // c["seqs"]))
        c["rotated"] = rng.choice([c["dim"], 2 * rng.randint(4, c["dim"] // 2)])
        c.update(interleaved=rng.random() < 0.5, scaling=rng.choice([1.0, 1.0, 4.0]), grad=rng.random() < 0.5)
    else:
        c["v_dim"] = rng.choice([c["dim"], 64, 128, 8 * rng.randint(2, 16)])
        c["seqs"] = log_int(1, 512 if op == "step" else 64)
        if op == "attention":
            c["moments"] = log_int(1, 32768 // c["seqs"])
            c.update(ragged=rng.random() < 0.4, grad=rng.random() < 0.6)
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _table(positions: int, rotated: int, scaling: float) -> torch.Tensor:
    """(cos, sin) of each position and pair of values, [positions, rotated / 2, 2]: angle = position / scaling x 10000^(-2i /
    rotated).  Made once by a program, in 64 bits."""
    turn = 10000.0 ** (-np.arange(0, rotated, 2, dtype=np.float64) / rotated) / scaling
    a = np.arange(positions, dtype=np.float64)[:, None] * turn
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).to(DEV)


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
    op, N, Hq, Hk, D = case["op"], case["seqs"], case["q_heads"], case["k_heads"], case["dim"]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    st = {"op": op, "grad": case.get("grad", False)}
    if op in ("rotary", "norm"):
        T = case["moments"]
        p = normal(N, T, (Hq + 2 * Hk) * D)                     # the projection's output: queries, keys and values
        st["q"] = p[..., :Hq * D].unflatten(-1, (Hq, D))
        st["k"] = p[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
        longest = T if T > 1 else 4096
        st["table"], st["interleaved"] = _table(longest, case["rotated"], case["scaling"]), case["interleaved"]
        st["positions"] = (torch.arange(T, device=DEV, dtype=torch.int32).expand(N, T).contiguous() if T > 1 else
                           torch.randint(0, longest, (N, 1), device=DEV, dtype=torch.int32, generator=g))
        if op == "norm":
            st["wq"], st["wk"] = (1 + 0.1 * normal(D, dtype=torch.float32) for _ in range(2))
        if st["grad"]:
            st["gq"], st["gk"] = normal(N, T, Hq, D), normal(N, T, Hk, D)
            leaves = ("q", "k", "wq", "wk") if op == "norm" else ("q", "k")
            st.update({k: st[k].detach().requires_grad_() for k in leaves})
        return st
    K, V = D, case["v_dim"]
    # each head's memory: from 8 moments to about 2,000
    st["log_decay"] = -(2.0 ** -torch.linspace(3, 11, Hq, device=DEV))
    st["scale"] = K ** -0.5
    if op == "step":
        st["q"], st["k"], st["v"] = normal(N, Hq, K), normal(N, Hk, K), normal(N, Hk, V)
        st["state"] = normal(N, Hq, K, V, dtype=torch.float32)
        st["next"] = torch.empty_like(st["state"])
        return st
    lengths = _lengths(case)
    total = sum(lengths)
    p = normal(total, Hk * (K + V))                             # keys come rotated, values as the projection gives them
    st["q"], st["k"] = normal(total, Hq, K), normal(total, Hk, K)
    st["v"] = p[:, Hk * K:].unflatten(-1, (Hk, V))
    st["state"] = normal(N, Hq, K, V, dtype=torch.float32)
    st["starts"], st["longest"] = None, max(lengths)
    if case["ragged"]:
        st["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=DEV)
    else:
        st.update({k: st[k].unflatten(0, (N, -1)) for k in ("q", "k", "v")})
    if st["grad"]:
        st["go"] = normal(*st["q"].shape[:-1], V)
        st["gs"] = normal(N, Hq, K, V, dtype=torch.float32)
        st.update({k: st[k].detach().requires_grad_() for k in ("q", "k", "v", "state")})
    return st


# ------------------------------------------------------------------------------------------------ a pass
def run(st: dict):
    if own:
        return _own(st)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "norm": _plain_norm, "attention": _plain_attention, "step": _plain_step}[st["op"]](st)


def _own(st: dict):
    from flyguy_amd import memory_hip as m
    if st["op"] == "step":
        o = m.decay_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"], into=st["next"], scale=st["scale"])
        return o, st["next"]
    if st["op"] == "attention":
        out = m.decay_attention(st["q"], st["k"], st["v"], st["log_decay"], st["state"], st["starts"], scale=st["scale"])
        leaves, grads = ("q", "k", "v", "state"), ("go", "gs")
    elif st["op"] == "norm":
        out = m.norm_rotary(st["q"], st["k"], st["wq"], st["wk"], st["table"], st["positions"],
                            interleaved=st["interleaved"], eps=EPS)
        leaves, grads = ("q", "k", "wq", "wk"), ("gq", "gk")
    else:
        out = m.rotary(st["q"], st["k"], st["table"], st["positions"], interleaved=st["interleaved"])
        leaves, grads = ("q", "k"), ("gq", "gk")
    if not st["grad"]:
        return out
    return (*(x.detach() for x in out), *torch.autograd.grad(out, [st[k] for k in leaves], [st[k] for k in grads]))


def _turn(x, cs, interleaved):
    """x [N, T, H, D] in 32 bits with the first values of each head turned by cs [N, T, 1, R/2, 2]."""
    R = 2 * cs.shape[-2]
    cos, sin = cs[..., 0], cs[..., 1]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _plain_rotary(st):
    cs = st["table"][st["positions"].long()][:, :, None]
    back = torch.stack([cs[..., 0], -cs[..., 1]], -1)
    q, k, il = st["q"], st["k"], st["interleaved"]
    out = _turn(q.float(), cs, il).to(q.dtype), _turn(k.float(), cs, il).to(k.dtype)
    if not st["grad"]:
        return out
    return (*out, _turn(st["gq"].float(), back, il).to(q.dtype), _turn(st["gk"].float(), back, il).to(k.dtype))


def _plain_norm(st):
    cs = st["table"][st["positions"].long()][:, :, None]
    back = torch.stack([cs[..., 0], -cs[..., 1]], -1)

    def forward(x, w):
        x = x.float()
        return _turn(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w, cs, st["interleaved"])

    def backward(x, w, g):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xh, g = x * r, _turn(g.float(), back, st["interleaved"])
        gw = (g * xh).sum((0, 1, 2))
        g = g * w
        return r * (g - xh * (g * xh).mean(-1, keepdim=True)), gw

    q, k, wq, wk = st["q"], st["k"], st["wq"], st["wk"]
    out = forward(q, wq).to(q.dtype), forward(k, wk).to(k.dtype)
    if not st["grad"]:
        return out
    (dq, dwq), (dk, dwk) = backward(q, wq, st["gq"]), backward(k, wk, st["gk"])
    return (*out, dq.to(q.dtype), dk.to(k.dtype), dwq, dwk)


def _plain_step(st):
    share = st["q"].shape[1] // st["k"].shape[1]
    k, v = (st[x].float().repeat_interleave(share, 1) for x in ("k", "v"))
    s = torch.exp(st["log_decay"])[:, None, None] * st["state"] + k[..., :, None] * v[..., None, :]
    o = st["scale"] * (st["q"].float()[..., None, :] @ s).squeeze(-2)
    return o.to(st["q"].dtype), s


def _decayed(x, y, v, z, g, first):
    """sum over j <= i of l^(i - j) (x_i . y_j) v_j + l^(i + first) x_i z, of [N, H, T, .] inputs, chunk by chunk all at once:
    products inside a chunk, and each chunk's start state by a product over chunks."""
    N, H, T, V = v.shape
    pad = -T % CHUNK
    x, y, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).unflatten(2, (-1, CHUNK)) for t in (x, y, v))
    n = x.shape[2]
    at = torch.arange(CHUNK, device=x.device, dtype=torch.float32)
    of = torch.arange(n, device=x.device, dtype=torch.float32)
    g1, g2 = g[:, None], g[:, None, None]
    apart = at[:, None] - at
    within = torch.where(apart >= 0, torch.exp(g2 * apart.clamp_min(0)), 0.0)                     # [H, C, C]
    out = (x @ y.transpose(-1, -2) * within[:, None]) @ v
    kv = (y * torch.exp(g1 * (CHUNK - at))[:, None, :, None]).transpose(-1, -2) @ v               # [N, H, n, K, V]
    chunks = of[:, None] - of - 1
    between = torch.where(chunks >= 0, torch.exp(g2 * CHUNK * chunks.clamp_min(0)), 0.0)          # [H, n, n]
    before = (between @ kv.flatten(-2)).unflatten(-1, kv.shape[-2:])
    before = before + torch.exp(g1 * (CHUNK * of + first))[..., None, None] * z[:, :, None]
    out = out + torch.exp(g1 * at)[:, None, :, None] * (x @ before)
    return out.flatten(2, 3)[:, :, :T]


def _carried(y, v, z, g, lengths, last):
    """l^n z + sum over j < n of l^(n - 1 - j + last) y_j v_j^T of [N, H, T, .] inputs, n a sequence's length: the state after
    it (last 0), or the gradient of the state before it, with the sequence backwards (last 1)."""
    at = torch.arange(y.shape[2], device=y.device)
    left = (lengths[:, None] - 1 - at).clamp_min(0).float() + last
    w = torch.exp(g[:, None] * left[:, None])                                                     # [N, H, T]
    return (y * w[..., None]).transpose(-1, -2) @ v + torch.exp(g * lengths[:, None].float())[..., None, None] * z


def _plain_attention(st):
    q, k, v, g, c = st["q"], st["k"], st["v"], st["log_decay"], st["scale"]
    share = q.shape[-2] // k.shape[-2]
    N, T = st["state"].shape[0], st["longest"]
    starts = st["starts"]
    if starts is None:
        starts = torch.arange(N + 1, device=q.device) * T
    starts = starts.long()
    lengths = starts[1:] - starts[:-1]
    at = torch.arange(T, device=q.device)
    there = at < lengths[:, None]                                                                 # [N, T]
    fore = torch.where(there, starts[:-1, None] + at, 0)
    back = torch.where(there, starts[1:, None] - 1 - at, 0)
    flat = {n: (st[n].flatten(0, -3) if st[n].dim() == 4 else st[n]).float() for n in ("q", "k", "v", "go") if n in st}

    def laid(name, order):                                     # [N, H, T, .], zeros past a sequence's end
        x = flat[name]
        if name in ("k", "v") and share > 1:
            x = x.repeat_interleave(share, 1)
        return (x[order] * there[..., None, None]).transpose(1, 2)

    def packed(x, order, like, heads_shared=False):            # back to the inputs' layout
        if heads_shared and share > 1:
            x = x.unflatten(1, (-1, share)).sum(2)
        out = torch.empty(flat["q"].shape[0], x.shape[1], x.shape[3], device=x.device)
        out[order[there]] = x.transpose(1, 2)[there]
        return out.to(like.dtype).reshape(like.shape[:-1] + (x.shape[3],))

    qf, kf, vf = (laid(n, fore) for n in ("q", "k", "v"))
    o = packed(c * _decayed(qf, kf, vf, st["state"], g, 1), fore, q)
    s = _carried(kf, vf, st["state"], g, lengths, 0)
    if not st["grad"]:
        return o, s
    gf = laid("go", fore)
    dq = packed(c * _decayed(gf, vf, kf, st["state"].transpose(-1, -2), g, 1), fore, q)
    qb, kb, vb, gb = (laid(n, back) for n in ("q", "k", "v", "go"))
    dk = packed(_decayed(vb, c * gb, qb, st["gs"].transpose(-1, -2), g, 0), back, k, True)
    dv = packed(_decayed(kb, c * qb, gb, st["gs"], g, 0), back, v, True)
    ds = _carried(c * qb, gb, st["gs"], g, lengths, 1)
    return o, s, dq, dk, dv, ds


# ------------------------------------------------------------------------------------------------ what a pass has to do
def work(case: dict) -> dict:
    """Each input read once and each output written once, and the products' operations (recurrent form of the attention: a
    state is multiplied and added to once a moment and read once, twice more of each for the gradients)."""
    size = 4 if case["dtype"] == "float32" else 2
    N, Hq, Hk, D = case["seqs"], case["q_heads"], case["k_heads"], case["dim"]
    if case["op"] in ("rotary", "norm"):
        T = case["moments"]
        values = N * T * (Hq + Hk) * D
        table = 4 * case["rotated"] * min(N * T, T if T > 1 else 4096)
        # forward: x read, y written; gradients: g read, gx written, and x read once for both where the norm needs it
        return {"bytes": values * size * (4 if case["grad"] else 2) + table + 4 * N * T,
                "flops": values * ((4 if case["op"] == "rotary" else 8) * (3 if case["grad"] else 1))}
    V = case["v_dim"]
    state = 4 * N * Hq * D * V
    moments = N if case["op"] == "step" else sum(_lengths(case))
    ins = moments * (Hq * D + Hk * (D + V)) * size
    out = moments * Hq * V * size
    flops = moments * Hq * 4 * D * V
    if case.get("grad"):
        # q, k, v, the output's and the state's gradients read; the output, the state and all gradients written
        return {"bytes": 2 * ins + 2 * out + 4 * state, "flops": 3.5 * flops}
    return {"bytes": ins + out + 2 * state, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    """The definitions in 64 bits: rotations as complex products, the attention moment by moment."""
    st = {k: (v.detach() if isinstance(v, torch.Tensor) else v) for k, v in prepare(case, seed).items()}
    st = {k: (v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in st.items()}
    if st["op"] in ("rotary", "norm"):
        turn = torch.view_as_complex(st["table"])[st["positions"].long()][:, :, None]
        R = 2 * turn.shape[-1]

        def rotated(x, t):
            head = x[..., :R].unflatten(-1, (-1, 2) if st["interleaved"] else (2, -1))
            head = head if st["interleaved"] else head.transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * t)
            y = y if st["interleaved"] else y.transpose(-1, -2)
            return torch.cat([y.flatten(-2), x[..., R:]], -1)

        outs, grads, weights = [], [], []
        for n in ("q", "k"):
            x = st[n]
            if st["op"] == "rotary":
                outs.append(rotated(x, turn))
                if st["grad"]:
                    grads.append(rotated(st["g" + n], turn.conj()))
                continue
            w, D = st["w" + n], x.shape[-1]
            rms = ((x ** 2).sum(-1, keepdim=True) / D + EPS).sqrt()
            outs.append(rotated(x / rms * w, turn))
            if st["grad"]:
                gz = rotated(st["g" + n], turn.conj())
                grads.append(gz * w / rms - x * (gz * w * x).sum(-1, keepdim=True) / (D * rms ** 3))
                weights.append((gz * x / rms).flatten(0, 2).sum(0))
        return (*outs, *grads, *weights)
    l, c = torch.exp(st["log_decay"])[:, None, None], st["scale"]
    q, k, v, s = st["q"], st["k"], st["v"], st["state"].clone()
    share = q.shape[-2] // k.shape[-2]
    if st["op"] == "step":
        k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
        s = l * s + k[..., :, None] * v[..., None, :]
        return c * (q[..., :, None] * s).sum(-2), s
    lengths = _lengths(case)
    first = np.concatenate([[0], np.cumsum(lengths)[:-1]])
    shapes = {n: st[n].shape for n in ("q", "k", "v", "go") if n in st}
    flat = {n: st[n].reshape(-1, *st[n].shape[-2:]) for n in shapes}
    for n in ("k", "v"):
        flat[n] = flat[n].repeat_interleave(share, 1)
    order = np.argsort(-np.asarray(lengths), kind="stable")    # the longest first: at any moment a prefix of them runs
    begin = torch.from_numpy(first[order].astype(np.int64)).to(DEV)
    count = torch.from_numpy(np.asarray(lengths, np.int64)[order]).to(DEV)
    running = [int((np.asarray(lengths) > t).sum()) for t in range(max(lengths))]
    if sum(running) and max(lengths) * s.numel() > 3e11:
        return None
    o = torch.empty(*flat["q"].shape[:2], v.shape[-1], dtype=torch.float64, device=DEV)
    s = s[torch.from_numpy(order.copy()).to(DEV)]
    if st["grad"]:
        gs = st["gs"][torch.from_numpy(order.copy()).to(DEV)].clone()
        dq, dk, dv = (torch.empty_like(flat[n]) for n in ("q", "k", "v"))
    for t, m in enumerate(running):
        at = begin[:m] + t
        s[:m].mul_(l).add_(flat["k"][at][..., :, None] * flat["v"][at][..., None, :])
        o[at] = c * (flat["q"][at][..., None, :] @ s[:m]).squeeze(-2)
        if st["grad"]:
            dq[at] = c * (s[:m] @ flat["go"][at][..., None]).squeeze(-1)
    undo = torch.from_numpy(np.argsort(order)).to(DEV)
    o = o.reshape(*shapes["q"][:-1], v.shape[-1])
    if not st["grad"]:
        return o, s[undo]
    for t, m in enumerate(running):
        at = begin[:m] + count[:m] - 1 - t
        gs[:m].add_(c * flat["q"][at][..., :, None] * flat["go"][at][..., None, :])
        dk[at] = (gs[:m] @ flat["v"][at][..., None]).squeeze(-1)
        dv[at] = (flat["k"][at][..., None, :] @ gs[:m]).squeeze(-2)
        gs[:m].mul_(l)
    shared = lambda x, like: x.unflatten(1, (-1, share)).sum(2).reshape(like)       # noqa: E731
    return o, s[undo], dq.reshape(shapes["q"]), shared(dk, shapes["k"]), shared(dv, shapes["v"]), gs[undo]
