"""A fly actor that remembers: a memory over decisions between the descending neurons and the read-out.

The reference's actor decides each moment alone (flyguy/fly.py:286-305).  MemoryActor keeps that network as it is and adds
to its logits what one layer of linear attention makes of the descending neurons' firing, moment after moment: queries,
keys and values are projections of the firing, queries and keys are normed per head and turned by the moment's number, and
each head remembers with a decay of its own (flyguy_amd/memory_hip.py).  With rule "delta" a head corrects what it remembers
instead of only adding to it: what its state holds under a moment's key is moved towards the moment's value, at a rate, and
after a decay, that the firing sets.  The firing may be normed first, and a share of what is read dropped while teaching.  A recorded stretch is read at once; a car in play
is decided one moment at a time from its state.  The read-out of the memory starts at zero, so that a fresh MemoryActor
decides as its actor does.

On the GPU the library's kernels run; on the CPU the same formulas in PyTorch, moment by moment.
"""
from __future__ import annotations

import math

import torch
from torch import nn

from .fly import FlyActor
from .memory_hip import decay_attention, decay_step, delta_attention, delta_step, norm_rotary, rotary_table
from .rows_hip import dropout, layer_norm

EPS = 1e-6


def _norm_rotary_cpu(q, k, wq, wk, table, positions):
    cs = table[positions.long()][:, :, None]
    half = cs.shape[-2]

    def turn(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1], rest], -1)
    return turn(q, wq), turn(k, wk)


def _decay_attention_cpu(q, k, v, log_decay, state):
    share = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(share, 2), v.repeat_interleave(share, 2)
    l, out = torch.exp(log_decay)[:, None, None], []
    for t in range(q.shape[1]):
        state = l * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append(q.shape[-1] ** -0.5 * (q[:, t, :, None, :] @ state).squeeze(-2))
    return (torch.stack(out, 1) if out else q.new_zeros(*q.shape[:3], v.shape[-1])), state


def _delta_attention_cpu(q, k, v, log_decay, beta, state):
    share = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(share, 2), v.repeat_interleave(share, 2)
    out = []
    for t in range(q.shape[1]):
        state = torch.exp(log_decay[:, t])[..., None, None] * state
        e = v[:, t] - (k[:, t, :, None, :] @ state).squeeze(-2)
        state = state + k[:, t, :, :, None] * (beta[:, t, :, None] * e)[..., None, :]
        out.append(q.shape[-1] ** -0.5 * (q[:, t, :, None, :] @ state).squeeze(-2))
    return (torch.stack(out, 1) if out else q.new_zeros(*q.shape[:3], v.shape[-1])), state


def _dropout_cpu(x, share, counter):
    """rows_hip.dropout's numbers: Philox4x32 of 10 rounds in 64-bit integers."""
    n, low = x.numel(), 0xFFFFFFFF
    b = torch.arange(-(-n // 8))
    c0, c1, c2, c3 = b & low, b >> 32, (counter[1] & low).expand_as(b), (counter[1] >> 32 & low).expand_as(b)
    k0, k1 = counter[0] & low, counter[0] >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], -1)
    t = round(share * 65536)
    kept = (torch.stack([words & 0xFFFF, words >> 16], -1).flatten()[:n] >= t).view(x.shape)
    return torch.where(kept, x * (65536 / (65536 - t) if t < 65536 else 0.0), torch.zeros((), dtype=x.dtype))


class MemoryActor(nn.Module):
    """actor: a FlyActor.  heads query heads of dim values share k_heads key / value heads; the slowest head remembers about
    `longest` moments, the fastest 8.  positions: moments of the rotation's table.  A stretch from an empty memory may not be
    longer; a car that goes on past it keeps its memory, whose moments from there on all count as the table's last one, so that
    newer ones are no longer told apart by their distance.  On the GPU a call takes up to 16384 stretches, a step 65535 cars.
    rule: "decay", a memory that adds, each head with its decay, or "delta", one that corrects: keys of length 1, and a rate and
    a decay of each moment and head (the head's own where the firing says nothing).  norm: the firing goes through a layer norm
    first.  dropout: the share of what is read from the memory that is dropped in training mode (nn.Module.train), each pass
    another: by a seed that each actor draws from torch's generator when it is made or loaded, and the number of the pass.  A
    copy.deepcopy goes on as its original would.  Under activation checkpointing, whose second pass would drop others, it is
    refused."""

    def __init__(self, actor: FlyActor, heads: int = 8, k_heads: int | None = None, dim: int = 64, longest: float = 2048.0,
                 positions: int = 65536, rule: str = "decay", norm: bool = False, dropout: float = 0.0):
        super().__init__()
        if positions < 1:
            raise ValueError("MemoryActor: at least one position")
        k_heads = heads if k_heads is None else k_heads
        if heads % k_heads:
            raise ValueError("MemoryActor: heads must be a multiple of k_heads")
        if rule not in ("decay", "delta"):
            raise ValueError("MemoryActor: rule is decay or delta")
        if not 0 <= dropout <= 1:
            raise ValueError("MemoryActor: dropout is a share from 0 to 1")
        self.actor, self.heads, self.k_heads, self.dim = actor, heads, k_heads, dim
        firing, actions = actor.out.in_features, actor.out.out_features
        self.proj = nn.Linear(firing, (heads + 2 * k_heads) * dim, bias=False)
        self.rule, self.dropout = rule, float(dropout)
        self.wq = nn.Parameter(torch.ones(dim))
        if rule == "decay":
            self.wk = nn.Parameter(torch.ones(dim))
        else:
            self.register_buffer("wk", torch.full((dim,), dim ** -0.5))       # (keys stay of length 1)
        self.back = nn.Linear(heads * dim, actions, bias=False)
        nn.init.zeros_(self.back.weight)
        memory = torch.logspace(0, 1, heads, dtype=torch.float64).log10() * (torch.tensor(longest).log2() - 3) + 3
        self.register_buffer("log_decay", -torch.exp2(-memory).float())
        self.register_buffer("table", rotary_table(positions, dim - dim % 2), persistent=False)
        if rule == "delta":
            self.gates = nn.Linear(firing, 2 * heads)
            nn.init.zeros_(self.gates.weight)
            nn.init.zeros_(self.gates.bias)
        self.norm_w, self.norm_b = (nn.Parameter(torch.ones(firing)), nn.Parameter(torch.zeros(firing))) if norm else (None, None)
        if self.dropout:
            # (seed, pass): the seed is drawn, so that no two actors of a process drop the same numbers
            self.register_buffer("drops", torch.cat([torch.randint(1 << 62, (1,)), torch.zeros(1, dtype=torch.int64)]), persistent=False)

    def checkpoint(self, graph: str) -> dict:
        """What MemoryActor.load reads: the memory, and the actor that it was taught on (as flyguy_amd.teach writes actors)."""
        held = {k: v.detach().cpu() for k, v in self.state_dict().items()}
        return {"memory": {k: v for k, v in held.items() if not k.startswith("actor.")},
                "model": {k: v for k, v in held.items() if k.startswith("actor.")},
                "config": {"heads": self.heads, "k_heads": self.k_heads, "dim": self.dim, "positions": len(self.table),
                           "rule": self.rule, "norm": self.norm_w is not None, "dropout": self.dropout,
                           "observation": self.actor.obs_dim, "actions": self.actor.out.out_features,
                           "model": {"fly_graph": str(graph), "fly_hops": self.actor.hops, "fly_fan": self.actor.fan}}}

    @classmethod
    def load(cls, path, graph: str | None = None) -> "MemoryActor":
        """A MemoryActor from a checkpoint (flyguy_amd.remember writes them); graph: where the actor's graph lies now."""
        ck = torch.load(path, map_location="cpu", weights_only=True)
        c = ck["config"]
        m = c["model"]
        net = cls(FlyActor(graph or m["fly_graph"], c["observation"], c["actions"], hops=m["fly_hops"], fan=m["fly_fan"]),
                  heads=c["heads"], k_heads=c["k_heads"], dim=c["dim"], positions=c["positions"],
                  rule=c.get("rule", "decay"), norm=c.get("norm", False), dropout=c.get("dropout", 0.0))
        net.load_state_dict({**ck["memory"], **ck["model"]})
        return net

    def state(self, cars: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The memory of cars that have seen nothing: (states, moments seen)."""
        dev = self.log_decay.device
        return (torch.zeros(cars, self.heads, self.dim, self.dim, device=dev),
                torch.zeros(cars, dtype=torch.int32, device=dev))

    def _see(self, obs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(the actor's logits, its descending neurons' firing) of moments [n, observation]."""
        n = obs.shape[0]
        if obs.is_cuda and n % 32:                # (the library's products take batches of whole tiles)
            obs = torch.cat([obs, obs.new_zeros(-n % 32, obs.shape[1])])
        logits, firing = self.actor.with_firing(obs)
        return logits[:n], firing[:n]

    def _heads(self, firing: torch.Tensor):
        """(queries, keys, values, log decays, rates) of moments [.., firing]; decays of a head, and no rates, where the memory adds."""
        if self.norm_w is not None:
            firing = layer_norm(firing, self.norm_w, self.norm_b) if firing.is_cuda else \
                nn.functional.layer_norm(firing, firing.shape[-1:], self.norm_w, self.norm_b)
        split = self.proj(firing).split([self.heads * self.dim, self.k_heads * self.dim, self.k_heads * self.dim], -1)
        heads = [x.unflatten(-1, (-1, self.dim)) for x in split]
        if self.rule == "decay":
            return (*heads, self.log_decay, None)
        forget, rate = self.gates(firing).to(self.log_decay.dtype).unflatten(-1, (2, -1)).unbind(-2)   # (float32 under autocast too)
        return (*heads, self.log_decay * (nn.functional.softplus(forget) / math.log(2)), torch.sigmoid(rate))

    def _dropped(self, o: torch.Tensor) -> torch.Tensor:
        if not self.dropout:
            return o
        if torch._C._current_graph_task_id() >= 0:
            raise RuntimeError("MemoryActor: a pass that is made again while gradients are taken (activation checkpointing) would drop "
                               "other numbers than the first; checkpoint without dropout, or take the memory out of it")
        now = self.drops.clone()
        self.drops[1:] += 1
        return dropout(o, self.dropout, now) if o.is_cuda else _dropout_cpu(o, self.dropout, now)

    def _at(self, moments: torch.Tensor) -> torch.Tensor:
        return moments.clamp_max(len(self.table) - 1)

    def forward(self, obs: torch.Tensor, state: tuple | None = None):
        """Stretches of consecutive moments obs [cars, moments, observation] -> (logits [cars, moments, actions], the
        memory after them)."""
        return self._stretches(obs, state, self.training)

    def _stretches(self, obs: torch.Tensor, state: tuple | None, drops: bool):
        N, T = obs.shape[:2]
        if state is None and T > len(self.table):
            raise ValueError(f"MemoryActor: a stretch of {T} moments; positions is {len(self.table)}")
        mem, seen = self.state(N) if state is None else state
        logits, firing = self._see(obs.flatten(0, 1))
        q, k, v, decay, rate = self._heads(firing.unflatten(0, (N, T)))
        at = self._at(seen[:, None] + torch.arange(T, device=obs.device, dtype=torch.int32))
        if obs.is_cuda:
            q, k = norm_rotary(q, k, self.wq, self.wk, self.table, at, eps=EPS)
            o, mem = decay_attention(q, k, v, decay, mem) if rate is None else delta_attention(q, k, v, decay, rate, mem)
        else:
            q, k = _norm_rotary_cpu(q, k, self.wq, self.wk, self.table, at)
            o, mem = _decay_attention_cpu(q, k, v, decay, mem) if rate is None else _delta_attention_cpu(q, k, v, decay, rate, mem)
        o = self._dropped(o.flatten(-2)) if drops else o.flatten(-2)
        return logits.unflatten(0, (N, T)) + self.back(o), (mem, seen + T)

    @torch.no_grad()
    def step(self, obs: torch.Tensor, state: tuple) -> torch.Tensor:
        """One new moment of each car, obs [cars, observation] -> logits; the cars' memory is updated in place.  Nothing is dropped."""
        mem, seen = state
        if not obs.is_cuda:
            logits, (after, _) = self._stretches(obs[:, None], state, False)
            mem.copy_(after)
            seen += 1
            return logits[:, 0]
        logits, firing = self._see(obs)
        q, k, v, decay, rate = self._heads(firing)
        q, k = norm_rotary(q[:, None], k[:, None], self.wq, self.wk, self.table, self._at(seen[:, None]), eps=EPS)
        o = decay_step(q[:, 0], k[:, 0], v, decay, mem) if rate is None else delta_step(q[:, 0], k[:, 0], v, decay, rate, mem)
        seen += 1
        return logits + self.back(o.flatten(-2))
