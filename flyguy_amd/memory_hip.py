"""A memory over decisions on the MI355X library: rotary positions, per-head norms with the rotation, and linear attention
with a decay for each head (include/flyguy_memory.h).  An addition: the reference remembers nothing from one decision to
the next (flyguy/fly.py:286-305 decides each moment alone).

    q, k = rotary(q, k, table, positions)                       # turned by their positions
    q, k = norm_rotary(q, k, wq, wk, table, positions)          # each head's norm and the turn, in one pass
    o, state = decay_attention(q, k, v, log_decay, state)       # whole stretches, from a state and to a state
    o = decay_step(q, k, v, log_decay, state)                   # one new moment, the state updated in place

Queries and keys are [stretches, moments, heads, values] (decay_step: [rows, heads, values]), float32, bfloat16 or
binary16, on the GPU, with any strides whose last is 1 (another last stride costs a copy); query heads share key / value
heads in consecutive groups.  The first three have gradients (backwards, of the first order; tables and decays are fixed).
Work goes to the current stream; nothing synchronises.
"""
from __future__ import annotations

import struct

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from ._lib import LibraryError, check, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TURN = struct.Struct("=44qd")
_ATTENTION = struct.Struct("=36qd")
_STEP = struct.Struct("=24qd")
_PARTIAL_ROWS = 2 * 1024                # fm_turn_partial's most, in rows of a head's values


def rotary_table(positions: int, dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 taught: int = 0, slow: float = 1.0, fast: float = 32.0, device=None) -> torch.Tensor:
    """The table of (cos, sin) a rotation of `dim` values (even) reads, float32 [positions, dim / 2, 2], computed in 64
    bits: pair i of position p turns by p base^(-2i / dim).  For stretches `factor` times longer than the `taught` ones:
      linear  every position divided by factor
      base    the base raised to base factor^(dim / (dim - 2)): the slowest pair turns by 1 / factor, the fastest is kept
      bands   pairs that turn more than `fast` times over `taught` positions are kept, those that turn fewer than `slow`
              times are divided by factor, and between the two the division is blended in linearly
    """
    if dim < 2 or dim % 2 or positions < 0:
        raise ValueError("rotary_table: an even number of values, from 2, and at least 0 positions")
    if factor <= 0 or base <= 0:
        raise ValueError("rotary_table: base and factor must be positive")
    i = np.arange(0, dim, 2, dtype=np.float64)
    if scaling == "base":
        if dim < 4:
            raise ValueError("rotary_table: scaling 'base' takes at least 4 values")
        base = base * factor ** (dim / (dim - 2))
    turn = float(base) ** (-i / dim)
    if scaling == "linear":
        turn = turn / factor
    elif scaling == "bands":
        if taught <= 0 or not fast > slow:
            raise ValueError("rotary_table: scaling 'bands' takes the taught length, and fast > slow")
        keep = np.clip((taught * turn / (2 * np.pi) - slow) / (fast - slow), 0.0, 1.0)
        turn = turn * (keep + (1 - keep) / factor)
    elif scaling not in ("none", "base"):
        raise ValueError("rotary_table: scaling is none, linear, base or bands")
    a = np.arange(positions, dtype=np.float64)[:, None] * turn
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).to(device or "cpu")


# ------------------------------------------------------------------------------------------------ calls
_functions: dict = {}


def _call(name: str, x: torch.Tensor, args: bytes) -> None:
    """The call on x's device and its current stream."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(lib(), name)
    dev = x.get_device()
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _call(name, x, args)
    if fn(args, torch._C._cuda_getCurrentRawStream(dev)):
        check(name)
        raise LibraryError(f"{name} failed")


def _ptr(x: torch.Tensor | None) -> int:
    return 0 if x is None else x.data_ptr()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with its heads' values side by side."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _like(x: torch.Tensor | None) -> torch.Tensor | None:
    """Memory for as many values as x, in x's order where that leaves a head's values side by side (views whose rows overlap,
    as unfold's, can come out with another dimension innermost)."""
    if x is None:
        return None
    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 or y.shape[-1] == 1 else x.new_empty(x.shape)


def _heads(what: str, dims: int, *tensors) -> None:
    """Every tensor on one GPU, of one type and `dims` dimensions."""
    first = tensors[0]
    for i, x in enumerate(tensors):
        if not isinstance(x, torch.Tensor) or not x.is_cuda:
            raise ValueError(f"{what}: {'qkv'[i]} must be a tensor on the GPU")
        if x.dtype not in _TYPES or x.dim() != dims:
            raise ValueError(f"{what}: {'qkv'[i]} must be float32, bfloat16 or float16 of {dims} dimensions")
        if x.dtype != first.dtype or x.device != first.device:
            raise ValueError(f"{what}: {'qkv'[i]} is of another type or on another device")


def _floats(what: str, name: str, x, shape: tuple, device) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.device != device or x.shape != shape:
        raise ValueError(f"{what}: {name} must be float32 {list(shape)} on the same GPU")
    return x if x.is_contiguous() else x.contiguous()


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors)


def _no_tangents(what: str, *tensors) -> None:
    """The library's calls take no tangents along: forward-mode derivatives would come out as zero."""
    if forward_ad._current_level >= 0 and any(isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None
                                              for x in tensors):
        raise RuntimeError(f"{what}: has no forward-mode derivative")


_NONE = (0, 0, 0, 0)


def _view4(x: torch.Tensor | None) -> tuple:
    return _NONE if x is None else (x.data_ptr(), *x.stride()[:3])


def _view3(x: torch.Tensor | None) -> tuple:
    return _NONE if x is None else (x.data_ptr(), 0, *x.stride()[:2])


def _once(what: str) -> None:
    """A gradient that is asked for with a graph of its own (create_graph) would be taken for a constant there."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what}: its gradient has no gradient (create_graph)")


# ------------------------------------------------------------------------------------------------ rotation and norm
class _Plan:
    """What a turn of queries and keys shares with its gradient."""
    __slots__ = ("table", "positions", "pos", "heads", "shape", "rotated", "interleaved", "eps", "type")

    def pack(self, x, y, g, weight, gweight, partial) -> bytes:
        return _TURN.pack(*_view4(x[0]), *_view4(x[1]), *_view4(y[0]), *_view4(y[1]), *_view4(g[0]), *_view4(g[1]),
                          _ptr(weight[0]), _ptr(weight[1]), _ptr(gweight[0]), _ptr(gweight[1]), _ptr(partial),
                          _ptr(self.table), _ptr(self.positions), *self.pos, *self.heads, *self.shape, self.rotated,
                          self.interleaved, self.table.shape[0] if self.table is not None else 0, self.type, self.eps)


def _plan(what, q, k, table, positions, interleaved, eps) -> _Plan:
    _no_tangents(what, q, k, table)
    _heads(what, 4, q) if k is None else _heads(what, 4, q, k)
    N, T, H, D = q.shape
    if k is not None and (k.shape[:2] != q.shape[:2] or k.shape[3] != D):
        raise ValueError(f"{what}: q and k must be of the same stretches, moments and values per head")
    if not 1 <= D <= 512:
        raise ValueError(f"{what}: heads of 1 to 512 values")
    p = _Plan()
    p.rotated = 0
    if table is not None:
        if not isinstance(table, torch.Tensor) or table.dim() != 3 or table.shape[2] != 2 or \
                table.dtype != torch.float32 or table.device != q.device:
            raise ValueError(f"{what}: the table must be float32 [positions, rotated / 2, 2] on the same GPU (rotary_table)")
        if _wants_grad(table):
            raise ValueError(f"{what}: the table is fixed; one that requires a gradient would get none")
        table = table if table.is_contiguous() else table.contiguous()
        p.rotated = 2 * table.shape[1]
        if p.rotated > D:
            raise ValueError(f"{what}: the table turns more values than a head has")
    p.table, p.positions, p.pos = table, None, (0, 0, 0, 0)
    if isinstance(positions, torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device or positions.dim() > 2 or \
                positions.dim() < 1:
            raise ValueError(f"{what}: positions must be int32 or int64 [moments] or [stretches, moments] on the same GPU")
        try:
            p.positions = positions if positions.shape == (N, T) else positions.expand(N, T)
        except RuntimeError:
            raise ValueError(f"{what}: positions do not fit [stretches, moments]") from None
        p.pos = (*p.positions.stride(), 0, int(positions.dtype == torch.int64))
    elif positions is not None:
        p.pos = (0, 0, int(positions), 0)
    p.heads = (H, 0 if k is None else k.shape[2])
    p.shape, p.interleaved, p.eps, p.type = (N, T, D), int(bool(interleaved)), float(eps), _TYPES[q.dtype]
    return p


def _turn(p: _Plan, q, k, wq, wk):
    q, k = _rows(q), None if k is None else _rows(k)
    yq, yk = _like(q), _like(k)
    _call("fm_turn", q, p.pack((q, k), (yq, yk), (None, None), (wq, wk), (None, None), None))
    return yq, yk


class TurnHip(torch.autograd.Function):
    """rotary / norm_rotary with gradients: apply(q, k, wq, wk, plan) (k, wq, wk may be None)."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, p):
        ctx.p = p
        # (table and positions, so that one that is changed before the gradient is found out)
        ctx.save_for_backward(*((q, k) if wq is not None else (None, None)), wq, wk, p.table, p.positions)
        return _turn(p, q, k, wq, wk)

    @staticmethod
    def backward(ctx, gq, gk):
        _once("rotary, norm_rotary")
        q, k, wq, wk = ctx.saved_tensors[:4]
        p = ctx.p
        q, k, gq = None if q is None else _rows(q), None if k is None else _rows(k), _rows(gq)
        gk = None if not p.heads[1] else _rows(gk)
        yq, yk = _like(gq), _like(gk)
        gwq = torch.empty_like(wq) if wq is not None and ctx.needs_input_grad[2] else None
        gwk = torch.empty_like(wk) if wk is not None and ctx.needs_input_grad[3] else None
        partial = None
        if gwq is not None or gwk is not None:
            partial = wq.new_empty(_PARTIAL_ROWS * p.shape[2])
        _call("fm_turn_bwd", gq, p.pack((q, k), (yq, yk), (gq, gk), (wq, wk), (gwq, gwk), partial))
        return yq, yk, gwq, gwk, None


def rotary(q, k, table, positions=None, interleaved: bool = False):
    """q and k (k may be None) turned by their positions: the pairs of the first 2 table.shape[1] values of each head, (i,
    i + half) or, interleaved, (2i, 2i + 1); the rest passes through.  positions: int32 / int64 tensor [moments] or
    [stretches, moments], the first moment's position (an int), or None for 0, 1, ...  A position outside the table gives
    NaN.  Returns the turned (q, k), without gaps."""
    if table is None:
        raise ValueError("rotary: no table")
    p = _plan("rotary", q, k, table, positions, interleaved, 0.0)
    if _wants_grad(q, k):
        return TurnHip.apply(q, k, None, None, p)
    return _turn(p, q, k, None, None)


def norm_rotary(q, k, wq, wk, table=None, positions=None, interleaved: bool = False, eps: float = 1e-6):
    """Each head of q and k divided by its root mean square (eps added to the mean square) and multiplied by wq / wk
    (float32 [values], shared by the heads), then turned as by rotary (table None: not turned), in one pass over memory."""
    _no_tangents("norm_rotary", wq, wk)
    p = _plan("norm_rotary", q, k, table, positions, interleaved, eps)
    D = q.shape[3]
    wq = _floats("norm_rotary", "wq", wq, (D,), q.device)
    if k is None and wk is not None:
        raise ValueError("norm_rotary: wk without k")
    wk = None if k is None else _floats("norm_rotary", "wk", wk, (D,), q.device)
    if _wants_grad(q, k, wq, wk):
        return TurnHip.apply(q, k, wq, wk, p)
    return _turn(p, q, k, wq, wk)


# ------------------------------------------------------------------------------------------------ linear attention
class _Stretches:
    __slots__ = ("starts", "sizes", "state", "V", "scale", "log_decay")

    def pack(self, q, k, v, go=None, state=None, o=None, state_out=None, gstate_out=None, gq=None, gk=None, gv=None,
             gstate=None, work=None) -> bytes:
        vq, vk, vv, vg = (_view4(q), _view4(k), _view4(v), _view4(go)) if self.starts is None else \
            (_view3(q), _view3(k), _view3(v), _view3(go))
        return _ATTENTION.pack(*vq, *vk, *vv, *vg, _ptr(self.log_decay), _ptr(state), _ptr(self.starts), _ptr(o),
                               _ptr(state_out), _ptr(gstate_out), _ptr(gq), _ptr(gk), _ptr(gv), _ptr(gstate), _ptr(work),
                               0 if work is None else work.numel(), *self.sizes, self.scale)

    def workspace(self, q, k, v, backward: bool, **given) -> torch.Tensor | None:
        sizes = (self.starts is None, backward, *self.sizes)
        n = _workspaces.get(sizes)
        if n is None:
            if len(_workspaces) >= 4096:
                _workspaces.clear()
            n = _workspaces[sizes] = lib().fm_attention_workspace(self.pack(q, k, v, **given), int(backward))
        return q.new_empty(n, dtype=torch.uint8) if n else None


_workspaces: dict = {}                  # bytes by sizes: the library's answer depends on nothing else


def _attend(p: _Stretches, q, k, v, state):
    q, k, v = _rows(q), _rows(k), _rows(v)
    o = q.new_empty((*q.shape[:-1], p.V))
    state_out = p.log_decay.new_empty(p.state)
    work = p.workspace(q, k, v, False)
    _call("fm_attention", q, p.pack(q, k, v, state=state, o=o, state_out=state_out, work=work))
    return o, state_out


class DecayHip(torch.autograd.Function):
    """decay_attention with gradients: apply(q, k, v, state, stretches) (state may be None)."""

    @staticmethod
    def forward(ctx, q, k, v, state, p):
        ctx.p = p
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, state, p.log_decay, p.starts)
        return _attend(p, q, k, v, state)

    @staticmethod
    def backward(ctx, go, gstate_out):
        _once("decay_attention")
        p = ctx.p
        q, k, v, state = ctx.saved_tensors[:4]
        want = ctx.needs_input_grad
        q, k, v = _rows(q), _rows(k), _rows(v)
        go = q.new_zeros((*q.shape[:-1], p.V)) if go is None else _rows(go)
        gstate_out = None if gstate_out is None else gstate_out.contiguous()
        gq, gk, gv = (x.new_empty(x.shape) if w else None
                      for x, w in zip((q, k, v), want))
        gstate = torch.empty_like(state) if state is not None and want[3] else None
        given = dict(go=go, state=state, gstate_out=gstate_out, gq=gq, gk=gk, gv=gv, gstate=gstate)
        work = p.workspace(q, k, v, True, **given)
        _call("fm_attention_bwd", q, p.pack(q, k, v, work=work, **given))
        return gq, gk, gv, gstate, None


def _decays(what, log_decay, heads, device) -> torch.Tensor:
    if isinstance(log_decay, torch.Tensor) and log_decay.requires_grad:
        raise ValueError(f"{what}: the decays are fixed; a log_decay that requires a gradient would get none")
    return _floats(what, "log_decay", log_decay, (heads,), device)


def _shared(what, q, k, v, first: int) -> None:
    if k.shape[:first] != q.shape[:first] or v.shape[:first] != q.shape[:first] or k.shape[-1] != q.shape[-1] or \
            v.shape[first] != k.shape[first]:
        raise ValueError(f"{what}: q, k and v do not fit together")
    if not k.shape[first] or not q.shape[first] or q.shape[first] % k.shape[first]:
        raise ValueError(f"{what}: the query heads must be a multiple of the key heads")
    if not (1 <= q.shape[-1] <= 128 and 1 <= v.shape[-1] <= 128):
        raise ValueError(f"{what}: heads of 1 to 128 values")


def decay_attention(q, k, v, log_decay, state=None, starts=None, scale: float | None = None):
    """Linear attention with a decay for each query head, l = exp(log_decay[head]) (log_decay at most 1): S_t = l S_{t-1} +
    k_t v_t^T, o_t = scale q_t S_t (scale: values^-0.5 unless given), from `state` (float32 [stretches, q heads, values, v values]; None: zeros).
    starts (int32 / int64 [stretches + 1] on the GPU): q, k, v are packed, [moments, heads, values], and stretch n is
    moments starts[n] .. starts[n + 1] - 1 (any length, 0 too; moments of no stretch give zeros; where starts fall, stretches
    are cut short so that no two share a moment).  At most 16384 stretches.
    Returns (o in q's type, the state after each stretch).  Gradients of q, k, v and state; the decays are fixed."""
    what = "decay_attention"
    _no_tangents(what, q, k, v, log_decay, state)
    dims = 4 if starts is None else 3
    _heads(what, dims, q, k, v)
    _shared(what, q, k, v, dims - 2)
    p = _Stretches()
    p.starts, wide = None, 0
    if starts is None:
        n, moments = q.shape[:2]
    else:
        if not isinstance(starts, torch.Tensor) or starts.dtype not in (torch.int32, torch.int64) or starts.dim() != 1 or \
                starts.numel() < 1 or starts.device != q.device:
            raise ValueError(f"{what}: starts must be int32 or int64 [stretches + 1] on the same GPU")
        p.starts, wide = starts.contiguous(), int(starts.dtype == torch.int64)
        n, moments = starts.numel() - 1, q.shape[0]
    H, K = q.shape[-2:]
    p.V = v.shape[-1]
    p.state = (n, H, K, p.V)
    p.sizes = (wide, n, moments, H, k.shape[-2], K, p.V, _TYPES[q.dtype])
    p.scale = float(K ** -0.5 if scale is None else scale)
    p.log_decay = _decays(what, log_decay, H, q.device)
    if state is not None:
        state = _floats(what, "state", state, p.state, q.device)
    if _wants_grad(q, k, v, state):
        return DecayHip.apply(q, k, v, state, p)
    return _attend(p, q, k, v, state)


def decay_step(q, k, v, log_decay, state, slots=None, scale: float | None = None, into=None):
    """One new moment of decay_attention for each row: q [rows, q heads, values], k, v -> o [rows, q heads, v values].
    state (float32 [states, q heads, values, v values], dense) is updated in place, or the new states are written to
    `into`, another tensor like it that shares none of its memory.  slots (int32 [rows] on the GPU): the state each row goes
    on from, by default its own number; below 0: the row is idle (zeros, no state touched); past the states: NaN, no state
    touched.  No two rows of a call may name one slot.  At most 65535 rows.  No gradients."""
    what = "decay_step"
    _no_tangents(what, q, k, v, log_decay, state, into)
    _heads(what, 3, q, k, v)
    _shared(what, q, k, v, 1)
    if _wants_grad(q, k, v, state, into):
        raise ValueError(f"{what}: has no gradients; decay_attention has")
    n, Hq, K = q.shape
    V, dev = v.shape[2], q.device
    into = state if into is None else into
    for name, x in (("state", state), ("into", into)):
        if not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.device != dev or x.dim() != 4 or \
                tuple(x.shape[1:]) != (Hq, K, V) or not x.is_contiguous():
            raise ValueError(f"{what}: {name} must be dense float32 [states, {Hq}, {K}, {V}] on the same GPU")
    if into.shape != state.shape:
        raise ValueError(f"{what}: into must hold as many states")
    if slots is None:
        if state.shape[0] != n:
            raise ValueError(f"{what}: one state per row, or slots")
    elif not isinstance(slots, torch.Tensor) or slots.dtype != torch.int32 or slots.device != dev or \
            tuple(slots.shape) != (n,):
        raise ValueError(f"{what}: slots must be int32 [rows] on the same GPU")
    else:
        slots = slots.contiguous()
    log_decay = _decays(what, log_decay, Hq, dev)
    q, k, v = _rows(q), _rows(k), _rows(v)
    o = q.new_empty((n, Hq, V))
    views = [f for x in (q, k, v) for f in (x.data_ptr(), x.stride(0), 0, x.stride(1))]
    _call("fm_step", q, _STEP.pack(*views, log_decay.data_ptr(), state.data_ptr(), into.data_ptr(), _ptr(slots),
                                    o.data_ptr(), n, state.shape[0], Hq, k.shape[1], K, V, _TYPES[q.dtype],
                                    float(K ** -0.5 if scale is None else scale)))
    if not into.is_inference():
        increment_version(into)               # (autograd does not see the library's write)
    return o
