"""The memory over decisions (flyguy_amd.memory_hip: rotary, norm_rotary, decay_attention, decay_step) against 64-bit
restatements, at the sizes, layouts and values where such kernels go wrong."""
from __future__ import annotations

import math
import random

import pytest
import torch
from torch.autograd import forward_ad

import memory_helpers as ref
from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def draw(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def laid_out(x, how):
    """x [N, T, H, D] with the same values: dense, part of a wider projection (16-byte rows kept or not), or heads first."""
    N, T, H, D = x.shape
    if how == "dense":
        return x
    if how == "packed" or how == "odd":
        pad = 8 if how == "packed" else 3
        wide = torch.zeros(N, T, H * D + 2 * pad, dtype=x.dtype, device=x.device)
        part = wide[..., pad:pad + H * D].unflatten(-1, (H, D))
        part.copy_(x)
        return part
    if how == "heads first":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "values first":
        return x.movedim(3, 0).contiguous().movedim(0, 3)
    raise ValueError(how)


# ------------------------------------------------------------------------------------------------ rotation and norm
TURNS = [  # N, T, Hq, Hk, D, R, interleaved, type, layout
    (1, 1, 1, 0, 2, 2, False, F32, "dense"),
    (1, 1, 8, 8, 64, 64, False, F32, "dense"),
    (2, 5, 3, 1, 64, 64, True, BF16, "packed"),
    (3, 17, 4, 2, 128, 128, False, BF16, "packed"),
    (2, 33, 16, 4, 128, 64, True, BF16, "packed"),
    (2, 9, 5, 5, 80, 32, False, F32, "packed"),
    (2, 9, 5, 5, 80, 32, False, BF16, "odd"),
    (1, 70, 2, 2, 96, 96, False, F16, "heads first"),
    (1, 7, 3, 3, 100, 50, False, F32, "dense"),
    (1, 7, 3, 3, 100, 50, True, F16, "dense"),
    (2, 3, 2, 1, 33, 6, True, BF16, "values first"),
    (1, 3, 9, 4, 512, 512, False, F32, "dense"),
    (1, 40, 7, 2, 256, 192, False, BF16, "dense"),
    (2, 300, 1, 1, 8, 8, False, BF16, "dense"),
    (4, 100, 4, 4, 16, 16, True, F16, "dense"),
    (1, 4, 300, 1, 64, 16, False, BF16, "dense"),
    (1, 1, 1, 1, 1, 0, False, F32, "dense"),
    (1, 65, 2, 2, 24, 8, True, BF16, "packed"),
    (1, 65, 2, 2, 40, 16, False, BF16, "packed"),
    (2, 37, 5, 3, 128, 106, False, F32, "packed"),
    (1, 130, 9, 1, 128, 34, False, BF16, "packed"),
    (3, 11, 4, 4, 64, 62, False, F16, "dense"),
    (1, 9, 3, 2, 512, 298, False, BF16, "dense"),
    (2, 21, 4, 2, 64, 50, True, BF16, "packed"),
    (1, 5, 6, 6, 16, 2, False, F32, "dense"),
    (1, 5, 6, 6, 8, 6, False, BF16, "dense"),
]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("case", TURNS, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_turns_and_their_gradients(gpu_lib, case, norm):
    from flyguy_amd.memory_hip import norm_rotary, rotary, rotary_table
    N, T, Hq, Hk, D, R, il, dt, how = case
    say(f"turn {case} norm {norm}")
    if not norm and not R:
        pytest.skip("nothing to turn")
    gen = torch.Generator().manual_seed(N + T + D + R)
    q = laid_out(draw(gen, N, T, Hq, D, dtype=dt), how).requires_grad_()
    k = laid_out(draw(gen, N, T, Hk, D, dtype=dt), how).requires_grad_() if Hk else None
    table = rotary_table(2 * T + 3, R, scaling="linear", factor=2.0).cuda() if R else None
    pos = torch.randint(0, 2 * T + 3, (N, T), generator=gen, dtype=torch.int64 if D % 3 else torch.int32)
    ws = [(1 + 0.3 * draw(gen, D)).requires_grad_() for _ in range(2 if k is not None else 1)] if norm else []
    gs = [laid_out(draw(gen, *x.shape, dtype=dt), how) for x in (q, k) if x is not None]
    eps = 1e-5
    if norm:
        out = norm_rotary(q, k, ws[0], ws[1] if k is not None else None, table, pos.cuda(), interleaved=il, eps=eps)
    else:
        out = rotary(q, k, table, pos.cuda(), interleaved=il)
    out = [y for y in out if y is not None]
    xs = [x for x in (q, k) if x is not None]
    grads = torch.autograd.grad(out, xs + ws, gs)
    cs = table.cpu().double()[pos][:, :, None] if R else torch.zeros(N, T, 1, 0, 2, dtype=torch.float64)
    for i, (x, g, y, gx) in enumerate(zip(xs, gs, out, grads)):
        x, g = x.detach().cpu().double(), g.cpu().double()
        w = ws[i].detach().cpu().double() if norm else torch.ones(D, dtype=torch.float64)
        r = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if norm else torch.ones(1, dtype=torch.float64)
        z = x * r * w
        n = D if norm else 0                       # the norm's sum of D squares, then a few roundings
        ref.within(y, ref.turned(z, cs, il), ref.turned_magnitude(z, cs, il), n + 12, "value")
        gz, gm = ref.turned(g, cs, il, back=True), ref.turned_magnitude(g, cs, il)
        if not norm:
            ref.within(gx, gz, gm, 12, "gradient")
            continue
        xh, u, um = x * r, gz * w, gm * w.abs()
        want = r * (u - xh * (u * xh).mean(-1, keepdim=True))
        mag = r * (um + xh.abs() * (um * xh.abs()).mean(-1, keepdim=True))
        ref.within(gx, want, mag, 3 * D + 40, "gradient")
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        ref.within(grads[len(xs) + i], (gz * xh).sum((0, 1, 2)), (gm * xh.abs()).sum((0, 1, 2)), rows + D + 20, "weight's")


def test_norm_gradient_against_differences(gpu_lib):
    """The loss <g, y> along a direction d: (L(x + h d) - L(x - h d)) / 2h is the gradient's <gx, d> up to h^2 / 6 of the
    third derivative (of the order of the terms' magnitudes: values of order 1) and 2^-24 of L's terms / h."""
    from flyguy_amd.memory_hip import norm_rotary, rotary_table
    gen = torch.Generator().manual_seed(5)
    q, k, d = draw(gen, 2, 9, 3, 64), draw(gen, 2, 9, 2, 64), draw(gen, 2, 9, 3, 64)
    wq, wk, g = 1 + 0.2 * draw(gen, 64), 1 + 0.2 * draw(gen, 64), draw(gen, 2, 9, 3, 64)
    dw = draw(gen, 64)
    table = rotary_table(9, 32).cuda()
    loss = lambda x, w: (norm_rotary(x, k, w, wk, table)[0].double() * g.double()).sum()          # noqa: E731
    x, w = q.clone().requires_grad_(), wq.clone().requires_grad_()
    gx, gw = torch.autograd.grad(loss(x, w), [x, w])
    h = 2.0 ** -7
    for grad, way, fore, back in ((gx, d, (q + h * d, wq), (q - h * d, wq)), (gw, dw, (q, wq + h * dw), (q, wq - h * dw))):
        want = (loss(*fore) - loss(*back)) / (2 * h)
        terms = float((grad.double() * way.double()).abs().sum())
        noise = 24 * 2.0 ** -24 * float(g.abs().double().sum() * 4) / h
        assert abs(float((grad.double() * way.double()).sum()) - float(want)) <= 8 * h * h * terms + noise


OVERLAPPING = [((1, 3, 2, 4), (50, 8, 1, 1)), ((2, 5, 3, 64), (40, 3, 1, 1)), ((2, 9, 2, 8), (0, 1, 0, 1)),
               ((2, 20, 1, 24), (64, 1, 1, 1)), ((1, 7, 3, 16), (0, 0, 0, 1))]


@pytest.mark.parametrize("shape,strides", OVERLAPPING)
def test_rows_that_overlap(gpu_lib, shape, strides):
    """Views whose rows share values (windows, expanded tensors): what a copy of them gives, in memory of its own, and its
    gradients too."""
    from flyguy_amd.memory_hip import decay_attention, norm_rotary, rotary, rotary_table
    say(f"overlapping {shape} {strides}")
    gen = torch.Generator().manual_seed(20)
    q = draw(gen, 400).as_strided(shape, strides)
    D, w, g = shape[-1], draw(gen, shape[-1]), draw(gen, 400).as_strided(shape, strides)
    table = rotary_table(shape[1], D, device="cuda")
    d = decays(shape[2])

    def all_of(q, g):
        x = q.detach().requires_grad_()
        a, b = rotary(x, x, table)
        c, _ = norm_rotary(x, None, w, None, table)
        o, _ = decay_attention(x, x, x, d)
        for y in (a, b, c, o):
            assert y.stride(-1) == 1
        return [a, b, c, o, *(torch.autograd.grad(y, x, g, retain_graph=True)[0] for y in (a, b, c, o))]
    # (the copy's strides may take another form of the kernels: the same numbers up to a few roundings)
    for y, want in zip(all_of(q, g), all_of(q.contiguous(), g.contiguous())):
        torch.testing.assert_close(y, want, rtol=1e-5, atol=1e-5 * float(want.detach().abs().max()))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,R,il,dt,how", [(100, 50, False, F32, "dense"), (100, 100, False, BF16, "odd"), (100, 98, True, F16, "odd"),
                                           (33, 32, False, F32, "dense"), (511, 510, False, BF16, "dense"),
                                           (128, 128, False, F32, "odd"), (128, 106, False, BF16, "dense"),
                                           (64, 64, False, BF16, "packed"), (96, 64, True, F32, "packed"), (200, 130, False, F16, "odd")])
def test_in_place(gpu_lib, D, R, il, dt, how, norm):
    """The library writes over what it reads, queries and keys alike, bit for bit what it writes elsewhere; gradients over the
    outputs' and over the inputs."""
    from flyguy_amd.memory_hip import _call, _plan, rotary_table
    say(f"in place {D} {R} {il} {dt} {how} {norm}")
    gen = torch.Generator().manual_seed(21)
    x = [laid_out(draw(gen, 2, 9, h, D, dtype=dt), how) for h in (3, 2)]
    g = [laid_out(draw(gen, 2, 9, h, D, dtype=dt), how) for h in (3, 2)]
    w = [1 + 0.2 * draw(gen, D) for _ in range(2)] if norm else [None, None]
    p = _plan("test", *x, rotary_table(9, R, device="cuda"), None, il, 1e-6)

    def copies(xs):
        return [laid_out(y.contiguous().clone(), how) for y in xs]

    def forward(xs, ys):
        _call("fm_turn", xs[0], p.pack(xs, ys, (None, None), w, (None, None), None))
        return ys

    def backward(xs, gs, ys):
        _call("fm_turn_bwd", gs[0], p.pack(xs, ys, gs, w, (None, None), None))
        return ys
    want, a = forward(x, copies(x)), copies(x)
    for y, z in zip(want, forward(a, a)):
        assert torch.equal(y, z)
    want, a, b = backward(x, g, copies(x)), copies(g), copies(x)
    for y, z, u in zip(want, backward(x, a, a), backward(b, g, b)):
        assert torch.equal(y, z) and torch.equal(y, u)


def test_positions(gpu_lib):
    """None, an int, one row for all, int32, int64, and strided positions name the same turns; outside the table: NaN."""
    from flyguy_amd.memory_hip import rotary, rotary_table
    gen = torch.Generator().manual_seed(1)
    q = draw(gen, 2, 6, 3, 16)
    table = rotary_table(20, 8).cuda()
    at = torch.arange(6, device="cuda")
    first = rotary(q, None, table)[0]
    for pos in (0, at, at.int(), at.expand(2, 6), torch.stack([at, at], 1).int().t(), torch.stack([at, at + 1], 1)[:, 0]):
        assert torch.equal(rotary(q, None, table, pos)[0], first)
    assert torch.equal(rotary(q, None, table, 3)[0], rotary(q, None, table, at + 3)[0])
    out = rotary(q, None, table, torch.tensor([[0, -1, 19, 20, 5, 2 ** 40]], device="cuda"))[0]
    bad = torch.tensor([False, True, False, True, False, True], device="cuda")
    assert torch.isnan(out[:, bad][..., :8]).all() and torch.equal(out[..., 8:], q[..., 8:])
    assert torch.isfinite(out[:, ~bad]).all()
    assert torch.isnan(rotary(q, None, table, 18)[0][:, 2:, :, :8]).all()


def test_many_rows(gpu_lib):
    """70 million heads of two values: more workgroups than a grid's x takes threads for."""
    from flyguy_amd.memory_hip import rotary, rotary_table
    q = torch.randn(1, 70, 1000000, 2, device="cuda").bfloat16()
    table = rotary_table(70, 2).cuda()
    got = rotary(q, None, table)[0]
    c, s = table[:, 0, 0, None], table[:, 0, 1, None]
    a, b = q[0, ..., 0].float(), q[0, ..., 1].float()
    for x, y in ((got[0, ..., 0], a * c - b * s), (got[0, ..., 1], b * c + a * s)):
        assert float((x.float() - y).abs().max()) <= 2.0 ** -8 * float(y.abs().max())


@pytest.mark.parametrize("il", [False, True])
def test_values_that_are_not_turned_pass_through(gpu_lib, il):
    """Whatever they are: infinities and NaN among them touch nothing else, turned values' only their own pair."""
    from flyguy_amd.memory_hip import rotary, rotary_table
    gen = torch.Generator().manual_seed(7)
    for dt in (F32, BF16):
        q = draw(gen, 2, 5, 3, 96, dtype=dt)
        table = rotary_table(5, 32).cuda()
        clean = rotary(q, None, table, interleaved=il)[0]
        bad = q.clone()
        bad[0, 1, 2, 40], bad[0, 1, 2, 95], bad[1, 4, 0, 57], bad[1, 2, 1, 4] = (float(x) for x in ("inf", "nan", "-inf", "inf"))
        got = rotary(bad, None, table, interleaved=il)[0]
        assert torch.equal(got[..., 32:].view(torch.uint8), bad[..., 32:].view(torch.uint8))
        off = ~torch.isfinite(got[..., :32])
        pair = torch.zeros_like(off)
        pair[1, 2, 1, [4, 5] if il else [4, 20]] = True
        assert torch.equal(off, pair) and torch.equal(got[..., :32][~pair], clean[..., :32][~pair])


def test_a_norm_keeps_rows_apart(gpu_lib):
    """A row of zeros, one of infinity and one of NaN: the others are what they are without them, the row of zeros is zeros."""
    from flyguy_amd.memory_hip import norm_rotary, rotary_table
    gen = torch.Generator().manual_seed(2)
    for dt in (F32, BF16):
        q = draw(gen, 2, 8, 4, 64, dtype=dt)
        w, table = torch.ones(64, device="cuda"), rotary_table(8, 64).cuda()
        clean = norm_rotary(q, None, w, None, table)[0]
        bad = q.clone()
        bad[0, 1, 2], bad[0, 3, 1, 5], bad[1, 7, 0, 63] = 0, float("inf"), float("nan")
        got = norm_rotary(bad, None, w, None, table)[0]
        touched = torch.zeros(2, 8, 4, dtype=torch.bool)
        touched[0, 1, 2] = touched[0, 3, 1] = touched[1, 7, 0] = True
        assert torch.equal(got[~touched], clean[~touched])
        assert (got[0, 1, 2] == 0).all() and torch.isnan(got[1, 7, 0]).all() and torch.isnan(got[0, 3, 1]).any()


# ------------------------------------------------------------------------------------------------ linear attention
ATTENTION = [  # N, T, Hq, Hk, K, V, type, layout, start state
    (1, 1, 1, 1, 1, 1, F32, "dense", True),
    (1, 1, 2, 1, 64, 64, BF16, "dense", True),
    (2, 15, 2, 2, 16, 16, BF16, "packed", False),
    (1, 16, 1, 1, 128, 128, BF16, "dense", True),
    (2, 17, 3, 3, 40, 56, F16, "packed", True),
    (1, 63, 2, 2, 64, 64, F32, "packed", True),
    (2, 64, 2, 1, 64, 128, BF16, "packed", True),
    (1, 65, 4, 2, 128, 64, BF16, "dense", True),
    (1, 130, 2, 2, 128, 128, F32, "heads first", True),
    (1, 200, 1, 1, 5, 7, BF16, "odd", True),
    (1, 150, 2, 1, 72, 100, BF16, "odd", False),
    (1, 150, 2, 1, 72, 104, F32, "values first", False),
    (1, 300, 3, 1, 24, 8, F16, "dense", True),
    (2, 700, 1, 1, 32, 32, BF16, "dense", True),
    (1, 1100, 1, 1, 64, 16, F32, "dense", True),
    (1, 2500, 1, 1, 16, 64, BF16, "dense", True),
]


def decays(H):
    """From none to all at once: heads remember everything, about 1,000 / 20 / 1 moments, or nothing."""
    return torch.tensor([0.0, -1e-3, -0.05, -1.0, -30.0, -math.inf])[torch.arange(H) * 5 % 6].cuda()


def inputs(gen, N, T, Hq, Hk, K, V, dt, how, state):
    q, k, v = (laid_out(draw(gen, N, T, h, d, dtype=dt), how) for h, d in ((Hq, K), (Hk, K), (Hk, V)))
    return q, k, v, draw(gen, N, Hq, K, V) if state else None


def check_attention(q, k, v, g, s, starts=None, scale=None):
    """Values and gradients against the restatement; the bounds count a sum over K or V values inside a sum over moments,
    the powers of the decay (a rounding a chunk, and 2^-24 of an exponent of at most 88 where the power still counts), and in
    bfloat16 two terms of 8 bits each for what a product rounds (2^-16 with both operands)."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(9)
    K, V = q.shape[-1], v.shape[-1]
    c = K ** -0.5 if scale is None else scale
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([s.clone().requires_grad_()] if s is not None else [])
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    o, end = decay_attention(*leaves[:3], g, leaves[3] if s is not None else None, st, scale=scale)
    go, ge = draw(gen, *o.shape, dtype=o.dtype), draw(gen, *end.shape)
    grads = torch.autograd.grad([o, end], leaves, [go, ge])
    f = [x.detach().cpu().double() if x is not None else None for x in (q, k, v, s, go, ge)]
    args = dict(log_decay=g.cpu(), starts=starts)
    want = ref.attention(*f[:3], state=f[3], scale=c, go=f[4], gs=f[5], **args)
    m = [x.abs() if x is not None else None for x in f]
    mag = ref.attention(*m[:3], state=m[3], scale=abs(c), go=m[4], gs=m[5], **args)
    T = max(e - b for b, e in zip(starts[:-1], starts[1:])) if starts else q.shape[1]
    count, extra = K + V + T + 200, 2.0 ** -16 if q.dtype == BF16 else 0.0
    for i, what in enumerate(("o", "end state", "gradient of q", "of k", "of v", "of the state")):
        got = (o, end, *grads)[i] if i < 5 or s is not None else None
        if got is not None:
            ref.within(got, want[i], mag[i], count, what, extra)
    return o, end


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_attention_and_its_gradients(gpu_lib, case):
    say(f"attention {case}")
    N, T, Hq, Hk, K, V, dt, how, state = case
    gen = torch.Generator().manual_seed(T + K)
    check_attention(*inputs(gen, N, T, Hq, Hk, K, V, dt, how, state)[:3], decays(Hq),
                    draw(gen, N, Hq, K, V) if state else None)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("lengths", [[0], [1], [0, 3, 0, 64, 1, 129, 0], [65, 63, 2, 700, 17, 16], [1200, 5], [0, 700, 0, 600, 0]])
def test_packed_stretches(gpu_lib, dt, lengths):
    say(f"packed {lengths} {dt}")
    gen = torch.Generator().manual_seed(len(lengths))
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    H, Hk, K, V = 4, 2, 48, 40
    q, k, v = (draw(gen, starts[-1], h, d, dtype=dt) for h, d in ((H, K), (Hk, K), (Hk, V)))
    check_attention(q, k, v, decays(H), draw(gen, len(lengths), H, K, V), starts)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_many_short_stretches_and_a_few_long_ones(gpu_lib, dt):
    """The long ones are cut, wherever they lie among the short ones; moments before the first stretch belong to none."""
    say(f"many packed {dt}")
    rng = random.Random(5)
    lengths = [rng.randint(0, 12) for _ in range(300)]
    for n, at in ((64, 0), (500, 1), (65, 70), (129, 200), (777, 299)):
        lengths[at] = n
    gen = torch.Generator().manual_seed(6)
    starts = [70]
    for n in lengths:
        starts.append(starts[-1] + n)
    q, k, v = (draw(gen, starts[-1], h, d, dtype=dt) for h, d in ((2, 24), (1, 24), (1, 32)))
    check_attention(q, k, v, decays(2), draw(gen, len(lengths), 2, 24, 32), starts)


def test_more_chains_than_half_of_what_fits(gpu_lib):
    """So many heads that the gradient's first segments are shorter than the rest: a few heads against the restatement."""
    say("uneven segments")
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(8)
    H, T, K = 128, 2100, 128
    q, k, v, go = (draw(gen, 1, T, H, K, dtype=BF16) for _ in range(4))
    s, ge, g = draw(gen, 1, H, K, K), draw(gen, 1, H, K, K), decays(H)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, s)]
    o, end = decay_attention(*leaves[:3], g, leaves[3])
    grads = torch.autograd.grad([o, end], leaves, [go, ge])
    few = [0, 61, 127]
    f = [x[..., few, :].cpu().double() for x in (q, k, v)] + [x[:, few].cpu().double() for x in (s, ge)]
    args = dict(log_decay=g[few].cpu(), starts=None, scale=K ** -0.5)
    do = go[..., few, :].cpu().double()
    want = ref.attention(*f[:3], state=f[3], go=do, gs=f[4], **args)
    m = [x.abs() for x in f]
    mag = ref.attention(*m[:3], state=m[3], go=do.abs(), gs=m[4], **args)
    for i, (got, what) in enumerate(zip((o, end, *grads), ("o", "end state", "gradient of q", "of k", "of v", "of the state"))):
        got = got[:, few] if i in (1, 5) else got[..., few, :]
        ref.within(got, want[i], mag[i], 2 * K + T + 200, what, 2.0 ** -16)


def test_starts_of_another_kind(gpu_lib):
    """int64 starts give the int32 ones' results; moments of no stretch give zeros, and take no gradient; starts beyond the
    moments, or falling, read nothing outside."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(3)
    q, k, v = (draw(gen, 200, 2, 32) .requires_grad_() for _ in range(3))
    g = decays(2)
    starts = torch.tensor([10, 70, 70, 190], dtype=torch.int32, device="cuda")
    o, s = decay_attention(q, k, v, g, None, starts)
    o64, s64 = decay_attention(q, k, v, g, None, starts.long())
    assert torch.equal(o, o64) and torch.equal(s, s64)
    assert (o[:10] == 0).all() and (o[190:] == 0).all() and (o[10:190].abs().sum((1, 2)) > 0).all()
    for x in torch.autograd.grad([o, s], [q, k, v], [torch.ones_like(o), torch.ones_like(s)]):
        assert (x[:10] == 0).all() and (x[190:] == 0).all() and torch.isfinite(x).all()
    o2, s2 = decay_attention(q, k, v, g, None, torch.tensor([-5, 100, 500], dtype=torch.int32, device="cuda"))
    w, sw = decay_attention(q, k, v, g, None, torch.tensor([0, 100, 200], dtype=torch.int32, device="cuda"))
    assert torch.equal(o2, w) and torch.equal(s2, sw)
    decay_attention(q, k, v, g, None, torch.tensor([150, 20, 400, -3], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dt,V", [(F32, 24), (BF16, 7), (F16, 40)])
@pytest.mark.parametrize("Hk", [3, 1])
def test_a_pack_with_room_before_and_behind(gpu_lib, dt, V, Hk):
    """Two stretches in the middle of a place for many times as much: the values and gradients of the stretches alone, zeros
    elsewhere, whatever the memory held."""
    from flyguy_amd.memory_hip import decay_attention
    say(f"room {dt} {V} {Hk}")
    gen = torch.Generator().manual_seed(19)
    M, b, n = 5003, 1501, 333
    q, k, v, go = (draw(gen, M, h, d, dtype=dt) for h, d in ((3, 8), (Hk, 8), (Hk, V), (3, V)))

    def both(q, k, v, go, starts):
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
        held = [torch.full((M, 3, d), float("nan"), dtype=dt, device="cuda") for d in (8, 8, V, V, V)]
        del held
        o, e = decay_attention(*leaves, decays(3), None, torch.tensor(starts, dtype=torch.int32, device="cuda"))
        return (o, *torch.autograd.grad([o, e], leaves, [go, torch.ones_like(e)])), e
    got, e = both(q, k, v, go, [b, b + 100, b + n])
    want, e2 = both(*(x[b:b + n] for x in (q, k, v, go)), [0, 100, n])
    for x, y in zip(got, want):
        small = {F32: 1e-5, BF16: 2.0 ** -7, F16: 2.0 ** -10}[dt]      # (other segments: sums in another order, one more rounding)
        torch.testing.assert_close(x[b:b + n], y, rtol=small, atol=small * float(y.detach().abs().max()))
        assert (x[:b] == 0).all() and (x[b + n:] == 0).all()
    torch.testing.assert_close(e, e2, rtol=1e-5, atol=1e-5 * float(e2.detach().abs().max()))


FALLING = [[150, 20, 400, -3], [0, 60, 30, 200], [7, 190, 3, 195, 100, 110, 200], [200, 0], [90, 10, 20, 30], [0, 0, -9, 5, 5]]


@pytest.mark.parametrize("dt,wide", [(F32, False), (BF16, True)])
@pytest.mark.parametrize("case", range(len(FALLING) + 5))
def test_starts_that_fall(gpu_lib, case, dt, wide):
    """No two stretches share a moment, whatever the starts: values and gradients are those of starts that do not fall with the
    same stretches; of a few stretches, those that begin at the largest start so far."""
    from flyguy_amd.memory_hip import decay_attention
    say(f"falling {case} {dt}")
    rng = random.Random(case)
    if case < len(FALLING):
        starts, M = FALLING[case], 200
    else:
        n_seq, M = ((5, 3000), (63, 4000), (64, 4000), (700, 9000), (4100, 30000))[case - len(FALLING)]
        starts = sorted(rng.randint(-50, M + 50) for _ in range(n_seq + 1))
        for _ in range(max(2, n_seq // 9)):
            starts[rng.randrange(n_seq + 1)] = rng.randint(-50, M + 50)
    same = ref.risen(starts, M)
    if len(starts) <= 8:
        b, top = [min(max(x, 0), M) for x in starts], 0
        for n, x in enumerate(b):
            top = max(top, x)
            assert same[n] == top
    gen = torch.Generator().manual_seed(case)
    q, k, v = (draw(gen, M, h, d, dtype=dt).requires_grad_() for h, d in ((2, 24), (1, 24), (1, 32)))
    n = len(starts) - 1
    s, go, ge = draw(gen, n, 2, 24, 32).requires_grad_(), draw(gen, M, 2, 32, dtype=dt), draw(gen, n, 2, 24, 32)
    outs = []
    for st in (starts, same):
        st = torch.tensor(st, dtype=torch.int64 if wide else torch.int32, device="cuda")
        held = [torch.full((M, 2, 32), float("nan"), dtype=dt, device="cuda") for _ in range(6)]
        del held
        o, e = decay_attention(q, k, v, decays(2), s, st)
        outs.append((o, e, *torch.autograd.grad([o, e], [q, k, v, s], [go, ge])))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert (outs[0][0][:same[0]] == 0).all() and (outs[0][0][same[-1]:] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_no_moments(gpu_lib, dt):
    """No moments pass the state on, both ways; no stretches give nothing."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(4)
    s = draw(gen, 3, 2, 16, 24).requires_grad_()
    q, k, v = (torch.empty(3, 0, 2, d, dtype=dt, device="cuda") for d in (16, 16, 24))
    o, e = decay_attention(q, k, v, decays(2), s)
    assert o.shape == (3, 0, 2, 24) and torch.equal(e, s)
    assert torch.equal(torch.autograd.grad(e, s, 2 * torch.ones_like(e))[0], 2 * torch.ones_like(e))
    o, e = decay_attention(q[:0], k[:0], v[:0], decays(2))
    assert o.shape == (0, 0, 2, 24) and e.shape == (0, 2, 16, 24)


@pytest.mark.parametrize("lengths", [None, [0, 0], [0, 5, 0], [70, 0, 2500, 0]])
def test_no_moments_pass_any_state_on(gpu_lib, lengths):
    """Infinities and NaN too, bit for bit, and so the end state's gradient; at any decay."""
    from flyguy_amd.memory_hip import decay_attention
    say(f"pass on {lengths}")
    gen = torch.Generator().manual_seed(22)
    n = 3 if lengths is None else len(lengths)
    s, ge = (draw(gen, n, 6, 16, 24) for _ in range(2))
    for x in (s, ge):
        x[:, :, 3, 5], x[:, :, 0, 1], x[:, :, 15, 23] = math.inf, -math.inf, math.nan
    if lengths is None:
        q, k, v = (torch.empty(3, 0, 6, d, device="cuda") for d in (16, 16, 24))
        st, empty = None, range(3)
    else:
        starts = [0]
        for x in lengths:
            starts.append(starts[-1] + x)
        q, k, v = (draw(gen, starts[-1], 6, d) for d in (16, 16, 24))
        st, empty = torch.tensor(starts, dtype=torch.int32, device="cuda"), [i for i, x in enumerate(lengths) if not x]
    s.requires_grad_()
    _, e = decay_attention(q, k, v, decays(6), s, st)
    g, = torch.autograd.grad(e, s, ge)
    for i in empty:
        assert torch.equal(e[i].view(torch.int32), s[i].view(torch.int32)), i
        assert torch.equal(g[i].view(torch.int32), ge[i].view(torch.int32)), i


@pytest.mark.parametrize("T", [1, 64, 130, 3000])
def test_a_state_kept_whole(gpu_lib, T):
    """A decay of 1 leaves an infinite entry of the state infinite."""
    from flyguy_amd.memory_hip import decay_attention, decay_step
    gen = torch.Generator().manual_seed(23)
    q, k, v, s = inputs(gen, 1, T, 1, 1, 32, 32, F32, "dense", True)
    s[0, 0, 3, 5], s[0, 0, 9, 1] = math.inf, -math.inf
    g, into = torch.zeros(1, device="cuda"), torch.empty_like(s)
    decay_step(q[:, 0], k[:, 0], v[:, 0], g, s, into=into)
    for e in (decay_attention(q, k, v, g, s)[1], into):
        assert e[0, 0, 3, 5] == math.inf and e[0, 0, 9, 1] == -math.inf
        assert torch.equal(torch.isfinite(e), torch.isfinite(s))


@pytest.mark.parametrize("K,V", [(16, 16), (128, 128)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_growing_states_that_are_zero_for_long(gpu_lib, dt, K, V):
    """log_decay 1: what is zero stays zero over any number of moments, forwards and backwards."""
    from flyguy_amd.memory_hip import decay_attention
    say(f"growing {dt} {K}")
    gen = torch.Generator().manual_seed(24)
    T, n = 65536, 40
    q, k, v, go = (draw(gen, 1, T, 1, d, dtype=dt) for d in (K, K, V, V))
    g = torch.ones(1, device="cuda")
    late = k.clone()
    late[:, :-n] = 0
    o, e = decay_attention(q, late, v, g)
    f = [x[:, -n:].cpu().double() for x in (q, k, v)]
    want = ref.attention(*f, g.cpu(), None, K ** -0.5)
    mag = ref.attention(*[x.abs() for x in f], g.cpu(), None, K ** -0.5)
    extra = 2.0 ** -16 if dt == BF16 else 0.0
    assert (o[:, :-n] == 0).all()
    ref.within(o[:, -n:], want[0], mag[0], K + V + n + 200, "o", extra)
    ref.within(e, want[1], mag[1], K + V + n + 200, "end state", extra)
    early_q, leaves = q.clone(), [k.clone().requires_grad_(), v.clone().requires_grad_()]
    early_q[:, n:] = 0
    go[:, n:] = 0
    grads = torch.autograd.grad(decay_attention(early_q, *leaves, g)[0], leaves, go)
    f = [x[:, :n].cpu().double() for x in (q, k, v, go)]
    want = ref.attention(*f[:3], g.cpu(), None, K ** -0.5, go=f[3])
    mag = ref.attention(*[x.abs() for x in f[:3]], g.cpu(), None, K ** -0.5, go=f[3].abs())
    for i, x in zip((3, 4), grads):
        assert (x[:, n:] == 0).all()
        ref.within(x[:, :n], want[i], mag[i], K + V + n + 200, "gradient", extra)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("Hk", [4, 2])
def test_moments_of_no_stretch_at_all(gpu_lib, dt, Hk):
    """Packed moments and no stretches: zeros, and gradients of zero, whatever the memory held before."""
    from flyguy_amd.memory_hip import decay_attention
    say(f"no stretch {dt} {Hk}")
    gen = torch.Generator().manual_seed(18)
    q, k, v = (draw(gen, 200, h, d, dtype=dt).requires_grad_() for h, d in ((4, 24), (Hk, 24), (Hk, 40)))
    starts = torch.zeros(1, dtype=torch.int32, device="cuda")
    go = draw(gen, 200, 4, 40, dtype=dt)
    for _ in range(3):
        held = [torch.full((200, 4, d), float("nan"), dtype=dt, device="cuda") for d in (24, 40, 24, 40)]
        del held
        o, e = decay_attention(q, k, v, decays(4), None, starts)
        assert (o == 0).all() and e.shape == (0, 4, 24, 40)
        held = [torch.full((200, 4, d), float("nan"), dtype=dt, device="cuda") for d in (24, 24, 40, 40)]
        del held
        for x, g in zip((q, k, v), torch.autograd.grad(o, (q, k, v), go)):
            assert g.shape == x.shape and (g == 0).all()
    decay_attention(q[:0], k[:0], v[:0], decays(4), None, starts)


@pytest.mark.parametrize("dt,K,V", [(F32, 64, 64), (BF16, 64, 128), (BF16, 128, 48), (F16, 40, 40)])
def test_a_later_moment_does_not_reach_an_earlier_one(gpu_lib, dt, K, V):
    """NaN and infinities at a moment leave the outputs before it, and the gradients after it, as they were, bit for bit;
    another stretch's leave a stretch alone."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(6)
    q, k, v, _ = inputs(gen, 2, 200, 2, 2, K, V, dt, "dense", False)
    go = draw(gen, 2, 200, 2, V, dtype=dt)
    g = torch.tensor([-0.02, -1.0], device="cuda")

    def both(q, k, v, go):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        o, _ = decay_attention(*leaves, g)
        return (o.detach(), *torch.autograd.grad(o, leaves, go))
    clean = both(q, k, v, go)
    for t, bad in ((5, math.nan), (77, math.inf), (100, -math.inf), (64, math.nan), (199, math.inf), (120, math.nan)):
        for which in range(4):
            x = [y.clone() for y in (q, k, v, go)]
            x[which][0, t, 1, 3] = bad
            got = both(*x)
            # o at moments before t; the gradients of q before t (of k, v there t is among the later moments)
            for i in (0, 1):
                if which != 3 or i == 1:
                    assert torch.equal(got[i][0, :t], clean[i][0, :t]), (t, bad, which, i)
            for i in (2, 3):                       # the gradients of k and v at moments after t
                assert torch.equal(got[i][0, t + 1:], clean[i][0, t + 1:]), (t, bad, which, i)
            for i in range(4):
                assert torch.equal(got[i][1], clean[i][1]) and torch.equal(got[i][0, :, 0], clean[i][0, :, 0])
            if which < 3:
                assert not torch.isfinite(got[0][0, t, 1]).all()


def test_gradients_against_differences(gpu_lib):
    """The loss <go, o> + <ge, end> is linear in q, in k, in v and in the state, so its whole difference along any d is <gx,
    d>, up to the roundings of both sides: T + K + V + 200 of the terms' magnitudes (f32)."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(8)
    q, k, v, s = inputs(gen, 2, 150, 4, 2, 32, 24, F32, "dense", True)
    go, ge = draw(gen, 2, 150, 4, 24), draw(gen, 2, 4, 32, 24)
    g = decays(4)

    def loss(*x):
        o, e = decay_attention(*x[:3], g, x[3])
        return (o.double() * go.double()).sum() + (e.double() * ge.double()).sum()
    base = [q, k, v, s]
    leaves = [x.clone().requires_grad_() for x in base]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(4):
        d = draw(gen, *base[i].shape)
        moved = [x + d if j == i else x for j, x in enumerate(base)]
        mags = [x.abs().cpu().double() for x in (moved[i].abs() + base[i].abs() if j == i else base[j] for j in range(4))]
        o, e = ref.attention(mags[0], mags[1], mags[2], g.cpu(), mags[3], 32 ** -0.5)
        terms = float((o * go.abs().cpu().double()).sum() + (e * ge.abs().cpu().double()).sum())
        diff = float(loss(*moved) - loss(*base))
        assert abs(diff - float((grads[i].double() * d.double()).sum())) <= 406 * ref.U * terms


def test_parts_of_the_gradient(gpu_lib):
    """Any subset of inputs with gradients, and either output's gradient missing, gives the whole call's values."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(10)
    for Hk in (2, 1):
        base = inputs(gen, 1, 90, 2, Hk, 16, 24, F32, "dense", True)
        go, ge = draw(gen, 1, 90, 2, 24), draw(gen, 1, 2, 16, 24)

        def grads(wanted, outs):
            x = [b.clone().requires_grad_(i in wanted) for i, b in enumerate(base)]
            res = decay_attention(*x[:3], decays(2), x[3])
            gs = torch.autograd.grad([res[j] for j in outs], [x[i] for i in wanted], [(go, ge)[j] for j in outs])
            return dict(zip(wanted, gs))
        for outs in ((0, 1), (0,), (1,)):
            whole = grads((0, 1, 2, 3), outs) if 0 in outs else {**grads((1, 2, 3), outs)}
            for wanted in ((0,), (1,), (2,), (3,), (1, 3), (0, 2)):
                if outs == (1,) and 0 in wanted:
                    continue                      # (the end state does not depend on q)
                for i, x in grads(wanted, outs).items():
                    assert torch.equal(x, whole[i]), (Hk, outs, wanted, i)


def test_a_gradient_is_refused_where_it_would_be_wrong(gpu_lib):
    """Gradients of gradients, and a gradient after its inputs, positions, starts or decays were changed in place."""
    from flyguy_amd.memory_hip import decay_attention, norm_rotary, rotary_table
    gen = torch.Generator().manual_seed(12)
    q, k, v = (draw(gen, 6, 2, 16).requires_grad_() for _ in range(3))
    w = torch.ones(16, device="cuda", requires_grad=True)
    g, starts = decays(2), torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    at, table = torch.arange(6, dtype=torch.int32, device="cuda"), rotary_table(8, 16, device="cuda")

    def attend():
        return decay_attention(q, k, v, g, None, starts)[0]

    def turn():
        return norm_rotary(q[None], k[None], w, w, table, at)[0]
    for f in (attend, turn):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(f().sum(), q, create_graph=True)
    for f, changed in ((attend, g), (attend, starts), (turn, at), (turn, table)):
        out = f().sum()
        changed.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.backward()


def test_what_gets_no_gradient_is_refused(gpu_lib):
    """Tables, decays and a step's states that ask for one; where gradients are off, a table that would ask is taken."""
    from flyguy_amd.memory_hip import decay_attention, decay_step, norm_rotary, rotary, rotary_table
    q, w, s, g = torch.zeros(1, 6, 2, 16, device="cuda"), torch.ones(16, device="cuda"), torch.zeros(1, 2, 16, 16, device="cuda"), decays(2)
    table = rotary_table(8, 16, device="cuda").requires_grad_()
    for f in (lambda: rotary(q, q, table), lambda: norm_rotary(q, q, w, w, table)):
        with pytest.raises(ValueError, match="table is fixed"):
            f()
        with torch.no_grad():
            f()
    with pytest.raises(ValueError, match="decays are fixed"):
        decay_attention(q, q, q, g.clone().requires_grad_())
    with pytest.raises(ValueError, match="no gradients"):
        decay_step(q[:, 0], q[:, 0], q[:, 0], g, s, into=torch.zeros_like(s).requires_grad_())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        rotary(forward_ad.make_dual(q, q), None, table.detach())


def test_a_state_that_a_step_has_changed_is_found_out(gpu_lib):
    """A step's write counts as a change in place; in inference mode it is done all the same."""
    from flyguy_amd.memory_hip import decay_attention, decay_step
    gen = torch.Generator().manual_seed(13)
    q, k, v = (draw(gen, 1, 3, 2, 16).requires_grad_() for _ in range(3))
    s = draw(gen, 1, 2, 16, 16)
    o, _ = decay_attention(q, k, v, decays(2), s)
    with torch.no_grad():
        decay_step(q[:, 0], k[:, 0], v[:, 0], decays(2), s)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()
    with torch.inference_mode():
        t = torch.zeros(1, 2, 16, 16, device="cuda")
        decay_step(q[:, 0], k[:, 0], v[:, 0], decays(2), t)
        assert (t != 0).any()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_decay_that_is_not_a_number(gpu_lib, dt):
    """Its head's outputs and states are not numbers either; the other head's stay as they are."""
    from flyguy_amd.memory_hip import decay_attention, decay_step
    gen = torch.Generator().manual_seed(14)
    q, k, v = (draw(gen, 1, 70, 2, 32, dtype=dt) for _ in range(3))
    s = draw(gen, 1, 2, 32, 32)
    clean, bad = (torch.tensor([-0.1, x], device="cuda") for x in (-0.2, math.nan))
    for f in (lambda g: decay_attention(q, k, v, g, s),
              lambda g: (decay_step(q[:, 0], k[:, 0], v[:, 0], g, s, into=(n := torch.empty_like(s))), n)):
        (o, e), (ob, eb) = f(clean), f(bad)
        assert torch.equal(o[..., 0, :], ob[..., 0, :]) and torch.equal(e[:, 0], eb[:, 0])
        assert ob[..., 1, :].isnan().all() and eb[:, 1].isnan().all()


def test_a_decay_that_is_not_a_number_and_an_empty_state(gpu_lib):
    from flyguy_amd.memory_hip import decay_attention, decay_step
    gen = torch.Generator().manual_seed(25)
    q, k, v = (draw(gen, 1, 3000, 2, 16) for _ in range(3))
    g, s = torch.tensor([-0.1, math.nan], device="cuda"), torch.zeros(1, 2, 16, 16, device="cuda")
    decay_step(q[:, 0], k[:, 0], v[:, 0], g, s)
    for e in (s, decay_attention(q, k, v, g)[1], decay_attention(q, k, v, g, torch.zeros_like(s))[1]):
        assert e[:, 1].isnan().all() and e[:, 0].isfinite().all()


def test_pieces_of_a_stretch_and_single_moments(gpu_lib):
    """A stretch read in two pieces, or moment by moment with decay_step, is the stretch read at once, up to rounding."""
    from flyguy_amd.memory_hip import decay_attention, decay_step
    gen = torch.Generator().manual_seed(11)
    for dt in (F32, BF16):
        q, k, v, s = inputs(gen, 3, 150, 4, 2, 64, 32, dt, "packed", True)
        g = decays(4)
        o, e = decay_attention(q, k, v, g, s)
        f = [x.cpu().double() for x in (q, k, v)]
        want = ref.attention(*f, g.cpu(), s.cpu().double(), 0.125)
        mag = ref.attention(*[x.abs() for x in f], g.cpu(), s.abs().cpu().double(), 0.125)
        o1, e1 = decay_attention(q[:, :37], k[:, :37], v[:, :37], g, s)
        o2, e2 = decay_attention(q[:, 37:], k[:, 37:], v[:, 37:], g, e1)
        live, outs = s.clone(), []
        for t in range(150):
            outs.append(decay_step(q[:, t], k[:, t], v[:, t], g, live))
        extra = 2.0 ** -16 if dt == BF16 else 0.0
        for a, b in ((o, e), (torch.cat([o1, o2], 1), e2), (torch.stack(outs, 1), live)):
            ref.within(a, want[0], mag[0], 64 + 32 + 150 + 200, "o", extra)
            ref.within(b, want[1], mag[1], 64 + 32 + 150 + 200, "state", extra)


def test_long_stretches_keep_their_precision(gpu_lib):
    """20,000 moments of heads that hardly forget: the end state within a few roundings of its own size, as its moments'
    random signs add (errors of 20,000 roundings in one direction, as a rounded decay taken 300 times gives, would show)."""
    from flyguy_amd.memory_hip import decay_attention
    gen = torch.Generator().manual_seed(12)
    g = torch.tensor([-1e-5, -3e-4], device="cuda")
    for dt in (F32, BF16):
        q, k, v, _ = inputs(gen, 1, 20000, 2, 2, 16, 16, dt, "dense", False)
        _, e = decay_attention(q, k, v, g)
        f = [x.cpu().double() for x in (k, v)]
        w = torch.exp(g.cpu().double()[:, None] * torch.arange(19999, -1, -1, dtype=torch.float64))
        want = torch.einsum("ht,thk,thv->hkv", w, f[0][0], f[1][0])
        assert float((e[0].cpu().double() - want).norm() / want.norm()) <= 1e-6


def test_far_strides(gpu_lib):
    """Heads and moments more than 2^31 values apart (views of one 6 GB buffer)."""
    from flyguy_amd.memory_hip import decay_attention, rotary, rotary_table
    gen = torch.Generator().manual_seed(13)
    big = torch.empty(3 * 2 ** 30 + 65536, dtype=BF16, device="cuda")
    far = big.as_strided((1, 2, 2, 64), (0, 2 ** 30, 2 ** 31, 1))
    x = draw(gen, 1, 2, 2, 64, dtype=BF16)
    far.copy_(x)
    table = rotary_table(2, 64).cuda()
    assert torch.equal(rotary(far, None, table)[0], rotary(x, None, table)[0])
    g = decays(2)
    a, b = decay_attention(far, far, far, g), decay_attention(x, x, x, g)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------ single moments
@pytest.mark.parametrize("n,Hq,Hk,K,V,dt", [(1, 1, 1, 1, 1, F32), (1, 8, 8, 64, 64, F32), (3, 4, 2, 128, 128, BF16),
                                            (5, 6, 2, 40, 56, F16), (2, 3, 3, 7, 33, BF16), (70, 2, 1, 96, 20, BF16),
                                            (2, 2, 2, 128, 6, F32)])
def test_step(gpu_lib, n, Hq, Hk, K, V, dt):
    from flyguy_amd.memory_hip import decay_step
    say(f"step {n} {Hq} {Hk} {K} {V} {dt}")
    gen = torch.Generator().manual_seed(n + K)
    wide = draw(gen, n, Hq * K + Hk * (K + V) + 5, dtype=dt)
    q = wide[:, :Hq * K].unflatten(1, (Hq, K))
    k, v = wide[:, Hq * K:Hq * K + Hk * K].unflatten(1, (Hk, K)), wide[:, -Hk * V:].unflatten(1, (Hk, V))
    s = draw(gen, n, Hq, K, V)
    g = decays(Hq)
    f = [x.cpu().double()[:, None] for x in (q, k, v)]
    want = ref.attention(*f, g.cpu(), s.cpu().double(), K ** -0.5)
    mag = ref.attention(*[x.abs() for x in f], g.cpu(), s.abs().cpu().double(), K ** -0.5)
    into = torch.full_like(s, 7.0)
    o1 = decay_step(q, k, v, g, s, into=into)
    kept = s.clone()
    o2 = decay_step(q, k, v, g, s)
    assert torch.equal(o1, o2) and torch.equal(into, s) and not torch.equal(kept, s)
    ref.within(o1[:, None], want[0], mag[0], K + 10, "o")
    ref.within(s, want[1], mag[1], 10, "state")


def test_slots(gpu_lib):
    """Rows go on from their slots' states, idle rows touch none, a slot past the states gives NaN and touches none."""
    from flyguy_amd.memory_hip import decay_step
    gen = torch.Generator().manual_seed(15)
    q, k, v = draw(gen, 5, 2, 32), draw(gen, 5, 2, 32), draw(gen, 5, 2, 48)
    s, g = draw(gen, 7, 2, 32, 48), decays(2)
    slots = torch.tensor([6, -1, 0, 7, 3], dtype=torch.int32, device="cuda")
    was = s.clone()
    o = decay_step(q, k, v, g, s, slots)
    for row, slot in ((0, 6), (2, 0), (4, 3)):
        one = was[slot:slot + 1].clone()
        assert torch.equal(decay_step(q[row:row + 1], k[row:row + 1], v[row:row + 1], g, one)[0], o[row])
        assert torch.equal(one[0], s[slot])
    assert (o[1] == 0).all() and torch.isnan(o[3]).all()
    for slot in (1, 2, 4, 5):
        assert torch.equal(s[slot], was[slot])


# ------------------------------------------------------------------------------------------------ streams, graphs
def test_other_streams(gpu_lib):
    """Calls go to the current stream, and their gradients to it too."""
    from flyguy_amd.memory_hip import decay_attention, decay_step, norm_rotary, rotary_table
    gen = torch.Generator().manual_seed(16)
    q, k, v, s = inputs(gen, 2, 500, 4, 2, 64, 64, BF16, "packed", True)
    w, table, g = torch.ones(64, device="cuda"), rotary_table(500, 64).cuda(), decays(4)
    go = draw(gen, 2, 500, 4, 64, dtype=BF16)

    def all_of_it():
        x = [y.detach().requires_grad_() for y in (q, k, v)]
        a, b = norm_rotary(x[0], x[1], w, w, table)
        o, e = decay_attention(a, b, x[2], g, s)
        return (o.detach(), e.detach(), *torch.autograd.grad(o, x, go), decay_step(q[:, 0], k[:, 0], v[:, 0], g, s.clone()))
    want = all_of_it()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        burn = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            burn = burn @ burn * 1e-3             # (the stream is busy: work on another would overtake it)
        got = all_of_it()
    torch.cuda.current_stream().wait_stream(other)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_in_a_graph(gpu_lib):
    """A decision's calls recorded once and replayed, with eager work between the replays, give the eager results."""
    from flyguy_amd.memory_hip import decay_attention, decay_step, norm_rotary, rotary_table
    gen = torch.Generator().manual_seed(17)
    w, table, g = torch.ones(64, device="cuda"), rotary_table(64, 64).cuda(), decays(4)
    q, k, v = draw(gen, 3, 1, 4, 64), draw(gen, 3, 1, 2, 64), draw(gen, 3, 1, 2, 64)
    long = [draw(gen, 1, 700, 2, 32, dtype=BF16) for _ in range(3)]
    pos = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    s = draw(gen, 3, 4, 64, 64)
    start = s.clone()

    def decide(s):
        a, b = norm_rotary(q, k, w, w, table, pos)
        return decay_step(a[:, 0], b[:, 0], v[:, 0], g, s), decay_attention(*long, g[:2])[0]
    decide(s)                                     # (the first calls load the kernels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decide(s)
    s.copy_(start)
    eager = start.clone()
    for i in range(5):
        pos.fill_(i)
        q.normal_()
        long[0].normal_()
        graph.replay()
        want = decide(eager)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(s, eager)


# ------------------------------------------------------------------------------------------------ the actor that remembers
def test_memory_actor_on_the_gpu(gpu_lib):
    """MemoryActor through the library against its CPU form: logits, state and every gradient, to the bars of the actor's own
    tests (1e-5 and 1e-4 of the largest entry, the latter for what passes float32 norms and sums on both sides); and a
    stretch played moment by moment."""
    import copy

    from conftest import lively, toy
    from flyguy_amd.fly import FlyActor
    from flyguy_amd.memory import MemoryActor
    from gpu_helpers import rel
    torch.manual_seed(3)
    f = lively(FlyActor(toy("b"), 517, 90, hops=3), 3)
    f.kernel = "hip"
    m = MemoryActor(f, heads=4, k_heads=2, dim=24, positions=128)
    with torch.no_grad():
        m.back.weight.normal_(0, 0.3)
    x, R = torch.randn(3, 75, 517), torch.randn(3, 75, 90)
    g = copy.deepcopy(m).cuda()
    out, (mem, seen) = g(x.cuda())
    (out * R.cuda()).sum().backward()
    want, (want_mem, _) = m(x)
    (want * R).sum().backward()
    assert rel(out.detach().cpu(), want.detach()) <= 1e-4 and rel(mem.detach().cpu(), want_mem.detach()) <= 1e-4
    for (name, p), (_, q) in zip(g.named_parameters(), m.named_parameters()):
        assert p.grad is not None and rel(p.grad.cpu(), q.grad) <= 1e-4, name
    live = g.state(3)
    played = torch.stack([g.step(x[:, t].cuda(), live) for t in range(75)], 1)
    assert rel(played.cpu(), out.detach().cpu()) <= 1e-4 and live[1].tolist() == [75] * 3


def test_an_actor_past_its_table(gpu_lib):
    """Cars that play on past the table: the CPU form's logits and memory (to the bars above), by moments and by stretches."""
    import copy

    from conftest import lively, toy
    from flyguy_amd.fly import FlyActor
    from flyguy_amd.memory import MemoryActor
    from gpu_helpers import rel
    torch.manual_seed(4)
    f = lively(FlyActor(toy("a"), 517, 90, hops=3), 4)
    f.kernel = "hip"
    m = MemoryActor(f, heads=4, k_heads=2, dim=24, positions=10)
    with torch.no_grad():
        m.back.weight.normal_(0, 0.3)
        x, g = torch.randn(3, 25, 517), copy.deepcopy(m).cuda()
        live, cpu = g.state(3), m.state(3)
        played = torch.stack([g.step(x[:, t].cuda(), live) for t in range(25)], 1)
        want = torch.stack([m.step(x[:, t], cpu) for t in range(25)], 1)
        a, st = g(x[:, :7].cuda())
        b, (mem, _) = g(x[:, 7:].cuda(), st)
    assert rel(played.cpu(), want) <= 1e-4 and rel(live[0].cpu(), cpu[0]) <= 1e-4
    assert rel(torch.cat([a, b], 1).cpu(), want) <= 1e-4 and rel(mem.cpu(), cpu[0]) <= 1e-4


def test_the_teaching_command_on_the_gpu(gpu_lib, tmp_path, capsys):
    import numpy as np

    from conftest import GOLDEN
    from flyguy_amd.remember import main
    from oracle import trainer as ot
    rng = np.random.default_rng(4)
    ot.write_chunk(tmp_path / "game.bin", rng.standard_normal((300, 517)).astype(np.float16),
                   (3 * rng.standard_normal((300, 90))).astype(np.float16))
    assert main(["--data", str(tmp_path / "game.bin"), "--graph", str(GOLDEN / "toy_a.npz"), "--stretch", "100", "--cars", "8",
                 "--steps", "20", "--out", str(tmp_path / "m.pt")]) == 0
    assert "first choice the same in" in capsys.readouterr().out
