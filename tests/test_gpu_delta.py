"""The gated delta rule (flyguy_amd.memory_hip: delta_attention, delta_step) against a 64-bit restatement."""
from __future__ import annotations

import math

import pytest
import torch

import delta_helpers as ref
from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("q", "k", "v", "log_decay", "beta", "state")


def draw(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def laid_out(x, how):
    """The same values [.., H, D]: dense, in a wider projection (16-byte rows kept or not), or the values first."""
    if how == "dense":
        return x
    if how == "values first":
        return x.movedim(-1, 0).contiguous().movedim(0, -1)
    H, D = x.shape[-2:]
    pad = 8 if how == "packed" else 3
    wide = torch.full((*x.shape[:-2], H * D + 2 * pad), math.nan, dtype=x.dtype, device=x.device)
    part = wide[..., pad:pad + H * D].unflatten(-1, (H, D))
    part.copy_(x)
    return part


def inputs(gen, shape, H, Hk, K, V, dt, how="dense", state=None):
    """Queries, keys of length 1 (alike from moment to moment), values, decays and rates of moments [*shape], and states."""
    k = draw(gen, Hk, K) + draw(gen, *shape, Hk, K)
    k = (0.99 * k / k.square().sum(-1, keepdim=True).sqrt()).to(dt)
    q, v = draw(gen, *shape, H, K, dtype=dt), draw(gen, *shape, Hk, V, dtype=dt)
    g = -torch.rand(*shape, H, generator=gen).cuda() * torch.logspace(-3, 0, H).cuda()
    b = torch.rand(*shape, H, generator=gen).cuda()
    if how != "dense":                                      # (gates of another order too)
        g, b = g.movedim(-1, 0).contiguous().movedim(0, -1), torch.stack([b, b], -1)[..., 0]
    return [laid_out(x, how) for x in (q, k, v)] + [g, b] + [draw(gen, state, H, K, V) if state else None]


def check(ins, starts, dt, scale=None, grad=True, gen=None, end=True):
    """delta_attention and its gradients of these inputs against the restatement."""
    from flyguy_amd.memory_hip import delta_attention
    leaves = [None if x is None else x.detach().requires_grad_(grad) for x in ins]
    q, v = ins[0], ins[2]
    K, V, T = q.shape[-1], v.shape[-1], q.shape[0 if starts is not None else 1]
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    o, e = delta_attention(*leaves, st, scale=scale)
    assert o.dtype == dt and e.dtype == F32 and o.is_contiguous()
    go, ge = draw(gen, *o.shape, dtype=dt), draw(gen, *e.shape)
    f = [None if x is None else x.detach().cpu().double() for x in ins]
    c = K ** -0.5 if scale is None else scale
    want = ref.delta(*f, c, starts, *((go.cpu().double(), ge.cpu().double() if end else None) if grad else ()))
    near = lambda got, w, what: ref.near(got, w, K, V, T, dt, what)       # noqa: E731
    near(o, want[0], "o")
    near(e, want[1], "end state")
    if not grad:
        return
    named = [(n, x) for n, x in zip(NAMES, leaves) if x is not None]
    grads = torch.autograd.grad([o, e] if end else o, [x for _, x in named], [go, ge] if end else go)
    for (n, x), got in zip(named, grads):
        assert got.dtype == x.dtype
        near(got, want[2 + NAMES.index(n)], "gradient of " + n)


CASES = [  # N, T, H, Hk, K, V, type, layout, a start state
    (1, 1, 1, 1, 1, 1, F32, "dense", True),
    (2, 1, 2, 1, 8, 8, BF16, "dense", True),
    (2, 5, 3, 3, 16, 24, F32, "packed", True),
    (1, 16, 2, 2, 64, 64, BF16, "dense", False),
    (1, 17, 2, 2, 64, 64, F16, "packed", True),
    (3, 33, 4, 2, 64, 64, F32, "dense", True),
    (2, 63, 2, 1, 32, 128, BF16, "packed", True),
    (2, 64, 2, 2, 128, 64, BF16, "dense", True),
    (2, 65, 2, 2, 128, 128, BF16, "packed", True),
    (1, 65, 2, 2, 128, 128, F32, "dense", True),
    (2, 100, 6, 2, 40, 56, F16, "packed", True),
    (1, 130, 3, 1, 100, 70, F32, "odd", True),
    (2, 130, 3, 1, 33, 7, BF16, "odd", True),
    (1, 200, 2, 1, 128, 128, F16, "values first", True),
    (1, 257, 4, 4, 72, 96, BF16, "dense", False),
    (1, 257, 4, 4, 65, 65, F32, "dense", False),
    (5, 70, 1, 1, 16, 128, F32, "packed", False),
    (1, 700, 2, 2, 64, 128, BF16, "dense", True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_delta_attention_and_its_gradients(gpu_lib, case):
    N, T, H, Hk, K, V, dt, how, start = case
    say(f"delta {case}")
    gen = torch.Generator().manual_seed(N + T + K + V)
    check(inputs(gen, (N, T), H, Hk, K, V, dt, how, N if start else None), None, dt, gen=gen)


LONG = [  # few chains of many chunks: walked in segments
    (1, 2100, 2, 1, 64, 64, F32, "dense", True),
    (1, 3001, 2, 2, 128, 128, BF16, "packed", True),
    (2, 1500, 3, 1, 40, 56, F16, "dense", True),
    (1, 2500, 1, 1, 128, 64, F32, "dense", False),
    (1, 2300, 1, 1, 64, 128, BF16, "dense", True),
    (1, 1800, 2, 2, 100, 36, F16, "packed", True),
    (3, 1024, 1, 1, 16, 16, BF16, "dense", False),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_long_stretches_of_few_heads(gpu_lib, case):
    N, T, H, Hk, K, V, dt, how, start = case
    say(f"long {case}")
    gen = torch.Generator().manual_seed(N + T + K + V)
    check(inputs(gen, (N, T), H, Hk, K, V, dt, how, N if start else None), None, dt, gen=gen)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_long_packed_stretches(gpu_lib, dt):
    say(f"long packed {dt}")
    gen = torch.Generator().manual_seed(31)
    starts = [5]
    for x in [1900, 0, 700, 3, 2500, 64, 130]:
        starts.append(starts[-1] + x)
    check(inputs(gen, (starts[-1] + 7,), 2, 1, 48, 80, dt, "packed", 7), starts, dt, gen=gen)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("where", [0, 700, 2599])
def test_odd_moments_in_segments(gpu_lib, dt, where):
    """What is not finite reaches the same in a stretch that is walked in segments."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"odd in segments {dt} {where}")
    gen = torch.Generator().manual_seed(32)
    ins = inputs(gen, (1, 2600), 2, 2, 48, 40, dt, "dense", 1)
    want_o, want_e = delta_attention(*ins)
    for what in (1, 2, 4):
        given = [x.clone() for x in ins]
        given[what][(0, where, 1) + ((7,) if what < 3 else ())] = math.nan
        o, e = delta_attention(*given)
        columns = slice(7, 8) if what == 2 else slice(None)
        t, te = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(e, dtype=torch.bool)
        t[0, where:, 1, columns], te[0, 1, :, columns] = True, True
        assert torch.equal(o[~t], want_o[~t]) and torch.equal(e[~te], want_e[~te]), what
        assert torch.isnan(o[t]).all() and torch.isnan(e[te]).all(), what


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("lengths", [[1], [7, 64, 65, 1], [0, 130, 0, 3, 64, 0], [200, 1, 1, 90, 33, 31]])
def test_packed_stretches(gpu_lib, dt, lengths):
    say(f"packed {dt} {lengths}")
    gen = torch.Generator().manual_seed(sum(lengths))
    starts = [0]
    for x in lengths:
        starts.append(starts[-1] + x)
    check(inputs(gen, (starts[-1],), 4, 2, 48, 80, dt, "packed", len(lengths)), starts, dt, gen=gen)


@pytest.mark.parametrize("dt,V,Hk", [(BF16, 24, 4), (F32, 7, 2), (F16, 5, 4), (BF16, 3, 2)])
def test_a_pack_with_room_before_and_behind(gpu_lib, dt, V, Hk):
    """Moments of no stretch: zeros, and gradients of zero, whatever the memory held; starts of 64 bits too."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"room {dt} {V} {Hk}")
    gen = torch.Generator().manual_seed(V)
    M, starts = 300, [20, 90, 90, 221]
    ins = inputs(gen, (M,), 4, Hk, 24, V, dt, "dense", 3)
    junk = torch.full((1 << 22,), math.nan, device="cuda")
    del junk
    check(ins, starts, dt, gen=gen)
    leaves = [x.detach().requires_grad_() for x in ins]
    for wide in (torch.int32, torch.int64):
        o, e = delta_attention(*leaves, torch.tensor(starts, dtype=wide, device="cuda"))
        grads = torch.autograd.grad((o, e), leaves, (torch.ones_like(o), torch.ones_like(e)))
        for x in (o, *grads[:5]):
            assert (x[:20] == 0).all() and (x[221:] == 0).all()


def test_starts_out_of_order_or_out_of_range(gpu_lib):
    """Stretches then share no moment, and nothing outside is read: every moment's output is its own stretch's or zero."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(2)
    for starts in ([0, 90, 40, 150], [-50, 70, 1000], [150, 0], [10, 10, 5, 5, 149]):
        say(f"starts {starts}")
        ins = inputs(gen, (150,), 2, 2, 16, 16, F32, "dense", len(starts) - 1)
        leaves = [x.detach().requires_grad_() for x in ins]
        o, e = delta_attention(*leaves, torch.tensor(starts, device="cuda"))
        grads = torch.autograd.grad((o, e), leaves, (torch.ones_like(o), torch.ones_like(e)))
        for x in (o, e, *grads):
            assert torch.isfinite(x).all()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("packed", [False, True])
def test_no_moments(gpu_lib, dt, packed):
    """The state passes as it is, infinities too, and so does its gradient; no stretches give nothing."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(4)
    s, ge = draw(gen, 3, 2, 16, 24), draw(gen, 3, 2, 16, 24)
    for x in (s, ge):
        x[:, :, 3, 5], x[:, :, 0, 1] = math.inf, math.nan
    s.requires_grad_()
    shape, st = ((0,), torch.zeros(4, dtype=torch.int32, device="cuda")) if packed else ((3, 0), None)
    q, k, v = (torch.empty(*shape, 2, d, dtype=dt, device="cuda") for d in (16, 16, 24))
    gates = torch.empty(*shape, 2, device="cuda")
    o, e = delta_attention(q, k, v, gates, gates, s, st)
    assert o.shape == (*shape, 2, 24) and torch.equal(e.view(torch.int32), s.view(torch.int32))
    assert torch.equal(torch.autograd.grad(e, s, ge)[0].view(torch.int32), ge.view(torch.int32))
    if not packed:
        o, e = delta_attention(q[:0], k[:0], v[:0], gates[:0], gates[:0])
        assert o.shape == (0, 0, 2, 24) and e.shape == (0, 2, 16, 24)
    else:
        z = torch.ones(5, 2, 16, dtype=dt, device="cuda", requires_grad=True)
        g = torch.ones(5, 2, device="cuda", requires_grad=True)
        o, e = delta_attention(z, z, z, g, g, None, torch.zeros(1, dtype=torch.int32, device="cuda"))
        assert (o == 0).all() and e.shape == (0, 2, 16, 16)
        for x in torch.autograd.grad(o, (z, g), torch.ones_like(o)):
            assert (x == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_parts_of_the_gradient(gpu_lib, dt):
    """Each gradient alone, or of one output alone, is what it is among all."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(6)
    ins = inputs(gen, (2, 70), 4, 2, 32, 40, dt, "dense", 2)
    go, ge = draw(gen, 2, 70, 4, 40, dtype=dt), draw(gen, 2, 4, 32, 40)
    leaves = [x.detach().requires_grad_() for x in ins]
    want = torch.autograd.grad(delta_attention(*leaves), leaves, (go, ge))
    for i in range(6):
        one = [x.detach().requires_grad_(j == i) for j, x in enumerate(ins)]
        assert torch.equal(torch.autograd.grad(delta_attention(*one), one[i], (go, ge))[0], want[i]), NAMES[i]
    check(ins, None, dt, gen=gen, end=False)
    leaves = [x.detach().requires_grad_() for x in ins]
    o, e = delta_attention(*leaves)
    for a, b in zip(torch.autograd.grad(e, leaves, ge, retain_graph=True),
                    torch.autograd.grad((o, e), leaves, (torch.zeros_like(go), ge))):
        assert torch.equal(a, b)
    delta_attention(*leaves)[0].sum().backward()            # (a gradient of one number for all)


def test_broadcast_inputs(gpu_lib):
    """Keys, values and gates expanded over stretches, heads or moments: strides of 0, gradients summed by autograd."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(7)
    q, k, v, g, b, s = inputs(gen, (1, 1), 4, 4, 16, 16, F32, "dense", 3)
    small = [q, k, v, g, b]
    wide = [x.expand(3, 70, *x.shape[2:]) for x in small]
    check([*wide, s], None, F32, gen=gen)
    leaves = [x.detach().requires_grad_() for x in small]
    o, _ = delta_attention(*[x.expand(3, 70, *x.shape[2:]) for x in leaves], s)
    full = [x.contiguous().detach().requires_grad_() for x in wide]
    p, _ = delta_attention(*full, s)
    assert torch.equal(o, p)
    for a, c in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), torch.autograd.grad(p, full, torch.ones_like(o))):
        torch.testing.assert_close(a, c.sum((0, 1), keepdim=True), rtol=1e-5, atol=1e-4)


def test_gradients_against_differences(gpu_lib):
    """The loss <go, o> + <ge, e> along a direction d: (L(x + h d) - L(x - h d)) / 2h is <gradient, d> up to h^2 / 6 of the third
    derivative (some hundred moments' terms of order 1, h = 1e-2: 1e-5 of them) and u of L's terms / h (6e-6 of them)."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(8)
    ins = inputs(gen, (1, 70), 2, 1, 16, 16, F32, "dense", 1)
    ds = [draw(gen, *x.shape) for x in ins]
    ds[1], ds[3] = 0.1 * ds[1], 0.1 * ds[3]
    leaves = [x.detach().requires_grad_() for x in ins]
    out = delta_attention(*leaves)
    gs = [draw(gen, *x.shape) for x in out]
    grads = torch.autograd.grad(out, leaves, gs)
    for i, name in enumerate(NAMES):
        def loss(h):
            out = delta_attention(*[x + h * ds[j] if j == i else x for j, x in enumerate(ins)])
            return sum(float((x.double() * y.double()).sum()) for x, y in zip(out, gs))
        got = float((grads[i].double() * ds[i].double()).sum())
        assert abs((loss(1e-2) - loss(-1e-2)) / 2e-2 - got) < 0.02 * (10 + abs(got)), name


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_pieces_of_a_stretch_and_single_moments(gpu_lib, dt):
    """A stretch in pieces, its state handed on, and moment by moment in place: as all at once, up to rounding."""
    from flyguy_amd.memory_hip import delta_attention, delta_step
    gen = torch.Generator().manual_seed(9)
    q, k, v, g, b, s = inputs(gen, (2, 150), 4, 2, 64, 48, dt, "dense", 2)
    f = [x.cpu().double() for x in (q, k, v, g, b, s)]
    want = ref.delta(*f, 64 ** -0.5)
    state, outs = s, []
    for a, z in ((0, 1), (1, 70), (70, 134), (134, 150)):
        o, state = delta_attention(*[x[:, a:z] for x in (q, k, v, g, b)], state)
        outs.append(o)
    ref.near(torch.cat(outs, 1), want[0], 64, 48, 150, dt, "pieces")
    ref.near(state, want[1], 64, 48, 150, dt, "pieces' state")
    state = s.clone()
    outs = [delta_step(*[x[:, t] for x in (q, k, v, g, b)], state) for t in range(150)]
    ref.near(torch.stack(outs, 1), want[0], 64, 48, 150, dt, "moments")
    ref.near(state, want[1], 64, 48, 150, F32, "moments' state")


@pytest.mark.parametrize("dt", [F32, BF16])
def test_forgetting_and_not_writing(gpu_lib, dt):
    """-inf forgets what was there, infinities and all the finite; a huge decay too; rates of 0 write nothing; and the sums of
    decays lose nothing by what was forgotten before."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"forget {dt}")
    gen = torch.Generator().manual_seed(10)
    q, k, v, g, b, s = inputs(gen, (1, 140), 2, 2, 32, 32, dt, "dense", 1)
    g[:, 3], g[:, 5], g[:, 70], g[:, 71], g[:, 9:40] = -math.inf, -1e30, -5000.0, -math.inf, -1000.0
    b[:, 50:60] = 0
    b[:, 100:] = 0
    g[:, 100:] = 0
    check([q, k, v, g.clamp_min(-1e4), b, s], None, dt, gen=gen)
    one, two = delta_attention(q, k, v, g, b, s), delta_attention(q, k, v, g.clamp_min(-1e4), b, s)
    for x, y in zip(one, two):
        assert torch.equal(x, y)
    assert torch.equal(one[1], delta_attention(*[x[:, :100] for x in (q, k, v, g, b)], s)[1])
    leaves = [x.detach().requires_grad_() for x in (q, k, v, g, b, s)]
    for x in torch.autograd.grad(delta_attention(*leaves), leaves, [torch.ones_like(x) for x in one]):
        assert torch.isfinite(x).all()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("where", [0, 10, 63, 64, 100])
def test_a_later_moment_does_not_reach_an_earlier_one(gpu_lib, dt, where):
    """A value that is not finite: a query's reaches its own output, a value's its column from its moment on, a key's, decay's or
    rate's everything of its heads from there on; other stretches and heads stay bit for bit."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"odd {dt} {where}")
    gen = torch.Generator().manual_seed(11)
    ins = inputs(gen, (2, 150), 4, 2, 48, 40, dt, "dense", 2)
    want_o, want_e = delta_attention(*ins)
    for what in range(5):
        for odd in (math.nan, math.inf, -math.inf):
            if what == 3 and odd == -math.inf:
                continue
            given = [x.clone() for x in ins]
            heads = slice(1, 2) if what in (0, 3, 4) else slice(2, 4)         # (key head 1's query heads)
            given[what][(1, where, 1) + ((7,) if what < 3 else ())] = odd
            o, e = delta_attention(*given)
            touched = torch.zeros_like(o, dtype=torch.bool)
            touched_e = torch.zeros_like(e, dtype=torch.bool)
            if what == 0:
                touched[1, where, heads] = True
            elif what == 2:
                touched[1, where:, heads, 7], touched_e[1, heads, :, 7] = True, True
            else:
                touched[1, where:, heads], touched_e[1, heads] = True, True
            assert torch.equal(o[~touched], want_o[~touched]) and torch.equal(e[~touched_e], want_e[~touched_e]), (what, odd)
            assert not torch.isfinite(o[touched]).any() and not torch.isfinite(e[touched_e]).any(), (what, odd)
            leaves = [x.requires_grad_() for x in given]
            grads = torch.autograd.grad(delta_attention(*leaves), leaves, (torch.ones_like(o), torch.ones_like(e)))
            for i, x in enumerate(grads):                                     # (no other stretch)
                assert torch.isfinite(x[0]).all(), (what, odd, NAMES[i])


def test_a_zero_rate_hides_no_key(gpu_lib):
    """Rates of exactly 0 and 1 have gradients like any other; errors are not divided by them."""
    gen = torch.Generator().manual_seed(12)
    for dt in (F32, BF16):
        ins = inputs(gen, (2, 90), 2, 1, 32, 32, dt, "dense", 2)
        ins[4] = (ins[4] > 0.5).float()
        check(ins, None, dt, gen=gen)


def test_keys_all_alike(gpu_lib):
    """The hardest system a chunk can have: every key the same, rate 1 and no decay, so that each moment replaces the last."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(13)
    for dt in (F32, BF16, F16):
        say(f"alike {dt}")
        q, k, v, g, b, s = inputs(gen, (1, 200), 2, 2, 64, 64, dt, "dense", 1)
        k = torch.zeros_like(k)
        k[..., 5] = 1
        check([q, k, v, torch.zeros_like(g), torch.ones_like(b), s], None, dt, gen=gen)
        e = delta_attention(q, k, v, torch.zeros_like(g), torch.ones_like(b), s)[1]
        torch.testing.assert_close(e[0, :, 5], v[0, -1].float(), rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_long_stretches_keep_their_precision(gpu_lib, dt):
    """20,000 moments that forget next to nothing: against the recurrence in 64 bits on the GPU."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(14)
    T = 20000
    q, k, v, g, b, s = inputs(gen, (1, T), 2, 2, 32, 32, dt, "dense", 1)
    g, b = torch.full_like(g, -1e-6), 0.01 * b
    o, e = delta_attention(q, k, v, g, b, s)
    x, w = s.double()[0], torch.empty(T, 2, 32, dtype=torch.float64, device="cuda")
    qd, kd, vd, gd, bd = (t.double()[0] for t in (q, k, v, g, b))
    for t in range(T):
        x = torch.exp(gd[t])[:, None, None] * x
        u = bd[t][:, None] * (vd[t] - (kd[t][:, :, None] * x).sum(1))
        x = x + kd[t][:, :, None] * u[:, None, :]
        w[t] = 32 ** -0.5 * (qd[t][:, :, None] * x).sum(1)
    ref.near(e, x[None].cpu(), 32, 32, T, F32, "end state")
    ref.near(o, w[None].cpu(), 32, 32, T, dt, "o")


STEPS = [(1, 8, 8, 64, 64, F32), (3, 4, 2, 40, 56, F16), (5, 2, 1, 128, 128, BF16), (2, 3, 3, 7, 5, F32), (1, 1, 1, 1, 1, BF16),
         (70, 2, 2, 33, 100, F32), (70, 8, 4, 64, 64, BF16), (140, 8, 8, 33, 57, F32), (33, 8, 8, 128, 127, F16)]


@pytest.mark.parametrize("n,H,Hk,K,V,dt", STEPS)
def test_step(gpu_lib, n, H, Hk, K, V, dt):
    from flyguy_amd.memory_hip import delta_step
    say(f"step {n} {H} {K} {V} {dt}")
    gen = torch.Generator().manual_seed(n + K)
    for how in ("dense", "odd"):
        q, k, v, g, b, s = inputs(gen, (n,), H, Hk, K, V, dt, how, n)
        want = ref.delta(*[x.cpu().double()[:, None] for x in (q, k, v, g, b)], s.cpu().double(), K ** -0.5)
        into, mine = torch.empty_like(s), s.clone()
        for o in (delta_step(q, k, v, g, b, s, into=into), delta_step(q, k, v, g, b, mine)):
            ref.near(o, want[0][:, 0], K, V, 1, dt, "o")
        ref.near(into, want[1], K, V, 1, F32, "state")
        assert torch.equal(into, mine)


def test_slots(gpu_lib):
    """Rows go on from the slots they name; idle rows give zeros, rows past the states NaN, and neither touches a state."""
    from flyguy_amd.memory_hip import delta_step
    gen = torch.Generator().manual_seed(15)
    q, k, v, g, b, s = inputs(gen, (5,), 2, 2, 24, 16, F32, "dense", 7)
    slots = torch.tensor([6, -1, 0, 99, 3], dtype=torch.int32, device="cuda")
    mine = s.clone()
    o = delta_step(q, k, v, g, b, mine, slots)
    live = [0, 2, 4]
    rows = [slots[i].item() for i in live]
    want, into = s[rows].clone(), None
    w = delta_step(*[x[live] for x in (q, k, v, g, b)], want, into=into)
    assert torch.equal(o[live], w) and torch.equal(mine[rows], want)
    assert (o[1] == 0).all() and torch.isnan(o[3]).all()
    rest = [i for i in range(7) if i not in rows]
    assert torch.equal(mine[rest], s[rest])


def test_refusals(gpu_lib):
    from flyguy_amd.memory_hip import delta_attention, delta_step
    gen = torch.Generator().manual_seed(16)
    ins = inputs(gen, (2, 5), 4, 2, 16, 16, F32, "dense", 2)
    q, k, v, g, b, s = ins
    for i, bad in ((0, q.double()), (1, k[:, :4]), (1, k[..., :8]), (2, v.half()), (3, g[..., :2]), (3, g.double()), (4, b.cpu()),
                   (4, None), (5, s[:1]), (5, s.half()), (1, k[:, :, :0])):
        given = [bad if j == i else x for j, x in enumerate(ins)]
        with pytest.raises(ValueError, match="delta_attention"):
            delta_attention(*given)
        if i == 5 or i == 1 and bad.shape[1] == 4:
            continue
        rows = [x[:, 0] if isinstance(x, torch.Tensor) else x for x in given[:5]]
        with pytest.raises(ValueError, match="delta_step"):
            delta_step(*rows, s)
    with pytest.raises(ValueError, match="starts"):
        delta_attention(*[x[0] for x in ins[:5]], s[:1], torch.zeros(2, device="cuda"))
    wide = torch.zeros(1, 2, 1, 129, device="cuda")
    with pytest.raises(ValueError, match="128"):
        delta_attention(wide, wide, wide, wide[..., 0], wide[..., 0])
    row = [x[:, 0] for x in ins[:5]]
    with pytest.raises(ValueError, match="gradients"):
        delta_step(*row[:3], row[3].clone().requires_grad_(), row[4], s)
    with pytest.raises(ValueError, match="state"):
        delta_step(*row, s.transpose(2, 3))
    leaves = [x.detach().requires_grad_() for x in ins]
    with pytest.raises(RuntimeError, match="has no gradient"):
        torch.autograd.grad(delta_attention(*leaves)[0].sum(), leaves, create_graph=True)
    s2 = s.clone().requires_grad_()
    e = delta_attention(q, k, v, g, b, s2)[1]
    loss = (e * e).sum()
    delta_step(*row, e.detach())                            # (writes over what the loss has kept)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    o, _ = delta_attention(*leaves)
    with torch.no_grad():
        leaves[4].mul_(0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()


def test_another_stream_and_a_graph(gpu_lib):
    """A forward, its gradients and a step captured once and replayed on new inputs, with eager work between."""
    from flyguy_amd.memory_hip import delta_attention, delta_step
    gen = torch.Generator().manual_seed(17)
    ins = inputs(gen, (2, 140), 4, 2, 48, 80, BF16, "dense", 2)
    go = draw(gen, 2, 140, 4, 80, dtype=BF16)

    def work(given):
        leaves = [x.clone().requires_grad_() for x in given]
        o, e = delta_attention(*leaves)
        grads = torch.autograd.grad((o, e), leaves, (go, torch.ones_like(e)))
        s = e.detach().clone()
        row = delta_step(*[x[:, 3] for x in given[:5]], s)
        return (o.detach(), e.detach(), *grads, row, s)

    want = work(ins)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work(ins)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    held = [x.clone() for x in ins]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(held)
    for i in range(3):
        new = inputs(gen, (2, 140), 4, 2, 48, 80, BF16, "dense", 2)
        for h, x in zip(held, new):
            h.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(work(new), outs):
            assert torch.equal(a, b), i


def test_a_gradient_taken_twice(gpu_lib):
    """What the forward leaves for its gradient stays as it was: a second pass gives the same numbers."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(41)
    for dt, shape in ((BF16, (2, 150)), (F32, (1, 2100))):
        leaves = [x.detach().requires_grad_() for x in inputs(gen, shape, 2, 1, 64, 64, dt, "dense", shape[0])]
        outs = delta_attention(*leaves)
        given = [torch.randn_like(x) for x in outs]
        first = torch.autograd.grad(outs, leaves, given, retain_graph=True)
        for a, b in zip(first, torch.autograd.grad(outs, leaves, given)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_states_that_grow(gpu_lib, dt):
    """Log decays from 0 to 1: what an early moment leaves is 1e17 times larger in the end.  What a moment is off by grows as what
    it leaves does, so that against the largest number the bound of decaying states holds."""
    gen = torch.Generator().manual_seed(44)
    ins = inputs(gen, (2, 40), 2, 1, 64, 64, dt, "dense", 2)
    ins[3] = 1 - torch.rand(2, 40, 2, generator=gen).cuda() * 0.1
    check(ins, None, dt, gen=gen)


def test_two_at_once_and_two_graphs(gpu_lib):
    """Calls of the same sizes on two streams at the same time, and two graphs of them replayed in turn and side by side, each
    with its own inputs, give what they give alone."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(42)
    both = [inputs(gen, (1, 2100), 2, 1, 64, 64, BF16, "dense", 1) for _ in range(2)]
    go = draw(gen, 1, 2100, 2, 64, dtype=BF16)

    def work(given):
        leaves = [x.detach().requires_grad_() for x in given]
        o, e = delta_attention(*leaves)
        return (o.detach(), e.detach(), *torch.autograd.grad((o, e), leaves, (go, torch.ones_like(e))))

    want = [work(x) for x in both]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for i in range(3):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[n].append(work(both[n]))
    torch.cuda.synchronize()
    for n in range(2):
        for run in got[n]:
            for a, b in zip(want[n], run):
                assert torch.equal(a, b), n
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for n, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            outs.append(work(both[n]))
    for i in range(4):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st if i >= 2 else streams[0]):
                graphs[n].replay()
        torch.cuda.synchronize()
        for n in range(2):
            for a, b in zip(want[n], outs[n]):
                assert torch.equal(a, b), (i, n)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_tensors_at_odd_places(gpu_lib, dt):
    """States and values that begin inside other memory, at no multiple of 16 bytes, and one tensor given as two of the three."""
    from flyguy_amd.memory_hip import delta_attention, delta_step
    gen = torch.Generator().manual_seed(43)

    def moved(x):
        room = torch.full((x.numel() + 3,), math.nan, dtype=x.dtype, device="cuda")
        return room[3:].view(x.shape).copy_(x)

    q, k, v, g, b, s = inputs(gen, (2, 70), 2, 2, 64, 64, dt, "dense", 2)
    for x, y in zip(delta_attention(q, k, v, g, b, s), delta_attention(*map(moved, (q, k, v, g, b, s)))):
        assert torch.equal(x, y)
    for x, y in zip(delta_attention(k, k, k, g, b, s), delta_attention(k, k.clone(), moved(k), g, b, s)):
        assert torch.equal(x, y)
    one = [x[:, 0] for x in (q, k, v, g, b)]
    there, odd = s.clone(), moved(s)
    o, p = delta_step(*one, there), delta_step(*map(moved, one), odd)
    assert torch.equal(o, p) and torch.equal(there, odd)
    into = moved(torch.zeros_like(s))
    assert torch.equal(delta_step(*one, s, into=into), o) and torch.equal(into, there)


def test_far_strides(gpu_lib):
    """Moments more than 2^31 bytes apart."""
    from flyguy_amd.memory_hip import delta_attention
    gen = torch.Generator().manual_seed(18)
    q, k, v, g, b, s = inputs(gen, (1, 3), 1, 1, 16, 16, BF16, "dense", 1)
    far = torch.empty(3 * (1 << 30), dtype=BF16, device="cuda")
    view = far.as_strided((1, 3, 1, 16), (0, 1 << 30, 16, 1))
    view.copy_(k)
    for x, y in zip(delta_attention(q, view, v, g, b, s), delta_attention(q, k, v, g, b, s)):
        assert torch.equal(x, y)


def test_more_than_2_31_values(gpu_lib):
    """Two stretches of 1.1e9 values: the one that lies beyond 2^31 bytes, and partly values, gives what it gives as the first."""
    from flyguy_amd.memory_hip import delta_attention
    T, H = 140000, 64
    torch.manual_seed(45)
    q = torch.randn(2, T, H, 128, dtype=BF16, device="cuda")
    k, v = (torch.randn(2, T, 1, 128, dtype=BF16, device="cuda") * 0.08 for _ in range(2))
    g, b = -torch.rand(2, T, H, device="cuda"), torch.rand(2, T, H, device="cuda")
    o, e = delta_attention(q, k, v, g, b)
    turned, end = delta_attention(*(x.flip(0) for x in (q, k, v, g, b)))
    assert torch.isfinite(e).all()
    for n in range(2):
        assert torch.equal(o[n], turned[1 - n]) and torch.equal(e[n], end[1 - n])
        assert float(o[n, -64:].abs().max()) > 0


@pytest.mark.parametrize("kw", [dict(rule="delta", norm=True, dropout=0.25), dict(rule="delta"), dict(norm=True, dropout=0.1)])
def test_memory_actor_on_the_gpu(gpu_lib, kw):
    """The layer norm, the projections, the rotation, the delta rule and the dropout together: MemoryActor against its CPU form,
    the same numbers dropped; logits, state and every gradient to 1e-4 of the largest entry, as its other tests; then played."""
    import copy

    from conftest import lively, toy
    from flyguy_amd.fly import FlyActor
    from flyguy_amd.memory import MemoryActor
    from gpu_helpers import rel
    say(f"actor {kw}")
    torch.manual_seed(3)
    f = lively(FlyActor(toy("b"), 517, 90, hops=3), 3)
    f.kernel = "hip"
    m = MemoryActor(f, heads=4, k_heads=2, dim=24, positions=128, **kw)
    with torch.no_grad():
        m.back.weight.normal_(0, 0.3)
        if m.rule == "delta":
            m.gates.weight.normal_(0, 0.05)
            m.gates.bias.normal_(0, 1)
    x, R = torch.randn(3, 75, 517), torch.randn(3, 75, 90)
    g = copy.deepcopy(m).cuda()
    for _ in range(2):                                      # (the second pass drops others)
        out, (mem, _) = g(x.cuda())
        (out * R.cuda()).sum().backward()
        want, (want_mem, _) = m(x)
        (want * R).sum().backward()
        assert rel(out.detach().cpu(), want.detach()) <= 1e-4 and rel(mem.detach().cpu(), want_mem.detach()) <= 1e-4
    for (name, p), (_, q) in zip(g.named_parameters(), m.named_parameters()):
        assert p.grad is not None and rel(p.grad.cpu(), q.grad) <= 1e-4, name
    g.eval()
    with torch.no_grad():
        want, _ = g(x.cuda())
        live = g.state(3)
        played = torch.stack([g.step(x[:, t].cuda(), live) for t in range(75)], 1)
    assert rel(played.cpu(), want.cpu()) <= 1e-4 and live[1].tolist() == [75] * 3


def test_the_teaching_command_on_the_gpu(gpu_lib, tmp_path, capsys):
    import numpy as np

    from conftest import GOLDEN
    from flyguy_amd.remember import main
    from oracle import trainer as ot
    rng = np.random.default_rng(4)
    ot.write_chunk(tmp_path / "game.bin", rng.standard_normal((300, 517)).astype(np.float16),
                   (3 * rng.standard_normal((300, 90))).astype(np.float16))
    assert main(["--data", str(tmp_path / "game.bin"), "--graph", str(GOLDEN / "toy_a.npz"), "--stretch", "100", "--cars", "8",
                 "--steps", "20", "--rule", "delta", "--norm", "--dropout", "0.1", "--out", str(tmp_path / "m.pt")]) == 0
    assert float(capsys.readouterr().out.split("logits off by ")[1].split()[0]) < 1e-4
