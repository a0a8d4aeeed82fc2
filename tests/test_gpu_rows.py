"""Layer norm and dropout (flyguy_amd.rows_hip) against 64-bit restatements."""
from __future__ import annotations

import math

import pytest
import torch

import memory_helpers as ref
import rows_helpers as rows_ref
from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


def draw(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def laid_out(x, how):
    """x [rows, D] with the same values: dense, rows apart (16 bytes kept or not), or columns first."""
    if how == "dense":
        return x
    if how == "columns first":
        return x.t().contiguous().t()
    pad = 16 if how == "apart" else 3
    wide = torch.full((x.shape[0], x.shape[1] + 2 * pad), math.nan, dtype=x.dtype, device=x.device)
    part = wide[:, pad:pad + x.shape[1]]
    part.copy_(x)
    return part


NORMS = [  # rows, width, type, layout, weight, bias
    (1, 1, F32, "dense", True, True),
    (5, 2, BF16, "dense", True, False),
    (3, 8, F16, "apart", False, False),
    (70, 13, F32, "odd", True, True),
    (33, 64, BF16, "dense", False, True),
    (1001, 96, F32, "dense", True, True),
    (17, 255, F16, "odd", True, True),
    (9, 512, BF16, "apart", True, True),
    (6, 513, F32, "dense", True, False),
    (50, 1000, F32, "apart", True, True),
    (4, 1024, BF16, "columns first", True, True),
    (130, 1332, F32, "dense", True, True),
    (7, 1332, F32, "odd", True, True),
    (5, 2056, F16, "apart", True, True),
    (3, 4096, BF16, "dense", True, False),
    (3, 4096, F32, "odd", True, True),
    (2, 4097, BF16, "dense", True, True),
    (3, 8192, F32, "dense", True, True),
    (2, 8200, F16, "apart", True, True),
    (5, 20001, F32, "dense", True, True),
    (4200, 40, BF16, "dense", True, True),
    (900, 252, BF16, "dense", True, True),
    (9, 1002, F32, "dense", True, True),
    (6, 1332, F16, "dense", True, True),
    (3, 5001, F32, "dense", True, True),
    (4, 5002, F32, "dense", True, False),
    (3, 5002, BF16, "dense", False, True),
    (3, 6004, BF16, "dense", True, True),
    (2100, 4096, BF16, "dense", True, True),
]


@pytest.mark.parametrize("case", NORMS, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_layer_norm_and_its_gradients(gpu_lib, case):
    from flyguy_amd.rows_hip import layer_norm
    n, D, dt, how, has_w, has_b = case
    say(f"layer norm {case}")
    gen = torch.Generator().manual_seed(n + D)
    x = laid_out((draw(gen, n, D) * draw(gen, n, 1) + 2 * draw(gen, n, 1)).to(dt), how).requires_grad_()
    w = (1 + 0.3 * draw(gen, D)).requires_grad_() if has_w else None
    b = (0.3 * draw(gen, D)).requires_grad_() if has_b else None
    g = laid_out(draw(gen, n, D, dtype=dt), how)
    y = layer_norm(x, w, b, eps=EPS)
    assert y.is_contiguous() and y.dtype == dt
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps=EPS), y)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([i for i, t in enumerate((x, w, b)) if t is not None], torch.autograd.grad(y, leaves, g)))
    f = [None if t is None else t.detach().cpu().double() for t in (x, w, b)]
    want = rows_ref.layer_norm(*f, EPS, g.cpu().double())
    A = f[0].abs().mean(1, keepdim=True)
    r = ((f[0] - f[0].mean(1, keepdim=True)).square().mean(1, keepdim=True) + EPS).rsqrt()
    second = float(((D + 2) * ref.U * A * r).square().max())        # a mean that is off by d makes the deviation off by d^2 r^2 / 2
    ref.within(y, *want[0], D + 20, "y", second)
    ref.within(grads[0], *want[1], 3 * D + 60, "gx", 3 * second)
    if has_w:
        ref.within(grads[1], *want[2], n + D + 40, "gweight", second)
    if has_b:
        ref.within(grads[2], *want[3], n + 5, "gbias")


def test_layer_norm_of_more_dimensions_and_parts_of_its_gradient(gpu_lib):
    from flyguy_amd.rows_hip import layer_norm
    gen = torch.Generator().manual_seed(3)
    x, w, b = draw(gen, 4, 6, 40).transpose(0, 1), draw(gen, 40), draw(gen, 40)
    y = layer_norm(x, w, b)
    assert y.shape == x.shape and torch.equal(y, layer_norm(x.reshape(24, 40), w, b).view(6, 4, 40))
    assert torch.equal(layer_norm(x[0, 0], w, b), y[0, 0])
    g = draw(gen, 6, 4, 40)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*full), full, g)
    for i in range(3):
        given = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(layer_norm(*given), given[i], g)[0], want[i])
    one = x.clone().requires_grad_()                       # (a gradient of one number for all)
    layer_norm(one, w, b).sum().backward()
    assert torch.equal(one.grad, torch.autograd.grad(layer_norm(one, w, b), one, torch.ones_like(y))[0])


def test_layer_norm_without_rows(gpu_lib):
    from flyguy_amd.rows_hip import layer_norm
    x, w = torch.empty(0, 24, device="cuda", requires_grad=True), torch.ones(24, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == gx.shape == (0, 24) and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.parametrize("D", [24, 700, 1332, 9000])
def test_layer_norm_keeps_rows_apart(gpu_lib, D):
    """Infinities and NaN stay in their row; a row of one value is all bias."""
    from flyguy_amd.rows_hip import layer_norm
    gen = torch.Generator().manual_seed(D)
    x, w, b, g = draw(gen, 40, D), draw(gen, D), draw(gen, D), draw(gen, 40, D)
    odd = x.clone()
    odd[3, 5], odd[17, D - 1], odd[30] = math.nan, math.inf, 7.0
    outs = []
    for t in (x, odd):
        t.requires_grad_()
        y = layer_norm(t, w, b)
        outs.append((y.detach(), torch.autograd.grad(y, t, g)[0]))
    same = [i for i in range(40) if i not in (3, 17, 30)]
    for a, c in zip(*outs):
        assert torch.equal(a[same], c[same]) and torch.isnan(c[3]).all() and torch.isnan(c[17]).all()
    assert torch.equal(outs[1][0][30], b)


def test_layer_norm_gradient_against_differences(gpu_lib):
    """The loss <g, y> along a direction d of order 1: (L(x + h d) - L(x - h d)) / 2h is <gx, d> up to h^2 / 6 of the third
    derivative (a few times the terms' magnitudes) and u of L's terms / h: 1e-4 and 6e-8 x 320 x 40 / 1e-2 of values of order 10."""
    from flyguy_amd.rows_hip import layer_norm
    gen = torch.Generator().manual_seed(5)
    ts = [draw(gen, 8, 40), draw(gen, 40), draw(gen, 40)]
    ds = [draw(gen, *t.shape) for t in ts]
    g, h = draw(gen, 8, 40), 1e-2
    given = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(layer_norm(*given), given, g)
    for i in range(3):
        def loss(s):
            return float((g.double() * layer_norm(*[t + s * ds[j] if j == i else t for j, t in enumerate(ts)]).double()).sum())
        got = float((grads[i].double() * ds[i].double()).sum())
        assert abs((loss(h) - loss(-h)) / (2 * h) - got) < 0.02 * (1 + abs(got)), i


def test_layer_norm_refuses(gpu_lib):
    from flyguy_amd.rows_hip import layer_norm
    x = torch.zeros(3, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda")
    for bad in (lambda: layer_norm(x.double()), lambda: layer_norm(x, w[:4]), lambda: layer_norm(x, w.half()),
                lambda: layer_norm(x, w, w.cpu()), lambda: layer_norm(x, eps=-1), lambda: layer_norm(x[:, :0]),
                lambda: layer_norm(x.sum())):
        with pytest.raises(ValueError, match="layer_norm"):
            bad()
    with pytest.raises(RuntimeError, match="has no gradient"):
        torch.autograd.grad(layer_norm(x, w).sum(), x, create_graph=True)


DROPS = [  # shape, type, share
    ((1,), F32, 0.5), ((7,), BF16, 0.3), ((8,), F16, 0.9), ((3, 5), F32, 0.1), ((2, 3, 64), BF16, 0.25), ((1001, 13), F32, 0.05),
    ((130, 512), F16, 0.1), ((4, 8192), BF16, 0.5), ((40, 40), F32, 0.0), ((40, 40), BF16, 1.0), ((40, 40), F32, 1e-7),
    ((3, 999), F16, 1 - 2.0 ** -16),
]


@pytest.mark.parametrize("case", DROPS, ids=str)
def test_dropout_and_its_gradient(gpu_lib, case):
    """Bit for bit: one product in float32, rounded once."""
    from flyguy_amd.rows_hip import dropout
    shape, dt, share = case
    say(f"dropout {case}")
    gen = torch.Generator().manual_seed(len(shape))
    x, g = draw(gen, *shape, dtype=dt), draw(gen, *shape, dtype=dt)
    for counter in ((1, 2), (0x123456789ABCDEF, (1 << 40) + 5), (-3, -1)):
        c = torch.tensor(counter, device="cuda")
        t = x.clone().requires_grad_()
        y = dropout(t, share, c)
        assert torch.equal(y.cpu(), rows_ref.dropout(x.cpu(), share, counter))
        assert torch.equal(torch.autograd.grad(y, t, g)[0].cpu(), rows_ref.dropout(g.cpu(), share, counter))
        with torch.no_grad():
            assert torch.equal(dropout(x, share, c), y)


def test_dropout_of_any_strides(gpu_lib):
    """The mask goes by a number's place in the tensor's order, not in memory."""
    from flyguy_amd.rows_hip import dropout
    gen = torch.Generator().manual_seed(8)
    x, c = draw(gen, 50, 40), torch.tensor([5, 6], device="cuda")
    want = rows_ref.dropout(x.cpu(), 0.4, (5, 6))
    for how in ("apart", "odd", "columns first"):
        assert torch.equal(dropout(laid_out(x, how), 0.4, c).cpu(), want), how
    assert torch.equal(dropout(x[:, None].expand(50, 2, 40), 0.4, c).cpu(),
                       rows_ref.dropout(x.cpu()[:, None].expand(50, 2, 40), 0.4, (5, 6)))
    one = x.clone().requires_grad_()
    dropout(one, 0.4, c).sum().backward()                  # (a gradient of one number for all)
    assert torch.equal(one.grad.cpu(), rows_ref.dropout(torch.ones(50, 40), 0.4, (5, 6)))
    assert dropout(x[:0], 0.4, c).shape == (0, 40)


def test_dropped_numbers_are_zero_whatever_they_were(gpu_lib):
    from flyguy_amd.rows_hip import dropout
    x = torch.full((64, 64), math.nan, device="cuda")
    y = dropout(x, 0.5, torch.tensor([1, 1], device="cuda"))
    kept = torch.isnan(y)
    assert 0.4 < float(kept.float().mean()) < 0.6 and (y[~kept] == 0).all()


def test_dropout_draws(gpu_lib):
    """The share dropped is p within 6 standard deviations, and other offsets or seeds give unrelated masks."""
    from flyguy_amd.rows_hip import dropout
    x, n, p = torch.ones(1 << 20, device="cuda"), 1 << 20, 0.3
    masks = [dropout(x, p, torch.tensor(c, device="cuda")) == 0 for c in ((0, 0), (0, 1), (1, 0))]
    for m in masks:
        assert abs(float(m.double().mean()) - p) < 6 * math.sqrt(p * (1 - p) / n)
    for a, b in ((0, 1), (0, 2), (1, 2)):
        q = p * p
        assert abs(float((masks[a] & masks[b]).double().mean()) - q) < 6 * math.sqrt(q * (1 - q) / n)


def test_dropout_refuses(gpu_lib):
    from flyguy_amd.rows_hip import dropout
    x, c = torch.zeros(3, 8, device="cuda", requires_grad=True), torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (lambda: dropout(x, -0.1, c), lambda: dropout(x, 1.1, c), lambda: dropout(x, math.nan, c), lambda: dropout(x, 0.5, c[:1]),
                lambda: dropout(x, 0.5, c.int()), lambda: dropout(x, 0.5, c.cpu()), lambda: dropout(x.double(), 0.5, c),
                lambda: dropout(x, 0.5, 3)):
        with pytest.raises(ValueError, match="dropout"):
            bad()
    with pytest.raises(RuntimeError, match="has no gradient"):
        torch.autograd.grad(dropout(x, 0.5, c).sum(), x, create_graph=True)
    y = dropout(x, 0.5, c)
    c += 1                                                  # another mask by now
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_rows_on_another_stream_and_in_a_graph(gpu_lib):
    """Captured once: every replay has its own mask by the counter that it moves on, and matches the calls one by one."""
    from flyguy_amd.rows_hip import dropout, layer_norm
    gen = torch.Generator().manual_seed(9)
    x, w, b, g = draw(gen, 300, 1332), draw(gen, 1332), draw(gen, 1332), draw(gen, 300, 1332)
    count = torch.tensor([77, 0], device="cuda")

    def work():
        t = [v.clone().requires_grad_() for v in (x, w, b)]
        now = count.clone()
        y = dropout(layer_norm(*t), 0.2, now)
        grads = torch.autograd.grad(y, t, g)
        count[1:] += 1
        return (y.detach(), *grads)

    want = [work() for _ in range(4)]
    count[1:] = 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(want[0], other):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for i in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(want[i], outs):
            assert torch.equal(a, c), i


def test_rows_at_odd_places(gpu_lib):
    """One row for all, every second row, rows and weights at no multiple of 16 bytes, a counter inside other memory."""
    from flyguy_amd.rows_hip import dropout, layer_norm
    gen = torch.Generator().manual_seed(19)
    room = draw(gen, 70, 1333)
    w, b = room[0, 1:257], room[1, 3:259]
    for x in (room[2, 5:261].expand(9, 256), room[::2, 1:257], room[4:, 2:258].unflatten(0, (6, 11))):
        # (bounds as above; not the dense copies' numbers, bit for bit: those are read in units of 16 bytes, these one by one, so
        # that a row's 256 numbers are summed in another order)
        leaves, n, D = [t.detach().requires_grad_() for t in (x, w, b)], x.numel() // 256, 256
        y, g = layer_norm(*leaves), room[5, 7:263].expand(x.shape)
        f = [t.detach().cpu().double() for t in (x.reshape(-1, D), w, b)]
        want = rows_ref.layer_norm(*f, 1e-5, g.reshape(-1, D).cpu().double())
        r = (f[0].var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
        second = float(((D + 2) * ref.U * f[0].abs().mean(1, keepdim=True) * r).square().max())
        gx, gw, gb = torch.autograd.grad(y, leaves, g)
        ref.within(y.view(-1, D), *want[0], D + 20, "y", second)
        ref.within(gx.reshape(-1, D), *want[1], 3 * D + 60, "gx", 3 * second)
        ref.within(gw, *want[2], n + D + 40, "gweight", second)
        ref.within(gb, *want[3], n + 5, "gbias")
        counts = torch.tensor([9, 5, 9, 3], device="cuda")
        assert torch.equal(dropout(x, 0.5, counts[::2]), dropout(x.clone(), 0.5, torch.tensor([9, 9], device="cuda")))
        assert torch.equal(dropout(x, 0.5, counts[2:]), dropout(x.clone(), 0.5, torch.tensor([9, 3], device="cuda")))
