"""Layer norm and its gradients keep to their rooms: workspaces, statistics, and outputs whose rows lie apart."""
from __future__ import annotations

import pytest
import torch

from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def guarded(n, dtype=F32, guard=4096):
    room = torch.full((n * dtype.itemsize + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
    part = room[guard:guard + n * dtype.itemsize].view(dtype)
    return part, lambda: bool((room[:guard] == 0xA5).all() and (room[guard + n * dtype.itemsize:] == 0xA5).all())


@pytest.mark.parametrize("gap", [0, 8, 5])
@pytest.mark.parametrize("n,D,dt", [(1, 1, F32), (33, 7, BF16), (700, 64, F16), (5, 1002, F32), (2100, 1332, F32), (9, 4097, BF16), (3, 8192, F16),
                                    (40, 8196, F32), (2, 20001, BF16)])
def test_nothing_is_written_outside_its_room(gpu_lib, n, D, dt, gap):
    from flyguy_amd._lib import lib
    from flyguy_amd.rows_hip import _call, _pack_norm, layer_norm
    say(f"rooms {n} {D} {dt} {gap}")
    gen = torch.Generator().manual_seed(n + D)
    draw = lambda *s: torch.randn(*s, generator=gen)          # noqa: E731
    x, g = (draw(n, D + gap).to(dt).cuda()[:, :D] for _ in range(2))
    w, b = draw(D).cuda(), draw(D).cuda()
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    want_y = layer_norm(*leaves)
    want = torch.autograd.grad(want_y, leaves, g)
    row = D + gap
    (y, y_kept), (gx, gx_kept) = (guarded(n * row, dt) for _ in range(2))
    before = y.clone()
    y, gx, before = (t.view(n, row) for t in (y, gx, before))
    (stats, stats_kept), (gw, gw_kept), (gb, gb_kept) = guarded(2 * n), guarded(D), guarded(D)
    size = lib().fm_norm_partial(_pack_norm(x, *[None] * 9, 0.0))
    partial, partial_kept = guarded(size)
    _call("fm_norm", x, _pack_norm(x, y[:, :D], None, None, w, b, None, None, stats, None, 1e-5))
    _call("fm_norm_bwd", x, _pack_norm(x, None, g, gx[:, :D], w, None, gw, gb, stats, partial, 1e-5))
    for kept in (y_kept, gx_kept, stats_kept, gw_kept, gb_kept, partial_kept):
        assert kept()
    bits = torch.int32 if dt == F32 else torch.int16
    for t in (y, gx):                                         # (the gaps between rows)
        assert torch.equal(t[:, D:].contiguous().view(bits), before[:, D:].contiguous().view(bits))
    # (rows apart may be read in other units than dense ones, whose sums run in another order: a few roundings of sums of D or n numbers)
    for got, w64, count in ((y[:, :D], want_y, D), (gx[:, :D], want[0], 3 * D), (gw, want[1], n + D), (gb, want[2], n)):
        w64 = w64.detach()
        off = (got.double() - w64.double()).abs()
        step = {F32: 2.0 ** -24, BF16: 2.0 ** -7, F16: 2.0 ** -10}[got.dtype]     # (two roundings of half a step, of values as good as alike)
        scale = float(w64.double().abs().max()) + float(g.double().abs().max())
        assert float((off - step * w64.double().abs()).max()) <= (count + 60) * 2.0 ** -24 * scale * max(1.0, n ** 0.5), (n, D)
