"""Layer norm, its gradient and dropout written over what they read, as include/flyguy_memory.h allows: the same numbers, bit for
bit, as in memory of their own (the same kernels on the same values)."""
from __future__ import annotations

import pytest
import torch

from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# (rows of a wave end at 1,024 values, those held in registers at 8,192)
SIZES = [(70, 40, F32), (9, 1024, BF16), (9, 1025, F32), (70, 1332, F32), (5, 8192, F16), (5, 8193, F32), (70, 9000, BF16), (3, 20001, F16)]


def inputs(n, D, dt, pad=0):
    gen = torch.Generator().manual_seed(n + D)
    draw = lambda *s: torch.randn(*s, generator=gen)                      # noqa: E731
    rows = lambda: draw(n, D + pad).to(dt).cuda()[:, :D]                  # noqa: E731
    return rows(), rows(), (1 + 0.3 * draw(D)).cuda(), (0.3 * draw(D)).cuda()


def norm(x, y, w, b, stats):
    from flyguy_amd.rows_hip import _call, _pack_norm
    _call("fm_norm", x, _pack_norm(x, y, None, None, w, b, None, None, stats, None, 1e-5))


def norm_bwd(x, g, gx, w, stats):
    from flyguy_amd.rows_hip import _call, _pack_norm, _partial
    gw, gb = torch.empty_like(w), torch.empty_like(w)
    _call("fm_norm_bwd", x, _pack_norm(x, None, g, gx, w, None, gw, gb, stats, _partial(x, stats), 1e-5))
    return gw, gb


@pytest.mark.parametrize("pad", [0, 8])
@pytest.mark.parametrize("n,D,dt", SIZES)
def test_layer_norm_in_place(gpu_lib, n, D, dt, pad):
    say(f"in place {n} {D} {dt} {pad}")
    x, g, w, b = inputs(n, D, dt, pad)
    like = lambda t: torch.empty(n, D + pad, dtype=dt, device="cuda")[:, :D]      # noqa: E731
    stats, again = (torch.empty(n, 2, device="cuda") for _ in range(2))
    y, gx = like(x), like(x)
    norm(x, y, w, b, stats)
    gw, gb = norm_bwd(x, g, gx, w, stats)
    over = like(x).copy_(x)
    norm(over, over, w, b, again)
    assert torch.equal(over, y) and torch.equal(again, stats)
    for which in ("x", "g"):                                # gx over x, over g
        given = {"x": like(x).copy_(x), "g": like(x).copy_(g)}
        got = norm_bwd(given["x"], given["g"], given[which], w, stats)
        assert torch.equal(given[which], gx), which
        assert torch.equal(got[0], gw), ("gweight", which)
        assert torch.equal(got[1], gb), ("gbias", which)
        other = "g" if which == "x" else "x"
        assert torch.equal(given[other], {"x": x, "g": g}[other])


@pytest.mark.parametrize("n,dt", [(7, F32), (4096, BF16), (100003, F16)])
def test_dropout_in_place(gpu_lib, n, dt):
    from flyguy_amd.rows_hip import _DROP, _TYPES, _call, dropout
    gen = torch.Generator().manual_seed(n)
    c = torch.tensor([n, 3], device="cuda")
    for at in (0, 1):                                       # (whole units, and at no multiple of 16 bytes)
        x = torch.randn(n + at, generator=gen).to(dt).cuda()[at:]
        want = dropout(x, 0.3, c)
        _call("fm_drop", x, _DROP.pack(x.data_ptr(), x.data_ptr(), c.data_ptr(), n, 1, n, _TYPES[dt], 0.3))
        assert torch.equal(x, want)
