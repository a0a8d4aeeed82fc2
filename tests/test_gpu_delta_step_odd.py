"""One moment of the gated delta rule with numbers that are not finite: what each reaches is NaN, as include/flyguy_memory.h says of
stretches, and nothing else changes."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("n,K,V", [(3, 24, 20), (3, 128, 7), (140, 64, 128)])
def test_what_is_not_finite(gpu_lib, dt, n, K, V):
    """A query's reaches its own output, a value's its column of its heads, a key's, decay's or rate's all of its heads.  States and
    keys hold zeros too, among them a whole column and a whole head of the state, which infinities times zero go through."""
    from flyguy_amd.memory_hip import delta_attention, delta_step
    say(f"odd step {dt} {n} {K} {V}")
    gen = torch.Generator().manual_seed(n + K + V)
    draw = lambda *s, dtype=F32: torch.randn(*s, generator=gen).to(dtype).cuda()  # noqa: E731
    q, k, v = draw(n, 4, K, dtype=dt), 0.1 * draw(n, 2, K, dtype=dt), draw(n, 2, V, dtype=dt)
    k[..., 3:9] = 0
    g, b, s = -draw(n, 4).abs(), draw(n, 4).sigmoid(), draw(n, 4, K, V)
    s[..., V - 1] = 0
    s[1, 2] = 0
    ins = [q, k, v, g, b]
    want_s = s.clone()
    want = delta_step(*ins, want_s)
    for what in range(5):
        for odd in (math.nan, math.inf, -math.inf):
            if what == 3 and odd == -math.inf:              # (forgets everything)
                continue
            for value in (4, V - 1):                        # (a column of numbers, and the one of zeros; of a key or query, one or other)
                given = [x.clone() for x in ins]
                heads = slice(2, 3) if what in (0, 3, 4) else slice(2, 4)     # (key head 1's query heads)
                given[what][(1, 2 if what in (0, 3, 4) else 1) + ((min(value, K - 1 if what < 2 else V - 1),) if what < 3 else ())] = odd
                after = s.clone()
                o = delta_step(*given, after)
                hit, hit_s = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(s, dtype=torch.bool)
                if what == 0:
                    hit[1, heads] = True
                elif what == 2:
                    hit[1, heads, value], hit_s[1, heads, :, value] = True, True
                else:
                    hit[1, heads], hit_s[1, heads] = True, True
                assert torch.equal(o[~hit], want[~hit]) and torch.equal(after[~hit_s], want_s[~hit_s]), (what, odd, value)
                assert not torch.isfinite(o[hit]).any(), (what, odd, value)
                if what:
                    assert torch.isnan(o[hit]).all() and torch.isnan(after[hit_s]).all(), (what, odd, value)
                # the same of a stretch of one moment
                w, end = delta_attention(*[x[:, None] for x in given], s)
                assert torch.equal(torch.isfinite(w[:, 0]), torch.isfinite(o)), (what, odd, value)
                assert torch.equal(torch.isnan(end), torch.isnan(after)), (what, odd, value)


def test_forgetting_everything(gpu_lib):
    """A log decay of -inf, and rates of 0 and 1: finite numbers stay finite."""
    from flyguy_amd.memory_hip import delta_step
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, 2, 16, generator=gen).cuda() for _ in range(3))
    s = torch.randn(2, 2, 16, 16, generator=gen).cuda()
    g, b = torch.full((2, 2), -math.inf, device="cuda"), torch.tensor([[0.0, 1.0], [1.0, 0.0]], device="cuda")
    o = delta_step(q, k, v, g, b, s)
    u = b[..., None] * v
    assert torch.equal(s, k[..., :, None] * u[..., None, :] + 0.0) and torch.isfinite(o).all()
