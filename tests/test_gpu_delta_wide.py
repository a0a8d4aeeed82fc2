"""The gated delta rule with so many heads that moments lie 2^22 values apart and more, whose tensors the library copies."""
from __future__ import annotations

import pytest
import torch

from gpu_helpers import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hk,K,V", [(32768, 32768, 16, 128), (32768, 16, 64, 128), (32768, 32768, 128, 8)])
def test_heads_by_the_ten_thousand(gpu_lib, H, Hk, K, V):
    """All heads at once give what each half of them gives, bit for bit; gradients too, and with tensors broadcast over moments."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"wide {H} {Hk} {K} {V}")
    gen = torch.Generator(device="cuda").manual_seed(H + K)
    draw = lambda *s, dt=torch.bfloat16: torch.randn(*s, device="cuda", generator=gen).to(dt)     # noqa: E731
    T = 2
    ins = [draw(1, T, H, K), draw(1, T, Hk, K) * K ** -0.5, draw(1, T, Hk, V), -draw(1, T, H, dt=torch.float32).abs(),
           draw(1, T, H, dt=torch.float32).sigmoid()]
    go = draw(1, T, H, V)

    def work(given, go):
        leaves = [x.detach().requires_grad_() for x in given]
        o, e = delta_attention(*leaves)
        return o.detach(), e.detach(), torch.autograd.grad(o, leaves, go)

    for how in ("broadcast", "dense"):                      # (the same sizes: one must not leave the other too little room)
        given, g = ins, go
        if how == "broadcast":
            given, g = [x[:, :1].expand(x.shape[0], T, *x.shape[2:]) for x in ins], go[:, :1].expand(1, T, H, V)
        o, e, grads = work(given, g)
        for half in range(2):
            q, kv = slice(half * H // 2, (half + 1) * H // 2), slice(half * Hk // 2, (half + 1) * Hk // 2)
            heads = [q, kv, kv, q, q]
            po, pe, pg = work([x[:, :, s].contiguous() for x, s in zip(given, heads)], g[:, :, q].contiguous())
            assert torch.equal(po, o[:, :, q]) and torch.equal(pe, e[:, q]), (how, half)
            for x, y, s in zip(grads, pg, heads):
                assert torch.equal(x[:, :, s], y), (how, half)
