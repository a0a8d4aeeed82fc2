"""The gated delta rule keeps to the room it asks for, and many short stretches."""
from __future__ import annotations

import pytest
import torch

from gpu_helpers import say

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
GUARD = 1 << 16

# lengths of stretches (one number: alike), moments before and behind, q heads, k heads, K, V
ROOMS = [([1], 0, 1, 1, 1, 1), (3, 65, 2, 2, 64, 64), ([0, 130, 7, 64, 0], 3, 4, 2, 40, 72), (1, 2100, 2, 1, 128, 128),
         ([1900, 0, 700, 3, 2500, 64], 5, 2, 1, 48, 80), (2, 33, 6, 3, 128, 33), ([150, 1], 40, 1, 1, 7, 128), (1, 1, 32768, 32768, 16, 128)]


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("case", ROOMS, ids=str)
def test_nothing_is_written_outside_its_room(gpu_lib, case, dt, monkeypatch):
    """What lies before and behind the workspaces, what the forward keeps, outputs and gradients stays as it was, and results are what
    they are in rooms of torch's own."""
    from flyguy_amd import memory_hip
    say(f"rooms {case} {dt}")
    gen = torch.Generator().manual_seed(71)
    draw = lambda *s: torch.randn(*s, generator=gen)          # noqa: E731
    packed = isinstance(case[0], list)
    lengths, rest, H, Hk, K, V = case
    if packed:
        bounds = [rest]
        for x in lengths:
            bounds.append(bounds[-1] + x)
        shape, n, starts = (bounds[-1] + rest,), len(lengths), torch.tensor(bounds, device="cuda")
    else:
        shape, n, starts = (lengths, rest), lengths, None
    ins = [draw(*shape, H, K).to(dt).cuda(), (draw(*shape, Hk, K) * K ** -0.5).to(dt).cuda(), draw(*shape, Hk, V).to(dt).cuda(),
           -draw(*shape, H).abs().cuda(), draw(*shape, H).sigmoid().cuda(), draw(n, H, K, V).cuda()]
    go, gs = draw(*shape, H, V).to(dt).cuda(), draw(n, H, K, V).cuda()

    def work():
        leaves = [x.detach().requires_grad_() for x in ins]
        with torch.no_grad():
            play = memory_hip.delta_attention(*leaves, starts)
        out = memory_hip.delta_attention(*leaves, starts)
        return (*play, *(x.detach() for x in out), *torch.autograd.grad(out, leaves, (go, gs)))

    want, guarded, plain = work(), [], torch.Tensor.new_empty

    def new_empty(self, *size, dtype=None, **kw):
        """Memory of that size inside a larger one."""
        size = size[0] if len(size) == 1 and not isinstance(size[0], int) else size
        like = plain(self, 0, dtype=dtype, **kw)
        if not like.is_cuda:
            return plain(self, size, dtype=dtype, **kw)
        count = 1
        for s in size:
            count *= s
        data = -(-count * like.element_size() // 16) * 16
        room = torch.full((data + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=like.device)
        guarded.append((room, count * like.element_size()))
        return room[GUARD:GUARD + count * like.element_size()].view(like.dtype).view(size)

    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    got = work()
    monkeypatch.undo()
    assert len(guarded) >= 10
    for room, used in guarded:
        assert (room[:GUARD] == 0xA5).all() and (room[GUARD + used:] == 0xA5).all(), used
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_as_many_packed_stretches_as_there_may_be(gpu_lib, dt):
    """16,384 stretches of 0 to 5 moments and a few long ones: each what it is among stretches of its own length."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"many {dt}")
    gen = torch.Generator().manual_seed(72)
    n, H, Hk, K, V = 16384, 2, 1, 24, 16
    lengths = torch.randint(0, 6, (n,), generator=gen)
    lengths[torch.tensor([0, 5000, n - 1])] = 70
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    M = int(starts[-1])
    draw = lambda *s, to=F32: torch.randn(*s, generator=gen).to(to).cuda()        # noqa: E731
    q, k, v = draw(M, H, K, to=dt), 0.2 * draw(M, Hk, K, to=dt), draw(M, Hk, V, to=dt)
    g, b, s = -draw(M, H).abs(), draw(M, H).sigmoid(), draw(n, H, K, V)
    go, gs = draw(M, H, V, to=dt), draw(n, H, K, V)
    leaves = [x.requires_grad_() for x in (q, k, v, g, b, s)]
    o, e = delta_attention(*leaves, starts.cuda())
    grads = torch.autograd.grad((o, e), leaves, (go, gs))
    seen = 0
    for length in sorted(set(lengths.tolist())):
        of = (lengths == length).nonzero()[:, 0]
        at = (starts[of][:, None] + torch.arange(length)).cuda()
        rows, of = [x.detach()[at].requires_grad_() for x in (q, k, v, g, b)], of.cuda()
        given = [*rows, s.detach()[of].requires_grad_()]
        po, pe = delta_attention(*given)
        pg = torch.autograd.grad((po, pe), given, (go[at], gs[of]))
        assert torch.equal(o[at], po) and torch.equal(e[of], pe), length
        for x, y, i in zip(grads, pg, [at] * 5 + [of]):
            assert torch.equal(x[i], y), length
        seen += at.numel()
    assert seen == M
    with pytest.raises(Exception, match="stretches"):
        delta_attention(q, k, v, g, b, None, torch.zeros(n + 2, dtype=torch.int64, device="cuda"))
