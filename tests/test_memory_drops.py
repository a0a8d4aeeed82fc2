"""Which numbers MemoryActor's dropout drops: each actor and each pass others, and never others in a pass that is made again."""
from __future__ import annotations

import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from conftest import GOLDEN, lively, toy
from flyguy_amd.fly import FlyActor
from flyguy_amd.memory import MemoryActor


def net(**kw):
    f = lively(FlyActor(toy("a"), 517, 90, hops=3), 1)
    m = MemoryActor(f, **(dict(heads=4, k_heads=2, dim=16, positions=64, dropout=0.5) | kw))
    with torch.no_grad():
        m.back.weight.fill_(0.1)
    return m


def dropped(m):
    """The mask of the actor's next pass."""
    return m._dropped(torch.ones(1, 1, 64)) == 0


def test_two_actors_drop_different_numbers(tmp_path):
    torch.manual_seed(7)
    a, b = net(), net()
    assert a.drops[0] != b.drops[0] and not torch.equal(dropped(a), dropped(b))
    torch.save(a.checkpoint(str(GOLDEN / "toy_a.npz")), tmp_path / "m.pt")
    c, d = MemoryActor.load(tmp_path / "m.pt"), MemoryActor.load(tmp_path / "m.pt")
    assert len({int(x.drops[0]) for x in (a, b, c, d)}) == 4
    torch.manual_seed(7)                                    # (the same program again: the same numbers)
    again = net()
    assert torch.equal(again.drops[0], a.drops[0])


def test_a_copy_goes_on_as_its_original_would():
    torch.manual_seed(8)
    a = net()
    dropped(a)
    b = copy.deepcopy(a)
    for _ in range(3):
        assert torch.equal(dropped(a), dropped(b))
    assert torch.equal(a.drops, b.drops) and int(a.drops[1]) == 4


def test_weights_are_as_without_dropout():
    """Drawing the seed comes after all weights are drawn."""
    torch.manual_seed(9)
    a = net(dropout=0.0)
    torch.manual_seed(9)
    b = net()
    for (name, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert torch.equal(p, q), name


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_pass_made_again_for_its_gradient_is_refused(reentrant):
    """Activation checkpointing would make the pass again with the next mask, and so the gradients of another one."""
    m = net()
    x = torch.randn(2, 6, 517, requires_grad=True)
    out = checkpoint(lambda x: m(x)[0], x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="drop"):
        out.square().mean().backward()
    m.eval()                                                # (nothing is dropped: nothing to refuse)
    checkpoint(lambda x: m(x)[0], x, use_reentrant=reentrant).square().mean().backward()
    m = net(dropout=0.0)
    checkpoint(lambda x: m(x)[0], x, use_reentrant=reentrant).square().mean().backward()
