"""MemoryActor with a memory that corrects itself, a normed firing and dropout, on the CPU."""
from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import rows_helpers
from conftest import GOLDEN, lively, toy
from flyguy_amd.fly import FlyActor
from flyguy_amd.memory import MemoryActor, _delta_attention_cpu, _dropout_cpu
from flyguy_amd.remember import main
from oracle import trainer as ot

import delta_helpers


def net(**kw):
    torch.manual_seed(1)
    f = lively(FlyActor(toy("a"), 517, 90, hops=3), 1)
    m = MemoryActor(f, **(dict(heads=4, k_heads=2, dim=16, positions=64, rule="delta", norm=True) | kw))
    with torch.no_grad():
        m.back.weight.normal_(0, 0.3)
        if m.rule == "delta":
            m.gates.weight.normal_(0, 0.05)
            m.gates.bias.normal_(0, 1)
    return m


def test_the_rule():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, 9, h, d, generator=g).double() for h, d in ((4, 6), (2, 6), (2, 5)))
    k = k / k.norm(dim=-1, keepdim=True)
    l, b, s = -torch.rand(2, 9, 4, generator=g).double(), torch.rand(2, 9, 4, generator=g).double(), torch.randn(2, 4, 6, 5, generator=g).double()
    for got, want in zip(_delta_attention_cpu(q, k, v, l, b, s), delta_helpers.delta(q, k, v, l, b, s, 6 ** -0.5)):
        torch.testing.assert_close(got, want)


@pytest.mark.parametrize("share", [0.0, 0.25, 1.0])
def test_dropped_numbers(share):
    x = torch.randn(3, 5, 7, generator=torch.Generator().manual_seed(3))
    for c in ((1, 2), ((1 << 62) + 12345, 1 << 40), (-7, -1)):
        assert torch.equal(_dropout_cpu(x, share, torch.tensor(c)), rows_helpers.dropout(x, share, c))


@pytest.mark.parametrize("kw", [{}, {"norm": False}, {"rule": "decay"}])
def test_pieces_and_single_moments(kw):
    m = net(**kw)
    x = torch.randn(3, 20, 517)
    with torch.no_grad():
        whole, (mem, seen) = m(x)
        a, st = m(x[:, :8])
        b, (mem2, _) = m(x[:, 8:], st)
        live = m.state(3)
        played = torch.stack([m.step(x[:, t], live) for t in range(20)], 1)
    for y, want in ((torch.cat([a, b], 1), whole), (played, whole), (mem2, mem), (live[0], mem)):
        torch.testing.assert_close(y, want, rtol=1e-4, atol=1e-4)


def test_dropout_in_training_alone():
    m = net(dropout=0.3)
    x = torch.randn(2, 6, 517)
    with torch.no_grad():
        a, b = m(x)[0], m(x)[0]
        m.eval()
        c, d = m(x)[0], m(x)[0]
        assert not torch.equal(a, b) and torch.equal(c, d) and m.drops[1] == 2
        m.train()                                           # (a step drops nothing, whatever the mode)
        live = m.state(2)
        played = torch.stack([m.step(x[:, t], live) for t in range(6)], 1)
    torch.testing.assert_close(played, c, rtol=1e-4, atol=1e-4)
    assert net().dropout == 0.0 and not hasattr(net(), "drops")


def test_what_learns():
    m = net(dropout=0.1)
    m.actor.requires_grad_(False)
    m(torch.randn(2, 6, 517))[0].square().mean().backward()
    learns = {n for n, p in m.named_parameters() if p.requires_grad}
    assert learns == {"proj.weight", "wq", "back.weight", "gates.weight", "gates.bias", "norm_w", "norm_b"}
    assert all(m.get_parameter(n).grad.abs().max() > 0 for n in learns)


@pytest.mark.parametrize("kw", [{"rule": "other"}, {"dropout": -0.1}, {"dropout": 1.5}])
def test_refusals(kw):
    with pytest.raises(ValueError, match="MemoryActor"):
        net(**kw)


def test_a_checkpoint_and_a_copy(tmp_path):
    m = net(dropout=0.2).eval()
    torch.save(m.checkpoint(str(GOLDEN / "toy_a.npz")), tmp_path / "m.pt")
    back = MemoryActor.load(tmp_path / "m.pt").eval()
    x = torch.randn(2, 5, 517)
    with torch.no_grad():
        want = m(x)[0]
        assert torch.equal(back(x)[0], want) and torch.equal(copy.deepcopy(m)(x)[0], want)
    assert (back.rule, back.dropout, back.norm_w is not None) == ("delta", 0.2, True)
    old = net(rule="decay", norm=False).checkpoint("g")                      # a file from before there was a choice
    for k in ("rule", "norm", "dropout"):
        del old["config"][k]
    old["config"]["model"]["fly_graph"] = str(GOLDEN / "toy_a.npz")
    torch.save(old, tmp_path / "old.pt")
    assert MemoryActor.load(tmp_path / "old.pt").rule == "decay"


def test_the_teaching_command(tmp_path, capsys):
    rng = np.random.default_rng(4)
    ot.write_chunk(tmp_path / "game.bin", rng.standard_normal((80, 517)).astype(np.float16),
                   (3 * rng.standard_normal((80, 90))).astype(np.float16))
    args = ["--data", str(tmp_path / "game.bin"), "--graph", str(GOLDEN / "toy_a.npz"), "--stretch", "12", "--cars", "3", "--steps", "3",
            "--heads", "2", "--dim", "8", "--device", "cpu", "--kernel", "torch", "--rule", "delta", "--norm", "--dropout", "0.2",
            "--out", str(tmp_path / "m.pt")]
    assert main(args) == 0
    said = capsys.readouterr().out
    off = float(said.split("logits off by ")[1].split()[0])
    assert off < 1e-4                                       # (play drops nothing)
    assert MemoryActor.load(tmp_path / "m.pt").rule == "delta"
    with pytest.raises(SystemExit, match="dropout"):
        main(args[:-2] + ["--dropout", "2", "--out", str(tmp_path / "m.pt")])
