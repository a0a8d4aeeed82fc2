"""The actor that remembers (flyguy_amd.memory.MemoryActor) and its teaching command, on the CPU: a fresh one decides as its
actor, a stretch in pieces or moment by moment is the stretch at once, nothing reaches an earlier moment, and a memory can be
taught what no single moment shows."""
from __future__ import annotations

import copy
import pickle
import re
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from conftest import GOLDEN, lively, toy
from flyguy_amd.fly import FlyActor
from flyguy_amd.memory import MemoryActor
from flyguy_amd.remember import main
from oracle import trainer as ot


def net(**kw):
    torch.manual_seed(1)
    f = lively(FlyActor(toy("a"), 517, 90, hops=3), 1)
    m = MemoryActor(f, **(dict(heads=4, k_heads=2, dim=16, positions=64) | kw))
    with torch.no_grad():
        m.back.weight.normal_(0, 0.3)
    return m


def test_a_fresh_memory_changes_nothing():
    m = net()
    torch.nn.init.zeros_(m.back.weight)
    x = torch.randn(2, 7, 517)
    with torch.no_grad():
        want = m.actor(x.flatten(0, 1)).unflatten(0, (2, 7))
        torch.testing.assert_close(m(x)[0], want, rtol=1e-5, atol=1e-5)


def test_pieces_and_single_moments():
    m = net()
    x = torch.randn(3, 20, 517)
    with torch.no_grad():
        whole, (mem, seen) = m(x)
        a, st = m(x[:, :8])
        b, (mem2, seen2) = m(x[:, 8:], st)
        live = m.state(3)
        played = torch.stack([m.step(x[:, t], live) for t in range(20)], 1)
    torch.testing.assert_close(torch.cat([a, b], 1), whole, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(played, whole, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(mem2, mem, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(live[0], mem, rtol=1e-4, atol=1e-4)
    assert seen.tolist() == seen2.tolist() == live[1].tolist() == [20] * 3


def test_only_what_was_seen_counts():
    m = net()
    x = torch.randn(1, 12, 517)
    y = x.clone()
    y[:, 9:] = torch.randn(1, 3, 517)
    with torch.no_grad():
        a, b = m(x)[0], m(y)[0]
    torch.testing.assert_close(a[:, :9], b[:, :9], rtol=1e-5, atol=1e-5)
    assert (a[:, 9:] - b[:, 9:]).abs().max() > 1e-3


def test_past_the_table():
    """A car that goes on past the table keeps a memory of numbers, its later moments at the table's last position, however it is
    read; a stretch from the start that is longer is refused."""
    m, x = net(positions=8), torch.randn(2, 30, 517)
    far = net(positions=64)
    far.table[8:] = far.table[7]
    with torch.no_grad():
        want, (mem, _) = far(x)
        live = m.state(2)
        played = torch.stack([m.step(x[:, t], live) for t in range(30)], 1)
        a, st = m(x[:, :6])
        b, (mem2, seen) = m(x[:, 6:], st)
    assert torch.isfinite(played).all() and live[1].tolist() == seen.tolist() == [30] * 2
    torch.testing.assert_close(played, want, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(torch.cat([a, b], 1), want, rtol=1e-4, atol=1e-4)
    for got in (live[0], mem2):
        torch.testing.assert_close(got, mem, rtol=1e-4, atol=1e-4)
    with pytest.raises(ValueError, match="positions is 8"):
        m(x[:, :9])
    with pytest.raises(ValueError, match="one position"):
        net(positions=0)


@pytest.mark.parametrize("grad", [False, True])
def test_threads_that_share_an_actor(grad):
    """Two threads play through one MemoryActor, and a third through another with the same actor: each gets what it gets alone."""
    m, other = net(), net()
    other.actor = m.actor
    xs = [torch.randn(60, 1, 517) for _ in range(3)]

    def play(m, x):
        live, out = m.state(1), []
        with torch.set_grad_enabled(grad):
            for t in range(60):
                if grad:
                    y, live = m(x[t][:, None], live)
                    out.append(y[:, 0].detach())
                else:
                    out.append(m.step(x[t], live))
        return torch.stack(out), live[0].detach()
    nets = (m, m, other)
    alone = [play(n, x) for n, x in zip(nets, xs)]
    with ThreadPoolExecutor(3) as pool:
        for _ in range(3):
            for got, want in zip(pool.map(play, nets, xs), alone):
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_cpu_play_is_the_actors(monkeypatch):
    """A step on the CPU decides in compiled code, without gradients: a fresh memory gives the actor's logits bit for bit, and
    both forms of play the same firing."""
    m = net()
    torch.nn.init.zeros_(m.back.weight)
    x, grads = torch.randn(4, 517), []
    walk = FlyActor._walk
    monkeypatch.setattr(FlyActor, "_walk", lambda *a, **kw: grads.append(torch.is_grad_enabled()) or walk(*a, **kw))
    with torch.no_grad():
        want = m.actor(x)
        assert torch.equal(m.step(x, m.state(4)), want) and not grads
        _, firing = m.actor.with_firing(x)
        top = m.actor._firing(x)
    assert grads == [False] and (firing > 0).any()
    torch.testing.assert_close(firing, top, rtol=1e-5, atol=1e-5)
    logits, again = m.actor.with_firing(x)                     # (with gradients)
    torch.testing.assert_close(again, firing, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(logits, want, rtol=1e-5, atol=1e-5)


def test_copies_of_an_actor_that_has_played():
    """A copy and a pickle of an actor that has decided on the CPU decide by themselves."""
    m, x = net(), torch.randn(3, 517)
    with torch.no_grad():
        want = m.step(x, m.state(3))
        copies = [copy.deepcopy(m), pickle.loads(pickle.dumps(m))]
        m.actor.out.bias.add_(1.0)
        moved = m.step(x, m.state(3))
        for c in copies:
            assert torch.equal(c.step(x, c.state(3)), want)
            assert c.actor._decider[1] is not None and c.actor._decider[1] is not m.actor._decider[1]
    torch.testing.assert_close(moved, want + 1.0)


def test_heads_must_share():
    with pytest.raises(ValueError, match="multiple"):
        net(heads=4, k_heads=3)


def test_teaching_a_memory(tmp_path, capsys):
    """Answers that depend on the moment before: with a memory the distance falls."""
    rng = np.random.default_rng(4)
    obs = rng.standard_normal((400, 517)).astype(np.float16)
    ans = np.zeros((400, 90), np.float16)
    side = np.concatenate([[False], obs[:-1, 0] > 0])
    ans[side, 3], ans[~side, 7] = 6, 6
    data = tmp_path / "game.bin"
    ot.write_chunk(data, obs, ans)
    torch.manual_seed(5)
    f = lively(FlyActor(toy("a"), 517, 90, hops=3), 5)
    ck = tmp_path / "actor.pt"
    torch.save({"model": {"actor." + k: v for k, v in f.state_dict().items()}}, ck)
    out = tmp_path / "memory.pt"
    assert main(["--data", str(data), "--graph", str(GOLDEN / "toy_a.npz"), "--start", str(ck), "--stretch", "24", "--cars", "4",
                 "--steps", "40", "--heads", "2", "--dim", "8", "--lr", "1e-2", "--device", "cpu", "--out", str(out)]) == 0
    text = capsys.readouterr().out
    first, last = (float(v) for v in re.search(r"KL ([0-9.]+) -> ([0-9.]+)", text).groups())
    assert last < 0.7 * first
    assert float(re.search(r"off by ([0-9.e+-]+)", text).group(1)) <= 1e-4
    saved = torch.load(out, weights_only=True)
    assert set(saved["memory"]) == {"proj.weight", "wq", "wk", "back.weight", "log_decay"}


def test_a_taught_memory_is_read_back(tmp_path, monkeypatch):
    """What the command writes decides as what it taught, with the actor it was taught on: a fresh one, or a checkpoint's with
    hops and a fan of its own."""
    rng = np.random.default_rng(6)
    data = tmp_path / "game.bin"
    ot.write_chunk(data, rng.standard_normal((60, 517)).astype(np.float16), (3 * rng.standard_normal((60, 90))).astype(np.float16))
    f = lively(FlyActor(toy("a"), 517, 90, hops=2, fan=7), 6)
    torch.save({"model": {"actor." + k: v for k, v in f.state_dict().items()}, "config": {"model": {"fly_hops": 2, "fly_fan": 7}}},
               tmp_path / "actor.pt")
    taught, init = [], MemoryActor.__init__
    monkeypatch.setattr(MemoryActor, "__init__", lambda self, *a, **kw: taught.append(self) or init(self, *a, **kw))
    x = torch.randn(2, 11, 517)
    for start in ([], ["--start", str(tmp_path / "actor.pt")]):
        assert main(["--data", str(data), "--graph", str(GOLDEN / "toy_a.npz"), "--stretch", "12", "--cars", "3", "--steps", "4",
                     "--heads", "4", "--dim", "12", "--device", "cpu", "--out", str(tmp_path / "m.pt"), *start]) == 0
        net = MemoryActor.load(tmp_path / "m.pt")
        with torch.no_grad():
            assert torch.equal(net(x)[0], taught[-2](x)[0])
        assert net.actor.hops == (2 if start else 3) and len(net.table) == 65536
        if start:
            assert torch.equal(net.actor.w, f.w) and torch.equal(net.actor.in_w, f.in_w)
    (tmp_path / "elsewhere.npz").write_bytes((GOLDEN / "toy_a.npz").read_bytes())
    again = MemoryActor.load(tmp_path / "m.pt", graph=str(tmp_path / "elsewhere.npz"))
    with torch.no_grad():
        assert torch.equal(again(x)[0], net(x)[0])


@pytest.mark.parametrize("what", ["--steps", "--cars", "--stretch"])
def test_nothing_to_teach(tmp_path, what):
    with pytest.raises(SystemExit, match="at least 1"):
        main(["--data", str(tmp_path / "none.bin"), "--graph", str(GOLDEN / "toy_a.npz"), "--device", "cpu", what, "0"])


def test_too_short_a_recording(tmp_path):
    data = tmp_path / "game.bin"
    ot.write_chunk(data, np.zeros((5, 517), np.float16), np.zeros((5, 90), np.float16))
    with pytest.raises(SystemExit, match="no file holds"):
        main(["--data", str(data), "--graph", str(GOLDEN / "toy_a.npz"), "--device", "cpu"])
