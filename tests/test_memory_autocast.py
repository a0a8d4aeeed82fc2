"""MemoryActor under torch.autocast: projections in 16 bits, gates, states and norms in float32."""
from __future__ import annotations

import pytest
import torch

from conftest import lively, toy
from flyguy_amd.fly import FlyActor
from flyguy_amd.memory import EPS, MemoryActor


def net(**kw):
    torch.manual_seed(5)
    m = MemoryActor(lively(FlyActor(toy("b"), 517, 90, hops=3), 5), heads=4, k_heads=2, dim=24, positions=128, **kw)
    with torch.no_grad():
        m.back.weight.normal_(0, 0.3)
        if m.rule == "delta":
            m.gates.weight.normal_(0, 0.05)
            m.gates.bias.normal_(0, 1)
    return m


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gates_are_float32(dt):
    m = net(rule="delta")
    firing = torch.rand(2, 3, m.proj.in_features)
    with torch.no_grad(), torch.autocast("cpu", dtype=dt):
        q, k, v, decay, rate = m._heads(firing)
        gates = m.gates(firing).float().unflatten(-1, (2, -1)).unbind(-2)
    assert q.dtype == k.dtype == v.dtype == dt and decay.dtype == rate.dtype == torch.float32
    # (not 16-bit numbers made float32: what the gates' product rounds is rounded once)
    assert torch.equal(rate, torch.sigmoid(gates[1]))


def test_an_actor_in_64_bits_keeps_them():
    m = net(rule="delta").double()
    firing = torch.rand(2, 3, m.proj.in_features, dtype=torch.float64)
    with torch.no_grad():
        assert all(x.dtype == torch.float64 for x in m._heads(firing))


@pytest.mark.parametrize("kw", [{"rule": "decay"}, {"rule": "delta"}, {"rule": "delta", "norm": True, "dropout": 0.2}])
def test_a_pass_on_the_cpu(kw):
    m = net(**kw)
    x = torch.randn(2, 6, 517)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        out, (mem, _) = m(x)
        out.float().square().mean().backward()
        live = m.state(2)
        with torch.no_grad():
            m.step(x[:, 0], live)
    assert torch.isfinite(out).all() and mem.dtype == live[0].dtype == torch.float32
    assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [{"rule": "decay"}, {"rule": "delta"}, {"rule": "delta", "norm": True, "dropout": 0.2}])
def test_a_pass_on_the_gpu(gpu_lib, kw, dt):
    """The 16-bit kernels, reached through the actor: what the operators give one by one on what the actor hands them, bit for
    bit; gradients for all that learns; and a step."""
    from flyguy_amd.memory_hip import decay_attention, decay_step, delta_attention, delta_step, norm_rotary
    m = net(**kw)
    m.actor.kernel = "hip"
    m = m.cuda()
    x = torch.randn(3, 70, 517, device="cuda")
    with torch.autocast("cuda", dtype=dt):
        out, _ = m(x)
        out.float().square().mean().backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    m.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=dt):
        out, (mem, seen) = m(x)
        logits, firing = m._see(x.flatten(0, 1))
        q, k, v, decay, rate = m._heads(firing.unflatten(0, (3, 70)))
        assert q.dtype == k.dtype == v.dtype == dt and decay.dtype == torch.float32
        at = torch.arange(70, device="cuda", dtype=torch.int32).expand(3, 70)
        q, k = norm_rotary(q, k, m.wq, m.wk, m.table, at, eps=EPS)
        first = m.state(3)[0]
        o, end = decay_attention(q, k, v, decay, first) if rate is None else delta_attention(q, k, v, decay, rate, first)
        assert o.dtype == dt and torch.equal(end, mem) and seen.tolist() == [70] * 3
        assert torch.equal(out, logits.unflatten(0, (3, 70)) + m.back(o.flatten(-2)))
        live, before = (mem.clone(), seen.clone()), mem.clone()
        got = m.step(x[:, 0], live)
        logits, firing = m._see(x[:, 0])
        q, k, v, decay, rate = m._heads(firing)
        q, k = norm_rotary(q[:, None], k[:, None], m.wq, m.wk, m.table, m._at(seen[:, None]), eps=EPS)
        o = decay_step(q[:, 0], k[:, 0], v, decay, before) if rate is None else delta_step(q[:, 0], k[:, 0], v, decay, rate, before)
        assert torch.equal(got, logits + m.back(o.flatten(-2))) and torch.equal(before, live[0])
