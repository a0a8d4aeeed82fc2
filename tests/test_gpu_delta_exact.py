"""How exact the gated delta rule's float32 results are, head by head, and stretches whose starts fall."""
from __future__ import annotations

import math

import pytest
import torch

import delta_chunks
import delta_helpers as ref
import memory_helpers
from gpu_helpers import say

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("o", "end state", "q", "k", "v", "log_decay", "beta", "state")
HEADS_AT = {"o": 2, "end state": 1, "q": 2, "k": 2, "v": 2, "log_decay": 2, "beta": 2, "state": 1}
# What stays float32 whatever the inputs are
FLOATS = ("end state", "log_decay", "beta", "state")
SIZES = [(2, 200, 3, 64, 64), (1, 333, 2, 128, 96), (1, 2100, 2, 64, 128)]        # (the last is walked in segments)


def inputs(N, T, H, K, V, dt, seed=61):
    """Keys alike from moment to moment; the first head forgets within thousands of moments, the last within one."""
    gen = torch.Generator().manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=gen)          # noqa: E731
    k = draw(1, 1, H, K) + draw(N, T, H, K)
    k = 0.99 * k / k.square().sum(-1, keepdim=True).sqrt()
    g = -torch.rand(N, T, H, generator=gen) * torch.logspace(-3, 0, H)
    ins = [draw(N, T, H, K).to(dt), k.to(dt), draw(N, T, H, V).to(dt), g, torch.rand(N, T, H, generator=gen), draw(N, H, K, V)]
    return ins, draw(N, T, H, V).to(dt), draw(N, H, K, V)


def errors(outs, want):
    return {n: delta_chunks.off_by_head(x, w, HEADS_AT[n]) for n, x, w in zip(NAMES, outs, want)}


# A float32 sum of n products is off by n + 1 roundings of u = 2^-24.  Three bfloat16 terms of each operand (halves of a last bit:
# 2^-9, 2^-18, 2^-27 of a number) leave 2^-27 of each, and the pairs of terms that are dropped 2 x 2^-27 + 2^-36: together u / 2 of a
# product, less than one rounding more; its exponentials are off by 3 u and |x| u where the plain ones are by 1 u.  So the kernels'
# errors are those of the same chunks in plain float32, made of other roundings, and at most one more for each: twice as large,
# and 4 times where a head's few numbers make both sides' errors a matter of luck (the norm of some hundred independent roundings is within
# 20% of its expectation).  With two terms a product is off by 3 x 2^-18 of itself, 190 u: that shows far beyond it.
TIMES = 4.0


def test_the_bound_sees_sixteen_bits():
    """On the CPU: the same chunks with operands of 16 bits break the bound at every float32 result, in each head; other chunk
    lengths of plain float32 keep it."""
    for N, T, H, K, V in SIZES[:2]:
        ins, go, gs = inputs(N, T, H, K, V, BF16)
        f = [x.double() for x in ins]
        want = ref.delta(*f, K ** -0.5, None, go.double(), gs.double())
        plain = errors(delta_chunks.chunked(*ins, K ** -0.5, go, gs, 32), want)
        other = errors(delta_chunks.chunked(*ins, K ** -0.5, go, gs, 64), want)
        short = errors(delta_chunks.chunked(*ins, K ** -0.5, go, gs, 32, bits=16), want)
        for n in FLOATS:
            assert (other[n] <= TIMES * plain[n]).all(), (n, other[n] / plain[n])
            assert (short[n] > TIMES * plain[n]).all(), (n, short[n] / plain[n])
        again = errors(delta_chunks.chunked(*f, K ** -0.5, go, gs, 32, dtype=torch.float64), want)
        for n, w in zip(NAMES, want):                         # (the chunks are the rule)
            assert float(again[n].max()) <= 1e-12 * float(w.norm()), n


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("N,T,H,K,V", SIZES)
def test_float32_results_are_float32s(gpu_lib, N, T, H, K, V, dt):
    from flyguy_amd.memory_hip import delta_attention
    say(f"exact {N} {T} {H} {K} {V} {dt}")
    ins, go, gs = inputs(N, T, H, K, V, dt)
    leaves = [x.cuda().requires_grad_() for x in ins]
    out = delta_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, (go.cuda(), gs.cuda()))
    want = ref.delta(*[x.double() for x in ins], K ** -0.5, None, go.double(), gs.double())
    plain = errors(delta_chunks.chunked(*ins, K ** -0.5, go, gs, 64 if dt == BF16 else 32), want)
    got = errors((*out, *grads), want)
    for n, w in zip(NAMES, want):
        if n in FLOATS or dt == F32:
            bound = TIMES * plain[n]
        else:                                                 # 16 bits: its rounding, and two terms a product (190 u: as above) of 1 u's sums
            w = w.movedim(HEADS_AT[n], 0).flatten(1)
            bound = memory_helpers.ROUND[dt] * w.norm(dim=1) + 190 * plain[n] + (2.0 ** -25 * math.sqrt(w.shape[1]) if dt == F16 else 0)
        assert (got[n] <= bound).all(), (n, (got[n] / bound).tolist())


FALLING = [[0, 90, 40, 150], [-50, 70, 1000], [150, 0], [10, 10, 5, 5, 149], [120, 60, 90, 30, 140, 20], [3, 9, 8, 7, 6, 5, 4, 60, 61, 40, 130]]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("starts", FALLING, ids=str)
def test_starts_that_fall_cut_stretches_short(gpu_lib, starts, dt):
    check_spans(starts, 150, 2, 1, 16, 24, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("starts", [[5, 1900, 1200, 4000, 3900, 4100], [2000, 0, 2600, 2500, 4000, 9000], [-7, 2100, 2100, 300, 4090]], ids=str)
def test_long_stretches_whose_starts_fall(gpu_lib, starts, dt):
    """Long enough for segments, more than one a stretch."""
    check_spans(starts, 4100, 2, 1, 48, 40, dt)


def check_spans(starts, moments, H, Hk, K, V, dt):
    """Outputs, end states and gradients are those of the stretches that the library gives moments to (memory_helpers.risen:
    such as share none), and exactly zero at all other moments, whatever the memory held."""
    from flyguy_amd.memory_hip import delta_attention
    say(f"spans {starts} {dt}")
    n = len(starts) - 1
    gen = torch.Generator().manual_seed(n + moments)
    draw = lambda *s: torch.randn(*s, generator=gen)          # noqa: E731
    k = draw(Hk, K) + draw(moments, Hk, K)
    ins = [draw(moments, H, K).to(dt), (0.99 * k / k.norm(dim=-1, keepdim=True)).to(dt), draw(moments, Hk, V).to(dt),
           -draw(moments, H).abs(), torch.rand(moments, H, generator=gen), draw(n, H, K, V)]
    go, gs = draw(moments, H, V).to(dt), draw(n, H, K, V)
    bounds = memory_helpers.risen(starts, moments)
    want = ref.delta(*[x.double() for x in ins], K ** -0.5, bounds, go.double(), gs.double())
    outside = torch.ones(moments, dtype=torch.bool)
    outside[bounds[0]:bounds[-1]] = False
    for wide in (torch.int32, torch.int64):
        leaves = [x.cuda().requires_grad_() for x in ins]
        st = torch.tensor(starts, dtype=wide, device="cuda")
        junk = [torch.full((1 << 20,), math.nan, device="cuda") for _ in range(8)] + [torch.full((1 << 24,), math.nan, device="cuda")]
        del junk
        out = delta_attention(*leaves, st)
        grads = torch.autograd.grad(out, leaves, (go.cuda(), gs.cuda()))
        for name, x, w in zip(NAMES, (*out, *grads), want):
            ref.near(x, w, K, V, moments, dt, name)
            if name not in ("end state", "state"):
                assert (x.detach().cpu()[outside] == 0).all(), name
    with torch.no_grad():                                     # (and without gradients: other kernels)
        o, e = delta_attention(*[x.cuda() for x in ins], st)
    for name, x, w in zip(NAMES, (o, e), want):
        ref.near(x, w, K, V, moments, dt, name)
    assert (o.cpu()[outside] == 0).all()
