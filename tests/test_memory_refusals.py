"""What the memory operators refuse, and the rotation's tables: no GPU needed."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from flyguy_amd._lib import LibraryError, check, lib
from flyguy_amd.memory_hip import _ATTENTION, _STEP, _TURN, _like, decay_attention, decay_step, norm_rotary, rotary, rotary_table


def test_tables():
    """Angles in 64 bits, rounded once: far positions keep their digits."""
    t = rotary_table(100001, 8)
    a = 100000 * 10000.0 ** (-np.arange(0, 8, 2) / 8)
    assert t.shape == (100001, 4, 2) and t.dtype == torch.float32
    np.testing.assert_array_equal(t[100000].numpy(), np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32))
    np.testing.assert_array_equal(rotary_table(50, 8, scaling="linear", factor=4.0)[40].numpy(), rotary_table(50, 8)[10].numpy())
    # base: the fastest pair as before, the slowest 1 / factor of its angle
    b, p = rotary_table(2, 64, scaling="base", factor=8.0), rotary_table(2, 64)
    angle = lambda x: torch.atan2(x[1, :, 1].double(), x[1, :, 0].double())                       # noqa: E731
    assert abs(float(angle(b)[0] - angle(p)[0])) < 1e-6 and abs(float(angle(b)[-1] * 8 / angle(p)[-1]) - 1) < 1e-3
    # bands: pairs of many turns as before, pairs of less than one divided, the others in between and in order
    n = rotary_table(2, 64, scaling="bands", factor=4.0, taught=2048)
    turns = 2048 * 10000.0 ** (-np.arange(0, 64, 2) / 64) / (2 * math.pi)
    share = (angle(n) / angle(p)).numpy()
    np.testing.assert_allclose(share[turns > 32], 1.0, rtol=1e-5)
    np.testing.assert_allclose(share[turns < 1], 0.25, rtol=1e-3)
    assert (np.diff(share) <= 1e-6).all()
    assert rotary_table(0, 4).shape == (0, 2, 2)


@pytest.mark.parametrize("args", [dict(positions=4, dim=3), dict(positions=4, dim=0), dict(positions=-1, dim=4),
                                  dict(positions=4, dim=4, scaling="other"), dict(positions=4, dim=4, factor=0.0),
                                  dict(positions=4, dim=4, scaling="bands"), dict(positions=4, dim=2, scaling="base", factor=2.0)])
def test_tables_refuse(args):
    with pytest.raises(ValueError):
        rotary_table(**args)


def test_tensors_off_the_gpu():
    q = torch.zeros(1, 2, 3, 4)
    w = torch.ones(4)
    for call in (lambda: rotary(q, q, rotary_table(2, 4)), lambda: norm_rotary(q, q, w, w),
                 lambda: decay_attention(q, q, q, torch.zeros(3)), lambda: decay_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(3),
                                                                                     torch.zeros(1, 3, 4, 4))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_memory_like_a_view():
    """As many values, a head's side by side, whatever view asks."""
    for shape, strides in (((1, 3, 2, 4), (50, 8, 1, 1)), ((2, 5, 3, 64), (40, 3, 1, 1)), ((2, 9, 2, 8), (0, 1, 0, 1)),
                           ((2, 3, 4, 8), (96, 8, 24, 1)), ((2, 3, 4, 1), (12, 4, 1, 7))):
        y = _like(torch.zeros(1000).as_strided(shape, strides))
        assert y.shape == shape and (y.stride(-1) == 1 or shape[-1] == 1) and y.untyped_storage().nbytes() == 4 * y.numel()
    x = torch.zeros(2, 4, 3, 8).transpose(1, 2)
    assert _like(x).stride() == x.stride() and _like(None) is None


def test_forward_mode():
    """A tangent is refused wherever it comes in: it would be dropped."""
    q, w, s, g = torch.zeros(1, 2, 3, 4), torch.ones(4), torch.zeros(1, 3, 4, 4), torch.zeros(3)
    table = rotary_table(2, 4)
    calls = {"rotary": (rotary, [q, q, table], (0, 1, 2)), "norm_rotary": (norm_rotary, [q, q, w, w, table], range(5)),
             "decay_attention": (decay_attention, [q, q, q, g, s], range(5)),
             "decay_step": (decay_step, [q[:, 0], q[:, 0], q[:, 0], g, s], range(5))}
    for name, (f, args, places) in calls.items():
        for i in places:
            with forward_ad.dual_level():
                given = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(args)]
                with pytest.raises(RuntimeError, match=f"{name}: has no forward-mode"):
                    f(*given)

            def at(x):
                return f(*[x if j == i else y for j, y in enumerate(args)])
            with pytest.raises(RuntimeError, match=f"{name}: has no forward-mode"):
                torch.func.jvp(at, (args[i],), (torch.ones_like(args[i]),))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="GPU"):      # (no tangent among them)
        rotary(q, q, table)


def refuses(name, args):
    assert getattr(lib(), name)(args, None) == -1
    with pytest.raises(LibraryError, match=name):
        check()


TURN = ["xq", "qs", "qm", "qh", "xk", "ks", "km", "kh", "yq", "a", "b", "c", "yk", "d", "e", "f", "gq", "g", "h", "i", "gk", "j",
        "k", "l", "wq", "wk", "gwq", "gwk", "partial", "table", "positions", "pos_seq", "pos_moment", "first", "wide", "Hq",
        "Hk", "N", "T", "D", "R", "interleaved", "P", "type", "eps"]


def turn(**given):
    v = dict.fromkeys(TURN, 0) | dict(xq=256, xk=256, yq=256, yk=256, gq=256, gk=256, Hq=2, Hk=1, N=1, T=1, D=8, eps=1e-6)
    return _TURN.pack(*[(v | given)[n] for n in TURN])


@pytest.mark.parametrize("given", [dict(type=3), dict(type=-1), dict(N=-1), dict(D=0), dict(D=513), dict(R=3, table=256, P=1),
                                   dict(R=10, table=256, P=1), dict(R=4), dict(xq=0), dict(yk=0), dict(N=1 << 36, T=1 << 36)])
def test_the_library_refuses_turns(given):
    refuses("fm_turn", turn(**given))


def test_the_library_refuses_turns_gradients():
    refuses("fm_turn_bwd", turn(gq=0))
    refuses("fm_turn_bwd", turn(wq=256, xq=0))
    refuses("fm_turn_bwd", turn(wq=256, gwq=256))
    refuses("fm_turn_bwd", turn(gwq=256, partial=256))


def attention(**given):
    names = [f"{t}{f}" for t in ("q", "k", "v", "go") for f in ("", "_seq", "_moment", "_head")]
    names += ["decay", "state", "starts", "o", "end", "gend", "gq", "gk", "gv", "gstate", "work", "bytes", "wide", "n", "T", "Hq",
              "Hk", "K", "V", "type", "scale"]
    v = dict.fromkeys(names, 0) | dict(q=256, k=256, v=256, go=256, decay=256, o=256, end=256, n=1, T=4, Hq=2, Hk=1, K=8, V=8,
                                       scale=1.0)
    return _ATTENTION.pack(*[(v | given)[n] for n in names])


@pytest.mark.parametrize("given", [dict(type=3), dict(Hq=3, Hk=2), dict(Hq=0), dict(Hk=0), dict(K=0), dict(K=129), dict(V=129),
                                   dict(n=-1), dict(n=20000), dict(T=-1), dict(q=0), dict(o=0), dict(decay=0),
                                   dict(state=256, end=256)])
def test_the_library_refuses_attention(given):
    refuses("fm_attention", attention(**given))


def test_the_library_refuses_packed_moments_without_an_output():
    refuses("fm_attention", attention(n=0, starts=256, o=0))


def test_the_library_refuses_states_that_share_memory():
    refuses("fm_attention", attention(state=256, end=512))
    refuses("fm_attention", attention(state=512, end=256))
    refuses("fm_step", step(state=256, next=768))
    refuses("fm_step", step(state=768, next=256))


def test_the_library_refuses_attention_gradients():
    refuses("fm_attention_bwd", attention(go=0, gk=256))
    refuses("fm_attention_bwd", attention(gk=256))                         # shared heads: a workspace is needed
    refuses("fm_attention_bwd", attention(gk=256, work=256, bytes=16))


def step(**given):
    names = [f"{t}{f}" for t in ("q", "k", "v") for f in ("", "_seq", "_moment", "_head")]
    names += ["decay", "state", "next", "slots", "o", "n", "states", "Hq", "Hk", "K", "V", "type", "scale"]
    v = dict.fromkeys(names, 0) | dict(q=256, k=256, v=256, decay=256, state=256, next=256, o=256, n=2, states=2, Hq=2, Hk=1,
                                       K=8, V=8, scale=1.0)
    return _STEP.pack(*[(v | given)[n] for n in names])


@pytest.mark.parametrize("given", [dict(type=7), dict(Hq=3, Hk=2), dict(K=0), dict(V=200), dict(n=-1), dict(n=70000), dict(k=0),
                                   dict(state=0), dict(states=1), dict(states=-1)])
def test_the_library_refuses_steps(given):
    refuses("fm_step", step(**given))
