"""What the gated delta rule refuses: no GPU needed."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from flyguy_amd._lib import LibraryError, check, lib
from flyguy_amd.memory_hip import _DELTA, _DELTA_STEP, _units, delta_attention, delta_step


def test_off_the_gpu():
    q, g, s = torch.zeros(1, 2, 3, 4), torch.zeros(1, 2, 3), torch.zeros(1, 3, 4, 4)
    for call in (lambda: delta_attention(q, q, q, g, g), lambda: delta_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_forward_mode():
    q, g, s = torch.zeros(1, 2, 3, 4), torch.zeros(1, 2, 3), torch.zeros(1, 3, 4, 4)
    calls = {"delta_attention": (delta_attention, [q, q, q, g, g, s]),
             "delta_step": (delta_step, [q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s])}
    for name, (f, args) in calls.items():
        for i in range(6):
            with forward_ad.dual_level():
                given = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(args)]
                with pytest.raises(RuntimeError, match=f"{name}: has no forward-mode"):
                    f(*given)


def test_whole_units():
    """Tensors that the library can load as they are stay; others of whole 16-byte units are copied; the rest is its own matter."""
    x = torch.zeros(2, 5, 3, 8)
    assert _units(x) is x
    wide = torch.zeros(2, 5, 30)
    for y in (wide[..., 3:27].unflatten(-1, (3, 8)), x.transpose(-1, -2).contiguous().transpose(-1, -2),
              wide[..., 1:25].unflatten(-1, (3, 8))):
        z = _units(y)
        assert z is not y and z.is_contiguous() and torch.equal(z, y)
    odd = wide[..., 3:24].unflatten(-1, (3, 7))
    assert _units(odd) is odd


def refuses(name, args):
    assert getattr(lib(), name)(args, None) == -1
    with pytest.raises(LibraryError, match=name):
        check()


NAMES = [f"{t}{f}" for t in ("q", "k", "v", "go") for f in ("", "_seq", "_moment", "_head")] + [
    "decay", "beta", "ls", "lm", "lh", "bs", "bm", "bh", "state", "starts", "o", "end", "saved", "saved_bytes", "gend", "gq", "gk", "gv", "gl",
    "gb", "gstate", "work", "bytes", "wide", "n", "T", "Hq", "Hk", "K", "V", "type", "scale"]


def delta(**given):
    v = dict.fromkeys(NAMES, 0) | dict(q=256, k=256, v=256, go=256, decay=256, beta=256, o=256, end=256, work=256, bytes=1 << 40,
                                       saved=256, saved_bytes=1 << 40, n=1, T=4, Hq=2, Hk=1, K=8, V=8, scale=1.0)
    return _DELTA.pack(*[(v | given)[n] for n in NAMES])


@pytest.mark.parametrize("given", [dict(type=3), dict(type=-1), dict(Hq=3, Hk=2), dict(Hq=0), dict(Hk=0), dict(K=0), dict(K=129), dict(V=0),
                                   dict(V=129), dict(n=-1), dict(n=20000), dict(T=-1), dict(T=(1 << 31) + 1), dict(n=16384, T=1 << 31),
                                   dict(q=0), dict(k=0), dict(v=0), dict(o=0), dict(decay=0), dict(beta=0), dict(state=256),
                                   dict(work=0), dict(bytes=64), dict(saved_bytes=64)])
def test_the_library_refuses(given):
    refuses("fm_delta", delta(**given))


@pytest.mark.parametrize("given", [dict(go=0), dict(saved=0), dict(work=0), dict(bytes=64), dict(saved_bytes=64), dict(K=200)])
def test_the_library_refuses_gradients(given):
    refuses("fm_delta_bwd", delta(**given))


def test_no_arguments():
    for name in ("fm_delta", "fm_delta_bwd", "fm_delta_step"):
        refuses(name, None)
    assert lib().fm_delta_workspace(None, 0) == 0 and lib().fm_delta_saved(None) == 0
    assert lib().fm_delta_workspace(delta(K=0), 0) == 0


def test_workspaces_hold_what_they_must():
    """Never less than the tensors that go there, for many sizes, alike and packed; and the same for any strides that need no copy."""
    for T in (1, 31, 32, 33, 64, 65, 700, 5000, 40000):
        for n in (1, 3, 60):
            for dt, chunk in ((0, 32), (1, 64), (2, 32)):
                for packed in (0, 256):
                    for K, V in ((8, 8), (72, 128)):
                        a = dict(T=T, n=n, type=dt, starts=packed, K=K, V=V, Hq=4, Hk=2)
                        slots = (T // chunk + n if T > chunk else n) if packed else n * -(-T // chunk)
                        states = slots * 4 * (64 if K <= 64 else 128) * (64 if V <= 64 else 128) * 4
                        saved = lib().fm_delta_saved(delta(**a))
                        assert saved >= states and lib().fm_delta_workspace(delta(**a), 0) > 0
                        assert lib().fm_delta_workspace(delta(**a), 1) >= states
                        assert lib().fm_delta_workspace(delta(**a, q_head=512, k_head=64), 1) == lib().fm_delta_workspace(delta(**a), 1)


STEP = [f"{t}{f}" for t in ("q", "k", "v") for f in ("", "_seq", "_moment", "_head")] + [
    "decay", "beta", "lr", "lh", "br", "bh", "state", "next", "slots", "o", "n", "states", "Hq", "Hk", "K", "V", "type", "scale"]


@pytest.mark.parametrize("given", [dict(type=7), dict(Hq=3, Hk=2), dict(K=0), dict(V=200), dict(n=-1), dict(n=70000), dict(k=0), dict(beta=0),
                                   dict(decay=0), dict(state=0), dict(next=0), dict(o=0), dict(states=1), dict(states=-1),
                                   dict(state=256, next=768), dict(state=768, next=256)])
def test_the_library_refuses_steps(given):
    v = dict.fromkeys(STEP, 0) | dict(q=256, k=256, v=256, decay=256, beta=256, state=256, next=256, o=256, n=2, states=2, Hq=2, Hk=1,
                                      K=8, V=8, scale=1.0)
    refuses("fm_delta_step", _DELTA_STEP.pack(*[(v | given)[n] for n in STEP]))
