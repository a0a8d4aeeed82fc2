"""The room that the gated delta rule's gradient is given holds what its call needs: no GPU needed."""
from __future__ import annotations

import pytest
import torch

from flyguy_amd._lib import lib
from flyguy_amd.memory_hip import _DELTA, _Corrections

NAMES = [f"{t}{f}" for t in ("q", "k", "v", "go") for f in ("", "_seq", "_moment", "_head")] + [
    "decay", "beta", "ls", "lm", "lh", "bs", "bm", "bh", "state", "starts", "o", "end", "saved", "saved_bytes", "gend", "gq", "gk", "gv", "gl",
    "gb", "gstate", "work", "bytes", "wide", "n", "T", "Hq", "Hk", "K", "V", "type", "scale"]


def dense(heads, width):
    return dict(zip(("_seq", "_moment", "_head"), (heads * width * 4, heads * width, width)))


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("Hq,Hk,K,V", [(32768, 32768, 64, 128), (32768, 1, 128, 64), (65535, 1, 64, 64), (65535, 3, 64, 72), (32768, 2, 16, 128),
                                       (32767, 32767, 128, 128), (8, 8, 64, 64), (8, 4, 33, 7)])
@pytest.mark.parametrize("packed", [0, 256])
def test_room_by_sizes_alone(Hq, Hk, K, V, dt, packed):
    """Asked for without the output's gradient, or by tensors broadcast over moments: as much as dense tensors of these sizes take.
    (From 2^22 values a moment on, the library copies even dense ones.)"""
    base = dict.fromkeys(NAMES, 0) | dict(q=256, k=256, v=256, go=256, decay=256, beta=256, starts=packed, n=1, T=1, Hq=Hq, Hk=Hk, K=K, V=V,
                                          type=dt, scale=1.0)
    sizes = {"q": (Hq, K), "k": (Hk, K), "v": (Hk, V), "go": (Hq, V)}

    def asked(which, backward):
        given = dict(base)
        for t, (heads, width) in sizes.items():
            if t in which:
                given |= {t + f: x for f, x in dense(heads, width).items()}
        return lib().fm_delta_workspace(_DELTA.pack(*[given[n] for n in NAMES]), backward)

    for backward in (0, 1):
        whole = asked("q k v go".split(), backward)
        assert whole > 0
        for which in ([], ["q"], ["q", "k"], ["q", "k", "v"], ["go"]):
            assert asked(which, backward) >= whole, (which, backward)


def test_the_python_side_asks_for_enough(monkeypatch):
    """delta_attention's gradient of 32,768 heads: the room that it caches against what the library wants with the call's own go."""
    from flyguy_amd import memory_hip
    monkeypatch.setattr(memory_hip, "_workspaces", {})
    H, K, V = 32768, 64, 128
    # (strides of dense tensors, without their memory)
    q, v = (torch.empty(0, dtype=torch.bfloat16).as_strided((0, 1, H, d), (H * d, H * d, d, 1)) for d in (K, V))
    gates = torch.empty(0, 1, H)
    p = _Corrections()
    p.starts, p.V, p.state, p.scale = None, V, (1, H, K, V), 1.0
    p.sizes = (0, 1, 1, H, H, K, V, 1)
    rooms = []
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda self, n, dtype=None: rooms.append(n))
    p.room("gradient", q, q, v, gates, gates)
    given = p.pack(q, q, v, gates, gates, go=v)
    assert rooms == [lib().fm_delta_workspace(given, 1)]
