"""What layer norm and dropout refuse, and the generator's published numbers: no GPU needed."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from flyguy_amd._lib import LibraryError, check, lib
from flyguy_amd.rows_hip import _DROP, _NORM, dropout, layer_norm
from rows_helpers import philox


def test_the_generators_published_numbers():
    """The three known answers of philox4x32-10 that its authors publish with it (counter, key, result)."""
    for c, k, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                       ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                       ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                        (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = philox([c[0] | c[1] << 32], c[2] | c[3] << 32, k[0] | k[1] << 32)
        assert tuple(int(x) for x in got[0]) == want


def test_off_the_gpu():
    x, c = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: layer_norm(x), lambda: dropout(x, 0.5, c)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_forward_mode():
    x, w, c = torch.zeros(2, 8), torch.ones(8), torch.zeros(2, dtype=torch.int64)
    with forward_ad.dual_level():
        d, e = forward_ad.make_dual(x, x), forward_ad.make_dual(w, w)
        for f in (lambda: layer_norm(d), lambda: layer_norm(x, e), lambda: layer_norm(x, w, e), lambda: dropout(d, 0.5, c)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()


def refuses(name, args):
    assert getattr(lib(), name)(args, None) == -1
    with pytest.raises(LibraryError, match=name):
        check()


NORM = ["x", "y", "g", "gx", "x_row", "y_row", "g_row", "gx_row", "weight", "bias", "gweight", "gbias", "stats", "partial",
        "rows", "width", "type", "eps"]


def norm(**given):
    v = dict.fromkeys(NORM, 0) | dict(x=256, y=256, g=256, gx=256, stats=256, x_row=8, y_row=8, g_row=8, gx_row=8, rows=2, width=8,
                                      eps=1e-5)
    return _NORM.pack(*[(v | given)[n] for n in NORM])


@pytest.mark.parametrize("given", [dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 41), dict(width=0),
                                   dict(width=(1 << 24) + 1), dict(x=0), dict(y=0), dict(eps=-1.0), dict(eps=float("nan"))])
def test_the_library_refuses_norms(given):
    refuses("fm_norm", norm(**given))


@pytest.mark.parametrize("given", [dict(g=0), dict(stats=0), dict(gweight=256), dict(gbias=256), dict(x=0)])
def test_the_library_refuses_norms_gradients(given):
    refuses("fm_norm_bwd", norm(**given))


@pytest.mark.parametrize("given", [dict(type=5), dict(rows=-1), dict(width=-1), dict(rows=1 << 39, width=1 << 39), dict(share=-0.1),
                                   dict(share=1.01), dict(share=float("nan")), dict(x=0), dict(y=0), dict(counter=0)])
def test_the_library_refuses_dropout(given):
    v = dict(x=256, y=256, counter=256, x_row=8, rows=2, width=8, type=0, share=0.5) | given
    refuses("fm_drop", _DROP.pack(*[v[n] for n in ("x", "y", "counter", "x_row", "rows", "width", "type", "share")]))
