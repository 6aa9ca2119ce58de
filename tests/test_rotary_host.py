"""Frequencies and refusals of the norm and rotation, on the CPU (no kernel is launched)."""

from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from streamindex_amd import _lib, norm_rotary, rotary, rotary_freqs
from streamindex_amd.build import LIB_PATH

FAKE = 0x1000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB_PATH):
        pytest.skip("libstreamindex.so not built (run __graft_entry__.build())")
    return _lib.load()


def test_frequencies():
    f = rotary_freqs(64, 10000.0, device="cpu")
    assert f.dtype is torch.float64 and f.shape == (32,)
    assert torch.allclose(f, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    g = rotary_freqs(64, 10000.0, factor=16.0, original_length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    ratio = f / g
    assert (ratio[turns > 40] == 1).all() and torch.allclose(ratio[turns < 0.7], torch.tensor(16.0, dtype=torch.float64))
    assert (ratio[1:] >= ratio[:-1] - 1e-12).all() and ((ratio > 1.01) & (ratio < 15.9)).any()
    assert rotary_freqs(0, device="cpu").shape == (0,)
    for bad in ({"dims": 3}, {"dims": -2}, {"dims": 4, "base": 0.0}, {"dims": 4, "factor": 0.5}, {"dims": 4, "fast": 1.0, "slow": 1.0},
                {"dims": 4, "original_length": 0}):
        with pytest.raises(ValueError):
            rotary_freqs(**bad, device="cpu")


def test_cpu_tensors_are_refused():
    x, p, f = torch.zeros(3, 2, 8), torch.zeros(3, dtype=torch.int32), rotary_freqs(8, device="cpu")
    with pytest.raises(AssertionError):
        rotary(x, p, f)
    with pytest.raises(AssertionError):
        norm_rotary(x, p, f)
    with pytest.raises(ValueError):
        norm_rotary(x, p, f, eps=-1.0)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def fwd(lib, x=FAKE, xs=i64(128, 64), norm=1, weight=None, pos=FAKE, npos=4, freqs=FAKE, pairs=16, start=32, T=4, H=2, D=64, dtype=1,
        y=FAKE):
    return lib.si_norm_rotary(x, xs, norm, weight, 1e-6, pos, 0, npos, freqs, pairs, start, 0, 1.0, 0, T, H, D, dtype, y, None)


def bwd(lib, dy=FAKE, ds=i64(128, 64), x=FAKE, xs=i64(128, 64), weight=None, pos=FAKE, npos=4, freqs=FAKE, pairs=16, start=32, T=4, H=2,
        D=64, dtype=1, dx=FAKE, dw=None, ws=None, size=0):
    return lib.si_norm_rotary_bwd(dy, ds, x, xs, weight, 1e-6, pos, 0, npos, freqs, pairs, start, 0, 1.0, 0, T, H, D, dtype, dx, dw, ws,
                                  size, None)


BAD = [({"dtype": 3}, 2), ({"T": -1}, 1), ({"H": 0}, 1), ({"D": 0}, 1), ({"D": 1025}, 2), ({"pairs": 33}, 1), ({"start": 33}, 1),
       ({"start": -1}, 1), ({"pairs": -1}, 1), ({"T": 1 << 40}, 2), ({"H": 1 << 31}, 2), ({"xs": None}, 1), ({"x": None}, 1),
       ({"pos": None}, 1), ({"freqs": None}, 1), ({"npos": 3}, 1), ({"npos": 0}, 1)]


@pytest.mark.parametrize("kw,rc", BAD + [({"y": None}, 1), ({"norm": 0, "weight": FAKE}, 1)])
def test_forward_refusals(lib, kw, rc):
    assert fwd(lib, **kw) == rc and lib.si_last_error()


@pytest.mark.parametrize("kw,rc", BAD + [({"dx": None}, 1), ({"dy": None}, 1), ({"ds": None}, 1), ({"dw": FAKE}, 1),
                                         ({"dw": FAKE, "ws": FAKE, "size": 255}, 1)])
def test_backward_refusals(lib, kw, rc):
    assert bwd(lib, **kw) == rc and lib.si_last_error()


def test_nothing_to_do(lib):
    assert fwd(lib, T=0, x=None, y=None, pos=None, freqs=None) == 0
    assert bwd(lib, T=0, x=None, dx=None, dy=None, pos=None, freqs=None) == 0


def test_workspace(lib):
    need = lib.si_norm_rotary_bwd_workspace_bytes
    assert need(4, 2, 64, 16) >= 64 * 4
    assert need(0, 2, 64, 16) == need(4, 2, 2000, 16) == need(4, 2, 64, 33) == 0
    assert need(1 << 20, 64, 576, 32) < 1 << 28
