"""Refusals of the operators over a paged cache in 8 bits, on the CPU (no kernel is launched)."""

from __future__ import annotations

import os

import pytest
import torch

from streamindex_amd import _lib, paged_write_q
from streamindex_amd.build import LIB_PATH

FAKE = 0x1000  # never dereferenced: every call fails its checks, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB_PATH):
        pytest.skip("libstreamindex.so not built (run __graft_entry__.build())")
    return _lib.load()


def test_cpu_tensors_are_refused():
    with pytest.raises(AssertionError):
        paged_write_q(torch.zeros(4, 64), torch.zeros(2, 4, 64).to(torch.float8_e4m3fn), torch.zeros(2, 4),
                      torch.zeros(4, dtype=torch.int64))


def write(lib, rows=FAKE, rs=64, dtype=1, slots=FAKE, n=4, D=64, codes=FAKE, ps=256, ss=64, scales=FAKE, sst=4, pages=2, page=4, block=1):
    return lib.si_paged_write_q(rows, rs, dtype, slots, n, D, codes, ps, ss, scales, sst, pages, page, block, None)


@pytest.mark.parametrize("kw,word,rc", [
    ({"dtype": 3}, b"dtype", 2), ({"dtype": -1}, b"dtype", 2), ({"n": -1}, b"dimension", 1), ({"D": 0}, b"dimension", 1),
    ({"pages": -1}, b"dimension", 1), ({"page": 0}, b"dimension", 1), ({"block": 0}, b"dimension", 1), ({"block": 3}, b"dimension", 1),
    ({"rs": -1}, b"dimension", 1), ({"n": 1 << 31}, b"int32", 2), ({"D": (1 << 20) + 1, "ss": 1 << 21}, b"width", 2),
    ({"pages": 1 << 31}, b"int32", 2), ({"rows": None}, b"null", 1), ({"slots": None}, b"null", 1), ({"codes": None}, b"null", 1),
    ({"scales": None}, b"null", 1), ({"ss": 63}, b"overlap", 1), ({"ps": 255}, b"overlap", 1), ({"sst": 3}, b"overlap", 1),
])
def test_write_refusals(lib, kw, word, rc):
    assert write(lib, **kw) == rc and word in lib.si_last_error(), lib.si_last_error()


def test_nothing_to_write(lib):
    assert write(lib, n=0, rows=None, slots=None, codes=None, scales=None) == 0
    assert write(lib, pages=0, codes=None, scales=None) == 0
