"""Refusals of the paged serving operators, on the CPU (no kernel is launched)."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from streamindex_amd import _lib, paged_attn_fwd, paged_compress, paged_plan, paged_write
from streamindex_amd.build import LIB_PATH

FAKE = 0x1000  # never dereferenced: every call fails its checks, or has nothing to do


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB_PATH):
        pytest.skip("libstreamindex.so not built (run __graft_entry__.build())")
    return _lib.load()


def test_cpu_tensors_are_refused():
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        paged_plan(z, z, torch.zeros(2, 3, dtype=torch.int32), z, 16, 4)
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        paged_write(x[0], x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(AssertionError):
        paged_compress(x, x, torch.zeros(4, 64), z.view(1, 2), z, z, x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(AssertionError):
        paged_attn_fwd(x, x, z.view(1, 2), z, z[:1], torch.zeros(4))


def plan(lib, R=4, ratio=1, tstride=8, P=8, F=5, page=16, rows=10, table=FAKE, cu=FAKE, free=FAKE, slots=FAKE):
    return lib.si_paged_plan(FAKE, FAKE, R, ratio, table, tstride, P, free, F, None, page, rows, cu, FAKE, slots, FAKE, FAKE,
                             FAKE, None)


@pytest.mark.parametrize("kw,word,rc", [
    ({"ratio": 0}, b"dimension", 1), ({"page": 0}, b"dimension", 1), ({"rows": -1}, b"dimension", 1), ({"R": -1}, b"dimension", 1),
    ({"rows": 1 << 31}, b"int32", 2), ({"page": 1 << 31}, b"int32", 2), ({"tstride": 7}, b"overlap", 1),
    ({"table": None}, b"null", 1), ({"cu": None}, b"null", 1), ({"free": None}, b"null", 1), ({"slots": None}, b"null", 1),
])
def test_plan_refusals(lib, kw, word, rc):
    assert plan(lib, **kw) == rc and word in lib.si_last_error()


def test_write_refusals(lib):
    call = lambda *a: lib.si_paged_write(*a, None)  # noqa: E731
    assert call(FAKE, 8, FAKE, -1, 8, FAKE, 64, 8, 2, 8) == 1
    assert call(FAKE, 8, FAKE, 4, 8, FAKE, 64, 8, 2, 0) == 1
    assert call(FAKE, -8, FAKE, 4, 8, FAKE, 64, 8, 2, 8) == 1
    assert call(None, 8, FAKE, 4, 8, FAKE, 64, 8, 2, 8) == 1 and b"null" in lib.si_last_error()
    assert call(FAKE, 8, FAKE, 1 << 31, 8, FAKE, 64, 8, 2, 8) == 2
    assert call(None, 8, None, 0, 8, None, 64, 8, 2, 8) == 0  # nothing to do


def compress(lib, dtype=1, pages=2, ps=4, C=64, m=4, R=1, P=2, E=3, out_pages=2, ca=FAKE, cb=None, cb_strides=None,
             strides=i64(256, 64, 1), out_strides=i64(256, 64, 1), slots=FAKE):
    return lib.si_paged_compress(ca, strides, FAKE, i64(256, 64, 1), FAKE, cb, cb_strides, None, None, None, dtype, pages, ps, C,
                                 m, FAKE, P, R, P, FAKE, FAKE, slots, E, FAKE, out_strides, out_pages, 4, None)


@pytest.mark.parametrize("kw,rc", [
    ({"m": 0}, 1), ({"ps": 0}, 1), ({"E": -1}, 1), ({"dtype": 3}, 2), ({"C": 1 << 31}, 2), ({"ca": None}, 1), ({"slots": None}, 1),
    ({"cb": FAKE}, 1), ({"cb": FAKE, "cb_strides": i64(256, 64, 1)}, 1), ({"strides": None}, 1), ({"strides": i64(256, 64, 2)}, 1),
    ({"out_strides": i64(256, -64, 1)}, 1),
])
def test_compress_refusals(lib, kw, rc):
    assert compress(lib, **kw) == rc


def attn(lib, N=3, H=4, D=64, R=2, window=0, ratio=0, qs=i64(256, 64, 1), ks=i64(1024, 64, 1), pages=5, ps=16, P=4, q=FAKE,
         kv=FAKE, kv2=FAKE, ks2=i64(1024, 64, 1), dtype=0, table=FAKE, cu=FAKE, scratch=None, o=FAKE):
    return lib.si_paged_attn_fwd(q, qs, kv, ks, pages, ps, table, P, P, kv2, ks2, 5, 16, FAKE, 4, 4, window, ratio, cu, FAKE, FAKE,
                                 N, H, D, R, 0.125, dtype, o, FAKE, scratch, 0, None)


@pytest.mark.parametrize("kw,word,rc", [
    ({"D": 96}, b"head dim", 2), ({"dtype": 2}, b"qkv_dtype", 1), ({"H": 0}, b"dimension", 1), ({"window": -1}, b"dimension", 1),
    ({"N": 1 << 30, "H": 4}, b"int32", 2), ({"qs": i64(256, 60, 1)}, b"multiples of 8", 1), ({"qs": i64(256, 64, 2)}, b"contiguous", 1),
    ({"q": None}, b"null", 1), ({"cu": None}, b"null", 1), ({"table": None}, b"null", 1), ({"kv": None}, b"null", 1),
    ({"kv": FAKE + 8}, b"alignment", 1), ({"o": FAKE + 8}, b"aligned", 1), ({"scratch": FAKE + 8}, b"aligned", 1),
    ({"ks": i64(1024, 64, 2)}, b"contiguous", 1), ({"ks": i64(1020, 64, 1)}, b"16-byte", 1), ({"ps": 0}, b"dimension", 1),
    ({"pages": 5, "ks": i64(1 << 33, 64, 1)}, b"64 GiB", 2), ({"pages": 1 << 30, "ks": i64(1 << 40, 64, 1)}, b"64 GiB", 2),
    ({"pages": 1 << 31}, b"int32", 2), ({"ratio": 4, "ks2": None}, b"kv2", 1), ({"ratio": 4, "kv2": None}, b"kv2", 1),
])
def test_attn_refusals(lib, kw, word, rc):
    assert attn(lib, **kw) == rc and word in lib.si_last_error(), lib.si_last_error()


def test_attn_scratch(lib):
    need = lib.si_paged_attn_fwd_scratch_bytes
    assert need(1, 64, 576, 1, 128, 64 * 64, 64 * 64) > 0
    assert need(1, 64, 576, 1, 0, 128, 0) == 0  # four tiles: never split
    assert need(0, 64, 576, 1, 0, 4096, 0) == 0 and need(4, 64, 96, 1, 0, 4096, 0) == 0
    # bounded whatever the lengths
    assert 0 < need(1 << 20, 64, 576, 64, 0, 1 << 40, 1 << 40) < 1 << 28
