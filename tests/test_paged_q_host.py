"""Refusals of the operators over a paged cache in 8 bits, on the CPU (no kernel is launched)."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from streamindex_amd import _lib, paged_attn_q_fwd, paged_write_q
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
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        paged_attn_q_fwd(torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 64).to(torch.float8_e4m3fn), torch.zeros(2, 4),
                         z.view(1, 2), z, z[:1], torch.zeros(4))


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


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def attn(lib, N=3, H=4, D=64, R=2, window=0, ratio=0, qs=i64(256, 64, 1), ks=i64(1024, 64, 1), pages=5, ps=16, P=4, q=FAKE, kv=FAKE,
         kv2=FAKE, ks2=i64(1024, 64, 1), dtype=0, table=FAKE, cu=FAKE, scratch=None, o=FAKE, scales=FAKE, sst=16, block=1, scales2=FAKE,
         sst2=16, block2=1):
    return lib.si_paged_attn_q_fwd(q, qs, kv, ks, scales, sst, block, pages, ps, table, P, P, kv2, ks2, scales2, sst2, block2, 5, 16, FAKE, 4,
                                   4, window, ratio, cu, FAKE, FAKE, N, H, D, R, 0.125, dtype, o, FAKE, scratch, 0, None)


@pytest.mark.parametrize("kw,word,rc", [
    ({"D": 96}, b"head dim", 2), ({"dtype": 2}, b"qkv_dtype", 1), ({"H": 0}, b"dimension", 1), ({"window": -1}, b"dimension", 1),
    ({"N": 1 << 30, "H": 4}, b"int32", 2), ({"qs": i64(256, 60, 1)}, b"multiples of 8", 1), ({"qs": i64(256, 64, 2)}, b"contiguous", 1),
    ({"q": None}, b"null", 1), ({"cu": None}, b"null", 1), ({"table": None}, b"null", 1), ({"kv": None}, b"null", 1),
    ({"kv": FAKE + 8}, b"alignment", 1), ({"o": FAKE + 8}, b"aligned", 1), ({"scratch": FAKE + 8}, b"aligned", 1),
    ({"ks": i64(1024, 64, 2)}, b"contiguous", 1), ({"ks": i64(1024, 72, 1)}, b"16-byte", 1), ({"ps": 0}, b"dimension", 1),
    ({"pages": 5, "ks": i64(1 << 34, 64, 1)}, b"64 GiB", 2), ({"pages": 1 << 30, "ks": i64(1 << 40, 64, 1)}, b"64 GiB", 2),
    ({"pages": 1 << 31}, b"int32", 2), ({"ratio": 4, "ks2": None}, b"kv2", 1), ({"ratio": 4, "kv2": None}, b"kv2", 1),
    ({"block": 0}, b"block", 1), ({"block": 3}, b"block", 1), ({"block": 32}, b"block", 1), ({"sst": -1}, b"scale stride", 1),
    ({"scales": None}, b"scales", 1), ({"ratio": 4, "block2": 5}, b"kv2: the block", 1), ({"ratio": 4, "scales2": None}, b"kv2", 1),
    ({"R": (1 << 30) + 1}, b"2^30", 2),
])
def test_attn_refusals(lib, kw, word, rc):
    assert attn(lib, **kw) == rc and word in lib.si_last_error(), lib.si_last_error()


def test_attn_scratch(lib):
    need = lib.si_paged_attn_q_fwd_scratch_bytes
    assert need(1, 64, 576, 1, 128, 64 * 64, 64 * 64) > 0
    assert need(1, 64, 576, 1, 0, 128, 0) == 0  # two tiles: never split
    assert need(0, 64, 576, 1, 0, 4096, 0) == 0 and need(4, 64, 96, 1, 0, 4096, 0) == 0
    # bounded whatever the lengths
    assert 0 < need(1 << 20, 64, 576, 64, 0, 1 << 40, 1 << 40) < 1 << 28
