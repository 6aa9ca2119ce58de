"""Refusals of the paged serving operators at the ends of their sizes, on the CPU (no kernel is launched)."""

from __future__ import annotations

from tests.test_paged_host import attn, lib, plan  # noqa: F401


def test_requests(lib):  # noqa: F811
    """2^31 - 1 requests fit 32 bits, but a thread's share of them would end past it."""
    for R in ((1 << 30) + 1, (1 << 31) - 1):
        assert plan(lib, R=R) == 2 and b"requests" in lib.si_last_error()
        assert attn(lib, R=R) == 2 and b"requests" in lib.si_last_error()
    assert attn(lib, N=0, R=1 << 30) == 0  # nothing to do
