"""Stretched frequencies at contexts and bases where the share of no pair, or of every pair, is between the two (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from streamindex_amd import rotary_freqs


@pytest.mark.parametrize("dims", [2, 8, 64, 128])
@pytest.mark.parametrize("base", [1.5, 100.0, 10000.0, 1e6])
@pytest.mark.parametrize("length,fast,slow", [
    (1, 32.0, 1.0), (3, 32.0, 1.0), (6, 32.0, 1.0), (7, 32.0, 1.0), (100, 32.0, 1.0), (4096, 32.0, 1.0), (4096, 2000.0, 700.0), (4096, 651.0, 650.0),
    (10**9, 32.0, 1.0), (4096, 1e-3, 1e-4)])
def test_few_and_many_turns(dims, base, length, fast, slow):
    """Pairs that turn fewer than `slow` times are divided by the factor, those that turn more than `fast` times stay, others are between."""
    f = rotary_freqs(dims, base, device="cpu")
    g = rotary_freqs(dims, base, factor=16.0, original_length=length, fast=fast, slow=slow, device="cpu")
    ratio, turns = f / g, length * f / (2 * math.pi)
    assert (ratio[turns > fast * (1 + 1e-9)] == 1).all()
    assert torch.allclose(ratio[turns < slow * (1 - 1e-9)], torch.tensor(16.0, dtype=torch.float64), rtol=1e-12)
    assert ((ratio >= 1) & (ratio <= 16 * (1 + 1e-12))).all() and (ratio[1:] >= ratio[:-1] - 1e-12).all()


def test_a_base_that_orders_no_pairs_is_refused():
    for base in (1.0, 0.5):
        assert rotary_freqs(8, base, device="cpu").shape == (4,)
        with pytest.raises(ValueError):
            rotary_freqs(8, base, factor=2.0, device="cpu")
    for bad in ({"base": math.nan}, {"factor": math.nan}, {"factor": math.inf}, {"base": math.inf}):
        with pytest.raises(ValueError):
            rotary_freqs(**{"dims": 8, "base": 100.0, "factor": 2.0, **bad}, device="cpu")
