"""Host-only check of the feed-forward oracle's gate functions far from zero, against the
standard library's."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import ffn as off


@pytest.mark.parametrize("z", [-30.0, -10.0, -8.5, -5.0, -1.0, 0.0, 2.0, 10.0])
def test_gelu_keeps_its_digits_in_both_tails(z):
    cdf = math.erfc(-z / math.sqrt(2)) / 2
    density = math.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    # 64 bits and an erfc of a few ulp, its argument's rounding times z^2 under 2^10
    assert off.gate(torch.tensor(z, dtype=torch.float64), "gelu").item() == pytest.approx(z * cdf, rel=2.0 ** -40, abs=0)
    slope = off.slope(torch.tensor(z, dtype=torch.float64), "gelu").item()
    assert slope == pytest.approx(cdf + z * density, rel=2.0 ** -30, abs=0)
