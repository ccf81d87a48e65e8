"""CPU: the tables of the position rotation."""
from __future__ import annotations

import math

import pytest


@pytest.mark.parametrize("rotary", [0, 2, 64])
def test_angles(rotary):
    from kbb200 import lm

    cos, sin = lm.rope_tables(5, rotary, base=100.0, device="cpu")
    assert cos.shape == sin.shape == (5, rotary // 2)
    for p in range(5):
        for i in range(rotary // 2):
            angle = p * 100.0 ** (-2 * i / rotary)
            assert abs(float(cos[p, i]) - math.cos(angle)) < 1e-7 and abs(float(sin[p, i]) - math.sin(angle)) < 1e-7


@pytest.mark.parametrize("rotary", [1, 5, 65, -2])
def test_half_a_pair_is_refused(rotary):
    """An odd size made tables for one element more, which then turned with the rest."""
    from kbb200 import lm

    with pytest.raises(RuntimeError, match="even"):
        lm.rope_tables(5, rotary, device="cpu")
