"""Rows of cosines and sines for the rotation kernel, on the CPU."""

import math

import pytest
import torch

from smaq_b200 import ops


def test_rope_table():
    """Frequencies on the CPU: plain, linear, ntk; yarn keeps fast pairs and divides slow ones."""
    t = ops.rope_table(50, 8, 100.0, device="cpu")
    for p in (0, 7, 49):
        for i in range(4):
            a = p * 100.0 ** (-2 * i / 8)
            assert abs(t[p, i] - math.cos(a)) < 1e-6 and abs(t[p, 4 + i] - math.sin(a)) < 1e-6
    assert torch.equal(ops.rope_table(50, 8, 100.0, linear=2.0, device="cpu")[::2], t[:25])
    assert torch.allclose(ops.rope_table(50, 8, 100.0, ntk=2.0, device="cpu"), ops.rope_table(50, 8, 100.0 * 2 ** (8 / 6), device="cpu"))
    y = ops.rope_table(200, 64, 10000.0, yarn=dict(factor=4.0, original=4096, attention=1.0), device="cpu")
    plain = ops.rope_table(200, 64, 10000.0, device="cpu")
    slow = ops.rope_table(200, 64, 10000.0, linear=4.0, device="cpu")
    assert torch.allclose(y[:, 0], plain[:, 0], atol=1e-6) and torch.allclose(y[:, 63], slow[:, 63], atol=1e-6)
    z = ops.rope_table(3, 64, yarn=dict(factor=4.0, original=4096), device="cpu")
    assert abs(float(z[0, 0]) - (0.1 * math.log(4) + 1)) < 1e-6
    for bad in (dict(max_positions=0, rotary_dim=8), dict(max_positions=4, rotary_dim=7), dict(max_positions=4, rotary_dim=8, linear=0)):
        with pytest.raises(ValueError):
            ops.rope_table(**bad, device="cpu")
