"""The rotation at positions up to the documented limit: its cosines and sines alone
(vectors of a 1 and a 0), against the exact angle reduced in whole numbers.

Bound: 2 u for the series and the reduction, u = 2^-24 for the product with 1."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from conftest import announce
from sbq.state import qk_norm_rope

U = 2.0 ** -24
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def _turn(pos, f):
    angle = Fraction(int(pos)) * Fraction(float(f))
    x = float(angle - TWO_PI * (angle // TWO_PI))
    return np.cos(x), np.sin(x)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 17, 30, 40, 47, 49, 50, 51, 52, 53])
def test_far_angles(dev, bits):
    announce(f"angles up to 2^{bits}")
    g = np.random.default_rng(bits)
    n = 64
    pos = g.integers(1 << (bits - 1), 1 << bits, 400)
    pos[::5] *= -1
    f = np.where(np.arange(n) % 2, 1 - np.arange(n) / 200, 1e6 ** -(np.arange(n) / n)).astype(np.float32)
    q = torch.zeros(len(pos), 1, 2 * n, device=dev)
    q[..., :n] = 1.0
    out, _ = qk_norm_rope(q, None, torch.from_numpy(pos).to(dev), torch.from_numpy(f).to(dev))
    got = out[:, 0].double().cpu().numpy()
    want = np.array([[_turn(p, x) for x in f] for p in pos])
    bad = np.maximum(np.abs(got[:, :n] - want[..., 0]), np.abs(got[:, n:] - want[..., 1]))
    assert bad.max() <= 3 * U, bad.max() / U
