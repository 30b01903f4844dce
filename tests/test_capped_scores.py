"""CPU: the cap of the shaped scores as the kernels compute it, restated in 32 bits with the coefficients of the source."""
import re
from pathlib import Path

import numpy as np
import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "nanopd_b200" / "csrc" / "capped_scores.cuh").read_text()
R = [float(x.strip().rstrip("f")) for x in re.search(r"kR\[4\] = \{([^}]*)\}", SOURCE).group(1).split(",")]
f32 = np.float32


def capped_log2(x, scale, cap):
    per = f32(max(float(scale) / float(cap), 1.2e-38))
    with np.errstate(over="ignore", invalid="ignore"):
        z = x * per
        w = z * z
        r = f32(R[3])
        for c in R[2::-1]:
            r = r * w + f32(c)
        y = x * f32(scale * 1.4426950408889634)
        near = (y * w) * r + y
        log2 = f32(f32(cap) * f32(1.4426950408889634))
        far = np.copysign(log2 - f32(2) * log2 / (f32(1) + np.exp2(np.abs(x) * f32(2 * 1.4426950408889634 * float(per)))), x)
        return np.where(np.abs(x) < f32(0.6 / float(per)), near, far)


def test_coefficients():
    z = np.linspace(-0.6, 0.6, 20001)
    z = z[z != 0]
    w = z * z
    t = z * (1 + w * sum(c * w ** k for k, c in enumerate(R)))
    assert np.abs(t / np.tanh(z) - 1).max() < 9e-8


@pytest.mark.parametrize("cap", [1e-30, 1e-3, 1.0, 30.0, 880.0, 1e5, 1e6, 1e9, 1e20, 1e38])
def test_every_cap_keeps_the_relative_accuracy_of_the_score(cap):
    """The polynomial is off by 8.4e-8, its evaluation by a few roundings of 2^-24; the exponential's form at z = 0.6 by
    2 / (1 + e^1.2) / tanh 0.6 = 0.87 times what its exponential, sum and quotient are off by (2^-22 each here, in numpy less)."""
    rng = np.random.default_rng(0)
    scale = 128 ** -0.5
    x = np.concatenate([rng.standard_normal(4000) * 11.3, rng.standard_normal(4000) * 300,
                        rng.uniform(-4, 4, 4000) * min(cap, 1e30) / scale]).astype(f32)
    x = x[np.abs(x) > 1e-30]
    exact = cap * np.tanh(x.astype(np.float64) * scale / cap) * 1.4426950408889634
    off = np.abs(capped_log2(x, scale, cap).astype(np.float64) - exact)
    assert (off <= 1.2e-6 * np.abs(exact)).all()


def test_the_short_form_serves_small_caps_only():
    """Its absolute error, 2^-23 cap in log2 units times 1.44, stays below what scores of 60 are off by (3e-5)."""
    assert float(re.search(r"kLowCap = ([0-9.]+)f", SOURCE).group(1)) * 1.4427 * 2 ** -23 < 3e-5


def test_infinite_scores_are_capped():
    for cap in (1e-3, 50.0, 1e9):
        y = capped_log2(np.array([np.inf, -np.inf], dtype=f32), 0.1, cap)
        assert np.allclose(y, [cap * 1.4426950408889634, -cap * 1.4426950408889634], rtol=1e-6)
