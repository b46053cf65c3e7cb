"""The polynomial 2^x of the paged prompt record, with the coefficients that stand in its source, in the order of its operations:
a fused multiply-add is one rounding of the exact result (here by 64 bits, which hold the product of two fp32 numbers)."""
import os
import re

import numpy as np

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vsa_lm_b200", "csrc", "paged_prompt.cu")


def _coefficients():
    body = open(SRC).read().split("float2 ex2_fma(float2 x) {")[1].split("\n}\n")[0]
    found = re.findall(r"y = (?:fma2\(y, f, )?pair\(([0-9.]+)f, ([0-9.]+)f\)", body)
    assert len(found) == 6 and all(a == b for a, b in found)
    return [np.float32(a) for a, _ in found]


def _error(x):
    n = np.rint(x).astype(np.float32)
    f = x - n                                             # exact
    y = np.full_like(f, _coefficients()[0])
    for c in _coefficients()[1:]:
        y = (y.astype(np.float64) * f.astype(np.float64) + np.float64(c)).astype(np.float32)
    return np.abs(y.astype(np.float64) * np.exp2(n.astype(np.float64)) / np.exp2(x.astype(np.float64)) - 1).max()


def test_the_polynomial_is_as_near_as_its_comment_says():
    rng = np.random.default_rng(0)
    for x in (np.linspace(-0.5, 0.5, (1 << 21) + 1), rng.uniform(-126, 0, 1 << 21), -np.exp2(rng.uniform(-30, 6.9, 1 << 20))):
        assert _error(x.astype(np.float32)) <= 2 ** -22.6
    assert _error(np.zeros(1, dtype=np.float32)) == 0


def test_the_coefficients_alone():
    f = np.linspace(-0.5, 0.5, (1 << 20) + 1)
    y = np.polyval([np.float64(c) for c in _coefficients()], f)
    assert np.abs(y / np.exp2(f) - 1).max() <= 2 ** -23.3
