"""CPU: the polynomial of the 8-bit rows' GELU, with the coefficients that the kernel's source holds, against erfc in 64 bits."""

import os
import re

import numpy as np
from scipy.special import erfcx

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flower_amd", "csrc", "flw_rows8.hip")


def test_the_tail_polynomial_is_as_near_as_its_comment_says():
    """R(z) = Q(z) exp(z^2 / 2) = erfcx(z / sqrt 2) / 2 by a polynomial in t = 1 / (1 + z / 4), relative to R, z <= 14."""
    with open(SOURCE) as f:
        text = f.read()
    body = text[text.index("float gelu(float x) {"):]
    body = body[:body.index("\n}")]
    found = re.findall(r"(?:, r = |r = fmaf\(r, t, )(-?[0-9.]+(?:e-?\d+)?)f", body)
    assert len(found) == 10
    z = np.linspace(0.0, 14.0, 200001)
    t, r = 1.0 / (1.0 + 0.25 * z), np.zeros_like(z)
    for c in found:
        r = r * t + np.float64(np.float32(c))
    worst = np.abs(r / (0.5 * erfcx(z / np.sqrt(2.0))) - 1.0).max()
    stated = float(re.search(r"relative error ([0-9.e-]+) with its", text).group(1))
    assert stated * 0.9 < worst <= stated * 1.01, worst
