"""CPU: YaRN's frequencies pair by pair, from the published formula.

Pair i turns at f_i = base^(-2 i / R). The (fractional) pair that turns n times in L positions is R ln(L / (2 pi n)) / (2 ln base);
between floor(that of beta_fast), at least 0, and ceil(that of beta_slow), at most R - 1, a line over i goes from f_i to f_i / s.

Tolerance: the tables' entries at position 1 are cos and sin of an angle of at most 1, times the attention factor, each
rounded to half a step (2^-24 of itself), so that the angle read back is off by at most 2^-24 |sin 2 a| <= 2^-23 a: 2^-22 of it.
"""

import math

import pytest
import torch

from flower_amd.attention import rotary_tables


def formula(R, L, s, base, fast, slow):
    pair = lambda n: R * math.log(L / (2 * math.pi * n)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), R - 1)
    out = []
    for i in range(R // 2):
        f = base ** (-2.0 * i / R)
        w = min(max((i - low) / (high - low), 0.0), 1.0)
        out.append(f * (1 - w) + f / s * w)
    return out


@pytest.mark.parametrize("R,L,s,base,fast,slow", [
    (64, 2048, 16.0, 10000.0, 32, 1),        # the ramp ends within the pairs
    (64, 32768, 8.0, 10000.0, 32, 1),        # just behind the last
    (64, 65536, 8.0, 10000.0, 32, 1),        # behind the last pair: it still turns more than once, and is not slowed in full
    (128, 131072, 8.0, 10000.0, 32, 1),
    (16, 32768, 4.0, 10000.0, 32, 1),
    (8, 8192, 8.0, 10000.0, 32, 1),
    (128, 4096, 2.0, 500000.0, 32, 1),
    (64, 2048, 4.0, 10000.0, 8, 2),
])
def test_every_pairs_frequency(R, L, s, base, fast, slow):
    cos, sin = rotary_tables(R, 2, base, {"type": "yarn", "factor": s, "original_positions": L, "beta_fast": fast, "beta_slow": slow})
    got = torch.atan2(sin[1].double(), cos[1].double()).tolist()
    want = formula(R, L, s, base, fast, slow)
    assert [i for i, (a, b) in enumerate(zip(got, want)) if abs(a - b) > 2.0 ** -22 * b] == []
    for i, f in enumerate(want):             # and what the formula is for
        turns, plain = L * base ** (-2.0 * i / R) / (2 * math.pi), base ** (-2.0 * i / R)
        assert turns <= slow or f > plain / s * (1 + 1e-9)
