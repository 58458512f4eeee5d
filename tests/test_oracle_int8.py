"""Pins oracle/int8.py against torch on the CPU."""

import numpy as np
import pytest
import torch

from oracle.int8 import gelu, product, rms_norm, rows8, swiglu


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 64), (2, 1031)])
def test_rows8_is_torchs_division_and_rounding(kind, shape):
    h = torch.randn(*shape, generator=torch.Generator().manual_seed(1)) * 3
    h[0] = 0
    top = torch.full((), 127.0 if kind == "int8" else 448.0)
    scale = torch.maximum(h.abs().amax(1) / top, torch.full((), 1e-12))
    units = h / scale[:, None]
    want = units.round().to(torch.int8) if kind == "int8" else units.to(torch.float8_e4m3fn).view(torch.uint8)
    codes, s = rows8(h.numpy(), kind)
    assert np.array_equal(s, scale.numpy()) and np.array_equal(codes, want.numpy())
    if kind == "int8":
        assert np.abs(codes.astype(int)).max() <= 127


def test_rows8_of_rows_that_are_not_finite():
    h = np.ones((3, 4), np.float32)
    h[0, 1], h[1, 2] = np.nan, -np.inf
    codes, s = rows8(h)
    assert np.isnan(s[:2]).all() and not codes[:2].any() and (codes[2] == 127).all()


def test_activations_norm_and_product():
    g = torch.Generator().manual_seed(2)
    x, u, w = (torch.randn(4, 33, generator=g, dtype=torch.float64) * 2 for _ in range(3))
    np.testing.assert_allclose(gelu(x.numpy()), torch.nn.functional.gelu(x).numpy(), rtol=1e-13, atol=1e-16)
    np.testing.assert_allclose(swiglu(x.numpy(), u.numpy()), (torch.nn.functional.silu(x) * u).numpy(), rtol=1e-13)
    np.testing.assert_allclose(rms_norm(x.numpy(), w[0].numpy(), 1e-6), torch.nn.functional.rms_norm(x, (33,), w[0], 1e-6).numpy(),
                               rtol=1e-13)
    a, b = (torch.randint(-128, 128, (n, 300), generator=g) for n in (5, 7))
    assert np.array_equal(product(a.numpy().astype(np.int8), b.numpy().astype(np.int8)), (a @ b.t()).numpy())
