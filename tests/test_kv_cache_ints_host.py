"""CPU: counts and places that are no whole numbers are refused, not cut."""

import numpy as np
import pytest
import torch

from flower_amd.kv_cache import PagedKVCache


@pytest.mark.parametrize("values", [[1.5, 2.0], torch.tensor([1.0, 2.0]), np.array([0.7, 1.0]), torch.tensor([1j, 0])])
def test_refused(values):
    cache = PagedKVCache(1, 4, 1, 64, sequences=2, max_len=64, device="cpu")
    for call in (cache.reserve, cache.reorder, cache.take_back):
        with pytest.raises(TypeError, match="whole numbers"):
            call(values)
