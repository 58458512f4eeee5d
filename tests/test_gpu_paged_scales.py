"""GPU: paged_attention where a head's scores are multiplied by zero: every key that a row sees weighs the same, and one that it
does not see nothing, whichever way the work is cut. Tolerances: test_gpu_paged's (the oracle's slack has no scores' part)."""

import pytest
import torch

from gpu_util import seeded
from test_gpu_paged import check_attention, ints, make_cache, values

pytestmark = pytest.mark.gpu

CASES = [
    # KV, G, T, D, page, cache, lens, counts, window
    (2, 1, 1, 64, 64, "bf16", [1, 0, 63, 64, 65, 130], None, None),
    (2, 2, 1, 64, 16, "bf16", [5, 200, 701], None, 77),
    (1, 4, 3, 128, 32, "e4m3", [7, 150, 411], [3, 1, 2], None),
    (1, 4, 1, 64, 64, "bf16", [20001], None, None),                 # cut into parts
    (1, 8, 8, 64, 32, "e4m3", [1500], None, 1000),                  # four waves of rows
    (4, 3, 1, 32, 64, "bf16", [250, 1, 129], None, None),           # four waves an item
]


@pytest.mark.parametrize("KV,G,T,D,page,cache,lens,counts,window", CASES)
@pytest.mark.parametrize("scale", [0.0, -0.0])
def test_a_scale_of_zero_is_the_mean_of_the_seen_values(KV, G, T, D, page, cache, lens, counts, window, scale):
    print("[scale 0]", KV, G, T, D, page, cache, lens, counts, window, flush=True)
    k, v, tables, ks, vs = make_cache(len(lens), KV, D, page, lens, cache)
    q = seeded((len(lens), T, KV * G, D), 9, torch.bfloat16, scale=1.5).transpose(1, 2)
    out = check_attention(q, k, v, tables, lens, counts, window, ks, vs, scale=scale)
    assert torch.isfinite(out).all()


def test_a_head_whose_k_scale_is_zero():
    k, v, tables, ks, vs = make_cache(3, 3, 64, 16, [40, 9, 333], "e4m3")
    ks[1] = 0.0
    q = seeded((3, 2, 6, 64), 9, torch.bfloat16).transpose(1, 2)
    assert torch.isfinite(check_attention(q, k, v, tables, [40, 9, 333], None, None, ks, vs)).all()


def test_zero_times_what_is_not_finite_is_nan():
    """As the product says: a query, or a seen key, that is not finite; not a key behind the window."""
    from flower_amd.kernels import paged_attention
    k, v, tables, _, _ = make_cache(4, 1, 64, 16, [40] * 4, "bf16")
    q = seeded((4, 1, 1, 64), 9, torch.bfloat16)
    q[0, 0, 0, 5], q[1, 0, 0, 63] = float("inf"), float("nan")
    k[int(tables[2, 1]), 0, 3, 7] = float("-inf")
    out = paged_attention(q, k, v, tables, ints([40] * 4), scale=0.0)
    assert torch.isnan(out[:3]).all() and torch.isfinite(out[3]).all()
    out = paged_attention(q, k, v, tables, ints([40] * 4), scale=0.0, window=20)
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2:]).all()
    mean = values(v)[[int(t) for t in tables[3, 1:3]]]               # positions 20 .. 39
    mean = (mean[0, 0, :, 4:].sum(-1) + mean[1, 0, :, :8].sum(-1)) / 20
    assert (abs(values(out)[3, 0, 0] - mean) <= 2.0 ** -8 * abs(mean) + 2.0 ** -12).all()
