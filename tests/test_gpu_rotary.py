"""GPU: apply_rotary against the float64 oracle, forward and gradient.

Tolerance: an output value is fma(a, c, -(b s)) (or fma(b, c, a s)) in fp32, two roundings of at most
2^-24 (|a c| + |b s|) each, then one rounding to the dtype (half a step: bf16 2^-8, fp32 2^-24 of the value; the fp32 one is
the fma's own). Values that are only copied are equal.
"""

import numpy as np
import pytest
import torch

from oracle import paged as O

from gpu_util import seeded, to_np

pytestmark = pytest.mark.gpu


def tables(rows, R, seed=3):
    g = np.random.default_rng(seed)
    a = g.uniform(-3.0, 3.0, (rows, R // 2))
    return torch.tensor(np.cos(a), dtype=torch.float32).cuda(), torch.tensor(np.sin(a), dtype=torch.float32).cuda()


def check(got, x, cos, sin, pos, layout, dtype, inverse=False):
    want, size = O.rotary(to_np(x).astype(np.float64), to_np(cos), to_np(sin), pos, layout, inverse)
    got = to_np(got).astype(np.float64)
    assert got.shape == want.shape
    step = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    bad = ~((np.abs(got - want) <= step * np.abs(want) + 2.0 ** -22 * size) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4])
    R = 2 * cos.shape[1]
    assert np.array_equal(got[..., R:], to_np(x).astype(np.float64)[..., R:])


CASES = [
    # B, H, KV, T, D, R, layout, dtype, positions
    (2, 4, 2, 33, 64, 64, "interleaved", torch.bfloat16, "none"),
    (2, 4, 2, 33, 64, 64, "half", torch.bfloat16, "row"),
    (3, 3, 1, 1, 128, 64, "half", torch.bfloat16, "batch"),
    (1, 2, 2, 257, 32, 8, "half", torch.float32, "batch"),
    (1, 5, 5, 130, 128, 128, "half", torch.float32, "long"),
    (2, 2, 1, 65, 32, 32, "interleaved", torch.float32, "batch"),
    (4, 20, 20, 70, 64, 16, "interleaved", torch.bfloat16, "long"),
    (1, 1, 1, 1, 32, 8, "interleaved", torch.bfloat16, "row"),
]


def positions_of(kind, B, T, rows):
    g = torch.Generator().manual_seed(7)
    if kind == "none":
        return None, np.broadcast_to(np.arange(T), (B, T))
    if kind == "row":
        p = torch.randint(0, rows, (T,), generator=g, dtype=torch.int32)
        return p.cuda(), np.broadcast_to(p.numpy(), (B, T))
    p = torch.randint(0, rows, (B, T), generator=g, dtype=torch.int64 if kind == "long" else torch.int32)
    return p.cuda(), p.numpy()


@pytest.mark.parametrize("B,H,KV,T,D,R,layout,dtype,kind", CASES)
@pytest.mark.parametrize("packed", [False, True])
def test_forward_and_gradient(B, H, KV, T, D, R, layout, dtype, kind, packed):
    rows = max(T, 50)
    cos, sin = tables(rows, R)
    if packed:                      # views of a fused projection's (B, T, heads x D)
        y = seeded((B, T, H + 2 * KV, D), 1, dtype).transpose(1, 2)
        q, k = y[:, :H].detach().requires_grad_(), y[:, H:H + KV].detach().requires_grad_()
    else:
        q, k = seeded((B, H, T, D), 1, dtype).requires_grad_(), seeded((B, KV, T, D), 2, dtype).requires_grad_()
    from flower_amd.kernels import apply_rotary
    pos, pos_np = positions_of(kind, B, T, rows)
    qo, ko = apply_rotary(q, k, cos, sin, pos, layout=layout)
    check(qo, q, cos, sin, pos_np, layout, dtype)
    check(ko, k, cos, sin, pos_np, layout, dtype)
    gq, gk = seeded(qo.shape, 5, dtype), seeded(ko.shape, 6, dtype)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    check(dq, gq, cos, sin, pos_np, layout, dtype, inverse=True)
    check(dk, gk, cos, sin, pos_np, layout, dtype, inverse=True)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient_against_differences(layout):
    """The map is linear: <g, f(x + d) - f(x - d)> / 2 = <grad, d>, to fp32 rounding (2^-22 of the sums of magnitudes)."""
    from flower_amd.kernels import apply_rotary
    cos, sin = tables(9, 16)
    x, d = seeded((1, 2, 9, 32), 1), seeded((1, 2, 9, 32), 2)
    g = seeded((1, 2, 9, 32), 3)
    f = lambda z: apply_rotary(z, None, cos, sin, layout=layout)[0].double()  # noqa: E731
    x1 = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(apply_rotary(x1, None, cos, sin, layout=layout)[0], x1, g)
    lhs = ((f(x + d) - f(x - d)) * g.double()).sum() / 2
    rhs = (grad.double() * d.double()).sum()
    size = (f(x.abs() + d.abs()).abs() * g.abs().double()).sum() * 4 + (grad.abs() * d.abs()).sum()
    assert abs(float(lhs - rhs)) <= 2.0 ** -21 * float(size)


def test_second_gradient_and_one_output_only():
    from flower_amd.kernels import apply_rotary
    cos, sin = tables(20, 64)
    q, k = seeded((2, 2, 20, 64), 1).requires_grad_(), seeded((2, 1, 20, 64), 2).requires_grad_()
    g = seeded((2, 2, 20, 64), 3).requires_grad_()
    qo, ko = apply_rotary(q, k, cos, sin)
    (dq,) = torch.autograd.grad(qo, q, g, create_graph=True)
    w = seeded(dq.shape, 4)
    (gg,) = torch.autograd.grad(dq, g, w)                    # the gradient's gradient is the forward rotation
    assert torch.equal(gg, apply_rotary(w, None, cos, sin)[0])
    (dk,) = torch.autograd.grad(ko, k, seeded(ko.shape, 6))  # without q's gradient
    check(dk, seeded(ko.shape, 6), cos, sin, np.broadcast_to(np.arange(20), (2, 20)), "interleaved", torch.float32, True)


def test_positions_outside_the_tables_are_nan_and_touch_nothing_else():
    from flower_amd.kernels import apply_rotary
    cos, sin = tables(10, 32)
    pos = torch.tensor([0, 9, 10, -1, 2 ** 31 - 1, 5], dtype=torch.int32).cuda()
    x = seeded((1, 2, 6, 64), 1, torch.bfloat16)
    y, none = apply_rotary(x, None, cos, sin, pos, layout="half")
    assert none is None
    check(y, x, cos, sin, to_np(pos)[None], "half", torch.bfloat16)
    assert torch.isnan(y[:, :, 2:5, :32]).all() and torch.isfinite(y[:, :, 2:5, 32:]).all()
    y64, _ = apply_rotary(x, None, cos, sin, pos.long() + 2 ** 40 * (pos == 5), layout="half")
    assert torch.isnan(y64[:, :, 5, :32]).all() and torch.equal(y64[:, :, :2], y[:, :, :2])


def test_infinite_and_nan_values_stay_in_their_pair():
    from flower_amd.kernels import apply_rotary
    cos, sin = tables(4, 32)
    x = seeded((1, 1, 4, 32), 1)
    x[0, 0, 1, 3], x[0, 0, 2, 7] = float("inf"), float("nan")
    y, _ = apply_rotary(x, None, cos, sin)
    bad = ~torch.isfinite(y)
    assert bad[0, 0, 1, 2:4].all() and bad[0, 0, 2, 6:8].all() and int(bad.sum()) == 4


def test_unaligned_rows_and_a_side_stream():
    from flower_amd.kernels import apply_rotary
    cos, sin = tables(30, 64)
    base = seeded((2, 3, 30, 67), 1, torch.bfloat16)
    x = base[..., 1:65]                                      # rows of 134 bytes, 2 bytes off
    want, _ = apply_rotary(x.contiguous(), None, cos, sin)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = apply_rotary(x, None, cos, sin)
    s.synchronize()
    assert torch.equal(got, want)
