"""GPU: 8-bit rows, the int8 product and the int8 linear against plain 64-bit arithmetic (oracle/int8.py).

Tolerances. A code is at most half a step from h / scale; what fp32 adds to that: the sum of K squares in chains and trees of
at most 64 additions, the mean, the square root, the division and three products, (64 / 2 + 6) 2^-24 = 2.3e-6 of h and of the
scale each, so 6e-4 of a step of int8 (127 steps) beside the half one. GELU and SwiGLU: a few 2^-24 of the argument's size each
for erf, exp, the sum and the quotient, 2^-21 of |x| (|h| for SwiGLU) with a margin: 127 * 2^-21 * |x| / max|h| steps.
A bf16 result is at most 2^-8 from its value (half a step of the coarsest place), each further rounding 2^-8 of what it rounds.
"""

import math

import numpy as np
import pytest
import torch

from flower_amd.kernels import gelu_quant, int8_linear, int8_scaled_mm, quant_rows, rms_norm_quant, swiglu_quant
from oracle import int8 as O
from oracle.e4m3 import e4m3_to_f32
from oracle.int8 import gelu
from tests.gpu_util import seeded, to_np

pytestmark = pytest.mark.gpu

COLS = [1, 7, 8, 31, 64, 257, 512, 1031, 1280, 2048, 2056, 4096, 6145, 8192, 8200, 16392, 32768]
FP32 = (64 / 2 + 6) * 2.0 ** -24


def kinds():
    return [(torch.int8, "int8"), (torch.float8_e4m3fn, "e4m3")]


def near(codes, scale, h, kind, slack):
    """codes and scale stand for the rows h (64 bits): slack (a row's values) in units of h."""
    amax = np.abs(h).max(axis=1)
    want = np.maximum(amax / (127.0 if kind == "int8" else 448.0), 1e-12)
    slack = np.broadcast_to(slack, h.shape)
    assert np.all(np.abs(scale - want) <= want * 2.0 ** -22 + slack.max(axis=1) / (127.0 if kind == "int8" else 448.0))
    s = scale.astype(np.float64)[:, None]
    off = np.abs((codes.astype(np.float64) if kind == "int8" else e4m3_to_f32(codes).astype(np.float64)) * s - h)
    half = s / 2 if kind == "int8" else np.maximum(np.abs(h) * 2.0 ** -4, s * 2.0 ** -10)
    bad = off > half * (1 + 2.0 ** -20) + slack * (1 + 2.0 ** -4) + np.abs(h) * 2.0 ** -22
    assert not bad.any(), (kind, off[bad][:4], half[np.broadcast_to(bad, half.shape)][:4])


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_bit_for_bit(cols, dtype):
    for rows in (1, 5):
        x = seeded((rows, cols), cols + rows, dtype, scale=3.0)
        x[0, 0] = 100.0
        for out, kind in kinds():
            codes, scale = quant_rows(x, dtype=out)
            want, s = O.rows8(to_np(x), kind)
            assert codes.dtype == out and codes.shape == x.shape and scale.shape == (rows,)
            assert np.array_equal(to_np(scale), s) and np.array_equal(to_np(codes), want), (cols, dtype, kind)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(cols, dtype, residual):
    x, a = seeded((6, cols), 1, dtype, scale=2.0), seeded((6, cols), 2, dtype)
    x[2] = a[2] = 0                                                    # a row of nothing
    for w in (seeded((cols,), 3, dtype), seeded((cols,), 3)):
        for out, kind in kinds():
            got = rms_norm_quant(x, w, 1e-5, residual=a if residual else None, dtype=out)
            assert len(got) == 2 + residual
            t = x
            if residual:
                t = (x.float() + a.float()).to(dtype)
                assert torch.equal(got[2], t)
            h = O.rms_norm(to_np(t), to_np(w), 1e-5)
            near(to_np(got[0]), to_np(got[1]), h, kind, np.abs(h) * FP32)


@pytest.mark.parametrize("cols", [1, 8, 31, 1280, 3392, 6145, 16392])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_activations(cols, dtype):
    x, u = seeded((5, cols), 4, dtype, scale=2.0), seeded((5, cols), 5, dtype)
    x[1] = -x[1].abs() - 3.0                                           # all of GELU's left tail
    x[2], x[3, 0] = 0.0, -100.0
    xn = to_np(x)
    for out, kind in kinds():
        codes, scale = gelu_quant(x, dtype=out)
        near(to_np(codes), to_np(scale), O.gelu(xn), kind, np.abs(xn) * 2.0 ** -21)
        codes, scale = swiglu_quant(x, u, dtype=out)
        h = O.swiglu(xn, to_np(u))
        near(to_np(codes), to_np(scale), h, kind, np.abs(h) * 2.0 ** -21)


@pytest.mark.parametrize("cols", [9, 1280, 4104])
def test_rows_that_are_not_finite_or_tiny(cols):
    x = seeded((7, cols), 6, torch.bfloat16)
    x[0, cols - 1], x[1, 0], x[2, cols // 2] = float("nan"), float("inf"), -float("inf")
    x[3] = 1e-30
    x[4, 0] = 3e38
    w = torch.ones(cols, device="cuda")
    codes, scale = quant_rows(x)
    want, s = O.rows8(to_np(x))
    assert np.array_equal(to_np(codes), want) and np.array_equal(to_np(scale), s, equal_nan=True)
    assert torch.isnan(scale[:3]).all() and not codes[:3].any()
    e, es = quant_rows(x, dtype=torch.float8_e4m3fn)
    want, s = O.rows8(to_np(x), "e4m3")
    assert np.array_equal(to_np(es), s, equal_nan=True)
    assert np.array_equal(to_np(e) & 0x7F, want & 0x7F)                # a NaN's sign is nobody's
    for got in (rms_norm_quant(x, w), gelu_quant(x), swiglu_quant(x, x)):
        codes, scale = got
        assert torch.isnan(scale[0]) and not codes[0].any() and torch.isfinite(scale[[3, 5, 6]]).all()
    y = int8_linear(x[[0, 5, 1, 6]], torch.ones(3, cols, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
    assert torch.isnan(y[[0, 2]]).all() and torch.isfinite(y[[1, 3]]).all()


def test_infinities_into_e4m3():
    """What an activation makes of an infinity is its limit: inf at inf and 0 at -inf. A row that holds an infinity has an infinite
    scale, and with it codes 0 but for its own."""
    x = torch.ones(4, 64, device="cuda")
    x[0, 3], x[1, 4], x[2, 5] = float("inf"), -float("inf"), float("nan")
    codes, scale = gelu_quant(x, dtype=torch.float8_e4m3fn)
    assert torch.isinf(scale[0]) and torch.isnan(scale[2]) and torch.isfinite(scale[[1, 3]]).all()
    assert torch.isnan(codes[0, 3].float()) and codes[0, 4].float() == 0 and codes[1, 4].float() == 0
    want = 0.5 * (1 + math.erf(math.sqrt(0.5)))
    assert (codes[1, 0].float() * scale[1] - want).abs() <= want * 2 ** -4 and torch.equal(codes[1, 5:], codes[3, 5:])
    codes, scale = swiglu_quant(x, torch.ones_like(x), dtype=torch.float8_e4m3fn)
    assert torch.isinf(scale[0]) and torch.isnan(scale[2]) and torch.isfinite(scale[[1, 3]]).all() and codes[1, 4].float() == 0
    for quant in (gelu_quant, lambda t: swiglu_quant(t, torch.ones_like(t))):       # the largest that are finite stay so
        big = torch.full((1, 64), 3e38, device="cuda")
        codes, scale = quant(big)
        assert torch.isfinite(scale).all() and (codes == 127).all()
        codes, scale = quant(-big)
        assert torch.isfinite(scale).all() and not codes.any()


def test_gelu_of_far_values():
    """Rows of negative values alone, where gelu is small: the exponential's argument, z^2 / 2 = 18 at -6, is off by its own 2^-24
    three times (its constant, z^2, the product), 18 * 3 * 2^-24 = 2^-18.2 of the value; 2^-17 is asked beside the codes' half step."""
    for lo, hi in ((-1.0, -0.1), (-3.0, -2.0), (-6.0, -5.0)):
        x = torch.linspace(lo, hi, 512, device="cuda").reshape(4, 128)
        codes, scale = gelu_quant(x)
        h = torch.from_numpy(gelu(to_np(x)))
        got = codes.cpu().double() * scale.cpu().double()[:, None]
        peak = h.abs().amax(1, keepdim=True)
        assert ((got - h).abs() <= peak * (0.5 / 127 + 2.0 ** -17)).all()


def test_rows_of_any_stride_and_shape():
    big = seeded((9, 3, 200), 7, torch.bfloat16)
    views = [big[:, 1, 3:131], big[:, :, 8:72], big.transpose(0, 1)[..., :64], big[..., ::2], big[:1, 0].expand(4, 200), big[:0], big[0, 0],
             big[:, 0, :1], big.permute(2, 1, 0)]
    w = seeded((200,), 8)
    for v in views:
        for call in (lambda t: quant_rows(t), lambda t: rms_norm_quant(t, w[:t.shape[-1]]), lambda t: gelu_quant(t),
                     lambda t: swiglu_quant(t, t), lambda t: rms_norm_quant(t, w[:t.shape[-1]], residual=t)):
            got, want = call(v), call(v.contiguous())
            assert got[0].shape == v.shape and got[1].shape == v.shape[:-1]
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def product(M, N, K, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * M + 11 * N + 13 * K)
    a, b = (torch.randint(-128, 128, (n, K), generator=g).to(torch.int8).cuda() for n in (M, N))
    sa, sb = (torch.rand(n, generator=g).add(0.5).mul(1e-3).cuda() for n in (M, N))
    return a, sa, b, sb


def check_product(y, a, sa, b, sb, bias=None, res=None):
    """To the bit without a bias; with one, a fused multiply-add may leave out a rounding of fp32."""
    acc = torch.from_numpy(O.product(a.cpu().numpy(), b.cpu().numpy()))
    v = acc.float() * sa.cpu().reshape(-1, 1) * sb.cpu().reshape(1, -1)
    if bias is None:
        want = v.bfloat16()
        if res is not None:
            want = (res.cpu().float() + want.float()).bfloat16()
        assert torch.equal(y.cpu(), want)
        return
    exact = acc.double() * sa.cpu().double().reshape(-1, 1) * sb.cpu().double().reshape(1, -1) + bias.cpu().double()
    slack = exact.abs() * 2.0 ** -8 + (v.double().abs() + bias.cpu().double().abs()) * 2.0 ** -22
    if res is not None:
        exact = exact + res.cpu().double()
        slack = slack + (exact.abs() + slack) * 2.0 ** -8
    assert ((y.cpu().double() - exact).abs() <= slack).all()


SIZES = [(1, 1, 1), (1, 64, 64), (1, 3840, 1280), (2, 5, 15), (3, 130, 16), (5, 17, 17), (7, 33, 100), (15, 1280, 80), (16, 96, 3392), (17, 1003, 127),
         (31, 64, 128), (32, 1280, 1280), (33, 100, 192), (48, 2000, 320), (64, 64, 4096), (65, 129, 8192), (100, 1283, 1291), (127, 640, 1040),
         (128, 128, 256), (129, 260, 336), (255, 512, 1280), (300, 1500, 272), (517, 1288, 1296), (1000, 1024, 2064)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K):
    a, sa, b, sb = product(M, N, K)
    check_product(int8_scaled_mm(a, sa, b, sb), a, sa, b, sb)
    res = seeded((M, N), 1, torch.bfloat16)
    check_product(int8_scaled_mm(a, sa, b, sb, residual=res), a, sa, b, sb, res=res)
    for bias in (seeded((N,), 2), seeded((N,), 2, torch.bfloat16)):
        check_product(int8_scaled_mm(a, sa, b, sb, bias=bias), a, sa, b, sb, bias)
        check_product(int8_scaled_mm(a, sa, b, sb, bias=bias, residual=res), a, sa, b, sb, bias, res)
    one = torch.full((1,), 2e-3, device="cuda")
    check_product(int8_scaled_mm(a, one, b, sb), a, one.expand(M), b, sb)
    check_product(int8_scaled_mm(a, sa, b, one), a, sa, b, one.expand(N))


@pytest.mark.parametrize("M,N,K", [(4096, 2304, 1296), (4100, 2312, 256), (8200, 8200, 144), (2500, 3000, 384), (4097, 2307, 272), (3000, 1280, 3392),
                                   (5000, 1024, 128)])
def test_large_products(M, N, K):
    """To the bit, against sums in float64 (exact: below 2^53) on the GPU: more tiles than one a compute unit, ragged ones, outputs
    of both sides of the size from which they pass the caches by."""
    a, sa, b, sb = product(M, N, K)
    v = (a.double() @ b.double().t()).float().mul_(sa[:, None]).mul_(sb).bfloat16()
    assert torch.equal(int8_scaled_mm(a, sa, b, sb), v)
    res = seeded((M, N), 1, torch.bfloat16)
    assert torch.equal(int8_scaled_mm(a, sa, b, sb, residual=res), (res.float() + v.float()).bfloat16())
    bias = seeded((N,), 2)
    few = [0, 1, M // 2, M - 1]
    assert torch.equal(int8_scaled_mm(a, sa, b, sb, bias=bias)[few], int8_scaled_mm(a[few], sa[few], b, sb, bias=bias))


@pytest.mark.parametrize("M,N,K", [(4100, 2312, 256), (4096, 4096, 1296), (9000, 4104, 144)])
def test_large_products_with_everything(M, N, K):
    """Bias and a residual of its own row stride, over every row: as in parts of 200 rows, which another kernel computes."""
    a, sa, b, sb = product(M, N, K)
    wide, odd = seeded((M, N + 24), 1, torch.bfloat16), seeded((M, N + 3), 1, torch.bfloat16)
    for bias in (seeded((N,), 2), seeded((N,), 2, torch.bfloat16), None):
        for res in (wide[:, 8:8 + N], odd[:, 1:1 + N], None):
            y = int8_scaled_mm(a, sa, b, sb, bias=bias, residual=res)
            parts = [int8_scaled_mm(a[r:r + 200], sa[r:r + 200], b, sb, bias=bias, residual=None if res is None else res[r:r + 200])
                     for r in range(0, M, 200)]
            assert torch.equal(y, torch.cat(parts))


@pytest.mark.parametrize("M", [1, 40, 700])
def test_product_at_the_ends_of_its_range(M):
    """The longest K that int32 holds, with every product the largest: 128 * 128 * 131071 and its negative."""
    K, N = 131071, 24
    for K in (131071, 131056):
        a = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
        b = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
        b[1::2] = 127
        one = torch.ones(1, device="cuda")
        y = int8_scaled_mm(a, one, b, one).float().cpu()
        want = torch.tensor([16384.0 * K, -16256.0 * K]).bfloat16().float()
        assert (y[:, ::2] == want[0]).all() and (y[:, 1::2] == want[1]).all()


@pytest.mark.parametrize("K", [64, 100, 1280])
def test_product_of_views(K):
    """Row strides that vectors take and others, a leading shape, the rows behind the output's left as they were."""
    big, w = product(20, 30, 2 * K + 48)[0::2]
    sa, sb = torch.rand(20, device="cuda"), torch.rand(30, device="cuda")
    for a, b in ((big[:, :K], w[:, 16:16 + K]), (big[:, 3:3 + K], w[:, 5:5 + K]), (big[::2, 32:32 + K], w[::3, :K]),
                 (big.view(4, 5, -1)[:, 1:4, :K], w[:, :K]), (big[:, :2 * K:2], w[:, 1:2 * K:2]), (big[:1, :K].expand(6, K), w[:, :K])):
        rows = a.reshape(-1, K)
        s, t = sa[:rows.shape[0]].contiguous(), sb[:b.shape[0]].contiguous()
        y = int8_scaled_mm(a, s, b, t)
        assert y.shape == (*a.shape[:-1], b.shape[0])
        check_product(y.reshape(-1, b.shape[0]), rows, s, b, t)
    res = seeded((20, 61), 3, torch.bfloat16)
    for r in (res[:, 1:31], res[:, ::2][:, :30]):
        check_product(int8_scaled_mm(big[:, :K], sa, w[:, :K], sb, residual=r), big[:, :K], sa, w[:, :K], sb, res=r)
    assert int8_scaled_mm(big[:0, :K], sa[:0], w[:, :K], sb).shape == (0, 30)


def test_a_row_alone_is_the_row_in_a_batch():
    """Whatever way the work is cut by the number of rows."""
    a, sa, b, sb = product(700, 1344, 1280)
    res = seeded((700, 1344), 4, torch.bfloat16)
    whole = int8_scaled_mm(a, sa, b, sb, residual=res)
    for rows in ([3], [0, 699], list(range(5)), list(range(13)), list(range(100, 133)), list(range(600, 697)), list(range(260))):
        part = int8_scaled_mm(a[rows], sa[rows], b, sb, residual=res[rows])
        assert torch.equal(part, whole[rows]), len(rows)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 3840, 1280), (3, 130, 17), (4, 1280, 3392), (16, 100, 31), (2, 96, 2064), (3, 1288, 1296), (5, 64, 16),
                                   (16, 1003, 4112), (7, 320, 8192), (1, 48, 16), (48, 1280, 1280), (517, 1283, 1291),
                                   (300, 512, 4096), (1, 64, 32768)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_is_its_two_parts(M, N, K, dtype):
    x, w = seeded((M, K), 5, dtype), seeded((N, K), 6)
    w8, sw = quant_rows(w)
    bias, res = seeded((N,), 7, torch.bfloat16), seeded((M, N), 8, torch.bfloat16)
    codes, scale = quant_rows(x)
    for how in ({}, dict(bias=bias), dict(residual=res), dict(bias=bias, residual=res)):
        assert torch.equal(int8_linear(x, w8, sw, **how), int8_scaled_mm(codes, scale, w8, sw, **how))
    check_product(int8_linear(x, w8, sw), codes, scale, w8, sw)


def test_linear_is_near_the_unquantised_one():
    """Each operand's error is uniform within half a step: scale / sqrt 12 a value, so for normal rows with maxima of about 4 sigma
    4 / 127 / sqrt 12 = 0.9 % of sigma each, 1.3 % of the result's size together; 2 % is asked."""
    x, w = seeded((300, 1280), 9, torch.bfloat16), seeded((640, 1280), 10, torch.bfloat16)
    w8, sw = quant_rows(w)
    y = int8_linear(x.view(3, 100, 1280), w8, sw).view(300, 640).double()
    want = x.double() @ w.double().t()
    assert ((y - want).norm() / want.norm()).item() < 0.02


def test_on_a_stream_of_its_own_and_in_a_graph():
    x, a, w = seeded((40, 1280), 11, torch.bfloat16), seeded((40, 1280), 12, torch.bfloat16), seeded((1280,), 13)
    w8, sw = quant_rows(seeded((512, 1280), 14))

    def step():
        codes, scale, total = rms_norm_quant(x, w, residual=a)
        y = int8_scaled_mm(codes, scale, w8, sw)
        codes, scale = gelu_quant(y)
        g, s2 = swiglu_quant(y, y)
        return total, y, codes, scale, g, s2, int8_linear(x[:1], w8, sw), int8_linear(x, w8, sw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apart = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(apart, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        x.copy_(seeded((40, 1280), 20 + seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step()))


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes apart, and an output of more than that: each as at its place in a small one."""
    K, N, far = 144, 40, 2 ** 31 + 64
    base = torch.empty(2 * far + K, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((3, K), (far, 1))
    x.copy_(seeded((3, K), 1, torch.bfloat16))
    near = x.contiguous()
    for got, want in zip((*quant_rows(x), *swiglu_quant(x, x), *rms_norm_quant(x, near[0], residual=x)),
                         (*quant_rows(near), *swiglu_quant(near, near), *rms_norm_quant(near, near[0], residual=near))):
        assert torch.equal(got, want)
    w8, sw = quant_rows(seeded((N, K), 2, torch.bfloat16))
    assert torch.equal(int8_linear(x, w8, sw), int8_linear(near, w8, sw))
    bytes_ = base.view(torch.int8).as_strided((3, K), (2 * far, 1))
    codes, s = quant_rows(near)
    bytes_.copy_(codes)
    assert torch.equal(int8_scaled_mm(bytes_, s, w8, sw), int8_scaled_mm(codes, s, w8, sw))
    assert torch.equal(int8_scaled_mm(w8, sw, bytes_, s), int8_scaled_mm(w8, sw, codes, s))
    del base, x, bytes_
    for M, N, K in ((70000, 32768, 144), (70000, 32768, 128), (70001, 32767, 40)):      # the stream, tiles, any
        a, b = (torch.randint(-128, 128, (r, K), dtype=torch.int8, device="cuda") for r in (M, N))
        sa, sb = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
        y = int8_scaled_mm(a, sa, b, sb)
        assert y.numel() * 2 > 2 ** 32
        for rows in (slice(0, 40), slice(M // 2, M // 2 + 33), slice(M - 50, M)):
            assert torch.equal(y[rows], int8_scaled_mm(a[rows], sa[rows], b, sb))
        del y
