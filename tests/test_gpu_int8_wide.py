"""GPU: int8 linears at the ends of what they take: outputs wider than a pass over 8-bit rows, more rows than a column sum,
the few-row kernel's largest LDS.

Tolerances as in test_gpu_int8_linear.py: a gradient is off by its bf16 rounding, 2^-8, and the matrix unit's fp32 sums, a thousandth
of the largest.
"""

import numpy as np
import pytest
import torch

from flower_amd import int8
from flower_amd.kernels import int8_linear, int8_scaled_mm, quant_rows
from oracle.gemm import fp8_linear_backward
from tests.gpu_util import seeded, to_np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [32768, 32784, 50304, 128256])
@pytest.mark.parametrize("bias", [False, True])
def test_gradients_of_wide_outputs(N, bias):
    """A vocabulary's width: the output's gradient is cast by rows of N values."""
    M, K = 5, 48
    x, w, b = seeded((M, K), 1, torch.bfloat16), seeded((N, K), 2, torch.bfloat16, scale=K ** -0.5), seeded((N,), 3, torch.bfloat16)
    g = seeded((M, N), 4, torch.bfloat16) * seeded((M, 1), 5, torch.bfloat16).exp()
    leaves = [t.requires_grad_() for t in ((x, w, b) if bias else (x, w))]
    y = int8.int8_linear_train(*leaves)
    assert torch.equal(y.detach(), int8_linear(x.detach(), *quant_rows(w.detach()), bias=b.detach() if bias else None))
    grads = torch.autograd.grad(y, leaves, g)
    for got, want in zip(grads, fp8_linear_backward(to_np(g), to_np(x), to_np(w), "rowwise")):
        assert np.abs(to_np(got) - want).max() <= np.abs(want).max() * (2.0 ** -8 + 1e-3)
    if bias:
        s, total = g.double().sum(0), g.double().abs().sum(0)
        assert ((grads[2].double() - s).abs() <= s.abs() * 2.0 ** -8 + total * M * 2.0 ** -24).all()


@pytest.mark.parametrize("N", [32784, 50304])
def test_a_wide_modules_input_gradient(N):
    """Through the module, the weight's codes kept or not, a gradient whose rows are apart: the bits of one call."""
    from flower_amd.precision import fp8_weight_cache

    mod = int8.Int8Linear(64, N, bias=False, device="cuda", dtype=torch.bfloat16)
    x = seeded((33, 64), 6, torch.bfloat16).requires_grad_()
    g = seeded((33, N + 24), 7, torch.bfloat16)[:, :N]
    want = torch.autograd.grad(mod(x), x, g.contiguous())[0]
    assert torch.equal(torch.autograd.grad(mod(x), x, g)[0], want)
    with fp8_weight_cache(torch.nn.ModuleList([mod])):
        assert torch.equal(torch.autograd.grad(mod(x), x, g)[0], want)


@pytest.mark.parametrize("rows", [65535 * 128, 65535 * 128 + 1])
def test_gradients_of_very_many_rows(rows):
    """More rows than one column sum takes. The bias's gradient: chains of 32 + 3 + 4096 + 16 additions in fp32 of each part, and the
    parts', each off by 2^-24 of the absolute sum, then the rounding. Rows of the input's gradient are the same bits as alone."""
    N = K = 16
    rng = torch.Generator(device="cuda").manual_seed(1)
    x, g = (torch.randn(rows, n, generator=rng, device="cuda").bfloat16() for n in (K, N))
    w, b = seeded((N, K), 2, torch.bfloat16, scale=0.25), seeded((N,), 3, torch.bfloat16)
    s, total = g.double().sum(0), g.abs().sum(0, dtype=torch.float64)
    for bias in (b, b.float()):
        leaves = [t.detach().requires_grad_() for t in (x, w, bias)]
        gx, gw, gb = torch.autograd.grad(int8.int8_linear_train(*leaves), leaves, g)
        half = 2.0 ** -8 if bias.dtype == torch.bfloat16 else 2.0 ** -24
        assert gb.dtype == bias.dtype and ((gb.double() - s).abs() <= s.abs() * half + total * 4150 * 2.0 ** -24).all()
    some = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    few = [x[some].clone().requires_grad_(), w.detach(), b.detach()]
    assert torch.equal(gx[some], torch.autograd.grad(int8.int8_linear_train(*few), few[0], g[some])[0])
    assert torch.isfinite(gw).all() and gw.any()


@pytest.mark.parametrize("M,N,K", [(16, 64, 8960), (15, 100, 9600), (9, 33, 15984), (4, 1283, 32768)])
def test_few_rows_in_the_most_lds(M, N, K):
    """Rows that fill the few-row kernel's 150 KB, and those that just do not fit: to the bit, as their float64 sums."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = (torch.randint(-128, 128, (n, K), generator=g).to(torch.int8).cuda() for n in (M, N))
    sa, sb = (torch.rand(n, generator=g).add(0.5).mul(1e-3).cuda() for n in (M, N))
    want = (a.double() @ b.double().t()).float().mul_(sa[:, None]).mul_(sb).bfloat16()
    assert torch.equal(int8_scaled_mm(a, sa, b, sb), want)
    x = seeded((M, K), 8, torch.bfloat16)
    codes, scale = quant_rows(x)
    assert torch.equal(int8_linear(x, b, sb), int8_scaled_mm(codes, scale, b, sb))
