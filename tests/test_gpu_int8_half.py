"""GPU: Int8Linear where its input, weight or autocast is float16: as the e4m3 linears, what is neither bfloat16 nor float32 is cast to
bfloat16 first, and a gradient comes back in its leaf's type."""

import pytest
import torch
import torch.nn as nn

from flower_amd import int8
from flower_amd.kernels import quant_rows
from flower_amd.precision import fp8_weight_cache
from tests.gpu_util import seeded

pytestmark = pytest.mark.gpu


def pair(dtype, bias, M=37, N=96, K=64):
    """(module of that dtype, module of the same values in bfloat16, input, output gradient)"""
    own = int8.Int8Linear(K, N, bias=bias, device="cuda", dtype=dtype)
    own.weight.data.copy_(seeded((N, K), 1))
    if bias:
        own.bias.data.copy_(seeded((N,), 2))
    same = int8.Int8Linear(K, N, bias=bias, device="cuda", dtype=torch.bfloat16)
    same.load_state_dict(own.state_dict())
    return own, same, seeded((M, K), 3, torch.float16), seeded((M, N), 4, torch.bfloat16)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("bias", [False, True])
def test_a_float16_module(bias, fp8):
    own, same, x, g = pair(torch.float16, bias)
    own.backward_fp8 = same.backward_fp8 = fp8
    want_x = x.bfloat16().requires_grad_()
    want = same(want_x)
    want.backward(g)
    for cached in (False, True):
        own.zero_grad()
        leaf = x.clone().requires_grad_()
        with fp8_weight_cache(nn.ModuleList([own] if cached else [])):
            y = own(leaf)
            y.backward(g)
            with torch.no_grad():
                assert torch.equal(own(x), want) and torch.equal(own.forward_codes(*quant_rows(x.bfloat16())), want)
        assert torch.equal(y, want)
        for got, ref in zip((leaf.grad, *(p.grad for p in own.parameters())), (want_x.grad, *(p.grad for p in same.parameters()))):
            assert got.dtype == torch.float16 and torch.equal(got, ref.half())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_float16_autocast(dtype):
    own, _, x, g = pair(dtype, True)
    want_x = x.bfloat16().requires_grad_()
    want = own(want_x)
    want.backward(g)
    grads = [p.grad.clone() for p in own.parameters()]
    own.zero_grad()
    leaf = x.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.float16):
        y = own(leaf)
    y.backward(g)
    assert y.dtype == torch.bfloat16 and torch.equal(y, want) and torch.equal(leaf.grad, want_x.grad.float())
    assert all(torch.equal(p.grad, q) for p, q in zip(own.parameters(), grads))
