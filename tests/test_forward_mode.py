"""Forward-mode differentiation of the native operators, and gradients of what the forward-only ones take, are refused, never
dropped."""

import pytest
import torch
from torch.autograd import forward_ad

from flower_amd.kernels import apply_rotary, paged_append, paged_attention


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("which", ["q", "k", "cos", "sin"])
@pytest.mark.parametrize("grad", [True, False])
def test_rotary(which, grad):
    a = dict(q=torch.zeros(2, 4, 3, 64), k=torch.zeros(2, 2, 3, 64), cos=torch.zeros(8, 32), sin=torch.zeros(8, 32))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        a[which] = dual(a[which])
        with pytest.raises(RuntimeError, match="forward-mode"):
            apply_rotary(*a.values())
    with pytest.raises(RuntimeError, match="only on a ROCm GPU"):         # the level is left: as any other tensors
        apply_rotary(*a.values())


@pytest.mark.parametrize("which", [0, 1, 2])
def test_paged_append_and_attention(which):
    heads = [torch.zeros(2, n, 1, 64, dtype=torch.bfloat16) for n in (4, 2, 2)]
    pool = (torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, 16, dtype=torch.bfloat16),
            torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with forward_ad.dual_level(), torch.no_grad():
        heads[which] = dual(heads[which])
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_append(*heads, *pool)
        if which == 0:
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged_attention(heads[0], *pool)


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_paged_operators_refuse_gradients_of_pages_and_scales(which):
    heads = [torch.zeros(2, n, 1, 64, dtype=torch.bfloat16) for n in (4, 2, 2)]
    floats = [torch.zeros(5, 2, 16, 64).to(torch.float8_e4m3fn), torch.zeros(5, 2, 64, 16).to(torch.float8_e4m3fn), torch.ones(2), torch.ones(2)]
    floats[which].requires_grad_()
    k_pages, v_pages, ks, vs = floats
    pool, how = (k_pages, v_pages, torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)), dict(k_scale=ks, v_scale=vs)
    for call in (lambda: paged_append(*heads, *pool, **how), lambda: paged_attention(heads[0], *pool, **how)):
        with pytest.raises(RuntimeError, match="forward-only"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="only on a ROCm GPU"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("create_graph", [False, True])
def test_a_tangent_of_rotarys_output_gradient(create_graph):
    q = torch.randn(1, 2, 5, 64, device="cuda", requires_grad=True)
    t = torch.randn(8, 32, device="cuda")
    y, _ = apply_rotary(q, None, t, t)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode|jvp"):
        torch.autograd.grad(y, q, dual(torch.ones_like(y)), create_graph=create_graph)
