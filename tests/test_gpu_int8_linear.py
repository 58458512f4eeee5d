"""GPU: Int8Linear and int8_linear_train: outputs, gradients, the weight cache.

The gradient is straight through the quantisers, its products the e4m3 ones of the rowwise recipe: against the oracle's, in
64 bits on the same codes, a result is off by its bf16 rounding, 2^-8, and the matrix unit's fp32 sums (a thousandth of the
largest is asked, as of the e4m3 linears). Against the gradient of the unquantised linear the two operands' e4m3 rounding, at most
2^-4 of a value each, uniform within it, is 2^-4 / sqrt 3 * sqrt 2 = 5.1 % of the result's size at the most; 6 % is asked.
"""

import ctypes

import numpy as np
import pytest
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from flower_amd import _lib, int8
from flower_amd.kernels import int8_linear, quant_rows
from flower_amd.precision import fp8_weight_cache, quantize_cols
from oracle.gemm import fp8_linear_backward
from tests.gpu_util import seeded, to_np

pytestmark = pytest.mark.gpu


class _Job(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                ("out_t", ctypes.c_void_p), ("ld", ctypes.c_int64), ("scale_out", ctypes.c_void_p)]


def tensors(M, N, K, dtype=torch.bfloat16):
    x, w, b = seeded((M, K), 1, dtype), seeded((N, K), 2, dtype, scale=K ** -0.5), seeded((N,), 3, dtype)
    g = seeded((M, N), 4, torch.bfloat16) * seeded((M, 1), 5, torch.bfloat16).exp()
    return x, w, b, g


def off(a, b):
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (3, 48, 64), (130, 256, 80), (517, 1280, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(M, N, K, dtype):
    x, w, b, g = tensors(M, N, K, dtype)
    r = seeded((M, N), 6, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = int8.int8_linear_train(*leaves)
    w8, sw = quant_rows(w.detach())
    assert torch.equal(y.detach(), int8_linear(x.detach(), w8, sw, bias=b.detach(), residual=r.detach()))
    gx, gw, gb, gr = torch.autograd.grad(y, leaves, g)
    assert all(t.dtype == s.dtype and t.shape == s.shape for t, s in zip((gx, gw, gb, gr), leaves))
    half = lambda t: to_np(t.detach().to(torch.bfloat16))  # noqa: E731
    # the e4m3 casts read the input as it is, the weight too
    want_x, want_w = fp8_linear_backward(to_np(g), to_np(x), to_np(w), "rowwise")
    for got, want in ((gx, want_x), (gw, want_w)):
        assert np.abs(to_np(got) - want).max() <= np.abs(want) .max() * (2.0 ** -8 + 1e-3)
    assert torch.equal(gr, g)
    s = g.double().sum(0).cpu().numpy()
    slack = np.abs(s) * 2.0 ** -8 + g.double().abs().sum(0).cpu().numpy() * M * 2.0 ** -24
    assert np.all(np.abs(to_np(gb).astype(np.float64) - s) <= slack)
    assert half(gx).shape == (M, K)


def test_gradients_are_near_the_linears_own_and_its_differences():
    x, w, b, g = tensors(300, 256, 512)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(int8.int8_linear_train(*leaves), leaves, g)
    xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
    for got, want in ((gx, gd @ wd), (gw, gd.t() @ xd)):
        assert off(got.double().cpu().numpy(), want.cpu().numpy()) < 0.06
    # along the gradient itself: (f(x + h d) - f(x - h d)) / 2 h of the linear that is quantised
    for leaf, grad, f in ((xd, gx, lambda t: (t @ wd.t() * gd).sum()), (wd, gw, lambda t: (xd @ t.t() * gd).sum())):
        d = grad.double() / grad.double().norm()
        slope = (f(leaf + 1e-3 * d) - f(leaf - 1e-3 * d)) / 2e-3
        assert abs(slope / (grad.double() * d).sum() - 1) < 0.06
    # the bias enters the output unquantised: its differences are the output's, to the roundings
    with torch.no_grad():
        up, down = (int8.int8_linear_train(x, w, b.float() + s) for s in (4.0, -4.0))
    slope = ((up.double() - down.double()) * gd).sum() / 8
    most = (gd.abs() * (up.double().abs() + down.double().abs())).sum() * 2.0 ** -8 / 8
    assert abs(slope - gb.double().sum()) <= most + gd.abs().sum() * 2.0 ** -8


@pytest.mark.parametrize("N,K", [(33, 80), (64, 40), (256, 128)])
def test_bf16_backward_of_odd_widths_and_on_request(N, K):
    x, w, b, g = tensors(65, N, K)
    mod = int8.Int8Linear(K, N, device="cuda", dtype=torch.bfloat16)
    mod.load_state_dict({"weight": w, "bias": b})
    mod.backward_fp8 = False
    x.requires_grad_()
    mod(x).backward(g)
    for got, want in ((x.grad, g.double() @ w.double()), (mod.weight.grad, g.double().t() @ x.detach().double())):
        assert off(got.double().cpu().numpy(), want.cpu().numpy()) < 2.0 ** -8
    if N % 16 or K % 16:                                               # the same without being asked
        plain = [t.detach().requires_grad_() for t in (x, w, b)]
        got = torch.autograd.grad(int8.int8_linear_train(*plain), plain, g)
        assert torch.equal(got[0], x.grad) and torch.equal(got[1], mod.weight.grad) and torch.equal(got[2], mod.bias.grad)


@pytest.mark.parametrize("M,N,K", [(1, 48, 64), (70, 48, 64), (70, 33, 40)])
def test_gradients_of_any_layout(M, N, K):
    """Inputs and an output's gradient that do not start on 16 bytes, with odd or no strides, or all one row: as their copies."""
    x, w, b, g = tensors(M, N, K)

    def grads(x, w, g):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = int8.int8_linear_train(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    def odd(t):
        out = torch.empty(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device="cuda")[:, :t.shape[1]]
        return out.copy_(t)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    def columns(t):
        return t.t().contiguous().t()

    one = seeded((N,), 9, torch.bfloat16)
    for a, v, h in ((odd(x), w, g), (shifted(x), shifted(w), shifted(g)), (x, odd(w), odd(g)), (columns(x), columns(w), columns(g)),
                    (x, w, one.expand(M, N)), (x, w, one[:1].expand(M, N)), (x[:1].expand(M, K), w, g)):
        for got, want in zip(grads(a, v, h), grads(a.contiguous().clone(), v.contiguous().clone(), h.contiguous().clone())):
            assert torch.equal(got, want)
    leaf = x.clone().requires_grad_()
    int8.int8_linear_train(leaf, w).sum(0).pow(2).sum().backward()                      # a gradient that autograd expands
    assert leaf.grad.any()


@pytest.mark.parametrize("shapes", [[(5, 8, 16)], [(300, 136, 304), (1, 64, 16)], [(517, 1280, 640), (1280, 640, 1280), (517, 640, 768)],
                                    [(256, 64, 256), (257, 72, 272), (600, 8, 608)]])
def test_casts_by_columns_together(shapes):
    """The casts of one to three matrices in one call: the bits of each one's own."""
    lib = _lib.load()
    xs = [seeded((r, c + 8), 20 + k, torch.bfloat16)[:, :c] for k, (r, c, _) in enumerate(shapes)]
    outs = [(torch.full((c, ld), 7, dtype=torch.uint8, device="cuda"), torch.zeros(c, device="cuda")) for _, c, ld in shapes]
    jobs = (_Job * 3)(*(_Job(x.data_ptr(), r, c, c + 8, o.data_ptr(), ld, s.data_ptr()) for x, (r, c, ld), (o, s) in zip(xs, shapes, outs)))
    ws = torch.full((sum(lib.flw_quant_cols_workspace_bytes(r, c) for r, c, _ in shapes),), 255, dtype=torch.uint8, device="cuda")
    _lib.check(lib.flw_quant_cols_e4m3_several(ctypes.byref(jobs), len(shapes), ws.data_ptr(), ws.numel(), _lib.stream_of(ws)), "several")
    for x, (_, _, ld), (o, s) in zip(xs, shapes, outs):
        want, scale = quantize_cols(x, "column", ld=ld)
        assert torch.equal(o, want.view(torch.uint8)) and torch.equal(s, scale)


@pytest.mark.parametrize("rows", [1, 3, 32, 33, 2048, 2049, 5000])
@pytest.mark.parametrize("cols,stride", [(1, 1), (7, 7), (8, 24), (513, 520), (1280, 1280)])
def test_column_sums(rows, cols, stride):
    """Chains of at most 32 + 3 + 3 + 16 additions in fp32 of any rows here, each off by 2^-24 of the absolute sum; then the type's
    rounding. The same bits every time."""
    lib = _lib.load()
    x = seeded((rows, stride), 8, torch.bfloat16)[:, :cols]
    want, total = x.double().sum(0), x.double().abs().sum(0)
    ws = torch.empty(lib.flw_col_sum_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    for dtype, code, half in ((torch.float32, _lib.F32, 0.0), (torch.bfloat16, _lib.BF16, 2.0 ** -8)):
        out = torch.full((2, cols + 1), 7.0, dtype=dtype, device="cuda")
        for o in out:
            ws.fill_(255)
            _lib.check(lib.flw_col_sum(x.data_ptr(), rows, cols, stride, o.data_ptr(), code, ws.data_ptr(), ws.numel(), _lib.stream_of(x)), "sum")
        assert torch.equal(out[0], out[1]) and (out[:, cols] == 7).all()
        assert ((out[0, :cols].double() - want).abs() <= want.abs() * half + total * 54 * 2.0 ** -24 * (1 + half)).all()


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (0, 2), (1, 3), (2, 3)])
@pytest.mark.parametrize("K", [64, 40])
def test_gradients_that_are_asked_for(which, K):
    """Any of the inputs alone, with and without a bias and a residual before it in the call: as in the call for all of them."""
    x, w, b, g = tensors(33, 48, K)
    given = [x, w, b, seeded((33, 48), 6, torch.bfloat16)]
    leaves = [t.clone().requires_grad_() for t in given]
    want = torch.autograd.grad(int8.int8_linear_train(*leaves), leaves, g)
    some = [t.clone().requires_grad_(i in which) for i, t in enumerate(given)]
    y = int8.int8_linear_train(*some)
    for got, i in zip(torch.autograd.grad(y, [some[i] for i in which], g), which):
        assert torch.equal(got, want[i])
    # all require gradients, some are taken
    got = torch.autograd.grad(int8.int8_linear_train(*leaves), [leaves[i] for i in which], g)
    assert all(torch.equal(got[n], want[i]) for n, i in enumerate(which))
    if 2 not in which:
        some = [t.clone().requires_grad_(i in which) for i, t in enumerate(given)]
        y = int8.int8_linear_train(some[0], some[1], None, some[3])
        for got, i in zip(torch.autograd.grad(y, [some[i] for i in which], g), which):
            assert torch.equal(got, want[i])


def test_second_derivatives_and_tangents_are_refused():
    x, w, b, g = tensors(3, 16, 16)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(int8.int8_linear_train(x, w), x, g, create_graph=True)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        int8.int8_linear_train(forward_ad.make_dual(x.detach(), x.detach()), w)
    y = int8.int8_linear_train(x, w.requires_grad_())
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)


def test_empty_batch():
    x, w, b, _ = tensors(4, 32, 48)
    leaves = [t.requires_grad_() for t in (x[:0].detach(), w, b)]
    y = int8.int8_linear_train(*leaves)
    assert y.shape == (0, 32)
    gx, gw, gb = torch.autograd.grad(y.sum(), leaves)
    assert gx.shape == (0, 48) and not gw.any() and not gb.any()


def test_module_and_weight_cache():
    x, w, b, g = tensors(130, 256, 512)
    lin = nn.Linear(512, 256, device="cuda", dtype=torch.bfloat16)
    lin.load_state_dict({"weight": w, "bias": b})
    mod = int8.Int8Linear.from_linear(lin)
    assert mod.weight is lin.weight
    x.requires_grad_()
    y = mod(x.view(2, 65, 512))
    y.backward(g.view(2, 65, 256))
    want = [t.clone() for t in (y.detach(), x.grad, mod.weight.grad, mod.bias.grad)]
    codes, scale = quant_rows(x.detach())
    assert torch.equal(mod.forward_codes(codes, scale), want[0].view(130, 256))
    r = seeded((130, 256), 7, torch.bfloat16)
    assert torch.equal(mod(x.detach(), residual=r), mod.forward_codes(codes, scale, residual=r))
    x.grad = mod.weight.grad = mod.bias.grad = None
    with fp8_weight_cache(nn.ModuleList([mod])):
        assert mod.weight_codes()[0].dtype == torch.int8
        for _ in range(2):
            x.grad = mod.weight.grad = mod.bias.grad = None
            y = mod(x.view(2, 65, 512))
            y.backward(g.view(2, 65, 256))
            assert all(torch.equal(p, q) for p, q in zip((y.detach(), x.grad, mod.weight.grad, mod.bias.grad), want))
        assert torch.equal(mod.forward_codes(codes, scale), want[0].view(130, 256))
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        assert torch.equal(mod(x.float()), want[0].view(130, 256))
    with pytest.raises(RuntimeError, match="stale"):
        with fp8_weight_cache(nn.ModuleList([mod])):
            mod.weight.data += 1


def test_training_step_in_a_graph():
    x, w, _, g = tensors(64, 128, 256)
    lin = int8.Int8Linear(256, 128, bias=False, device="cuda", dtype=torch.bfloat16)
    lin.weight.data.copy_(w)
    held = x.detach().clone().requires_grad_()

    def step():
        return torch.autograd.grad(lin(held), [held, lin.weight], g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        with torch.no_grad():
            held.copy_(seeded((64, 256), 30 + seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        own = held.detach().clone().requires_grad_()
        y = lin(own)
        want = torch.autograd.grad(y, [own, lin.weight], g)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
