"""CPU: what the 8-bit rows and the int8 product refuse, and Int8Linear's conversion rules."""

import ctypes

import pytest
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from flower_amd import int8
from flower_amd.kernels import gelu_quant, int8_linear, int8_scaled_mm, quant_rows, rms_norm_quant, swiglu_quant

X, W = torch.zeros(2, 3, 8), torch.ones(8)
CODES, S = torch.zeros(3, 8, dtype=torch.int8), torch.ones(3)
B8, BS = torch.zeros(5, 8, dtype=torch.int8), torch.ones(5)


def every(x=X):
    return [lambda **k: quant_rows(x, **k), lambda **k: rms_norm_quant(x, W, **k), lambda **k: gelu_quant(x, **k),
            lambda **k: swiglu_quant(x, x, **k)]


def test_good_calls_reach_the_gpu_check():
    for call in (*every(), lambda: rms_norm_quant(X, W, residual=X), lambda: int8_scaled_mm(CODES, S, B8, BS),
                 lambda: int8_linear(X, B8, BS, bias=torch.ones(5), residual=torch.zeros(2, 3, 5).bfloat16())):
        with pytest.raises(RuntimeError, match="only on a ROCm GPU"):
            call()


def test_rows_refuse_types_and_shapes():
    for call in every():
        with pytest.raises(ValueError, match="int8 or float8_e4m3fn"):
            call(dtype=torch.uint8)
    for x in (torch.zeros(3, 8, dtype=torch.float16), torch.zeros(3, 8, dtype=torch.int32)):
        for call in every(x):
            with pytest.raises(TypeError, match="bfloat16 or float32"):
                call()
    for x in (torch.zeros(3, 0), torch.zeros(())):
        for call in every(x):
            with pytest.raises(ValueError, match="K > 0"):
                call()
    for w in (torch.ones(7), torch.ones(1, 8), torch.ones(8, dtype=torch.float64), torch.ones(8).bfloat16()):
        with pytest.raises(ValueError, match="weight must be"):
            rms_norm_quant(X, w)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            rms_norm_quant(X, W, eps)
    for r in (torch.zeros(3, 8), X.bfloat16()):
        with pytest.raises(ValueError, match="residual must be"):
            rms_norm_quant(X, W, residual=r)
        with pytest.raises(ValueError, match="up must be"):
            swiglu_quant(X, r)


def test_the_product_refuses_types_and_shapes():
    with pytest.raises(TypeError, match="int8 codes"):
        int8_scaled_mm(CODES.to(torch.uint8), S, B8, BS)
    bad = [dict(weight=B8.to(torch.uint8)), dict(weight=B8[:, :7]), dict(weight=B8[0]), dict(weight=B8[:0]), dict(a_scale=torch.ones(2)),
           dict(a_scale=S.double()), dict(weight_scale=torch.ones(4)), dict(weight_scale=torch.ones(10)[::2]), dict(bias=torch.ones(4)),
           dict(bias=torch.ones(5, dtype=torch.float16)), dict(residual=torch.zeros(3, 5)), dict(residual=torch.zeros(2, 5).bfloat16())]
    for change in bad:
        with pytest.raises(ValueError, match="int8_scaled_mm: "):
            int8_scaled_mm(**{**dict(a=CODES, a_scale=S, weight=B8, weight_scale=BS), **change})
        if "a_scale" not in change:
            with pytest.raises(ValueError, match="int8_linear: "):
                int8_linear(**{**dict(x=X, weight=B8, weight_scale=BS), **change})
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        int8_linear(CODES, B8, BS)


def test_gradients_and_tangents_are_refused_not_dropped():
    x, w, s = X.clone().requires_grad_(), W.clone().requires_grad_(), BS.clone().requires_grad_()
    calls = [*every(x), lambda: rms_norm_quant(X, w), lambda: rms_norm_quant(X, W, residual=x), lambda: swiglu_quant(X, x),
             lambda: int8_linear(x, B8, BS), lambda: int8_linear(X, B8, s), lambda: int8_linear(X, B8, BS, bias=s),
             lambda: int8_scaled_mm(CODES, S, B8, s)]
    for call in calls:
        with pytest.raises(RuntimeError, match="forward-only"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="only on a ROCm GPU"):
            call()
    with forward_ad.dual_level():
        for call in every(forward_ad.make_dual(X, X)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_int8_linear_train_refuses():
    for x, w in ((X, torch.ones(5, 7)), (X, W), (torch.zeros(()), torch.ones(5, 8)), (X, torch.ones(5, 8, device="meta"))):
        with pytest.raises(ValueError, match="takes a weight"):
            int8.int8_linear_train(x, w)
    with pytest.raises(RuntimeError, match="only on a ROCm GPU"):
        int8.int8_linear_train(X, torch.ones(5, 8))
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        int8.int8_linear_train(X, torch.ones(5, 8).half())


class Model(nn.Module):
    def __init__(self, blocks=4):
        super().__init__()
        self.blocks = nn.ModuleList(nn.ModuleDict({"a": nn.Linear(32, 48), "odd": nn.Linear(32, 40)}) for _ in range(blocks))
        self.head = nn.Linear(32, 64)


def test_conversion_shares_parameters_and_follows_the_filter():
    m = Model()
    weight = m.blocks[1]["a"].weight
    m, info = int8.convert_model_to_int8(m, verbose=False)
    assert info == {"int8_keep_bf16_blocks": 1, "int8_converted_linears": 2, "int8_total_linears": 9}
    assert [type(b["a"]) is int8.Int8Linear for b in m.blocks] == [False, True, True, False]
    assert type(m.blocks[1]["odd"]) is nn.Linear and type(m.head) is nn.Linear
    assert m.blocks[1]["a"].weight is weight and "recipe=int8" in repr(m.blocks[1]["a"])
    with pytest.raises(RuntimeError, match="no `blocks`"):
        int8.convert_model_to_int8(nn.Linear(32, 32), verbose=False)
    with pytest.raises(RuntimeError, match="tensorwise"):
        m.blocks[1]["a"].tensorwise_codes()


def test_c_entries_refuse_on_the_host():
    """Sizes, strides, types and workspaces that no kernel takes (made-up aligned addresses: only where no GPU is visible)."""
    if torch.cuda.is_available():
        pytest.skip("passes fake device pointers: CPU-only host check")
    from flower_amd import _lib
    lib, P = _lib.load(), 1 << 20
    rows = lambda **k: lib.flw_rows8(*{**dict(x=P, dtype=1, rows=2, cols=64, xs=64, type=3, codes=P, cs=64, scale=P, stream=None), **k}.values())  # noqa: E731
    for change, rc in ((dict(x=None), 1), (dict(dtype=3), 2), (dict(cols=0), 1), (dict(cols=32769, xs=32769, cs=32769), 2), (dict(xs=63), 1),
                       (dict(type=1), 2), (dict(cs=63), 1), (dict(scale=None), 1), (dict(rows=-1), 1), (dict(rows=2 ** 31), 2),
                       (dict(x=P + 1), 1)):
        assert rows(**change) == rc, change
    assert rows(rows=0, x=None) == 0
    for cols, most in ((512, 2 ** 26), (2048, 2 ** 26), (8192, 2 ** 24), (8200, 2 ** 22)):        # a launch's 2^32 threads
        assert rows(rows=most, cols=cols, xs=cols, cs=cols) == 2, cols
    norm = lambda **k: lib.flw_rows8_rmsnorm(*{**dict(x=P, a=P, dtype=1, rows=2, cols=64, xs=64, as_=64, w=P, wd=1, eps=0.0, sum=P, ss=64, type=3,  # noqa: E731
                                                      codes=P, cs=64, scale=P, stream=None), **k}.values())
    for change, rc in ((dict(sum=None), 1), (dict(w=None), 1), (dict(wd=2), 2), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(as_=8), 1), (dict(ss=8), 1),
                       (dict(dtype=0, wd=1), 2)):
        assert norm(**change) == rc, change
    mm = lambda **k: lib.flw_int8_scaled_mm(*{**dict(a=P, M=2, K=64, as_=64, b=P, N=8, bs=64, sa=P, sac=2, sb=P, sbc=8, bias=None, bd=1, res=None,  # noqa: E731
                                                     rs=0, y=P, ys=8, stream=None), **k}.values())
    for change, rc in ((dict(a=None), 1), (dict(K=0), 1), (dict(K=131072, as_=131072, bs=131072), 2), (dict(sac=3), 1), (dict(sbc=2), 1),
                       (dict(as_=63), 1), (dict(ys=7), 1), (dict(res=P, rs=7), 1), (dict(bias=P, bd=2), 1), (dict(bias=P + 1), 1),
                       (dict(y=P + 1), 1), (dict(M=-1), 1), (dict(N=2 ** 31), 2)):
        assert mm(**change) == rc, change
    assert mm(M=0, a=None, sac=0) == 0
    assert mm(M=2 ** 30, sac=1, N=64, sbc=1, ys=64, K=65, as_=65, bs=65) == 2 and b"tiles" in lib.flw_last_error()
    need = lib.flw_int8_linear_workspace_bytes(3, 65)
    assert need == 3 * 80 + 12
    lin = lambda **k: lib.flw_int8_linear(*{**dict(x=P, dtype=1, M=3, K=65, xs=65, b=P, N=8, bs=65, sb=P, sbc=8, bias=None, bd=1, res=None, rs=0, y=P,  # noqa: E731
                                                   ys=8, ws=P, wb=need, stream=None), **k}.values())
    for change, rc in ((dict(wb=need - 1), 3), (dict(ws=None), 3), (dict(ws=P + 8), 3), (dict(K=0), 1), (dict(M=-1), 1)):
        assert lin(**change) == rc, change
    act = lambda **k: lib.flw_rows8_swiglu(*{**dict(x=P, u=P, dtype=1, rows=2, cols=64, xs=64, us=64, type=2, codes=P, cs=64, scale=P, stream=None),  # noqa: E731
                                             **k}.values())
    for change, rc in ((dict(u=None), 1), (dict(us=63), 1), (dict(u=P + 1), 1), (dict(dtype=2), 2), (dict(type=0), 2)):
        assert act(**change) == rc, change
    assert lib.flw_rows8_gelu(P, 1, 2, 64, 63, 3, P, 64, P, None) == 1
    # chunks of 32 rows, of 128 from 2049 rows on
    assert [lib.flw_col_sum_workspace_bytes(r, 5) for r in (0, 1, 33, 2048, 2049)] == [0, 20, 40, 1280, 340]
    tot = lambda **k: lib.flw_col_sum(*{**dict(x=P, rows=3, cols=5, xs=5, out=P, dtype=0, ws=P, wb=20, stream=None), **k}.values())  # noqa: E731
    for change, rc in ((dict(x=None), 1), (dict(out=None), 1), (dict(rows=0), 1), (dict(cols=0), 1), (dict(xs=4), 1), (dict(dtype=3), 2), (dict(wb=19), 3),
                       (dict(ws=None), 3), (dict(ws=P + 4), 3), (dict(x=P + 1), 1), (dict(out=P + 2), 1), (dict(rows=2 ** 24, wb=2 ** 30), 2)):
        assert tot(**change) == rc, change

    class Job(ctypes.Structure):
        _fields_ = [("x", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                    ("out_t", ctypes.c_void_p), ("ld", ctypes.c_int64), ("scale_out", ctypes.c_void_p)]

    size = lib.flw_quant_cols_workspace_bytes(20, 64)
    good = dict(x=P, rows=20, cols=64, row_stride=64, out_t=P, ld=32, scale_out=P)

    def casts(count=2, ws=P, wb=2 * size, **change):
        jobs = (Job * 2)(Job(*good.values()), Job(*{**good, **change}.values()))
        return lib.flw_quant_cols_e4m3_several(ctypes.byref(jobs), count, ws, wb, None)

    for change, rc in ((dict(x=None), 1), (dict(out_t=None), 1), (dict(scale_out=None), 1), (dict(rows=0), 1), (dict(cols=0), 1), (dict(cols=60), 1),
                       (dict(row_stride=56), 1), (dict(row_stride=68), 1), (dict(x=P + 8), 1), (dict(out_t=P + 8), 1), (dict(ld=16), 1),
                       (dict(ld=24), 1), (dict(rows=2 ** 40, ld=2 ** 40), 2), (dict(count=0), 1), (dict(count=4), 1), (dict(ws=None), 3),
                       (dict(wb=2 * size - 1), 3)):
        assert casts(**change) == rc, change
