"""CPU: what an int8 linear's training takes, refused before its forward rather than behind it, and which linears are
converted."""

import pytest
import torch
import torch.nn as nn

from flower_amd import int8

MOST = 65535 * 256                      # fp32 rows of one cast by columns


def test_float32_rows_that_the_backward_cannot_cast_are_refused_at_once():
    """Views of one row: no memory."""
    row, w = torch.zeros(1, 16), torch.ones(16, 16)
    many, wide = row.expand(MOST + 1, 16), torch.ones(1, 16).expand(MOST + 16 - MOST % 16, 16)
    leaf = lambda t: t.detach().requires_grad_()  # noqa: E731
    for x, v in ((many, leaf(w)), (leaf(many), leaf(w)), (many.view(1, -1, 16), leaf(w)), (leaf(row), wide)):
        with pytest.raises(ValueError, match="at most 16776960 float32 rows"):
            int8.int8_linear_train(x, v)
    # taken: as many, bfloat16, where the cast is not needed, and where the gradients are no e4m3 products
    for x, v in ((row.expand(MOST, 16), leaf(w)), (row.bfloat16().expand(MOST + 1, 16), leaf(w)), (leaf(many), w), (row, leaf(wide)),
                 (many[:, :8], leaf(w[:, :8])), (many, w)):
        with pytest.raises(RuntimeError, match="only on a ROCm GPU"):
            int8.int8_linear_train(x, v)


def test_linears_too_wide_for_a_row_stay_as_they_are():
    wide = nn.Linear(32784, 16, device="meta")
    with pytest.raises(ValueError, match="at most 32768 input features, got 32784"):
        int8.Int8Linear.from_linear(wide)
    with pytest.raises(ValueError, match="at most 32768 input features, got 32784"):
        int8.Int8Linear(32784, 16, device="meta")
    m = nn.Module()
    m.blocks = nn.ModuleList([nn.ModuleDict({"wide": wide, "full": nn.Linear(32768, 16, device="meta"),
                                             "out": nn.Linear(16, 65536, device="meta")})])
    m, info = int8.convert_model_to_int8(m, keep_bf16_blocks=0, verbose=False)
    assert info["int8_converted_linears"] == 2 and m.blocks[0]["wide"] is wide
    assert type(m.blocks[0]["full"]) is type(m.blocks[0]["out"]) is int8.Int8Linear
