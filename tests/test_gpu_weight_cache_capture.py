"""GPU: the weight cache's transposed codes, first asked for while a graph is captured."""

import gc

import pytest
import torch

from flower_amd.int8 import Int8Linear
from flower_amd.precision import Fp8Linear, fp8_weight_cache
from tests.gpu_util import seeded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["int8", "rowwise", "tensorwise"])
def test_a_capture_leaves_no_codes_behind_that_were_never_made(kind):
    """A captured call records the codes' kernels and does not run them: a later call outside of the graph makes its own."""
    x, g = seeded((64, 256), 1, torch.bfloat16), seeded((64, 128), 2, torch.bfloat16)
    lin = (Int8Linear(256, 128, bias=False, device="cuda", dtype=torch.bfloat16) if kind == "int8" else
           Fp8Linear(256, 128, bias=False, device="cuda", dtype=torch.bfloat16, recipe=kind))
    leaf = x.clone().requires_grad_()

    def step():
        return torch.autograd.grad(lin(leaf), leaf, g)[0]

    want = step()
    lin.weight_col_codes()                             # no cache is active: nothing is kept
    torch.cuda.synchronize()
    gc.collect()                                       # no graph is let go while another is captured
    same = []
    with fp8_weight_cache(torch.nn.ModuleList([lin])):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        same.append(torch.equal(step(), want))
        for _ in range(3):
            held.zero_()
            graph.replay()
            torch.cuda.synchronize()
            same += [torch.equal(held, want), torch.equal(step(), want)]
        del graph, held
    assert same == [True] * 7
