"""GPU: a captured step goes on reading its rotary tables when the module is used at other lengths afterwards."""

import pytest
import torch

from gpu_util import seeded
from test_attention_host import _cfg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg", [dict(), dict(rope_layout="half", rope_dim=32)], ids=["plain", "half"])
@torch.no_grad()
def test_a_captured_step_after_longer_and_shorter_ones(cfg):
    from flower_amd.attention import CausalSelfAttention
    from flower_amd.kv_cache import PagedKVCache
    torch.manual_seed(0)
    m = CausalSelfAttention(_cfg(attn_precision="bf16", max_seq_len=32, **cfg), local_window=16).cuda().bfloat16()

    def cache_of(n):
        return PagedKVCache(1, 20, 2, 64, sequences=2, max_len=n, page_size=16, window=16)

    cache, twin = cache_of(64), cache_of(64)
    gate = torch.zeros(2, dtype=torch.int32, device="cuda")
    x, y = torch.zeros((2, 1, 128), dtype=torch.bfloat16, device="cuda"), seeded((2, 20, 128), 5, torch.bfloat16)

    def step(c):
        c.reserve(gate)
        return m.forward_cached(x, c, 0), m(y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(cache)                                  # (changes nothing: no token is granted)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    gate.fill_(1)
    for n in range(6):
        other = cache_of(200 * (n + 1))                  # longer than the tables, and the last ones
        other.reserve(7)
        m.forward_cached(seeded((2, 7, 128), 40 + n, torch.bfloat16), other, 0)
        m(seeded((1, 50 + n, 128), 60 + n, torch.bfloat16))
        junk = [torch.full((n + 1, 64, 64), float("nan"), device="cuda") for _ in range(50)]     # what was freed is taken again
        x.copy_(seeded((2, 1, 128), 20 + n, torch.bfloat16))
        graph.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and bool(torch.isfinite(out[0]).all()), n
        del junk
