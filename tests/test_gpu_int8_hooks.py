"""GPU: what a user hangs on a converted block's modules runs without gradients as it runs with them."""

import pytest
import torch

from flower_amd import int8
from flower_amd.kv_cache import PagedKVCache
from flower_amd.precision import fp8_weight_cache
from tests.gpu_util import seeded
from tests.test_gpu_int8_block import model

pytestmark = pytest.mark.gpu

GATED = ["attn", "attn.qkv", "attn.out", "ff", "ff.gate", "ff.up", "ff.down"]
GELU = ["attn", "ff", "ff.net", "ff.net.0", "ff.net.1", "ff.net.2", "ff.net.3"]


def converted(gelu):
    m = model(ffn_activation="gelu" if gelu else "swiglu")
    return int8.convert_model_to_int8(m, keep_bf16_blocks=0, verbose=False)[0]


def modules_route(block, x):
    """The modules one after the other, as with gradients."""
    with torch.enable_grad():
        return block(x)[0].detach()


def cached_step(block, x):
    cache = PagedKVCache(1, 64, 4, 64, sequences=x.shape[0], max_len=128, page_size=16, window=128)
    cache.reserve([x.shape[1]] * x.shape[0])
    return block.forward_cached(x, cache, 0)


@pytest.mark.parametrize("name,gelu", [(n, False) for n in GATED] + [(n, True) for n in GELU])
@pytest.mark.parametrize("how", ["hook", "pre-hook", "forward"])
@torch.no_grad()
def test_hooks_and_own_forwards_run(name, gelu, how):
    b, x, seen = converted(gelu).blocks[0], seeded((2, 40, 256), 1, torch.bfloat16), []
    fused = b(x)[0]
    mod = b.get_submodule(name)
    if how == "hook":
        handle = mod.register_forward_hook(lambda m, a, out: seen.append(m))
    elif how == "pre-hook":
        handle = mod.register_forward_pre_hook(lambda m, a: seen.append(m))
    else:
        own = mod.forward
        mod.forward = lambda *a, **k: (seen.append(mod), own(*a, **k))[1]
    y = b(x)[0]
    assert seen == [mod]
    assert torch.equal(y, modules_route(b, x)) and seen == [mod, mod]
    if name != "attn":                                 # forward_cached is another method of it
        cached_step(b, x)
        assert seen == [mod] * 3
    if how == "forward":
        del mod.forward
    else:
        handle.remove()
    assert torch.equal(b(x)[0], fused)


@torch.no_grad()
def test_a_hook_changes_the_output():
    b, x = converted(False).blocks[0], seeded((2, 40, 256), 1, torch.bfloat16)
    b.ff.register_forward_hook(lambda m, a, out: torch.zeros_like(out))
    assert not b(x)[0].any() and not cached_step(b, x).any()


@torch.no_grad()
def test_hooks_of_every_module_run():
    b, x, seen = converted(False).blocks[0], seeded((2, 40, 256), 1, torch.bfloat16), []
    fused = b(x)[0]
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: seen.append(m))
    try:
        b(x)
    finally:
        handle.remove()
    assert all(b.get_submodule(n) in seen for n in GATED)
    assert torch.equal(b(x)[0], fused)


@torch.no_grad()
def test_other_modules_in_their_places_run():
    """Subclasses and modules put in the place of the block's own."""
    b, x = converted(True).blocks[0], seeded((2, 40, 256), 1, torch.bfloat16)

    class Twice(type(b.attn)):
        def forward(self, *a, **k):
            return 2 * super().forward(*a, **k)

    b.attn.__class__ = Twice
    assert torch.equal(b(x)[0], modules_route(b, x))
    b = converted(True).blocks[0]
    b.ff.net[1] = torch.nn.GELU(approximate="tanh")
    assert torch.equal(b(x)[0], modules_route(b, x))
    b.ff.net[1] = torch.nn.ReLU()
    assert torch.equal(b(x)[0], modules_route(b, x))
    b.ff.net = torch.nn.Linear(256, 256, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(b(x)[0], modules_route(b, x))
    b = converted(False).blocks[0]
    b.ff.down = torch.nn.Sequential(b.ff.down)
    assert torch.equal(b(x)[0], modules_route(b, x))


@torch.no_grad()
def test_the_weight_cache_keeps_the_int8_route():
    m, x = converted(False), seeded((2, 40, 256), 1, torch.bfloat16)
    b = m.blocks[0]
    fused, apart = b(x)[0], modules_route(b, x)
    assert not torch.equal(fused, apart)               # the norms' roundings
    for _ in range(2):
        with fp8_weight_cache(m):
            assert torch.equal(b(x)[0], fused)
        assert torch.equal(b(x)[0], fused)
    with fp8_weight_cache(m):
        b.ff.up.register_forward_hook(lambda mod, a, out: 0 * out)
        assert torch.equal(b(x)[0], modules_route(b, x))
