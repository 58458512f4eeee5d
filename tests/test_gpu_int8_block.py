"""GPU: a model's blocks on int8 linears, as they are used: converted, with a prompt and decode steps over a paged cache, eager and in
a captured graph.

The route is the operators' calls one after the other, to the bit. Against the unconverted block: an int8 linear's output is off by
1.3 % of its size (each operand's values by a uniform half step, 4 / 127 / sqrt 12 of sigma), and three follow on each other in a
residual branch, the norm and the attention passing an error on as it is; the branches are added to a stream of at least their size.
sqrt 3 * 1.3 % = 2.3 % of a branch each, twice in a block: 3.2 %, so 4 % is asked of the block's own addition, y - x, for one block.
"""

import pytest
import torch
import torch.nn as nn

from flower_amd import int8
from flower_amd.block import TransformerBlock, block_config
from flower_amd.kernels import gelu_quant, rms_norm_quant, swiglu_quant
from flower_amd.kv_cache import PagedKVCache
from flower_amd.precision import fp8_weight_cache
from tests.gpu_util import seeded

pytestmark = pytest.mark.gpu


class Model(nn.Module):
    def __init__(self, layers, **config):
        super().__init__()
        self.blocks = nn.ModuleList(TransformerBlock(block_config(max_seq_len=512, **config)) for _ in range(layers))


def model(layers=1, **config):
    torch.manual_seed(3)
    m = Model(layers, **{**dict(d_model=256, num_heads=4, ffn_dim=768, local_window=128), **config})
    for mod in m.modules():
        if isinstance(mod, nn.Linear):
            nn.init.normal_(mod.weight, std=mod.in_features ** -0.5)
            if mod.bias is not None:
                nn.init.normal_(mod.bias, std=0.1)
    for b in m.blocks:
        nn.init.normal_(b.ln1.weight, 1.0, 0.1)
        nn.init.normal_(b.ln2.weight, 1.0, 0.1)
    return m.cuda().to(torch.bfloat16)


def off(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm()).item()


@pytest.mark.parametrize("config", [dict(), dict(ffn_activation="gelu", use_bias=True), dict(d_model=320, num_heads=5, qk_norm=False)])
@torch.no_grad()
def test_forward(config):
    m = model(**config)
    x = seeded((3, 77, m.blocks[0].attn.qkv.in_features), 1, torch.bfloat16)
    want = m.blocks[0](x)[0]
    int8.convert_model_to_int8(m, keep_bf16_blocks=0, verbose=False)
    b = m.blocks[0]
    got = b(x)[0]
    assert off(got - x, want - x) < 0.04
    # the calls one by one
    c, s = rms_norm_quant(x, b.ln1.weight, b.ln1.eps)
    a = b.attn.out(b.attn.attend(*b.attn.heads(b.attn.qkv.forward_codes(c, s))))
    c, s, t = rms_norm_quant(x, b.ln2.weight, b.ln2.eps, residual=a)
    assert torch.equal(t, x + a)
    if b.ff.activation == "gelu":
        c, s = gelu_quant(b.ff.net[0].forward_codes(c, s))
    else:
        c, s = swiglu_quant(b.ff.gate.forward_codes(c, s), b.ff.up.forward_codes(c, s))
    assert torch.equal(got, b.ff.linears()[-1].forward_codes(c, s, residual=t))
    # with gradients the modules run one after the other, the norms' outputs rounded to bf16 (2^-8 at most) on the way: the same
    # approximation as above of the same block. Between the two routes the weights' codes are the same and the activations' half
    # steps, 4 / 127 / sqrt 12 = 0.9 % of sigma, are each route's own once a value has moved by a fraction of a step:
    # sqrt 2 * 0.9 % = 1.3 % a linear, as between a linear and its int8 form, and the rest of the sum is the same: 4 % again
    with torch.enable_grad():
        y = b(x)[0]
    assert y.requires_grad and off(y.detach() - x, want - x) < 0.04 and off(y.detach() - x, got - x) < 0.04


def test_training_reaches_every_parameter():
    m = model(ffn_activation="gelu", use_bias=True)
    plain = model(ffn_activation="gelu", use_bias=True)
    int8.convert_model_to_int8(m, keep_bf16_blocks=0, verbose=False)
    x = seeded((2, 64, 256), 2, torch.bfloat16)
    g = seeded((2, 64, 256), 3, torch.bfloat16)
    grads = []
    for net in (m, plain):
        leaf = x.clone().requires_grad_()
        net.blocks[0](leaf)[0].backward(g)
        grads.append({"x": leaf.grad, **{n: p.grad for n, p in net.named_parameters()}})
    for name, want in grads[1].items():
        # e4m3 products, 5.1 % each, and the forward's 1.3 %, through at most four linears of a branch
        assert off(grads[0][name], want) < 0.12, name


@torch.no_grad()
@pytest.mark.parametrize("pages", [torch.bfloat16, torch.float8_e4m3fn])
def test_decoding(pages):
    m = model(2)
    B, lens = 5, [40, 3, 64, 17, 1]
    x = seeded((B, 64, 256), 4, torch.bfloat16)
    steps = [seeded((B, 1, 256), 10 + i, torch.bfloat16) for i in range(6)]

    def decode(net, graphed):
        cache = PagedKVCache(2, 64, 4, 64, sequences=B, max_len=256, page_size=16, dtype=pages, window=128)
        cache.reserve(lens)

        def run(h, prompt):
            for i, block in enumerate(net.blocks):
                h = block.forward_cached(h, cache, i, prompt=prompt)
            return h

        out = [run(x, True)]
        held, one = steps[0].clone(), torch.ones(B, dtype=torch.int32, device="cuda")
        if graphed:                                     # what a step needs once is made before the capture; the step is taken back
            cache.reserve(one)
            run(held, False)
            cache.take_back(one)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                cache.reserve(one)
                y = run(held, False)
        for s in steps:
            held.copy_(s)
            if graphed:
                graph.replay()
                torch.cuda.synchronize()
            else:
                cache.reserve(one)
                y = run(held, False)
            out.append(y.clone())
        return out

    want = decode(m, False)
    int8.convert_model_to_int8(m, keep_bf16_blocks=0, verbose=False)
    with fp8_weight_cache(m):
        eager, replayed = decode(m, False), decode(m, True)
    again = decode(m, False)                            # the weights quantised at every call
    for b, n in enumerate(lens):
        assert torch.equal(eager[0][b, :n], again[0][b, :n]) and torch.equal(eager[0][b, :n], replayed[0][b, :n])
        assert off(eager[0][b, :n], want[0][b, :n]) < 0.06
    for e, r, a, w in zip(eager[1:], replayed[1:], again[1:], want[1:]):
        assert torch.equal(e, r) and torch.equal(e, a)
        assert off(e, w) < 0.06                         # two blocks' 4 %, of a stream that holds more than what they add


@torch.no_grad()
def test_a_sequence_decodes_alone_as_in_a_batch():
    """Every linear gives a row the same bits in any batch, and the paged attention is each sequence's own."""
    m = model(1)
    int8.convert_model_to_int8(m, keep_bf16_blocks=0, verbose=False)
    x, token = seeded((6, 48, 256), 5, torch.bfloat16), seeded((6, 1, 256), 6, torch.bfloat16)

    def last(rows):
        cache = PagedKVCache(1, 64, 4, 64, sequences=len(rows), max_len=128, page_size=16, window=128)
        cache.reserve(48)
        m.blocks[0].forward_cached(x[rows], cache, 0)
        cache.reserve(1)
        return m.blocks[0].forward_cached(token[rows], cache, 0)

    whole = last(list(range(6)))
    for b in (0, 3, 5):
        assert torch.equal(last([b])[0], whole[b])
