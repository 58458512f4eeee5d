"""GPU: the cache's operators as a model runs them together: PagedKVCache, the attention module's and the block's cached
forward, a captured decode step, and the rotary options of the module.

Tolerances. The attention of written keys and values: test_gpu_paged's (2^-8 of the value for the rounding to bf16, on
sum p |v| / sum p the weights' 2^-15 and `slack`). The module against the definition from its exact inputs: besides these, q
and k are rounded to bf16 (half a step each: 2^-8 of the value, so 2^-7 of sum |q k| scale =: delta on a score, and 2^-14 of
it both at once), so that a weight is off by exp(2 delta) - 1 relative to the sum, which the output's size takes; an e4m3
cache's keys and values by 2^-4 instead, 2^-10 scale below the normal range.
"""

import numpy as np
import pytest
import torch

from oracle import paged as O

from gpu_util import seeded, to_np
from test_attention_host import _cfg

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().cpu().float().numpy().astype(np.float64)


def within(got, want, size, slack):
    ok = np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + size * (2.0 ** -15 + 2 * slack)
    assert ok.all(), (int((~ok).sum()), np.argwhere(~ok)[:4], got[~ok][:4], want[~ok][:4])


# ---------------------------------------------------------------- a run of the operators

@pytest.mark.parametrize("dtype,window", [(torch.bfloat16, None), (torch.bfloat16, 21), (torch.float8_e4m3fn, None)])
def test_a_run_of_reserve_append_attend_fork_free_and_compact(dtype, window):
    """Random steps of a server: tokens, forks, drops, compactions. Beside the cache each sequence's keys and values as
    they were written, in plain lists; every answer is checked against those. The pool is kept nearly full, so that some
    sequences are refused room; nothing but the granted counts tells the lists so."""
    from flower_amd.kv_cache import PagedKVCache
    rng = np.random.default_rng(5)
    S, H, KV, D, L, page = 5, 4, 2, 64, 2, 16
    scales = dict(k_scale=torch.rand(L, KV) / 8 + 0.05, v_scale=torch.rand(L, KV) / 8 + 0.05) if dtype != torch.bfloat16 else {}
    cache = PagedKVCache(L, 17, KV, D, sequences=S, max_len=160, page_size=page, dtype=dtype, window=window, **scales)
    cache.k_pages.view(torch.uint8).fill_(0xFF)              # NaN in every place that nothing is written to
    cache.v_pages.view(torch.uint8).fill_(0xFF)
    keys = [[(np.zeros((0, KV, D)),) * 2 for _ in range(S)] for _ in range(L)]          # [layer][place]: (k, v) of all positions
    granted_some = refused_some = 0
    for step in range(40):
        kind = rng.integers(0, 10)
        if kind == 0:
            parents = rng.integers(-1, S, S)
            cache.reorder(parents.tolist())
            kept = to_np(cache.lens)
            keys = [[row[p] if p >= 0 and kept[s] > 0 else (np.zeros((0, KV, D)),) * 2 for s, p in enumerate(parents)] for row in keys]
        elif kind == 1:
            s = int(rng.integers(0, S))
            cache.free([s])
            for row in keys:
                row[s] = (np.zeros((0, KV, D)),) * 2
        elif kind == 2:
            live = int(cache.compact())
            assert live == int((cache.refs > 0).sum()) and bool((cache.refs[:live] > 0).all())
        T = int(rng.choice([1, 1, 1, 4, 23]))
        want = rng.integers(0, T + 1, S) if T > 1 else rng.integers(0, 2, S)
        counts = to_np(cache.reserve(want.tolist()))
        assert ((counts == want) | (counts == 0)).all()
        granted_some += int((counts > 0).sum())
        refused_some += int(((counts == 0) & (want > 0)).sum())
        x = [seeded((S, T, H + 2 * KV, D), 100 * step + i, torch.bfloat16).transpose(1, 2) for i in range(L)]
        for layer in range(L):
            y = x[layer]
            q, k = cache.append(layer, y[:, :H], y[:, H:H + KV], y[:, H + KV:], norm_eps=1e-6, return_k=True)
            out = f64(cache.attend(layer, q))
            kn, vn = f64(k), f64(y[:, H + KV:])
            for s in range(S):
                n = int(counts[s])
                if scales:      # what the codes hold, rounded from fp32 (k is not: to bf16 first), within half a step of k, v
                    at = int(cache.lens[s]) - n + torch.arange(n, device="cuda")
                    ids, off = cache.tables[s].long()[at // page], at % page
                    for new, pages, scale in ((kn, cache.k_pages[layer][ids, :, off], scales["k_scale"][layer]),
                                              (vn, cache.v_pages[layer].transpose(-1, -2)[ids, :, off], scales["v_scale"][layer])):
                        scale = scale.double().numpy()[None, :, None]
                        code = f64(pages) * scale
                        value = np.clip(new[s, :, :n].transpose(1, 0, 2), -448 * scale, 448 * scale)
                        assert (np.abs(code - value) <= (2.0 ** -4 + 2.0 ** -7) * np.abs(value) + 2.0 ** -10 * scale).all()
                        new[s, :, :n] = code.transpose(1, 0, 2)
                old = keys[layer][s]
                keys[layer][s] = new = (np.concatenate([old[0], kn[s, :, :n].transpose(1, 0, 2)]),
                                        np.concatenate([old[1], vn[s, :, :n].transpose(1, 0, 2)]))
                total = len(new[0])
                assert int(cache.lens[s]) == total
                if total == 0 or n == 0:
                    assert (out[s] == 0).all()
                    continue
                # the sequence alone, in one page that holds it whole
                want_o, _, size, slack = O.attention(f64(q[s:s + 1]), new[0].transpose(1, 0, 2)[None], new[1].transpose(1, 2, 0)[None],
                                                     np.zeros((1, 1), np.int64), np.array([total]), np.array([n]),
                                                     2 ** 31 - 1 if window is None else window, D ** -0.5)
                within(out[s:s + 1], want_o, size, slack)
    assert granted_some > 50 and (refused_some > 3 or window is not None)        # (a window's pages come back)
    held = to_np(cache.tables)
    assert (np.bincount(held[held >= 0], minlength=17) == to_np(cache.refs)).all()


# ---------------------------------------------------------------- the module and the block

def exact_module(H, D, window, **cfg):
    """A module whose projections are exact in any order of sums: q, k, v are x's values in other orders, out is x's order."""
    from flower_amd.attention import CausalSelfAttention
    d = H * D
    m = CausalSelfAttention(_cfg(d_model=d, num_heads=H, attn_precision="bf16", **cfg), local_window=window).cuda().bfloat16()
    perms = [torch.randperm(d, generator=torch.Generator().manual_seed(i)) for i in range(3)]
    with torch.no_grad():
        m.qkv.weight.copy_(torch.cat([torch.eye(d)[p] for p in perms]))
        m.out.weight.copy_(torch.eye(d))
    return m, perms


def defined(x, m, perms, H, D, window, lens):
    """(out, size, delta) of the module's definition in 64 bits on whole sequences x (B, T, d), rotary tables as it uses them."""
    B, T, d = x.shape
    q, k, v = (x[..., p.numpy()].reshape(B, T, H, D).transpose(0, 2, 1, 3) for p in perms)
    if m.qk_norm is not None:
        q, k = O.head_norm(q, m.qk_norm.eps), O.head_norm(k, m.qk_norm.eps)
    cos, sin = (to_np(t) for t in m.rope.pair_tables(T, torch.bfloat16, "cuda"))
    pos = np.tile(np.arange(T), (B, 1))
    q, k = (O.rotary(t, cos, sin, pos, m.rope.layout)[0] for t in (q, k))
    s = np.einsum("bhid,bhjd->bhij", q, k) * D ** -0.5
    mass = np.einsum("bhid,bhjd->bhij", np.abs(q), np.abs(k)) * D ** -0.5
    i, j = np.arange(T)[:, None], np.arange(T)[None]
    see = (j <= i) & (i - j < (window or T))
    p = np.exp(np.where(see, s - np.where(see, s, -np.inf).max(-1, keepdims=True), -np.inf))
    p /= p.sum(-1, keepdims=True)
    rows = lambda t: t.transpose(0, 2, 1, 3).reshape(B, T, d)
    delta = np.where(see, mass, 0).max(-1, keepdims=True) * np.ones((1, 1, 1, D))
    return rows(p @ v), rows(p @ np.abs(v)), rows(delta)


MODULES = [dict(qk_norm=False), dict(qk_norm=True), dict(qk_norm=True, rope_layout="half", rope_dim=32),
           dict(qk_norm=False, rope_scaling={"type": "yarn", "factor": 4.0, "original_positions": 16})]


@pytest.mark.parametrize("cfg", MODULES, ids=["plain", "norm", "half", "yarn"])
@pytest.mark.parametrize("window", [None, 9])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_cached_forward_is_the_modules_definition(cfg, window, dtype):
    """Ragged prompts (in one call, or two), then tokens one by one."""
    from flower_amd.kv_cache import PagedKVCache
    H, D, T, first = 2, 64, 45, [20, 1, 33]
    m, perms = exact_module(H, D, window, **cfg)
    x = seeded((3, T, H * D), 4, torch.bfloat16, scale=0.5)
    want, size, mass = defined(f64(x), m, perms, H, D, window, first)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -4
    delta = mass * (half + 2.0 ** -8 + half * 2.0 ** -8) + (0 if dtype == torch.bfloat16 else D ** 0.5 * 2.0 ** -10 * 4)
    tol = 2.0 ** -8 * np.abs(want) + (size * (1 + half) + 2.0 ** -10) * (np.exp(2 * delta) - 1) + size * half + 2.0 ** -10
    for prompt in (True, False):
        cache = PagedKVCache(1, 16, H, D, sequences=3, max_len=64, page_size=16, dtype=dtype, window=window)
        got, at = np.full(want.shape, np.nan), [0, 0, 0]

        def feed(counts, prompt=False):
            n = max(counts)
            chunk = torch.zeros((3, n, H * D), dtype=torch.bfloat16, device="cuda")
            for b, c in enumerate(counts):
                chunk[b, :c] = x[b, at[b]:at[b] + c]
            assert cache.reserve(counts).tolist() == list(counts)
            out = f64(m.forward_cached(chunk, cache, 0, prompt=prompt))
            for b, c in enumerate(counts):
                got[b, at[b]:at[b] + c] = out[b, :c]
                at[b] += c
                assert prompt or (out[b, c:] == 0).all()

        if prompt:
            feed(first, prompt=True)
        else:
            feed([7, 0, 30])
            feed([13, 1, 3])
        while min(at) < T:
            feed([int(a < T) for a in at])
        off = np.abs(got - want) / tol
        assert off.max() <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))


def test_default_rope_options_change_nothing():
    """The module's forward with the options at their defaults, and named: the same bits."""
    from flower_amd.attention import CausalSelfAttention
    outs = []
    for cfg in ({}, dict(rope_layout="interleaved", rope_dim=64, rope_scaling=None)):
        torch.manual_seed(0)
        m = CausalSelfAttention(_cfg(attn_precision="bf16", **cfg), local_window=16).cuda().bfloat16()
        outs.append(m(seeded((2, 40, 128), 1, torch.bfloat16)))
    assert torch.equal(*outs)


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_rope_options_train_and_infer(precision):
    """Half layout on a part of the head, scaled: the module runs forward and backward and every parameter has a finite
    gradient; its two routes without gradients agree bit for bit."""
    from flower_amd.attention import CausalSelfAttention
    torch.manual_seed(0)
    cfg = _cfg(attn_precision=precision, rope_layout="half", rope_dim=32, rope_scaling={"type": "linear", "factor": 2.0})
    m = CausalSelfAttention(cfg, local_window=16).cuda().bfloat16()
    x = seeded((2, 40, 128), 1, torch.bfloat16).requires_grad_()
    m(x).float().square().sum().backward()
    assert all(bool(torch.isfinite(t.grad).all()) and bool((t.grad != 0).any()) for t in (x, m.qkv.weight, m.out.weight))
    with torch.no_grad():
        y = m(x)
        assert precision == "bf16" or torch.equal(y, m.forward_unfused(x))


def test_rotary_embedding_gradient_against_differences():
    """RotaryEmbedding beyond the plain form, fp32: the rotation is linear, so a difference over a step of one is the
    derivative; off by the roundings of the two outputs (each 2^-23 of |a c| + |b s|, at most 2 |x|) and of the sum."""
    from flower_amd.attention import RotaryEmbedding
    r = RotaryEmbedding(64, 32, layout="half", rotary_dim=48, scaling={"type": "ntk", "factor": 2.0})
    q, k = seeded((2, 3, 20, 64), 1).requires_grad_(), seeded((2, 1, 20, 64), 2).requires_grad_()
    wq, wk = seeded((2, 3, 20, 64), 3), seeded((2, 1, 20, 64), 4)

    def loss(q, k):
        a, b = r(q, k)
        return (a.double() * wq.double()).sum() + (b.double() * wk.double()).sum()

    loss(q, k).backward()
    for t, at in ((q, (1, 2, 19, 5)), (q, (0, 0, 7, 40)), (q, (1, 1, 3, 60)), (k, (1, 0, 13, 30))):
        e = torch.zeros_like(t)
        e[at] = 1.0
        with torch.no_grad():
            d = loss(*(x + e if x is t else x for x in (q, k))) - loss(q, k)
        assert abs(float(d) - float(t.grad[at])) <= 16 * 2.0 ** -23 * (1 + float(t.detach().abs().max())) * 4


# ---------------------------------------------------------------- graphs

def blocks(n, dtype=torch.bfloat16):
    from flower_amd.block import TransformerBlock, block_config
    torch.manual_seed(3)
    cfg = block_config(d_model=128, num_heads=2, ffn_dim=256, local_window=24, max_seq_len=64)
    return [TransformerBlock(cfg).cuda().to(dtype).eval() for _ in range(n)]


def make_cache(layers, dtype=torch.bfloat16):
    from flower_amd.kv_cache import PagedKVCache
    return PagedKVCache(layers, 40, 2, 64, sequences=4, max_len=96, page_size=16, window=24, dtype=dtype)


def test_the_block_decodes_as_it_prompts():
    """The last token's row of a block run on a growing prompt, against the decode of that token: the two routes' attention
    (each within its bf16 roundings of the same numbers) and the same layers behind it. A block's row is x + a + ff: where
    the attentions agree bit for bit so must it; checked here to the sum of the two routes' roundings carried through."""
    (b,) = blocks(1)
    x = seeded((4, 30, 128), 8, torch.bfloat16)
    cache, outs = make_cache(1), []
    with torch.no_grad():
        cache.reserve(20)
        outs.append(b.forward_cached(x[:, :20], cache, 0, prompt=True))
        for t in range(20, 30):
            cache.reserve(1)
            outs.append(b.forward_cached(x[:, t:t + 1], cache, 0))
        got, want = torch.cat(outs, dim=1).float(), b(x)[0].float()
    # |da| <= 2^-6 of a's scale (roundings of q, k, products, tables: about ten half steps), ff's gain here below 4
    assert float((got - want).abs().max()) <= (1 + 4) * 2.0 ** -6 * float(want.abs().max())


def test_the_fp8_block_decodes():
    """Fp8DecoderBlock over the cache: the composition of its modules, bit for bit, prompt and decode; one token a call or
    several, a row's result is the same to the attention's own rounding (per-row activation scales)."""
    from flower_amd.block import Fp8DecoderBlock
    torch.manual_seed(1)
    b = Fp8DecoderBlock(128, 2, 256, 24).cuda().bfloat16().eval()
    x = seeded((4, 30, 128), 8, torch.bfloat16)
    cache, twin = make_cache(1), make_cache(1)
    with torch.no_grad():
        for t0, t1 in ((0, 20), (20, 21), (21, 25)):
            cache.reserve(t1 - t0), twin.reserve(t1 - t0)
            got = b.forward_cached(x[:, t0:t1], cache, 0, prompt=t0 == 0)
            h = x[:, t0:t1] + b.attn.forward_cached(b.ln1(x[:, t0:t1]), twin, 0, prompt=t0 == 0)
            assert torch.equal(got, h + b.ff(b.ln2(h))) and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_captured_decode_steps_replay_as_eager_ones(dtype):
    """Two graphs of whole decode steps (pages reserved, two blocks, with a beam reorder in the one), each with a cache of
    its own, replayed in turn with eager steps of a twin cache and synchronisations in between: every step's outputs and the
    caches' states equal the twins' bit for bit."""
    layers = blocks(2)
    counts, parents = torch.ones(4, dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")

    def step(cache, x, reorder):
        if reorder:
            cache.reorder(parents)
        cache.reserve(counts)
        for i, b in enumerate(layers):
            x = b.forward_cached(x, cache, i)
        return x

    def fill(cache):
        x = seeded((4, 18, 128), 1, torch.bfloat16)
        cache.reserve([18, 1, 0, 7])
        for i, b in enumerate(layers):
            x = b.forward_cached(x, cache, i, prompt=True)

    runs = []
    with torch.no_grad():
        for reorder in (False, True):
            cache, twin = make_cache(2, dtype), make_cache(2, dtype)
            x = torch.zeros((4, 1, 128), dtype=torch.bfloat16, device="cuda")
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(2):
                    step(cache, x, reorder)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(cache, x, reorder)
            cache.free(range(4))
            fill(cache), fill(twin)
            runs.append((reorder, cache, twin, x, graph, out))
        for n in range(30):
            for reorder, cache, twin, x, graph, out in runs:
                new = seeded((4, 1, 128), 50 + n, torch.bfloat16)
                parents.copy_(torch.tensor([0, 1, 2, 3] if n % 7 else [3, 1, 1, -1], dtype=torch.int32))
                counts.copy_(torch.tensor([1, 1, n % 2, 1], dtype=torch.int32))
                x.copy_(new)
                graph.replay()
                want = step(twin, new, reorder)
                torch.cuda.synchronize()
                assert torch.equal(out, want), (n, reorder)
                for a in ("tables", "lens", "refs", "counts"):
                    assert torch.equal(getattr(cache, a), getattr(twin, a)), (n, reorder, a)
                assert bool(torch.isfinite(out).all())
        assert int(runs[0][1].lens[0]) == 48


def test_captured_rotary_backward():
    """Forward and backward of the rotary pass in one graph, leaves of the graph's own, replayed between eager calls on
    other leaves."""
    from flower_amd.attention import RotaryEmbedding
    r = RotaryEmbedding(64, 32, layout="half", rotary_dim=32)
    r.pair_tables(32, torch.bfloat16, "cuda")
    w = seeded((2, 2, 20, 64), 9, torch.bfloat16)

    def grads(q, k):
        a, b = r(q, k)
        return (a, b, *torch.autograd.grad((a, b), (q, k), (w, w)))

    def leaves(seed):
        return [seeded((2, 2, 20, 64), seed + i, torch.bfloat16).requires_grad_() for i in (0, 1)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            grads(*leaves(5))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    static = leaves(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = grads(*static)
    for n in range(4):
        new = leaves(20 + n)
        with torch.no_grad():
            for a, b in zip(static, new):
                a.copy_(b)
        w.copy_(seeded((2, 2, 20, 64), 70 + n, torch.bfloat16))
        graph.replay()
        want = grads(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), n
