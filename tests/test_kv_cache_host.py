"""CPU: the rotary tables and options, and what the rotary and paged-cache operators refuse before anything runs."""

import math

import pytest
import torch

from flower_amd.attention import CausalSelfAttention, RotaryEmbedding, rotary_tables
from flower_amd.kernels import (apply_rotary, compact_pages, paged_append, paged_attention, reorder_pages, reserve_pages)
from flower_amd.kv_cache import PagedKVCache

from test_abi import fake_pointers
from test_attention_host import _cfg


# ---------------------------------------------------------------- tables

def angles(cos, sin):
    return torch.atan2(sin.double(), cos.double())


@pytest.mark.parametrize("R", [8, 32, 64, 128])
def test_tables_are_the_formula_rounded_once(R):
    cos, sin = rotary_tables(R, 500, 10000.0)
    assert cos.shape == sin.shape == (500, R // 2) and cos.dtype == torch.float32
    for p in (0, 1, 77, 499):
        for i in range(R // 2):
            a = p * 10000.0 ** (-2.0 * i / R)
            # half a step of fp32, and the angle's own 64-bit rounding
            assert abs(float(cos[p, i]) - math.cos(a)) <= 2.0 ** -24 + 1e-12
            assert abs(float(sin[p, i]) - math.sin(a)) <= 2.0 ** -24 + 1e-12


def test_linear_scaling_interpolates_positions():
    cos, sin = rotary_tables(64, 400, scaling={"type": "linear", "factor": 4.0})
    c0, s0 = rotary_tables(64, 100)
    assert torch.equal(cos[::4], c0) and torch.equal(sin[::4], s0)


def test_ntk_scaling_keeps_the_fastest_pair_and_slows_the_slowest_by_the_factor():
    cos, sin = rotary_tables(64, 3, base=500.0, scaling={"type": "ntk", "factor": 8.0})
    a, a0 = angles(cos, sin)[1], angles(*rotary_tables(64, 3, base=500.0))[1]
    assert float(a[0]) == float(a0[0])
    # fp32 tables: sin and cos off by 2^-24 each, an angle of 0.0026 by 2^-24 / 0.0026 of itself at most
    assert abs(float(a0[-1] / a[-1]) - 8.0) < 8.0 * 2 * 2.0 ** -24 / float(a[-1])
    assert bool((a <= a0).all())


def test_yarn_scaling_keeps_fast_pairs_slows_slow_ones_and_scales_the_tables():
    R, L, s = 64, 2048, 16.0
    cos, sin = rotary_tables(R, 2, scaling={"type": "yarn", "factor": s, "original_positions": L})
    gain = 0.1 * math.log(s) + 1.0
    freq0 = [10000.0 ** (-2.0 * i / R) for i in range(R // 2)]
    freq = angles(cos, sin)[1]
    radius = (cos.double() ** 2 + sin.double() ** 2).sqrt()
    assert float((radius - gain).abs().max()) < 4 * 2.0 ** -24 * gain
    kept = slowed = between = 0
    for i, f in enumerate(freq0):
        turns, tol = L * f / (2 * math.pi), 4 * 2.0 ** -24
        if turns > 40:                                   # the ramp's ends are rounded outwards to whole pairs
            assert abs(float(freq[i]) - f) <= tol
            kept += 1
        elif turns < 0.7:
            assert abs(float(freq[i]) - f / s) <= tol
            slowed += 1
        else:
            assert f / s - tol <= float(freq[i]) <= f + tol
            between += 1
    assert kept and slowed and between
    same = rotary_tables(R, 9, scaling={"type": "yarn", "factor": 1.0, "original_positions": L})
    assert all(torch.equal(a, b) for a, b in zip(same, rotary_tables(R, 9)))


@pytest.mark.parametrize("scaling", [{"type": "cubic", "factor": 2.0}, {"factor": 2.0}, {"type": "linear", "factor": 0.5},
                                     {"type": "linear", "factor": float("nan")}, {"type": "yarn", "factor": 2.0},
                                     {"type": "yarn", "factor": 2.0, "original_positions": 64, "beta_fast": 1, "beta_slow": 2},
                                     {"type": "ntk", "factor": 2.0, "original_positions": 64}])
def test_scalings_that_are_refused(scaling):
    with pytest.raises(ValueError):
        rotary_tables(32, 4, scaling=scaling)
    with pytest.raises(ValueError):
        RotaryEmbedding(32, 4, scaling=scaling)


def test_rotary_embedding_options():
    plain = RotaryEmbedding(64, 16)
    assert plain.plain
    cos, sin = plain.pair_tables(40, torch.bfloat16, "cpu")          # longer than its tables: extended
    whole = plain.tables(40, torch.bfloat16, "cpu")
    assert cos.dtype == torch.float32 and torch.equal(cos, whole[0][:, ::2].float()) and torch.equal(sin, whole[1][:, 1::2].float())
    half = RotaryEmbedding(64, 16, layout="half", rotary_dim=32).to(torch.bfloat16)
    assert not half.plain
    cos, sin = half.pair_tables(24, torch.bfloat16, "cpu")
    assert all(torch.equal(a, b) for a, b in zip((cos, sin), rotary_tables(32, 24)))         # fp32 under any cast
    with pytest.raises(ValueError, match="pair_tables"):
        half.tables(4, torch.bfloat16, "cpu")
    for bad in (dict(layout="quarter"), dict(rotary_dim=12), dict(rotary_dim=72), dict(rotary_dim=0)):
        with pytest.raises(ValueError):
            RotaryEmbedding(64, 16, **bad)


# ---------------------------------------------------------------- refusals of the operators

def args(B=2, H=4, KV=2, T=1, D=64, P=5, page=16, M=3, dtype=torch.bfloat16):
    return dict(q=torch.zeros(B, H, T, D, dtype=torch.bfloat16), k=torch.zeros(B, KV, T, D, dtype=torch.bfloat16),
                v=torch.zeros(B, KV, T, D, dtype=torch.bfloat16), k_pages=torch.zeros(P, KV, page, D).to(dtype),
                v_pages=torch.zeros(P, KV, D, page).to(dtype), tables=torch.zeros(B, M, dtype=torch.int32),
                lens=torch.ones(B, dtype=torch.int32))


def refused(call, a, error, **change):
    a = dict(a, **change)
    pos = [a.pop(n) for n in (("q", "k", "v") if call is paged_append else ("q",))]
    if call is paged_attention:
        a.pop("k", None), a.pop("v", None)
    pos += [a.pop(n) for n in ("k_pages", "v_pages", "tables", "lens")]
    with pytest.raises(error):
        call(*pos, a.pop("counts", None), **a)


BAD = [
    (ValueError, dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16))),
    (ValueError, dict(q=torch.zeros(2, 4, 0, 64, dtype=torch.bfloat16))),
    (ValueError, dict(q=torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16))),               # heads not shared evenly
    (ValueError, dict(q=torch.zeros(2, 4, 1, 32, dtype=torch.bfloat16))),               # another head size than the pool's
    (ValueError, dict(q=torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16))),               # more sequences than tables
    (TypeError, dict(q=torch.zeros(2, 4, 1, 64))),
    (TypeError, dict(k_pages=torch.zeros(5, 2, 16, 64))),
    (ValueError, dict(v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16))),        # V is (pages, heads, D, page)
    (ValueError, dict(k_pages=torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16))),
    (ValueError, dict(tables=torch.zeros(2, 3, dtype=torch.int64))),
    (ValueError, dict(tables=torch.zeros(3, 2, dtype=torch.int32).t())),
    (ValueError, dict(lens=torch.ones(3, dtype=torch.int32))),
    (ValueError, dict(lens=torch.ones(2))),
    (ValueError, dict(counts=torch.ones(2, dtype=torch.int64))),
    (ValueError, dict(k_scale=torch.ones(2), v_scale=torch.ones(2))),                   # a bf16 cache takes none
]


@pytest.mark.parametrize("call", [paged_append, paged_attention])
@pytest.mark.parametrize("error,change", BAD)
def test_append_and_attention_refuse(call, error, change):
    refused(call, args(), error, **change)


@pytest.mark.parametrize("call", [paged_append, paged_attention])
def test_append_and_attention_refuse_scales_pages_gradients_and_the_cpu(call):
    e4m3 = args(dtype=torch.float8_e4m3fn)
    refused(call, e4m3, ValueError)                                                     # scales missing
    refused(call, e4m3, ValueError, k_scale=torch.ones(2))
    refused(call, e4m3, ValueError, k_scale=torch.ones(3), v_scale=torch.ones(3))
    refused(call, args(), RuntimeError, q=torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, requires_grad=True))
    refused(call, args(), RuntimeError)                                                 # CPU tensors
    refused(call, e4m3, RuntimeError, k_scale=torch.ones(2), v_scale=torch.ones(2))


def test_append_refuses_its_own_arguments():
    a = args()
    table = torch.zeros(4, 32)
    for change in (dict(k=torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)), dict(v=torch.zeros(2, 2, 2, 64, dtype=torch.bfloat16)),
                   dict(cos=table), dict(cos=table, sin=torch.zeros(4, 16)), dict(cos=table.double(), sin=table.double()),
                   dict(cos=torch.zeros(4, 34), sin=torch.zeros(4, 34)), dict(cos=torch.zeros(4, 6), sin=torch.zeros(4, 6)),
                   dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)), dict(layout="quarter"), dict(norm_eps=-1.0),
                   dict(norm_eps=float("nan"))):
        refused(paged_append, a, ValueError, **change)


def test_rotary_refuses():
    q, k, t = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64), torch.zeros(8, 32)
    for error, a in [(ValueError, (q[0], k, t, t)), (ValueError, (q, k[:, :, :2], t, t)), (ValueError, (q, k.bfloat16(), t, t)),
                     (TypeError, (q.half(), k.half(), t, t)), (ValueError, (q, k, t, t[:4])), (ValueError, (q, k, t[:, :6], t[:, :6])),
                     (ValueError, (torch.zeros(1, 1, 1, 48), None, t, t)),
                     (ValueError, (q, k, t, t, torch.zeros(4, dtype=torch.int32))),
                     (ValueError, (q, k, t, t, torch.zeros(3))), (RuntimeError, (q, k, t, t)), (RuntimeError, (q, None, t, t))]:
        with pytest.raises(error):
            apply_rotary(*a)
    with pytest.raises(ValueError, match="layout"):
        apply_rotary(q, k, t, t, layout="quarter")
    with pytest.raises(ValueError, match="gradient"):
        apply_rotary(q, k, t.clone().requires_grad_(), t)


def test_pages_refuse():
    i32 = dict(dtype=torch.int32)
    tables, lens, refs, counts = torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(5, **i32), torch.ones(2, **i32)
    k, v = torch.zeros(1, 5, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(1, 5, 2, 64, 16, dtype=torch.bfloat16)
    for a in [(tables[0], lens, refs, counts, 16), (tables.long(), lens, refs, counts, 16), (tables, lens[:1], refs, counts, 16),
              (tables, lens, refs[None], counts, 16), (tables, lens, refs, counts[:1], 16), (tables, lens, refs[:0], counts, 16)]:
        with pytest.raises(ValueError):
            reserve_pages(*a)
    for window in (0, -3):
        with pytest.raises(ValueError):
            reserve_pages(tables, lens, refs, counts, 16, window=window)
    for a in [(k, v, tables, lens, refs[:4], counts), (k, v[:, :, :, :, :8], tables, lens, refs, counts),
              (k, v[0], tables, lens, refs, counts), (k, v, tables, lens, refs, counts.long())]:
        with pytest.raises(ValueError):
            reorder_pages(*a)
    with pytest.raises(ValueError):
        compact_pages(k, v, tables, refs[:4])
    with pytest.raises(TypeError):
        compact_pages(k.float(), v.float(), tables, refs)
    for call in (lambda: reserve_pages(tables, lens, refs, counts, 16), lambda: reorder_pages(k, v, tables, lens, refs, counts),
                 lambda: compact_pages(k, v, tables, refs)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# ---------------------------------------------------------------- the cache object and the module

def test_cache_shapes_and_refusals():
    c = PagedKVCache(2, 7, 3, 64, sequences=4, max_len=100, page_size=16, device="cpu")
    assert c.k_pages.shape == (2, 7, 3, 16, 64) and c.v_pages.shape == (2, 7, 3, 64, 16) and c.tables.shape == (4, 7)
    assert c.max_len == 112 and c.sequences == 4 and int(c.tables.max()) == -1 and c.k_scale is None
    scale = torch.rand(2, 3)
    c8 = PagedKVCache(2, 7, 3, 64, sequences=4, max_len=100, dtype=torch.float8_e4m3fn, k_scale=scale, device="cpu")
    assert torch.equal(c8.k_scale, scale) and c8.k_scale.data_ptr() != scale.data_ptr() and bool((c8.v_scale == 1).all())
    for change in (dict(sequences=0), dict(max_len=0), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(window=0),
                   dict(k_scale=scale)):
        with pytest.raises(ValueError):
            PagedKVCache(2, 7, 3, 64, **dict(dict(sequences=4, max_len=100, device="cpu"), **change))
    with pytest.raises(ValueError):
        PagedKVCache(2, 7, 3, 48, sequences=4, max_len=100, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(2, 7, 3, 64, sequences=4, max_len=100, dtype=torch.float8_e4m3fn, v_scale=scale[:1], device="cpu")
    with pytest.raises(TypeError):
        PagedKVCache(2, 7, 3, 64, sequences=4, max_len=100, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="no place"):
        c.free([4])
    w = PagedKVCache(1, 7, 3, 64, sequences=4, max_len=100, window=32, device="cpu")
    with pytest.raises(ValueError, match="window of 32"):
        w.attend(0, torch.zeros(4, 3, 1, 64, dtype=torch.bfloat16), window=33)


def test_cached_forward_refuses():
    cache = PagedKVCache(1, 8, 2, 64, sequences=3, max_len=64, window=32, device="cpu")
    x = torch.zeros(3, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be \\(3, T, d\\)"):
        CausalSelfAttention(_cfg(), local_window=32).forward_cached(x[:2], cache, 0)
    with pytest.raises(ValueError, match="window of 32"):
        CausalSelfAttention(_cfg()).forward_cached(x, cache, 0)
    with pytest.raises(ValueError, match="window of 32"):
        CausalSelfAttention(_cfg(), local_window=33).forward_cached(x, cache, 0)
    with pytest.raises(ValueError, match="fp8_attention_sim"):
        CausalSelfAttention(_cfg(fp8_attention_sim=True), local_window=32).forward_cached(x, cache, 0)
    with pytest.raises(RuntimeError, match="GPU"):
        CausalSelfAttention(_cfg(), local_window=32).bfloat16().forward_cached(x, cache, 0)


# ---------------------------------------------------------------- the C entry points

A = 1 << 20            # an aligned address that is no memory: the calls below are refused before anything reads it


def c_call(name, **change):
    from flower_amd import _lib
    lib = _lib.load()
    st = (_lib.ctypes.c_int64 * 3)(64, 64, 64)
    lists = {
        "flw_rope": dict(q=A, q_strides=st, H=4, k=A, k_strides=st, KV=2, dtype=1, B=2, T=1, D=64, cos=A, sin=A, table_rows=8,
                         rotary_dim=64, layout=0, inverse=0, positions=None, bits=0, stride_b=0, q_out=A, k_out=A, stream=None),
        "flw_paged_attention": dict(q=A, q_strides=st, k_pages=A, v_pages=A, cache=1, P=5, page=16, tables=A, M=3, lens=A,
                                    counts=None, k_scale=None, v_scale=None, B=2, H=4, KV=2, T=1, D=64, window=100, scale=1.0,
                                    out=A, out_strides=st, lse=None, workspace=None, bytes=0, stream=None),
        "flw_reserve_pages": dict(tables=A, lens=A, refs=A, counts=A, S=2, M=3, P=5, page=16, window=0, to=A, to_lens=A, to_refs=A,
                                  granted=A, workspace=A, bytes=1 << 20, stream=None),
    }
    a = dict(lists[name])
    assert set(change) <= set(a)
    a.update(change)
    rc = getattr(lib, name)(*a.values())
    return rc, lib.flw_last_error().decode()


@fake_pointers
@pytest.mark.parametrize("name,change", [
    ("flw_rope", dict(q=None)), ("flw_rope", dict(cos=None)), ("flw_rope", dict(D=48)), ("flw_rope", dict(rotary_dim=12)),
    ("flw_rope", dict(rotary_dim=72)), ("flw_rope", dict(layout=2)), ("flw_rope", dict(dtype=2)), ("flw_rope", dict(B=0)),
    ("flw_rope", dict(table_rows=0)), ("flw_rope", dict(q_out=A + 2)), ("flw_rope", dict(positions=A, bits=16)),
    ("flw_rope", dict(k_out=None)), ("flw_rope", dict(B=1 << 40)),
    ("flw_paged_attention", dict(q=None)), ("flw_paged_attention", dict(q_strides=None)), ("flw_paged_attention", dict(lens=None)),
    ("flw_paged_attention", dict(D=48)), ("flw_paged_attention", dict(H=3)), ("flw_paged_attention", dict(page=24)),
    ("flw_paged_attention", dict(page=8)), ("flw_paged_attention", dict(page=2048)), ("flw_paged_attention", dict(cache=0)),
    ("flw_paged_attention", dict(cache=2)), ("flw_paged_attention", dict(k_scale=A, v_scale=A)),
    ("flw_paged_attention", dict(cache=2, k_scale=A)), ("flw_paged_attention", dict(k_pages=A + 8)),
    ("flw_paged_attention", dict(B=1 << 20)), ("flw_paged_attention", dict(T=1 << 20)),
    ("flw_paged_attention", dict(P=1 << 31)), ("flw_paged_attention", dict(M=1 << 40)), ("flw_paged_attention", dict(M=0)),
    ("flw_reserve_pages", dict(tables=None)), ("flw_reserve_pages", dict(granted=None)), ("flw_reserve_pages", dict(S=0)),
    ("flw_reserve_pages", dict(page=0)), ("flw_reserve_pages", dict(workspace=None)), ("flw_reserve_pages", dict(bytes=8)),
])
def test_c_entry_points_refuse(name, change):
    rc, message = c_call(name, **change)
    assert rc != 0 and message
