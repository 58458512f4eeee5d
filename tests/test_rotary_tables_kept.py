"""CPU: the tables that RotaryEmbedding hands out stay in place while the module lives (a captured graph reads them), are shared by
the lengths that they cover, and can be saved for a backward pass whoever asked for them first."""

import copy
import gc
import weakref

import pytest
import torch

from flower_amd.attention import RotaryEmbedding, rotary_tables

OPTIONS = [dict(), dict(layout="half", rotary_dim=32), dict(scaling={"type": "linear", "factor": 2.0})]


def asked(r, n):
    """Every kind of table that r has, of n rows."""
    kinds = [r.pair_tables, r.tables] if r.plain else [r.pair_tables]
    return [t for f in kinds for dtype in (torch.bfloat16, torch.float32) for t in f(n, dtype, "cpu")]


@pytest.mark.parametrize("options", OPTIONS)
def test_what_was_handed_out_is_never_freed(options):
    r = RotaryEmbedding(64, 16, **options)
    for n in (40, 10, 200, 41, 3000):                    # within the module's length and past it, shorter and longer
        tables = asked(r, n)
        refs = [weakref.ref(t._base if t._base is not None else t) for t in tables]
        want = [t.clone() for t in tables]
        places = [t.data_ptr() for t in tables]
        del tables
        for other in (5, 64, 7 * n, 41):
            asked(r, other)
        gc.collect()
        assert all(ref() is not None for ref in refs)
        assert all(torch.equal(ref().reshape(-1, t.shape[1])[:n], t) and ref().data_ptr() == p for ref, t, p in zip(refs, want, places))
        for got, t in zip(asked(r, n), want):
            assert got.shape[0] == n and got.is_contiguous() and torch.equal(got, t)


@pytest.mark.parametrize("options", OPTIONS)
def test_lengths_in_turn_make_no_new_tables(options):
    """Two caches of different lengths, a step of each in turn."""
    r = RotaryEmbedding(64, 16, **options)
    asked(r, 100), asked(r, 60)
    first = [t.data_ptr() for n in (60, 100) for t in asked(r, n)]
    for _ in range(3):
        assert [t.data_ptr() for n in (60, 100) for t in asked(r, n)] == first


@pytest.mark.parametrize("options", OPTIONS)
def test_lengths_that_grow_by_one_make_few_tables(options):
    r = RotaryEmbedding(64, 16, **options)
    seen = {asked(r, n)[0].data_ptr() for n in range(1, 600)}
    assert len(seen) <= 12                               # 1, 2, 4, .. 1024, and one more where the module's own length ends


@pytest.mark.parametrize("options", OPTIONS)
def test_tables_first_asked_for_in_inference_mode(options):
    r = RotaryEmbedding(64, 16, **options)
    with torch.inference_mode():
        asked(r, 40)
    assert not any(t.is_inference() for t in asked(r, 40) + asked(r, 30))
    if r.plain:
        x = torch.randn(1, 2, 40, 64, requires_grad=True)
        sum(t.sum() for t in r(x, x)).backward()
        assert bool(torch.isfinite(x.grad).all())


def test_a_cast_or_copied_module_has_its_own_values():
    r = RotaryEmbedding(64, 16)
    exact = [t.clone() for t in r.pair_tables(16, torch.float32, "cpu")]
    twin = copy.deepcopy(r)
    rounded = r.to(torch.bfloat16).pair_tables(16, torch.float32, "cpu")          # the buffers are rounded: so is forward
    assert all(torch.equal(a, b.bfloat16().float()) for a, b in zip(rounded, exact))
    assert all(torch.equal(a, b) for a, b in zip(twin.pair_tables(16, torch.float32, "cpu"), exact))
    half = RotaryEmbedding(64, 16, layout="half").to(torch.bfloat16)
    assert all(torch.equal(a, b) for a, b in zip(half.pair_tables(24, torch.bfloat16, "cpu"), rotary_tables(64, 24)))
