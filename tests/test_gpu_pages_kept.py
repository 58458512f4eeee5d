"""GPU: reorder_pages and PagedKVCache.reorder say which places hold positions of their parents; every number has to be equal."""

import numpy as np
import pytest
import torch

from oracle import paged as O

from gpu_util import seeded, to_np
from test_gpu_pages import ints, pools, state

pytestmark = pytest.mark.gpu


def check(tables, lens, refs, parents, page, in_place):
    """One call against the oracle; returns how many places lost their copy."""
    from flower_amd.kernels import reorder_pages
    S, P = len(lens), len(refs)
    k, v = pools(1, P, 1, page, 32, torch.bfloat16)
    real = (parents >= 0) & (parents < S)
    want = O.reorder(k.cpu().float().numpy(), v.cpu().float().numpy(), tables, lens, refs, parents, page)
    there = np.where(real, lens[np.where(real, parents, 0)], 0) > 0
    holds = want[1] > 0
    assert not (holds & ~there).any()
    t, n, r = ints(tables), ints(lens), ints(refs)
    *got, kept = reorder_pages(k, v, t, n, r, ints(parents), out=(t, n, r) if in_place else None, return_kept=True)
    for name, a, b in zip(("tables", "lens", "refs", "kept"), (*got, kept), (*want, holds.astype(np.int32))):
        assert np.array_equal(to_np(a), b), name
    assert kept.dtype == torch.int32
    return int((there & ~holds).sum())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,M,P,page", [(1, 1, 1, 16), (6, 3, 18, 16), (20, 4, 60, 32), (300, 3, 500, 16), (1100, 2, 1300, 16)])
def test_kept_is_who_holds_its_copy(S, M, P, page, in_place):
    rng = np.random.default_rng(S)
    for trial in range(6):
        tables, lens, refs = state(rng, S, M, P, page, share=trial % 2 == 1)
        lens[rng.integers(0, S)] = -2
        parents = rng.integers(-2, S + 2, S) if trial % 3 else np.full(S, rng.integers(0, S))
        if trial >= 4:                           # every page held: by nobody's table, for what a fork would need
            refs[refs == 0] = 1
        check(tables, lens, refs, parents, page, in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,spare", [(4, 0), (40, 3), (1500, 100)])
def test_forks_into_empty_places_of_a_pool_that_runs_out(S, spare, in_place):
    """Half of the places hold a sequence whose last page is not full, the others fork one each; `spare` pages are free."""
    rng = np.random.default_rng(S)
    lens = np.where(np.arange(S) % 2 == 0, rng.integers(17, 32, S), 0)
    tables, lens, refs = state(rng, S, 2, S + spare, 16, lens=lens)
    parents = np.where(np.arange(S) % 2 == 0, np.arange(S), 2 * rng.integers(0, S // 2, S))
    assert check(tables, lens, refs, parents, 16, in_place) == S // 2 - spare


def fork_step(cache, parents, x, gate):
    kept = cache.reorder(parents)
    cache.reserve(kept * gate)
    q = cache.append(0, x[:, :2], x[:, 2:3], x[:, 3:])
    return kept, cache.attend(0, q)


def full_cache():
    """Three sequences of 20, 33 and 7 positions in all six pages of a pool, and an empty place."""
    from flower_amd.kv_cache import PagedKVCache
    cache = PagedKVCache(1, 6, 1, 64, sequences=4, max_len=64, page_size=16)
    cache.reserve([20, 33, 7, 0])
    x = seeded((4, 33, 4, 64), 1, torch.bfloat16).transpose(1, 2)
    cache.append(0, x[:, :2], x[:, 2:3], x[:, 3:])
    return cache


def test_a_fork_without_a_page_is_told():
    cache = full_cache()
    x = seeded((4, 1, 4, 64), 2, torch.bfloat16).transpose(1, 2)
    kept, out = fork_step(cache, [0, 1, 2, 1], x, 1)                 # the copy of 1's last page finds none
    assert kept.tolist() == [1, 1, 1, 0] and cache.lens.tolist() == [21, 34, 8, 0] and cache.counts.tolist() == [1, 1, 1, 0]
    assert (out[3] == 0).all() and (out[:3] != 0).any()
    kept, _ = fork_step(cache, [0, 1, 2, 3], x, 1)                   # what is empty stays so
    assert kept.tolist() == [1, 1, 1, 0] and cache.lens.tolist() == [22, 35, 9, 0]
    kept, _ = fork_step(cache, [0, 1, -1, 1], x, 1)                  # place 2's page is let go in the same call
    assert kept.tolist() == [1, 1, 0, 1] and cache.lens.tolist() == [23, 36, 0, 36]


def test_a_captured_step_masks_the_forks_that_failed():
    """reorder and reserve(kept) in one graph, replayed with other parents, against eager steps of a twin cache."""
    cache, twin = full_cache(), full_cache()
    parents, gate = torch.arange(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros((4, 4, 1, 64), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fork_step(cache, parents, x, gate)                       # (changes nothing: places stay, no token is granted)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, out = fork_step(cache, parents, x, gate)
    gate.fill_(1)
    for n, row in enumerate(([0, 1, 2, 1], [0, 1, 2, 3], [0, 1, -1, 1], [3, 1, 0, 3], [0, 1, 2, 2])):
        parents.copy_(torch.tensor(row, dtype=torch.int32))
        x.copy_(seeded((4, 4, 1, 64), 30 + n, torch.bfloat16))
        graph.replay()
        want = fork_step(twin, parents, x, gate)
        torch.cuda.synchronize()
        assert torch.equal(kept, want[0]) and torch.equal(out, want[1]), n
        assert all(torch.equal(getattr(cache, a), getattr(twin, a)) for a in ("tables", "lens", "refs", "counts")), n
        assert n > 0 or kept.tolist() == [1, 1, 1, 0]
