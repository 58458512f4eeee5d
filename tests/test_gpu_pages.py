"""GPU: reserve_pages, reorder_pages and compact_pages against the oracle's plain loops; every number has to be equal."""

import numpy as np
import pytest
import torch

from oracle import paged as O

from gpu_util import to_np

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def state(rng, S, M, P, page, lens=None, share=False):
    """Random tables whose sequences hold their lens, some of it shared, and refs that fit."""
    lens = rng.integers(0, M * page + 1, S) if lens is None else np.asarray(lens)
    ids = list(rng.permutation(P))
    tables = np.full((S, M), -1, np.int32)
    for s in range(S):
        for j in range(-(-int(lens[s]) // page)):
            if share and s and (j + 1) * page <= min(lens[s], lens[s - 1]) and j < 2:
                tables[s, j] = tables[s - 1, j]
            elif ids:
                tables[s, j] = ids.pop()
            else:
                lens[s] = j * page
                break
    refs = np.bincount(tables[tables >= 0], minlength=P).astype(np.int32)
    return tables, lens.astype(np.int32), refs


def run_reserve(tables, lens, refs, counts, page, window, in_place):
    from flower_amd.kernels import reserve_pages
    t, n, r = ints(tables), ints(lens), ints(refs)
    out = reserve_pages(t, n, r, ints(counts), page, window=window, out=(t, n, r) if in_place else None)
    if in_place:
        assert out[0] is t and out[1] is n and out[2] is r
    else:
        assert np.array_equal(to_np(t), tables) and np.array_equal(to_np(n), lens) and np.array_equal(to_np(r), refs)
    return [to_np(x) for x in out]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,M,P,page,window,new", [
    (1, 1, 1, 16, None, 1), (5, 4, 30, 16, None, 1), (5, 4, 12, 16, None, 20), (7, 9, 100, 32, 40, 3),
    (300, 6, 5000, 16, 20, 5), (1100, 3, 2000, 64, None, 100), (3, 700, 3000, 16, 100, 4000), (40, 5, 40, 16, 1, 2),
    (2, 3, 9000, 1024, 5, 1),
])
def test_reserve(S, M, P, page, window, new, in_place):
    rng = np.random.default_rng(S * 7 + M)
    print("[reserve]", S, M, P, page, window, new, flush=True)
    for trial in range(3):
        tables, lens, refs = state(rng, S, M, P, page, share=trial == 1)
        counts = rng.integers(-1, new + 1, S)
        if trial == 2:                # a sequence rolled back holds pages past its lens; strange entries and lens
            lens = np.maximum(lens - rng.integers(0, 2 * page, S), 0).astype(np.int32)
            tables[rng.integers(0, S), rng.integers(0, M)] = -1
            refs = np.bincount(tables[tables >= 0], minlength=P).astype(np.int32)
            lens[0] = -4
        want = O.reserve(tables, lens, refs, counts, page, window)
        got = run_reserve(tables, lens, refs, counts, page, window, in_place)
        for name, a, b in zip(("tables", "lens", "refs", "granted"), got, want):
            assert np.array_equal(a, b), (trial, name)


def test_reserve_refuses_only_who_does_not_fit():
    page, P = 16, 6
    tables, lens, refs = state(np.random.default_rng(0), 4, 4, P, page, lens=[16, 30, 0, 5])       # 4 pages held, 2 free
    got = run_reserve(tables, lens, refs, [1, 2, 40, 1], page, None, False)
    assert got[3].tolist() == [1, 2, 0, 1]                  # 1, 0, 3 pages wanted; the last wants none
    got = run_reserve(tables, lens, refs, [0, 2 ** 31 - 1, 1, 64 - 5], page, None, False)
    assert got[3].tolist() == [0, 0, 1, 0]


def pools(L, P, KV, page, D, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(L, P, KV, page, D, generator=g), torch.randn(L, P, KV, D, page, generator=g)
    return k.to(dtype).cuda(), v.to(dtype).cuda()


def raw(t):
    return t.view(torch.int16 if t.element_size() == 2 else torch.uint8).cpu().numpy()


def run_reorder(k, v, tables, lens, refs, parents, page, in_place):
    from flower_amd.kernels import reorder_pages
    wk, wv = raw(k).copy(), raw(v).copy()
    t, n, r = ints(tables), ints(lens), ints(refs)
    want = O.reorder(wk, wv, tables, lens, refs, parents, page)
    got = reorder_pages(k, v, t, n, r, ints(parents), out=(t, n, r) if in_place else None)
    for name, a, b in zip(("tables", "lens", "refs"), got, want):
        assert np.array_equal(to_np(a), b), name
    assert np.array_equal(raw(k), wk) and np.array_equal(raw(v), wv)
    return [to_np(x) for x in got]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,M,P,page,KV,D,L,dtype", [
    (1, 1, 2, 16, 1, 32, 1, torch.bfloat16), (6, 3, 30, 16, 2, 64, 2, torch.bfloat16),
    (6, 3, 30, 32, 3, 128, 1, torch.float8_e4m3fn), (20, 4, 60, 16, 1, 32, 3, torch.float8_e4m3fn),
    (300, 3, 700, 16, 1, 32, 1, torch.bfloat16), (1100, 2, 1500, 16, 1, 32, 1, torch.float8_e4m3fn),
    (5, 40, 210, 16, 1, 64, 1, torch.bfloat16),
])
def test_reorder(S, M, P, page, KV, D, L, dtype, in_place):
    rng = np.random.default_rng(S + M)
    print("[reorder]", S, M, P, page, KV, D, L, dtype, flush=True)
    k, v = pools(L, P, KV, page, D, dtype)
    for trial in range(4):
        tables, lens, refs = state(rng, S, M, P, page, share=trial % 2 == 1)
        parents = rng.integers(0, S, S) if trial != 2 else rng.integers(-2, S + 2, S)
        if trial == 3:
            parents = np.full(S, rng.integers(0, S))        # one sequence everywhere
        run_reorder(k, v, tables, lens, refs, parents, page, in_place)


def test_reorder_swaps_empties_and_runs_out():
    page = 16
    k, v = pools(2, 7, 2, page, 32, torch.bfloat16)
    tables, lens, refs = state(np.random.default_rng(0), 3, 3, 7, page, lens=[20, 33, 16])         # 2 + 3 + 1 pages, 1 free
    t, n, r = run_reorder(k, v, tables, lens, refs, np.array([1, 0, 2]), page, True)
    assert np.array_equal(t, tables[[1, 0, 2]]) and n.tolist() == [33, 20, 16] and np.array_equal(r, refs)
    t, n, r = run_reorder(k, v, tables, lens, refs, np.array([-1, -1, -1]), page, False)
    assert (t == -1).all() and (n == 0).all() and (r == 0).all()
    t, n, r = run_reorder(k, v, tables, lens, refs, np.array([0, 0, 0]), page, False)              # 4 pages are let go
    assert n.tolist() == [20, 20, 20] and r.sum() == 6
    tables, lens, refs = state(np.random.default_rng(0), 4, 3, 7, page, lens=[20, 33, 16, 8])      # none free
    t, n, r = run_reorder(k, v, tables, lens, refs, np.array([0, 1, 0, 1]), page, False)           # 2 wanted, 2 let go
    assert n.tolist() == [20, 33, 20, 33]
    tables, lens, refs = state(np.random.default_rng(0), 4, 3, 7, page, lens=[20, 33, 0, 20])
    t, n, r = run_reorder(k, v, tables, lens, refs, np.array([0, 1, 1, 3]), page, False)           # 1 wanted, none free
    assert n.tolist() == [20, 33, 0, 20] and (t[2] == -1).all() and np.array_equal(r, refs)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,M,P,page,KV,D,L,dtype,fill", [
    (1, 1, 1, 16, 1, 32, 1, torch.bfloat16, 1.0), (3, 5, 40, 16, 2, 64, 2, torch.bfloat16, 0.5),
    (10, 20, 900, 32, 1, 128, 1, torch.float8_e4m3fn, 0.2), (60, 90, 6000, 16, 1, 32, 1, torch.bfloat16, 0.9),
    (4, 4, 50, 16, 3, 32, 2, torch.float8_e4m3fn, 0.0),
])
def test_compact(S, M, P, page, KV, D, L, dtype, fill, in_place):
    from flower_amd.kernels import compact_pages
    rng = np.random.default_rng(P)
    print("[compact]", S, M, P, page, KV, D, L, dtype, fill, flush=True)
    k, v = pools(L, P, KV, page, D, dtype)
    for trial in range(2):
        tables, lens, refs = state(rng, S, M, P, page, lens=(rng.random(S) * fill * M * page).astype(int), share=trial == 1)
        wk, wv = raw(k).copy(), raw(v).copy()
        want = O.compact(wk, wv, tables, refs)
        t, r = ints(tables), ints(refs)
        got = compact_pages(k, v, t, r, out=(t, r) if in_place else None)
        assert np.array_equal(to_np(got[0]), want[0]) and np.array_equal(to_np(got[1]), want[1])
        assert int(got[2]) == want[2] == int((refs != 0).sum())
        assert np.array_equal(raw(k), wk) and np.array_equal(raw(v), wv)


def test_one_layer_pools_and_a_side_stream():
    from flower_amd.kernels import compact_pages, reorder_pages
    k, v = pools(1, 20, 2, 16, 32, torch.bfloat16)
    tables, lens, refs = state(np.random.default_rng(2), 4, 3, 20, 16)
    k1, v1 = k[0].clone(), v[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    parents = ints([1, 1, 3, -1])
    a = reorder_pages(k, v, ints(tables), ints(lens), ints(refs), parents)
    args = ints(tables), ints(lens), ints(refs)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = reorder_pages(k1, v1, *args, parents)
        c = compact_pages(k1, v1, b[0], b[2])
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x, y) for x, y in zip(compact_pages(k, v, a[0], a[2]), c))
    assert torch.equal(k[0], k1) and torch.equal(v[0], v1)


def test_reorder_of_very_many_places():
    """More places than one grid dimension takes: forks into the first, the middle and the last ones."""
    from flower_amd.kernels import reorder_pages
    S, P = 40000, 12
    k, v = pools(2, P, 1, 16, 32, torch.bfloat16)
    wk, wv = k.clone(), v.clone()
    tables, lens, refs, parents = torch.full((S, 1), -1, dtype=torch.int32), torch.zeros(S, dtype=torch.int32), \
        torch.zeros(P, dtype=torch.int32), torch.arange(S, dtype=torch.int32)
    for s in range(3):                       # places 0, 1, 2 hold pages 3, 4, 5 and 5 + s positions
        tables[s], lens[s], refs[3 + s] = 3 + s, 5 + s, 1
    forks = [(5, 2), (32767, 0), (32768, 1), (32769, 2), (39999, 0)]
    for place, parent in forks:
        parents[place] = parent
    t, n, r = (x.cuda() for x in (tables, lens, refs))
    t, n, r = reorder_pages(k, v, t, n, r, parents.cuda(), out=(t, n, r))
    for (place, parent), page in zip(forks, (0, 1, 2, 6, 7)):        # the free pages in the order of the places
        tables[place], lens[place], refs[page] = page, 5 + parent, 1
        wk[:, page, :, :5 + parent] = wk[:, 3 + parent, :, :5 + parent]
        wv[:, page, :, :, :5 + parent] = wv[:, 3 + parent, :, :, :5 + parent]
    assert torch.equal(t.cpu(), tables) and torch.equal(n.cpu(), lens) and torch.equal(r.cpu(), refs)
    assert torch.equal(k, wk) and torch.equal(v, wv)
