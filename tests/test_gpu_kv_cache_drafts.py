"""GPU: PagedKVCache.take_back. A cache in which tokens are drafted and some of them taken back answers as its twin that was given
the accepted ones only, bit for bit: the same keys in ranges of the same length go through the same sums."""

import numpy as np
import pytest
import torch

from gpu_util import seeded, to_np

pytestmark = pytest.mark.gpu

S, H, KV, D = 3, 4, 2, 64


def make(dtype, window):
    from flower_amd.kv_cache import PagedKVCache
    cache = PagedKVCache(1, 40, KV, D, sequences=S, max_len=160, page_size=16, dtype=dtype, window=window)
    for pages in (cache.k_pages, cache.v_pages):
        pages.view(torch.uint8).fill_(0xFF)              # NaN in every place that nothing is written to
    return cache


def feed(cache, x, counts):
    assert cache.reserve(counts).tolist() == list(counts)
    q = cache.append(0, x[:, :H], x[:, H:H + KV], x[:, H + KV:])
    return cache.attend(0, q)


def heads(T, seed):
    return seeded((S, T, H + 2 * KV, D), seed, torch.bfloat16).transpose(1, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("window", [None, 21])
def test_drafts_taken_back_leave_no_trace(dtype, window):
    rng = np.random.default_rng(3)
    cache, twin = make(dtype, window), make(dtype, window)
    x = heads(30, 1)
    assert torch.equal(feed(cache, x, [30, 13, 1]), feed(twin, x, [30, 13, 1]))
    for step in range(14):
        drafted = rng.integers(1, 6, S)
        accepted = np.minimum(rng.integers(0, 6, S), drafted)
        x = heads(5, 10 + step)
        feed(cache, x, drafted.tolist())
        before = cache.lens.clone()
        back = drafted - accepted
        if step % 2:                                     # in two goes, from the GPU
            first = torch.tensor(back // 2, dtype=torch.int32, device="cuda")
            cache.take_back(first)
            cache.take_back(torch.tensor(back, dtype=torch.int64, device="cuda") - first)
        else:
            cache.take_back(back.tolist())
        assert cache.counts.tolist() == accepted.tolist() and (before - cache.lens).tolist() == back.tolist()
        feed(twin, x, accepted.tolist())
        x = heads(1, 50 + step)
        got, want = feed(cache, x, [1] * S), feed(twin, x, [1] * S)
        assert torch.equal(cache.lens, twin.lens) and torch.equal(got, want), step
        assert bool(torch.isfinite(got).all())
        if step % 5 == 4:
            assert cache.reorder([0, 1, 1]).tolist() == twin.reorder([0, 1, 1]).tolist() == [1, 1, 1]
        held = to_np(cache.tables)
        assert (np.bincount(held[held >= 0], minlength=40) == to_np(cache.refs)).all()


def test_no_more_is_taken_back_than_was_granted():
    cache = make(torch.bfloat16, None)
    feed(cache, heads(20, 1), [20, 3, 0])
    cache.take_back([5, -4, 7])
    assert cache.lens.tolist() == [15, 3, 0] and cache.counts.tolist() == [15, 3, 0]
    cache.take_back(4)
    assert cache.lens.tolist() == [11, 0, 0]
    cache.reserve([30, 20, 10])
    cache.reorder([0, 1, 1])                             # forks share full pages: what was granted before stays
    cache.take_back(100)
    assert cache.lens.tolist() == [41, 20, 20] and cache.counts.tolist() == [0, 0, 0]
    for bad in (torch.ones(2, dtype=torch.int32), torch.ones((S, 1), dtype=torch.int32)):
        with pytest.raises(ValueError, match="counts must be"):
            cache.take_back(bad)


def test_a_captured_draft_and_its_taking_back():
    cache, twin = make(torch.bfloat16, 21), make(torch.bfloat16, 21)
    counts, back = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(2))
    x = torch.zeros((S, H + 2 * KV, 3, D), dtype=torch.bfloat16, device="cuda")

    def step(c):
        c.reserve(counts)
        q = c.append(0, x[:, :H], x[:, H:H + KV], x[:, H + KV:])
        out = c.attend(0, q)
        c.take_back(back)
        return out

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
    for n in range(12):
        counts.copy_(torch.tensor([3, n % 4, 1], dtype=torch.int32))
        back.copy_(torch.tensor([n % 3, 1, 0], dtype=torch.int32))
        x.copy_(seeded(x.shape, 70 + n, torch.bfloat16))
        graph.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool(torch.isfinite(out).all()), n
        assert all(torch.equal(getattr(cache, a), getattr(twin, a)) for a in ("tables", "lens", "refs", "counts")), n
    assert cache.lens.tolist() == [24, 9, 12]


def test_whole_numbers_beyond_32_bits_are_not_cut():
    cache = make(torch.bfloat16, None)
    far = torch.tensor([2 ** 32 + 1, 2 ** 31, -2 ** 32 + 3], device="cuda")
    for counts in (far, far.tolist(), far.cpu().numpy()):
        assert cache.reserve(counts).tolist() == [0, 0, 0] and cache.lens.tolist() == [0, 0, 0]
    cache.reserve([3, 2, 1])
    assert cache.reorder(torch.tensor([2 ** 32, 1, -2 ** 32 + 2], device="cuda")).tolist() == [0, 1, 0]
    assert cache.lens.tolist() == [0, 2, 0]
