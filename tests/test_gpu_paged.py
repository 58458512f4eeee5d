"""GPU: paged_append and paged_attention against the float64 oracle, on pools whose unused places hold NaN.

Tolerances. attention: the output's rounding to bf16 (half a step: 2^-8 of the value), and on A = sum p |v| / sum p: what
the weights lose as two bf16 terms (2^-16, twice for the sum they are divided by), the fp32 sums' rounding (a 2^-24 a term)
and the scores' (D products of fp32, 2^-24 of sum |q k| each, exp turning an absolute error of the score into a relative one
of the weight): `slack` of the oracle, doubled for the quotient. append: rounding once from fp32, the norm's factor off by
(D + 8) 2^-24 at most, the rotation by 2^-22. e4m3: half a step is 2^-4 of the value, 2^-10 below the normal range.
"""

import numpy as np
import pytest
import torch

from oracle import paged as O

from gpu_util import seeded, to_np
from test_gpu_rotary import tables as rotary_tables

pytestmark = pytest.mark.gpu

NAN = float("nan")


def values(t):
    """A pool's values as float64 numpy, (e4m3: of the codes)."""
    return t.detach().cpu().float().numpy().astype(np.float64)


def make_cache(B, KV, D, page, lens, cache, *, spare=2, M=None, hold=None, seed=0):
    """A pool with every place NaN except the held positions of each sequence, and tables of shuffled pages; entries
    outside hold[b] = (first, end) positions are -1."""
    g = torch.Generator().manual_seed(seed)
    hold = [(0, n) for n in lens] if hold is None else hold
    M = max([1] + [-(-e // page) for _, e in hold]) if M is None else M
    held = [(b, j) for b, (f, e) in enumerate(hold) for j in range(f // page, -(-e // page))]
    P = len(held) + spare
    ids = torch.randperm(P, generator=g)
    tables = torch.full((B, M), -1, dtype=torch.int32)
    k, v = torch.full((P, KV, page, D), NAN), torch.full((P, KV, D, page), NAN)
    for n, (b, j) in enumerate(held):
        p = int(ids[n])
        tables[b, j] = p
        f, e = max(hold[b][0], j * page) - j * page, min(hold[b][1], (j + 1) * page) - j * page
        k[p, :, f:e] = torch.randn(KV, e - f, D, generator=g)
        v[p, :, :, f:e] = torch.randn(KV, D, e - f, generator=g)
    if cache == "e4m3":
        k, v = (k * 60).to(torch.float8_e4m3fn), (v * 60).to(torch.float8_e4m3fn)
        ks, vs = torch.rand(KV, generator=g) / 40 + 0.01, torch.rand(KV, generator=g) / 40 + 0.01
        return k.cuda(), v.cuda(), tables.cuda(), ks.cuda(), vs.cuda()
    return k.bfloat16().cuda(), v.bfloat16().cuda(), tables.cuda(), None, None


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def check_attention(q, k, v, tables, lens, counts, window, ks, vs, scale=None):
    from flower_amd.kernels import paged_attention
    T, D = q.shape[2], q.shape[3]
    out, lse = paged_attention(q, k, v, tables, ints(lens), None if counts is None else ints(counts), window=window,
                               scale=scale, k_scale=ks, v_scale=vs, return_lse=True)
    counts = [T] * len(lens) if counts is None else counts
    w = 2 ** 31 - 1 if window is None else window
    sc = D ** -0.5 if scale is None else scale
    want, wlse, size, slack = O.attention(values(q), values(k), values(v), to_np(tables), np.array(lens), np.array(counts), w, sc,
                                          None if ks is None else to_np(ks), None if vs is None else to_np(vs))
    got, glse = values(out), to_np(lse).astype(np.float64)
    assert out.dtype == torch.bfloat16 and out.shape == q.shape
    ok = np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + size * (2.0 ** -15 + 2 * slack)
    ok |= np.isnan(got) & np.isnan(want)
    assert ok.all(), (int((~ok).sum()), np.argwhere(~ok)[:4], got[~ok][:4], want[~ok][:4])
    with np.errstate(invalid="ignore"):
        okl = np.abs(glse - wlse) <= slack[..., 0] + 2.0 ** -22 * (1 + np.abs(wlse))
    okl |= (np.isnan(glse) & np.isnan(wlse)) | (glse == wlse)
    assert okl.all(), (np.argwhere(~okl)[:4], glse[~okl][:4], wlse[~okl][:4])
    return out


ATTENTION = [
    # KV, G, T, D, page, cache, lens, counts, window
    (2, 1, 1, 64, 64, "bf16", [1], None, None),
    (2, 1, 1, 64, 64, "bf16", [0, 1, 2, 63, 64, 65, 129], None, None),
    (3, 1, 1, 32, 16, "bf16", [17, 300, 1000], None, None),
    (3, 1, 1, 32, 16, "e4m3", [17, 300, 1000], None, None),
    (1, 8, 1, 128, 32, "bf16", [1, 31, 500], None, None),
    (1, 8, 1, 128, 16, "e4m3", [1, 31, 500], None, None),
    (2, 16, 1, 64, 128, "bf16", [777], None, None),
    (2, 20, 1, 64, 16, "bf16", [500, 90], None, None),              # 20 rows: two row tiles
    (4, 1, 1, 64, 64, "bf16", [5, 200, 700], None, 64),
    (4, 1, 1, 64, 64, "bf16", [5, 200, 700], None, 1),
    (2, 2, 1, 64, 16, "e4m3", [5, 200, 701], None, 77),
    (2, 1, 5, 64, 64, "bf16", [5, 6, 64, 68, 300], None, None),
    (2, 4, 5, 64, 16, "bf16", [5, 6, 64, 68, 300], [5, 3, 1, 5, 0], None),
    (2, 4, 7, 128, 32, "bf16", [7, 150, 411], [7, 7, 2], 50),
    (2, 3, 16, 128, 64, "e4m3", [16, 150, 411], [16, 7, 16], 100),
    (1, 1, 33, 32, 16, "bf16", [33, 90], None, 20),
    (1, 5, 16, 64, 256, "e4m3", [40, 600], None, 3),
    (1, 1, 1, 64, 1024, "bf16", [9000], None, None),
    (1, 4, 1, 64, 64, "bf16", [20000], None, None),                 # cut into parts
    (1, 4, 2, 128, 64, "e4m3", [20001, 3], None, None),
    (1, 4, 6, 64, 64, "bf16", [3000, 9, 1500], [6, 6, 0], None),    # two, four waves of rows, whole items and parts
    (1, 4, 5, 128, 16, "bf16", [2100, 700], None, 1900),
    (2, 8, 5, 128, 16, "e4m3", [2100, 5], [5, 2], None),
    (1, 8, 8, 64, 32, "e4m3", [1500], None, 1000),
    (1, 6, 16, 32, 64, "bf16", [1200, 40], [16, 11], None),         # two groups of rows
    (1, 8, 16, 128, 128, "bf16", [1100], None, 600),
    (4, 3, 1, 64, 64, "bf16", [256, 1, 0, 65, 129], None, None),    # four waves an item, some without a block
    (2, 2, 4, 128, 32, "bf16", [200, 4, 90], [4, 4, 1], 70),
    (2, 1, 2, 32, 16, "e4m3", [255, 2, 64], None, None),
    (40, 1, 1, 64, 16, "e4m3", [500, 3, 130], None, None),
    (70, 2, 1, 32, 64, "bf16", [900, 1000], None, None),
    (1, 5, 8, 128, 64, "bf16", [3000, 8], [8, 3], None),            # three waves of rows
    (2, 3, 16, 32, 16, "e4m3", [1800, 16], None, None),
    (1, 9, 5, 64, 32, "e4m3", [1300, 40], None, 900),
]


@pytest.mark.parametrize("KV,G,T,D,page,cache,lens,counts,window", ATTENTION)
def test_attention(KV, G, T, D, page, cache, lens, counts, window):
    print("[attention]", KV, G, T, D, page, cache, lens, counts, window, flush=True)
    hold = None
    if window is not None:          # pages behind the first new token's window are gone
        cs = [T] * len(lens) if counts is None else counts
        hold = [(max(0, n - c - window + 1), n) for n, c in zip(lens, cs)]
    k, v, tables, ks, vs = make_cache(len(lens), KV, D, page, lens, cache, hold=hold)
    q = seeded((len(lens), T, KV * G, D), 9, torch.bfloat16, scale=1.5).transpose(1, 2)
    check_attention(q, k, v, tables, lens, counts, window, ks, vs)


def test_window_of_nothing_scale_and_wide_tables():
    k, v, tables, _, _ = make_cache(3, 2, 64, 16, [50, 0, 9], "bf16", M=300)
    q = seeded((3, 2, 1, 64), 9, torch.bfloat16)
    out = check_attention(q, k, v, tables, [50, 0, 9], None, 0, None, None)
    assert (out == 0).all()
    check_attention(q, k, v, tables, [50, 0, 9], None, None, None, None, scale=-0.7)


def test_lengths_and_pages_that_are_wrong():
    """A key without a page, an entry that is no page, a query past its table: NaN there, and nothing else changes; a count
    larger than the length, a negative length: no keys. No access leaves the buffers."""
    k, v, tables, _, _ = make_cache(7, 2, 64, 16, [60, 60, 60, 60, 60, 60, 60], "bf16")
    tables[0, 1] = -1
    tables[1, 3] = 10 ** 9
    tables[2, 0] = -5
    tables[6, 0] = k.shape[0]
    q = seeded((7, 2, 1, 64), 9, torch.bfloat16)
    lens = [60, 60, 60, 60, 2 ** 31 - 1, -3, 60]
    out = check_attention(q, k, v, tables, lens, None, None, None, None)
    assert torch.isnan(out[[0, 1, 2, 4, 6]]).all() and torch.isfinite(out[3]).all() and (out[5] == 0).all()
    out = check_attention(q, k, v, tables, lens, None, 20, None, None)      # the bad entries 0 and 1 are behind the window
    assert torch.isfinite(out[[0, 2, 6]]).all() and torch.isnan(out[[1, 4]]).all()
    q = seeded((7, 2, 3, 64), 9, torch.bfloat16)
    check_attention(q, k, v, tables, [2, 0, 60, 65, 66, 64, 1], [9, 3, -2, 3, 3, 2 ** 31 - 1, 3], 15, None, None)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [None, 6])
def test_values_that_are_not_finite_reach_only_who_sees_them(cache, window):
    """A later token's V of NaN (or infinity) is not seen by the tokens before it, nor one that a window has passed."""
    lens, T = [40, 70], 5
    k, v, tables, ks, vs = make_cache(2, 2, 64, 16, lens, cache)
    tab = to_np(tables)
    for b, pos in ((0, 37), (1, 68), (1, 61)):
        if cache == "e4m3":
            v.view(torch.uint8)[tab[b, pos // 16], 1, 3:9, pos % 16] = 0x7F
        else:
            v[tab[b, pos // 16], 1, 3:9, pos % 16] = float("inf")
    q = seeded((2, T, 4, 64), 9, torch.bfloat16).transpose(1, 2)
    from flower_amd.kernels import paged_attention
    got = values(paged_attention(q, k, v, tables, ints(lens), window=window, k_scale=ks, v_scale=vs))
    with np.errstate(invalid="ignore"):
        want, _, size, slack = O.attention(values(q), values(k), values(v), tab, np.array(lens), np.array([T, T]),
                                           window or 2 ** 31 - 1, 0.125, None if ks is None else to_np(ks),
                                           None if vs is None else to_np(vs))
    bad = ~np.isfinite(want)
    assert bad.any() and not bad.all()
    assert np.array_equal(np.isfinite(got), ~bad)
    d = np.abs(got[~bad] - want[~bad])
    assert (d <= 2.0 ** -8 * np.abs(want)[~bad] + (size * (2.0 ** -15 + 2 * slack))[~bad]).all()


def test_scores_that_are_large_low_or_not_finite():
    k, v, tables, _, _ = make_cache(4, 1, 32, 16, [40] * 4, "bf16")
    tab = to_np(tables)
    q = seeded((4, 1, 1, 32), 9, torch.bfloat16)
    q[0] *= 300                                              # one key takes it all
    q[1] = 0                                                 # every key the same
    k[tab[2, 1], 0, 3] = NAN                                 # a seen key
    k[tab[3, 0]] = torch.finfo(torch.bfloat16).min * torch.sign(q[3, 0, 0].float()).bfloat16()      # scores of -inf
    from flower_amd.kernels import paged_attention
    out = paged_attention(q, k, v, tables, ints([40] * 4))
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1, 3]]).all()
    check_attention(q[:2].contiguous(), k, v, tables[:2].contiguous(), [40, 40], None, None, None, None)
    k2 = k.clone()
    k2[tab[3, 0]] = 0.0
    # -inf scores weigh nothing: as a window that begins behind that page
    want = paged_attention(q[3:], k2, v, tables[3:].contiguous(), ints([40]), window=24)
    assert torch.equal(out[3:], want)


def test_offsets_past_32_bits():
    """A pool of 2.6e9 values: pages on both sides of 2^31 and 2^32 bytes, and of 2^31 values."""
    from flower_amd.kernels import paged_append, paged_attention
    P, KV, page, D = 41000, 8, 64, 128
    k = torch.empty((P, KV, page, D), dtype=torch.bfloat16, device="cuda")
    v = torch.empty((P, KV, D, page), dtype=torch.bfloat16, device="cuda")
    ids = [0, 16383, 16384, 32767, 32768, 40999]
    small_k, small_v = seeded((6, KV, page, D), 1, torch.bfloat16), seeded((6, KV, D, page), 2, torch.bfloat16)
    k[ids], v[ids] = small_k, small_v
    q = seeded((2, KV, 1, D), 3, torch.bfloat16)
    lens = ints([300, 384])
    far, near = ints([ids, ids]), ints([list(range(6))] * 2)
    assert torch.equal(paged_attention(q, k, v, far, lens), paged_attention(q, small_k, small_v, near, lens))
    x = seeded((1, 70, 3 * KV, D), 4, torch.bfloat16).transpose(1, 2)
    one = ints([384])
    a = paged_append(x[:, :KV], x[:, KV:2 * KV], x[:, 2 * KV:], k, v, far[:1].contiguous(), one)
    b = paged_append(x[:, :KV], x[:, KV:2 * KV], x[:, 2 * KV:], small_k, small_v, near[:1].contiguous(), one)
    assert torch.equal(a, b) and torch.equal(k[ids], small_k) and torch.equal(v[ids], small_v)


APPEND = [
    # B, H, KV, T, D, R, layout, norm, page, cache, starts, counts
    (1, 4, 4, 1, 64, 64, "interleaved", True, 64, "bf16", [0], None),
    (9, 4, 2, 1, 64, 32, "half", False, 16, "bf16", [0, 1, 15, 16, 17, 63, 64, 100, 7], [1, 1, 1, 1, 0, 1, 1, 1, 1]),
    (2, 2, 1, 5, 128, 128, "half", True, 32, "e4m3", [30, 0], [5, 2]),
    (2, 2, 2, 3, 32, 8, "half", True, 16, "bf16", [14, 31], None),
    (1, 3, 3, 3, 32, 0, "interleaved", False, 16, "e4m3", [14], None),
    (2, 4, 2, 16, 64, 64, "interleaved", True, 16, "bf16", [3, 60], None),
    (3, 4, 2, 130, 64, 64, "interleaved", False, 64, "bf16", [0, 61, 5], [130, 67, 0]),
    (2, 8, 2, 200, 128, 64, "half", True, 16, "e4m3", [9, 64], [200, 1]),
    (1, 2, 1, 77, 32, 32, "half", True, 128, "bf16", [51], None),
]


@pytest.mark.parametrize("B,H,KV,T,D,R,layout,norm,page,cache,starts,counts", APPEND)
def test_append(B, H, KV, T, D, R, layout, norm, page, cache, starts, counts):
    from flower_amd.kernels import paged_append
    print("[append]", B, H, KV, T, D, R, layout, norm, page, cache, starts, counts, flush=True)
    cs = [T] * B if counts is None else counts
    lens = [s + c for s, c in zip(starts, cs)]
    k_pages, v_pages, tables, ks, vs = make_cache(B, KV, D, page, lens, cache)
    before_k, before_v = k_pages.clone(), v_pages.clone()
    x = seeded((B, T, H + 2 * KV, D), 3, torch.bfloat16).transpose(1, 2)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    cos, sin = rotary_tables(max(lens) + 1, R) if R else (None, None)
    qo, ko = paged_append(q, k, v, k_pages, v_pages, tables, ints(lens), None if counts is None else ints(counts), cos=cos,
                          sin=sin, layout=layout, norm_eps=1e-6 if norm else None, k_scale=ks, v_scale=vs, return_k=True)
    pos, live = O.new_positions(np.array(lens), np.array(cs), T)
    rel = (D + 8) * 2.0 ** -24 + 2.0 ** -22

    def turned(x):
        x = O.head_norm(values(x), 1e-6) if norm else values(x)
        return O.rotary(x, to_np(cos), to_np(sin), np.minimum(pos, cos.shape[0] - 1), layout) if R else (x, np.abs(x))
    want, size = turned(q)
    want[~np.broadcast_to(live[:, None], want.shape[:3])] = 0
    assert qo.is_contiguous() and qo.shape == (B, H, T, D)
    assert (np.abs(values(qo) - want) <= 2.0 ** -8 * np.abs(want) + rel * size).all()
    want, size = turned(k)
    m = np.broadcast_to(live[:, None], want.shape[:3])
    assert (np.abs(values(ko) - want)[m] <= (2.0 ** -8 * np.abs(want) + rel * size)[m]).all()
    wk, wv = values(before_k), values(before_v)
    gk, gv = values(k_pages), values(v_pages)
    tab, vn = to_np(tables), values(v)
    untouched = np.ones(wk.shape[:3], bool)
    for b in range(B):
        for t in range(T):
            if not live[b, t]:
                continue
            p, off = tab[b, pos[b, t] // page], pos[b, t] % page
            untouched[p, :, off] = False
            if cache == "bf16":
                assert np.array_equal(gk[p, :, off], values(ko)[b, :, t])
                assert np.array_equal(gv[p, :, :, off], vn[b, :, t])
                continue
            y = np.clip(want[b, :, t] / to_np(ks).astype(np.float64)[:, None], -448, 448)
            slack = rel * size[b, :, t] / to_np(ks)[:, None] * 2
            assert (np.abs(gk[p, :, off] - y) <= 2.0 ** -4 * np.abs(y) + 2.0 ** -10 + slack).all()
            z = (v[b, :, t].float().cpu() / vs.cpu()[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).float().numpy()
            assert np.array_equal(gv[p, :, :, off], z)
    raw = lambda t: t.view(torch.uint8).cpu().numpy().reshape(*t.shape[:3], -1)  # noqa: E731
    assert np.array_equal(raw(k_pages)[untouched], raw(before_k)[untouched])
    same_v = np.broadcast_to(untouched[:, :, None], wv.shape)
    width = k_pages.element_size()
    bytes_v = lambda t: t.view(torch.uint8).cpu().numpy().reshape(*wv.shape, width)  # noqa: E731
    assert np.array_equal(bytes_v(v_pages)[same_v], bytes_v(before_v)[same_v])


@pytest.mark.parametrize("T", [2, 40])
def test_append_without_a_page_or_past_the_tables(T):
    """Positions without a page, and negative ones, are not written; past the rotary tables a token's k is NaN."""
    from flower_amd.kernels import paged_append
    k_pages, v_pages, tables, _, _ = make_cache(5, 2, 64, 16, [100] * 5, "bf16", spare=1)
    before = k_pages.clone(), v_pages.clone()
    x = seeded((5, T, 6, 64), 3, torch.bfloat16).transpose(1, 2)
    bad = tables.clone()
    bad[0, :] = -1
    bad[1, :] = k_pages.shape[0]
    bad[2, :] = 10 ** 9
    cos, sin = rotary_tables(4, 64)
    args = x[:, :2], x[:, 2:4], x[:, 4:], k_pages, v_pages
    q = paged_append(*args, bad, ints([100, 100, 100, 7 * 16 + T, T - 1 - 2]), ints([T, T, T, T, T]), cos=cos, sin=sin)
    assert torch.isnan(q[:4]).all()
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))  # noqa: E731
    tab = to_np(tables)
    new = max(0, T - 3)                                      # of the last sequence, at positions 0 ..
    k_old, v_old = before[0].clone(), before[1].clone()
    for t in range(new):
        k_old[tab[4, t // 16], :, t % 16] = k_pages[tab[4, t // 16], :, t % 16]
        v_old[tab[4, t // 16], :, :, t % 16] = x[4, 4:, t + 3]
        assert torch.isfinite(k_pages[tab[4, t // 16], :, t % 16]).all() == (t < 4)
    assert same(k_pages, k_old) and same(v_pages, v_old)
    assert (q[4, :, :3] == 0).all()


def test_e4m3_append_of_large_and_odd_values():
    """Beyond the scale's range a value saturates at 448 (infinity too), NaN stays NaN."""
    from flower_amd.kernels import paged_append
    k_pages, v_pages, tables, _, _ = make_cache(1, 1, 32, 16, [20], "e4m3")
    s = torch.tensor([0.5]).cuda()
    x = torch.zeros((1, 1, 20, 32), dtype=torch.bfloat16, device="cuda")
    x[0, 0, :, 0], x[0, 0, :, 1], x[0, 0, :, 2], x[0, 0, :, 3] = 1e30, float("-inf"), NAN, 223.0
    paged_append(x, x, x, k_pages, v_pages, tables, ints([20]), k_scale=s, v_scale=s)
    tab = to_np(tables)
    for pos in (0, 15, 16, 19):
        for row in (values(k_pages)[tab[0, pos // 16], 0, pos % 16], values(v_pages)[tab[0, pos // 16], 0, :, pos % 16]):
            assert row[0] == 448 and row[1] == -448 and np.isnan(row[2]) and row[3] == 448 and (row[4:] == 0).all()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_decode_equals_the_prompt_at_once(cache):
    """A prompt appended and attended at once, in pieces, and token by token, each in a cache of its own: the same keys and
    values in the pages bit for bit, and the attention of every token within its tolerance of the definition."""
    from flower_amd.kernels import paged_append, paged_attention
    T, H, KV, D, page, W = 24, 4, 2, 64, 16, 10
    x = seeded((1, T, H + 2 * KV, D), 3, torch.bfloat16).transpose(1, 2)
    cos, sin = rotary_tables(T, D)
    first = None
    for chunks in ([T], [1] * T, [7, 1, 9, 7]):
        k_pages, v_pages, tables, ks, vs = make_cache(1, KV, D, page, [T], cache)
        at, got, qs = 0, [], []
        for n in chunks:
            y = x[:, :, at:at + n]
            at += n
            q = paged_append(y[:, :H], y[:, H:H + KV], y[:, H + KV:], k_pages, v_pages, tables, ints([at]), cos=cos, sin=sin,
                             norm_eps=1e-6, k_scale=ks, v_scale=vs)
            qs.append(q)
            got.append(paged_attention(q, k_pages, v_pages, tables, ints([at]), window=W, k_scale=ks, v_scale=vs))
        q, got = torch.cat(qs, dim=2), values(torch.cat(got, dim=2))
        pages = k_pages.view(torch.uint8).cpu(), v_pages.view(torch.uint8).cpu(), q
        first = pages if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(first, pages))
        want, _, size, slack = O.attention(values(q), values(k_pages), values(v_pages), to_np(tables), np.array([T]),
                                           np.array([T]), W, D ** -0.5, None if ks is None else to_np(ks),
                                           None if vs is None else to_np(vs))
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + size * (2.0 ** -15 + 2 * slack)).all()


def test_strided_q_side_streams_and_two_at_once():
    """q with other strides, calls on two streams at once: each as alone."""
    from flower_amd.kernels import paged_attention
    k, v, tables, _, _ = make_cache(2, 2, 64, 64, [9000, 3000], "bf16")
    lens = ints([9000, 3000])
    q = seeded((2, 2, 4, 1, 64), 9, torch.bfloat16)          # every other head of a wider tensor
    wide = torch.zeros((2, 8, 3, 72), dtype=torch.bfloat16, device="cuda")
    wide[:, ::2, 1:2, :64] = q[:, 0]
    want = [paged_attention(q[:, i].contiguous(), k, v, tables, lens) for i in (0, 1)]
    assert torch.equal(paged_attention(wide[:, ::2, 1:2, :64], k, v, tables, lens), want[0])
    odd = torch.zeros((2, 4, 1, 65), dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = q[:, 0]
    assert torch.equal(paged_attention(odd[..., 1:], k, v, tables, lens), want[0])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(q[:, i].contiguous(), k, v, tables, lens))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
