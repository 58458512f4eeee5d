"""The operators of serving from a paged key-value cache, and the rotary positions that feed it, as they are measured.

``rotary``    rotary positions of q and k, forward and gradients: pairs next to each other or half a rotation apart, the
              whole head or its first part, positions given per token.
``append``    the new tokens' heads on their way into the cache: QK-norm and rotary positions of q and k, then k and v
              written to their pages in bf16, or in e4m3 with one scale a head.
``attention`` one or a few new tokens of each sequence against its pages, under a sliding window or none.
``pages``     the cache's bookkeeping on the device: ``reserve`` (room for the next tokens, pages behind the window given
              back), ``reorder`` (sequences forked, dropped or put in another order, as a beam search does), ``compact``
              (the pages in use moved to the front of the pool).

A cache holds, for each of L layers, keys as (pages, kv heads, page size, D) and values as (pages, kv heads, D, page size);
``tables`` (sequences, entries) int32 names the page of each run of ``page size`` positions of a sequence, -1 where it
holds none; ``lens`` (sequences) int32 counts its positions; ``refs`` (pages) int32 how many tables hold a page.

Each case is a dict of plain values. ``prepare`` makes what a program holds before the call, ``run`` is one call,
``work`` the bytes and operations that it cannot do without, ``exact`` the same results in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
EPS = 1e-6


# ---------------------------------------------------------------------------------------- cases

def listed():
    return [
        # A short prompt of a small model: launches and host time. Half of each head turns, halves layout.
        dict(name="rotary_short", kind="rotary", B=2, H=8, KV=8, T=77, D=64, R=32, layout="half", dtype="bf16", factor=1.0),
        # One training step's heads of the 450M model, interleaved as the model has it.
        dict(name="rotary_train_450m", kind="rotary", B=2, H=20, KV=20, T=8192, D=64, R=64, layout="interleaved",
             dtype="bf16", factor=1.0),
        # A decode step of 64 sequences of the 450M model: its heads into a bf16 cache.
        dict(name="append_decode_450m", kind="append", B=64, H=20, KV=20, T=1, D=64, R=64, layout="interleaved",
             norm=True, page=64, cache="bf16", start=1500),
        # A prompt of 8192 tokens into an e4m3 cache with shared heads, odd start.
        dict(name="append_prompt_8k_e4m3", kind="append", B=1, H=16, KV=4, T=8192, D=128, R=64, layout="half",
             norm=False, page=64, cache="e4m3", start=13),
        # One user's first tokens: what a call costs when there is next to nothing to read.
        dict(name="attention_one_short", kind="attention", B=1, H=16, KV=16, T=1, D=64, page=64, cache="bf16", lo=100,
             hi=100, window=0),
        # A full batch of the 450M model with its window, lengths mixed.
        dict(name="attention_450m_batch", kind="attention", B=64, H=20, KV=20, T=1, D=64, page=64, cache="bf16", lo=300,
             hi=8192, window=2048),
        # Few long sequences with shared heads: work has to be split over the length.
        dict(name="attention_long_gqa", kind="attention", B=4, H=32, KV=4, T=1, D=128, page=64, cache="bf16", lo=70001,
             hi=131072, window=0),
        # Five drafted tokens checked at once, e4m3 cache, small pages, odd lengths.
        dict(name="attention_verify_e4m3", kind="attention", B=16, H=16, KV=2, T=5, D=128, page=16, cache="e4m3", lo=37,
             hi=9001, window=0),
        # Two beam groups of a small model: latency.
        dict(name="reorder_small", kind="reorder", S=8, beams=4, keep=2, L=2, KV=8, D=64, page=64, len=421, cache="bf16"),
        # Sixteen groups of four beams over twelve layers of the 450M model's heads.
        dict(name="reorder_450m", kind="reorder", S=64, beams=4, keep=2, L=12, KV=20, D=64, page=64, len=1007, cache="bf16"),
        # Room for the next token of 256 sequences under the 450M model's window.
        dict(name="reserve_256", kind="reserve", S=256, M=512, pages=12288, page=64, new=1, window=2048, lo=1, hi=16000),
        # A pool half in use drawn together before it is shrunk.
        dict(name="compact_1k", kind="compact", S=32, M=64, pages=1024, live=500, L=4, KV=8, D=64, page=64, cache="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "append", "append", "attention", "attention", "attention", "attention",
                       "reorder", "reorder", "reserve", "compact"))
    D = rng.choice((32, 64, 64, 128, 128))
    KV = rng.choice((1, 2, 4, 8, 16, 20))
    H = KV * rng.choice((1, 1, 2, 4, 8) if KV <= 8 else (1, 1, 2))
    page = rng.choice((16, 32, 64, 64, 128))
    cache = rng.choice(("bf16", "bf16", "e4m3"))
    if kind == "rotary":
        R = rng.choice((D, D, D // 2, D // 4))
        T = _log_int(rng, 1, 8192)
        B = rng.randint(1, max(1, min(8, 2 * 8192 * 40 * 64 // (T * (H + KV) * D))))
        return dict(kind=kind, B=B, H=H, KV=KV, T=T, D=D, R=R, layout=rng.choice(("interleaved", "half")),
                    dtype=rng.choice(("bf16", "bf16", "fp32")), factor=rng.choice((1.0, 4.0)))
    if kind == "append":
        T = rng.choice((1, 1, rng.randint(2, 9), _log_int(rng, 10, 4000)))
        B = _log_int(rng, 1, max(1, min(128, 8192 // T)))
        return dict(kind=kind, B=B, H=H, KV=KV, T=T, D=D, R=rng.choice((D, D, D // 2)),
                    layout=rng.choice(("interleaved", "half")), norm=rng.random() < 0.5, page=page, cache=cache,
                    start=_log_int(rng, 1, 2000) - 1)
    if kind == "attention":
        T = rng.choice((1, 1, 1, 1, 2, rng.randint(3, 16)))
        hi = _log_int(rng, 1, 60000)
        most = 4 * 4 * 131072 * 128 // 8                 # an eighth of the largest listed case's keys
        B = _log_int(rng, 1, max(1, min(128, most // (hi * KV * D))))
        return dict(kind=kind, B=B, H=H, KV=KV, T=T, D=D, page=page, cache=cache, lo=max(1, int(hi * rng.random())), hi=hi,
                    window=rng.choice((0, 0, _log_int(rng, 1, 4096))))
    if kind == "reorder":
        beams = rng.randint(2, 8)
        S = beams * rng.randint(1, 6)
        KV = rng.choice((1, 2, 4, 8))
        return dict(kind=kind, S=S, beams=beams, keep=rng.randint(1, beams), L=rng.randint(1, 4), KV=KV, D=D, page=page,
                    len=_log_int(rng, 1, 1500), cache=cache)
    if kind == "reserve":
        hi = _log_int(rng, 10, 16000)
        new = rng.choice((1, 1, rng.randint(2, 300)))
        S = _log_int(rng, 1, 256)
        M = -(-hi // page) + rng.randint(0, 8)
        return dict(kind=kind, S=S, M=M, pages=S * (-(-hi // page) + 1) + rng.randint(1, 4000), page=page, new=new,
                    window=rng.choice((0, 0, _log_int(rng, 1, 4096))), lo=1, hi=hi)
    M = rng.randint(1, 64)
    S = rng.randint(1, 32)
    pages = rng.randint(max(2, S * M), S * M + 500)
    return dict(kind=kind, S=S, M=M, pages=pages, live=rng.randint(1, S * M), L=rng.randint(1, 2), KV=rng.choice((1, 2, 4)),
                D=D, page=page, cache=cache)


# ---------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(rows, R, factor):
    """cos and sin [rows, R / 2] fp32 of position / factor x 10000^(-2 i / R), the angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] / factor * freq
    return angle.cos().float(), angle.sin().float()


def _heads(g, B, H, KV, T, D, dtype):
    """q, k, v as a fused projection gives them: (B, heads, T, D) views of one (B, T, (H + 2 KV) D) tensor, heads of
    different scale."""
    n = H + 2 * KV
    x = _randn(g, B, T, n, D) * (0.5 * _randn(g, 1, 1, n, 1)).exp()
    x = x.to(dtype).transpose(1, 2)
    return x[:, :H], x[:, H:H + KV], x[:, H + KV:]


def _pool(g, L, pages, KV, page, D, cache):
    """Keys and values that earlier tokens left, (L, pages, KV, page, D) and (L, pages, KV, D, page)."""
    k, v = _randn(g, L, pages, KV, page, D), _randn(g, L, pages, KV, D, page)
    if cache == "bf16":
        return k.bfloat16(), v.bfloat16()
    return (k * 80).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), (v * 80).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _scales(g, KV, cache):
    if cache == "bf16":
        return None, None
    return (torch.rand(KV, generator=g, device="cuda") + 0.5) / 80, (torch.rand(KV, generator=g, device="cuda") + 0.5) / 80


def _spread(n, lo, hi):
    """n lengths from lo to hi, both among them where n allows."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def prepare(case, seed):
    g, c = _gen(seed), case
    kind = c["kind"]
    if kind == "rotary":
        dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
        q, k, _ = _heads(g, c["B"], c["H"], c["KV"], c["T"], c["D"], dtype)
        gq, gk, _ = _heads(g, c["B"], c["H"], c["KV"], c["T"], c["D"], dtype)
        cos, sin = _tables(c["T"] + 64, c["R"], c["factor"])
        start = torch.randint(0, 64, (c["B"], 1), generator=g, device="cuda")
        positions = (start + torch.arange(c["T"], device="cuda")).to(torch.int32)
        return dict(case=c, q=q.requires_grad_(), k=k.requires_grad_(), gq=gq.contiguous(), gk=gk.contiguous(), cos=cos,
                    sin=sin, positions=positions)
    if kind == "append":
        B, T, page = c["B"], c["T"], c["page"]
        q, k, v = _heads(g, B, c["H"], c["KV"], T, c["D"], torch.bfloat16)
        # sequences at different lengths; one in eight (never the first) is idle, one in eight has fewer new tokens
        starts = [(c["start"] + 37 * b) % (c["start"] + 700) if b else c["start"] for b in range(B)]
        counts = [0 if b % 8 == 5 else (T + 1) // 2 if b % 8 == 3 else T for b in range(B)]
        lens = [s + n for s, n in zip(starts, counts)]
        M = -(-max(lens) // page) + 1
        pages = sum(-(-n // page) for n in lens) + 3
        tables = torch.full((B, M), -1, dtype=torch.int32, device="cuda")
        ids = _perm(g, pages).to(torch.int32)
        held = torch.arange(M, device="cuda") < _ints([-(-n // page) for n in lens])[:, None]
        tables[held] = ids[:int(held.sum())]
        k_pages, v_pages = _pool(g, 1, pages, c["KV"], page, c["D"], c["cache"])
        ks, vs = _scales(g, c["KV"], c["cache"])
        cos, sin = _tables(max(lens) + 1, c["R"], 1.0)
        if ks is not None:
            ks, vs = ks * 3, vs * 3                      # the widest heads still saturate
        return dict(case=c, q=q, k=k, v=v, k_pages=k_pages[0], v_pages=v_pages[0], tables=tables, lens=_ints(lens),
                    counts=_ints(counts), cos=cos, sin=sin, k_scale=ks, v_scale=vs)
    if kind == "attention":
        B, T, page = c["B"], c["T"], c["page"]
        lens = torch.tensor(_spread(B, c["lo"], c["hi"]))
        lens = lens.to("cuda", torch.int32)[_perm(g, B)]
        counts = lens.clamp(max=T)
        M = -(-c["hi"] // page)
        first = (lens - counts - c["window"] + 1).clamp(min=0) // page if c["window"] else torch.zeros_like(lens)
        j = torch.arange(M, device="cuda")
        held = (j >= first[:, None]) & (j * page < lens[:, None])
        pages = int(held.sum())
        tables = torch.full((B, M), -1, dtype=torch.int32, device="cuda")
        tables[held] = _perm(g, pages).to(torch.int32)
        k_pages, v_pages = _pool(g, 1, pages, c["KV"], page, c["D"], c["cache"])
        ks, vs = _scales(g, c["KV"], c["cache"])
        q = (1.5 * _randn(g, B, T, c["H"], c["D"])).bfloat16().transpose(1, 2)
        return dict(case=c, q=q, k_pages=k_pages[0], v_pages=v_pages[0], tables=tables, lens=lens, counts=counts, k_scale=ks,
                    v_scale=vs)
    if kind == "reorder":
        S, page, n, beams = c["S"], c["page"], c["len"], c["beams"]
        M = -(-n // page) + 1
        full, shared = n // page, (n // page) // 2           # the first half of a group's full pages is its prompt's
        ids = _perm(g, S * M + S).to(torch.int32)
        tables = torch.full((S, M), -1, dtype=torch.int32, device="cuda")
        rows = torch.arange(S, device="cuda")
        j = torch.arange(M, device="cuda")
        owner = torch.where(j < shared, rows[:, None] // beams * beams, rows[:, None])
        held = (j < -(-n // page)).expand(S, M)
        tables[held] = ids[(owner * M + j)[held]]
        refs = torch.zeros(S * M + S, dtype=torch.int32, device="cuda")
        refs.scatter_add_(0, tables[held].long(), torch.ones(int(held.sum()), dtype=torch.int32, device="cuda"))
        # each group continues `keep` of its beams, in any order and any number of times
        pick = torch.rand(S // beams, beams, generator=g, device="cuda").argsort(dim=1)[:, :c["keep"]]
        again = torch.randint(0, c["keep"], (S // beams, beams), generator=g, device="cuda")
        again[:, :c["keep"]] = torch.arange(c["keep"], device="cuda")
        again = again.gather(1, torch.rand(S // beams, beams, generator=g, device="cuda").argsort(dim=1))
        parents = (pick.gather(1, again) + torch.arange(S // beams, device="cuda")[:, None] * beams).reshape(-1).to(torch.int32)
        k_pages, v_pages = _pool(g, c["L"], S * M + S, c["KV"], page, c["D"], c["cache"])
        return dict(case=c, k_pages=k_pages, v_pages=v_pages, tables=tables, lens=torch.full_like(parents, n), refs=refs,
                    parents=parents, out=(torch.empty_like(tables), torch.empty_like(parents), torch.empty_like(refs)))
    if kind == "reserve":
        S, M, page = c["S"], c["M"], c["page"]
        lens = torch.tensor(_spread(S, c["lo"], c["hi"])).to("cuda", torch.int32)[_perm(g, S)]
        counts = torch.where(torch.rand(S, generator=g, device="cuda") < 0.1, 0, c["new"]).to(torch.int32)
        j = torch.arange(M, device="cuda")
        held = j * page < lens[:, None]
        if c["window"]:                                      # the step before gave back what its window had passed
            held &= ((j + 1) * page > lens[:, None] - c["window"]) | (torch.rand(S, 1, generator=g, device="cuda") < 0.1)
        tables = torch.full((S, M), -1, dtype=torch.int32, device="cuda")
        ids = _perm(g, c["pages"]).to(torch.int32)
        tables[held] = ids[torch.arange(int(held.sum()), device="cuda") % c["pages"]]
        refs = torch.zeros(c["pages"], dtype=torch.int32, device="cuda")
        refs.scatter_add_(0, tables[held].long(), torch.ones(int(held.sum()), dtype=torch.int32, device="cuda"))
        return dict(case=c, tables=tables, lens=lens, refs=refs, counts=counts,
                    out=(torch.empty_like(tables), torch.empty_like(lens), torch.empty_like(refs)))
    S, M, P = c["S"], c["M"], c["pages"]
    ids = _perm(g, P)[:c["live"]].to(torch.int32)
    tables = torch.full((S, M), -1, dtype=torch.int32, device="cuda")
    tables.view(-1)[_perm(g, S * M)[:c["live"]]] = ids
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    refs[ids.long()] = 1
    tables.view(-1)[_perm(g, S * M)[:2]] = ids[0]            # a page that several tables hold
    refs.zero_().scatter_add_(0, tables.view(-1).clamp(min=0).long(), (tables.view(-1) >= 0).int())
    k_pages, v_pages = _pool(g, c["L"], P, c["KV"], c["page"], c["D"], c["cache"])
    return dict(case=c, k_pages=k_pages, v_pages=v_pages, tables=tables, refs=refs,
                out=(torch.empty_like(tables), torch.empty_like(refs)))


# ---------------------------------------------------------------------------------------- plain forms

def _turn(x, cos, sin, layout, back=False):
    """x (..., D) fp32 with its first R = 2 cos.shape[-1] values turned by the angles (the other way with ``back``)."""
    R = 2 * cos.shape[-1]
    sin = -sin if back else sin
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if layout == "interleaved" else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), dim=-1).flatten(-2) if layout == "interleaved" else torch.cat((a, b), dim=-1)
    return torch.cat((turned, x[..., R:]), dim=-1)


def _plain_rotary(s):
    layout, pos = s["case"]["layout"], s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    with torch.no_grad():
        return [_turn(s[n].float(), cos, sin, layout, back).to(s[n].dtype)
                for n, back in (("q", False), ("k", False), ("gq", True), ("gk", True))]


def _plain_append(s):
    c = s["case"]
    page, T = c["page"], c["T"]
    t = torch.arange(T, device="cuda")
    live = t < s["counts"][:, None]
    pos = torch.where(live, (s["lens"] - s["counts"])[:, None] + t, 0).long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS)
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS)
    q, k = _turn(q, cos, sin, c["layout"]), _turn(k, cos, sin, c["layout"])
    q = torch.where(live[:, None, :, None], q, 0).bfloat16()
    k, v = k.transpose(1, 2)[live], v.transpose(1, 2)[live]              # (tokens, KV, D)
    ids = s["tables"].gather(1, pos // page)[live].long()
    at = (pos % page)[live]
    dtype = s["k_pages"].dtype
    if dtype != torch.bfloat16:
        k = (k / s["k_scale"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        v = (v / s["v_scale"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        s["k_pages"].view(torch.uint8)[ids, :, at] = k.to(dtype).view(torch.uint8)
        s["v_pages"].view(torch.uint8)[ids, :, :, at] = v.to(dtype).view(torch.uint8)
    else:
        s["k_pages"][ids, :, at] = k.to(dtype)
        s["v_pages"][ids, :, :, at] = v.to(dtype)
    return [q, s["k_pages"], s["v_pages"]]


def _plain_attention(s):
    c = s["case"]
    B, H, T, D = s["q"].shape
    KV, page = c["KV"], c["page"]
    M = s["tables"].shape[1]
    ids = s["tables"].clamp(min=0).long()
    byte = torch.uint8 if s["k_pages"].element_size() == 1 else torch.bfloat16
    k = s["k_pages"].view(byte)[ids].view(s["k_pages"].dtype).float().transpose(1, 2).reshape(B, KV, M * page, D)
    v = s["v_pages"].view(byte)[ids].view(s["v_pages"].dtype).float().permute(0, 2, 1, 4, 3).reshape(B, KV, M * page, D)
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    q = s["q"].float().reshape(B, KV, H // KV * T, D)
    t = torch.arange(T, device="cuda")
    at = torch.where(t < s["counts"][:, None], (s["lens"] - s["counts"])[:, None] + t, -1)       # a query's position
    j = torch.arange(M * page, device="cuda")
    seen = j <= at[..., None]
    if c["window"]:
        seen &= j > at[..., None] - c["window"]
    seen = seen[:, None, None].expand(B, KV, H // KV, T, M * page).reshape(B, KV, H // KV * T, M * page)
    x = torch.where(seen, torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D), -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return torch.where(m == -math.inf, 0.0, o).bfloat16().reshape(B, H, T, D)


def _held(refs, tables, sign):
    """refs with `sign` added for every entry of tables that holds a page."""
    flat = tables.reshape(-1)
    return refs.scatter_add(0, flat.clamp(min=0).long(), sign * (flat >= 0).to(torch.int32))


def _free_first(refs):
    """The pages' numbers, the free ones first, each part in ascending order."""
    return torch.argsort((refs != 0).to(torch.int32), stable=True).to(torch.int32)


def _plain_reserve(s):
    c = s["case"]
    page, M, P = c["page"], c["M"], c["pages"]
    lens, counts, tables, refs = s["lens"], s["counts"], s["tables"], s["refs"]
    j = torch.arange(M, device="cuda", dtype=torch.int32)
    if c["window"]:
        gone = (tables >= 0) & ((j + 1) * page <= (lens - c["window"] + 1)[:, None])
        refs = _held(refs, torch.where(gone, tables, -1), -1)
        tables = torch.where(gone, -1, tables)
    fits = (counts > 0) & (lens >= 0) & (lens + counts <= M * page)
    wanted = fits[:, None] & ((j + 1) * page > lens[:, None]) & (j * page < (lens + counts)[:, None]) & (tables < 0)
    need = wanted.sum(1)
    upto = need.cumsum(0)
    given = fits & ((need == 0) | (upto <= (refs == 0).sum()))
    place = (upto - need)[:, None] + wanted.cumsum(1) - 1
    tables = torch.where(wanted & given[:, None], _free_first(refs)[place.clamp(0, P - 1)], tables)
    refs = _held(refs, torch.where(wanted & given[:, None], tables, -1), 1)
    return [tables, torch.where(given, lens + counts, lens), refs, torch.where(given, counts, 0)]


def _plain_reorder(s):
    c = s["case"]
    page, S, M = c["page"], c["S"], s["tables"].shape[1]
    parents, tables = s["parents"].long(), s["tables"]
    P = s["refs"].shape[0]
    me, j = torch.arange(S, device="cuda"), torch.arange(M, device="cuda")
    real = (parents >= 0) & (parents < S)
    pr = torch.where(real, parents, 0)
    n = torch.where(real, s["lens"][pr], 0)
    # of a sequence's children, the one in its own place keeps its last page, or else the first
    rank = torch.where(parents == me, -1, me)
    best = torch.full((S + 1,), S, device="cuda").scatter_reduce(0, torch.where(real, parents, S), rank, "amin")
    keeps = real & (best[pr] == rank)
    last = tables[pr].gather(1, (n // page).clamp(max=M - 1)[:, None].long())[:, 0]
    need = real & ~keeps & (n % page != 0) & (last >= 0)
    rows = torch.where(keeps[:, None] | (real[:, None] & (j < (n // page)[:, None])), tables[pr], -1)
    refs = _held(_held(s["refs"], tables, -1), rows, 1)
    upto = need.to(torch.int32).cumsum(0)
    given = ~need | (upto <= (refs == 0).sum())
    new = _free_first(refs)[(upto - 1).clamp(0, P - 1)]
    copied = need & given
    refs = _held(refs, torch.where(given[:, None], -1, rows), -1)
    rows = torch.where(given[:, None], rows, -1)
    rows = torch.where(copied[:, None] & (j == (n // page)[:, None]), new[:, None], rows)
    refs = _held(refs, torch.where(copied, new, -1), 1)
    dst, src, used = new[copied].long(), last[copied].long(), (n % page)[copied]
    mine = torch.arange(page, device="cuda") < used[:, None]             # (copies, page)
    for_bytes = torch.uint8 if s["k_pages"].element_size() == 1 else torch.bfloat16
    k, v = s["k_pages"].view(for_bytes), s["v_pages"].view(for_bytes)
    k[:, dst] = torch.where(mine[:, None, :, None], k[:, src], k[:, dst])
    v[:, dst] = torch.where(mine[:, None, None, :], v[:, src], v[:, dst])
    return [rows, torch.where(given, n, 0).to(torch.int32), refs, s["k_pages"], s["v_pages"]]


def _plain_compact(s):
    tables, refs = s["tables"], s["refs"]
    P = refs.shape[0]
    ids = torch.arange(P, device="cuda")
    used = refs != 0
    n = used.sum()
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    to = ids.clone()
    to[src] = dst
    for_bytes = torch.uint8 if s["k_pages"].element_size() == 1 else torch.bfloat16
    k, v = s["k_pages"].view(for_bytes), s["v_pages"].view(for_bytes)
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    moved = refs.clone()
    moved[dst] = refs[src]
    moved[src] = 0
    return [torch.where(tables >= 0, to[tables.clamp(min=0).long()], -1).to(torch.int32), moved, n.to(torch.int32).reshape(1),
            s["k_pages"], s["v_pages"]]


# ---------------------------------------------------------------------------------------- the calls

def _own(s):
    import flower_amd.kernels as K
    c = s["case"]
    kind = c["kind"]
    if kind == "rotary":
        turned = K.apply_rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], layout=c["layout"])
        return [t.detach() for t in turned] + list(torch.autograd.grad(turned, (s["q"], s["k"]), (s["gq"], s["gk"])))
    if kind == "append":
        q = K.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["counts"],
                           cos=s["cos"], sin=s["sin"], layout=c["layout"], norm_eps=EPS if c["norm"] else None,
                           k_scale=s["k_scale"], v_scale=s["v_scale"])
        return [q, s["k_pages"], s["v_pages"]]
    if kind == "attention":
        return K.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["counts"],
                                 window=c["window"] or None, k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "reserve":
        return list(K.reserve_pages(s["tables"], s["lens"], s["refs"], s["counts"], c["page"], window=c["window"] or None,
                                    out=s["out"]))
    if kind == "reorder":
        return [*K.reorder_pages(s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["refs"], s["parents"], out=s["out"]),
                s["k_pages"], s["v_pages"]]
    return [*K.compact_pages(s["k_pages"], s["v_pages"], s["tables"], s["refs"], out=s["out"]), s["k_pages"], s["v_pages"]]


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "reserve": _plain_reserve,
          "reorder": _plain_reorder, "compact": _plain_compact}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------- work

def work(case):
    c = case
    kind = c["kind"]
    if kind == "rotary":
        size = 2 if c["dtype"] == "bf16" else 4
        values = c["B"] * c["T"] * (c["H"] + c["KV"]) * c["D"]
        return {"bytes": 4 * size * values + 4 * c["T"] * c["R"] + 4 * c["B"] * c["T"], "flops": 6 * values * c["R"] // c["D"]}
    if kind == "append":
        size = 2 if c["cache"] == "bf16" else 1
        tokens = sum(0 if b % 8 == 5 else (c["T"] + 1) // 2 if b % 8 == 3 else c["T"] for b in range(c["B"]))
        q, kv = c["H"] * c["D"], 2 * c["KV"] * c["D"]
        return {"bytes": tokens * (2 * q + 2 * kv + size * kv + 4 * c["R"]) + 2 * c["B"] * c["T"] * q, "flops": 6 * tokens * (q + kv)}
    if kind == "attention":
        size = 2 if c["cache"] == "bf16" else 1
        lens = _spread(c["B"], c["lo"], c["hi"])
        reach = c["window"] or c["hi"] + 1
        keys = sum(min(n, reach + min(n, c["T"]) - 1) for n in lens)
        pairs = sum(min(n - t, reach) for n in lens for t in range(min(n, c["T"])))
        return {"bytes": 2 * size * keys * c["KV"] * c["D"] + 4 * c["B"] * c["T"] * c["H"] * c["D"] + 4 * keys // c["page"],
                "flops": 4 * pairs * c["H"] * c["D"]}
    if kind == "reserve":
        return {"bytes": 8 * c["S"] * c["M"] + 8 * c["pages"] + 16 * c["S"], "flops": 0}
    size = 2 if c["cache"] == "bf16" else 1
    token = 2 * size * c["L"] * c["KV"] * c["D"]
    if kind == "reorder":
        copies = c["S"] // c["beams"] * (c["beams"] - c["keep"])
        M = -(-c["len"] // c["page"]) + 1
        return {"bytes": 2 * copies * (c["len"] % c["page"]) * token + 8 * c["S"] * M + 8 * c["S"] * (M + 1) + 12 * c["S"],
                "flops": 0}
    moved = c["live"] * (c["pages"] - c["live"]) // c["pages"]
    return {"bytes": 2 * moved * c["page"] * token + 8 * c["S"] * c["M"] + 8 * c["pages"], "flops": 0}


# ---------------------------------------------------------------------------------------- the definition in 64 bits

def _rotation(cos, sin, D, layout):
    """(..., D, D) matrices of the rotary positions: y = x M^T."""
    half = cos.shape[-1]
    m = torch.eye(D, dtype=torch.float64, device="cuda").expand(*cos.shape[:-1], D, D).clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + half)
        m[..., a, a], m[..., b, b] = cos[..., i], cos[..., i]
        m[..., a, b], m[..., b, a] = -sin[..., i], sin[..., i]
    return m


def _exact_turn(x, cos, sin, positions, layout, transpose=False):
    """x (B, H, T, D): every token's head vectors times that token's matrix, some tokens at a time."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    B, H, T, D = x.shape
    step = max(1, (1 << 26) // (D * D))
    for b in range(B):
        for t in range(0, T, step):
            pos = positions[b, t:t + step].long()
            m = _rotation(cos[pos].double(), sin[pos].double(), D, layout)
            m = m.transpose(1, 2) if transpose else m
            out[b, :, t:t + step] = torch.matmul(m, x[b, :, t:t + step].double().permute(1, 2, 0).contiguous()).permute(2, 0, 1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    kind = c["kind"]
    if kind == "rotary":
        with torch.no_grad():
            turn = lambda x, back: _exact_turn(x, s["cos"], s["sin"], s["positions"], c["layout"], back)  # noqa: E731
            return [turn(s["q"], False), turn(s["k"], False), turn(s["gq"], True), turn(s["gk"], True)]
    if kind == "append":
        lens, counts = s["lens"].tolist(), s["counts"].tolist()
        B, T, page = c["B"], c["T"], c["page"]
        pos = (s["lens"] - s["counts"])[:, None] + torch.arange(T, device="cuda")
        pos = pos.clamp(max=s["cos"].shape[0] - 1)
        norm = lambda x: x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() if c["norm"] else x  # noqa: E731
        q = _exact_turn(norm(s["q"].double()), s["cos"], s["sin"], pos, c["layout"])
        k = _exact_turn(norm(s["k"].double()), s["cos"], s["sin"], pos, c["layout"])
        if c["cache"] == "bf16":
            k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        for b in range(B):
            q[b, :, counts[b]:] = 0
            if c["cache"] == "bf16" and counts[b]:
                at = torch.arange(lens[b] - counts[b], lens[b], device="cuda")
                ids = s["tables"][b].long()[at // page]
                k_pages[ids, :, at % page] = k[b, :, :counts[b]].transpose(0, 1)
                v_pages[ids, :, :, at % page] = s["v"][b, :, :counts[b]].double().transpose(0, 1)
        return [q, k_pages, v_pages] if c["cache"] == "bf16" else [q, None, None]
    if kind == "attention":
        B, H, T, D = s["q"].shape
        KV, page, G = c["KV"], c["page"], H // c["KV"]
        out = torch.zeros(B, H, T, D, dtype=torch.float64, device="cuda")
        lens, counts = s["lens"].tolist(), s["counts"].tolist()
        for b in range(B):
            for t in range(counts[b]):
                last = lens[b] - counts[b] + t
                first = max(0, last - c["window"] + 1) if c["window"] else 0
                at = torch.arange(first, last + 1, device="cuda")
                ids = s["tables"][b].long()[at // page]
                byte = torch.uint8 if c["cache"] == "e4m3" else torch.bfloat16
                k = s["k_pages"].view(byte)[ids, :, at % page].view(s["k_pages"].dtype).double()             # (n, KV, D)
                v = s["v_pages"].view(byte)[ids, :, :, at % page].view(s["v_pages"].dtype).double()
                if s["k_scale"] is not None:
                    k, v = k * s["k_scale"].double()[:, None], v * s["v_scale"].double()[:, None]
                q = s["q"][b, :, t].double().view(KV, G, D)
                p = torch.softmax(torch.matmul(q, k.permute(1, 2, 0).contiguous()) / D ** 0.5, dim=-1)
                out[b, :, t] = torch.matmul(p, v.transpose(0, 1).contiguous()).view(H, D)
        return out
    return None


