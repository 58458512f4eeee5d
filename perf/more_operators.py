"""The operators of 8-bit integer linears, and the passes that feed them, as they are measured.

``norm``    root-mean-square norm of rows, with the residual's addition before it, straight into 8 bits with a scale a row.
``act``     GELU, or SwiGLU's product, of rows into 8 bits with a scale a row.
``mm``      the product of two int8 matrices with a scale for each token (row) and channel (column), bias and residual added.
``linear``  the same on activations in bf16: each token's row quantised, then the product.
``train``   an int8 linear's training step: its output, and the gradients of its input, weight and bias.

A row h in 8 bits is codes and a float32 scale s = max(max|h| / Q, 1e-12): int8 codes rne(h / s), Q = 127, or e4m3 codes
of h / s, Q = 448, the quotient a float32 too. The codes are returned as their values in bf16 (which holds each of them), the scales beside them.

Each case is a dict of plain values. ``prepare`` makes what a program holds before the call, ``run`` is one call,
``work`` the bytes and operations that it cannot do without, ``exact`` the same results in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
FLOOR = 1e-12
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------- cases

def listed():
    return [
        # The second norm of a block in a decode step of one sequence: launch and latency.
        dict(name="norm_token", kind="norm", M=1, K=1280, dtype="bf16", residual=True, codes="int8"),
        # A float32 stream of an odd width, the first norm of a stack (nothing to add), into e4m3.
        dict(name="norm_odd", kind="norm", M=4093, K=1031, dtype="f32", residual=False, codes="e4m3"),
        # A prefill of 32 prompts of 2048 tokens, a wide model.
        dict(name="norm_prefill", kind="norm", M=65536, K=4096, dtype="bf16", residual=True, codes="int8"),
        # The SwiGLU product of 24 sequences' decode step (the 450M block's width).
        dict(name="act_step", kind="act", M=24, K=3392, act="swiglu", dtype="bf16", codes="int8"),
        # GELU of a decoder block's prefill, into e4m3.
        dict(name="act_prefill", kind="act", M=32768, K=4096, act="gelu", dtype="bf16", codes="e4m3"),
        # Odd in every size: rows that no vector load takes.
        dict(name="mm_odd", kind="mm", M=517, N=1283, K=1291, bias=False, residual=True),
        # The LM head over the new tokens of 48 sequences.
        dict(name="mm_head", kind="mm", M=48, N=16384, K=1280, bias=False, residual=False),
        # The second projection of a decoder block's MLP over a prefill, with the residual stream.
        dict(name="mm_prefill", kind="mm", M=32768, N=1024, K=4096, bias=False, residual=True),
        # The qkv projection of one new token: the weights' bytes and the launches.
        dict(name="linear_token", kind="linear", M=1, N=3840, K=1280, bias=True, residual=False),
        # The gate projection of a prompt.
        dict(name="linear_prompt", kind="linear", M=8192, N=3392, K=1280, bias=False, residual=False),
        # Fine-tuning on one short, ragged batch.
        dict(name="train_short", kind="train", M=517, N=1280, K=1280, bias=True),
        # The MLP's first projection in a training step of 16384 tokens.
        dict(name="train_batch", kind="train", M=16384, N=5120, K=1280, bias=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "act", "mm", "linear", "train"))
    if kind in ("norm", "act"):
        K = _log_int(rng, 32, 8192)
        K = K if rng.random() < 0.4 else max(32, K // 64 * 64)
        M = _log_int(rng, 1, min(65536, 65536 * 2048 // K))
        how = dict(M=M, K=K, dtype=rng.choice(("bf16", "bf16", "f32")), codes=rng.choice(("int8", "e4m3")))
        if kind == "norm":
            return dict(kind=kind, residual=rng.random() < 0.6, **how)
        return dict(kind=kind, act=rng.choice(("gelu", "swiglu")), **how)
    N, K = _log_int(rng, 64, 16384), _log_int(rng, 64, 8192)
    if kind == "train" or rng.random() < 0.7:
        N, K = max(64, N // 16 * 16), max(64, K // 64 * 64)
    top = 32768 * 1024 * 4096 / (N * K) / (3 if kind == "train" else 1)
    M = _log_int(rng, 16 if kind == "train" else 1, max(17, min(32768, top)))
    if kind == "train":
        return dict(kind=kind, M=M, N=N, K=K, bias=rng.random() < 0.5)
    return dict(kind=kind, M=M, N=N, K=K, bias=rng.random() < 0.5, residual=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------- states

def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _stream(g, M, K, size):
    """Rows as a residual stream has them: a few channels much larger than the others."""
    channels = _normal(g, K).mul_(0.6).exp_().mul_(size)
    return _normal(g, M, K).mul_(channels)


def _int8_of(t):
    """What a weight, or an activation, is as int8 codes and a scale a row."""
    scale = (t.abs().amax(dim=1) / 127.0).clamp(min=FLOOR)
    return (t / scale[:, None]).round().to(torch.int8), scale


def prepare(case, seed):
    c, g = case, _rng(seed)
    s = dict(case)
    if c["kind"] in ("norm", "act"):
        dtype = DTYPE[c["dtype"]]
        if c["kind"] == "norm":
            s["x"] = _stream(g, c["M"], c["K"], 3.0).to(dtype)
            s["a"] = _stream(g, c["M"], c["K"], 0.5).to(dtype) if c["residual"] else None
            s["weight"] = (1.0 + 0.2 * _normal(g, c["K"])).to(dtype)
        else:
            s["x"] = _normal(g, c["M"], c["K"]).to(dtype)
            s["up"] = _normal(g, c["M"], c["K"]).to(dtype) if c["act"] == "swiglu" else None
        return s
    w = _normal(g, c["N"], c["K"]).mul_(c["K"] ** -0.5)
    x = _stream(g, c["M"], c["K"], 1.0)
    s["bias"] = (0.1 * _normal(g, c["N"])).bfloat16() if c["bias"] else None
    if c["kind"] == "train":
        s["weight"], s["x"] = w.bfloat16().requires_grad_(), x.bfloat16().requires_grad_()
        s["g"] = _normal(g, c["M"], c["N"]).mul_(1e-3 * _normal(g, c["M"], 1).exp_()).bfloat16()
        s["bias"] = s["bias"].requires_grad_() if c["bias"] else None
        return s
    s["residual"] = _normal(g, c["M"], c["N"]).bfloat16() if c["residual"] else None
    s["w8"], s["w_scale"] = _int8_of(w)
    if c["kind"] == "mm":
        s["x8"], s["x_scale"] = _int8_of(x)
    else:
        s["x"] = x.bfloat16()
    return s


# ---------------------------------------------------------------------------------------- passes

def _codes(h, kind):
    """The values of rows h (float32) in 8 bits, in units of their scales, and the scales. A row's maximum is divided in 64 bits,
    as torch multiplies by a rounded 1 / Q in 32: a scale one step off moves every value that lies on the border of two codes."""
    scale = (h.abs().amax(dim=1).double() / TOP[kind]).float().clamp(min=FLOOR)
    units = h / scale[:, None]
    return units.round() if kind == "int8" else units.to(torch.float8_e4m3fn).float(), scale


def _normed(s):
    x = s["x"] if s["a"] is None else (s["x"].float() + s["a"].float()).to(s["x"].dtype)
    f = x.float()
    return f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float(), x


def _activated(s):
    x = s["x"].float()
    if s["act"] == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return x / (1.0 + torch.exp(-x)) * s["up"].float()


def _product(x, x_scale, w, w_scale, bias, residual=None):
    y = (x @ w.t()) * x_scale[:, None] * w_scale
    y = y if bias is None else y + bias.float()
    return (y if residual is None else residual.float() + y).bfloat16()


def _gradients(s):
    """Straight through: the products of the gradient with the weight and the input, all in e4m3 with scales along the kept axes."""
    x, w, g = (s[n].detach().float() for n in ("x", "weight", "g"))
    (gr, gr_s), (wc, wc_s) = _codes(g, "e4m3"), _codes(w.t(), "e4m3")
    (gc, gc_s), (xc, xc_s) = _codes(g.t(), "e4m3"), _codes(x.t(), "e4m3")
    dx = (gr @ wc.t()) * gr_s[:, None] * wc_s
    dw = (gc @ xc.t()) * gc_s[:, None] * xc_s
    return dx.bfloat16(), dw.bfloat16(), g.sum(0).bfloat16()


def run(s):
    kind = s["kind"]
    if own:
        from flower_amd import int8
        from flower_amd.kernels import gelu_quant, int8_linear, int8_scaled_mm, rms_norm_quant, swiglu_quant

        if kind == "norm":
            out = rms_norm_quant(s["x"], s["weight"], EPS, residual=s["a"], dtype=_code_type(s))
            return {"codes": out[0].to(torch.bfloat16), "scale": out[1], "sum": out[2] if s["residual"] else None}
        if kind == "act":
            codes, scale = (gelu_quant(s["x"], dtype=_code_type(s)) if s["act"] == "gelu" else
                            swiglu_quant(s["x"], s["up"], dtype=_code_type(s)))
            return {"codes": codes.to(torch.bfloat16), "scale": scale}
        if kind == "mm":
            return int8_scaled_mm(s["x8"], s["x_scale"], s["w8"], s["w_scale"], bias=s["bias"], residual=s["residual"])
        if kind == "linear":
            return int8_linear(s["x"], s["w8"], s["w_scale"], bias=s["bias"], residual=s["residual"])
        leaves = [s[n] for n in ("x", "weight", "bias") if s[n] is not None]
        y = int8.int8_linear_train(s["x"], s["weight"], s["bias"])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["g"])]
    if kind in ("norm", "act"):
        h, total = _normed(s) if kind == "norm" else (_activated(s), None)
        codes, scale = _codes(h, s["codes"])
        out = {"codes": codes.bfloat16(), "scale": scale}
        return {**out, "sum": total if s["residual"] else None} if kind == "norm" else out
    if kind == "mm":
        return _product(s["x8"].float(), s["x_scale"], s["w8"].float(), s["w_scale"], s["bias"], s["residual"])
    x8, x_scale = _codes(s["x"].detach().float(), "int8")
    if kind == "linear":
        return _product(x8, x_scale, s["w8"].float(), s["w_scale"], s["bias"], s["residual"])
    w8, w_scale = _codes(s["weight"].detach().float(), "int8")
    y = _product(x8, x_scale, w8, w_scale, None if s["bias"] is None else s["bias"].detach())
    return [y, *_gradients(s)[:3 if s["bias"] is not None else 2]]


def _code_type(s):
    return torch.int8 if s["codes"] == "int8" else torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    M, K = c["M"], c["K"]
    if c["kind"] in ("norm", "act"):
        size = 2 if c["dtype"] == "bf16" else 4
        if c["kind"] == "norm":
            return {"bytes": M * K * (size * (3 if c["residual"] else 1) + 1) + size * K + 4 * M, "flops": 0}
        return {"bytes": M * K * (size * (2 if c["act"] == "swiglu" else 1) + 1) + 4 * M, "flops": 0}
    N = c["N"]
    if c["kind"] == "train":
        return {"bytes": 2 * (2 * M * K + 2 * M * N + 2 * N * K), "flops": 6 * M * N * K}
    a = M * K + 4 * M if c["kind"] == "mm" else 2 * M * K
    return {"bytes": a + N * K + 4 * N + 2 * M * N * (2 if c["residual"] else 1) + (2 * N if c["bias"] else 0), "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------------------- in 64 bits

def _rounded(x, bits, low):
    """x to the nearest of the numbers with `bits` bits of fraction and exponents from `low`, ties to even."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** low)))
    step = torch.exp2(exponent - bits)
    return torch.round(x / step) * step


def _quantised64(h, kind, axis):
    # the scale is a float32, and so is the quotient: a short number over another lies on the border of two codes often
    s = torch.clamp(torch.linalg.vector_norm(h, ord=math.inf, dim=axis, keepdim=True) / TOP[kind], min=FLOOR).float().double()
    units = (h / s).float().double()
    return torch.round(units) if kind == "int8" else _rounded(units, 3, -6), s


def exact(case, seed):
    s = prepare(case, seed)
    d = {n: t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t for n, t in s.items()}
    if case["kind"] == "norm":
        x = d["x"]
        if case["residual"]:
            # the stream is held in x's type, and the norm is of what is held
            x = (x + d["a"]).to(s["x"].dtype).double()
        h = x / torch.sqrt((x * x).sum(1, keepdim=True) / case["K"] + EPS) * d["weight"]
        codes, scale = _quantised64(h, case["codes"], 1)
        return {"codes": codes, "scale": scale[:, 0], "sum": x if case["residual"] else None}
    if case["kind"] == "act":
        x = d["x"]
        h = torch.special.ndtr(x) * x if case["act"] == "gelu" else torch.sigmoid(x) * x * d["up"]
        codes, scale = _quantised64(h, case["codes"], 1)
        return {"codes": codes, "scale": scale[:, 0]}
    if case["kind"] == "mm":
        a, b = s["x8"].double() * d["x_scale"][:, None], s["w8"].double() * d["w_scale"][:, None]
    else:
        codes, scale = _quantised64(d["x"], "int8", 1)
        a = codes * scale
        if case["kind"] == "train":
            codes, scale = _quantised64(d["weight"], "int8", 1)
            b = codes * scale
        else:
            b = s["w8"].double() * d["w_scale"][:, None]
    y = torch.mm(a, b.t())
    if case["bias"]:
        y = y + d["bias"]
    if case["kind"] != "train":
        return y + d["residual"] if case["residual"] else y
    whole = lambda t, axis: torch.mul(*_quantised64(t, "e4m3", axis))  # noqa: E731
    dx = torch.mm(whole(d["g"], 1), whole(d["weight"], 0))
    dw = torch.mm(whole(d["g"], 0).t(), whole(d["x"], 0))
    return [y, dx, dw, d["g"].sum(0)] if case["bias"] else [y, dx, dw]
