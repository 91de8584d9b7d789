"""Measured work of the 8-bit operators: block-scaled quantisation, residual add + RMSNorm with 8-bit output, and linear
layers whose products run in 8-bit floating point, forward (serving) and forward + backward (training).

Format: codes in e4m3 (or e5m2 for gradients), and for every 128 consecutive elements along the contraction one scale
2^e with the smallest e >= -126 for which the block's largest finite magnitude is at most FMAX * 2^e.  Weights share one
scale per 128 x 128 block.  Widths come from the Qwen3.5-0.8B shape (hidden 1024, feed-forward 3584, gate|up 7168) and
token counts from its benchmark micro-batch (16 x 1280), from decoding batches and from single tokens.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BLOCK = 128
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
TYPE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
MOST = 20480 * 7168 * 1024      # multiply-adds of the largest linear layer


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the hidden state of one token, before a projection of a decode step
        {"name": "quant_token_1x1024", "kind": "quant", "rows": 1, "cols": 1024, "pair": False, "type": "e4m3"},
        # the feed-forward activations of a training micro-batch, for the forward product and for the weight gradient
        {"name": "quant_pair_20480x3584", "kind": "quant", "rows": 20480, "cols": 3584, "pair": True, "type": "e4m3"},
        # the norm of one decoded token
        {"name": "norm_token_1x1024", "kind": "norm", "rows": 1, "cols": 1024, "resid": True},
        # the norms of every layer on a training micro-batch of 32 sequences
        {"name": "norm_train_40960x1024", "kind": "norm", "rows": 40960, "cols": 1024, "resid": True},
        # gate|up projection of one decoded token: the weights are read once
        {"name": "linear_token_1x1024x7168", "kind": "linear", "rows": 1, "k": 1024, "n": 7168},
        # down projection of a decode step of 128 sequences
        {"name": "linear_decode_128x3584x1024", "kind": "linear", "rows": 128, "k": 3584, "n": 1024},
        # a short prompt and widths that are no multiple of anything
        {"name": "linear_ragged_333x1111x1003", "kind": "linear", "rows": 333, "k": 1111, "n": 1003},
        # gate|up projection of a prefill or a scoring pass
        {"name": "linear_prefill_20480x1024x7168", "kind": "linear", "rows": 20480, "k": 1024, "n": 7168},
        # down projection of a training micro-batch, forward and both gradients
        {"name": "train_20480x3584x1024", "kind": "train", "rows": 20480, "k": 3584, "n": 1024, "grad": "e4m3"},
        # a ragged micro-batch with gradients in e5m2
        {"name": "train_ragged_1301x1000x520", "kind": "train", "rows": 1301, "k": 1000, "n": 520, "grad": "e5m2"},
        # norm and gate|up projection of a training micro-batch, forward and all gradients
        {"name": "normlinear_20480x1024x7168", "kind": "normlinear", "rows": 20480, "k": 1024, "n": 7168, "grad": "e4m3"},
        # the same on a few short sequences
        {"name": "normlinear_77x512x1536", "kind": "normlinear", "rows": 77, "k": 512, "n": 1536, "grad": "e4m3"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths of model layers, mostly multiples of 64, and odd ones."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.35 else max(64, (w + 32) // 64 * 64)


def draw(rng):
    kind = rng.choice(["quant", "norm", "linear", "linear", "linear", "train", "train", "normlinear", "normlinear"])
    if kind in ("quant", "norm"):
        cols = _width(rng, 64, 8192)
        rows = min(_log(rng, 1, 20480), 20480 * 3584 // cols)
        if kind == "norm":
            return {"kind": kind, "rows": rows, "cols": cols, "resid": rng.random() < 0.8}
        return {"kind": kind, "rows": rows, "cols": cols, "pair": rng.random() < 0.5,
                "type": rng.choice(["e4m3", "e4m3", "e5m2"])}
    k, n = _width(rng, 64, 8192), _width(rng, 64, 8192)
    room = max(1, MOST // (k * n))
    if kind == "linear":
        return {"kind": kind, "rows": _log(rng, 1, min(20480, room)), "k": k, "n": n}
    return {"kind": kind, "rows": _log(rng, 1, min(20480, room)), "k": k, "n": n, "grad": rng.choice(["e4m3", "e5m2"])}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape, std=1.0):
        return (torch.randn(shape, device=DEV, generator=g) * std).to(torch.bfloat16)

    def acts(rows, cols):
        # activations: a few channels are much larger than the others, rows differ in size
        chan = torch.exp(torch.randn(cols, device=DEV, generator=g))
        row = torch.exp(0.5 * torch.randn((rows, 1), device=DEV, generator=g))
        return (torch.randn((rows, cols), device=DEV, generator=g) * chan * row).to(torch.bfloat16)

    s = dict(case)
    if case["kind"] in ("quant", "norm"):
        s["x"] = acts(case["rows"], case["cols"])
        if case["kind"] == "norm":
            s["r"] = rand(case["rows"], case["cols"]) if case["resid"] else None
            s["wn"] = rand(case["cols"], std=0.1)
        return s
    m, k, n = case["rows"], case["k"], case["n"]
    s["x"] = acts(m, k)
    s["w"] = rand(n, k, std=k ** -0.5)
    if case["kind"] == "linear":        # serving: the weights are converted once and kept
        if own:
            from cverl_b200 import ops
            s["q"] = ops.quantize_fp8_weight(s["w"])
        else:
            s["q"] = _quant_plain(s["w"].float(), "e4m3", BLOCK)
        return s
    s["dy"] = rand(m, n, std=1e-3)
    if case["kind"] == "normlinear":
        s["r"], s["wn"], s["dh"] = rand(m, k), rand(k, std=0.1), rand(m, k, std=1e-3)
        s["r"].requires_grad_(), s["wn"].requires_grad_()
    s["x"].requires_grad_(), s["w"].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------- plain form
def _quant_plain(x, kind, block_rows=1):
    """Codes [R, C] (8-bit floats) and scales [R, ceil(C / 128)] (fp32) of an fp32 matrix."""
    rows, cols = x.shape
    nr, nb = -(-rows // block_rows), -(-cols // BLOCK)
    p = torch.nn.functional.pad(x, (0, nb * BLOCK - cols, 0, nr * block_rows - rows))
    p = p.view(nr, block_rows, nb, BLOCK)
    mag = torch.where(torch.isfinite(p), p.abs(), torch.zeros_like(p)).amax(dim=(1, 3), keepdim=True)
    frac, exp = torch.frexp(mag)
    top, at = math.frexp(FMAX[kind])
    e = torch.where(mag > 0, exp - at + (frac > top).int(), torch.full_like(exp, -126)).clamp(min=-126)
    codes = torch.ldexp(p, -e).to(TYPE[kind]).view(nr * block_rows, nb * BLOCK)[:rows, :cols]
    scale = torch.ldexp(torch.ones_like(mag), e).view(nr, nb).repeat_interleave(block_rows, 0)[:rows]
    return codes, scale


def _value(q):
    codes, scale = q
    return codes.float() * scale.repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _through(x, kind, block_rows=1):
    return _value(_quant_plain(x, kind, block_rows))


def _norm_plain(x, r, wn):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS)
    return hf * rstd * (1.0 + wn.float()), h, rstd


def _linear_grads_plain(x, w, dy, kind):
    """dx (fp32, before rounding) and dW of y = Q(x) Q(w)^T; x and dy fp32."""
    dx = _through(dy, kind) @ _through(w.float(), "e4m3", BLOCK)
    dw = _through(dy.t(), kind) @ _through(x.t(), "e4m3").t()
    return dx, dw.to(w.dtype)


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    kind = s["kind"]
    e8 = torch.float8_e8m0fnu
    if kind == "quant":
        q = _quant_plain(s["x"].float(), s["type"])
        out = {"q": q[0], "s": q[1].to(e8)}
        if s["pair"]:
            t = _quant_plain(s["x"].float().t(), s["type"])
            out |= {"qt": t[0], "st": t[1].to(e8)}
        return out
    if kind == "norm":
        y, h, _ = _norm_plain(s["x"], s["r"], s["wn"])
        q = _quant_plain(y, "e4m3")
        return {"q": q[0], "s": q[1].to(e8), "h": h}
    if kind == "linear":
        return (_through(s["x"].float(), "e4m3") @ _value(s["q"]).t()).to(torch.bfloat16)
    with torch.no_grad():
        x, w, dy = s["x"], s["w"], s["dy"].float()
        if kind == "train":
            y = _through(x.float(), "e4m3") @ _through(w.float(), "e4m3", BLOCK).t()
            dx, dw = _linear_grads_plain(x.float(), w, dy, s["grad"])
            return {"y": y.to(torch.bfloat16), "dx": dx.to(torch.bfloat16), "dw": dw}
        n, h, rstd = _norm_plain(x, s["r"], s["wn"])
        y = _through(n, "e4m3") @ _through(w.float(), "e4m3", BLOCK).t()
        dn, dw = _linear_grads_plain(n, w, dy, s["grad"])
        xhat, g = h.float() * rstd, dn * (1.0 + s["wn"].float())
        dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True)) + s["dh"].float()
        return {"y": y.to(torch.bfloat16), "h": h, "dx": dx.to(torch.bfloat16), "dr": dx.to(torch.bfloat16),
                "dwn": (dn * xhat).sum(0).to(torch.bfloat16), "dw": dw}


# ------------------------------------------------------------------------------------------------- the framework
def _run_own(s):
    from cverl_b200 import ops
    kind = s["kind"]
    if kind == "quant":
        if s["pair"]:
            q, t = ops.quantize_fp8_pair(s["x"], TYPE[s["type"]])
            return {"q": q.values, "s": q.scales(), "qt": t.values, "st": t.scales()}
        q = ops.quantize_fp8(s["x"], TYPE[s["type"]])
        return {"q": q.values, "s": q.scales()}
    if kind == "norm":
        q, h = ops.add_rmsnorm_fp8(s["x"], s["r"], s["wn"], EPS, 1.0)
        return {"q": q.values, "s": q.scales(), "h": h}
    if kind == "linear":
        return ops.linear_fp8(s["x"], s["q"])
    if kind == "train":
        y = ops.linear_fp8(s["x"], s["w"], grad_dtype=TYPE[s["grad"]])
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y, h = ops.add_rmsnorm_linear_fp8(s["x"], s["r"], s["wn"], s["w"], EPS, 1.0, grad_dtype=TYPE[s["grad"]])
    dx, dr, dwn, dw = torch.autograd.grad((y, h), (s["x"], s["r"], s["wn"], s["w"]), (s["dy"], s["dh"]))
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dr": dr, "dwn": dwn, "dw": dw}


# ------------------------------------------------------------------------------------------------- floors, exact values
def work(case):
    if case["kind"] in ("quant", "norm"):
        m, k = case["rows"], case["cols"]
        form = m * k + m * -(-k // BLOCK)
        if case["kind"] == "quant":
            return {"bytes": 2 * m * k + form + (m * k + k * -(-m // BLOCK) if case["pair"] else 0), "flops": 2 * m * k}
        return {"bytes": (6 if case["resid"] else 4) * m * k + form + 2 * k, "flops": 8 * m * k}
    m, k, n = case["rows"], case["k"], case["n"]
    if case["kind"] == "linear":        # the kept weights are 8-bit
        return {"bytes": 2 * m * k + n * k + n * -(-k // BLOCK) + 2 * m * n, "flops": 2 * m * n * k}
    out = 2 * (m * k + n * k + m * n) + 2 * (m * n + m * k + n * k)     # x, w, dy in; y, dx, dw out
    if case["kind"] == "normlinear":
        out += 2 * (4 * m * k + 2 * k)                                 # resid, dh, h, dr; norm weight and its gradient
    return {"bytes": out, "flops": 6 * m * n * k}


def _round64(v, kind):
    """fp64 values rounded to the 8-bit type, ties to even."""
    bits, low = (3, -6) if kind == "e4m3" else (2, -14)
    _, ex = torch.frexp(v)
    ulp = torch.exp2(torch.clamp(ex.double() - 1, min=low) - bits)
    return torch.round(v / ulp) * ulp


def _quant64(x, kind, tall=1):
    """Codes and scales of an fp64 matrix, element by element from the definition; `tall` rows share a scale."""
    rows, cols = x.shape
    nb, nr = -(-cols // BLOCK), -(-rows // tall)
    big = torch.zeros((nr * tall, nb * BLOCK), dtype=torch.float64, device=x.device)
    big[:rows, :cols] = x.abs()
    big = big.reshape(nr, tall, nb, BLOCK).amax((1, 3))
    part, e = torch.frexp(torch.clamp(big, min=1e-300) / FMAX[kind])     # part in [0.5, 1): 2^(e-1) <= ratio < 2^e
    e = torch.where(part == 0.5, e - 1, e).double().clamp(min=-126)
    scale = torch.exp2(e)[torch.arange(rows, device=x.device) // tall]
    return _round64(x / scale[:, torch.arange(cols, device=x.device) // BLOCK], kind), scale


def _near64(x, kind, tall=1):
    q, s = _quant64(x, kind, tall)
    return q * s[:, torch.arange(x.shape[1], device=x.device) // BLOCK]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x = s["x"].double()
        kind = case["kind"]
        if kind == "quant":
            q, sc = _quant64(x, case["type"])
            out = {"q": q, "s": sc}
            if case["pair"]:
                out["qt"], out["st"] = _quant64(x.t().contiguous(), case["type"])
            return out
        if kind in ("norm", "normlinear"):
            h16 = s["x"] if s["r"] is None else (x + s["r"].double()).to(torch.bfloat16)
            h, gain = h16.double(), 1.0 + s["wn"].double()
            inv = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
            x = h * inv * gain
        if kind == "norm":
            q, sc = _quant64(x, "e4m3")
            return {"q": q, "s": sc, "h": h}
        w = _near64(s["w"].double(), "e4m3", BLOCK)
        y = _near64(x, "e4m3") @ w.t()
        if kind == "linear":
            return y
        dy = s["dy"].double()
        dx = _near64(dy, case["grad"]) @ w
        dw = _near64(dy.t().contiguous(), case["grad"]) @ _near64(x.t().contiguous(), "e4m3").t()
        if kind == "train":
            return {"y": y, "dx": dx, "dw": dw}
        dwn = (dx * h * inv).sum(0)
        dx = dx * gain
        dx = inv * dx - h * inv ** 3 * (dx * h).mean(1, keepdim=True) + s["dh"].double()
        return {"y": y, "h": h, "dx": dx, "dr": dx, "dwn": dwn, "dw": dw}
