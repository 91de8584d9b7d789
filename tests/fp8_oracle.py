"""Plain 64-bit statements of the block-scaled 8-bit operators, element by element from their definition."""
import torch

FMAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
MANT = {torch.float8_e4m3fn: (3, -6), torch.float8_e5m2: (2, -14)}   # mantissa bits, smallest normal exponent
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def quantize(x, dtype=E4M3, tall=1):
    """(values in units of their scales, scales per element) of a matrix; one scale per `tall` x 128 block."""
    x = x.double()
    R, C = x.shape
    rb, cb = torch.arange(R, device=x.device) // tall, torch.arange(C, device=x.device) // 128
    mag = torch.where(x.isfinite(), x.abs(), 0.0)
    big = torch.zeros((int(rb.max()) + 1, int(cb.max()) + 1), dtype=torch.float64, device=x.device)
    block = rb[:, None] * big.shape[1] + cb[None, :]
    big.view(-1).scatter_reduce_(0, block.reshape(-1), mag.reshape(-1), "amax")
    part, e = torch.frexp(big / FMAX[dtype])
    e = torch.where(part == 0.5, e - 1, e).clamp(min=-126)
    e = torch.where(big == 0, -126, e)
    s = torch.ldexp(torch.ones_like(big), e)[rb][:, cb]
    v = x / s
    bits, low = MANT[dtype]
    _, ve = torch.frexp(torch.where(v.isfinite(), v, 0.0))
    ulp = torch.ldexp(torch.ones_like(v), (ve - 1).clamp(min=low) - bits)
    q = torch.round(v / ulp) * ulp
    q = torch.where(v == 0, 0.0, q)
    if dtype == E4M3:
        q = torch.where(v.isinf(), float("nan"), q)
    else:
        q = torch.where(v.isinf(), v, q)
    return q, s


def through(x, dtype=E4M3, tall=1):
    q, s = quantize(x, dtype, tall)
    return q * s


def value(t):
    """An Fp8Tensor as fp64, from its codes and scales."""
    s = t.scales().double().repeat_interleave(128, 1)[:, :t.cols]
    return t.values.double() * s


def norm(x, r, w, eps, off):
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    hd = h.double()
    rstd = 1.0 / torch.sqrt((hd * hd).mean(-1, keepdim=True) + eps)
    return hd * rstd * (off + w.double()), h, rstd


def norm_grads(h, rstd, w, off, dn, dh):
    xh = h.double() * rstd
    g = dn * (off + w.double())
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
    return dx, (dn * xh).sum(0)
