"""Linear layers in 8-bit floating point with power-of-two block scales (``cuda/fp8_quant.cu``, ``cuda/fp8_gemm.cu``).

A matrix ``[R, C]`` is held as 8-bit codes (``torch.float8_e4m3fn``, or ``torch.float8_e5m2`` for gradients) and one
scale ``2^e`` for every 128 consecutive elements of a row; ``e >= -126`` is the smallest exponent for which the largest
finite magnitude of the block is at most ``FMAX * 2^e`` (448 or 57344).  ``code = round(x * 2^-e)``, ties to even.  NaN
stays NaN; infinities become NaN in e4m3, which has none, and stay infinite in e5m2.  Weights take one scale per
128 x 128 block, so that a weight and its transpose hold the same values.

* ``quantize_fp8`` / ``quantize_fp8_t`` / ``quantize_fp8_pair`` - a matrix, its transpose, or both from one read
* ``quantize_fp8_weight`` - a weight in both orders, kept by the caller (``Fp8Weight``)
* ``gemm_fp8_nt(a, b)`` - ``a @ b.T``; the tensor core applies the scales
* ``add_rmsnorm_fp8`` - residual add + RMSNorm whose result leaves in 8 bits
* ``linear_fp8`` - ``x @ w.T`` with gradients;  ``add_rmsnorm_linear_fp8`` - the norm and the linear layer after it

Gradients pass through the roundings as if they were not there (straight-through):

    y = Q(x) Q(w)^T       dx = Q(dy) Q(w)       dw = Q(dy^T) Q(x^T)^T

with blocks of 128 along each product's own contraction.  CUDA tensors run the kernels; CPU tensors run the PyTorch
statement of the same math, which is also the test oracle.  The reference has no 8-bit path.
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _native as nv
from .gemm import _alloc_out, count_launch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BLOCK = 128
MAX_NORM_WIDTH = 16384
_FMT = {E4M3: 0, E5M2: 1}
_TOP = {E4M3: 8, E5M2: 15}                 # FMAX = 1.75 * 2^TOP
_ROWS, _COLS, _TILES = 1, 2, 4             # mode bits of cvb_fp8_quantize
_OUT = {torch.bfloat16: 0, torch.float32: 1}


def _ceil(a: int, b: int) -> int:
    return (a + b - 1) // b


def _device(t: torch.Tensor):
    """Launches go to the tensor's device and to that device's current stream."""
    if t.device.index is None or t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


# ----------------------------------------------------------------------------
# the 8-bit matrix
# ----------------------------------------------------------------------------
class Fp8Tensor:
    """``[rows, cols]`` in 8 bits.  One buffer: codes, row-major with rows padded to 16 bytes, then the scale bytes in
    the order in which the tensor core reads them (see ``cuda/fp8_common.cuh``)."""

    __slots__ = ("buf", "rows", "cols", "dtype", "ld")

    def __init__(self, buf: torch.Tensor, rows: int, cols: int, dtype: torch.dtype):
        self.buf, self.rows, self.cols, self.dtype = buf, rows, cols, dtype
        self.ld = _ceil(cols, 16) * 16

    @staticmethod
    def nbytes_of(rows: int, cols: int) -> int:
        return rows * _ceil(cols, 16) * 16 + _ceil(rows, BLOCK) * _ceil(cols, 4 * BLOCK) * 512

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.buf.device

    @property
    def sf_ptr(self) -> int:
        return self.buf.data_ptr() + self.rows * self.ld

    @property
    def values(self) -> torch.Tensor:
        """The codes as an 8-bit float view ``[rows, cols]`` (in units of their scales)."""
        return self.buf[:self.rows * self.ld].view(self.dtype).view(self.rows, self.ld)[:, :self.cols]

    def scales(self) -> torch.Tensor:
        """The scales ``[rows, ceil(cols / 128)]`` as ``torch.float8_e8m0fnu`` (powers of two)."""
        nb = _ceil(self.cols, BLOCK)
        out = torch.empty((self.rows, nb), dtype=torch.uint8, device=self.device)
        if out.numel() == 0:
            pass
        elif self.buf.is_cuda:
            with _device(self.buf):
                nv.check(nv.cuda().cvb_fp8_scales(self.sf_ptr, out.data_ptr(), self.rows, nb, nv.stream()),
                         "cvb_fp8_scales")
            count_launch()
        else:
            out.copy_(_scale_cells(self.buf, self.rows, self.cols, self.ld)[:self.rows, :nb])
        return out.view(torch.float8_e8m0fnu)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        s = self.scales().float().repeat_interleave(BLOCK, 1)[:, :self.cols]
        return (self.values.float() * s).to(dtype)


@dataclass
class Fp8Weight:
    """A weight ``[N, K]`` in 8 bits (``w``) and, for gradients of the input, its transpose ``[K, N]`` (``wt``)."""
    w: Fp8Tensor
    wt: Optional[Fp8Tensor]

    @property
    def shape(self) -> Tuple[int, int]:
        return self.w.shape


def _scale_cells(buf: torch.Tensor, rows: int, cols: int, ld: int) -> torch.Tensor:
    """CPU: the scale bytes of a buffer as a fresh plain ``[rows up to 128, blocks up to 4]`` matrix."""
    rt, kg = _ceil(rows, BLOCK), _ceil(cols, 4 * BLOCK)
    cells = buf[rows * ld:rows * ld + rt * kg * 512].view(rt, kg, 32, 4, 4)       # [.., r % 32, r / 32, b % 4]
    return cells.permute(0, 3, 2, 1, 4).reshape(rt * BLOCK, kg * 4)


def _quantize_ref(x: torch.Tensor, dtype: torch.dtype, block_rows: int = 1):
    """Codes (8-bit float ``[R, C]``) and scale bytes (uint8 ``[R, blocks]``) of a matrix, in PyTorch."""
    R, C = x.shape
    nr, nb = _ceil(R, block_rows), _ceil(C, BLOCK)
    p = torch.zeros((nr * block_rows, nb * BLOCK), dtype=torch.float32, device=x.device)
    p[:R, :C] = x.float()
    p = p.view(nr, block_rows, nb, BLOCK)
    amax = torch.where(p.isfinite(), p.abs(), 0.0).amax(dim=(1, 3), keepdim=True)
    byte = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - _TOP[dtype]).clamp(min=1)
    inv = ((254 - byte) << 23).view(torch.float32)
    codes = (p * inv).to(dtype).view(nr * block_rows, nb * BLOCK)[:R, :C]
    return codes, byte.to(torch.uint8).view(nr, nb).repeat_interleave(block_rows, 0)[:R]


def _pack_ref(x: torch.Tensor, dtype: torch.dtype, block_rows: int = 1) -> Fp8Tensor:
    R, C = x.shape
    out = Fp8Tensor(torch.zeros(Fp8Tensor.nbytes_of(R, C), dtype=torch.uint8, device=x.device), R, C, dtype)
    if R == 0 or C == 0:
        return out
    codes, byte = _quantize_ref(x, dtype, block_rows)
    out.buf[:R * out.ld].view(R, out.ld)[:, :C] = codes.contiguous().view(torch.uint8)
    rt, kg = _ceil(R, BLOCK), _ceil(C, 4 * BLOCK)
    cells = torch.ones((rt * BLOCK, kg * 4), dtype=torch.uint8, device=x.device)
    cells[:R, :byte.shape[1]] = byte
    out.buf[R * out.ld:] = cells.view(rt, 4, 32, kg, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    return out


def _check_matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: a tensor is wanted, got {type(x).__name__}")
    if x.dim() != 2:
        raise ValueError(f"{what}: a matrix is wanted, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: bfloat16 or float32 is wanted, got {x.dtype}")
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


def _check_dtype(dtype: torch.dtype, what: str) -> None:
    if dtype not in _FMT:
        raise TypeError(f"{what}: the 8-bit type is torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}")


def _quantize(x: torch.Tensor, dtype: torch.dtype, mode: int, rstd=None, w=None, w_offset: float = 0.0):
    """(row form or None, transposed form or None) by the mode's bits.  With ``rstd`` the values are
    ``x * rstd[row] * (w_offset + w[col])``."""
    R, C = x.shape
    tall = BLOCK if mode & _TILES else 1
    if not x.is_cuda:
        v = x.float() if rstd is None else x.float() * rstd[:, None] * (w_offset + w.float())
        return (_pack_ref(v, dtype, tall) if mode & _ROWS else None,
                _pack_ref(v.t(), dtype, tall) if mode & _COLS else None)
    n_q = Fp8Tensor.nbytes_of(R, C) if mode & _ROWS else 0
    n_t = Fp8Tensor.nbytes_of(C, R) if mode & _COLS else 0
    q = Fp8Tensor(torch.empty(n_q, dtype=torch.uint8, device=x.device), R, C, dtype) if n_q or mode & _ROWS else None
    t = Fp8Tensor(torch.empty(n_t, dtype=torch.uint8, device=x.device), C, R, dtype) if n_t or mode & _COLS else None
    if R and C:
        with _device(x):
            nv.check(nv.cuda().cvb_fp8_quantize(
                x.data_ptr(), int(x.dtype == torch.float32), R, C, x.stride(0), _FMT[dtype], mode,
                q.buf.data_ptr() if q else None, q.sf_ptr if q else None, q.ld if q else 0,
                t.buf.data_ptr() if t else None, t.sf_ptr if t else None, t.ld if t else 0,
                nv.ptr(rstd), nv.ptr(w), w_offset, nv.stream()), "cvb_fp8_quantize")
        count_launch()
    return q, t


@torch.no_grad()
def quantize_fp8(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x [R, C]`` (bf16 or fp32) in 8 bits, one scale per 128 elements of a row."""
    _check_dtype(dtype, "quantize_fp8")
    return _quantize(_check_matrix(x, "quantize_fp8"), dtype, _ROWS)[0]


@torch.no_grad()
def quantize_fp8_t(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x.T [C, R]`` in 8 bits, one scale per 128 rows of ``x``."""
    _check_dtype(dtype, "quantize_fp8_t")
    return _quantize(_check_matrix(x, "quantize_fp8_t"), dtype, _COLS)[1]


@torch.no_grad()
def quantize_fp8_pair(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, Fp8Tensor]:
    """``(quantize_fp8(x), quantize_fp8_t(x))`` from one read of ``x``."""
    _check_dtype(dtype, "quantize_fp8_pair")
    return _quantize(_check_matrix(x, "quantize_fp8_pair"), dtype, _ROWS | _COLS)


@torch.no_grad()
def quantize_fp8_weight(w: torch.Tensor, transposed: bool = True) -> Fp8Weight:
    """A weight ``[N, K]`` in e4m3 with one scale per 128 x 128 block.  ``transposed=False`` leaves the transpose out,
    which only gradients of the layer's input need."""
    w = _check_matrix(w, "quantize_fp8_weight")
    q, t = _quantize(w, E4M3, _ROWS | _TILES | (_COLS if transposed else 0))
    return Fp8Weight(q, t)


# ----------------------------------------------------------------------------
# product
# ----------------------------------------------------------------------------
def gemm_fp8_nt(a: Fp8Tensor, b: Fp8Tensor, out: Optional[torch.Tensor] = None, *,
                out_dtype: Optional[torch.dtype] = None, accumulate: bool = False) -> torch.Tensor:
    """``a [M, K] @ b [N, K].T -> [M, N]`` in bf16 (default) or fp32; ``accumulate`` adds to an fp32 ``out``.
    Either operand may be e4m3 or e5m2.  Sums are fp32; a bf16 result is rounded once."""
    if not isinstance(a, Fp8Tensor) or not isinstance(b, Fp8Tensor):
        raise TypeError("gemm_fp8_nt: both operands are Fp8Tensor")
    if a.cols != b.cols:
        raise ValueError(f"gemm_fp8_nt: {a.shape} and {b.shape} have different contraction lengths")
    if a.device != b.device:
        raise ValueError(f"gemm_fp8_nt: operands on {a.device} and {b.device}")
    M, N, K = a.rows, b.rows, a.cols
    if out is None:
        if accumulate:
            raise ValueError("gemm_fp8_nt: accumulate needs an out")
        dt = out_dtype or torch.bfloat16
        if dt not in _OUT:
            raise TypeError(f"gemm_fp8_nt: the result is bfloat16 or float32, not {dt}")
        out = _alloc_out(M, N, dt, a.device)
    else:
        if tuple(out.shape) != (M, N) or out.device != a.device:
            raise ValueError(f"gemm_fp8_nt: out is {tuple(out.shape)} on {out.device}, not {(M, N)} on {a.device}")
        if out.dtype not in _OUT or (out_dtype is not None and out.dtype != out_dtype):
            raise TypeError(f"gemm_fp8_nt: out has dtype {out.dtype}")
        if accumulate and out.dtype != torch.float32:
            raise TypeError("gemm_fp8_nt: accumulate needs a float32 out")
        if (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"gemm_fp8_nt: out has strides {out.stride()}: rows of unit stride that do not overlap are wanted")
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out if accumulate else out.zero_()
    if not a.buf.is_cuda:
        r = a.dequantize() @ b.dequantize().t()
        return out.add_(r) if accumulate else out.copy_(r)
    with _device(a.buf):
        nv.check(nv.cuda().cvb_fp8_gemm(
            a.buf.data_ptr(), a.sf_ptr, a.ld, _FMT[a.dtype], b.buf.data_ptr(), b.sf_ptr, b.ld, _FMT[b.dtype], M, N, K,
            out.data_ptr(), max(out.stride(0), N), 2 if accumulate else _OUT[out.dtype],
            nv.status_word(a.device).data_ptr(), nv.stream()), "cvb_fp8_gemm")
    count_launch()
    return out


# ----------------------------------------------------------------------------
# residual add + RMSNorm with 8-bit output
# ----------------------------------------------------------------------------
def _check_norm(x, resid, w, what):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_WIDTH:
        raise ValueError(f"{what}: a last dimension of 1 to {MAX_NORM_WIDTH} is wanted, got shape {tuple(x.shape)}")
    if x.is_cuda and (x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16):
        raise TypeError(f"{what}: bfloat16 is wanted on the GPU, got {x.dtype} and a weight in {w.dtype}")
    if tuple(w.shape) != (x.shape[-1],) or w.device != x.device:
        raise ValueError(f"{what}: the weight is {tuple(w.shape)} on {w.device}, the rows have {x.shape[-1]} on {x.device}")
    if resid is not None and (resid.shape != x.shape or resid.dtype != x.dtype or resid.device != x.device):
        raise ValueError(f"{what}: resid is {tuple(resid.shape)} {resid.dtype} on {resid.device}, "
                         f"x is {tuple(x.shape)} {x.dtype} on {x.device}")


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _norm_forward(x2, r2, w, eps, w_offset, dtype, need_rstd: bool):
    """(8-bit rows, h or x2, rstd or None) of matrices."""
    R, D = x2.shape
    if not x2.is_cuda:
        h = x2 if r2 is None else (x2.float() + r2.float()).to(x2.dtype)
        rstd = torch.rsqrt(h.float().pow(2).mean(-1) + eps)
        return _pack_ref(h.float() * rstd[:, None] * (w_offset + w.float()), dtype), h, rstd
    q = Fp8Tensor(torch.empty(Fp8Tensor.nbytes_of(R, D), dtype=torch.uint8, device=x2.device), R, D, dtype)
    h = torch.empty((R, D), dtype=x2.dtype, device=x2.device) if r2 is not None else None
    rstd = torch.empty(R, dtype=torch.float32, device=x2.device) if need_rstd else None
    if R:
        w = w.contiguous()
        with _device(x2):
            nv.check(nv.cuda().cvb_fp8_add_rmsnorm(
                x2.data_ptr(), x2.stride(0), nv.ptr(r2), r2.stride(0) if r2 is not None else 0, w.data_ptr(),
                nv.ptr(h), q.buf.data_ptr(), q.sf_ptr, q.ld, nv.ptr(rstd), R, D, _FMT[dtype], eps, w_offset,
                nv.stream()), "cvb_fp8_add_rmsnorm")
        count_launch()
    return q, (h if h is not None else x2), rstd


@torch.no_grad()
def add_rmsnorm_fp8(x: torch.Tensor, resid: Optional[torch.Tensor], w: torch.Tensor, eps: float = 1e-6,
                    w_offset: float = 1.0, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, torch.Tensor]:
    """``(Q(rmsnorm(x + resid)), x + resid)``; ``resid`` may be None.  The norm is rounded once, from fp32 to 8 bits;
    rows of the result are the rows of ``x`` flattened to a matrix.  For gradients see ``add_rmsnorm_linear_fp8``."""
    _check_dtype(dtype, "add_rmsnorm_fp8")
    _check_norm(x, resid, w, "add_rmsnorm_fp8")
    q, h, _ = _norm_forward(_rows2d(x), _rows2d(resid) if resid is not None else None, w, eps, w_offset, dtype, False)
    return q, (x if resid is None else h.view(x.shape))


# ----------------------------------------------------------------------------
# linear layers
# ----------------------------------------------------------------------------
def _check_linear(K: int, device, w, weight: Optional[Fp8Weight], grad_dtype, what: str) -> None:
    _check_dtype(grad_dtype, what)
    shape = tuple(w.shape)
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f"{what}: a weight [N, {K}] is wanted, got {shape}")
    if isinstance(w, torch.Tensor) and w.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: the weight is bfloat16 or float32, not {w.dtype}")
    if (w.w.device if isinstance(w, Fp8Weight) else w.device) != device:
        raise ValueError(f"{what}: the weight and the input are on different devices")
    if weight is not None and (tuple(weight.shape) != shape or weight.w.device != device):
        raise ValueError(f"{what}: the 8-bit weight is {weight.shape} on {weight.w.device}, the weight {shape} on {device}")


def _weight_grad(qdyt: Fp8Tensor, qxt: Fp8Tensor, w: torch.Tensor):
    """dw = dy^T x: added to ``w.main_grad`` (fp32) where the parameter has one, else returned in its dtype."""
    main = getattr(w, "main_grad", None)
    if main is not None:
        gemm_fp8_nt(qdyt, qxt, main.view(w.shape), accumulate=True)
        return None
    return gemm_fp8_nt(qdyt, qxt, torch.empty(w.shape, dtype=w.dtype, device=w.device))


def _quantize_dy(dy, N, grad_dtype, need_dx, need_dw):
    dy2 = _check_matrix(dy.reshape(-1, N) if dy.numel() else dy.reshape(0, N), "linear_fp8 gradient")
    return _quantize(dy2, grad_dtype, (_ROWS if need_dx else 0) | (_COLS if need_dw else 0))


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, weight, grad_dtype):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        x2 = _rows2d(x)
        if weight is None:
            weight = quantize_fp8_weight(w, transposed=need_dx)
        elif need_dx and weight.wt is None:
            raise ValueError("linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        qx, qxt = _quantize(x2, E4M3, _ROWS | (_COLS if need_dw else 0))
        y = gemm_fp8_nt(qx, weight.w, out_dtype=torch.bfloat16 if x.is_cuda else x.dtype)
        # what the gradients need: x^T and w^T in 8 bits, half of what the bf16 layer keeps of x
        ctx.save_for_backward(w if need_dw else None, qxt.buf if need_dw else None, weight.wt.buf if need_dx else None)
        ctx.cfg = (x.shape, x.dtype, x2.shape[0], w.shape, grad_dtype)
        return y.reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):
        w, qxt, wt = ctx.saved_tensors
        shape, xdtype, M, (N, K), grad_dtype = ctx.cfg
        qdy, qdyt = _quantize_dy(dy, N, grad_dtype, wt is not None, qxt is not None)
        dx = dw = None
        if wt is not None:
            dx = gemm_fp8_nt(qdy, Fp8Tensor(wt, K, N, E4M3), out_dtype=xdtype).reshape(shape)
        if qxt is not None:
            dw = _weight_grad(qdyt, Fp8Tensor(qxt, K, M, E4M3), w)
        return dx, dw, None, None


def linear_fp8(x, w, *, weight: Optional[Fp8Weight] = None, grad_dtype: torch.dtype = E4M3) -> torch.Tensor:
    """``x [..., K] @ w [N, K].T`` with both operands rounded to 8 bits.

    ``w`` is a parameter (its 8-bit form is made in the call, or taken from ``weight`` where the caller keeps one for
    several micro-batches), or an ``Fp8Weight`` for serving and for frozen weights.  ``x`` is a tensor or, without
    gradients, an ``Fp8Tensor`` (from ``add_rmsnorm_fp8``) with a matrix as the result.  Gradients of ``y`` are rounded
    to ``grad_dtype``; the weight's gradient goes to ``w.main_grad`` when the parameter has one."""
    what = "linear_fp8"
    if weight is not None and isinstance(w, Fp8Weight):
        raise ValueError(f"{what}: the 8-bit weight is given twice")
    frozen = w if isinstance(w, Fp8Weight) else None
    if isinstance(x, Fp8Tensor):
        _check_linear(x.cols, x.device, w, weight, grad_dtype, what)
        if frozen is None:
            frozen = weight or quantize_fp8_weight(w, transposed=False)
        return gemm_fp8_nt(x, frozen.w)
    if x.dim() < 1:
        raise ValueError(f"{what}: x has no dimensions")
    if x.dtype != torch.bfloat16 and (x.is_cuda or x.dtype != torch.float32):
        raise TypeError(f"{what}: bfloat16 is wanted, got {x.dtype}")
    _check_linear(x.shape[-1], x.device, w, weight, grad_dtype, what)
    if frozen is not None:
        if not (torch.is_grad_enabled() and x.requires_grad):
            x2 = _rows2d(x)
            y = gemm_fp8_nt(_quantize(x2, E4M3, _ROWS)[0], frozen.w, out_dtype=x.dtype)
            return y.reshape(*x.shape[:-1], w.shape[0])
        return _LinearFp8.apply(x, _Shape(w.shape), frozen, grad_dtype)
    return _LinearFp8.apply(x, w, weight, grad_dtype)


class _Shape:
    """Stands for a frozen weight in the autograd function: only its shape is asked for."""

    def __init__(self, shape):
        self.shape = shape


class _NormLinearFp8(torch.autograd.Function):
    """(linear(rmsnorm(x + resid)), x + resid) with the norm's result in 8 bits only."""

    @staticmethod
    def forward(ctx, x, resid, wn, w, weight, eps, w_offset, grad_dtype):
        need_dn = any(ctx.needs_input_grad[:3])
        need_dw = ctx.needs_input_grad[3]
        if weight is None:
            weight = quantize_fp8_weight(w, transposed=need_dn)
        elif need_dn and weight.wt is None:
            raise ValueError("add_rmsnorm_linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        x2 = _rows2d(x)
        q, h, rstd = _norm_forward(x2, _rows2d(resid) if resid is not None else None, wn, eps, w_offset, E4M3, True)
        y = gemm_fp8_nt(q, weight.w, out_dtype=torch.bfloat16 if x.is_cuda else x.dtype)
        ctx.save_for_backward(h, rstd, wn, w if need_dw else None, weight.wt.buf if need_dn else None)
        ctx.cfg = (x.shape, w.shape, w_offset, grad_dtype, resid is not None, need_dn, need_dw)
        y = y.reshape(*x.shape[:-1], w.shape[0])
        if resid is None:
            return y
        return y, h.view(x.shape)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, rstd, wn, w, wt = ctx.saved_tensors
        shape, (N, K), w_offset, grad_dtype, has_resid, need_dn, need_dw = ctx.cfg
        qdy, qdyt = _quantize_dy(dy, N, grad_dtype, need_dn, need_dw)
        dx = dwn = dw = None
        if need_dw:
            # the norm's result is formed again from h and rstd while its transpose is quantised: it is never stored
            qnt = _quantize(h, E4M3, _COLS, rstd, wn.contiguous(), w_offset)[1]
            dw = _weight_grad(qdyt, qnt, w)
        if need_dn:
            # bf16 between the product and the norm's backward, as between the bf16 layers: half the traffic of fp32
            dn = gemm_fp8_nt(qdy, Fp8Tensor(wt, K, N, E4M3), out_dtype=h.dtype)
            dx, dwn = _norm_backward(dn, h, wn, rstd, dh, w_offset, ctx.needs_input_grad[2])
            dx = dx.view(shape)
        need_x, need_r = ctx.needs_input_grad[:2]
        return (dx if need_x else None), (dx if need_r and has_resid else None), dwn, dw, None, None, None, None


def _norm_backward(dn, h, wn, rstd, dh, w_offset, need_dwn):
    R, D = h.shape
    main = getattr(wn, "main_grad", None) if need_dwn else None
    dh2 = _rows2d(dh) if dh is not None else None
    if not h.is_cuda:
        xh, d32 = h.float() * rstd[:, None], dn.float()
        g = d32 * (w_offset + wn.float())
        dx = rstd[:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
        if dh2 is not None:
            dx = dx + dh2.float()
        dwn = (d32 * xh).sum(0)
        if main is not None:
            main.view(D).add_(dwn)
        return dx.to(h.dtype), dwn.to(wn.dtype) if need_dwn and main is None else None
    lib = nv.cuda()
    dx = torch.empty((R, D), dtype=h.dtype, device=h.device)
    dwn = torch.empty(D, dtype=wn.dtype, device=h.device) if need_dwn and main is None else None
    if R == 0:
        return dx, dwn.zero_() if dwn is not None else None
    part = torch.empty((min(R, lib.cvb_fp8_norm_bwd_parts()), D), dtype=torch.float32, device=h.device) if need_dwn else None
    wc = wn.contiguous()
    with _device(h):
        nv.check(lib.cvb_fp8_norm_bwd(dn.data_ptr(), dn.stride(0), h.data_ptr(), h.stride(0), wc.data_ptr(),
                                      rstd.data_ptr(), nv.ptr(dh2), dh2.stride(0) if dh2 is not None else 0,
                                      dx.data_ptr(), nv.ptr(part), nv.ptr(main), nv.ptr(dwn), R, D, w_offset,
                                      nv.stream()), "cvb_fp8_norm_bwd")
    count_launch(2 if need_dwn else 1)
    return dx, dwn


def add_rmsnorm_linear_fp8(x: torch.Tensor, resid: Optional[torch.Tensor], norm_w: torch.Tensor, w, eps: float = 1e-6,
                           w_offset: float = 1.0, *, weight: Optional[Fp8Weight] = None,
                           grad_dtype: torch.dtype = E4M3) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(rmsnorm(x + resid) @ w.T, x + resid)``; ``resid`` may be None.  The norm's result exists in 8 bits only: the
    backward pass forms it again from ``x + resid``.  ``w``, ``weight`` and ``grad_dtype`` as in ``linear_fp8``."""
    what = "add_rmsnorm_linear_fp8"
    if weight is not None and isinstance(w, Fp8Weight):
        raise ValueError(f"{what}: the 8-bit weight is given twice")
    _check_norm(x, resid, norm_w, what)
    _check_linear(x.shape[-1], x.device, w, weight, grad_dtype, what)
    if isinstance(w, Fp8Weight):
        w, weight = _Shape(w.shape), w
    out = _NormLinearFp8.apply(x, resid, norm_w, w, weight, eps, w_offset, grad_dtype)
    return (out, x) if resid is None else out
