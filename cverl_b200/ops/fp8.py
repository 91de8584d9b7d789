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

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _native as nv
from .gemm import count_launch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BLOCK = 128
MAX_NORM_WIDTH = 16384
_FMT = {E4M3: 0, E5M2: 1}
_TOP = {E4M3: 8, E5M2: 15}                 # FMAX = 1.75 * 2^TOP
_ROWS, _COLS, _TILES = 1, 2, 4             # mode bits of cvb_fp8_quantize
_OUT = {torch.bfloat16: 0, torch.float32: 1}


def _ceil(a: int, b: int) -> int:
    return (a + b - 1) // b


class _On:
    """Launches of a block go to one device: ``stream`` is that device's current stream, ``status`` its status word."""

    __slots__ = ("index", "before", "stream", "status")

    def __init__(self, t: torch.Tensor):
        self.index = t.get_device()

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        self.stream = nv.raw_stream(self.index)
        self.status = nv.status_word(self.index).data_ptr()
        return self

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _bytes(n: int, device: torch.device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


def _alloc_rows(M: int, N: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """``[M, N]`` whose rows start on 32 bytes (what the vector stores of the product want)."""
    per32 = 16 if dtype == torch.bfloat16 else 8
    if N % per32 == 0:
        return torch.empty((M, N), dtype=dtype, device=device)
    return torch.empty((M, _ceil(N, per32) * per32), dtype=dtype, device=device)[:, :N]


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
            with _On(out) as on:
                nv.check(nv.cuda().cvb_fp8_scales(self.sf_ptr, out.data_ptr(), self.rows, nb, on.stream), "cvb_fp8_scales")
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
        x = x.detach()
        v = x.float() if rstd is None else x.float() * rstd[:, None] * (w_offset + w.float())
        return (_pack_ref(v, dtype, tall) if mode & _ROWS else None,
                _pack_ref(v.t(), dtype, tall) if mode & _COLS else None)
    q = t = None
    q_args = t_args = (None, None, 0)
    if mode & _ROWS:
        q = Fp8Tensor(_bytes(Fp8Tensor.nbytes_of(R, C), x.device), R, C, dtype)
        q_args = (q.buf.data_ptr(), q.sf_ptr, q.ld)
    if mode & _COLS:
        t = Fp8Tensor(_bytes(Fp8Tensor.nbytes_of(C, R), x.device), C, R, dtype)
        t_args = (t.buf.data_ptr(), t.sf_ptr, t.ld)
    if R and C:
        with _On(x) as on:
            nv.check(nv.cuda().cvb_fp8_quantize(
                x.data_ptr(), x.dtype == torch.float32, R, C, x.stride(0), _FMT[dtype], mode, *q_args, *t_args,
                nv.ptr(rstd), nv.ptr(w), w_offset, on.stream), "cvb_fp8_quantize")
        count_launch()
    return q, t


def quantize_fp8(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x [R, C]`` (bf16 or fp32) in 8 bits, one scale per 128 elements of a row."""
    _check_dtype(dtype, "quantize_fp8")
    return _quantize(_check_matrix(x, "quantize_fp8"), dtype, _ROWS)[0]


def quantize_fp8_t(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x.T [C, R]`` in 8 bits, one scale per 128 rows of ``x``."""
    _check_dtype(dtype, "quantize_fp8_t")
    return _quantize(_check_matrix(x, "quantize_fp8_t"), dtype, _COLS)[1]


def quantize_fp8_pair(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, Fp8Tensor]:
    """``(quantize_fp8(x), quantize_fp8_t(x))`` from one read of ``x``."""
    _check_dtype(dtype, "quantize_fp8_pair")
    return _quantize(_check_matrix(x, "quantize_fp8_pair"), dtype, _ROWS | _COLS)


def quantize_fp8_weight(w: torch.Tensor, transposed: bool = True) -> Fp8Weight:
    """A weight ``[N, K]`` in e4m3 with one scale per 128 x 128 block.  ``transposed=False`` leaves the transpose out,
    which only gradients of the layer's input need."""
    q, t = _quantize(_check_matrix(w, "quantize_fp8_weight"), E4M3, _ROWS | _TILES | (_COLS if transposed else 0))
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
        out = _alloc_rows(M, N, dt, a.device)
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
    with _On(out) as on:
        nv.check(nv.cuda().cvb_fp8_gemm(
            a.buf.data_ptr(), a.sf_ptr, a.ld, _FMT[a.dtype], b.buf.data_ptr(), b.sf_ptr, b.ld, _FMT[b.dtype], M, N, K,
            out.data_ptr(), max(out.stride(0), N), 2 if accumulate else _OUT[out.dtype], on.status, on.stream),
            "cvb_fp8_gemm")
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
    q = Fp8Tensor(_bytes(Fp8Tensor.nbytes_of(R, D), x2.device), R, D, dtype)
    h = torch.empty((R, D), dtype=x2.dtype, device=x2.device) if r2 is not None else None
    rstd = torch.empty(R, dtype=torch.float32, device=x2.device) if need_rstd else None
    if R:
        w = w.contiguous()
        with _On(x2) as on:
            nv.check(nv.cuda().cvb_fp8_add_rmsnorm(
                x2.data_ptr(), x2.stride(0), nv.ptr(r2), r2.stride(0) if r2 is not None else 0, w.data_ptr(),
                nv.ptr(h), q.buf.data_ptr(), q.sf_ptr, q.ld, nv.ptr(rstd), R, D, _FMT[dtype], eps, w_offset,
                on.stream), "cvb_fp8_add_rmsnorm")
        count_launch()
    return q, (h if h is not None else x2), rstd


def add_rmsnorm_fp8(x: torch.Tensor, resid: Optional[torch.Tensor], w: torch.Tensor, eps: float = 1e-6,
                    w_offset: float = 1.0, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, torch.Tensor]:
    """``(Q(rmsnorm(x + resid)), x + resid)``; ``resid`` may be None.  The norm is rounded once, from fp32 to 8 bits;
    rows of the result are the rows of ``x`` flattened to a matrix.  For gradients see ``add_rmsnorm_linear_fp8``."""
    _check_dtype(dtype, "add_rmsnorm_fp8")
    _check_norm(x, resid, w, "add_rmsnorm_fp8")
    r2 = _rows2d(resid.detach()) if resid is not None else None
    q, h, _ = _norm_forward(_rows2d(x.detach()), r2, w.detach(), eps, w_offset, dtype, False)
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


def _forward(x2, xq, w, weight: Optional[Fp8Weight], M, N, K, need_wt: bool, need_xt: bool, dtype):
    """``(y, xt, wt)``: the product and the transposed 8-bit forms that gradients read (buffers or None).  ``x2`` is the
    input's rows or None where ``xq`` is its 8-bit form; ``w`` the weight or None where ``weight`` is."""
    device = (x2 if x2 is not None else xq.buf).device
    y = _alloc_rows(M, N, dtype, device)
    if not y.is_cuda:
        xt = None
        if x2 is not None:
            xq, xt = _quantize(x2, E4M3, _ROWS | (_COLS if need_xt else 0))
        weight = weight or quantize_fp8_weight(w, transposed=need_wt)
        gemm_fp8_nt(xq, weight.w, y)
        return y, xt.buf if xt else None, weight.wt.buf if need_wt else None
    xt = _bytes(Fp8Tensor.nbytes_of(K, M), device) if need_xt else None
    xb = xq.buf if xq is not None else _bytes(Fp8Tensor.nbytes_of(M, K), device)
    if weight is None:
        w = _check_matrix(w, "linear_fp8 weight")
        wq = _bytes(Fp8Tensor.nbytes_of(N, K), device)
        wt = _bytes(Fp8Tensor.nbytes_of(K, N), device) if need_wt else None
    else:
        w, wq, wt = None, weight.w.buf, weight.wt.buf if need_wt else None
    if M and N and K:
        with _On(y) as on:
            nv.check(nv.cuda().cvb_fp8_linear_fwd(
                nv.ptr(x2), x2 is not None and x2.dtype == torch.float32, x2.stride(0) if x2 is not None else 0,
                nv.ptr(w), w is not None and w.dtype == torch.float32, w.stride(0) if w is not None else 0, M, N, K,
                xb.data_ptr(), nv.ptr(xt), wq.data_ptr(), nv.ptr(wt) if weight is None else None,
                y.data_ptr(), max(y.stride(0), N), _OUT[dtype], on.status, on.stream), "cvb_fp8_linear_fwd")
        count_launch(1 + (x2 is not None) + (w is not None))
    else:
        if weight is None:      # no rows: the gradient of the input is empty too, and reads nothing
            weight = quantize_fp8_weight(w, transposed=need_wt)
            wt = weight.wt.buf if need_wt else None
        y.zero_()
    return y, xt, wt


def _backward(dy, M, N, K, grad_dtype, wt, xt, w, dx_dtype, norm=None):
    """``(dx or None, dw or None)`` of ``y = x w^T``: dx where ``wt`` is given, dw where the parameter ``w`` is (added
    to its fp32 ``main_grad`` where it has one, and then None).  ``norm = (h, rstd, wn, w_offset)`` stands for ``xt``."""
    dy2 = _check_matrix(dy.reshape(-1, N) if dy.numel() else dy.reshape(0, N), "linear_fp8 gradient")
    dx = _alloc_rows(M, K, dx_dtype, dy.device) if wt is not None else None
    main = getattr(w, "main_grad", None) if w is not None else None
    target = None
    if w is not None:
        target = main.view(N, K) if main is not None else _alloc_rows(N, K, w.dtype, dy.device)
    if not (M and N and K):
        if dx is not None:
            dx.zero_()
        if target is not None and main is None:
            target.zero_()
    elif not dy2.is_cuda:
        qdy, qdyt = _quantize(dy2, grad_dtype, (_ROWS if wt is not None else 0) | (_COLS if w is not None else 0))
        if dx is not None:
            gemm_fp8_nt(qdy, Fp8Tensor(wt, K, N, E4M3), dx)
        if target is not None:
            if norm is not None:
                xt = _quantize(norm[0], E4M3, _COLS, *norm[1:])[1].buf
            gemm_fp8_nt(qdyt, Fp8Tensor(xt, K, M, E4M3), target, accumulate=main is not None)
    else:
        if main is not None and (main.dtype != torch.float32 or not main.is_contiguous()):
            raise TypeError("linear_fp8: main_grad is a contiguous float32 tensor")
        dyq = _bytes(Fp8Tensor.nbytes_of(M, N), dy.device) if wt is not None else None
        dyt = _bytes(Fp8Tensor.nbytes_of(N, M), dy.device) if w is not None else None
        h = rstd = wn = None
        w_offset = 0.0
        if norm is not None and w is not None:
            h, rstd, wn, w_offset = norm
            xt = _bytes(Fp8Tensor.nbytes_of(K, M), dy.device)
        with _On(dy2) as on:
            nv.check(nv.cuda().cvb_fp8_linear_bwd(
                dy2.data_ptr(), dy2.dtype == torch.float32, dy2.stride(0), _FMT[grad_dtype], M, N, K, nv.ptr(dyq),
                nv.ptr(dyt), nv.ptr(wt), nv.ptr(xt), nv.ptr(h), h.stride(0) if h is not None else 0, nv.ptr(rstd),
                nv.ptr(wn), w_offset, nv.ptr(dx), max(dx.stride(0), K) if dx is not None else 0,
                _OUT[dx_dtype], nv.ptr(target), max(target.stride(0), K) if target is not None else 0,
                2 if main is not None else _OUT[w.dtype] if w is not None else 0, on.status, on.stream),
                "cvb_fp8_linear_bwd")
        count_launch(1 + (wt is not None) + (w is not None) + (h is not None))
    return dx, (target if main is None else None)


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, weight, grad_dtype):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        if need_dx and weight is not None and weight.wt is None:
            raise ValueError("linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        x2 = _rows2d(x)
        (M, K), N = x2.shape, w.shape[0]
        y, xt, wt = _forward(x2, None, w, weight, M, N, K, need_dx, need_dw, x.dtype)
        # what the gradients read: x^T and w^T in 8 bits, half of what the bf16 layer keeps of x
        ctx.save_for_backward(w if need_dw else None, xt, wt)
        ctx.cfg = (x.shape, x.dtype, M, N, K, grad_dtype)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        w, xt, wt = ctx.saved_tensors
        shape, xdtype, M, N, K, grad_dtype = ctx.cfg
        dx, dw = _backward(dy, M, N, K, grad_dtype, wt, xt, w, xdtype)
        if dx is not None and len(shape) != 2:
            dx = dx.reshape(shape)
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
    N = w.shape[0] if len(w.shape) else 0
    if isinstance(x, Fp8Tensor):
        _check_linear(x.cols, x.device, w, weight, grad_dtype, what)
        if x.dtype != E4M3:
            raise TypeError(f"{what}: inputs are torch.float8_e4m3fn, got {x.dtype}")
        with torch.no_grad():
            return _forward(None, x, w, frozen or weight, x.rows, N, x.cols, False, False, torch.bfloat16)[0]
    if x.dim() < 1:
        raise ValueError(f"{what}: x has no dimensions")
    if x.dtype != torch.bfloat16 and (x.is_cuda or x.dtype != torch.float32):
        raise TypeError(f"{what}: bfloat16 is wanted, got {x.dtype}")
    _check_linear(x.shape[-1], x.device, w, weight, grad_dtype, what)
    if not (torch.is_grad_enabled() and (x.requires_grad or (frozen is None and w.requires_grad))):
        x2 = _rows2d(x)
        y = _forward(x2, None, w, frozen or weight, x2.shape[0], N, x2.shape[1], False, False, x.dtype)[0]
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)
    if frozen is not None:
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
        need_dn, need_dw = any(ctx.needs_input_grad[:3]), ctx.needs_input_grad[3]
        if need_dn and weight is not None and weight.wt is None:
            raise ValueError("add_rmsnorm_linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        x2 = _rows2d(x)
        (M, K), N = x2.shape, w.shape[0]
        q, h, rstd = _norm_forward(x2, _rows2d(resid) if resid is not None else None, wn, eps, w_offset, E4M3,
                                   need_dn or need_dw)
        y, _, wt = _forward(None, q, w, weight, M, N, K, need_dn, False, x.dtype)
        ctx.save_for_backward(h, rstd, wn, w if need_dw else None, wt)
        ctx.cfg = (x.shape, M, N, K, w_offset, grad_dtype)
        if x.dim() != 2:
            y = y.reshape(*x.shape[:-1], N)
        return y if resid is None else (y, h.view(x.shape))

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, rstd, wn, w, wt = ctx.saved_tensors
        shape, M, N, K, w_offset, grad_dtype = ctx.cfg
        need_x, need_r, need_wn = ctx.needs_input_grad[:3]
        # The norm's result is formed again from h and rstd while its transpose is quantised: it is never stored.  Its
        # gradient stays fp32 between the product and the norm's backward.
        dn, dw = _backward(dy, M, N, K, grad_dtype, wt, None, w, torch.float32, (h, rstd, wn.contiguous(), w_offset))
        dx = dwn = None
        if dn is not None:
            dx, dwn = _norm_backward(dn, h, wn, rstd, dh, w_offset, need_wn)
            dx = dx.view(shape)
        return (dx if need_x else None), (dx if need_r else None), dwn, dw, None, None, None, None


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
    if main is not None and (main.dtype != torch.float32 or not main.is_contiguous()):
        raise TypeError("add_rmsnorm_linear_fp8: main_grad is a contiguous float32 tensor")
    wc = wn.contiguous()
    with _On(h) as on:
        nv.check(lib.cvb_fp8_norm_bwd(dn.data_ptr(), dn.stride(0), h.data_ptr(), h.stride(0), wc.data_ptr(),
                                      rstd.data_ptr(), nv.ptr(dh2), dh2.stride(0) if dh2 is not None else 0,
                                      dx.data_ptr(), nv.ptr(part), nv.ptr(main), nv.ptr(dwn), R, D, w_offset,
                                      on.stream), "cvb_fp8_norm_bwd")
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
    if not (torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, resid, norm_w, w))):
        q, h = add_rmsnorm_fp8(x, resid, norm_w, eps, w_offset)
        y = _forward(None, q, w, weight, q.rows, w.shape[0], q.cols, False, False, x.dtype)[0]
        return (y if x.dim() == 2 else y.reshape(*x.shape[:-1], w.shape[0])), h
    out = _NormLinearFp8.apply(x, resid, norm_w, w, weight, eps, w_offset, grad_dtype)
    return (out, x) if resid is None else out
