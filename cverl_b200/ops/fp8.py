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

with blocks of 128 along each product's own contraction.  CUDA tensors run the kernels, with workspaces and autograd
nodes in ``torch_ext/fp8_torch.cc``; CPU tensors run the PyTorch statement of the same math, which is also the test
oracle.  The reference has no 8-bit path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nv
from .gemm import count_launch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BLOCK = 128
MAX_NORM_WIDTH = 16384
MAX_EXTENT = 2 ** 31 - 1024                # rows or columns; sizes are 32-bit in the product
_FMT = {E4M3: 0, E5M2: 1}
_TOP = {E4M3: 8, E5M2: 15}                 # FMAX = 1.75 * 2^TOP
_ROWS, _COLS, _TILES = 1, 2, 4             # mode bits of cvb_fp8_quantize
_OUT = {torch.bfloat16: 0, torch.float32: 1}
_status_ptr: dict = {}


def _ceil(a: int, b: int) -> int:
    return (a + b - 1) // b


def _status(index: int) -> int:
    p = _status_ptr.get(index)
    if p is None:
        p = _status_ptr[index] = nv.status_word(index).data_ptr()      # one per device, never replaced
    return p


def _alloc_rows(M: int, N: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """``[M, N]`` whose rows start on 32 bytes (what the vector stores of the product want)."""
    per32 = 16 if dtype == torch.bfloat16 else 8
    if N % per32 == 0:
        return torch.empty((M, N), dtype=dtype, device=device)
    return torch.empty((M, _ceil(N, per32) * per32), dtype=dtype, device=device)[:, :N]


# ----------------------------------------------------------------------------
# the 8-bit matrix
# ----------------------------------------------------------------------------
def _nbytes(rows: int, cols: int) -> int:
    """Codes and scale cells: what the products read."""
    return rows * ((cols + 15) // 16 * 16) + ((rows + 127) // 128) * ((cols + 511) // 512) * 512


def _nbytes_plain(rows: int, cols: int) -> int:
    """The scale bytes once more, in plain order ``[rows, blocks]``: what a caller reads."""
    return rows * ((cols + 127) // 128)


class Fp8Tensor:
    """``[rows, cols]`` in 8 bits.  One buffer: codes, row-major with rows padded to 16 bytes; the scale bytes in the order
    in which the tensor core reads them (see ``cuda/fp8_common.cuh``); the scale bytes in plain order."""

    __slots__ = ("buf", "rows", "cols", "dtype", "ld")

    def __init__(self, buf: torch.Tensor, rows: int, cols: int, dtype: torch.dtype):
        if not (0 <= rows <= MAX_EXTENT and 0 <= cols <= MAX_EXTENT):
            raise ValueError(f"Fp8Tensor: at most {MAX_EXTENT} rows and columns, got [{rows}, {cols}]")
        if (buf.dtype != torch.uint8 or buf.dim() != 1 or buf.numel() != _nbytes(rows, cols) + _nbytes_plain(rows, cols)
                or not buf.is_contiguous() or buf.storage_offset() or dtype not in _FMT):
            raise ValueError(f"Fp8Tensor: not a buffer of a [{rows}, {cols}] matrix in {dtype}")
        self.buf, self.rows, self.cols, self.dtype = buf, rows, cols, dtype
        self.ld = (cols + 15) // 16 * 16

    @classmethod
    def _made(cls, buf: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> "Fp8Tensor":
        """Around a buffer that the extension has just made for these sizes: the checks take a tenth of a small call."""
        t = cls.__new__(cls)
        t.buf, t.rows, t.cols, t.dtype, t.ld = buf, rows, cols, dtype, (cols + 15) // 16 * 16
        return t

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
        if self.buf.is_cuda:
            return nv.torch_ext().view8(self.buf, self.rows, self.cols, _FMT[self.dtype])
        return self.buf.view(self.dtype).as_strided((self.rows, self.cols), (self.ld, 1))

    def scales(self) -> torch.Tensor:
        """The scales as a view ``[rows, ceil(cols / 128)]`` of ``torch.float8_e8m0fnu`` (powers of two)."""
        if self.buf.is_cuda:
            return nv.torch_ext().view8(self.buf, self.rows, self.cols, 2)
        nb = _ceil(self.cols, BLOCK)
        return self.buf.view(torch.float8_e8m0fnu).as_strided((self.rows, nb), (nb, 1), _nbytes(self.rows, self.cols))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        s = self.scales().float().repeat_interleave(BLOCK, 1)[:, :self.cols]
        return (self.values.float() * s).to(dtype)


class Fp8Weight:
    """A weight ``[N, K]`` in 8 bits (``w``) and, for gradients of the input, its transpose ``[K, N]`` (``wt``)."""

    __slots__ = ("w", "wt", "shape", "device")

    def __init__(self, w: Fp8Tensor, wt: Optional[Fp8Tensor] = None):
        if w.dtype != E4M3 or (wt is not None and (wt.dtype != E4M3 or wt.shape != w.shape[::-1] or wt.device != w.device)):
            raise ValueError("Fp8Weight: a weight and its transpose in torch.float8_e4m3fn on one device are wanted")
        self.w, self.wt = w, wt
        self.shape, self.device = w.shape, w.device


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
    out = Fp8Tensor(torch.zeros(_nbytes(R, C) + _nbytes_plain(R, C), dtype=torch.uint8, device=x.device), R, C, dtype)
    if R == 0 or C == 0:
        return out
    codes, byte = _quantize_ref(x, dtype, block_rows)
    out.buf[:R * out.ld].view(R, out.ld)[:, :C] = codes.contiguous().view(torch.uint8)
    rt, kg, at = _ceil(R, BLOCK), _ceil(C, 4 * BLOCK), _nbytes(R, C)
    cells = torch.ones((rt * BLOCK, kg * 4), dtype=torch.uint8, device=x.device)
    cells[:R, :byte.shape[1]] = byte
    out.buf[R * out.ld:at] = cells.view(rt, 4, 32, kg, 4).permute(0, 3, 2, 1, 4).reshape(-1)   # [.., r % 32, r / 32, b % 4]
    out.buf[at:] = byte.reshape(-1)
    return out


def _check_matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: a tensor is wanted, got {type(x).__name__}")
    if x.dim() != 2:
        raise ValueError(f"{what}: a matrix is wanted, got shape {tuple(x.shape)}")
    if x.dtype not in _OUT:
        raise TypeError(f"{what}: bfloat16 or float32 is wanted, got {x.dtype}")
    if x.shape[0] > MAX_EXTENT or x.shape[1] > MAX_EXTENT:
        raise ValueError(f"{what}: at most {MAX_EXTENT} rows and columns, got {tuple(x.shape)}")
    return x


def _check_dtype(dtype: torch.dtype, what: str) -> None:
    if dtype not in _FMT:
        raise TypeError(f"{what}: the 8-bit type is torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}")


def _quantize(x: torch.Tensor, dtype: torch.dtype, mode: int):
    """(row form or None, transposed form or None) by the mode's bits."""
    R, C = x.shape
    if x.is_cuda:
        q, t = nv.torch_ext().quantize(x, _FMT[dtype], mode)
        return (Fp8Tensor._made(q, R, C, dtype) if q is not None else None,
                Fp8Tensor._made(t, C, R, dtype) if t is not None else None)
    tall = BLOCK if mode & _TILES else 1
    v = x.detach().float()
    return (_pack_ref(v, dtype, tall) if mode & _ROWS else None), (_pack_ref(v.t(), dtype, tall) if mode & _COLS else None)


def _check_activations(x: torch.Tensor, dtype: torch.dtype, what: str) -> torch.Tensor:
    _check_dtype(dtype, what)
    _check_matrix(x, what)
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or linear_fp8 on the tensor itself")
    return x


def quantize_fp8(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x [R, C]`` (bf16 or fp32) in 8 bits, one scale per 128 elements of a row.  This, the transpose and the pair have
    no gradient and refuse an input that asks for one: ``linear_fp8`` rounds and differentiates."""
    return _quantize(_check_activations(x, dtype, "quantize_fp8"), dtype, _ROWS)[0]


def quantize_fp8_t(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x.T [C, R]`` in 8 bits, one scale per 128 rows of ``x``."""
    return _quantize(_check_activations(x, dtype, "quantize_fp8_t"), dtype, _COLS)[1]


def quantize_fp8_pair(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, Fp8Tensor]:
    """``(quantize_fp8(x), quantize_fp8_t(x))`` from one read of ``x``."""
    return _quantize(_check_activations(x, dtype, "quantize_fp8_pair"), dtype, _ROWS | _COLS)


def quantize_fp8_weight(w: torch.Tensor, transposed: bool = True) -> Fp8Weight:
    """A weight ``[N, K]`` in e4m3 with one scale per 128 x 128 block.  ``transposed=False`` leaves the transpose out,
    which only gradients of the layer's input need.  A copy without history, of a parameter too: ``linear_fp8`` takes
    both where the parameter trains."""
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
        if out.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("gemm_fp8_nt has no gradient: call it under torch.no_grad() for an out that asks for one")
        if (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"gemm_fp8_nt: out has strides {out.stride()}: rows of unit stride that do not overlap are wanted")
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out if accumulate else out.zero_()
    if not a.buf.is_cuda:
        r = a.dequantize() @ b.dequantize().t()
        return out.add_(r) if accumulate else out.copy_(r)
    index = out.get_device()
    args = (a.buf.data_ptr(), a.sf_ptr, a.ld, _FMT[a.dtype], b.buf.data_ptr(), b.sf_ptr, b.ld, _FMT[b.dtype], M, N, K,
            out.data_ptr(), max(out.stride(0), N), 2 if accumulate else _OUT[out.dtype], 0, _status(index))
    if index != torch._C._cuda_getDevice():       # launches go to the operands' device and its current stream
        with torch.cuda.device(index):
            nv.check(nv.cuda().cvb_fp8_gemm(*args, nv.raw_stream(index)), "cvb_fp8_gemm")
    else:
        nv.check(nv.cuda().cvb_fp8_gemm(*args, nv.raw_stream(index)), "cvb_fp8_gemm")
    count_launch()
    return out


# ----------------------------------------------------------------------------
# residual add + RMSNorm with 8-bit output
# ----------------------------------------------------------------------------
def _check_norm(x, resid, w, what):
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= MAX_NORM_WIDTH:
        raise ValueError(f"{what}: a last dimension of 1 to {MAX_NORM_WIDTH} is wanted, got shape {tuple(shape)}")
    if x.numel() // shape[-1] > MAX_EXTENT:
        raise ValueError(f"{what}: at most {MAX_EXTENT} rows, got shape {tuple(shape)}")
    if (x.is_cuda or w.is_cuda) and (x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16):
        raise TypeError(f"{what}: bfloat16 is wanted on the GPU, got {x.dtype} and a weight in {w.dtype}")
    if w.dim() != 1 or w.shape[0] != shape[-1] or w.device != x.device:
        raise ValueError(f"{what}: the weight is {tuple(w.shape)} on {w.device}, the rows have {shape[-1]} on {x.device}")
    if resid is not None and (resid.shape != shape or resid.dtype != x.dtype or resid.device != x.device):
        raise ValueError(f"{what}: resid is {tuple(resid.shape)} {resid.dtype} on {resid.device}, "
                         f"x is {tuple(shape)} {x.dtype} on {x.device}")


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 2 else t.reshape(t.shape[:-1].numel(), t.shape[-1])


def _norm_ref(x2, r2, w, eps, w_offset):
    """(fp32 norm, h, rstd) of matrices in PyTorch."""
    h = x2 if r2 is None else (x2.float() + r2.float()).to(x2.dtype)
    rstd = torch.rsqrt(h.float().pow(2).mean(-1) + eps)
    return h.float() * rstd[:, None] * (w_offset + w.float()), h, rstd


def add_rmsnorm_fp8(x: torch.Tensor, resid: Optional[torch.Tensor], w: torch.Tensor, eps: float = 1e-6,
                    w_offset: float = 1.0, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, torch.Tensor]:
    """``(Q(rmsnorm(x + resid)), x + resid)``; ``resid`` may be None.  The norm is rounded once, from fp32 to 8 bits;
    rows of the result are the rows of ``x`` flattened to a matrix.  It has no gradient and refuses inputs that ask for
    one: see ``add_rmsnorm_linear_fp8``."""
    _check_dtype(dtype, "add_rmsnorm_fp8")
    _check_norm(x, resid, w, "add_rmsnorm_fp8")
    if _needs_grad(x, resid, w):
        raise RuntimeError("add_rmsnorm_fp8 has no gradient: call it under torch.no_grad(), or add_rmsnorm_linear_fp8")
    D = x.shape[-1]
    if x.is_cuda:
        q, h = nv.torch_ext().norm(x, resid, w, eps, w_offset, _FMT[dtype])
        return Fp8Tensor._made(q, x.numel() // D, D, dtype), (x if h is None else h)
    with torch.no_grad():
        y, h, _ = _norm_ref(_rows2d(x), _rows2d(resid) if resid is not None else None, w, eps, w_offset)
        return _pack_ref(y, dtype), (x if resid is None else h.view(x.shape))


# ----------------------------------------------------------------------------
# linear layers
# ----------------------------------------------------------------------------
def _check_linear(rows: int, K: int, device, w, weight: Optional[Fp8Weight], grad_dtype, what: str) -> None:
    if grad_dtype not in _FMT:
        _check_dtype(grad_dtype, what)
    shape = w.shape
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f"{what}: a weight [N, {K}] is wanted, got {tuple(shape)}")
    if w.device != device:
        raise ValueError(f"{what}: the weight is on {w.device}, the input on {device}")
    if shape[0] > MAX_EXTENT or K > MAX_EXTENT or rows > MAX_EXTENT:
        raise ValueError(f"{what}: at most {MAX_EXTENT} rows and columns")
    if not isinstance(w, Fp8Weight):
        if w.dtype not in _OUT:
            raise TypeError(f"{what}: the weight is bfloat16 or float32, not {w.dtype}")
        if weight is not None and (weight.shape != tuple(shape) or weight.device != device):
            raise ValueError(f"{what}: the 8-bit weight is {weight.shape} on {weight.device}, the weight {tuple(shape)} on {device}")
    elif weight is not None:
        raise ValueError(f"{what}: the 8-bit weight is given twice")


# The PyTorch statement of the layers: the CPU path, and the oracle of the tests.  (CUDA: torch_ext/fp8_torch.cc.)
def _gradients_ref(dy2, xt, wt, w, grad_dtype, dx_dtype):
    """(dx or None, dw or None) from the transposed 8-bit forms; dw goes to the parameter's main_grad where it has one."""
    dx = dw = None
    if wt is not None:
        dx = gemm_fp8_nt(_pack_ref(dy2, grad_dtype), wt, out_dtype=dx_dtype)
    if w is not None:
        main = getattr(w, "main_grad", None)
        if main is None:
            dw = gemm_fp8_nt(_pack_ref(dy2.t(), grad_dtype), xt, out_dtype=w.dtype)
        elif main.dtype != torch.float32 or not main.is_contiguous() or main.numel() != w.numel():
            raise TypeError("main_grad is a contiguous float32 tensor of the parameter's size")
        else:
            gemm_fp8_nt(_pack_ref(dy2.t(), grad_dtype), xt, main.view(w.shape), accumulate=True)
    return dx, dw


class _LinearRef(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, weight, grad_dtype):
        x2 = _rows2d(x)
        weight = weight or quantize_fp8_weight(w)
        need_dx, need_dw = ctx.needs_input_grad[:2]
        if need_dx and weight.wt is None:
            raise ValueError("linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        ctx.forms = (_pack_ref(x2.t(), E4M3) if need_dw else None, weight.wt if need_dx else None)
        ctx.save_for_backward(w if need_dw else None)
        ctx.cfg = (x.shape, x.dtype, grad_dtype)
        return gemm_fp8_nt(_pack_ref(x2, E4M3), weight.w, out_dtype=x.dtype).reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        shape, dtype, grad_dtype = ctx.cfg
        dx, dw = _gradients_ref(_rows2d(dy), *ctx.forms, ctx.saved_tensors[0], grad_dtype, dtype)
        return (dx.reshape(shape) if dx is not None else None), dw, None, None


class _NormLinearRef(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, resid, wn, w, weight, eps, w_offset, grad_dtype):
        weight = weight or quantize_fp8_weight(w)
        need_dn, need_dw = any(ctx.needs_input_grad[:3]), ctx.needs_input_grad[3]
        if need_dn and weight.wt is None:
            raise ValueError("add_rmsnorm_linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        n, h, rstd = _norm_ref(_rows2d(x), _rows2d(resid) if resid is not None else None, wn, eps, w_offset)
        ctx.forms = (_pack_ref(n.t(), E4M3) if need_dw else None, weight.wt if need_dn else None)
        ctx.save_for_backward(h, rstd, wn, w if need_dw else None)
        ctx.cfg = (x.shape, w_offset, grad_dtype)
        y = gemm_fp8_nt(_pack_ref(n, E4M3), weight.w, out_dtype=x.dtype).reshape(*x.shape[:-1], w.shape[0])
        return y if resid is None else (y, h.view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, rstd, wn, w = ctx.saved_tensors
        shape, w_offset, grad_dtype = ctx.cfg
        dn, dw = _gradients_ref(_rows2d(dy), *ctx.forms, w, grad_dtype, torch.float32)
        dx = dwn = None
        if dn is not None:
            xh, g = h.float() * rstd[:, None], dn * (w_offset + wn.float())
            dx = rstd[:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
            if dh is not None:
                dx = dx + _rows2d(dh).float()
            dx = dx.to(h.dtype).view(shape)
            if ctx.needs_input_grad[2]:
                dwn = (dn * xh).sum(0)
                main = getattr(wn, "main_grad", None)
                if main is not None:
                    main.view(-1).add_(dwn)
                    dwn = None
                else:
                    dwn = dwn.to(wn.dtype)
        need_x, need_r = ctx.needs_input_grad[:2]
        return (dx if need_x else None), (dx if need_r else None), dwn, dw, None, None, None, None


def _parts(w, kept):
    """What the extension takes for a weight: (parameter, 8-bit weight, its transpose), each None where there is none."""
    if kept is None:
        return w, None, None
    return (None if kept is w else w), kept.w.buf, (kept.wt.buf if kept.wt is not None else None)


class _Shape:
    """Stands for a frozen weight in the autograd functions: only its shape is asked for."""

    def __init__(self, shape):
        self.shape = shape


def _needs_grad(*tensors) -> bool:
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            return True
    return False


def linear_fp8(x, w, *, weight: Optional[Fp8Weight] = None, grad_dtype: torch.dtype = E4M3) -> torch.Tensor:
    """``x [..., K] @ w [N, K].T`` with both operands rounded to 8 bits.

    ``w`` is a parameter (its 8-bit form is made in the call, or taken from ``weight`` where the caller keeps one for
    several micro-batches), or an ``Fp8Weight`` for serving and for frozen weights.  ``x`` is a tensor or, without
    gradients, an ``Fp8Tensor`` (from ``add_rmsnorm_fp8``) with a matrix as the result.  Gradients of ``y`` are rounded
    to ``grad_dtype``; the weight's gradient goes to ``w.main_grad`` when the parameter has one."""
    what = "linear_fp8"
    kept = w if isinstance(w, Fp8Weight) else weight
    if isinstance(x, Fp8Tensor):
        _check_linear(x.rows, x.cols, x.device, w, weight, grad_dtype, what)
        if x.dtype != E4M3:
            raise TypeError(f"{what}: inputs are torch.float8_e4m3fn, got {x.dtype}")
        if _needs_grad(w):
            raise RuntimeError(f"{what}: an 8-bit input carries no gradient: call it under torch.no_grad()")
        if not x.buf.is_cuda:
            return gemm_fp8_nt(x, (kept or quantize_fp8_weight(w, transposed=False)).w)
        p, wq, _ = _parts(w, kept)
        return nv.torch_ext().linear_rows8(x.buf, x.rows, x.cols, p, wq, w.shape[0], _status(x.buf.get_device()))
    shape = x.shape
    if not shape:
        raise ValueError(f"{what}: x has no dimensions")
    if x.dtype != torch.bfloat16 and (x.is_cuda or x.dtype != torch.float32):
        raise TypeError(f"{what}: bfloat16 is wanted, got {x.dtype}")
    K = shape[-1]
    _check_linear(x.numel() // K if K else 0, K, x.device, w, weight, grad_dtype, what)
    if x.is_cuda:
        return nv.torch_ext().linear(x, *_parts(w, kept), w.shape[0], _FMT[grad_dtype], _status(x.get_device()))
    return _LinearRef.apply(x, _Shape(w.shape) if kept is w else w, kept, grad_dtype)


def add_rmsnorm_linear_fp8(x: torch.Tensor, resid: Optional[torch.Tensor], norm_w: torch.Tensor, w, eps: float = 1e-6,
                           w_offset: float = 1.0, *, weight: Optional[Fp8Weight] = None,
                           grad_dtype: torch.dtype = E4M3) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(rmsnorm(x + resid) @ w.T, x + resid)``; ``resid`` may be None.  The norm's result exists in 8 bits only: the
    backward pass forms it again from ``x + resid``.  ``w``, ``weight`` and ``grad_dtype`` as in ``linear_fp8``."""
    what = "add_rmsnorm_linear_fp8"
    _check_norm(x, resid, norm_w, what)
    K, N = x.shape[-1], w.shape[0] if len(w.shape) else 0
    _check_linear(x.numel() // K, K, x.device, w, weight, grad_dtype, what)
    kept = w if isinstance(w, Fp8Weight) else weight
    if x.is_cuda:
        out = nv.torch_ext().norm_linear(x, resid, norm_w, *_parts(w, kept), N, eps, w_offset, _FMT[grad_dtype],
                                         _status(x.get_device()))
        return out[0], (x if resid is None else out[1])
    out = _NormLinearRef.apply(x, resid, norm_w, _Shape(w.shape) if kept is w else w, kept, eps, w_offset, grad_dtype)
    return (out, x) if resid is None else out
