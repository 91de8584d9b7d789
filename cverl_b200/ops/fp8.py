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

import functools
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


def _current_device() -> int:
    return torch._C._cuda_getDevice()


def _on_device(fn):
    """Runs ``fn`` with the device of its first argument as the current one: launches go to the tensors' device and to
    that device's current stream."""
    @functools.wraps(fn)
    def call(x, *args, **kwargs):
        t = x.buf if isinstance(x, Fp8Tensor) else x
        if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() != _current_device():
            with torch.cuda.device(t.device):
                return fn(x, *args, **kwargs)
        return fn(x, *args, **kwargs)
    return call


def _stream() -> int:
    return nv.raw_stream(_current_device())


def _status() -> int:
    index = _current_device()
    p = _status_ptr.get(index)
    if p is None:
        p = _status_ptr[index] = nv.status_word(index).data_ptr()      # one per device, never replaced
    return p


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
        self.buf, self.rows, self.cols, self.dtype = buf, rows, cols, dtype
        self.ld = (cols + 15) // 16 * 16

    @classmethod
    def empty(cls, rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> "Fp8Tensor":
        return cls(_bytes(_nbytes(rows, cols) + _nbytes_plain(rows, cols), device), rows, cols, dtype)

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.buf.device

    @property
    def sf_ptr(self) -> int:
        return self.buf.data_ptr() + self.rows * self.ld

    def _pointers(self):
        base = self.buf.data_ptr()
        return base, base + self.rows * self.ld, base + _nbytes(self.rows, self.cols), self.ld

    @property
    def values(self) -> torch.Tensor:
        """The codes as an 8-bit float view ``[rows, cols]`` (in units of their scales)."""
        return self.buf.view(self.dtype).as_strided((self.rows, self.cols), (self.ld, 1))

    def scales(self) -> torch.Tensor:
        """The scales as a view ``[rows, ceil(cols / 128)]`` of ``torch.float8_e8m0fnu`` (powers of two)."""
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
    out = Fp8Tensor.empty(R, C, dtype, x.device)
    out.buf.zero_()
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
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


def _check_dtype(dtype: torch.dtype, what: str) -> None:
    if dtype not in _FMT:
        raise TypeError(f"{what}: the 8-bit type is torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}")


def _quantize(x: torch.Tensor, dtype: torch.dtype, mode: int, rstd=None, w=None, w_offset: float = 0.0):
    """(row form or None, transposed form or None) by the mode's bits.  With ``rstd`` (on the CPU) the values are
    ``x * rstd[row] * (w_offset + w[col])``."""
    R, C = x.shape
    if not x.is_cuda:
        tall = BLOCK if mode & _TILES else 1
        x = x.detach()
        v = x.float() if rstd is None else x.float() * rstd[:, None] * (w_offset + w.float())
        return (_pack_ref(v, dtype, tall) if mode & _ROWS else None,
                _pack_ref(v.t(), dtype, tall) if mode & _COLS else None)
    q = t = None
    q_args = t_args = (None, None, None, 0)
    if mode & _ROWS:
        q = Fp8Tensor.empty(R, C, dtype, x.device)
        q_args = q._pointers()
    if mode & _COLS:
        t = Fp8Tensor.empty(C, R, dtype, x.device)
        t_args = t._pointers()
    if R and C:
        nv.check(nv.cuda().cvb_fp8_quantize(
            x.data_ptr(), x.dtype == torch.float32, R, C, x.stride(0), _FMT[dtype], mode, *q_args, *t_args, None, None,
            0.0, _stream()), "cvb_fp8_quantize")
        count_launch()
    return q, t


@_on_device
def quantize_fp8(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x [R, C]`` (bf16 or fp32) in 8 bits, one scale per 128 elements of a row."""
    _check_dtype(dtype, "quantize_fp8")
    return _quantize(_check_matrix(x, "quantize_fp8"), dtype, _ROWS)[0]


@_on_device
def quantize_fp8_t(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Fp8Tensor:
    """``x.T [C, R]`` in 8 bits, one scale per 128 rows of ``x``."""
    _check_dtype(dtype, "quantize_fp8_t")
    return _quantize(_check_matrix(x, "quantize_fp8_t"), dtype, _COLS)[1]


@_on_device
def quantize_fp8_pair(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, Fp8Tensor]:
    """``(quantize_fp8(x), quantize_fp8_t(x))`` from one read of ``x``."""
    _check_dtype(dtype, "quantize_fp8_pair")
    return _quantize(_check_matrix(x, "quantize_fp8_pair"), dtype, _ROWS | _COLS)


@_on_device
def quantize_fp8_weight(w: torch.Tensor, transposed: bool = True) -> Fp8Weight:
    """A weight ``[N, K]`` in e4m3 with one scale per 128 x 128 block.  ``transposed=False`` leaves the transpose out,
    which only gradients of the layer's input need."""
    q, t = _quantize(_check_matrix(w, "quantize_fp8_weight"), E4M3, _ROWS | _TILES | (_COLS if transposed else 0))
    return Fp8Weight(q, t)


# ----------------------------------------------------------------------------
# product
# ----------------------------------------------------------------------------
@_on_device
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
    nv.check(nv.cuda().cvb_fp8_gemm(
        a.buf.data_ptr(), a.sf_ptr, a.ld, _FMT[a.dtype], b.buf.data_ptr(), b.sf_ptr, b.ld, _FMT[b.dtype], M, N, K,
        out.data_ptr(), max(out.stride(0), N), 2 if accumulate else _OUT[out.dtype], _status(), _stream()),
        "cvb_fp8_gemm")
    count_launch()
    return out


# ----------------------------------------------------------------------------
# residual add + RMSNorm with 8-bit output
# ----------------------------------------------------------------------------
def _check_norm(x, resid, w, what):
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= MAX_NORM_WIDTH:
        raise ValueError(f"{what}: a last dimension of 1 to {MAX_NORM_WIDTH} is wanted, got shape {tuple(shape)}")
    if (x.is_cuda or w.is_cuda) and (x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16):
        raise TypeError(f"{what}: bfloat16 is wanted on the GPU, got {x.dtype} and a weight in {w.dtype}")
    if w.dim() != 1 or w.shape[0] != shape[-1] or w.device != x.device:
        raise ValueError(f"{what}: the weight is {tuple(w.shape)} on {w.device}, the rows have {shape[-1]} on {x.device}")
    if resid is not None and (resid.shape != shape or resid.dtype != x.dtype or resid.device != x.device):
        raise ValueError(f"{what}: resid is {tuple(resid.shape)} {resid.dtype} on {resid.device}, "
                         f"x is {tuple(shape)} {x.dtype} on {x.device}")


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _norm_forward(x2, r2, w, eps, w_offset, dtype, need_rstd: bool):
    """(8-bit rows, h or x2, rstd or None) of matrices."""
    R, D = x2.shape
    if not x2.is_cuda:
        x2, w = x2.detach(), w.detach()
        h = x2 if r2 is None else (x2.float() + r2.detach().float()).to(x2.dtype)
        rstd = torch.rsqrt(h.float().pow(2).mean(-1) + eps)
        return _pack_ref(h.float() * rstd[:, None] * (w_offset + w.float()), dtype), h, rstd
    q = Fp8Tensor.empty(R, D, dtype, x2.device)
    h = torch.empty((R, D), dtype=x2.dtype, device=x2.device) if r2 is not None else None
    rstd = torch.empty(R, dtype=torch.float32, device=x2.device) if need_rstd else None
    if R:
        if w.stride(0) != 1:
            w = w.contiguous()
        nv.check(nv.cuda().cvb_fp8_add_rmsnorm(
            x2.data_ptr(), x2.stride(0), nv.ptr(r2), r2.stride(0) if r2 is not None else 0, w.data_ptr(), nv.ptr(h),
            *q._pointers(), nv.ptr(rstd), R, D, _FMT[dtype], eps, w_offset, _stream()),
            "cvb_fp8_add_rmsnorm")
        count_launch()
    return q, (h if h is not None else x2), rstd


@_on_device
def add_rmsnorm_fp8(x: torch.Tensor, resid: Optional[torch.Tensor], w: torch.Tensor, eps: float = 1e-6,
                    w_offset: float = 1.0, dtype: torch.dtype = E4M3) -> Tuple[Fp8Tensor, torch.Tensor]:
    """``(Q(rmsnorm(x + resid)), x + resid)``; ``resid`` may be None.  The norm is rounded once, from fp32 to 8 bits;
    rows of the result are the rows of ``x`` flattened to a matrix.  It has no gradient and refuses inputs that ask for
    one: see ``add_rmsnorm_linear_fp8``."""
    _check_dtype(dtype, "add_rmsnorm_fp8")
    _check_norm(x, resid, w, "add_rmsnorm_fp8")
    if _needs_grad(x, resid, w):
        raise RuntimeError("add_rmsnorm_fp8 has no gradient: call it under torch.no_grad(), or add_rmsnorm_linear_fp8")
    q, h, _ = _norm_forward(_rows2d(x), _rows2d(resid) if resid is not None else None, w, eps, w_offset, dtype, False)
    if resid is None:
        return q, x
    return q, h if x.dim() == 2 else h.view(x.shape)


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


def _quantised_within(M: int, K: int) -> bool:
    """Whether the product quantises its bf16 rows itself (rows whose transpose nobody needs): every tile of 128 columns
    does it for its share of K, in series, so for few rows of moderate length.  Back to back, against two kernels: one row,
    K = 1024, N = 7168: 5.3 us against 6.6; 16 rows, K = 3584, N = 1024: 6.1 against 7.3; 32 rows, K = 2048: 7.2 against
    7.5; 64 rows: 10.6 against 8.2; 16 rows, K = N = 8192: 14.2 against 11.9.  And one launch less."""
    return M <= 16 and K <= 4096 or M <= 32 and K <= 2048


def _forward(x2, xq, w, weight: Optional[Fp8Weight], M, N, K, need_wt: bool, need_xt: bool, dtype):
    """``(y, xt, wt, wt_off)``: the product, and the transposed 8-bit forms that gradients read: ``xt`` at the start of
    its buffer, ``wt`` at ``wt_off`` bytes of its (buffers or None).  ``x2`` is the input's rows or None where ``xq`` is
    its 8-bit form; ``w`` the weight or None where ``weight`` is."""
    device = (x2 if x2 is not None else xq.buf).device
    y = _alloc_rows(M, N, dtype, device)
    if not y.is_cuda or not (M and N and K):
        xt = None
        if x2 is not None:
            xq, xt = _quantize(x2, E4M3, _ROWS | (_COLS if need_xt else 0))
        weight = weight or quantize_fp8_weight(w, transposed=need_wt)
        gemm_fp8_nt(xq, weight.w, y)
        return y, xt.buf if need_xt else None, weight.wt.buf if need_wt else None, 0
    # workspaces: 8-bit x and w for this product; 8-bit x^T and w^T kept for the gradients
    fused = xq is None and not need_xt and x2.dtype == torch.bfloat16 and _quantised_within(M, K)
    xq_n = 0 if xq is not None or fused else _nbytes(M, K)
    xt_n = _nbytes(K, M) if need_xt else 0
    wq_n = wt_n = x_stride = w_stride = 0
    x_fp32 = w_fp32 = False
    if weight is None:
        w = _check_matrix(w, "linear_fp8 weight")
        wq_n, wt_n = _nbytes(N, K), _nbytes(K, N) if need_wt else 0
        w_ptr, w_stride, w_fp32 = w.data_ptr(), w.stride(0), w.dtype == torch.float32
    else:
        w_ptr = None
    temp = _bytes(xq_n + wq_n, device) if xq_n + wq_n else None
    keep = _bytes(xt_n + wt_n, device) if xt_n + wt_n else None
    temp_ptr = temp.data_ptr() if temp is not None else 0
    keep_ptr = keep.data_ptr() if keep is not None else 0
    if x2 is not None:
        x_ptr, x_stride, x_fp32 = x2.data_ptr(), x2.stride(0), x2.dtype == torch.float32
    else:
        x_ptr = None
    nv.check(nv.cuda().cvb_fp8_linear_fwd(
        x_ptr, x_fp32, x_stride, w_ptr, w_fp32, w_stride, M, N, K,
        None if fused else temp_ptr if xq_n else xq.buf.data_ptr(),
        keep_ptr if xt_n else None, temp_ptr + xq_n if weight is None else weight.w.buf.data_ptr(),
        keep_ptr + xt_n if wt_n else None, y.data_ptr(), max(y.stride(0), N), _OUT[dtype], _status(), _stream()),
        "cvb_fp8_linear_fwd")
    count_launch(1 + (x_ptr is not None and not fused) + (w_ptr is not None))
    if need_wt and weight is not None:
        return y, keep, weight.wt.buf, 0
    return y, keep if need_xt else None, keep if need_wt else None, xt_n


def _backward(dy, M, N, K, grad_dtype, wt, wt_off, xt, w, dx_dtype, norm=None):
    """``(dx or None, dw or None)`` of ``y = x w^T``: dx where ``wt`` is given, dw where the parameter ``w`` is (added
    to its fp32 ``main_grad`` where it has one, and then None).  ``norm = (h, rstd, wn, w_offset)`` stands for ``xt`` on the CPU."""
    if dy.is_cuda and dy.get_device() != _current_device():
        with torch.cuda.device(dy.device):
            return _backward(dy, M, N, K, grad_dtype, wt, wt_off, xt, w, dx_dtype, norm)
    dy2 = _check_matrix(dy if dy.dim() == 2 else dy.reshape(-1, N) if dy.numel() else dy.reshape(0, N), "linear_fp8 gradient")
    dx = _alloc_rows(M, K, dx_dtype, dy.device) if wt is not None else None
    target, is_main = _grad_target(w, N, K, "linear_fp8") if w is not None else (None, False)
    if not (M and N and K):
        if dx is not None:
            dx.zero_()
        if target is not None and not is_main:
            target.zero_()
    elif not dy2.is_cuda:
        qdy, qdyt = _quantize(dy2, grad_dtype, (_ROWS if wt is not None else 0) | (_COLS if w is not None else 0))
        if dx is not None:
            gemm_fp8_nt(qdy, Fp8Tensor(wt, K, N, E4M3), dx)
        if target is not None:
            if norm is not None:
                xt = _quantize(norm[0], E4M3, _COLS, *norm[1:])[1].buf
            gemm_fp8_nt(qdyt, Fp8Tensor(xt, K, M, E4M3), target, accumulate=is_main)
    else:
        dyq_n = _nbytes(M, N) if wt is not None else 0
        dyt_n = _nbytes(N, M) if w is not None else 0
        temp = _bytes(dyq_n + dyt_n, dy.device)
        base = temp.data_ptr()
        dx_ptr = dw_ptr = wt_ptr = None
        dx_stride = dw_stride = dw_kind = 0
        if wt is not None:
            wt_ptr, dx_ptr, dx_stride = wt.data_ptr() + wt_off, dx.data_ptr(), max(dx.stride(0), K)
        if w is not None:
            dw_ptr, dw_stride, dw_kind = target.data_ptr(), max(target.stride(0), K), 2 if is_main else _OUT[w.dtype]
        nv.check(nv.cuda().cvb_fp8_linear_bwd(
            dy2.data_ptr(), dy2.dtype == torch.float32, dy2.stride(0), _FMT[grad_dtype], M, N, K, base, base + dyq_n,
            wt_ptr, nv.ptr(xt), None, 0, None, None, 0.0, dx_ptr, dx_stride, _OUT[dx_dtype], dw_ptr,
            dw_stride, dw_kind, _status(), _stream()), "cvb_fp8_linear_bwd")
        count_launch(1 + (wt is not None) + (w is not None))
    return dx, (None if is_main else target)


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, weight, grad_dtype):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        if need_dx and weight is not None and weight.wt is None:
            raise ValueError("linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        x2 = _rows2d(x)
        (M, K), N = x2.shape, w.shape[0]
        y, xt, wt, wt_off = _forward(x2, None, w, weight, M, N, K, need_dx, need_dw, x.dtype)
        # what the gradients read: x^T and w^T in 8 bits, half of what the bf16 layer keeps of x
        ctx.save_for_backward(w if need_dw else None, xt, wt)
        ctx.cfg = (x.shape, x.dtype, M, N, K, grad_dtype, wt_off)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, xt, wt = ctx.saved_tensors
        shape, xdtype, M, N, K, grad_dtype, wt_off = ctx.cfg
        dx, dw = _backward(dy, M, N, K, grad_dtype, wt, wt_off, xt, w, xdtype)
        if dx is not None and len(shape) != 2:
            dx = dx.reshape(shape)
        return dx, dw, None, None


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


@_on_device
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
        return _forward(None, x, w, kept, x.rows, w.shape[0], x.cols, False, False, torch.bfloat16)[0]
    shape = x.shape
    if not shape:
        raise ValueError(f"{what}: x has no dimensions")
    if x.dtype != torch.bfloat16 and (x.is_cuda or x.dtype != torch.float32):
        raise TypeError(f"{what}: bfloat16 is wanted, got {x.dtype}")
    K = shape[-1]
    _check_linear(x.numel() // K if K else 0, K, x.device, w, weight, grad_dtype, what)
    if not _needs_grad(x, w):
        x2 = _rows2d(x)
        N = w.shape[0]
        y = _forward(x2, None, w, kept, x2.shape[0], N, K, False, False, x.dtype)[0]
        return y if len(shape) == 2 else y.reshape(*shape[:-1], N)
    if kept is w:
        w = _Shape(w.shape)
    return _LinearFp8.apply(x, w, kept, grad_dtype)


def _norm_linear_forward(x2, r2, wn, w, weight, eps, w_offset, need_wt: bool, need_rstd: bool):
    """``(y, h, rstd, wt, wt_off)`` of matrices; ``h`` is ``x2`` without a residual, ``rstd`` None where not asked for."""
    (M, K), N = x2.shape, w.shape[0]
    if not x2.is_cuda or not (M and N and K):
        q, h, rstd = _norm_forward(x2, r2, wn, eps, w_offset, E4M3, need_rstd)
        y, _, wt, wt_off = _forward(None, q, w, weight, M, N, K, need_wt, False, x2.dtype)
        return y, h, rstd, wt, wt_off
    device = x2.device
    y = _alloc_rows(M, N, x2.dtype, device)
    h = torch.empty((M, K), dtype=x2.dtype, device=device) if r2 is not None else None
    if wn.stride(0) != 1:
        wn = wn.contiguous()
    rstd = torch.empty(M, dtype=torch.float32, device=device) if need_rstd else None
    xq_n = _nbytes(M, K)
    w_ptr = wt_ptr = keep = None
    wq_n = w_stride = 0
    w_fp32 = False
    if weight is None:
        w = _check_matrix(w, "linear_fp8 weight")
        w_ptr, w_stride, w_fp32, wq_n = w.data_ptr(), w.stride(0), w.dtype == torch.float32, _nbytes(N, K)
        if need_wt:
            keep = _bytes(_nbytes(K, N), device)
            wt_ptr = keep.data_ptr()
    temp = _bytes(xq_n + wq_n, device)
    temp_ptr = temp.data_ptr()
    nv.check(nv.cuda().cvb_fp8_norm_linear_fwd(
        x2.data_ptr(), x2.stride(0), nv.ptr(r2), r2.stride(0) if r2 is not None else 0, wn.data_ptr(), nv.ptr(h),
        nv.ptr(rstd), eps, w_offset, w_ptr, w_fp32, w_stride, M, N, K, temp_ptr,
        temp_ptr + xq_n if weight is None else weight.w.buf.data_ptr(), wt_ptr, y.data_ptr(), max(y.stride(0), N),
        _OUT[x2.dtype], _status(), _stream()), "cvb_fp8_norm_linear_fwd")
    count_launch(2 + (w_ptr is not None))
    if need_wt and weight is not None:
        keep = weight.wt.buf
    return y, (h if h is not None else x2), rstd, keep, 0


class _NormLinearFp8(torch.autograd.Function):
    """(linear(rmsnorm(x + resid)), x + resid) with the norm's result in 8 bits only."""

    @staticmethod
    def forward(ctx, x, resid, wn, w, weight, eps, w_offset, grad_dtype):
        need_dn, need_dw = any(ctx.needs_input_grad[:3]), ctx.needs_input_grad[3]
        if need_dn and weight is not None and weight.wt is None:
            raise ValueError("add_rmsnorm_linear_fp8: the gradient of the input needs the transposed 8-bit weight")
        y, h, rstd, wt, wt_off = _norm_linear_forward(
            _rows2d(x), _rows2d(resid) if resid is not None else None, wn, w, weight, eps, w_offset, need_dn, True)
        ctx.save_for_backward(h, rstd, wn, w if need_dw else None, wt)
        ctx.cfg = (x.shape, h.shape[0], w.shape[0], h.shape[1], w_offset, grad_dtype, wt_off)
        if x.dim() != 2:
            y, h = y.reshape(*x.shape[:-1], w.shape[0]), h.view(x.shape)
        return y if resid is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, rstd, wn, w, wt = ctx.saved_tensors
        shape, M, N, K, w_offset, grad_dtype, wt_off = ctx.cfg
        need_x, need_r, need_wn = ctx.needs_input_grad[:3]
        # The norm's result is formed again from h and rstd while its transpose is quantised: it is never stored.  Its
        # gradient stays fp32 between the product and the norm's backward.
        norm = (h, rstd, wn if wn.stride(0) == 1 else wn.contiguous(), w_offset)
        if dy.is_cuda and M and N and K:
            dx, dwn, dw = _norm_linear_backward(dy, dh, M, N, K, grad_dtype, wt, wt_off, w, norm, wn if need_wn else None)
        else:
            dn, dw = _backward(dy, M, N, K, grad_dtype, wt, wt_off, None, w, torch.float32, norm)
            dx, dwn = _norm_backward_ref(dn, h, wn, rstd, dh, w_offset, need_wn) if dn is not None else (None, None)
        if dx is not None and len(shape) != 2:
            dx = dx.view(shape)
        return (dx if need_x else None), (dx if need_r else None), dwn, dw, None, None, None, None


def _grad_target(w, rows: int, cols: int, what: str):
    """(where a weight's gradient goes, whether that is its main_grad)."""
    main = getattr(w, "main_grad", None)
    if main is None:
        return _alloc_rows(rows, cols, w.dtype, w.device), False
    if main.dtype != torch.float32 or not main.is_contiguous():
        raise TypeError(f"{what}: main_grad is a contiguous float32 tensor")
    return main.view(rows, cols), True


def _norm_linear_backward(dy, dh, M, N, K, grad_dtype, wt, wt_off, w, norm, wn_param):
    """``(dx, dwn, dw)``, each None where it is not wanted or went to a main_grad."""
    if dy.get_device() != _current_device():
        with torch.cuda.device(dy.device):
            return _norm_linear_backward(dy, dh, M, N, K, grad_dtype, wt, wt_off, w, norm, wn_param)
    h, rstd, wn, w_offset = norm
    device = dy.device
    dy2 = _check_matrix(dy if dy.dim() == 2 else dy.reshape(-1, N), "linear_fp8 gradient")
    dh2 = _rows2d(dh) if dh is not None and wt is not None else None
    lib = nv.cuda()
    # one workspace: dy in both forms, the norm's result transposed, its gradient, and the parts of dwn
    dyq_n = _nbytes(M, N) if wt is not None else 0
    dyt_n, xt_n = (_nbytes(N, M), _nbytes(K, M)) if w is not None else (0, 0)
    lddn = _ceil(K, 8) * 8
    dn_n = M * lddn * 4 if wt is not None else 0
    parts = min(M, lib.cvb_fp8_norm_bwd_parts()) if wn_param is not None else 0
    temp = _bytes(_ceil(dyq_n + dyt_n + xt_n, 32) * 32 + dn_n + parts * K * 4, device)
    base = temp.data_ptr()
    dn_at = base + _ceil(dyq_n + dyt_n + xt_n, 32) * 32
    wt_ptr = dx = dx_ptr = dw = dw_ptr = dwn = acc_ptr = dwn_ptr = part_ptr = None
    dw_stride = dw_kind = 0
    if wt is not None:
        wt_ptr = wt.data_ptr() + wt_off
        dx = torch.empty((M, K), dtype=h.dtype, device=device)
        dx_ptr = dx.data_ptr()
    if w is not None:
        target, is_main = _grad_target(w, N, K, "linear_fp8")
        dw_ptr, dw_stride, dw_kind = target.data_ptr(), max(target.stride(0), K), 2 if is_main else _OUT[w.dtype]
        dw = None if is_main else target
    if wn_param is not None:
        part_ptr = dn_at + dn_n
        if getattr(wn_param, "main_grad", None) is not None:
            acc_ptr = _grad_target(wn_param, 1, K, "add_rmsnorm_linear_fp8")[0].data_ptr()
        else:
            dwn = torch.empty(K, dtype=wn_param.dtype, device=device)
            dwn_ptr = dwn.data_ptr()
    nv.check(lib.cvb_fp8_norm_linear_bwd(
        dy2.data_ptr(), dy2.dtype == torch.float32, dy2.stride(0), _FMT[grad_dtype], M, N, K, base, base + dyq_n, wt_ptr,
        base + dyq_n + dyt_n, h.data_ptr(), h.stride(0), rstd.data_ptr(), wn.data_ptr(), w_offset, dn_at, lddn, dw_ptr,
        dw_stride, dw_kind, nv.ptr(dh2), dh2.stride(0) if dh2 is not None else 0, dx_ptr, part_ptr, acc_ptr, dwn_ptr,
        _status(), _stream()), "cvb_fp8_norm_linear_bwd")
    count_launch(1 + (2 if wt is not None else 0) + (2 if w is not None else 0) + (wn_param is not None))
    return dx, dwn, dw


def _norm_backward_ref(dn, h, wn, rstd, dh, w_offset, need_dwn):
    """``(dx, dwn)`` of the norm in PyTorch; without rows on any device."""
    D = h.shape[1]
    xh, d32 = h.float() * rstd[:, None], dn.float()
    g = d32 * (w_offset + wn.float())
    dx = rstd[:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + _rows2d(dh).float()
    dwn = None
    if need_dwn:
        dwn = (d32 * xh).sum(0)
        main = getattr(wn, "main_grad", None)
        if main is not None:
            main.view(D).add_(dwn)
            dwn = None
        else:
            dwn = dwn.to(wn.dtype)
    return dx.to(h.dtype), dwn


@_on_device
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
    if not _needs_grad(x, resid, norm_w, w):
        y, h, *_ = _norm_linear_forward(_rows2d(x), _rows2d(resid) if resid is not None else None, norm_w, w, kept, eps,
                                        w_offset, False, False)
        if x.dim() != 2:
            y, h = y.reshape(*x.shape[:-1], N), h.view(x.shape)
        return y, x if resid is None else h
    out = _NormLinearFp8.apply(x, resid, norm_w, _Shape(w.shape) if kept is w else w, kept, eps, w_offset, grad_dtype)
    return (out, x) if resid is None else out
