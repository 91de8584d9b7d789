"""8-bit operators on the CPU path: format, gradients, refusals."""
import pytest
import torch

import fp8_oracle as orc
from cverl_b200 import ops
from cverl_b200.ops import fp8
from fp8_oracle import E4M3, E5M2


def _rand(*shape, seed=0, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _same(got, want):
    return torch.equal(torch.nan_to_num(got.double(), nan=1e300), torch.nan_to_num(want, nan=1e300))


def awkward(R, C, dtype):
    """Rows that are zero, subnormal, huge, at the borders of a scale, infinite or NaN."""
    x = _rand(R, C, seed=R * 1000 + C) * torch.exp2(torch.arange(R).float() % 40 - 20)[:, None]
    rows = [torch.zeros(C), torch.full((C,), 2.0 ** -130), torch.full((C,), 3e38), torch.full((C,), 448.0 * 2 ** -9),
            torch.full((C,), 450.0), torch.full((C,), -1.0)]
    rows[5][::3] = float("inf")
    rows[5][1::5] = float("nan")
    rows[5][2::7] = float("-inf")
    for i, row in enumerate(rows[:R]):
        x[R - 1 - i] = row
    return x.to(dtype)


@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (6, 129), (130, 300), (257, 640)])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_codes_and_scales_are_the_definition(shape, dtype, src):
    x = awkward(*shape, src)
    q, t = ops.quantize_fp8_pair(x, dtype)
    for got, want in ((q, orc.quantize(x, dtype)), (t, orc.quantize(x.t(), dtype))):
        assert _same(got.values, want[0])
        assert torch.equal(got.scales().double(), want[1][:, ::128])
    assert _same(ops.quantize_fp8(x, dtype).values, orc.quantize(x, dtype)[0])
    assert _same(ops.quantize_fp8_t(x, dtype).values, orc.quantize(x.t(), dtype)[0])


def test_weight_and_its_transpose_hold_the_same_values():
    w = _rand(200, 300, seed=3)
    q = ops.quantize_fp8_weight(w)
    assert torch.equal(q.w.dequantize(), q.wt.dequantize().t())
    assert torch.equal(orc.value(q.w), orc.through(w, tall=128))
    assert ops.quantize_fp8_weight(w, transposed=False).wt is None


def test_product_and_accumulation():
    a, b = ops.quantize_fp8(_rand(5, 200)), ops.quantize_fp8(_rand(7, 200, seed=1), E5M2)
    want = orc.value(a) @ orc.value(b).t()
    # 200 products, each sum in fp32: at most 200 half steps of a sum of magnitudes
    tol = 200 * 2.0 ** -24 * (orc.value(a).abs() @ orc.value(b).abs().t())
    got = ops.gemm_fp8_nt(a, b, out_dtype=torch.float32)
    assert ((got - want).abs() <= tol).all()
    out = torch.ones(5, 7)
    ops.gemm_fp8_nt(a, b, out, accumulate=True)
    assert ((out - 1 - want).abs() <= tol + 2.0 ** -23 * (1 + want.abs())).all()


@pytest.mark.parametrize("grad", [E4M3, E5M2])
def test_linear_gradients_are_the_formula(grad):
    x, w = _rand(3, 50, 140, seed=1).requires_grad_(), _rand(130, 140, seed=2).requires_grad_()
    dy = _rand(3, 50, 130, seed=3, std=1e-3)
    y = ops.linear_fp8(x, w, grad_dtype=grad)
    y.backward(dy)
    x2, dy2 = x.detach().view(150, 140), dy.view(150, 130)
    qw = orc.through(w.detach(), tall=128)
    for got, want in ((y.detach().view(150, 130), orc.through(x2) @ qw.t()),
                      (x.grad.view(150, 140), orc.through(dy2, grad) @ qw),
                      (w.grad, orc.through(dy2.t(), grad) @ orc.through(x2.t()).t())):
        # fp32 sums of at most 150 terms, random signs: 150 half steps of 2^-24 of the norm at the very most
        assert (got - want).norm() <= 150 * 2.0 ** -24 * want.norm()


def test_gradients_agree_with_differences_of_the_smooth_layer():
    """Every rounding is at most 2^-4 of its value, three a product, independent over 96 or more terms: the gradient of
    the rounded layer lies within 3 * 2^-4 of the smooth layer's, whose gradient is taken by central differences."""
    x, r = _rand(40, 96, seed=1), _rand(40, 96, seed=2)
    wn, w = _rand(96, seed=3, std=0.1), _rand(100, 96, seed=4, std=0.1)
    dy, dh = _rand(40, 100, seed=5), _rand(40, 96, seed=6)
    leaves = [t.clone().requires_grad_() for t in (x, r, wn, w)]
    y, h = ops.add_rmsnorm_linear_fp8(*leaves, 1e-6, 1.0)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def loss(x, r, wn, w):
        n, h, _ = orc.norm(x.double(), r.double(), wn, 1e-6, 1.0)
        return ((n @ w.double().t()) * dy.double()).sum() + (h * dh.double()).sum()

    for i, g in enumerate(grads):
        d = _rand(*g.shape, seed=10 + i).double()
        d = 1e-5 * (d + g.double() / g.double().norm() * d.norm())      # not orthogonal to the gradient
        args = [t.double() for t in (x, r, wn, w)]
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + d, args[i] - d
        want = (loss(*hi) - loss(*lo)) / 2
        got = (g.double() * d).sum()
        assert abs(got - want) <= 3 * 2.0 ** -4 * abs(want)


def test_norm_then_linear_is_the_joint_layer():
    x, r = _rand(33, 200, seed=1), _rand(33, 200, seed=2)
    wn, w = _rand(200, seed=3, std=0.1), _rand(70, 200, seed=4)
    q, h = ops.add_rmsnorm_fp8(x, r, wn)
    kept = ops.quantize_fp8_weight(w)
    y = ops.linear_fp8(q, kept)
    y2, h2 = ops.add_rmsnorm_linear_fp8(x, r, wn, w)
    assert torch.equal(h, h2) and torch.equal(y.float(), y2.to(y.dtype).float())
    y3, h3 = ops.add_rmsnorm_linear_fp8(x, None, wn, kept)
    assert h3 is x and y3.shape == (33, 70)


def test_main_grad_takes_the_weight_gradients():
    x, w, wn = _rand(20, 130, seed=1), _rand(40, 130, seed=2), _rand(130, seed=3)
    plain = [t.clone().requires_grad_() for t in (wn, w)]
    y, _ = ops.add_rmsnorm_linear_fp8(x, None, *plain)
    want = torch.autograd.grad(y.sum(), plain)
    kept = [t.clone().requires_grad_() for t in (wn, w)]
    for p in kept:
        p.main_grad = torch.ones_like(p)
    y, _ = ops.add_rmsnorm_linear_fp8(x, None, *kept)
    y.sum().backward()
    for p, g in zip(kept, want):
        assert p.grad is None
        assert torch.allclose(p.main_grad - 1, g, rtol=1e-5, atol=1e-5)


def test_frozen_weights_pass_gradients_of_the_input():
    x, w = _rand(9, 150, seed=1).requires_grad_(), _rand(30, 150, seed=2)
    kept = ops.quantize_fp8_weight(w)
    y = ops.linear_fp8(x, kept)
    y.sum().backward()
    want = orc.through(torch.ones(9, 30)) @ orc.through(w, tall=128)
    assert (x.grad - want).norm() <= 30 * 2.0 ** -24 * want.norm()
    with pytest.raises(ValueError, match="transposed"):
        ops.linear_fp8(x, ops.quantize_fp8_weight(w, transposed=False))


@pytest.mark.parametrize("m,n,k", [(0, 5, 7), (5, 0, 7), (5, 7, 0)])
def test_empty_matrices(m, n, k):
    a, b = ops.quantize_fp8(torch.ones(m, k)), ops.quantize_fp8(torch.ones(n, k))
    y = ops.gemm_fp8_nt(a, b, out_dtype=torch.float32)
    assert y.shape == (m, n) and not y.any()
    assert a.values.shape == (m, k) and a.scales().shape == (m, (k + 127) // 128)


def test_no_tokens_give_zero_gradients():
    x, w = torch.zeros(0, 64, requires_grad=True), torch.randn(32, 64, requires_grad=True)
    y = ops.linear_fp8(x, w)
    y.sum().backward()
    assert y.shape == (0, 32) and x.grad.shape == (0, 64) and w.grad.shape == (32, 64) and not w.grad.any()


def test_what_has_no_gradient_says_so():
    x, w, wn = torch.ones(4, 8, requires_grad=True), torch.ones(3, 8, requires_grad=True), torch.ones(8)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.add_rmsnorm_fp8(x, None, wn)
    with torch.no_grad():
        q, _ = ops.add_rmsnorm_fp8(x, None, wn)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.linear_fp8(q, w)
    assert not ops.linear_fp8(q, ops.quantize_fp8_weight(w)).requires_grad
    g, = torch.autograd.grad(ops.linear_fp8(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        g.sum().backward()


def test_refusals():
    a, b = ops.quantize_fp8(torch.ones(4, 8)), ops.quantize_fp8(torch.ones(3, 9))
    good = ops.quantize_fp8(torch.ones(3, 8))
    bad = [
        (TypeError, lambda: ops.quantize_fp8(torch.ones(2, 2), torch.float16)),
        (TypeError, lambda: ops.quantize_fp8(torch.ones(2, 2, dtype=torch.float16))),
        (TypeError, lambda: ops.quantize_fp8(torch.ones(2, 2, dtype=torch.int32))),
        (TypeError, lambda: ops.quantize_fp8([1.0])),
        (ValueError, lambda: ops.quantize_fp8(torch.ones(2))),
        (ValueError, lambda: ops.quantize_fp8_weight(torch.ones(2, 2, 2))),
        (TypeError, lambda: ops.gemm_fp8_nt(torch.ones(4, 8), good)),
        (ValueError, lambda: ops.gemm_fp8_nt(a, b)),
        (TypeError, lambda: ops.gemm_fp8_nt(a, good, out_dtype=torch.float16)),
        (ValueError, lambda: ops.gemm_fp8_nt(a, good, accumulate=True)),
        (TypeError, lambda: ops.gemm_fp8_nt(a, good, torch.ones(4, 3, dtype=torch.bfloat16), accumulate=True)),
        (ValueError, lambda: ops.gemm_fp8_nt(a, good, torch.ones(3, 4))),
        (ValueError, lambda: ops.gemm_fp8_nt(a, good, torch.ones(3, 4).t())),
        (ValueError, lambda: ops.gemm_fp8_nt(a, good, torch.ones(1, 3).expand(4, 3))),
        (ValueError, lambda: ops.add_rmsnorm_fp8(torch.ones(2, 8), None, torch.ones(9))),
        (ValueError, lambda: ops.add_rmsnorm_fp8(torch.ones(2, 8), torch.ones(3, 8), torch.ones(8))),
        (ValueError, lambda: ops.add_rmsnorm_fp8(torch.ones(2, 16385), None, torch.ones(16385))),
        (ValueError, lambda: ops.linear_fp8(torch.ones(2, 8), torch.ones(4, 9))),
        (TypeError, lambda: ops.linear_fp8(torch.ones(2, 8), torch.ones(4, 8), grad_dtype=torch.bfloat16)),
        (TypeError, lambda: ops.linear_fp8(torch.ones(2, 8).half(), torch.ones(4, 8))),
        (TypeError, lambda: ops.linear_fp8(torch.ones(2, 8), torch.ones(4, 8).half())),
        (ValueError, lambda: ops.linear_fp8(torch.ones(2, 8), torch.ones(4, 8), weight=ops.quantize_fp8_weight(torch.ones(5, 8)))),
        (ValueError, lambda: ops.Fp8Tensor(torch.zeros(8, dtype=torch.uint8), 4, 8, E4M3)),
        (ValueError, lambda: ops.Fp8Tensor(good.buf, 3, 17, E4M3)),
        (ValueError, lambda: ops.Fp8Weight(ops.quantize_fp8(torch.ones(4, 8), E5M2))),
        (ValueError, lambda: ops.Fp8Weight(good, a)),
        (TypeError, lambda: ops.linear_fp8(ops.quantize_fp8(torch.ones(2, 8), E5M2), ops.quantize_fp8_weight(torch.ones(4, 8)))),
        (ValueError, lambda: ops.quantize_fp8(torch.ones(1).expand(2 ** 31, 1))),
        (ValueError, lambda: ops.linear_fp8(torch.ones(1).expand(2 ** 31, 1), torch.ones(4, 1))),
        (ValueError, lambda: ops.linear_fp8(torch.ones(2, 8), ops.quantize_fp8_weight(torch.ones(4, 8)),
                                            weight=ops.quantize_fp8_weight(torch.ones(4, 8)))),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()


def test_a_buffer_that_is_not_one_run_of_bytes_is_refused():
    """The kernels read a buffer from its first byte on, whatever its strides say."""
    q = ops.quantize_fp8(torch.ones(3, 8))
    n = q.buf.numel()
    for buf in (torch.zeros(1, dtype=torch.uint8).expand(n), torch.zeros(2 * n, dtype=torch.uint8)[::2],
                torch.zeros(n + 16, dtype=torch.uint8)[16:], q.buf.view(1, n), q.buf.view(torch.int8)):
        with pytest.raises(ValueError, match="not a buffer"):
            ops.Fp8Tensor(buf, 3, 8, E4M3)
    assert torch.equal(ops.Fp8Tensor(q.buf.clone(), 3, 8, E4M3).dequantize(), torch.ones(3, 8))


@pytest.mark.parametrize("rows", [2 ** 31 - 1023, 2 ** 31, -1])
def test_sizes_beyond_32_bits_are_refused_wherever_a_matrix_is_made(rows):
    n = max(rows, 0)
    with pytest.raises(ValueError):
        ops.Fp8Tensor(torch.empty(n * 16 + -(-n // 128) * 512 + n, dtype=torch.uint8, device="meta"), rows, 1, E4M3)
    with pytest.raises(ValueError):
        ops.Fp8Tensor(torch.empty(0, dtype=torch.uint8, device="meta"), 0, rows, E4M3)
    if rows > 0:
        x = torch.empty((1, 1), device="meta").expand(rows, 1)
        with pytest.raises(ValueError, match="rows"):
            ops.add_rmsnorm_fp8(x, None, torch.empty(1, device="meta"))


@pytest.mark.parametrize("quantize", [ops.quantize_fp8, ops.quantize_fp8_t, ops.quantize_fp8_pair])
def test_quantising_what_asks_for_a_gradient_is_refused(quantize):
    """The 8-bit form has no history: a product of it would drop the gradient without a word."""
    x, w = torch.ones(4, 8, requires_grad=True), torch.ones(3, 8, requires_grad=True)
    for t in (x, x * 2):
        with pytest.raises(RuntimeError, match="no gradient"):
            quantize(t)
        with torch.no_grad():
            quantize(t)
        quantize(t.detach())
    assert not ops.linear_fp8(ops.quantize_fp8(x.detach()), ops.quantize_fp8_weight(w)).requires_grad    # kept weights are copies


def test_a_product_into_what_asks_for_a_gradient_is_refused():
    a, b = ops.quantize_fp8(torch.ones(4, 8)), ops.quantize_fp8(torch.ones(3, 8))
    leaf = torch.zeros(4, 3, requires_grad=True)
    for out in (leaf, leaf * 1):
        for acc in (False, True):
            with pytest.raises(RuntimeError, match="no gradient"):
                ops.gemm_fp8_nt(a, b, out, accumulate=acc)
    with torch.no_grad():
        assert (ops.gemm_fp8_nt(a, b, leaf) == 8).all()


def test_8_bit_weights_without_the_native_step_are_refused():
    """The PyTorch step reads the parameters: with 8-bit weights in the state it would not do what was asked for."""
    from cverl_b200.models import decode
    from cverl_b200.models.config import Qwen35TextConfig
    from cverl_b200.models.qwen3_5 import Qwen35Model
    model = Qwen35Model(Qwen35TextConfig.tiny(), dtype=torch.float32, with_main_grad=False)
    model.init_weights(seed=1)
    with torch.no_grad():
        state, logits = decode.prefill(model, torch.arange(8).view(1, 8), max_len=12)
        decode.decode_step(model, state, logits.argmax(-1))
        state.fp8 = {}
        with pytest.raises(RuntimeError, match="native decode"):
            decode.decode_step(model, state, logits.argmax(-1))
        assert state.length == 9


def test_the_buffer_is_laid_out_as_the_kernels_lay_it_out():
    """Sizes and offsets of the Python side against those that the extension and the launchers are compiled with."""
    from cverl_b200 import _native as nv
    view = nv.torch_ext().view8
    for rows in (0, 1, 3, 127, 128, 129, 1000):
        for cols in (0, 1, 15, 16, 17, 128, 129, 511, 512, 513, 4100):
            q = ops.Fp8Tensor(torch.zeros(fp8._nbytes(rows, cols) + fp8._nbytes_plain(rows, cols), dtype=torch.uint8), rows, cols, E4M3)
            for got, want in ((view(q.buf, rows, cols, 0), q.values), (view(q.buf, rows, cols, 2), q.scales())):
                assert got.dtype == want.dtype and got.shape == want.shape and got.stride() == want.stride()
                assert got.storage_offset() == want.storage_offset()
            with pytest.raises(ValueError, match="not a buffer"):
                view(torch.zeros(q.buf.numel() + 1, dtype=torch.uint8), rows, cols, 0)
