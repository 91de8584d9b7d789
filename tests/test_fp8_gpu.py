"""8-bit operators on the kernels against plain 64-bit statements."""
import pytest
import torch

import fp8_oracle as orc
from cverl_b200 import ops
from fp8_oracle import E4M3, E5M2
from test_fp8_cpu import awkward

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _rand(*shape, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def _same(got, want):
    return torch.equal(torch.nan_to_num(got.double(), nan=1e300), torch.nan_to_num(want, nan=1e300))


def _check_quantised(got, want):
    assert _same(got.values, want[0])
    assert torch.equal(got.scales().double(), want[1][:, ::128])


# ----------------------------------------------------------------------------- quantisation: exact
SHAPES = [(1, 1), (1, 128), (1, 1024), (7, 129), (128, 128), (129, 127), (300, 1000), (257, 513), (515, 2055)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_codes_and_scales_are_the_definition(shape, dtype, src):
    x = awkward(*shape, src).cuda()
    rows, cols = orc.quantize(x, dtype), orc.quantize(x.t(), dtype)
    q, t = ops.quantize_fp8_pair(x, dtype)
    _check_quantised(q, rows)
    _check_quantised(t, cols)
    _check_quantised(ops.quantize_fp8(x, dtype), rows)
    _check_quantised(ops.quantize_fp8_t(x, dtype), cols)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_weight_blocks(shape, src):
    w = awkward(*shape, src).cuda()
    kept = ops.quantize_fp8_weight(w)
    _check_quantised(kept.w, orc.quantize(w, tall=128))
    assert _same(kept.wt.values, orc.quantize(w, tall=128)[0].t())
    assert _same(orc.value(kept.wt), orc.value(kept.w).t())
    _check_quantised(ops.quantize_fp8_weight(w, transposed=False).w, orc.quantize(w, tall=128))


def test_strides_and_alignments():
    base = _rand(300, 700, seed=1)
    for x in (base[:, 3:640], base[5:, 8:136], base[::3, 1:2], base.t(), base[:1].expand(140, 700), base[7]
              .unsqueeze(0), base.view(-1)[1:1 + 256 * 800].view(256, 800)):
        q, t = ops.quantize_fp8_pair(x)
        _check_quantised(q, orc.quantize(x))
        _check_quantised(t, orc.quantize(x.t()))


# ----------------------------------------------------------------------------- product
def _whole(rows, cols, seed):
    """Whole numbers up to 8 times a power of two per block: codes, scales and every partial sum are exact."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-8, 9, (rows, cols), device="cuda", generator=g).float()
    s = torch.randint(0, 4, (rows, -(-cols // 128)), device="cuda", generator=g).float()
    return v * torch.exp2(s).repeat_interleave(128, 1)[:, :cols]


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 7168, 1024), (2, 129, 513), (15, 300, 130), (16, 256, 2048), (17, 65, 16),
            (33, 127, 640), (64, 1000, 1000), (65, 512, 129), (128, 1024, 3584), (129, 130, 4096), (200, 4000, 256),
            (333, 1003, 1111), (512, 512, 512), (1000, 257, 385), (2049, 260, 131), (257, 2304, 1024),
            (1536, 1600, 640), (4100, 1024, 512), (300, 300, 9000), (300, 1, 200), (1000, 7, 129),
            (129, 128, 1)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_whole_numbers_is_exact(m, n, k):
    x, w = _whole(m, k, 1), _whole(n, k, 2)
    want = x.double() @ w.double().t()
    assert want.abs().max() < 2 ** 24                       # every sum is a whole number that fp32 holds
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w)
    got = ops.gemm_fp8_nt(a, b, out_dtype=torch.float32)
    assert torch.equal(got.double(), want)
    assert torch.equal(ops.gemm_fp8_nt(a, b), want.float().bfloat16())
    out = torch.full((m, n), 3.0, device="cuda")
    ops.gemm_fp8_nt(a, b, out, accumulate=True)
    assert torch.equal(out.double(), (want.float() + 3.0).double())


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("fa,fb", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2), (E4M3, E4M3)])
def test_product_of_random_values(m, n, k, fa, fb):
    a = ops.quantize_fp8(_rand(m, k, seed=m) * torch.exp(_rand(m, 1, seed=5)), fa)
    b = ops.quantize_fp8(_rand(n, k, seed=n, std=0.05), fb)
    x, w = orc.value(a), orc.value(b)
    got = ops.gemm_fp8_nt(a, b, out_dtype=torch.float32).double()
    # products of two 8-bit values are exact in fp32; each of the k additions is off by at most one step (2^-23) of a
    # partial sum, which is at most the sum of magnitudes
    assert ((got - x @ w.t()).abs() <= k * 2.0 ** -23 * (x.abs() @ w.abs().t())).all()


def test_output_that_is_a_range_of_a_wider_tensor():
    """Rows behind the last and columns beside the range keep what they held."""
    for m, n, k, c0 in [(5, 37, 200, 3), (300, 515, 140, 1), (129, 100, 128, 8), (700, 700, 300, 5)]:
        a, b = ops.quantize_fp8(_whole(m, k, 1)), ops.quantize_fp8(_whole(n, k, 2))
        want = ops.gemm_fp8_nt(a, b, out_dtype=torch.float32)
        for dt in (torch.float32, torch.bfloat16):
            wide = torch.full((m + 3, n + 11), 7.0, dtype=dt, device="cuda")
            ops.gemm_fp8_nt(a, b, wide[1:m + 1, c0:c0 + n])
            assert torch.equal(wide[1:m + 1, c0:c0 + n], want.to(dt))
            wide[1:m + 1, c0:c0 + n] = 7.0
            assert (wide == 7.0).all()


def test_non_finite_values_stay_in_their_rows():
    x, w = _rand(150, 300, seed=1), _rand(140, 300, seed=2)
    clean = ops.gemm_fp8_nt(ops.quantize_fp8(x), ops.quantize_fp8(w), out_dtype=torch.float32)
    x[3, 7], x[131, 299], w[5, 100] = float("inf"), float("nan"), float("-inf")
    got = ops.gemm_fp8_nt(ops.quantize_fp8(x), ops.quantize_fp8(w), out_dtype=torch.float32)
    bad = torch.zeros(150, 140, dtype=torch.bool, device="cuda")
    bad[3], bad[131], bad[:, 5] = True, True, True
    assert got[bad].isnan().all() and not got[~bad].isnan().any()
    same = ~bad
    same[[3, 131]] = False
    assert torch.equal(got[same], clean[same])


def test_product_is_the_same_from_run_to_run():
    for m, n, k in [(1, 1000, 3584), (128, 1024, 3584), (700, 900, 2000), (2048, 2048, 1024)]:
        a, b = ops.quantize_fp8(_rand(m, k, seed=1)), ops.quantize_fp8(_rand(n, k, seed=2))
        first = ops.gemm_fp8_nt(a, b, out_dtype=torch.float32)
        for _ in range(3):
            assert torch.equal(ops.gemm_fp8_nt(a, b, out_dtype=torch.float32), first)


# ----------------------------------------------------------------------------- rows quantised within the product
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (129, 127), (300, 130), (1000, 1000), (128, 4096), (7168, 1024), (520, 8200)])
def test_rows_quantised_within_the_product(m, n, k):
    kept = ops.quantize_fp8_weight(_whole(n, k, 2))
    x = _whole(m, k, 1).bfloat16()
    x[m // 2] = 0
    want = (orc.value(ops.quantize_fp8(x)) @ orc.value(kept.w).t()).float().bfloat16()
    assert torch.equal(ops.linear_fp8(x, kept), want)
    wide = torch.full((m, k + 3), 5.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:k + 1] = x
    assert torch.equal(ops.linear_fp8(wide[:, 1:k + 1], kept), want)
    # random values: the same codes and scales as the separate quantisation, fp32 sums of k products
    x = _rand(m, k, seed=m) * torch.exp(_rand(m, 1, seed=3))
    kept = ops.quantize_fp8_weight(_rand(n, k, seed=4))
    a, w = orc.value(ops.quantize_fp8(x)), orc.value(kept.w)
    got = ops.linear_fp8(x, kept).double()
    e = a @ w.t()
    assert ((got - e).abs() <= 2.0 ** -8 * e.abs() + k * 2.0 ** -23 * (1 + 2.0 ** -8) * (a.abs() @ w.abs().t())).all()


def test_rows_that_are_not_finite_within_the_product():
    kept = ops.quantize_fp8_weight(_rand(140, 300, seed=2))
    for m in (5, 20, 50, 128):
        x = _rand(m, 300, seed=1)
        clean = ops.linear_fp8(x, kept)
        x[1, 7], x[3, 299], x[4, 128] = float("inf"), float("nan"), float("-inf")
        got = ops.linear_fp8(x, kept)
        assert got[[1, 3, 4]].isnan().all()
        rest = [0, 2, *range(5, m)]
        assert torch.equal(got[rest], clean[rest])


# ----------------------------------------------------------------------------- norm
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 1024), (3, 129), (9, 128), (130, 256), (77, 500), (64, 513), (257, 1024),
                                    (31, 1111), (20, 2048), (33, 2560), (5, 4096), (7, 5000), (4, 8192), (3, 16384),
                                    (2, 16001), (5000, 64)])
@pytest.mark.parametrize("resid", [True, False])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_norm(rows, d, resid, dtype):
    x = _rand(rows, d, seed=rows, std=3.0)
    r = _rand(rows, d, seed=d) if resid else None
    w = _rand(d, seed=7, std=0.2)
    x[rows // 2] = 0.0
    if resid:
        r[rows // 2] = 0.0
    q, h = ops.add_rmsnorm_fp8(x, r, w, EPS, 1.0, dtype)
    y, want_h, _ = orc.norm(x, r, w, EPS, 1.0)
    assert torch.equal(h, want_h)
    # the fp32 row: sum of d squares (d half steps at most, one in practice halved by the root), root, two products
    fp32 = (d / 2 + 8) * 2.0 ** -24
    s = q.scales().double().repeat_interleave(128, 1)[:, :d]
    _, exact_s = orc.quantize(y, dtype)
    # a scale is the definition's, or the neighbour where the block's maximum is that close to the border
    big = torch.stack([b.abs().amax(1) for b in y.split(128, 1)], 1).repeat_interleave(128, 1)[:, :d]
    edge = orc.FMAX[dtype] * torch.minimum(s, exact_s)
    assert ((s == exact_s) | ((big / edge - 1).abs() <= fp32)).all()
    step, low = (2.0 ** -4, 2.0 ** -10) if dtype == E4M3 else (2.0 ** -3, 2.0 ** -17)
    assert ((orc.value(q) - y).abs() <= y.abs() * (step + 2 * fp32) + low * s).all()


def test_norm_strides_and_rows_of_no_number():
    x, r, w = _rand(40, 600, seed=1), _rand(40, 600, seed=2), _rand(512, seed=3, std=0.1)
    x[3, 9], x[4, 20] = float("nan"), float("inf")
    cols = (x[:, 5:517], r[:, 8:520])
    q, h = ops.add_rmsnorm_fp8(*cols, w)
    q2, h2 = ops.add_rmsnorm_fp8(cols[0].contiguous(), cols[1].contiguous(), w)
    assert _same(q.values, q2.values.double()) and torch.equal(q.scales().view(torch.uint8), q2.scales().view(torch.uint8))
    assert _same(h, h2.double())
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = True
    assert q.values[3].isnan().all()
    assert q.values[4].isnan().any() and not q.values[5:].float().isnan().any()


# ----------------------------------------------------------------------------- linear layers
def _near(got, want, terms):
    """bf16 result of fp32 sums: half a step of 2^-8, and the sums' 2^-24 a term of the norm."""
    assert (got.double() - want).norm() <= (2.0 ** -8 + terms * 2.0 ** -24) * want.norm()


LAYERS = [(1, 128, 64), (5, 100, 33), (77, 512, 1536), (130, 257, 129), (300, 1000, 520), (1301, 640, 384), (2100, 1024, 2048)]


@pytest.mark.parametrize("m,k,n", LAYERS)
@pytest.mark.parametrize("grad", [E4M3, E5M2])
def test_linear_and_gradients(m, k, n, grad):
    x, w, dy = _rand(m, k, seed=1), _rand(n, k, seed=2, std=k ** -0.5), _rand(m, n, seed=3, std=1e-3)
    x.requires_grad_(), w.requires_grad_()
    y = ops.linear_fp8(x, w, grad_dtype=grad)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    qw = orc.through(w.detach(), tall=128)
    _near(y.detach(), orc.through(x.detach()) @ qw.t(), k)
    _near(dx, orc.through(dy, grad) @ qw, n)
    _near(dw, orc.through(dy.t(), grad) @ orc.through(x.detach().t()).t(), m)
    assert torch.equal(ops.linear_fp8(x.detach(), ops.quantize_fp8_weight(w.detach())), y.detach())
    w.main_grad = torch.ones(n, k, device="cuda")
    dw32 = ops.linear_fp8(x, w, grad_dtype=grad, weight=ops.quantize_fp8_weight(w))
    dw32.backward(dy)
    assert w.grad is None
    want = orc.through(dy.t(), grad) @ orc.through(x.detach().t()).t()
    assert (w.main_grad.double() - 1 - want).norm() <= (m + 1) * 2.0 ** -24 * (want.norm() + (n * k) ** 0.5)


# tiles of the longer and of the shorter product: less than a round of 74 CTA pairs together; more than one round each,
# either product the longer; exactly one round; one tile; columns and rows that end inside a tile
@pytest.mark.parametrize("m,k,n", [(200, 520, 2000), (5000, 1300, 4000), (2900, 1300, 6400), (300, 18900, 256),
                                   (1301, 523, 1003), (129, 130, 131), (20000, 300, 260), (640, 5000, 8200)])
def test_both_gradients_of_whole_numbers_are_exact(m, k, n):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w, dy = (torch.randint(-8, 9, s, device="cuda", generator=g).bfloat16() for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_fp8(x, w), (x, w), dy)          # sums below 64 * 20000 < 2^24
    assert torch.equal(dx, (dy.double() @ w.detach().double()).float().bfloat16())
    assert torch.equal(dw, (dy.double().t() @ x.detach().double()).float().bfloat16())
    w.main_grad = torch.ones(n, k, device="cuda")
    sign = dy.sign()                                                        # e5m2 has three digits
    ops.linear_fp8(x, w, grad_dtype=E5M2).backward(sign)
    assert torch.equal(w.main_grad.double(), sign.double().t() @ x.detach().double() + 1)
    assert torch.equal(x.grad, (sign.double() @ w.detach().double()).float().bfloat16())


@pytest.mark.parametrize("m,k,n", LAYERS + [(40, 4100, 96), (9, 8192, 64), (6, 16384, 32)])
@pytest.mark.parametrize("resid", [True, False])
def test_norm_linear_and_gradients(m, k, n, resid):
    x, w, wn = _rand(m, k, seed=1), _rand(n, k, seed=2, std=k ** -0.5), _rand(k, seed=3, std=0.1)
    r = _rand(m, k, seed=4) if resid else None
    dy, dh = _rand(m, n, seed=5, std=1e-2), _rand(m, k, seed=6, std=1e-2)
    leaves = [t.requires_grad_() for t in (x, r, wn, w) if t is not None]
    y, h = ops.add_rmsnorm_linear_fp8(x, r, wn, w, EPS, 1.0)
    outs, seeds = ((y, h), (dy, dh)) if resid else ((y,), (dy,))
    grads = torch.autograd.grad(outs, leaves, seeds)
    with torch.no_grad():
        nrm, want_h, rstd = orc.norm(x, r, wn, EPS, 1.0)
        assert torch.equal(h, want_h)
        # what the kernel rounded, from its own fp32 norm: at a rounding border it may differ from the 64-bit norm's by
        # a step of 2^-3 of a value, which happens to at most one in 2^14 of them (fp32 steps against e4m3 steps)
        few = 2.0 ** -3 * 2.0 ** -7
        qw = orc.through(w, tall=128)
        want_y = orc.through(nrm) @ qw.t()
        assert (y.double() - want_y).norm() <= (2.0 ** -8 + k * 2.0 ** -24 + few) * want_y.norm()
        dn = orc.through(dy) @ qw
        want_dw = orc.through(dy.t()) @ orc.through(nrm.t()).t()
        dx, dwn = orc.norm_grads(want_h, rstd, wn, 1.0, dn, dh if resid else None)
        assert (grads[-1].double() - want_dw).norm() <= (2.0 ** -8 + m * 2.0 ** -24 + few) * want_dw.norm()
        # dn is bf16 between the product and the norm: one more half step of it, and of what it is subtracted from
        size = (rstd * dn * (1.0 + wn.double())).norm()
        tol = 2.0 ** -8 * dx.norm() + (2 * 2.0 ** -8 + n * 2.0 ** -24) * size
        for g in grads[:2 if resid else 1]:
            assert (g.double() - dx).norm() <= tol
        xh = want_h.double() * rstd
        assert (grads[-2].double() - dwn).norm() <= 2.0 ** -8 * dwn.norm() + 2.0 ** -8 * (dn * xh).abs().sum(0).norm()


def test_norm_weight_gradient_is_the_same_from_run_to_run():
    x, wn, w = _rand(3000, 384, seed=1), _rand(384, seed=2).requires_grad_(), _rand(64, 384, seed=3)
    kept = ops.quantize_fp8_weight(w)
    runs = []
    for _ in range(3):
        y, _ = ops.add_rmsnorm_linear_fp8(x, None, wn, kept)
        runs.append(torch.autograd.grad(y, wn, torch.ones_like(y))[0])
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    wn.main_grad = torch.zeros(384, device="cuda")
    y, _ = ops.add_rmsnorm_linear_fp8(x, None, wn, kept)
    y.backward(torch.ones_like(y))
    assert torch.equal(wn.main_grad.bfloat16(), runs[0])


# ----------------------------------------------------------------------------- together
def _mlp(x, r, wn, w1, w2):
    gu, h = ops.add_rmsnorm_linear_fp8(x, r, wn, w1)
    return ops.linear_fp8(ops.swiglu(gu), w2), h


def test_feed_forward_block_trains():
    """Norm, gate|up, SwiGLU and down projection as a model runs them, against the same block in 64 bits."""
    m, d, f = 700, 512, 896
    x, r = _rand(m, d, seed=1).requires_grad_(), _rand(m, d, seed=2).requires_grad_()
    wn = _rand(d, seed=3, std=0.1).requires_grad_()
    w1, w2 = _rand(2 * f, d, seed=4, std=d ** -0.5).requires_grad_(), _rand(d, f, seed=5, std=f ** -0.5).requires_grad_()
    leaves = (x, r, wn, w1, w2)
    y, h = _mlp(*leaves)
    dy = _rand(m, d, seed=6)
    grads = torch.autograd.grad((y, h), leaves, (dy, dy))
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    h64 = l64[0] + l64[1]
    n64 = h64 * torch.rsqrt((h64 * h64).mean(-1, keepdim=True) + EPS) * (1 + l64[2])
    g64, u64 = (n64 @ l64[3].t()).chunk(2, -1)
    y64 = (torch.nn.functional.silu(g64) * u64) @ l64[4].t()
    want = torch.autograd.grad((y64, h64), l64, (dy.double(), dy.double()))
    # each 8-bit rounding is at most 2^-4 of its value; the chain has at most 6 of them in any gradient
    for g, e in zip((y.detach(), *grads), (y64.detach(), *want)):
        assert (g.double() - e).norm() <= 6 * 2.0 ** -4 * e.norm()


def test_decoding_and_prefill_of_a_block_agree():
    """Tokens one by one give what they give together: rows do not depend on each other."""
    d, f, m = 1024, 3584, 9
    wn, w1, w2 = _rand(d, seed=1, std=0.1), _rand(2 * f, d, seed=2, std=0.03), _rand(d, f, seed=3, std=0.02)
    kept = ops.quantize_fp8_weight(w1, transposed=False), ops.quantize_fp8_weight(w2, transposed=False)
    x, r = _rand(m, d, seed=4), _rand(m, d, seed=5)

    def block(x, r):
        q, h = ops.add_rmsnorm_fp8(x, r, wn)
        return ops.linear_fp8(ops.swiglu(ops.linear_fp8(q, kept[0])), kept[1]), h

    with torch.no_grad():
        y, h = block(x, r)
        for i in range(m):
            yi, hi = block(x[i:i + 1], r[i:i + 1])
            assert torch.equal(hi, h[i:i + 1])
            assert (yi.double() - y[i:i + 1].double()).norm() <= 2.0 ** -7 * y[i].double().norm()


# ----------------------------------------------------------------------------- streams, graphs, refusals
def test_other_stream():
    x, w = _rand(300, 512, seed=1), _rand(256, 512, seed=2)
    want = ops.linear_fp8(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_fp8(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_two_streams_at_once():
    """Products and quantisations of two streams run side by side: nothing is shared between calls."""
    jobs = []
    for seed, (m, n, k) in enumerate([(700, 1500, 1024), (3, 2048, 2048)]):
        jobs.append((_rand(m, k, seed=seed), ops.quantize_fp8_weight(_rand(n, k, seed=seed + 10))))
    want = [ops.linear_fp8(x, w) for x, w in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(20):
        for i, (s, (x, w)) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i].append(ops.linear_fp8(x, w))
    torch.cuda.synchronize()
    for outs, e in zip(got, want):
        assert all(torch.equal(o, e) for o in outs)


def test_offsets_past_32_bits():
    """More than 2^31 elements in the input of a quantisation, in its codes and in a product's result."""
    rows, cols = 70016, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail = _rand(200, cols, seed=1)
    x[-200:] = tail
    q, t = ops.quantize_fp8_pair(x)
    del x
    want = orc.quantize(tail)
    assert _same(q.values[-200:], want[0]) and torch.equal(q.scales()[-200:].double(), want[1][:, ::128])
    # 70016 = 547 * 128: the last block of a transposed row is the last 128 rows
    assert _same(t.values[:, -128:], orc.quantize(tail[-128:].t())[0])
    del q, t
    a, b = _whole(rows, 128, 1), _whole(cols, 128, 2)
    y = ops.gemm_fp8_nt(ops.quantize_fp8(a), ops.quantize_fp8(b))
    at = [0, 1, 65535, 65537, rows - 129, rows - 1]
    assert torch.equal(y[at], (a[at] @ b.t()).bfloat16())


def test_two_captured_graphs_replayed_in_turn():
    w = ops.quantize_fp8_weight(_rand(700, 512, seed=1))
    wn = _rand(512, seed=2)
    xs = [_rand(5, 512, seed=3), _rand(130, 512, seed=4)]
    ops.linear_fp8(xs[0], w)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q, _ = ops.add_rmsnorm_fp8(x, None, wn)
            outs.append(ops.linear_fp8(q, w) + ops.linear_fp8(x, w))
        graphs.append(g)
    for seed in (10, 11):
        for x, g, out in zip(xs, graphs, outs):
            x.copy_(_rand(*x.shape, seed=seed))
            g.replay()
        for x, out in zip(xs, outs):
            want = ops.linear_fp8(ops.add_rmsnorm_fp8(x, None, wn)[0], w) + ops.linear_fp8(x, w)
            assert torch.equal(out, want)


def test_captured_training_step():
    x, w = _rand(200, 256, seed=1).requires_grad_(), _rand(300, 256, seed=2).requires_grad_()
    dy = _rand(200, 300, seed=3)
    want = torch.autograd.grad(ops.linear_fp8(x, w), (x, w), dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(ops.linear_fp8(x, w), (x, w), dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(ops.linear_fp8(x, w), (x, w), dy)
    for _ in range(2):
        g.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_backward_twice_and_expanded_gradient():
    x, w = _rand(20, 200, seed=1).requires_grad_(), _rand(30, 200, seed=2).requires_grad_()
    y = ops.linear_fp8(x, w)
    first = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    again = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_batches_of_sequences_and_computed_weights():
    """Leading dimensions are kept, a weight may be the result of an operation, a gradient may be missing or strided."""
    x, r = _rand(3, 7, 260, seed=1).requires_grad_(), _rand(3, 7, 260, seed=2).requires_grad_()
    w, wn = _rand(130, 260, seed=3).requires_grad_(), _rand(260, seed=4, std=0.1).requires_grad_()
    dy = _rand(3, 7, 130, seed=5)
    flat = torch.autograd.grad(ops.linear_fp8(x.view(21, 260), w), (x, w), dy.view(21, 130))
    got = torch.autograd.grad(ops.linear_fp8(x, w * 1.0), (x, w), dy.transpose(0, 1).contiguous().transpose(0, 1))
    assert got[0].shape == x.shape and all(torch.equal(a, b.view_as(a)) for a, b in zip(got, flat))
    y, h = ops.add_rmsnorm_linear_fp8(x, r, wn, w)
    assert y.shape == (3, 7, 130) and torch.equal(h, x + r)
    y2, h2 = ops.add_rmsnorm_linear_fp8(x.view(21, 260), r.view(21, 260), wn, w)
    assert torch.equal(y.view(21, 130), y2)
    a = torch.autograd.grad(y, (x, r, wn, w), dy, retain_graph=True)
    b = torch.autograd.grad(y2, (x, r, wn, w), dy.view(21, 130))
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    dh, = torch.autograd.grad(h, x, torch.ones_like(h))             # only h is used
    assert torch.equal(dh, torch.ones_like(dh))
    with torch.no_grad():
        q, h3 = ops.add_rmsnorm_fp8(x, r, wn)
        assert q.shape == (21, 260) and torch.equal(h3, h) and torch.equal(ops.linear_fp8(q, w), y2)
    one = torch.autograd.grad(ops.linear_fp8(x[0, 0], w), w, dy[0, 0])[0]        # a single row without dimensions
    assert one.shape == w.shape


def test_only_some_gradients():
    x, w, wn, r = _rand(40, 200, seed=1), _rand(30, 200, seed=2), _rand(200, seed=3), _rand(40, 200, seed=4)
    full = [t.clone().requires_grad_() for t in (x, r, wn, w)]
    dy = _rand(40, 30, seed=5)
    want = torch.autograd.grad(ops.add_rmsnorm_linear_fp8(*full)[0], full, dy)
    for i in range(4):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, r, wn, w))]
        got, = torch.autograd.grad(ops.add_rmsnorm_linear_fp8(*leaves)[0], leaves[i], dy)
        assert torch.equal(got, want[i])
    for t in (x, w):
        t.requires_grad_()
        g, = torch.autograd.grad(ops.linear_fp8(x, w), t, dy)
        t.requires_grad_(False)
        both = torch.autograd.grad(ops.linear_fp8(*(a := [v.clone().requires_grad_() for v in (x, w)])), a, dy)
        assert torch.equal(g, both[0 if t is x else 1])


def test_no_second_derivative():
    x, w = _rand(4, 64, seed=1).requires_grad_(), _rand(8, 64, seed=2).requires_grad_()
    g, = torch.autograd.grad(ops.linear_fp8(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.add_rmsnorm_fp8(x, None, _rand(64))
    with pytest.raises(ValueError, match="transposed"):
        ops.linear_fp8(x, ops.quantize_fp8_weight(w, transposed=False))


def test_launches_are_counted():
    from cverl_b200.ops.gemm import launch_counter
    x, w, wn = _rand(200, 256, seed=1).requires_grad_(), _rand(300, 256, seed=2).requires_grad_(), _rand(256).requires_grad_()
    n = launch_counter["n"]
    y = ops.linear_fp8(x, w)                                # weight, input, product
    assert launch_counter["n"] == n + 3
    y.backward(torch.ones_like(y))                          # gradient, both products
    assert launch_counter["n"] == n + 5
    y, _ = ops.add_rmsnorm_linear_fp8(x, None, wn, w)       # weight, norm, product
    y.backward(torch.ones_like(y))                          # gradient, norm's transpose, both products, norm, its weight
    assert launch_counter["n"] == n + 13


def test_empty_calls():
    w = _rand(30, 200, seed=2).requires_grad_()
    x = torch.empty(0, 200, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y, _ = ops.add_rmsnorm_linear_fp8(x, None, _rand(200), w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == (0, 200) and not dw.any()
    a, b = ops.quantize_fp8(_rand(4, 0)), ops.quantize_fp8(_rand(5, 0))
    assert not ops.gemm_fp8_nt(a, b).any()


def test_refusals():
    h = _rand(4, 64).half()
    for call in (lambda: ops.quantize_fp8(h), lambda: ops.linear_fp8(h, _rand(8, 64)),
                 lambda: ops.linear_fp8(_rand(4, 64).float(), _rand(8, 64)),
                 lambda: ops.add_rmsnorm_fp8(_rand(4, 64).float(), None, _rand(64).float()),
                 lambda: ops.linear_fp8(_rand(4, 64), _rand(8, 64), grad_dtype=torch.float16)):
        with pytest.raises(TypeError):
            call()
    a = ops.quantize_fp8(_rand(4, 64))
    for call in (lambda: ops.gemm_fp8_nt(a, ops.quantize_fp8(torch.ones(4, 64))),
                 lambda: ops.gemm_fp8_nt(a, ops.quantize_fp8(_rand(4, 65))),
                 lambda: ops.linear_fp8(torch.ones(4, 64), _rand(8, 64)),
                 lambda: ops.add_rmsnorm_fp8(_rand(4, 64), None, torch.ones(64))):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_values_and_scales_are_views_of_the_buffer():
    q = ops.quantize_fp8(_rand(3, 200), E5M2)
    v, s = q.values, q.scales()
    assert v.dtype == E5M2 and v.shape == (3, 200) and v.stride() == (208, 1) and v.device == q.device
    assert s.dtype == torch.float8_e8m0fnu and s.shape == (3, 2) and s.is_contiguous()
    assert v.untyped_storage().data_ptr() == s.untyped_storage().data_ptr() == q.buf.data_ptr()
    del q                                                    # the views keep the memory
    kept = v.float().clone()
    torch.empty(3 * 208 + 1024, dtype=torch.uint8, device="cuda").fill_(255)
    assert torch.equal(v.float(), kept) and not v.requires_grad and not v.clone().requires_grad
    assert torch.equal(torch.cat([v.view(torch.uint8), v.view(torch.uint8)])[3:], v.view(torch.uint8))
    e = ops.quantize_fp8(torch.empty(0, 5, device="cuda"))
    assert e.values.shape == (0, 5) and e.scales().shape == (0, 1)


@pytest.mark.parametrize("m", [1, 24, 40, 128, 300, 2048])
def test_overlapped_launches_give_what_separate_ones_give(m):
    """Layers without a pause, weights changed in between, against the same operators one at a time."""
    d, f = 1024, 2560
    x0, r0, wn = _rand(m, d, seed=1), _rand(m, d, seed=2), _rand(d, seed=3, std=0.1)
    up0, down0 = _rand(f, d, seed=4, std=d ** -0.5), _rand(d, f, seed=5, std=f ** -0.5)
    kept = ops.quantize_fp8_weight(_rand(d, d, seed=6, std=d ** -0.5))

    def fast():
        x, r, up, down = x0.clone(), r0.clone(), up0.clone(), down0.clone()
        for i in range(30):
            y, r = ops.add_rmsnorm_linear_fp8(x, r, wn, up)
            up.mul_(-1.001)
            x = ops.linear_fp8(y, down)
            down.mul_(-0.999)
            x = ops.linear_fp8(x, kept)
        return x, r, y

    def one_at_a_time():
        def product(q, w):
            torch.cuda.synchronize()
            y = ops.gemm_fp8_nt(q, w if isinstance(w, ops.Fp8Tensor) else ops.quantize_fp8_weight(w).w)
            torch.cuda.synchronize()
            return y
        x, r, up, down = x0.clone(), r0.clone(), up0.clone(), down0.clone()
        for i in range(30):
            q, r = ops.add_rmsnorm_fp8(x, r, wn)
            y = product(q, up)
            up.mul_(-1.001)
            x = product(ops.quantize_fp8(y), down)
            down.mul_(-0.999)
            x = product(ops.quantize_fp8(x), kept.w)
        return x, r, y

    with torch.no_grad():
        want = one_at_a_time()
        for got in (fast(), fast()):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            got = fast()
        for _ in range(2):
            g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_overlapped_backward_passes():
    """Training steps without a pause: whole numbers, so that every result is exact; and a norm in front, against the
    same steps with a pause before and after each."""
    m, k, n = 1500, 1024, 1280
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w0, dy = (torch.randint(-8, 9, s, device="cuda", generator=g).bfloat16() for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_()
    w = w0.clone().requires_grad_()
    w.main_grad = torch.zeros(n, k, device="cuda")
    got = []
    for i in range(30):
        got.append(torch.autograd.grad(ops.linear_fp8(x, w), (x, w), dy, allow_unused=True)[0])
        with torch.no_grad():
            w.mul_(-1.0 if i % 3 else 0.5 ** (i % 2))
            dy = dy.neg()
    want, main = [], torch.zeros(n, k, device="cuda", dtype=torch.float64)
    scale, sign = 1.0, 1.0
    dx0, dw0 = dy.double() @ w0.double(), dy.double().t() @ x.detach().double()
    for i in range(30):
        assert torch.equal(got[i], (dx0 * scale * sign).float().bfloat16())
        main += sign * dw0
        scale, sign = scale * (-1.0 if i % 3 else 0.5 ** (i % 2)), -sign
    assert torch.equal(w.main_grad.double(), main)

    r, wn, d = _rand(m, k, seed=4), _rand(k, seed=5, std=0.1), _rand(m, n, seed=6, std=1e-2)

    def steps(pause):
        a, b, c, e = (t.detach().clone().requires_grad_() for t in (_rand(m, k, seed=7), r, wn, _rand(n, k, seed=8)))
        for i in range(15):
            pause()
            y, h = ops.add_rmsnorm_linear_fp8(a, b, c, e)
            pause()
            grads = torch.autograd.grad((y, h), (a, b, c, e), (d, r))
            pause()
            with torch.no_grad():
                for t, u in zip((a, b, c, e), grads):
                    t.add_(u, alpha=-0.1)
        return y, h, a, b, c, e

    for u, v in zip(steps(lambda: None), steps(torch.cuda.synchronize)):
        assert torch.equal(u, v)


def test_two_threads_launch_into_one_stream():
    """Forward and backward passes of two host threads mix their launches in one stream."""
    import threading

    def work(m, seed, steps, out):
        x, w = _rand(m, 512, seed=seed).requires_grad_(), _rand(640, 512, seed=seed + 1, std=0.05).requires_grad_()
        wn, dy = _rand(512, seed=seed + 2, std=0.1).requires_grad_(), _rand(m, 640, seed=seed + 3)
        for i in range(steps):
            y = ops.linear_fp8(x, w)
            g = torch.autograd.grad(y, (x, w), dy)
            z, h = ops.add_rmsnorm_linear_fp8(x, None, wn, w)
            k = torch.autograd.grad(z, (x, wn, w), dy)
            out[:] = [y.detach(), z.detach(), *g, *k]

    want, got = {}, {}
    for m in (40, 600):
        work(m, m, 1, want.setdefault(m, []))
    for _ in range(3):
        threads = [threading.Thread(target=work, args=(m, m, 40, got.setdefault(m, []))) for m in (40, 600)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for m in want:
            assert len(got[m]) == len(want[m]) == 7 and all(torch.equal(a, b) for a, b in zip(got[m], want[m]))


@pytest.mark.parametrize("shape", [(40, 96), (2, 3, 129)])
def test_a_weight_without_rows_leaves_the_sum(shape):
    """y has no columns; x + resid and its gradients are what they always are."""
    def poison():                       # what the allocator hands out next
        torch.full(shape, 7.0, dtype=torch.bfloat16, device="cuda")

    x, r, wn = _rand(*shape, seed=1), _rand(*shape, seed=2), _rand(shape[-1], seed=3, std=0.1)
    w, dh = torch.empty(0, shape[-1], dtype=torch.bfloat16, device="cuda"), _rand(*shape, seed=4)
    for weight in (w, ops.quantize_fp8_weight(w)):
        poison()
        with torch.no_grad():
            y, h = ops.add_rmsnorm_linear_fp8(x, r, wn, weight)
        assert y.shape == (*shape[:-1], 0) and torch.equal(h, x + r)
    leaves = [t.clone().requires_grad_() for t in (x, r, wn, w)]
    poison()
    y, h = ops.add_rmsnorm_linear_fp8(*leaves)
    assert torch.equal(h, x + r)
    dx, dr, dwn, dw = torch.autograd.grad((y, h), leaves, (torch.empty_like(y), dh))
    assert torch.equal(dx, dh) and torch.equal(dr, dh) and not dwn.any() and dw.shape == w.shape
    y, h = ops.add_rmsnorm_linear_fp8(x, None, wn, w)
    assert h is x and y.numel() == 0


# rows per CTA 8, 4, 2 and 1 of the norm's backward pass, one row to more than its CTAs hold at once
@pytest.mark.parametrize("m,k", [(1, 200), (1301, 200), (37, 400), (900, 1000), (2100, 1024), (150, 2048), (40, 4100),
                                 (9, 8192), (300, 16384)])
def test_norm_gradients_keep_fp32_between_product_and_norm(m, k):
    """dy and w are whole numbers that 8 bits hold, so dn = dy w is exact in fp32, and mostly not in bf16."""
    n = 600
    g = torch.Generator(device="cuda").manual_seed(m + k)
    dy, w = (torch.randint(-8, 9, s, device="cuda", generator=g).bfloat16() for s in ((m, n), (n, k)))
    x, r, wn, dh = _rand(m, k, seed=1), _rand(m, k, seed=2), _rand(k, seed=3, std=0.1), _rand(m, k, seed=4)
    dn = dy.double() @ w.double()
    assert dn.abs().max() < 2 ** 24
    _, h, rstd = orc.norm(x, r, wn, EPS, 1.0)
    xh, gain = h.double() * rstd, 1.0 + wn.double()
    # rstd: k / 2 + 8 half steps (see test_norm); the mean of g xh: k additions; a handful of products and sums
    fp32 = (1.5 * k + 16) * 2.0 ** -24
    size = (rstd * dn * gain).abs() + rstd * xh.abs() * (dn * gain * xh).abs().mean(-1, keepdim=True) + dh.double().abs()
    want, dwn = orc.norm_grads(h, rstd, wn, 1.0, dn, dh)
    near = 2.0 ** -8 * want.abs() + fp32 * (1 + 2.0 ** -8) * size
    leaves = [t.requires_grad_() for t in (x, r, wn)]
    y, h_out = ops.add_rmsnorm_linear_fp8(*leaves, ops.quantize_fp8_weight(w), EPS, 1.0)
    dx, dr, dw16 = torch.autograd.grad((y, h_out), leaves, (dy, dh), retain_graph=True)
    assert torch.equal(dx, dr) and ((dx.double() - want).abs() <= near).all()
    if m * k > 10000:                              # a bf16 rounding of dn would show
        rounded, _ = orc.norm_grads(h, rstd, wn, 1.0, dn.bfloat16().double(), dh)
        assert not ((rounded.bfloat16().double() - want).abs() <= near).all()
    # m additions, and rstd's half steps
    sums = (m + k / 2 + 16) * 2.0 ** -24 * (dn * xh).abs().sum(0)
    assert ((dw16.double() - dwn).abs() <= 2.0 ** -8 * dwn.abs() + (1 + 2.0 ** -8) * sums).all()
    wn.main_grad = torch.zeros(k, device="cuda")
    torch.autograd.backward((y, h_out), (dy, dh), inputs=[wn], retain_graph=True)
    assert ((wn.main_grad.double() - dwn).abs() <= sums).all()
    # one row at a time: every share of the weight's gradient arrives, and none of it in another row's dx
    for row in {0, m // 3, m // 2, max(m - 2, 0), m - 1}:
        one = torch.zeros_like(dy)
        one[row] = dy[row]
        wn.main_grad.zero_()                       # every pass through the layer adds to it
        dx, = torch.autograd.grad((y, h_out), (x,), (one, dh), retain_graph=True)
        e = dn[row] * xh[row]
        assert ((wn.main_grad.double() - e).abs() <= (k / 2 + 16) * 2.0 ** -24 * e.abs()).all()
        assert ((dx[row].double() - want[row]).abs() <= near[row]).all()
        dx[row] = dh[row]
        assert torch.equal(dx, dh)


# the few-rows kernel with tiles of 16 (three), 32, 64 (two, one more last) and 128 rows, K shared by up to eight CTAs, and
# once CTA pairs
@pytest.mark.parametrize("m,n,k", [(1, 1000, 640), (16, 513, 3584), (5, 30000, 300), (24, 256, 2048), (40, 1024, 4000),
                                   (100, 300, 4096), (100, 5000, 1800), (128, 8192, 512), (300, 513, 700)])
@pytest.mark.parametrize("beside", [0, 3])
def test_overlapped_accumulating_products(m, n, k, beside):
    """Products that add to one matrix without a pause between them, their operands and their sum changed on the way."""
    steps = 30
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = (torch.randint(-8, 9, s, device="cuda", generator=g).bfloat16() for s in ((m, k), (n, k)))
    step = x.double() @ w.double().t()
    assert 2 * steps * step.abs().max() < 2 ** 24
    b = ops.quantize_fp8(w)
    wide = torch.full((m, n + beside), 5.0, device="cuda")
    out = wide[:, beside:]
    out.zero_()
    want, sign = torch.zeros_like(step), 1
    torch.cuda.synchronize()
    for i in range(steps):
        a = ops.quantize_fp8(x)
        ops.gemm_fp8_nt(a, b, out, accumulate=True)
        want += sign * step
        if i % 4 != 3:
            ops.gemm_fp8_nt(a, b, out, accumulate=True)
            want += sign * step
        if i % 3 == 1:
            x.neg_()
            sign = -sign
        if i % 5 == 2:
            out.neg_()
            want.neg_()
    assert torch.equal(out.double(), want)
    assert (wide[:, :beside] == 5.0).all()


def test_a_refusal_of_a_launcher_is_an_exception():
    """A buffer that does not start on 16 bytes: the launchers refuse it before anything runs."""
    q, kept = ops.quantize_fp8(_rand(20, 64, seed=1)), ops.quantize_fp8_weight(_rand(30, 64, seed=2))
    room = torch.empty(q.buf.numel() + 8, dtype=torch.uint8, device="cuda")
    room[8:] = q.buf
    odd = ops.Fp8Tensor(torch.from_dlpack(room[8:]), 20, 64, E4M3)
    assert odd.buf.data_ptr() % 16 == 8
    for call in (lambda: ops.gemm_fp8_nt(odd, kept.w), lambda: ops.linear_fp8(odd, kept)):
        with pytest.raises(RuntimeError, match="failed with code -3"):
            call()
    assert torch.equal(ops.linear_fp8(q, kept), ops.gemm_fp8_nt(q, kept.w))


def test_a_main_grad_that_does_not_fit_is_an_exception():
    """Raised from the backward pass, before anything is added anywhere."""
    x, w, wn = _rand(20, 64, seed=1).requires_grad_(), _rand(30, 64, seed=2).requires_grad_(), _rand(64, seed=3).requires_grad_()
    good, good_n = torch.zeros(30, 64, device="cuda"), torch.zeros(64, device="cuda")
    for bad, bad_n, err in ((good.bfloat16(), good_n, TypeError), (good.t().contiguous().t(), good_n, TypeError),
                            (good[:29], good_n, TypeError), (good.cpu(), good_n, TypeError), ("no tensor", good_n, RuntimeError),
                            (good, good_n.bfloat16(), TypeError)):
        w.main_grad, wn.main_grad = bad, bad_n
        if bad is not good:
            with pytest.raises(err):
                ops.linear_fp8(x, w).sum().backward()
        with pytest.raises(err):
            ops.add_rmsnorm_linear_fp8(x, None, wn, w)[0].sum().backward()
        assert not good.any() and not good_n.any() and x.grad is None
    w.main_grad, wn.main_grad = good, good_n
    ops.add_rmsnorm_linear_fp8(x, None, wn, w)[0].sum().backward()
    assert good.any() and good_n.any() and x.grad is not None
