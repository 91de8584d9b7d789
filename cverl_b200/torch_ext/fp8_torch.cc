// The 8-bit linear layers between autograd and the launchers of libcverl_b200_cuda.so: workspaces, autograd nodes and
// the choice of what a pass computes, for CUDA tensors.
//
// A small layer is bound by its host side, and most of that was Python: nodes, workspaces and launches through ctypes.
// The arguments are checked by the Python functions that call in here (ops/fp8.py); the launchers' addresses come from
// the ctypes library, so that it is loaded once.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include "fp8_launch.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---------------------------------------------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------------------------------------------
struct Launchers {
  decltype(&cvb_fp8_quantize) quantize;
  decltype(&cvb_fp8_add_rmsnorm) add_rmsnorm;
  decltype(&cvb_fp8_linear_fwd) linear_fwd;
  decltype(&cvb_fp8_linear_bwd) linear_bwd;
  decltype(&cvb_fp8_norm_linear_fwd) norm_linear_fwd;
  decltype(&cvb_fp8_norm_linear_bwd) norm_linear_bwd;
  decltype(&cvb_fp8_norm_bwd_parts) norm_bwd_parts;
  decltype(&cvb_fp8_gemm_grads_launches) gemm_grads_launches;
} fn;

PyObject* launch_counter = nullptr;   // ops.gemm.launch_counter

template <typename F>
void take(F& f, const pybind11::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}
void bind(const pybind11::dict& addresses, pybind11::dict counter) {
  take(fn.quantize, addresses, "cvb_fp8_quantize");
  take(fn.add_rmsnorm, addresses, "cvb_fp8_add_rmsnorm");
  take(fn.linear_fwd, addresses, "cvb_fp8_linear_fwd");
  take(fn.linear_bwd, addresses, "cvb_fp8_linear_bwd");
  take(fn.norm_linear_fwd, addresses, "cvb_fp8_norm_linear_fwd");
  take(fn.norm_linear_bwd, addresses, "cvb_fp8_norm_linear_bwd");
  take(fn.norm_bwd_parts, addresses, "cvb_fp8_norm_bwd_parts");
  take(fn.gemm_grads_launches, addresses, "cvb_fp8_gemm_grads_launches");
  launch_counter = counter.release().ptr();
}
void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed with code ", rc); }

// the caller holds the GIL
void count_launches(long n) {
  pybind11::handle counter(launch_counter);
  counter["n"] = pybind11::int_(counter["n"].cast<long>() + n);
}

// ---------------------------------------------------------------------------------------------------------------
// sizes and buffers
// ---------------------------------------------------------------------------------------------------------------
enum { ROWS = 1, COLS = 2 };
enum { OUT_BF16 = 0, OUT_F32 = 1, OUT_F32_ACC = 2 };

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t nbytes(int64_t rows, int64_t cols) { return fp8_operand_bytes(rows, cols); }
int64_t nbytes_whole(int64_t rows, int64_t cols) { return nbytes(rows, cols) + fp8_plain_scale_bytes(rows, cols); }

// straight from the allocator: the way through the dispatcher takes as long again
Tensor fresh(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}
Tensor bytes(int64_t n, const Tensor& like) { return fresh({n}, at::kByte, like); }
char* ptr(const Tensor& t) { return t.defined() ? static_cast<char*>(t.data_ptr()) : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// [M, N] whose rows start on 32 bytes (what the vector stores of the product want)
Tensor alloc_rows(int64_t M, int64_t N, at::ScalarType dtype, const Tensor& like) {
  const int64_t per32 = dtype == at::kBFloat16 ? 16 : 8;
  if (N % per32 == 0) return fresh({M, N}, dtype, like);
  return fresh({M, up(N, per32)}, dtype, like).narrow(1, 0, N);
}
Tensor matrix(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }
Tensor rows2d(const Tensor& t) {
  if (t.dim() == 2) return matrix(t);
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  return matrix(t.reshape({rows, t.size(-1)}));
}
Tensor unit_stride(const Tensor& w) { return w.size(0) <= 1 || w.stride(0) == 1 ? w : w.contiguous(); }
int fp32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
int out_kind(at::ScalarType t) { return t == at::kFloat ? OUT_F32 : OUT_BF16; }
Tensor shaped(const Tensor& y, at::IntArrayRef x_shape) {
  if (x_shape.size() == 2) return y;
  std::vector<int64_t> shape(x_shape.begin(), x_shape.end());
  shape.back() = y.size(1);
  return y.reshape(shape);
}

// Whether the product quantises its bf16 rows itself (rows whose transpose nobody needs): every tile of 128 columns
// does it for its share of K, in series, so for few rows of moderate length.  Back to back, against two kernels that
// overlap: one row, K = 1024, N = 7168: 5.0 us against 5.4; 16 rows, K = 3584, N = 1024: 5.2 against 5.4; 24 rows: 6.6
// against 5.7; 16 rows, K = N = 4096: 7.6 against 6.9, with K = 6144, N = 2048 6.9 against 6.7.  And one launch less.
bool quantised_within(int64_t M, int64_t K) { return M <= 16 && K <= 4096; }

// ---------------------------------------------------------------------------------------------------------------
// weights: a parameter to convert in the call, or 8-bit forms that the caller keeps
// ---------------------------------------------------------------------------------------------------------------
struct Weight {
  Tensor w;          // parameter (or undefined)
  Tensor wq, wt;     // buffers of the 8-bit weight and of its transpose (or undefined)
  int64_t N;
};

struct Forward {
  Tensor y, xt, wt;        // transposed forms that the gradients read: xt at the start of its buffer,
  int64_t wt_off = 0;      // wt at wt_off bytes of its
  Tensor h, rstd;
};

// x [M, K] rows (or xq: their 8-bit form, rows M of K), or norm(x + resid) with wn
Forward forward(const Tensor& x, const Tensor& xq, int64_t M, int64_t K, const Weight& wt, bool need_wt, bool need_xt,
                at::ScalarType dtype, int64_t status, const Tensor* resid, const Tensor* wn, double eps, double off,
                bool need_rstd) {
  const Tensor& like = x.defined() ? x : xq;
  const int64_t N = wt.N;
  Forward f;
  f.y = alloc_rows(M, N, dtype, like);
  const bool has_resid = resid && resid->defined();
  if (wn) {
    f.h = has_resid ? fresh({M, K}, x.scalar_type(), x) : x;
    if (need_rstd) f.rstd = fresh({M}, at::kFloat, x);
  }
  if (M == 0 || N == 0 || K == 0) {
    f.y.zero_();
    if (has_resid && M && K) at::add_out(f.h, x, *resid);   // no columns in y: the sum is a result all the same
    return f;
  }
  const bool convert = !wt.wq.defined();
  const Tensor w = convert ? matrix(wt.w) : Tensor();
  const bool within = !wn && x.defined() && !need_xt && x.scalar_type() == at::kBFloat16 && quantised_within(M, K);
  const int64_t xq_n = xq.defined() || within ? 0 : nbytes(M, K), wq_n = convert ? nbytes(N, K) : 0;
  const int64_t xt_n = need_xt ? nbytes(K, M) : 0, wt_n = need_wt && convert ? nbytes(K, N) : 0;
  Tensor temp, keep;
  if (xq_n + wq_n) temp = bytes(xq_n + wq_n, like);
  if (xt_n + wt_n) keep = bytes(xt_n + wt_n, like);
  if (need_xt) f.xt = keep;
  if (need_wt) f.wt = convert ? keep : wt.wt, f.wt_off = convert ? xt_n : 0;
  char* xq_ptr = xq_n ? ptr(temp) : ptr(xq);
  char* wq_ptr = convert ? ptr(temp) + xq_n : ptr(wt.wq);
  char* wt_ptr = wt_n ? ptr(keep) + xt_n : nullptr;
  int* st = reinterpret_cast<int*>(status);
  if (wn) {
    check(fn.norm_linear_fwd(ptr(x), x.stride(0), has_resid ? ptr(*resid) : nullptr, has_resid ? resid->stride(0) : 0,
                             ptr(*wn), has_resid ? ptr(f.h) : nullptr, reinterpret_cast<float*>(ptr(f.rstd)), eps, off,
                             ptr(w), convert && fp32(w), convert ? w.stride(0) : 0, M, N, K, xq_ptr, wq_ptr, wt_ptr,
                             ptr(f.y), std::max<int64_t>(f.y.stride(0), N), out_kind(dtype), st, stream_of(like)),
          "cvb_fp8_norm_linear_fwd");
    count_launches(2 + convert);
  } else {
    check(fn.linear_fwd(ptr(x), x.defined() && fp32(x), x.defined() ? x.stride(0) : 0, ptr(w), convert && fp32(w),
                        convert ? w.stride(0) : 0, M, N, K, xq_ptr, need_xt ? ptr(keep) : nullptr, wq_ptr, wt_ptr,
                        ptr(f.y), std::max<int64_t>(f.y.stride(0), N), out_kind(dtype), st, stream_of(like)),
          "cvb_fp8_linear_fwd");
    count_launches(1 + (x.defined() && !within) + convert);
  }
  return f;
}

// ---------------------------------------------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------------------------------------------
// the parameter's fp32 main_grad, or undefined; the caller holds the GIL
Tensor main_grad(const Tensor& w) {
  if (!w.defined()) return Tensor();
  auto owner = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(w));
  auto attr = pybind11::getattr(owner, "main_grad", pybind11::none());
  if (attr.is_none()) return Tensor();
  Tensor m = attr.cast<Tensor>();
  TORCH_CHECK_TYPE(m.scalar_type() == at::kFloat && m.is_contiguous() && m.device() == w.device() && m.numel() == w.numel(),
                   "main_grad is a contiguous float32 tensor of the parameter's size on its device");
  return m;
}

Tensor gradient_rows(const Tensor& dy) {
  TORCH_CHECK_TYPE(dy.scalar_type() == at::kBFloat16 || dy.scalar_type() == at::kFloat,
                   "gradient of an 8-bit linear layer: bfloat16 or float32 is wanted, got ", dy.scalar_type());
  return rows2d(dy);
}

// results that raise when somebody differentiates them again
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list fake;
  for (auto& g : grads) fake.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "an 8-bit linear layer is once_differentiable: it has no second derivative", static_cast<int64_t>(fake.size()));
  return (*error)(std::move(fake));
}

struct Sizes {
  int64_t M, N, K, grad_fmt, wt_off, status;
  void save(AutogradContext* ctx) const { ctx->saved_data["sizes"] = std::vector<int64_t>{M, N, K, grad_fmt, wt_off, status}; }
  explicit Sizes(AutogradContext* ctx) {
    const auto v = ctx->saved_data["sizes"].toIntVector();
    M = v[0], N = v[1], K = v[2], grad_fmt = v[3], wt_off = v[4], status = v[5];
  }
  Sizes(int64_t m, int64_t n, int64_t k, int64_t g, int64_t o, int64_t s) : M(m), N(n), K(k), grad_fmt(g), wt_off(o), status(s) {}
  bool empty() const { return M == 0 || N == 0 || K == 0; }
};

// where a weight gradient [N, K] goes
struct WeightGrad {
  Tensor target, result;     // result: what autograd gets (undefined where a main_grad took it)
  int kind = 0;
  WeightGrad(const Tensor& w, const Sizes& z) {
    if (!w.defined()) return;
    pybind11::gil_scoped_acquire gil;
    const Tensor m = main_grad(w);
    target = m.defined() ? m.view({z.N, z.K}) : alloc_rows(z.N, z.K, w.scalar_type(), w);
    if (!m.defined()) result = target;
    kind = m.defined() ? OUT_F32_ACC : out_kind(w.scalar_type());
  }
  int64_t stride(const Sizes& z) const { return target.defined() ? std::max<int64_t>(target.stride(0), z.K) : 0; }
};

void count_from_backward(long n) {
  pybind11::gil_scoped_acquire gil;
  count_launches(n);
}

// launches of the products of a backward pass
long products(const Sizes& z, bool dx, bool dw) { return dx && dw ? fn.gemm_grads_launches(z.M, z.N, z.K) : dx + dw; }

Tensor some(const OptTensor& t) { return t ? *t : Tensor(); }

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_in, const OptTensor& wq,
                        const OptTensor& wt, int64_t N, int64_t grad_fmt, int64_t status, bool need_dx, bool need_dw) {
    const Tensor w = some(w_in);
    const Tensor x2 = rows2d(x);
    const int64_t M = x2.size(0), K = x2.size(1);
    Forward f = ::forward(x2, Tensor(), M, K, {w, some(wq), some(wt), N}, need_dx, need_dw, x.scalar_type(), status, nullptr, nullptr,
                          0, 0, false);
    // what the gradients read: x^T and w^T in 8 bits, half of what the bf16 layer keeps of x
    ctx->save_for_backward({need_dw ? w : Tensor(), f.xt, f.wt});
    Sizes(M, N, K, grad_fmt, f.wt_off, status).save(ctx);
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["needs"] = std::vector<int64_t>{need_dx, need_dw, static_cast<int64_t>(x.scalar_type())};
    return shaped(f.y, x.sizes());
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &w = saved[0], &xt = saved[1], &wt = saved[2];
    const Sizes z(ctx);
    const auto needs = ctx->saved_data["needs"].toIntVector();
    const auto dtype = static_cast<at::ScalarType>(needs[2]);
    variable_list out(9);
    {
      at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard guard(grads[0].device());
      const Tensor dy = gradient_rows(grads[0]);
      Tensor dx = needs[0] ? alloc_rows(z.M, z.K, dtype, dy) : Tensor();
      const WeightGrad g(needs[1] ? w : Tensor(), z);
      if (z.empty()) {
        if (dx.defined()) dx.zero_();
        if (g.result.defined()) g.target.zero_();
      } else {
        const int64_t dyq_n = needs[0] ? nbytes(z.M, z.N) : 0;
        const Tensor temp = bytes(dyq_n + (needs[1] ? nbytes(z.N, z.M) : 0), dy);
        check(fn.linear_bwd(ptr(dy), fp32(dy), dy.stride(0), z.grad_fmt, z.M, z.N, z.K, ptr(temp), ptr(temp) + dyq_n,
                            needs[0] ? ptr(wt) + z.wt_off : nullptr, ptr(xt), nullptr, 0, nullptr, nullptr, 0.f, ptr(dx),
                            needs[0] ? std::max<int64_t>(dx.stride(0), z.K) : 0, out_kind(dtype), ptr(g.target),
                            g.stride(z), g.kind, reinterpret_cast<int*>(z.status), stream_of(dy)),
              "cvb_fp8_linear_bwd");
        count_from_backward(1 + products(z, needs[0], needs[1]));
      }
      const auto shape = ctx->saved_data["shape"].toIntVector();
      if (dx.defined()) out[0] = shape.size() == 2 ? dx : dx.reshape(shape);
      out[1] = g.result;
    }
    return once(std::move(out));
  }
};

struct NormLinearFn : torch::autograd::Function<NormLinearFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& resid_in, const Tensor& wn,
                               const OptTensor& w_in, const OptTensor& wq, const OptTensor& wt, int64_t N, double eps,
                               double off, int64_t grad_fmt, int64_t status, bool need_x, bool need_r, bool need_wn,
                               bool need_dw) {
    const Tensor resid = some(resid_in), w = some(w_in);
    const bool need_dn = need_x || need_r || need_wn;
    const Tensor x2 = rows2d(x), r2 = resid.defined() ? rows2d(resid) : Tensor(), wn1 = unit_stride(wn);
    const int64_t M = x2.size(0), K = x2.size(1);
    Forward f = ::forward(x2, Tensor(), M, K, {w, some(wq), some(wt), N}, need_dn, false, x.scalar_type(), status, &r2, &wn1, eps, off, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({f.h, f.rstd, wn, need_dw ? w : Tensor(), f.wt});
    Sizes(M, N, K, grad_fmt, f.wt_off, status).save(ctx);
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["needs"] = std::vector<int64_t>{need_x, need_r, need_wn, need_dw};
    ctx->saved_data["off"] = off;
    variable_list out{shaped(f.y, x.sizes())};
    if (resid.defined()) out.push_back(x.dim() == 2 ? f.h : f.h.view(x.sizes()));
    return out;
  }

  // The norm's result is formed again from h and rstd while its transpose is quantised: it is never stored.  Its
  // gradient stays fp32 between the product and the norm's backward.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &rstd = saved[1], &wn = saved[2], &w = saved[3], &wt = saved[4];
    const Sizes z(ctx);
    const auto needs = ctx->saved_data["needs"].toIntVector();
    const bool need_dn = needs[0] || needs[1] || needs[2], need_dw = needs[3], need_wn = needs[2];
    const float off = static_cast<float>(ctx->saved_data["off"].toDouble());
    variable_list out(15);
    {
      at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard guard(h.device());
      const Tensor dy = grads[0].defined() ? gradient_rows(grads[0]) : at::zeros({z.M, z.N}, h.options());
      const Tensor dh = grads.size() > 1 && grads[1].defined() && need_dn ? rows2d(grads[1].to(h.scalar_type())) : Tensor();
      const WeightGrad g(need_dw ? w : Tensor(), z);
      Tensor wn_main, dwn, dx;
      if (need_wn) {
        pybind11::gil_scoped_acquire gil;
        wn_main = main_grad(wn);
        if (!wn_main.defined()) dwn = fresh({z.K}, wn.scalar_type(), wn);
      }
      if (need_dn) dx = fresh({z.M, z.K}, h.scalar_type(), h);
      if (z.empty()) {      // no rows, or no columns in y: only dh is left
        if (dx.defined()) dh.defined() ? dx.copy_(dh) : dx.zero_();
        if (dwn.defined()) dwn.zero_();
        if (g.result.defined()) g.target.zero_();
      } else {
        const Tensor wn1 = unit_stride(wn);
        // one workspace: dy in both forms, the norm's result transposed, its gradient, and the parts of dwn
        const int64_t dyq_n = need_dn ? nbytes(z.M, z.N) : 0, dyt_n = need_dw ? nbytes(z.N, z.M) : 0;
        const int64_t xt_n = need_dw ? nbytes(z.K, z.M) : 0, head = up(dyq_n + dyt_n + xt_n, 32);
        const int64_t lddn = up(z.K, 8), dn_n = need_dn ? z.M * lddn * 4 : 0;
        const int64_t parts = need_wn ? std::min<int64_t>(z.M, fn.norm_bwd_parts()) : 0;
        const Tensor temp = bytes(head + dn_n + parts * z.K * 4, dy);
        char* base = ptr(temp);
        check(fn.norm_linear_bwd(ptr(dy), fp32(dy), dy.stride(0), z.grad_fmt, z.M, z.N, z.K, base, base + dyq_n,
                                 need_dn ? ptr(wt) + z.wt_off : nullptr, base + dyq_n + dyt_n, ptr(h), h.stride(0),
                                 reinterpret_cast<const float*>(ptr(rstd)), ptr(wn1), off,
                                 reinterpret_cast<float*>(base + head), lddn, ptr(g.target), g.stride(z), g.kind, ptr(dh),
                                 dh.defined() ? dh.stride(0) : 0, ptr(dx),
                                 need_wn ? reinterpret_cast<float*>(base + head + dn_n) : nullptr,
                                 reinterpret_cast<float*>(ptr(wn_main)), ptr(dwn), reinterpret_cast<int*>(z.status),
                                 stream_of(dy)),
              "cvb_fp8_norm_linear_bwd");
        count_from_backward(1 + products(z, need_dn, need_dw) + need_dn + need_dw + need_wn);
      }
      if (dx.defined()) {
        const auto shape = ctx->saved_data["shape"].toIntVector();
        if (shape.size() != 2) dx = dx.view(shape);
        if (needs[0]) out[0] = dx;
        if (needs[1]) out[1] = dx;
      }
      out[2] = dwn;
      out[3] = g.result;
    }
    return once(std::move(out));
  }
};

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// ---------------------------------------------------------------------------------------------------------------
// what Python calls
// ---------------------------------------------------------------------------------------------------------------
Tensor linear(const Tensor& x, const OptTensor& w, const OptTensor& wq, const OptTensor& wt, int64_t N, int64_t grad_fmt,
              int64_t status) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor wp = some(w);
  const bool grad = at::GradMode::is_enabled(), need_dx = grad && x.requires_grad(), need_dw = grad && wants_grad(wp);
  if (need_dx || need_dw) {
    TORCH_CHECK_VALUE(!need_dx || !wq || wt, "linear_fp8: the gradient of the input needs the transposed 8-bit weight");
    return LinearFn::apply(x, w, wq, wt, N, grad_fmt, status, need_dx, need_dw);
  }
  at::NoGradGuard no_grad;
  const Tensor x2 = rows2d(x);
  return shaped(::forward(x2, Tensor(), x2.size(0), x2.size(1), {wp, some(wq), Tensor(), N}, false, false,
                          x.scalar_type(), status, nullptr, nullptr, 0, 0, false).y, x.sizes());
}

// the rows come in 8 bits: the buffer of an [M, K] e4m3 matrix
Tensor linear_rows8(const Tensor& xq, int64_t M, int64_t K, const OptTensor& w, const OptTensor& wq, int64_t N, int64_t status) {
  const c10::cuda::CUDAGuard guard(xq.device());
  at::NoGradGuard no_grad;
  return ::forward(Tensor(), xq, M, K, {some(w), some(wq), Tensor(), N}, false, false, at::kBFloat16, status, nullptr,
                   nullptr, 0, 0, false).y;
}

variable_list norm_linear(const Tensor& x, const OptTensor& resid, const Tensor& wn, const OptTensor& w, const OptTensor& wq,
                          const OptTensor& wt, int64_t N, double eps, double off, int64_t grad_fmt, int64_t status) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor wp = some(w), r = some(resid);
  const bool grad = at::GradMode::is_enabled(), need_x = grad && x.requires_grad(), need_r = grad && wants_grad(r);
  const bool need_wn = grad && wn.requires_grad(), need_dw = grad && wants_grad(wp), need_dn = need_x || need_r || need_wn;
  if (need_dn || need_dw) {
    TORCH_CHECK_VALUE(!need_dn || !wq || wt,
                      "add_rmsnorm_linear_fp8: the gradient of the input needs the transposed 8-bit weight");
    return NormLinearFn::apply(x, resid, wn, w, wq, wt, N, eps, off, grad_fmt, status, need_x, need_r, need_wn, need_dw);
  }
  at::NoGradGuard no_grad;
  const Tensor x2 = rows2d(x), r2 = r.defined() ? rows2d(r) : Tensor(), wn1 = unit_stride(wn);
  Forward f = ::forward(x2, Tensor(), x2.size(0), x2.size(1), {wp, some(wq), Tensor(), N}, false, false, x.scalar_type(),
                        status, &r2, &wn1, eps, off, false);
  variable_list out{shaped(f.y, x.sizes())};
  if (r.defined()) out.push_back(x.dim() == 2 ? f.h : f.h.view(x.sizes()));
  return out;
}

// (buffer of the row form, buffer of the transposed form) by the bits of `mode`; buffers hold the plain scales too
std::pair<OptTensor, OptTensor> quantize(const Tensor& x_in, int64_t fmt, int64_t mode) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  at::NoGradGuard no_grad;
  const Tensor x = matrix(x_in);
  const int64_t R = x.size(0), C = x.size(1);
  OptTensor q, t;
  char *qp = nullptr, *tp = nullptr;
  if (mode & ROWS) q = bytes(nbytes_whole(R, C), x), qp = ptr(*q);
  if (mode & COLS) t = bytes(nbytes_whole(C, R), x), tp = ptr(*t);
  if (R && C) {
    check(fn.quantize(ptr(x), fp32(x), R, C, x.stride(0), fmt, mode, qp, qp ? qp + fp8_code_bytes(R, C) : nullptr,
                      qp ? qp + nbytes(R, C) : nullptr, fp8_row_bytes(C), tp, tp ? tp + fp8_code_bytes(C, R) : nullptr,
                      tp ? tp + nbytes(C, R) : nullptr, fp8_row_bytes(R), nullptr, nullptr, 0.f, 0, stream_of(x)),
          "cvb_fp8_quantize");
    count_launches(1);
  }
  return {q, t};
}

// The codes (fmt 0, 1) or plain scales (fmt 2) of a [rows, cols] matrix as a view of its buffer, without the two calls
// through the dispatcher that a view of another type takes from Python.
Tensor view8(const Tensor& buf, int64_t rows, int64_t cols, int64_t fmt) {
  constexpr at::ScalarType types[] = {at::kFloat8_e4m3fn, at::kFloat8_e5m2, at::kFloat8_e8m0fnu};
  TORCH_CHECK_VALUE(fmt >= 0 && fmt < 3 && rows >= 0 && cols >= 0 && buf.scalar_type() == at::kByte &&
                        buf.numel() == nbytes_whole(rows, cols),
                    "not a buffer of a [", rows, ", ", cols, "] matrix");
  Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()), buf.key_set(),
                                                      c10::scalarTypeToTypeMeta(types[fmt]));
  const int64_t width = fmt == 2 ? up(cols, 128) / 128 : cols, ld = fmt == 2 ? width : fp8_row_bytes(cols);
  const int64_t sizes[] = {rows, width}, strides[] = {ld, 1};
  v.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides, buf.storage_offset() + (fmt == 2 ? nbytes(rows, cols) : 0));
  return v;
}

// (buffer of the 8-bit rows, x + resid or None)
std::pair<Tensor, OptTensor> norm(const Tensor& x_in, const OptTensor& resid, const Tensor& w, double eps, double off, int64_t fmt) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  at::NoGradGuard no_grad;
  const Tensor x = rows2d(x_in), r = resid ? rows2d(*resid) : Tensor(), wn = unit_stride(w);
  const int64_t R = x.size(0), D = x.size(1);
  const Tensor q = bytes(nbytes_whole(R, D), x);
  const Tensor h = r.defined() ? fresh({R, D}, x.scalar_type(), x) : Tensor();
  if (R) {
    check(fn.add_rmsnorm(ptr(x), x.stride(0), ptr(r), r.defined() ? r.stride(0) : 0, ptr(wn), ptr(h), ptr(q),
                         ptr(q) + fp8_code_bytes(R, D), ptr(q) + nbytes(R, D), fp8_row_bytes(D), nullptr, R, D, fmt, eps, off, 0,
                         stream_of(x)),
          "cvb_fp8_add_rmsnorm");
    count_launches(1);
  }
  OptTensor out;
  if (h.defined()) out = x_in.dim() == 2 ? h : h.view(x_in.sizes());
  return {q, out};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("linear", &linear);
  m.def("linear_rows8", &linear_rows8);
  m.def("norm_linear", &norm_linear);
  m.def("quantize", &quantize);
  m.def("norm", &norm);
  m.def("view8", &view8);
}
