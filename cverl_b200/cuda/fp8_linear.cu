// The launches of an 8-bit linear layer, forward and backward, each behind one call: a small layer spends more time in
// the calls than in the kernels (five ctypes calls of a 77-token layer's step took longer than its ten launches).
#include "fp8_launch.h"

namespace {
constexpr int E4M3 = 0;
enum { ROWS = 1, COLS = 2, BLOCKS = 4 };

struct Mat8 {      // [rows, cols] in a buffer; null buffer: absent
  char* codes;
  char* sf;
  long long ld;
  Mat8(void* buf, long long rows, long long cols) : codes(static_cast<char*>(buf)), sf(nullptr), ld(fp8_row_bytes(cols)) {
    if (codes) sf = codes + fp8_code_bytes(rows, cols);
  }
};

int quantize(const void* x, int x_fp32, long long rows, long long cols, long long stride, int fmt, int extra,
             const Mat8& q, const Mat8& t, int beside, void* stream) {
  const int mode = (q.codes ? ROWS : 0) | (t.codes ? COLS : 0) | extra;
  return cvb_fp8_quantize(x, x_fp32, rows, cols, stride, fmt, mode, q.codes, q.sf, nullptr, q.ld, t.codes, t.sf,
                          nullptr, t.ld, nullptr, nullptr, 0.f, beside, stream);
}
int product(const Mat8& a, int a_fmt, const Mat8& b, int b_fmt, int M, int N, int K, void* c, long long ldc,
            int out_kind, bool b_ready, int* status, void* stream) {
  return cvb_fp8_gemm(a.codes, a.sf, a.ld, a_fmt, b.codes, b.sf, b.ld, b_fmt, M, N, K, c, ldc, out_kind, b_ready, status,
                      stream);
}
}  // namespace

// y [M, N] = x [M, K] w [N, K]^T.  x null: `xq` holds its 8-bit form already.  w null: `wq` does.  `xt` and `wt`
// (both may be null) take the transposed forms that the backward pass reads.  xq null: up to 16 bf16 rows, quantised
// within the product.
extern "C" int cvb_fp8_linear_fwd(const void* x, int x_fp32, long long x_stride, const void* w, int w_fp32,
                                  long long w_stride, int M, int N, int K, void* xq, void* xt, void* wq, void* wt,
                                  void* y, long long ldy, int out_kind, int* status, void* stream) {
  const Mat8 mxq(xq, M, K), mxt(xt, K, M), mwq(wq, N, K), mwt(wt, K, N);
  int rc = 0;
  if (w && (rc = quantize(w, w_fp32, N, K, w_stride, E4M3, BLOCKS, mwq, mwt, 0, stream))) return rc;
  if (x && !xq) {
    if (x_fp32 || xt) return -1;
    return cvb_fp8_gemm_rows(x, x_stride, mwq.codes, mwq.sf, mwq.ld, E4M3, M, N, K, y, ldy, out_kind, status, stream);
  }
  if (x && (rc = quantize(x, x_fp32, M, K, x_stride, E4M3, 0, mxq, mxt, w != nullptr, stream))) return rc;
  return product(mxq, E4M3, mwq, E4M3, M, N, K, y, ldy, out_kind, x && !w, status,
                 stream);
}

// h = x + resid, y = norm(h) w^T; without resid, h is null and the norm reads x.
extern "C" int cvb_fp8_norm_linear_fwd(const void* x, long long x_stride, const void* resid, long long r_stride,
                                       const void* wn, void* h, float* rstd, float eps, float w_offset, const void* w,
                                       int w_fp32, long long w_stride, int M, int N, int K, void* xq, void* wq, void* wt,
                                       void* y, long long ldy, int out_kind, int* status, void* stream) {
  const Mat8 mxq(xq, M, K), mwq(wq, N, K), mwt(wt, K, N);
  int rc = 0;
  if (w && (rc = quantize(w, w_fp32, N, K, w_stride, E4M3, BLOCKS, mwq, mwt, 0, stream))) return rc;
  if ((rc = cvb_fp8_add_rmsnorm(x, x_stride, resid, r_stride, wn, h, mxq.codes, mxq.sf, nullptr, mxq.ld, rstd, M, K, E4M3,
                                eps, w_offset, w != nullptr, stream)))
    return rc;
  return product(mxq, E4M3, mwq, E4M3, M, N, K, y, ldy, out_kind, !w, status, stream);
}

// dx [M, K] = dy w (where wt is given) and dw [N, K] (+)= dy^T x (where dw is given).  `dyq` and `dyt` are workspaces
// for the two forms of dy.  h given: x is h * rstd * (w_offset + wn), formed into the workspace `xt`.
extern "C" int cvb_fp8_linear_bwd(const void* dy, int dy_fp32, long long dy_stride, int grad_fmt, int M, int N, int K,
                                  void* dyq, void* dyt, void* wt, void* xt, const void* h, long long h_stride,
                                  const float* rstd, const void* wn, float w_offset, void* dx, long long lddx,
                                  int dx_kind, void* dw, long long lddw, int dw_kind, int* status, void* stream) {
  const Mat8 mdq(wt ? dyq : nullptr, M, N), mdt(dw ? dyt : nullptr, N, M), mwt(wt, K, N), mxt(xt, K, M);
  if (!mdq.codes && !mdt.codes) return 0;
  int rc = quantize(dy, dy_fp32, M, N, dy_stride, grad_fmt, 0, mdq, mdt, 0, stream);
  if (rc) return rc;
  if (!dw) return product(mdq, grad_fmt, mwt, E4M3, M, K, N, dx, lddx, dx_kind, true, status, stream);
  if (h && (rc = cvb_fp8_quantize(h, 0, M, K, h_stride, E4M3, COLS, nullptr, nullptr, nullptr, 0, mxt.codes, mxt.sf,
                                  nullptr, mxt.ld,
                                  rstd, wn, w_offset, 1, stream)))
    return rc;
  if (!wt) return product(mdt, grad_fmt, mxt, E4M3, N, K, M, dw, lddw, dw_kind, false, status, stream);
  return cvb_fp8_gemm_grads(mdq.codes, mdq.sf, mdq.ld, mwt.codes, mwt.sf, mwt.ld, mdt.codes, mdt.sf, mdt.ld, mxt.codes,
                            mxt.sf, mxt.ld, grad_fmt, M, N, K, dx, lddx, dx_kind, dw, lddw, dw_kind, status, stream);
}

// The gradients of the norm + linear layer.  wt given: `dn` (fp32 [M, lddn], a workspace) takes the gradient of the
// norm's result, dx that of x + resid (with dh added), and dwn (or dwn_acc, +=) that of the norm's weight, by way of
// the workspace `part`.  dw given: as above, with the workspace `xt`.
extern "C" int cvb_fp8_norm_linear_bwd(const void* dy, int dy_fp32, long long dy_stride, int grad_fmt, int M, int N,
                                       int K, void* dyq, void* dyt, void* wt, void* xt, const void* h,
                                       long long h_stride, const float* rstd, const void* wn, float w_offset, float* dn,
                                       long long lddn, void* dw, long long lddw, int dw_kind, const void* dh,
                                       long long dh_stride, void* dx, float* part, float* dwn_acc, void* dwn, int* status,
                                       void* stream) {
  constexpr int F32 = 1;
  const int rc = cvb_fp8_linear_bwd(dy, dy_fp32, dy_stride, grad_fmt, M, N, K, dyq, dyt, wt, xt, h, h_stride, rstd, wn,
                                    w_offset, dn, lddn, F32, dw, lddw, dw_kind, status, stream);
  if (rc || !wt) return rc;
  return cvb_fp8_norm_bwd(dn, lddn, h, h_stride, wn, rstd, dh, dh_stride, dx, part, dwn_acc, dwn, M, K, w_offset, stream);
}
