// Launchers of the 8-bit operators: what the kernels define, what they call of each other, and what the torch extension
// calls through addresses of the loaded library.  One declaration for all of them, so that a changed argument does not
// compile where it is not followed.  Every launcher returns 0 or an error code; arguments are explained at the definitions.
#pragma once

// Buffer of an 8-bit matrix [rows, cols]: codes, row-major with rows padded to 16 bytes; the scale cells, 512 bytes per 128
// rows and 512 columns; and, in buffers that leave the extension, the scale bytes once more in plain order.
inline long long fp8_row_bytes(long long cols) { return (cols + 15) / 16 * 16; }
inline long long fp8_code_bytes(long long rows, long long cols) { return rows * fp8_row_bytes(cols); }
inline long long fp8_operand_bytes(long long rows, long long cols) {      // what the products read
  return fp8_code_bytes(rows, cols) + (rows + 127) / 128 * ((cols + 511) / 512) * 512;
}
inline long long fp8_plain_scale_bytes(long long rows, long long cols) { return rows * ((cols + 127) / 128); }

extern "C" {

// fp8_quant.cu
int cvb_fp8_quantize(const void* x, int x_fp32, long long rows, long long cols, long long x_stride, int fmt, int mode,
                     void* q, void* sf, void* ps, long long q_ld, void* qt, void* sft, void* pst, long long qt_ld,
                     const float* rstd, const void* w, float w_offset, int beside, void* stream);
int cvb_fp8_add_rmsnorm(const void* x, long long x_stride, const void* resid, long long r_stride, const void* w,
                        void* h, void* q, void* sf, void* ps, long long q_ld, float* rstd, long long rows, int D,
                        int fmt, float eps, float w_offset, int beside, void* stream);
int cvb_fp8_norm_bwd_parts();
int cvb_fp8_norm_bwd(const float* dn, long long dn_stride, const void* h, long long h_stride, const void* w,
                     const float* rstd, const void* dh, long long dh_stride, void* dx, float* part, float* dw_acc,
                     void* dw, long long rows, int D, float w_offset, void* stream);

// fp8_gemm.cu
int cvb_fp8_gemm(const void* a, const void* a_sf, long long lda, int a_fmt, const void* b, const void* b_sf,
                 long long ldb, int b_fmt, int M, int N, int K, void* c, long long ldc, int out_kind, int b_ready,
                 int* status, void* stream_v);
int cvb_fp8_gemm_rows(const void* x, long long x_stride, const void* b, const void* b_sf, long long ldb, int b_fmt,
                      int M, int N, int K, void* c, long long ldc, int out_kind, int* status, void* stream_v);
int cvb_fp8_gemm_grads(const void* dy, const void* dy_sf, long long ld_dy, const void* wt, const void* wt_sf,
                       long long ld_wt, const void* dyt, const void* dyt_sf, long long ld_dyt, const void* xt,
                       const void* xt_sf, long long ld_xt, int grad_fmt, int M, int N, int K, void* dx,
                       long long lddx, int dx_kind, void* dw, long long lddw, int dw_kind, int* status,
                       void* stream_v);
int cvb_fp8_gemm_grads_launches(int M, int N, int K);

// fp8_linear.cu
int cvb_fp8_linear_fwd(const void* x, int x_fp32, long long x_stride, const void* w, int w_fp32, long long w_stride,
                       int M, int N, int K, void* xq, void* xt, void* wq, void* wt, void* y, long long ldy,
                       int out_kind, int* status, void* stream);
int cvb_fp8_norm_linear_fwd(const void* x, long long x_stride, const void* resid, long long r_stride, const void* wn,
                            void* h, float* rstd, float eps, float w_offset, const void* w, int w_fp32,
                            long long w_stride, int M, int N, int K, void* xq, void* wq, void* wt, void* y,
                            long long ldy, int out_kind, int* status, void* stream);
int cvb_fp8_linear_bwd(const void* dy, int dy_fp32, long long dy_stride, int grad_fmt, int M, int N, int K, void* dyq,
                       void* dyt, void* wt, void* xt, const void* h, long long h_stride, const float* rstd,
                       const void* wn, float w_offset, void* dx, long long lddx, int dx_kind, void* dw,
                       long long lddw, int dw_kind, int* status, void* stream);
int cvb_fp8_norm_linear_bwd(const void* dy, int dy_fp32, long long dy_stride, int grad_fmt, int M, int N, int K,
                            void* dyq, void* dyt, void* wt, void* xt, const void* h, long long h_stride,
                            const float* rstd, const void* wn, float w_offset, float* dn, long long lddn, void* dw,
                            long long lddw, int dw_kind, const void* dh, long long dh_stride, void* dx, float* part,
                            float* dwn_acc, void* dwn, int* status, void* stream);

}  // extern "C"
