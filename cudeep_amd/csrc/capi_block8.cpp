// extern "C" entry points of layer norm and the 8-bit block-scaled operators
// (declared in include/cudeep_amd.h).  As in capi.cpp every argument is checked
// on the host before any launch, nothing throws, and scratch is the caller's
// workspace or allocated stream-ordered.
#include <cmath>

#include "block8.hpp"
#include "capi_checks.hpp"

using namespace cdx::checks;
using cdx::set_error;

namespace {

bool scale_type(int d) { return d == CDX_DTYPE_E8M0 || d == CDX_DTYPE_F32; }
bool activation(int a) { return a >= CDX_EPI_RELU && a <= CDX_ACT_LEAKY_RELU; }
int64_t blocks_of(int64_t n) { return cdx::ceil_div(n, (int64_t)cdx::b8::kBlock); }

// An 8-bit matrix argument.
int check_mat8(const char* fn, const char* name, const void* q, int64_t ldq, const void* s,
               int64_t lds, int scale_dtype, int tile_rows, int64_t rows, int64_t cols) {
    if (!scale_type(scale_dtype)) return bad(fn, "scales must be CDX_DTYPE_E8M0 or CDX_DTYPE_F32");
    if (tile_rows != 1 && tile_rows != cdx::b8::kBlock) return bad(fn, "tile_rows must be 1 or 128");
    int st = check_matrix(fn, name, q, ldq, rows, cols);
    if (st) return st;
    return check_matrix(fn, (std::string(name) + "'s scale").c_str(), s, lds,
                        tile_rows == 1 ? rows : blocks_of(rows), blocks_of(cols));
}

cdx::b8::Mat8 mat8(const void* q, int64_t ldq, const void* s, int64_t lds, int scale_dtype) {
    return {static_cast<const uint8_t*>(q), ldq, s, lds, scale_dtype == CDX_DTYPE_E8M0};
}

int check_norm(const char* fn, int64_t rows, int64_t dim, int dtype, int param_dtype) {
    if (bad_dim(rows) || dim < 1 || dim > kMaxDim) return bad(fn, "rows must be in [0, 2^40], dim in [1, 2^40]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    if (param_dtype != dtype && param_dtype != CDX_DTYPE_F32)
        return bad(fn, "param_dtype must be dtype or float32");
    return CDX_OK;
}

int check_product(const char* fn, int64_t M, int64_t N, int64_t K, const void* B, int64_t ldb,
                  const void* b_scale, int64_t ldsb, int b_scale_dtype, const void* C, int64_t ldc,
                  int c_dtype, int epilogue) {
    if (bad_dim(M) || bad_dim(N) || bad_dim(K)) return bad(fn, "dimensions must be in [0, 2^40]");
    if (!float_dtype(c_dtype)) return bad(fn, "c_dtype must be float32, float16 or bfloat16");
    if (!gemm_epilogue(epilogue)) return bad(fn, "unknown epilogue");
    int st = check_mat8(fn, "B", B, ldb, b_scale, ldsb, b_scale_dtype, cdx::b8::kBlock, N, K);
    if (st) return st;
    return check_matrix(fn, "C", C, ldc, M, N);
}

}  // namespace

extern "C" {

int cdx_layer_norm_forward(const void* x, int64_t ldx, const void* weight, const void* bias,
                           void* y, int64_t ldy, float* mean, float* rstd, int64_t rows,
                           int64_t dim, double eps, int dtype, int param_dtype,
                           hipStream_t stream) {
    static const char fn[] = "cdx_layer_norm_forward";
    int st = check_norm(fn, rows, dim, dtype, param_dtype);
    if (!st) st = check_matrix(fn, "x", x, ldx, rows, dim);
    if (!st) st = check_matrix(fn, "y", y, ldy, rows, dim);
    if (!st) st = check_in_place(fn, "y and x", {y, ldy, rows, dim, dtype}, {x, ldx, rows, dim, dtype});
    if (st) return st;
    if (!(eps >= 0.0) || !std::isfinite(eps)) return bad(fn, "eps must be finite and not negative");
    if (rows == 0) return CDX_OK;
    return cdx::launch_layer_norm(x, ldx, weight, bias, y, ldy, mean, rstd, rows, dim, (float)eps,
                                  dtype, param_dtype, stream);
}

size_t cdx_layer_norm_backward_workspace_size(int64_t rows, int64_t dim, int dtype) {
    if (bad_dim(rows) || dim < 1 || dim > kMaxDim || !float_dtype(dtype) || rows == 0) return 0;
    return cdx::layer_norm_partial_floats(rows, dim, dtype) * sizeof(float);
}

int cdx_layer_norm_backward(const void* grad_out, int64_t ldg, const void* x, int64_t ldx,
                            const void* weight, const float* mean, const float* rstd,
                            void* grad_in, int64_t ldgi, void* grad_weight, void* grad_bias,
                            int64_t rows, int64_t dim, int dtype, int param_dtype,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
    static const char fn[] = "cdx_layer_norm_backward";
    int st = check_norm(fn, rows, dim, dtype, param_dtype);
    if (!st) st = check_matrix(fn, "grad_out", grad_out, ldg, rows, dim);
    if (!st) st = check_matrix(fn, "x", x, ldx, rows, dim);
    if (!st) st = check_matrix(fn, "grad_in", grad_in, ldgi, rows, dim);
    const Span in{grad_in, ldgi, rows, dim, dtype};
    if (!st) st = check_in_place(fn, "grad_in and x", in, {x, ldx, rows, dim, dtype});
    if (!st) st = check_in_place(fn, "grad_in and grad_out", in, {grad_out, ldg, rows, dim, dtype});
    if (st) return st;
    if (rows == 0) {   // empty sums
        if (grad_weight) st = cdx::launch_zero(grad_weight, dim, param_dtype, stream);
        if (!st && grad_bias) st = cdx::launch_zero(grad_bias, dim, param_dtype, stream);
        return st;
    }
    if (!mean || !rstd) return bad(fn, "mean or rstd is NULL");
    const size_t need = grad_weight || grad_bias
        ? cdx_layer_norm_backward_workspace_size(rows, dim, dtype) : 0;
    return with_workspace(fn, need, workspace, workspace_bytes, stream, [&](void* ws) {
        return cdx::launch_layer_norm_backward(grad_out, ldg, x, ldx, weight, mean, rstd, grad_in,
                                               ldgi, grad_weight, grad_bias, rows, dim, dtype,
                                               param_dtype, static_cast<float*>(ws), stream);
    });
}

int cdx_quantize_e4m3(const void* x, int64_t ldx, int64_t rows, int64_t cols, int dtype,
                      int tile_rows, void* q, int64_t ldq, void* scale, int64_t lds,
                      int scale_dtype, hipStream_t stream) {
    static const char fn[] = "cdx_quantize_e4m3";
    if (bad_dim(rows) || bad_dim(cols)) return bad(fn, "dimensions must be in [0, 2^40]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    int st = check_matrix(fn, "x", x, ldx, rows, cols);
    if (!st) st = check_mat8(fn, "q", q, ldq, scale, lds, scale_dtype, tile_rows, rows, cols);
    if (st || rows == 0 || cols == 0) return st;
    uint8_t* codes = static_cast<uint8_t*>(q);
    const int e8m0 = scale_dtype == CDX_DTYPE_E8M0;
    if (tile_rows == 1)
        return cdx::launch_quantize_rows(x, ldx, rows, cols, dtype, codes, ldq, scale, lds, e8m0,
                                         nullptr, 0, CDX_EPI_NONE, 0.0f, stream);
    return cdx::launch_quantize_tiles(x, ldx, rows, cols, dtype, codes, ldq, scale, lds, e8m0,
                                      stream);
}

int cdx_dequantize_e4m3(const void* q, int64_t ldq, const void* scale, int64_t lds,
                        int scale_dtype, int tile_rows, void* out, int64_t ldo, int64_t rows,
                        int64_t cols, int dtype, hipStream_t stream) {
    static const char fn[] = "cdx_dequantize_e4m3";
    if (bad_dim(rows) || bad_dim(cols)) return bad(fn, "dimensions must be in [0, 2^40]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    int st = check_mat8(fn, "q", q, ldq, scale, lds, scale_dtype, tile_rows, rows, cols);
    if (!st) st = check_matrix(fn, "out", out, ldo, rows, cols);
    if (st || rows == 0 || cols == 0) return st;
    return cdx::launch_dequantize(mat8(q, ldq, scale, lds, scale_dtype), tile_rows, rows, cols, out,
                                  ldo, dtype, stream);
}

size_t cdx_gemm_e4m3_workspace_size(int64_t M, int64_t N, int64_t K) {
    if (bad_dim(M) || bad_dim(N) || bad_dim(K)) return 0;
    return cdx::gemm8_workspace(M, N, K, false);
}

int cdx_gemm_e4m3(int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* a_scale,
                  int64_t ldsa, int a_scale_dtype, const void* B, int64_t ldb, const void* b_scale,
                  int64_t ldsb, int b_scale_dtype, void* C, int64_t ldc, int c_dtype,
                  const float* bias, int epilogue, void* workspace, size_t workspace_bytes,
                  hipStream_t stream) {
    static const char fn[] = "cdx_gemm_e4m3";
    int st = check_product(fn, M, N, K, B, ldb, b_scale, ldsb, b_scale_dtype, C, ldc, c_dtype, epilogue);
    if (!st) st = check_mat8(fn, "A", A, lda, a_scale, ldsa, a_scale_dtype, 1, M, K);
    if (st || M == 0 || N == 0) return st;
    cdx::Gemm8Args g{M, N, K, mat8(A, lda, a_scale, ldsa, a_scale_dtype),
                     mat8(B, ldb, b_scale, ldsb, b_scale_dtype)};
    g.C = C; g.ldc = ldc; g.cdtype = c_dtype; g.bias = bias; g.epilogue = epilogue;
    return with_workspace(fn, cdx_gemm_e4m3_workspace_size(M, N, K), workspace, workspace_bytes,
                          stream, [&](void* ws) {
                              g.ws = ws;
                              return cdx::launch_gemm8(g, stream);
                          });
}

size_t cdx_linear_e4m3_workspace_size(int64_t M, int64_t N, int64_t K) {
    if (bad_dim(M) || bad_dim(N) || bad_dim(K)) return 0;
    return cdx::gemm8_workspace(M, N, K, true);
}

int cdx_linear_e4m3(int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, int x_dtype,
                    const void* B, int64_t ldb, const void* b_scale, int64_t ldsb,
                    int b_scale_dtype, void* C, int64_t ldc, int c_dtype, const float* bias,
                    int epilogue, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    static const char fn[] = "cdx_linear_e4m3";
    int st = check_product(fn, M, N, K, B, ldb, b_scale, ldsb, b_scale_dtype, C, ldc, c_dtype, epilogue);
    if (st) return st;
    if (!float_dtype(x_dtype)) return bad(fn, "x_dtype must be float32, float16 or bfloat16");
    st = check_matrix(fn, "x", x, ldx, M, K);
    if (st || M == 0 || N == 0) return st;
    cdx::Gemm8Args g{M, N, K, {}, mat8(B, ldb, b_scale, ldsb, b_scale_dtype)};
    g.x = x; g.ldx = ldx; g.xdtype = x_dtype;
    g.C = C; g.ldc = ldc; g.cdtype = c_dtype; g.bias = bias; g.epilogue = epilogue;
    const size_t need = cdx_linear_e4m3_workspace_size(M, N, K);
    const bool small = workspace && workspace_bytes < need;
    // (few rows: every workgroup reads all of x while others already write C)
    if (!small && overlap({C, ldc, M, N, c_dtype}, {x, ldx, M, K, x_dtype})) return bad(fn, "C overlaps x");
    return with_workspace(fn, need, workspace, workspace_bytes,
                          stream, [&](void* ws) {
                              g.ws = ws;
                              return cdx::launch_gemm8(g, stream);
                          });
}

int cdx_activation_forward_e4m3(const void* z, int64_t ldz, void* y, int64_t ldy, void* q,
                                int64_t ldq, void* scale, int64_t lds, int scale_dtype,
                                int64_t rows, int64_t cols, int dtype, int act, float alpha,
                                hipStream_t stream) {
    static const char fn[] = "cdx_activation_forward_e4m3";
    if (bad_dim(rows) || bad_dim(cols)) return bad(fn, "dimensions must be in [0, 2^40]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    if (!activation(act)) return bad(fn, "unknown activation");
    int st = check_matrix(fn, "z", z, ldz, rows, cols);
    if (!st) st = check_matrix(fn, "y", y, ldy, rows, cols);
    if (!st) st = check_mat8(fn, "q", q, ldq, scale, lds, scale_dtype, 1, rows, cols);
    if (!st) st = check_in_place(fn, "y and z", {y, ldy, rows, cols, dtype}, {z, ldz, rows, cols, dtype});
    if (st || rows == 0 || cols == 0) return st;
    return cdx::launch_quantize_rows(z, ldz, rows, cols, dtype, static_cast<uint8_t*>(q), ldq, scale,
                                     lds, scale_dtype == CDX_DTYPE_E8M0, y, ldy, act, alpha, stream);
}

int cdx_activation_backward_e4m3(const void* grad_out, int64_t ldg, const void* q, int64_t ldq,
                                 const void* scale, int64_t lds, int scale_dtype, void* grad_in,
                                 int64_t ldgi, int64_t rows, int64_t cols, int dtype, int act,
                                 float alpha, hipStream_t stream) {
    static const char fn[] = "cdx_activation_backward_e4m3";
    if (bad_dim(rows) || bad_dim(cols)) return bad(fn, "dimensions must be in [0, 2^40]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    if (!activation(act)) return bad(fn, "unknown activation");
    int st = check_matrix(fn, "grad_out", grad_out, ldg, rows, cols);
    if (!st) st = check_matrix(fn, "grad_in", grad_in, ldgi, rows, cols);
    if (!st) st = check_mat8(fn, "q", q, ldq, scale, lds, scale_dtype, 1, rows, cols);
    if (!st) st = check_in_place(fn, "grad_in and grad_out", {grad_in, ldgi, rows, cols, dtype},
                                 {grad_out, ldg, rows, cols, dtype});
    if (st || rows == 0 || cols == 0) return st;
    return cdx::launch_activation_backward8(grad_out, ldg, mat8(q, ldq, scale, lds, scale_dtype),
                                            rows, cols, grad_in, ldgi, dtype, act, alpha, stream);
}

size_t cdx_linear_weight_grad_e4m3_workspace_size(int64_t batch, int64_t out_features,
                                                  int64_t in_features, int dtype) {
    if (bad_dim(batch) || bad_dim(out_features) || bad_dim(in_features) || !float_dtype(dtype)) return 0;
    return cdx::wgrad8_workspace(batch, out_features, in_features, dtype, true);
}

int cdx_linear_weight_grad_e4m3(const void* dz, int64_t lddz, int dtype, const void* q, int64_t ldq,
                                const void* scale, int64_t lds, float* grad_weight,
                                float* grad_bias, int64_t batch, int64_t out_features,
                                int64_t in_features, void* workspace, size_t workspace_bytes,
                                hipStream_t stream) {
    static const char fn[] = "cdx_linear_weight_grad_e4m3";
    if (bad_dim(batch) || bad_dim(out_features) || bad_dim(in_features))
        return bad(fn, "dimensions must be in [0, 2^40]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    int st = check_matrix(fn, "dz", dz, lddz, batch, out_features);
    if (!st) st = check_mat8(fn, "x", q, ldq, scale, lds, CDX_DTYPE_E8M0, 1, batch, in_features);
    if (!st) st = check_matrix(fn, "grad_weight", grad_weight, in_features, out_features, in_features);
    if (st || out_features == 0) return st;
    if (batch == 0) {   // empty sums
        if (in_features > 0) st = cdx::launch_zero(grad_weight, out_features * in_features, CDX_DTYPE_F32, stream);
        if (!st && grad_bias) st = cdx::launch_zero(grad_bias, out_features, CDX_DTYPE_F32, stream);
        return st;
    }
    if (in_features == 0 && !grad_bias) return CDX_OK;
    const size_t need = cdx::wgrad8_workspace(batch, out_features, in_features, dtype, grad_bias != nullptr);
    return with_workspace(fn, need, workspace, workspace_bytes, stream, [&](void* ws) {
        return cdx::launch_wgrad8(dz, lddz, dtype, mat8(q, ldq, scale, lds, CDX_DTYPE_E8M0),
                                  grad_weight, grad_bias, batch, out_features, in_features, ws,
                                  stream);
    });
}

}  // extern "C"

// Internal: the kernel of cdx_gemm_e4m3, or with from_x of cdx_linear_e4m3 (`aligned`: rows of the
// 8-bit operands begin at 16-byte addresses), and the plan of
// cdx_linear_weight_grad_e4m3 as 1000 * (side of its tiles) + slices of the batch.
extern "C" const char* cdxi_gemm8_kernel(int from_x, int c_dtype, int64_t M, int64_t N, int64_t K,
                                         int aligned) {
    return cdx::gemm8_kernel_name(M, N, K, aligned, c_dtype == CDX_DTYPE_F32, from_x);
}
extern "C" int cdxi_wgrad8_plan(int64_t M, int64_t N, int64_t K) {
    int side = 0, slices = 0;
    cdx::wgrad8_plan(M, N, K, &side, &slices);
    return 1000 * side + slices;
}
