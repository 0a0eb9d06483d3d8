// extern "C" entry points of the Linear layer in 16 bits (declared in include/cudeep_amd.h).  Every
// argument is checked on the host before any launch, nothing throws, and scratch is the caller's
// workspace or allocated stream-ordered.
#include "capi_checks.hpp"
#include "linear16.hpp"

using namespace cdx::checks;
using cdx::Linear16Kind;

namespace {

bool half_dtype(int d) { return d == CDX_DTYPE_F16 || d == CDX_DTYPE_BF16; }

int check_layer(const char* fn, int64_t M, int64_t N, int64_t K, int epilogue, int dtype, int other,
                const char* other_name) {
    if (bad_dim(M) || bad_dim(N) || bad_dim(K)) return bad(fn, "dimensions must be in [0, 2^40]");
    if (!half_dtype(dtype)) return bad(fn, "dtype must be float16 or bfloat16");
    if (other != dtype && other != CDX_DTYPE_F32)
        return bad(fn, (std::string(other_name) + " must be dtype or float32").c_str());
    if (!gemm_epilogue(epilogue)) return bad(fn, "unknown epilogue");
    return CDX_OK;
}

// Result `out` of a product must not touch `in`, which other workgroups still read.
int check_apart(const char* fn, const char* what, const Span& out, const Span& in) {
    return overlap(out, in) ? bad(fn, (std::string(what) + " overlap").c_str()) : (int)CDX_OK;
}

// Sizes that no checked call has (the queries come without one).
bool no_layer(int64_t M, int64_t N, int64_t K) {
    return bad_dim(M) || bad_dim(N) || bad_dim(K) || too_large(M, N) || too_large(M, K) || too_large(N, K);
}

// A vector's bytes as a row.
Span vector_span(const void* p, int64_t n, int dtype) { return {p, n, 1, n, dtype}; }

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

size_t slope_bytes(int64_t M, int64_t N, int epilogue) {
    if (epilogue == CDX_EPI_NONE) return 0;
    return round256((size_t)M * (size_t)(cdx::ceil_div(N, (int64_t)8) * 8) * 2);
}

// Whether dz is rounded (without an activation, and with ReLU, it is grad_out's own values and zeros): the bias
// gradient is summed beside the slopes then.
bool rounds_slope(int epilogue) { return epilogue != CDX_EPI_NONE && epilogue != CDX_EPI_RELU; }

size_t slope_sums_bytes(int64_t M, int64_t N, int epilogue) {
    return rounds_slope(epilogue) ? round256(cdx::linear16_slope_sums_workspace(M, N)) : 0;
}

}  // namespace

extern "C" {

size_t cdx_linear16_workspace_size(int64_t M, int64_t N, int64_t K) {
    if (no_layer(M, N, K)) return 0;
    return cdx::linear16_workspace(Linear16Kind::Forward, M, N, K, false);
}

size_t cdx_linear16_call_workspace_size(int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx,
                                        const void* weight, int64_t ldw) {
    if (no_layer(M, N, K)) return 0;
    return cdx::linear16_workspace(Linear16Kind::Forward, M, N, K,
                                   cdx::linear16_aligned(Linear16Kind::Forward, M, N, x, ldx, weight, ldw), false);
}

int cdx_linear16(int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const void* weight,
                 int64_t ldw, const void* bias, int bias_dtype, const void* residual, int64_t ldr,
                 void* y, int64_t ldy, void* z, int64_t ldz, int epilogue, int dtype,
                 void* workspace, size_t workspace_bytes, hipStream_t stream) {
    static const char fn[] = "cdx_linear16";
    int st = check_layer(fn, M, N, K, epilogue, dtype, bias ? bias_dtype : dtype, "bias_dtype");
    if (!st) st = check_matrix(fn, "x", x, ldx, M, K);
    if (!st) st = check_matrix(fn, "weight", weight, ldw, N, K);
    if (!st) st = check_matrix(fn, "y", y, ldy, M, N);
    if (!st && residual) st = check_matrix(fn, "residual", residual, ldr, M, N);
    if (!st && z) st = check_matrix(fn, "z", z, ldz, M, N);
    if (!st) st = check_workspace(fn, workspace);
    if (st || M == 0 || N == 0) return st;
    const Span sx{x, ldx, M, K, dtype}, sw{weight, ldw, N, K, dtype}, sy{y, ldy, M, N, dtype};
    st = check_apart(fn, "y and x", sy, sx);
    if (!st) st = check_apart(fn, "y and weight", sy, sw);
    if (!st && bias) st = check_apart(fn, "y and bias", sy, vector_span(bias, N, bias_dtype));
    if (!st && residual) st = check_in_place(fn, "y and residual", sy, {residual, ldr, M, N, dtype});
    if (!st && z) {
        const Span sz{z, ldz, M, N, dtype};
        st = check_apart(fn, "z and y", sz, sy);
        if (!st) st = check_apart(fn, "z and x", sz, sx);
        if (!st) st = check_apart(fn, "z and weight", sz, sw);
        if (!st && bias) st = check_apart(fn, "z and bias", sz, vector_span(bias, N, bias_dtype));
        if (!st && residual) st = check_apart(fn, "z and residual", sz, {residual, ldr, M, N, dtype});
    }
    if (st) return st;
    cdx::Linear16Product p{M, N, K, x, ldx, weight, ldw, dtype, {}};
    p.out.y = y; p.out.ldy = ldy;
    p.out.z = z; p.out.ldz = ldz;
    p.out.residual = residual; p.out.ldr = ldr;
    p.out.bias = bias; p.out.bias_f32 = bias_dtype == CDX_DTYPE_F32;
    p.out.act = epilogue;
    return with_workspace(fn, cdx_linear16_call_workspace_size(M, N, K, x, ldx, weight, ldw), workspace, workspace_bytes, stream,
                          [&](void* ws) {
                              return cdx::launch_linear16(Linear16Kind::Forward, p, false, nullptr, ws, stream);
                          });
}

size_t cdx_linear16_backward_workspace_size(int64_t M, int64_t N, int64_t K, int epilogue) {
    if (no_layer(M, N, K) || !gemm_epilogue(epilogue)) return 0;
    const size_t dx = cdx::linear16_workspace(Linear16Kind::Input, M, K, N, false);
    const size_t dw = cdx::linear16_workspace(Linear16Kind::Weight, N, K, M, true);
    return slope_bytes(M, N, epilogue) + slope_sums_bytes(M, N, epilogue) + (dx > dw ? dx : dw);
}

size_t cdx_linear16_backward_call_workspace_size(int64_t M, int64_t N, int64_t K, const void* grad_out, int64_t ldg,
                                                 const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                                 int epilogue, int input, int params, int bias) {
    if (no_layer(M, N, K) || !gemm_epilogue(epilogue)) return 0;
    // (dz in the workspace begins on 16 bytes, in rows of whole 8)
    const bool own = epilogue != CDX_EPI_NONE;
    const void* dz = own ? nullptr : grad_out;
    const int64_t lddz = own ? cdx::ceil_div(N, (int64_t)8) * 8 : ldg;
    const bool sums = bias && rounds_slope(epilogue);   // beside the slopes
    size_t dx = 0, dw = 0;
    if (input)
        dx = cdx::linear16_workspace(Linear16Kind::Input, M, K, N,
                                     cdx::linear16_aligned(Linear16Kind::Input, M, K, dz, lddz, weight, ldw), false);
    if (params)
        dw = cdx::linear16_workspace(Linear16Kind::Weight, N, K, M,
                                     cdx::linear16_aligned(Linear16Kind::Weight, N, K, dz, lddz, x, ldx), bias && !sums);
    if (!input && !params && !bias) return 0;
    return slope_bytes(M, N, epilogue) + (sums ? slope_sums_bytes(M, N, epilogue) : 0) + (dx > dw ? dx : dw);
}

int cdx_linear16_backward(int64_t M, int64_t N, int64_t K, const void* grad_out, int64_t ldg,
                          const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* z,
                          int64_t ldz, int epilogue, void* grad_x, int64_t ldgx, void* grad_weight,
                          void* grad_bias, int dtype, int param_dtype, void* workspace,
                          size_t workspace_bytes, hipStream_t stream) {
    static const char fn[] = "cdx_linear16_backward";
    int st = check_layer(fn, M, N, K, epilogue, dtype, param_dtype, "param_dtype");
    if (!st) st = check_matrix(fn, "grad_out", grad_out, ldg, M, N);
    if (!st && epilogue != CDX_EPI_NONE) st = check_matrix(fn, "z", z, ldz, M, N);
    if (!st && grad_weight) st = check_matrix(fn, "x", x, ldx, M, K);
    if (!st && grad_x) st = check_matrix(fn, "weight", weight, ldw, N, K);
    if (!st && grad_x) st = check_matrix(fn, "grad_x", grad_x, ldgx, M, K);
    if (!st && grad_weight) st = check_matrix(fn, "grad_weight", grad_weight, K, N, K);
    if (!st) st = check_workspace(fn, workspace);
    if (st) return st;
    if (grad_bias && !grad_weight && N > 0 && K > 0) return bad(fn, "grad_bias needs grad_weight");
    // grad_x is written first: everything that is read later has to be apart from it
    const NamedSpan reads[] = {{"grad_out", {grad_out, ldg, M, N, dtype}},
                               {"x", {x, ldx, M, grad_weight ? K : 0, dtype}},
                               {"weight", {weight, ldw, N, grad_x ? K : 0, dtype}},
                               {"z", {z, ldz, M, epilogue != CDX_EPI_NONE ? N : 0, dtype}}};
    const NamedSpan writes[] = {{"grad_x", {grad_x, ldgx, M, grad_x ? K : 0, dtype}},
                                {"grad_weight", {grad_weight, K, N, grad_weight ? K : 0, param_dtype}},
                                {"grad_bias", vector_span(grad_bias, grad_bias ? N : 0, param_dtype)}};
    st = check_results(fn, writes, reads);
    if (st) return st;
    const bool dx = grad_x && M > 0 && K > 0;
    const bool dw = N > 0 && ((grad_weight && K > 0) || grad_bias);
    if (!dx && !dw) return CDX_OK;
    // (a layer without inputs has a bias still: a product of one column that nobody stores, or the slopes' sums)
    if (M == 0) {   // empty sums
        if (grad_weight && K > 0) st = cdx::launch_zero(grad_weight, N * K, param_dtype, stream);
        if (!st && grad_bias) st = cdx::launch_zero(grad_bias, N, param_dtype, stream);
        return st;
    }
    return with_workspace(
        fn,
        cdx_linear16_backward_call_workspace_size(M, N, K, grad_out, ldg, x, ldx, weight, ldw, epilogue, dx,
                                                  grad_weight && K > 0, dw && grad_bias),
        workspace, workspace_bytes, stream,
        [&](void* ws) {
            const void* dz = grad_out;
            int64_t lddz = ldg;
            const bool f32 = param_dtype == CDX_DTYPE_F32;
            void* bias_sums = grad_bias;   // of the weight product
            uint8_t* part = static_cast<uint8_t*>(ws);
            if (epilogue != CDX_EPI_NONE && N > 0) {
                lddz = cdx::ceil_div(N, (int64_t)8) * 8;
                part += slope_bytes(M, N, epilogue);
                int e;
                if (grad_bias && rounds_slope(epilogue)) {   // (its parts are the workspace's too)
                    e = cdx::launch_linear16_slope_sums(grad_out, ldg, z, ldz, ws, lddz, M, N, dtype, epilogue, grad_bias,
                                                        f32, reinterpret_cast<float*>(part), stream);
                    bias_sums = nullptr;
                    part += slope_sums_bytes(M, N, epilogue);
                } else {
                    e = cdx::launch_linear16_slope(grad_out, ldg, z, ldz, ws, lddz, M, N, dtype, epilogue, stream);
                }
                if (e) return e;
                dz = ws;
            }
            if (dx) {
                cdx::Linear16Product p{M, K, N, dz, lddz, weight, ldw, dtype, {}};
                p.out.y = grad_x; p.out.ldy = ldgx;
                int e = cdx::launch_linear16(Linear16Kind::Input, p, false, nullptr, part, stream);
                if (e) return e;
            }
            if (!dw || (K == 0 && !bias_sums)) return (int)CDX_OK;
            cdx::Linear16Product p{N, K, M, dz, lddz, x, ldx, dtype, {}};
            p.out.y = grad_weight; p.out.ldy = K;
            return cdx::launch_linear16(Linear16Kind::Weight, p, f32, bias_sums, part, stream);
        });
}

}  // extern "C"

// Internal: the kernel of a product (kind 0 forward, 1 input gradient, 2 weight gradient; the product's own
// M, N and K) with operands that allow wide loads or not, and how many slices of k it takes.
extern "C" const char* cdxi_linear16_kernel(int kind, int64_t M, int64_t N, int64_t K, int aligned, int* slices) {
    return cdx::linear16_kernel_name((Linear16Kind)kind, M, N, K, aligned, slices);
}
