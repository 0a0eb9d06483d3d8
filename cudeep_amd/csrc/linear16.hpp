// A Linear layer in 16 bits (linear16_*.hip): operands, results and launchers.
#pragma once

#include "block8.hpp"

namespace cdx {

// What becomes of a row-major product's sums: z = sum + bias (kept in 16 bits where z is given),
// y = residual + act(z), rounded once.  Or, with `sums`, the fp32 sums themselves.
struct Linear16Out {
    void* y = nullptr; int64_t ldy = 0;
    void* z = nullptr; int64_t ldz = 0;
    const void* residual = nullptr; int64_t ldr = 0;
    const void* bias = nullptr; int bias_f32 = 0;
    int act = CDX_EPI_NONE;
    float* sums = nullptr;           // dense [M][N], slice s at sums + s * M * N
};

// The product sum_k A(m, k) B(n, k).  An operand's rows hold consecutive k (rows [extent][K]), or
// its columns do (kCols: rows [K][extent]).
struct Linear16Product {
    int64_t M, N, K;
    const void* a; int64_t lda;
    const void* b; int64_t ldb;
    int dtype;                       // CDX_DTYPE_F16 or _BF16: operands and 16-bit results
    Linear16Out out;
};

enum class Linear16Kind { Forward, Input, Weight };   // both rows; A rows, B columns; both columns

// Whether operands allow wide loads, which may choose the kernel.
bool linear16_aligned(Linear16Kind kind, int64_t M, int64_t N, const void* a, int64_t lda, const void* b, int64_t ldb);
// Bytes of partial sums that a product of this kind needs (0: none), with such operands or without; the larger of
// both.
size_t linear16_workspace(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned, bool col_sums);
size_t linear16_workspace(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool col_sums);
// col_y (Weight products; may be null): the column sums sum_k A(m, k).  out_f32: y, dense, and col_y
// hold fp32 instead of 16-bit values.
int launch_linear16(Linear16Kind kind, const Linear16Product& p, bool out_f32, void* col_y, void* ws,
                    hipStream_t stream);
// The kernel it runs (aligned: 16-byte rows and, for columns, extents of whole 8).
const char* linear16_kernel_name(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned,
                                 int* slices);

// dz = grad act'(z), all 16-bit [rows, cols].
int launch_linear16_slope(const void* grad, int64_t ldg, const void* z, int64_t ldz, void* dz,
                          int64_t lddz, int64_t rows, int64_t cols, int dtype, int act,
                          hipStream_t stream);
// The same for GELU, SiLU and sigmoid (the others' dz is exact), with `sums`[cols] = sum over rows of dz before its
// rounding, in 16 bits or fp32; part: the workspace's bytes.
size_t linear16_slope_sums_workspace(int64_t rows, int64_t cols);
int launch_linear16_slope_sums(const void* grad, int64_t ldg, const void* z, int64_t ldz, void* dz,
                               int64_t lddz, int64_t rows, int64_t cols, int dtype, int act, void* sums,
                               bool sums_f32, float* part, hipStream_t stream);

}  // namespace cdx
