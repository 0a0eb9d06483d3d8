// Shared by layer norm and the 8-bit block-scaled kernels: element types,
// unaligned vector loads and stores, lane reductions, and the 8-bit format.
//
// The format: e4m3 values (OCP: 3 fraction bits, largest 448, no infinities,
// one NaN code of each sign) with a scale for each 128 columns of a row, or
// for each 128 x 128 tile.  A value is code * scale.  The quantiser's scale
// is 2^e with the least e in [kScaleMin, kScaleMax] for which the block's
// largest finite magnitude is at most 448 * 2^e, and 1 for a block without a
// finite nonzero: multiplying by a power of two is exact, so a value is
// rounded once, and code * 2^e is exact in bf16 (the bounds keep the least
// code, 2^-9, times the scale a normal bf16 and 1 / scale a normal float), but for
// magnitudes of 248 * 2^120 and more, which round to 2^128 and come back infinite.
// Infinities and NaN take the NaN code and stay out of the scale, so that
// they stay visible and spoil no neighbour.
#pragma once

#include <type_traits>

#include "cdx_internal.hpp"

namespace cdx {
namespace b8 {

constexpr int kBlock = 128;       // columns (and tile rows) under one scale
constexpr int kScaleMin = -117, kScaleMax = 120;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

typedef _Float16 f16;
typedef __bf16 bf16;

// dtype codes of the C-ABI
template <class T> constexpr int dtype_of() {
    return std::is_same_v<T, float> ? CDX_DTYPE_F32
                                    : std::is_same_v<T, f16> ? CDX_DTYPE_F16 : CDX_DTYPE_BF16;
}

// Calls f with a value of the element type of `dtype` (f32, bf16 or f16).
template <class F> int with_dtype(int dtype, F f) {
    if (dtype == CDX_DTYPE_F32) return f(float{});
    if (dtype == CDX_DTYPE_BF16) return f(bf16{});
    return f(f16{});
}

// 16 bytes at any address: rows of odd widths and views begin anywhere, and
// gfx950's global loads take any alignment.
struct __attribute__((packed, aligned(1))) Bytes16 { u32x4 v; };
struct __attribute__((packed, aligned(1))) Bytes8 { u32x2 v; };

__device__ __forceinline__ u32x4 load16(const void* p) {
    return static_cast<const Bytes16*>(p)->v;
}
__device__ __forceinline__ void store16(void* p, u32x4 v) { static_cast<Bytes16*>(p)->v = v; }
__device__ __forceinline__ u32x2 load8b(const void* p) { return static_cast<const Bytes8*>(p)->v; }
__device__ __forceinline__ void store8b(void* p, u32x2 v) { static_cast<Bytes8*>(p)->v = v; }

// N consecutive elements as floats.  `n`: how many exist (the others read as
// `fill`); the full count is one or two 16-byte loads.
template <int N, class T>
__device__ __forceinline__ void load_n(const T* p, int n, float (&v)[N], float fill = 0.0f) {
    constexpr int PER = 16 / (int)sizeof(T);
    static_assert(N % PER == 0 || N * sizeof(T) == 8, "whole 16-byte (or one 8-byte) loads");
    if (n >= N) {
        if constexpr (N % PER == 0) {
#pragma unroll
            for (int i = 0; i < N / PER; ++i) {
                const u32x4 u = load16(p + i * PER);
                T e[PER];
                __builtin_memcpy(e, &u, 16);
#pragma unroll
                for (int j = 0; j < PER; ++j) v[i * PER + j] = (float)e[j];
            }
        } else {
            const u32x2 u = load8b(p);
            T e[N];
            __builtin_memcpy(e, &u, 8);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = (float)e[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < n ? (float)p[j] : fill;
    }
}

// Two floats rounded to bf16 in one register (the first in the low half).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
}

template <class T> __device__ __forceinline__ T round_to(float v) { return (T)v; }

template <int N, class T>
__device__ __forceinline__ void store_n(T* p, int n, const float (&v)[N]) {
    constexpr int PER = 16 / (int)sizeof(T);
    static_assert(N % PER == 0 || N * sizeof(T) == 8, "whole 16-byte (or one 8-byte) stores");
    if (n >= N) {
        T e[N];
        if constexpr (std::is_same_v<T, bf16>) {
            uint32_t w[N / 2];
#pragma unroll
            for (int j = 0; j < N / 2; ++j) w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
            __builtin_memcpy(e, w, sizeof(e));
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = round_to<T>(v[j]);
        }
        if constexpr (N % PER == 0) {
#pragma unroll
            for (int i = 0; i < N / PER; ++i) {
                u32x4 u;
                __builtin_memcpy(&u, e + i * PER, 16);
                store16(p + i * PER, u);
            }
        } else {
            u32x2 u;
            __builtin_memcpy(&u, e, 8);
            store8b(p, u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) p[j] = round_to<T>(v[j]);
    }
}

// Lane rotations within the 16 lanes of a DPP row.
template <int R> __device__ __forceinline__ float ror16(float v) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + R, 0xf, 0xf, false));
}

// The sum (largest) over the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ float sum16(float v) {
    v += ror16<8>(v);
    v += ror16<4>(v);
    v += ror16<2>(v);
    return v + ror16<1>(v);
}
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, ror16<8>(v));
    v = fmaxf(v, ror16<4>(v));
    v = fmaxf(v, ror16<2>(v));
    return fmaxf(v, ror16<1>(v));
}

__device__ __forceinline__ float lane_value(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// The sum over a wave, in all lanes (all 64 must be active).
__device__ __forceinline__ float sum64(float v) {
    v = sum16(v);
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ float max64(float v) {
    v = max16(v);
    return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)),
                 fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// ---- the format ---------------------------------------------------------------

// |v| where it is finite, else 0 (what the scale looks at).
__device__ __forceinline__ float finite_mag(float v) {
    const float a = __builtin_fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}

// The scale's biased exponent e + 127 of a block whose largest magnitude is
// amax: amax = 1.f * 2^E is at most 448 * 2^e = 1.75 * 2^(e + 8) from e = E - 8 on
// if 1.f <= 1.75, else from E - 7 on.  (Subnormal amax reads as E = -127, below
// the lower bound anyway.)
__device__ __forceinline__ int scale_exp(float amax) {
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    int e = (int)(u >> 23) - 8 + ((u & 0x7fffff) > 0x600000);
    e = e < 127 + kScaleMin ? 127 + kScaleMin : e;
    e = e > 127 + kScaleMax ? 127 + kScaleMax : e;
    return u ? e : 127;
}

__device__ __forceinline__ float exp_value(int biased) {   // 2^(biased - 127), 1 <= biased <= 254
    return __builtin_bit_cast(float, (uint32_t)biased << 23);
}

// A scale byte's value: 2^(b - 127) (0: the subnormal 2^-127), NaN for 255; no branches.
__device__ __forceinline__ float e8m0_value(uint32_t b) {
    uint32_t u = b << 23;
    u = u > 0x00400000u ? u : 0x00400000u;
    return __builtin_bit_cast(float, u | (b + 1) >> 8 << 22);
}

__device__ __forceinline__ float load_scale(const void* s, int64_t i, bool e8m0) {
    return e8m0 ? e8m0_value(static_cast<const uint8_t*>(s)[i]) : static_cast<const float*>(s)[i];
}

// Activations on values of T: fp32 results with the accurate functions of the
// elementwise kernels; results that are rounded to 16 bits with the hardware's
// exponential and reciprocal (relative error 2^-22, below 2^-9 and 2^-12 by far;
// with expf and divisions the GELU pair of 8-bit checkpoints is bound by them, not by memory).
template <class T> __device__ __forceinline__ float fast_exp(float x) {
    if constexpr (std::is_same_v<T, float>) return expf(x);
    else return __builtin_amdgcn_exp2f(x * 1.44269504f);
}
template <class T> __device__ __forceinline__ float inverse(float x) {
    if constexpr (std::is_same_v<T, float>) return 1.0f / x;
    else return __builtin_amdgcn_rcpf(x);
}

template <class T, int ACT>
__device__ __forceinline__ float act_value(float v, float alpha) {
    if constexpr (ACT == CDX_EPI_RELU) return v > 0.0f ? v : 0.0f;
    if constexpr (ACT == CDX_EPI_GELU) {
        const float u = 0.7978845608f * (v + 0.044715f * v * v * v);
        return v * inverse<T>(1.0f + fast_exp<T>(-2.0f * u));
    }
    if constexpr (ACT == CDX_EPI_SILU) return v * inverse<T>(1.0f + fast_exp<T>(-v));
    if constexpr (ACT == CDX_EPI_SIGMOID) return inverse<T>(1.0f + fast_exp<T>(-v));
    if constexpr (ACT == CDX_ACT_TANH) return tanhf(v);
    if constexpr (ACT == CDX_ACT_LEAKY_RELU) return v > 0.0f ? v : alpha * v;
    return v;
}

// Four values times `inv` (a power of two that brings them to at most 448 in
// magnitude), rounded to nearest even; infinities become NaN first.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d, float inv) {
    const float inf = __builtin_inff(), nan = __builtin_nanf("");
    a = __builtin_fabsf(a) == inf ? nan : a * inv;
    b = __builtin_fabsf(b) == inf ? nan : b * inv;
    c = __builtin_fabsf(c) == inf ? nan : c * inv;
    d = __builtin_fabsf(d) == inf ? nan : d * inv;
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// The four values of a word of codes (unscaled).
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float (&v)[4]) {
    const floatx2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const floatx2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
}

// The workgroup's tile number as its XCD's share (workgroup b runs on XCD b % 8):
// each XCD takes a run of neighbouring tiles, which share operands in its L2.
__device__ __forceinline__ int64_t xcd_tile(int64_t b, int64_t count) {
    const int64_t each = count / 8, more = count % 8, x = b % 8;
    return x * each + (x < more ? x : more) + b / 8;
}

// Whether one dimension of a launch holds these workgroups: its threads are counted in 32 bits, and
// a launch of more runs what is left of the number, without an error.
inline bool grid_fits(int64_t groups, int threads) {
    return groups < ((int64_t)1 << 31) && groups * threads < ((int64_t)1 << 32);
}

// An 8-bit matrix: codes with leading dimension ldq, scales [rows (or tiles
// of 128 rows)][ceil(cols / 128)] with leading dimension lds.
struct Mat8 {
    const uint8_t* q; int64_t ldq;
    const void* s; int64_t lds;
    int e8m0;        // scales: 1 e8m0 bytes, 0 floats
};

}  // namespace b8

// ---- launchers (no argument validation: the C-ABI validates first) -----------------

// n zeros of f32, f16 or bf16 (a kernel, so that calls can be captured).
int launch_zero(void* p, int64_t n, int dtype, hipStream_t stream);

// Layer norm (layer_norm.hip).  dtype: x, y and gradients; pdtype: weight, bias
// and their gradients (f32 or dtype).  mean, rstd, weight, bias may be null.
int launch_layer_norm(const void* x, int64_t ldx, const void* w, const void* b, void* y,
                      int64_t ldy, float* mean, float* rstd, int64_t rows, int64_t dim, float eps,
                      int dtype, int pdtype, hipStream_t stream);
// ws: layer_norm_partial_floats(...) floats where grad_w or grad_b is wanted.
size_t layer_norm_partial_floats(int64_t rows, int64_t dim, int dtype);
int launch_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                               const void* w, const float* mean, const float* rstd, void* dx,
                               int64_t lddx, void* dw, void* db, int64_t rows, int64_t dim,
                               int dtype, int pdtype, float* ws, hipStream_t stream);

// The 8-bit format (quantize8.hip).  act: CDX_EPI_* or CDX_ACT_* of `y`, or
// CDX_EPI_NONE with y null.
int launch_quantize_rows(const void* x, int64_t ldx, int64_t rows, int64_t cols, int dtype,
                         uint8_t* q, int64_t ldq, void* s, int64_t lds, int e8m0, void* y,
                         int64_t ldy, int act, float alpha, hipStream_t stream);
int launch_quantize_tiles(const void* x, int64_t ldx, int64_t rows, int64_t cols, int dtype,
                          uint8_t* q, int64_t ldq, void* s, int64_t lds, int e8m0,
                          hipStream_t stream);
// out = q * s, or out = grad * act'(q * s) where grad is given.
int launch_dequantize(const b8::Mat8& a, int tile_rows, int64_t rows, int64_t cols, void* out,
                      int64_t ldo, int dtype, hipStream_t stream);
int launch_activation_backward8(const void* grad, int64_t ldg, const b8::Mat8& a, int64_t rows,
                                int64_t cols, void* out, int64_t ldo, int dtype, int act,
                                float alpha, hipStream_t stream);

// C[M,N] = act(A B^T + bias) (gemm8.hip): A's scales by row, B's by 128 x 128
// tile.  x, when not null, stands for A: [M,K] elements of xdtype, quantised
// by the launch (scale bytes if B's are, into ws).
struct Gemm8Args {
    int64_t M, N, K;
    b8::Mat8 a, b;
    const void* x = nullptr; int64_t ldx = 0; int xdtype = CDX_DTYPE_F32;
    void* C; int64_t ldc; int cdtype;
    const float* bias; int epilogue;
    void* ws = nullptr;
};
size_t gemm8_workspace(int64_t M, int64_t N, int64_t K, bool from_x);
int launch_gemm8(const Gemm8Args& g, hipStream_t stream);
// The kernel it runs: aligned operands or not, 32-bit results (wide) or 16-bit ones.
const char* gemm8_kernel_name(int64_t M, int64_t N, int64_t K, bool aligned, bool wide, bool from_x);

// dw[N,K] = dz[M,N]^T * (q * s)[M,K], db[n] = sum_m dz[m,n] (wgrad8.hip; db may be
// null).  ws: wgrad8_workspace(...) bytes.
size_t wgrad8_workspace(int64_t M, int64_t N, int64_t K, int dtype, bool bias);
int launch_wgrad8(const void* dz, int64_t lddz, int dtype, const b8::Mat8& x, float* dw, float* db,
                  int64_t M, int64_t N, int64_t K, void* ws, hipStream_t stream);
// The side of its tiles and the number of slices of m.
void wgrad8_plan(int64_t M, int64_t N, int64_t K, int* side, int* slices);

}  // namespace cdx
