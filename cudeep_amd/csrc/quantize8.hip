// Into and out of the 8-bit block-scaled format (block8.hpp), alone or with an
// activation: all of them read and write each value once, by the thread that read it (an activation's
// result may take the place of its input, a gradient's that of the other: no __restrict__ there).
//
// Rows: the 16 lanes of a DPP row take the 128 columns of a block, eight values
// each (one 16-byte load of 16-bit values), so a block's largest magnitude is
// four lane rotations away and nothing goes through LDS.  Tiles of 128 x 128
// (weights): one workgroup of 1024 threads, 16 values a thread in registers, the
// largest magnitude through LDS.
//
// Bound by memory, all of them (bf16, bytes read and written over the time): rows of 8192 x
// 8192 34.3 us, 5.9 TB/s; tiles 35.1, 5.7; restoring 31.4, 6.4; 8192 x 4096 with GELU 26.7,
// 6.3 (28.7 with operands that no cache holds), its gradient 30.3, 5.5 (35.8).
#include "block8.hpp"

namespace cdx {
namespace {

using namespace b8;

constexpr int kLane = 8;   // values per lane: 16 lanes cover a block

// s = 1 / (1 + exp(-x)) and r = 1 - s, neither by subtraction.  fp32: from both
// exponentials, as the elementwise kernels.  16 bits: r = exp(-x) s from one exponential,
// held finite there: where s is 0, so is r (only s and s r are used).  The GELU backward
// pass is held up by its exponentials and reciprocals: 8192 x 4096 in bf16 45.6 us with two
// of each, 38.9 with one (operands that no cache holds).
template <class T> __device__ __forceinline__ void logistic(float x, float& s, float& r) {
    if constexpr (std::is_same_v<T, float>) {
        s = 1.0f / (1.0f + expf(-x));
        r = 1.0f / (1.0f + expf(x));
    } else {
        const float e = __builtin_amdgcn_exp2f(x * -1.44269504f);
        s = __builtin_amdgcn_rcpf(1.0f + e);
        r = fminf(e, 0x1p126f) * s;
    }
}

// v as a factor of s r.  In both tails s r is 0 and a slope is s itself, but v v overflows from
// 1.8e19 on (and v is infinite where its 8 bits round to 2^128), and 0 times infinity is no slope:
// 0 there, or for 16 bits, bound by their instructions, v within 2^30.  8192 x 4096 with GELU: fp32
// 74.5 us, clamped 78.5; bf16 30.3, chosen by s r > 0 32.5.
template <class T> __device__ __forceinline__ float beside(float v, float sr) {
    if constexpr (std::is_same_v<T, float>) return sr > 0.0f ? v : 0.0f;
    else return __builtin_amdgcn_fmed3f(v, -0x1p30f, 0x1p30f);
}

// grad * act'(v).
template <class T, int ACT>
__device__ __forceinline__ float act_slope(float g, float v, float alpha) {
    if constexpr (ACT == CDX_EPI_RELU) return v > 0.0f ? g : 0.0f;
    if constexpr (ACT == CDX_ACT_LEAKY_RELU) return v > 0.0f ? g : alpha * g;
    float s, r;
    if constexpr (ACT == CDX_EPI_GELU) {
        constexpr float c = 0.7978845608f, k = 0.044715f;
        logistic<T>(2.0f * c * (v + k * v * v * v), s, r);
        const float n = beside<T>(v, s * r);   // slope s + 2 v s r du, du = c (1 + 3 k v v)
        return g * (s + n * (s * r) * (2.0f * c + 6.0f * c * k * (n * n)));
    }
    if constexpr (ACT == CDX_EPI_SILU) {
        logistic<T>(v, s, r);
        return g * (s + beside<T>(v, s * r) * (s * r));
    }
    if constexpr (ACT == CDX_EPI_SIGMOID) {
        logistic<T>(v, s, r);
        return g * (s * r);
    }
    if constexpr (ACT == CDX_ACT_TANH) {
        const float t = tanhf(v);
        return g * (1.0f - t) * (1.0f + t);
    }
    return g;
}

// Calls f with the activation's code as a constant.
template <class F> int with_act(int act, F f) {
    using std::integral_constant;
    switch (act) {
        case CDX_EPI_RELU: return f(integral_constant<int, CDX_EPI_RELU>{});
        case CDX_EPI_GELU: return f(integral_constant<int, CDX_EPI_GELU>{});
        case CDX_EPI_SILU: return f(integral_constant<int, CDX_EPI_SILU>{});
        case CDX_EPI_SIGMOID: return f(integral_constant<int, CDX_EPI_SIGMOID>{});
        case CDX_ACT_TANH: return f(integral_constant<int, CDX_ACT_TANH>{});
        case CDX_ACT_LEAKY_RELU: return f(integral_constant<int, CDX_ACT_LEAKY_RELU>{});
        default: return f(integral_constant<int, CDX_EPI_NONE>{});
    }
}

// Walks [rows, cols] in pieces of eight columns, 16 pieces to a block of 128:
// piece p of row r is number (r * blocks + block) * 16 + p % 16.
struct Pieces {
    int64_t rows, cols, blocks, count;   // count: rows * blocks
    DivMagic by_blocks;                  // for count < 2^31
};

Pieces pieces_of(int64_t rows, int64_t cols) {
    const int64_t blocks = ceil_div(cols, (int64_t)kBlock);
    return {rows, cols, blocks, rows * blocks,
            blocks < ((int64_t)1 << 31) ? div_magic(blocks) : DivMagic{0, 0}};
}

__device__ __forceinline__ void row_of(const Pieces& p, int64_t i, int64_t& row, int64_t& blk) {
    if (p.count < ((int64_t)1 << 31)) {
        const uint32_t r = div_u31((uint32_t)i, p.by_blocks);
        row = r;
        blk = (uint32_t)i - r * (uint32_t)p.blocks;
    } else {
        row = i / p.blocks;
        blk = i - row * p.blocks;
    }
}

template <class T, int ACT, bool E8M0>
__global__ __launch_bounds__(256)
void quantize_rows_kernel(Pieces p, const T* x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
                          void* __restrict__ s, int64_t lds, T* y, int64_t ldy, float alpha) {
    const int lane = threadIdx.x & 15;
    for (int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); i < p.count;
         i += (int64_t)gridDim.x * 16) {
        int64_t row, blk;
        row_of(p, i, row, blk);
        const int64_t c = blk * kBlock + lane * kLane;
        const int64_t left = p.cols - c;
        const int n = left < 0 ? 0 : left > kLane ? kLane : (int)left;
        float v[kLane];
        load_n<kLane>(x + row * ldx + c, n, v);
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < kLane; ++j) m = fmaxf(m, finite_mag(v[j]));
        const int e = scale_exp(max16(m));
        const float inv = exp_value(254 - e);
        const uint32_t lo = pack_e4m3(v[0], v[1], v[2], v[3], inv);
        const uint32_t hi = pack_e4m3(v[4], v[5], v[6], v[7], inv);
        uint8_t* qr = q + row * ldq + c;
        if (n == kLane) {
            store8b(qr, u32x2{lo, hi});
        } else {
#pragma unroll
            for (int j = 0; j < kLane; ++j)
                if (j < n) qr[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
        }
        if (lane == 0) {
            if constexpr (E8M0) static_cast<uint8_t*>(s)[row * lds + blk] = (uint8_t)e;
            else static_cast<float*>(s)[row * lds + blk] = exp_value(e);
        }
        if constexpr (ACT != CDX_EPI_NONE) {
#pragma unroll
            for (int j = 0; j < kLane; ++j) v[j] = act_value<T, ACT>(v[j], alpha);
            store_n<kLane>(y + row * ldy + c, n, v);
        }
    }
}

template <class T, bool E8M0>
__global__ __launch_bounds__(1024)
void quantize_tiles_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols,
                           uint8_t* __restrict__ q, int64_t ldq, void* __restrict__ s,
                           int64_t lds) {
    __shared__ float red[16];
    const int lane = threadIdx.x & 15, line = threadIdx.x >> 4;   // rows `line` and line + 64
    const int64_t blk = blockIdx.x, tiles = ceil_div(rows, (int64_t)kBlock);
    const int64_t c = blk * kBlock + lane * kLane;
    const int64_t left = cols - c;
    const int width = left < 0 ? 0 : left > kLane ? kLane : (int)left;
    for (int64_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
        float v[2][kLane];
        float m = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = tile * kBlock + line + 64 * h;
            load_n<kLane>(x + row * ldx + c, row < rows ? width : 0, v[h]);
#pragma unroll
            for (int j = 0; j < kLane; ++j) m = fmaxf(m, finite_mag(v[h][j]));
        }
        m = max64(m);
        __syncthreads();   // the last tile's readers are done with red
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) m = fmaxf(m, red[k]);
        const int e = scale_exp(m);
        const float inv = exp_value(254 - e);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = tile * kBlock + line + 64 * h;
            if (row >= rows) continue;
            const uint32_t lo = pack_e4m3(v[h][0], v[h][1], v[h][2], v[h][3], inv);
            const uint32_t hi = pack_e4m3(v[h][4], v[h][5], v[h][6], v[h][7], inv);
            uint8_t* qr = q + row * ldq + c;
            if (width == kLane) {
                store8b(qr, u32x2{lo, hi});
            } else {
#pragma unroll
                for (int j = 0; j < kLane; ++j)
                    if (j < width) qr[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
            }
        }
        if (threadIdx.x == 0) {
            if constexpr (E8M0) static_cast<uint8_t*>(s)[tile * lds + blk] = (uint8_t)e;
            else static_cast<float*>(s)[tile * lds + blk] = exp_value(e);
        }
    }
}

// out = q * s, or grad * act'(q * s).
template <class T, int ACT, bool BWD>
__global__ __launch_bounds__(256)
void dequantize_kernel(Pieces p, Mat8 a, int tile_shift, const T* grad, int64_t ldg, T* out,
                       int64_t ldo, float alpha) {
    const int lane = threadIdx.x & 15;
    for (int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); i < p.count;
         i += (int64_t)gridDim.x * 16) {
        int64_t row, blk;
        row_of(p, i, row, blk);
        const int64_t c = blk * kBlock + lane * kLane;
        const int64_t left = p.cols - c;
        const int n = left < 0 ? 0 : left > kLane ? kLane : (int)left;
        const uint8_t* qr = a.q + row * a.ldq + c;
        u32x2 w = {0u, 0u};
        if (n == kLane) {
            w = load8b(qr);
        } else {
#pragma unroll
            for (int j = 0; j < kLane; ++j)
                if (j < n) w[j >> 2] |= (uint32_t)qr[j] << (8 * (j & 3));
        }
        const float scale = load_scale(a.s, (row >> tile_shift) * a.lds + blk, a.e8m0);
        float g[kLane];
        if constexpr (BWD) load_n<kLane>(grad + row * ldg + c, n, g);
        float lo[4], hi[4], v[kLane];
        unpack_e4m3(w[0], lo);
        unpack_e4m3(w[1], hi);
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            v[j] = (j < 4 ? lo[j] : hi[j - 4]) * scale;
            if constexpr (BWD) v[j] = act_slope<T, ACT>(g[j], v[j], alpha);
        }
        store_n<kLane>(out + row * ldo + c, n, v);
    }
}

unsigned piece_grid(const Pieces& p) {
    const int64_t g = ceil_div(p.count, (int64_t)16);
    return (unsigned)(g < 65536 * 16 ? g : 65536 * 16);
}

}  // namespace

int launch_quantize_rows(const void* x, int64_t ldx, int64_t rows, int64_t cols, int dtype,
                         uint8_t* q, int64_t ldq, void* s, int64_t lds, int e8m0, void* y,
                         int64_t ldy, int act, float alpha, hipStream_t stream) {
    const Pieces p = pieces_of(rows, cols);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return with_act(act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            if (e8m0)
                hipLaunchKernelGGL((quantize_rows_kernel<T, ACT, true>), dim3(piece_grid(p)),
                                   dim3(256), 0, stream, p, static_cast<const T*>(x), ldx, q, ldq,
                                   s, lds, static_cast<T*>(y), ldy, alpha);
            else
                hipLaunchKernelGGL((quantize_rows_kernel<T, ACT, false>), dim3(piece_grid(p)),
                                   dim3(256), 0, stream, p, static_cast<const T*>(x), ldx, q, ldq,
                                   s, lds, static_cast<T*>(y), ldy, alpha);
            return hip_error(hipGetLastError(), "quantize_rows_kernel launch");
        });
    });
}

int launch_quantize_tiles(const void* x, int64_t ldx, int64_t rows, int64_t cols, int dtype,
                          uint8_t* q, int64_t ldq, void* s, int64_t lds, int e8m0,
                          hipStream_t stream) {
    const int64_t tiles = ceil_div(rows, (int64_t)kBlock);
    constexpr int64_t most = (int64_t)1 << 21;   // blocks across a launch: 2^31 threads
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        for (int64_t c = 0, b = 0; c < cols; c += most * kBlock, b += most) {
            const int64_t part = cols - c < most * kBlock ? cols - c : most * kBlock;
            const dim3 grid((unsigned)ceil_div(part, (int64_t)kBlock),
                            (unsigned)(tiles < 65535 ? tiles : 65535));
            if (e8m0)
                hipLaunchKernelGGL((quantize_tiles_kernel<T, true>), grid, dim3(1024), 0, stream,
                                   static_cast<const T*>(x) + c, ldx, rows, part, q + c, ldq,
                                   static_cast<uint8_t*>(s) + b, lds);
            else
                hipLaunchKernelGGL((quantize_tiles_kernel<T, false>), grid, dim3(1024), 0, stream,
                                   static_cast<const T*>(x) + c, ldx, rows, part, q + c, ldq,
                                   static_cast<float*>(s) + b, lds);
            const int st = hip_error(hipGetLastError(), "quantize_tiles_kernel launch");
            if (st) return st;
        }
        return (int)CDX_OK;
    });
}

int launch_dequantize(const Mat8& a, int tile_rows, int64_t rows, int64_t cols, void* out,
                      int64_t ldo, int dtype, hipStream_t stream) {
    const Pieces p = pieces_of(rows, cols);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((dequantize_kernel<T, CDX_EPI_NONE, false>), dim3(piece_grid(p)),
                           dim3(256), 0, stream, p, a, tile_rows == 1 ? 0 : 7,
                           static_cast<const T*>(nullptr), (int64_t)0, static_cast<T*>(out), ldo,
                           0.0f);
        return hip_error(hipGetLastError(), "dequantize_kernel launch");
    });
}

int launch_activation_backward8(const void* grad, int64_t ldg, const Mat8& a, int64_t rows,
                                int64_t cols, void* out, int64_t ldo, int dtype, int act,
                                float alpha, hipStream_t stream) {
    const Pieces p = pieces_of(rows, cols);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return with_act(act, [&](auto ac) {
            constexpr int ACT = decltype(ac)::value;
            hipLaunchKernelGGL((dequantize_kernel<T, ACT, true>), dim3(piece_grid(p)), dim3(256), 0,
                               stream, p, a, 0, static_cast<const T*>(grad), ldg,
                               static_cast<T*>(out), ldo, alpha);
            return hip_error(hipGetLastError(), "dequantize_kernel launch");
        });
    });
}

}  // namespace cdx
