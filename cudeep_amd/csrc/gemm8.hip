// C[M,N] = act(A B^T + bias) of 8-bit operands with a scale for each 128
// columns of a row of A and each 128 x 128 tile of B:
//   C[m,n] = sum over blocks kb of sa[m,kb] sb[n/128,kb] sum_k qa[m,k] qb[n,k].
//
// Results of 16 bits: v_mfma_scale_f32_16x16x128_f8f6f4 takes one block of 128 per
// instruction, so a block's sum is one instruction's.  Scale bytes (e8m0) go into
// the instruction itself; float scales multiply the block's sum.  The
// instruction adds eight products at a time on a grid 2^-13 below the largest
// one's power of two (measured: beside 2^16 a product of 2^3 counts, one of 2^2
// does not) and everything else in 24 bits: a sum's error is a few 2^-14 of its
// larger terms (relative to the result 5e-5 to 1e-4 on random operands), which is below the
// result's rounding to 8 or 11 bits and above a 32-bit result's.
//
// Results of 32 bits: codes widen to bf16 (exact) and a block is four
// v_mfma_f32_16x16x32_bf16, whose sums keep 24 bits, at half the rate.
//
// The weights are the instruction's first operand and the activations its
// second: a lane then holds four consecutive n of one row m, all under the same
// two scales.
#include "block8.hpp"

namespace cdx {
namespace {

using namespace b8;

struct Params {
    const uint8_t* a; const uint8_t* b;
    const void* sa; const void* sb;
    int64_t M, N, K, lda, ldb, ldsa, ldsb, ldc;
    int64_t blocks;            // ceil(K / 128)
    int a_e8m0, b_e8m0;        // (float-scale kernels read either kind)
    void* C;
    const float* bias;
    int epilogue;
};

// 16 codes of a row from column k on, zeros past K.
__device__ __forceinline__ u32x4 load_codes(const uint8_t* p, int64_t k, int64_t K) {
    if (k + 16 <= K) return load16(p + k);
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (k + j < K) v[j >> 2] |= (uint32_t)p[k + j] << (8 * (j & 3));
    return v;
}

// How a block's product is formed.
constexpr int kBytes = 0;    // 8-bit instruction, scale bytes
constexpr int kFloats = 1;   // 8-bit instruction, float scales
constexpr int kWide = 2;     // bf16 instruction, float scales

// A lane's 32 codes of a row and block.
template <int MODE> struct Frag {
    intx8 q;
    __device__ __forceinline__ void set(u32x4 lo, u32x4 hi) {
        const u32x4 t[2] = {lo, hi};
        __builtin_memcpy(&q, t, 32);
    }
};
template <> struct Frag<kWide> {
    bf16x8 v[4];
    __device__ __forceinline__ static bf16x8 widen(uint32_t a, uint32_t b) {
        uint32_t w[4];
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
        bf16x8 r;
        __builtin_memcpy(&r, w, 16);
        return r;
    }
    __device__ __forceinline__ void set(u32x4 lo, u32x4 hi) {
        v[0] = widen(lo[0], lo[1]);
        v[1] = widen(lo[2], lo[3]);
        v[2] = widen(hi[0], hi[1]);
        v[3] = widen(hi[2], hi[3]);
    }
};

// acc += the block's sum under its scales: the bytes sa and sb, or s, the float
// product of both.
template <int MODE>
__device__ __forceinline__ floatx4 block_product(const Frag<MODE>& w, const Frag<MODE>& x,
                                                 floatx4 acc, int sa, int sb, float s) {
    if constexpr (MODE == kBytes) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.q, x.q, acc, 0, 0, 0, sb, 0, sa);
    } else {
        floatx4 t = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (MODE == kFloats) {
            t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.q, x.q, t, 0, 0, 0, 127, 0, 127);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[j], x.v[j], t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(t[r], s, acc[r]);
        return acc;
    }
}

// Four consecutive n (from n0) of row m: bias, activation, rounding, store.
template <class T>
__device__ __forceinline__ void store_four(const Params& p, int64_t m, int64_t n0, floatx4 v) {
    if (m >= p.M || n0 >= p.N) return;
    T* c = static_cast<T*>(p.C) + m * p.ldc + n0;
    const int n = p.N - n0 < 4 ? (int)(p.N - n0) : 4;
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float b = p.bias && r < n ? p.bias[n0 + r] : 0.0f;
        o[r] = apply_act(v[r] + b, p.epilogue);
    }
    store_n<4>(c, n, o);
}

// Operands of any alignment and any K, 64 x 64 tiles: four waves of 32 x 32,
// each block of 128 staged through registers into LDS.  A row's 16-byte pieces
// lie at piece ^ (row & 7), so that the 16 rows that lanes read together spread
// over all banks.
template <class T, int MODE>
__global__ __launch_bounds__(256)
void gemm8_any_kernel(Params p) {
    __shared__ u32x4 lds[2][64][8];   // A rows, B rows
    const int tid = threadIdx.x, wave = tid >> 6, l16 = tid & 15, g = (tid >> 4) & 3;
    const int wm = wave & 1, wn = wave >> 1;
    const int64_t tiles_m = ceil_div(p.M, (int64_t)64);
    const int64_t m0 = (blockIdx.x % tiles_m) * 64, n0 = (blockIdx.x / tiles_m) * 64;
    u32x4 stage[4];
    auto load = [&](int64_t kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int piece = tid + 256 * i, row = (piece >> 3) & 63, c = piece & 7;
            const bool is_b = piece >= 512;
            const int64_t last = (is_b ? p.N : p.M) - 1;
            int64_t r = (is_b ? n0 : m0) + row;
            r = r < last ? r : last;
            stage[i] = load_codes((is_b ? p.b : p.a) + r * (is_b ? p.ldb : p.lda), kb * kBlock + 16 * c, p.K);
        }
    };
    floatx4 acc[2][2] = {};
    int64_t am[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        am[j] = m0 + 32 * wm + 16 * j + l16;
        am[j] = am[j] < p.M ? am[j] : p.M - 1;
    }
    load(0);
    for (int64_t kb = 0; kb < p.blocks; ++kb) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int piece = tid + 256 * i, row = (piece >> 3) & 63, c = piece & 7;
            lds[piece >= 512][row][c ^ (row & 7)] = stage[i];
        }
        __syncthreads();
        if (kb + 1 < p.blocks) load(kb + 1);
        int sa[2] = {}, sb = 0;
        float s[2] = {};
        if constexpr (MODE == kBytes) {
            sb = static_cast<const uint8_t*>(p.sb)[(n0 / kBlock) * p.ldsb + kb];
#pragma unroll
            for (int j = 0; j < 2; ++j) sa[j] = static_cast<const uint8_t*>(p.sa)[am[j] * p.ldsa + kb];
        } else {
            const float fb = load_scale(p.sb, (n0 / kBlock) * p.ldsb + kb, p.b_e8m0);
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = fb * load_scale(p.sa, am[j] * p.ldsa + kb, p.a_e8m0);
        }
        Frag<MODE> xq[2], wq[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int ra = 32 * wm + 16 * j + l16, rb = 32 * wn + 16 * j + l16;
            xq[j].set(lds[0][ra][(2 * g) ^ (ra & 7)], lds[0][ra][(2 * g + 1) ^ (ra & 7)]);
            wq[j].set(lds[1][rb][(2 * g) ^ (rb & 7)], lds[1][rb][(2 * g + 1) ^ (rb & 7)]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = block_product<MODE>(wq[i], xq[j], acc[i][j], sa[j], sb, s[j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            store_four<T>(p, m0 + 32 * wm + 16 * j + l16, n0 + 32 * wn + 16 * i + 4 * g, acc[i][j]);
}

// K = 0: act(bias).
template <class T>
__global__ __launch_bounds__(256)
void gemm8_empty_kernel(Params p) {
    const int64_t four = ceil_div(p.N, (int64_t)4), n = p.M * four;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        store_four<T>(p, i / four, i % four * 4, floatx4{0.0f, 0.0f, 0.0f, 0.0f});
}

// Calls f with the way a result type and scale types call for.
template <class T, class F> int with_mode(const Params& p, F f) {
    using std::integral_constant;
    if constexpr (std::is_same_v<T, float>) return f(integral_constant<int, kWide>{});
    else if (p.a_e8m0 && p.b_e8m0) return f(integral_constant<int, kBytes>{});
    else return f(integral_constant<int, kFloats>{});
}

template <class T>
int run(const Params& p, hipStream_t stream) {
    if (p.K == 0) {
        const int64_t g = ceil_div(p.M * ceil_div(p.N, (int64_t)4), (int64_t)256);
        hipLaunchKernelGGL(gemm8_empty_kernel<T>, dim3((unsigned)(g < 65536 ? g : 65536)), dim3(256), 0,
                           stream, p);
        return hip_error(hipGetLastError(), "gemm8_empty_kernel launch");
    }
    const int64_t grid = ceil_div(p.M, (int64_t)64) * ceil_div(p.N, (int64_t)64);
    if (grid >= (int64_t)1 << 31) return set_error(CDX_ERR_UNSUPPORTED, "gemm8: too many output tiles");
    return with_mode<T>(p, [&](auto mode) {
        hipLaunchKernelGGL((gemm8_any_kernel<T, decltype(mode)::value>), dim3((unsigned)grid), dim3(256),
                           0, stream, p);
        return hip_error(hipGetLastError(), "gemm8_any_kernel launch");
    });
}

// Where a launch quantises x itself: codes, then scales behind them.
int64_t codes_ld(int64_t K) { return ceil_div(K, (int64_t)16) * 16; }
size_t codes_bytes(int64_t M, int64_t K) { return ((size_t)M * (size_t)codes_ld(K) + 255) / 256 * 256; }

}  // namespace

size_t gemm8_workspace(int64_t M, int64_t N, int64_t K, bool from_x) {
    (void)N;
    if (!from_x || M == 0 || K == 0) return 0;
    return codes_bytes(M, K) + (size_t)M * (size_t)ceil_div(K, (int64_t)kBlock) * 4;
}

int launch_gemm8(const Gemm8Args& g, hipStream_t stream) {
    const int64_t blocks = ceil_div(g.K, (int64_t)kBlock);
    Params p{g.a.q, g.b.q, g.a.s, g.b.s, g.M, g.N, g.K, g.a.ldq, g.b.ldq, g.a.lds, g.b.lds, g.ldc,
             blocks, g.a.e8m0, g.b.e8m0, g.C, g.bias, g.epilogue};
    if (g.x && g.K > 0) {
        uint8_t* q = static_cast<uint8_t*>(g.ws);
        void* s = q + codes_bytes(g.M, g.K);
        const int st = launch_quantize_rows(g.x, g.ldx, g.M, g.K, g.xdtype, q, codes_ld(g.K), s,
                                            blocks, g.b.e8m0, nullptr, 0, CDX_EPI_NONE, 0.0f, stream);
        if (st) return st;
        p.a = q; p.lda = codes_ld(g.K); p.sa = s; p.ldsa = blocks; p.a_e8m0 = g.b.e8m0;
    }
    return with_dtype(g.cdtype, [&](auto t) { return run<decltype(t)>(p, stream); });
}

}  // namespace cdx
