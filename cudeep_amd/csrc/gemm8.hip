// C[M,N] = act(A B^T + bias) of 8-bit operands with a scale for each 128
// columns of a row of A and each 128 x 128 tile of B:
//   C[m,n] = sum over blocks kb of sa[m,kb] sb[n/128,kb] sum_k qa[m,k] qb[n,k].
//
// Results of 16 bits: v_mfma_scale_f32_16x16x128_f8f6f4 takes one block of 128 per
// instruction, so a block's sum is one instruction's.  Scale bytes (e8m0) go into
// the instruction itself; float scales multiply the block's sum.  The
// instruction adds eight products at a time on a grid 2^-13 below the largest
// one's power of two (measured: beside 2^16 a product of 2^3 counts, one of 2^2
// does not) and everything else in 24 bits.  That is fewer than 32 bits, taken for
// twice the rate: a sum may lose 2^-10 of the largest of each eight products.  On random
// operands (1 to 2048 rows, K 1200 and 4096, both kinds of scales) it is 1.2e-5 to 2.6e-5 of the
// results' norm, a hundredth of bf16's rounding and a tenth of f16's (error against 64 bits 1.661e-3
// and 2.083e-4, the roundings alone 1.661e-3 and 2.073e-4); a sum that cancels loses more
// than its rounding.  Results of 32 bits are for those who mind.
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
    const int n = (int)(K - k);
#pragma unroll 1
    for (int j = n < 0 ? -1 : n - 1; j >= 0; --j) {   // the last code first
        v[3] = v[3] << 8 | v[2] >> 24;
        v[2] = v[2] << 8 | v[1] >> 24;
        v[1] = v[1] << 8 | v[0] >> 24;
        v[0] = v[0] << 8 | p[k + j];
    }
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

// Products with GELU and 16-bit results: 4096^3 72 us, with expf and a division 80.
template <class T, int ACT> __device__ __forceinline__ float result_act(float v) {
    if constexpr (std::is_same_v<T, float>) return act_fixed<ACT>(v);
    else return act_value<T, ACT>(v, 0.0f);
}

// A wave's FN x FM accumulators (first n and m: n0, m0) through bias and
// activation into C: a lane stores four consecutive n of a row at once.
template <class T, int ACT, int FN, int FM>
__device__ __forceinline__ void store_act(const Params& p, int64_t m0, int64_t n0,
                                          const floatx4 (&acc)[FN][FM]) {
    const int l16 = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const int64_t nn = n0 + 16 * i + 4 * g;
        const int n = p.N - nn < 0 ? 0 : p.N - nn < 4 ? (int)(p.N - nn) : 4;
        float b[4] = {};
        if (p.bias) load_n<4>(p.bias + nn, n, b);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int64_t m = m0 + 16 * j + l16;
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = result_act<T, ACT>(acc[i][j][r] + b[r]);
            if (m < p.M) store_n<4>(static_cast<T*>(p.C) + m * p.ldc + nn, n, o);
        }
    }
}

template <class T, int FN, int FM>
__device__ __forceinline__ void store_tile(const Params& p, int64_t m0, int64_t n0,
                                           const floatx4 (&acc)[FN][FM]) {
    switch (p.epilogue) {
        case CDX_EPI_RELU: store_act<T, CDX_EPI_RELU>(p, m0, n0, acc); break;
        case CDX_EPI_GELU: store_act<T, CDX_EPI_GELU>(p, m0, n0, acc); break;
        case CDX_EPI_SILU: store_act<T, CDX_EPI_SILU>(p, m0, n0, acc); break;
        case CDX_EPI_SIGMOID: store_act<T, CDX_EPI_SIGMOID>(p, m0, n0, acc); break;
        default: store_act<T, CDX_EPI_NONE>(p, m0, n0, acc); break;
    }
}

// The same for a whole workgroup's BM x BN tile through LDS (`buf`) that is no longer
// read or written, so that a wave stores whole rows: a product of 4096 x 4096 x 256 takes 17
// us, 25 with each lane's 8 bytes stored alone.
// Row m's 4-element units lie at unit ^ 4 (m & 15): 16 rows are then on all banks.
template <class T, int ACT, int BM, int BN, int NT, int FN, int FM>
__device__ __forceinline__ void store_rows_act(const Params& p, uint8_t* buf, int64_t m0, int64_t n0,
                                               int wm0, int wn0, const floatx4 (&acc)[FN][FM]) {
    constexpr int UNIT = 4 * sizeof(T), UNITS = BN / 4, ROW = BN * sizeof(T);
    constexpr int SWAP = UNITS / 4 - 1 < 15 ? UNITS / 4 - 1 : 15;
    const int l16 = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const int64_t nn = n0 + wn0 + 16 * i + 4 * g;
        float b[4] = {};
        if (p.bias) load_n<4>(p.bias + nn, p.N - nn < 0 ? 0 : p.N - nn < 4 ? (int)(p.N - nn) : 4, b);
        const int unit = (wn0 / 4 + 4 * i + g) ^ (4 * (l16 & SWAP));
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = result_act<T, ACT>(acc[i][j][r] + b[r]);
            store_n<4>(reinterpret_cast<T*>(buf + (wm0 + 16 * j + l16) * ROW + unit * UNIT), 4, o);
        }
    }
    __syncthreads();
    constexpr int CHUNKS = ROW / 16, PER = 16 / sizeof(T);
    const int c = threadIdx.x % CHUNKS, r0 = threadIdx.x / CHUNKS;
    const int64_t n = n0 + c * PER;
    T* out = static_cast<T*>(p.C) + m0 * p.ldc + n;
    const int rows = p.M - m0 < BM ? (int)(p.M - m0) : BM;
#pragma unroll 4
    for (int row = r0; row < rows; row += NT / CHUNKS) {
        const int chunk = UNIT == 16 ? c ^ (4 * (row & SWAP)) : c ^ (2 * (row & SWAP));
        const u32x4 v = *reinterpret_cast<const u32x4*>(buf + row * ROW + chunk * 16);
        T* dst = out + row * p.ldc;
        if (n + PER <= p.N) {
            store16(dst, v);
        } else {
            T e[PER];
            __builtin_memcpy(e, &v, 16);
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (n + k < p.N) dst[k] = e[k];
        }
    }
}

template <class T, int BM, int BN, int NT, int FN, int FM>
__device__ __forceinline__ void store_rows(const Params& p, uint8_t* buf, int64_t m0, int64_t n0,
                                           int wm0, int wn0, const floatx4 (&acc)[FN][FM]) {
#define CDX_ROWS(ACT) store_rows_act<T, ACT, BM, BN, NT>(p, buf, m0, n0, wm0, wn0, acc)
    switch (p.epilogue) {
        case CDX_EPI_RELU: CDX_ROWS(CDX_EPI_RELU); break;
        case CDX_EPI_GELU: CDX_ROWS(CDX_EPI_GELU); break;
        case CDX_EPI_SILU: CDX_ROWS(CDX_EPI_SILU); break;
        case CDX_EPI_SIGMOID: CDX_ROWS(CDX_EPI_SIGMOID); break;
        default: CDX_ROWS(CDX_EPI_NONE); break;
    }
#undef CDX_ROWS
}

// Operands of any alignment and any K, 64 x 64 tiles: four waves of 32 x 32,
// each block of 128 staged through registers into LDS.  A row's 16-byte pieces
// lie at piece ^ (row / 2 & 7), so that the 16 rows that lanes read together spread
// over all banks.  One block is in flight, two barriers a block: 4096 x 4096 x 4001 with rows
// of 4001 bytes 306 us, 0.44 PFLOP/s (rows of 4016 bytes take the kernel below: 68).
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
            lds[piece >= 512][row][c ^ (row >> 1 & 7)] = stage[i];
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
            xq[j].set(lds[0][ra][g ^ (ra >> 1 & 7)], lds[0][ra][(g + 4) ^ (ra >> 1 & 7)]);
            wq[j].set(lds[1][rb][g ^ (rb >> 1 & 7)], lds[1][rb][(g + 4) ^ (rb >> 1 & 7)]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = block_product<MODE>(wq[i], xq[j], acc[i][j], sa[j], sb, s[j]);
    }
    store_tile<T>(p, m0 + 32 * wm, n0 + 32 * wn, acc);
}

// Aligned operands (16-byte rows) of at least one whole block, BM x BN tiles (BM rows
// of A, BN of B), WM x WN waves.  A block of 128 columns is one step: its rows go
// from global memory straight into LDS, one step ahead of the products, two
// buffers, one barrier a step.  LDS is filled in the order of the lanes, so that
// the exchange of 16-byte pieces (piece ^ (row / 2 & 7); a lane takes pieces g and g + 4:
// the 16 rows that the hardware reads at a time then lie on all 64 banks, where pieces 2 g
// and 2 g + 1 under row & 7 took a tenth more time at 4096^3) is made on the side of the
// global addresses.  The scales of kPanel steps are laid out in LDS at once, the
// ones that a lane wants in a step side by side: as bytes they are the
// instruction's scale operand, which picks one byte of a register per 16 rows.
//
// bf16 results, scale bytes: 4096^3 58 to 70 us, 2.0 to 2.4 PFLOP/s, 8192 x 8192 x 4096 228,
// 2.4; float scales 83 and 282, 1.9.  No unit is full (matrix slots 41 % busy, VALU 25 to 39,
// LDS 20): a step's loads, LDS reads and products meet at its barrier.  32-bit results 134 and
// 483, 1.1 PFLOP/s of the bf16 instruction.
constexpr int64_t kMaxLd = 1 << 23;   // 256 rows within 32-bit offsets
template <int MODE> using Scale = std::conditional_t<MODE == kBytes, uint8_t, float>;
template <int MODE> constexpr int kPart = MODE == kBytes ? 16 : 8;   // a thread's share of a panel

// Offsets of a thread's 16-byte pieces (BM rows of A, then B's) from the tile's first row;
// rows past the last one read it again, and what they give is not stored.
template <int BM, int NT, int LOADS>
__device__ __forceinline__ void row_offsets(const Params& p, int rows_a, int rows_b, uint32_t (&off)[LOADS]) {
    const int tid = threadIdx.x, c16 = 16 * ((tid & 7) ^ ((tid >> 4) & 7));
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const bool is_b = i * NT >= BM * 8;
        const int row = (i * NT + tid) / 8 - (is_b ? BM : 0), rows = is_b ? rows_b : rows_a;
        off[i] = (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)(is_b ? p.ldb : p.lda) + c16;
    }
}

// One block's rows into LDS: `a` and `b` are the addresses of the tile's first rows in it.
template <int BM, int NT, int LOADS>
__device__ __forceinline__ void rows_to_lds(uint64_t a, uint64_t b, const uint32_t (&off)[LOADS],
                                            uint8_t* buf, int wave) {
    typedef const __attribute__((address_space(1))) uint32_t* G;
    typedef const __attribute__((address_space(1))) uint8_t* G8;
    typedef __attribute__((address_space(3))) uint32_t* L;
    // (kept apart from the offsets: scalar base + 32-bit offset, one VGPR a load)
    asm("" : "+s"(a), "+s"(b));
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        uint32_t o = off[i];
        asm("" : "+v"(o));
        __builtin_amdgcn_global_load_lds((G)((G8)(i * NT >= BM * 8 ? b : a) + o),
                                         (L)(buf + (i * NT + wave * 64) * 16), 16, 0, 0);
    }
}

// The scales of blocks kb .. kb + P - 1.  Of A a thread takes its row's next kPart: lanes
// along the rows meet no bank twice (along the blocks they took 8 us a panel).
template <int MODE, int BM, int BN, int NT, int WM, int FM, int P>
__device__ __forceinline__ void scales_to_lds(const Params& p, int64_t m0, int64_t n0, int rows_a,
                                              int64_t kb, Scale<MODE> (&panel)[P][WM][16][FM],
                                              Scale<MODE> (&panel_b)[P][(BN + kBlock - 1) / kBlock]) {
    constexpr int PART = kPart<MODE>;
    const int tid = threadIdx.x;
    for (int i = tid; i < P * ((BN + kBlock - 1) / kBlock); i += NT) {
        const int k = i % P;
        int64_t t = n0 / kBlock + i / P;
        t = t < (p.N - 1) / kBlock ? t : (p.N - 1) / kBlock;
        const int64_t at = t * p.ldsb + (kb + k < p.blocks ? kb + k : p.blocks - 1);
        if constexpr (MODE == kBytes) panel_b[k][i / P] = static_cast<const uint8_t*>(p.sb)[at];
        else panel_b[k][i / P] = load_scale(p.sb, at, p.b_e8m0);
    }
    const int row = tid % BM, from = tid / BM * PART;
    const int64_t at = (m0 + (row < rows_a ? row : rows_a - 1)) * p.ldsa;
    auto keep = [&](int k, Scale<MODE> v) { panel[from + k][row / (16 * FM)][row % 16][row % (16 * FM) / 16] = v; };
    if constexpr (MODE == kBytes) {
        const u32x4 v = load_codes(static_cast<const uint8_t*>(p.sa) + at, kb + from, p.blocks);
#pragma unroll
        for (int k = 0; k < PART; ++k) keep(k, (uint8_t)(v[k / 4] >> (8 * (k % 4))));
    } else {
        float v[PART];
        auto take = [&](bool e8m0) {
#pragma unroll
            for (int k = 0; k < PART; ++k) {
                const int64_t b = kb + from + k;
                v[k] = load_scale(p.sa, at + (b < p.blocks ? b : p.blocks - 1), e8m0);
            }
        };
        if (p.a_e8m0) take(true);
        else take(false);
#pragma unroll
        for (int k = 0; k < PART; ++k) keep(k, v[k]);
    }
}

template <class T, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2)   // (two waves a SIMD: 256 registers)
void gemm8_tile_kernel(Params p) {
    constexpr int NT = 64 * WM * WN, ROWS = BM + BN, LOADS = ROWS * 8 / NT;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int P = kPart<MODE> * NT / BM;
    static_assert(ROWS * 8 % NT == 0 && BM * 8 % NT == 0, "whole rounds of loads");
    static_assert(FM % 4 == 0, "whole registers of scale bytes");
    using S = Scale<MODE>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][ROWS * 128];
    __shared__ __attribute__((aligned(16))) S panel[P][WM][16][FM];
    __shared__ S panel_b[P][BN / kBlock];
    const int tid = threadIdx.x, lane = tid & 63, l16 = tid & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const int64_t tiles_m = ceil_div(p.M, (int64_t)BM), tiles_n = ceil_div(p.N, (int64_t)BN);
    // eight tiles of A's rows at a time, all of B's
    int64_t id = xcd_tile(blockIdx.x, tiles_m * tiles_n);
    const int64_t first = id / (8 * tiles_n) * 8;
    const int64_t high = tiles_m - first < 8 ? tiles_m - first : 8;
    id -= first * tiles_n;
    const int64_t m0 = (first + id % high) * BM, n0 = id / high * BN;

    const uint8_t* base_a = p.a + m0 * p.lda;
    const uint8_t* base_b = p.b + n0 * p.ldb;
    const int rows_a = p.M - m0 < BM ? (int)(p.M - m0) : BM, rows_b = p.N - n0 < BN ? (int)(p.N - n0) : BN;
    const int c16 = 16 * ((tid & 7) ^ ((tid >> 4) & 7));
    uint32_t off[LOADS];
    row_offsets<BM, NT>(p, rows_a, rows_b, off);
    const int64_t whole = p.K / kBlock;   // blocks without a ragged end
    auto fetch = [&](int64_t kb, int buf) {
        rows_to_lds<BM, NT>((uint64_t)(base_a + kb * kBlock), (uint64_t)(base_b + kb * kBlock), off, lds[buf], wave);
    };
    auto fetch_end = [&](int64_t kb, int buf) {   // the last, ragged block: zeros past K
#pragma unroll 1
        for (int i = 0; i < LOADS; ++i) {
            const bool is_b = i * NT >= BM * 8;
            const int row = (i * NT + tid) / 8 - (is_b ? BM : 0), rows = is_b ? rows_b : rows_a;
            const uint8_t* s = (is_b ? base_b : base_a) +
                               (int64_t)(row < rows ? row : rows - 1) * (is_b ? p.ldb : p.lda);
            *reinterpret_cast<u32x4*>(&lds[buf][(i * NT + tid) * 16]) = load_codes(s, kb * kBlock + c16, p.K);
        }
    };
    auto fetch_panel = [&](int64_t kb) {
        scales_to_lds<MODE, BM, BN, NT>(p, m0, n0, rows_a, kb, panel, panel_b);
    };
    floatx4 acc[FN][FM] = {};
    fetch(0, 0);
    fetch_panel(0);
    const int lo = (g ^ (l16 >> 1)) * 16, hi = lo ^ 64;   // pieces g and g + 4
    for (int64_t kb = 0; kb < p.blocks; ++kb) {
        const int buf = (int)(kb & 1), k = (int)(kb % P);
        if (k == 0 && kb > 0) {
            __syncthreads();   // the last panel's readers are done
            fetch_panel(kb);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this step's rows are in LDS
        __syncthreads();
        if (kb + 1 < p.blocks) {
            if (kb + 1 < whole) fetch(kb + 1, buf ^ 1);
            else fetch_end(kb + 1, buf ^ 1);
        }
        const uint8_t* xrow = &lds[buf][(wm * (BM / WM) + l16) * 128];
        const uint8_t* wrow = &lds[buf][(BM + wn * (BN / WN) + l16) * 128];
        Frag<MODE> xq[FM];
#pragma unroll
        for (int j = 0; j < FM; ++j)
            xq[j].set(*reinterpret_cast<const u32x4*>(xrow + j * 2048 + lo),
                      *reinterpret_cast<const u32x4*>(xrow + j * 2048 + hi));
        S sa[FM];
        __builtin_memcpy(sa, panel[k][wm][l16], sizeof(sa));
        const S cb = panel_b[k][wn * (BN / WN) / kBlock];   // the wave's rows of B lie in one tile
        int words[FM / 4];
        float cs[FM];
        if constexpr (MODE == kBytes) {
            __builtin_memcpy(words, sa, sizeof(words));
        } else {
#pragma unroll
            for (int j = 0; j < FM; ++j) cs[j] = sa[j] * cb;
        }
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            Frag<MODE> wq;
            wq.set(*reinterpret_cast<const u32x4*>(wrow + i * 2048 + lo),
                   *reinterpret_cast<const u32x4*>(wrow + i * 2048 + hi));
            if constexpr (MODE == kBytes) {
#pragma unroll
                for (int j = 0; j < FM; j += 4) {
#define CDX_MFMA8(J) \
    acc[i][j + J] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wq.q, xq[j + J].q, acc[i][j + J], \
                                                                     0, 0, 0, cb, J, words[j / 4])
                    CDX_MFMA8(0);
                    CDX_MFMA8(1);
                    CDX_MFMA8(2);
                    CDX_MFMA8(3);
#undef CDX_MFMA8
                }
            } else {
#pragma unroll
                for (int j = 0; j < FM; ++j)
                    acc[i][j] = block_product<MODE>(wq, xq[j], acc[i][j], 0, 0, cs[j]);
            }
        }
    }
    store_rows<T, BM, BN, NT>(p, lds[0], m0, n0, wm * (BM / WM), wn * (BN / WN), acc);
}

// Few tiles: a CU has one workgroup or two, whose time is that of their
// loads on their way.  64 x 64 tiles, four waves along B's rows, four LDS buffers: three
// blocks are in flight.  Buffers of their own names tell the compiler that a block's reads
// need not wait for the later blocks' loads.  64 x 4096 x 4096 9.9 us (64 tiles: three of four
// CUs have none, and each of these goes through all of K), 512 x 4096 x 4096 14 to 16, 1.1 PFLOP/s
// and more.
template <class T, int MODE>
__global__ __launch_bounds__(256, 2)
void gemm8_ring_kernel(Params p) {
    constexpr int D = 4, NT = 256, SIDE = 64, LOADS = 2 * SIDE * 8 / NT, FM = SIDE / 16;
    constexpr int P = kPart<MODE> * NT / SIDE, SIZE = 2 * SIDE * 128;
    static_assert(P % D == 0, "whole rounds of buffers");
    static_assert(SIZE >= SIDE * SIDE * (int)sizeof(T), "the results fit one buffer");
    using S = Scale<MODE>;
    __shared__ __attribute__((aligned(1024))) uint8_t r0[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t r1[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t r2[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t r3[SIZE];
    __shared__ __attribute__((aligned(16))) S panel[P][1][16][FM];
    __shared__ S panel_b[P][1];
    const int tid = threadIdx.x, lane = tid & 63, l16 = tid & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t tiles_m = ceil_div(p.M, (int64_t)SIDE);
    const int64_t id = xcd_tile(blockIdx.x, tiles_m * ceil_div(p.N, (int64_t)SIDE));
    const int64_t m0 = id % tiles_m * SIDE, n0 = id / tiles_m * SIDE;
    const uint8_t* base_a = p.a + m0 * p.lda;
    const uint8_t* base_b = p.b + n0 * p.ldb;
    const int rows_a = p.M - m0 < SIDE ? (int)(p.M - m0) : SIDE;
    const int rows_b = p.N - n0 < SIDE ? (int)(p.N - n0) : SIDE;
    uint32_t off[LOADS];
    row_offsets<SIDE, NT>(p, rows_a, rows_b, off);
    const int64_t whole = p.K / kBlock;   // blocks without a ragged end
    auto fetch = [&](int64_t kb, uint8_t* buf) {
        // (past the last block the last one again, which nobody reads: the waits count loads)
        kb = kb < whole ? kb : whole - 1;
        rows_to_lds<SIDE, NT>((uint64_t)(base_a + kb * kBlock), (uint64_t)(base_b + kb * kBlock), off, buf, wave);
    };
    floatx4 acc[1][FM] = {};
    const int lo = (g ^ (l16 >> 1)) * 16, hi = lo ^ 64;   // pieces g and g + 4
    const int xoff = l16 * 128, woff = (SIDE + 16 * wave + l16) * 128;
    auto block = [&](const uint8_t* rows, int k) {
        auto frag = [&](int o) {
            Frag<MODE> f;
            f.set(*reinterpret_cast<const u32x4*>(rows + o + lo), *reinterpret_cast<const u32x4*>(rows + o + hi));
            return f;
        };
        const Frag<MODE> wq = frag(woff);
        S sa[FM];
        __builtin_memcpy(sa, panel[k][0][l16], sizeof(sa));
        const S sb = panel_b[k][0];
        Frag<MODE> xq[FM];
#pragma unroll
        for (int j = 0; j < FM; ++j) xq[j] = frag(xoff + j * 2048);
        if constexpr (MODE == kBytes) {
            int word;
            __builtin_memcpy(&word, sa, sizeof(word));
#define CDX_MFMA8(J) \
    acc[0][J] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wq.q, xq[J].q, acc[0][J], 0, 0, 0, sb, J, word)
            CDX_MFMA8(0);
            CDX_MFMA8(1);
            CDX_MFMA8(2);
            CDX_MFMA8(3);
#undef CDX_MFMA8
        } else {
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[0][j] = block_product<MODE>(wq, xq[j], acc[0][j], 0, 0, sa[j] * sb);
        }
    };
    fetch(0, r0);
    fetch(1, r1);
    fetch(2, r2);
    for (int64_t k0 = 0; k0 < whole; k0 += P) {
        const int count = whole - k0 < P ? (int)(whole - k0) : P;
        __syncthreads();   // the last panel's readers are done
        scales_to_lds<MODE, SIDE, SIDE, NT>(p, m0, n0, rows_a, k0, panel, panel_b);
        auto step = [&](int k, const uint8_t* now, uint8_t* last) {
            constexpr int N = (D - 2) * LOADS;
            // vmcnt(N) lgkmcnt(0): this block's rows are in LDS, and the last block's are read
            __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
            asm volatile("s_barrier" ::: "memory");
            fetch(k0 + k + D - 1, last);
            block(now, k);
        };
#pragma unroll 1
        for (int k = 0; k < count;) {
            step(k, r0, r3);
            if (++k == count) break;
            step(k, r1, r0);
            if (++k == count) break;
            step(k, r2, r1);
            if (++k == count) break;
            step(k, r3, r2);
            ++k;
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);   // nothing is on its way to LDS
    if (whole < p.blocks) {   // the ragged block: zeros past K
        __syncthreads();
        if (whole % P == 0) scales_to_lds<MODE, SIDE, SIDE, NT>(p, m0, n0, rows_a, whole, panel, panel_b);
#pragma unroll 1
        for (int i = 0; i < LOADS; ++i) {
            const bool is_b = i * NT >= SIDE * 8;
            const int row = (i * NT + tid) / 8 - (is_b ? SIDE : 0), rows = is_b ? rows_b : rows_a;
            const uint8_t* src = (is_b ? base_b : base_a) + (int64_t)(row < rows ? row : rows - 1) * (is_b ? p.ldb : p.lda);
            *reinterpret_cast<u32x4*>(r0 + (i * NT + tid) * 16) =
                load_codes(src, whole * kBlock + 16 * ((tid & 7) ^ ((tid >> 4) & 7)), p.K);
        }
        __syncthreads();
        block(r0, (int)(whole % P));
    }
    store_rows<T, SIDE, SIDE, NT>(p, r0, m0, n0, 0, 16 * wave, acc);
}

// Few rows of A: operands from global memory straight into registers, a block's
// 128 columns split over eight waves, whose sums meet in LDS in the order of the
// waves.  A workgroup takes 16 NT rows of B and 16 MT of A; each wave has the codes of
// U blocks in flight.  With X the rows of A are quantised here, as they are used:
// every workgroup does it again.  Bound by B's bytes, the latency of a launch, and A, which
// every workgroup reads whole: with 16 rows of 4096 columns its 256 workgroups take as many
// bytes of A out of L2 as of B.  4096 x 4096 with 1 row 4.8 us, 3.5 TB/s, 16 rows 7.1, 32 rows 9.7;
// from unquantised rows 1 row 7.1, 16 rows 9.0: their loads stand behind B's in the queue, so that
// quantising begins when B is there.
constexpr int kDirectWaves = 8;

// A lane's 32 values of a row and block as loaded: those of all rows are on their way before
// the first is quantised.
template <class X> struct RawRow {
    u32x4 u[4][sizeof(X) / 2];
    __device__ __forceinline__ void load(const X* x, int n) {   // the first n, then zeros
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (n >= 8 * j + 8) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(X) / 2; ++i)
                    u[j][i] = load16(reinterpret_cast<const char*>(x + 8 * j) + 16 * i);
            } else {
                X e[8] = {};
                if (n > 8 * j) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (8 * j + k < n) e[k] = x[8 * j + k];
                }
                __builtin_memcpy(u[j], e, sizeof(e));
            }
        }
    }
};

template <class X, int MODE>
__device__ __forceinline__ void quantize_frag(const RawRow<X>& raw, Frag<MODE>& f, int& e) {
    float v[4][8];
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        X t[8];
        __builtin_memcpy(t, raw.u[j], sizeof(t));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[j][k] = (float)t[k];
            m = fmaxf(m, finite_mag(v[j][k]));
        }
    }
    m = fmaxf(m, __shfl_xor(m, 16));   // the four lanes of a row and block
    m = fmaxf(m, __shfl_xor(m, 32));
    e = scale_exp(m);
    const float inv = exp_value(254 - e);
    u32x4 q[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[j >> 1][2 * (j & 1)] = pack_e4m3(v[j][0], v[j][1], v[j][2], v[j][3], inv);
        q[j >> 1][2 * (j & 1) + 1] = pack_e4m3(v[j][4], v[j][5], v[j][6], v[j][7], inv);
    }
    f.set(q[0], q[1]);
}

template <class T, int MODE, int MT, int NT, class X>
__global__ __launch_bounds__(64 * kDirectWaves)
void gemm8_direct_kernel(Params p, const X* __restrict__ x, int64_t ldx) {
    constexpr bool CODES = std::is_same_v<X, uint8_t>;
    constexpr int NW = kDirectWaves, U = MT * NT == 1 || (CODES && MT * NT == 2) ? 4 : 2;
    __shared__ floatx4 red[NW][NT * MT][64];
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tiles_n = ceil_div(p.N, (int64_t)(16 * NT));
    const int64_t n0 = blockIdx.x % tiles_n * (16 * NT), m0 = blockIdx.x / tiles_n * (16 * MT);
    // a lane's row of each operand tile (rows past the last read it again)
    const uint8_t *b[NT], *a[MT];
    const X* xr[MT];
    int64_t sa_row[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int64_t n = n0 + 16 * i + l16;
        b[i] = p.b + (n < p.N ? n : p.N - 1) * p.ldb;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        int64_t m = m0 + 16 * j + l16;
        m = m < p.M ? m : p.M - 1;
        a[j] = p.a + m * p.lda;
        xr[j] = x + m * ldx;
        sa_row[j] = m * p.ldsa;
    }
    const int64_t sb_row = n0 / kBlock * p.ldsb;
    floatx4 acc[NT][MT] = {};
    // (the kind of the scales outside the loop, whose loads a branch would end)
    auto sums = [&](auto ae, auto be) {
        constexpr bool AE = decltype(ae)::value, BE = decltype(be)::value;
        auto product = [&](int64_t kb, const Frag<MODE> (&wq)[NT], auto ragged) {
            constexpr bool RAGGED = decltype(ragged)::value;
            const int64_t k = kb * kBlock + 32 * g;
            int sb = 0;
            float fb = 0.0f;
            if constexpr (MODE == kBytes) sb = static_cast<const uint8_t*>(p.sb)[sb_row + kb];
            else fb = load_scale(p.sb, sb_row + kb, BE);
            RawRow<std::conditional_t<CODES, float, X>> raw[CODES ? 1 : MT];
            if constexpr (!CODES) {
                const int64_t left = RAGGED ? p.K - k : 32;
#pragma unroll
                for (int j = 0; j < MT; ++j) raw[j].load(xr[j] + k, left < 32 ? (int)left : 32);
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                Frag<MODE> xq;
                int sa = 0;
                float s = 0.0f;
                if constexpr (CODES) {
                    if constexpr (RAGGED) xq.set(load_codes(a[j], k, p.K), load_codes(a[j], k + 16, p.K));
                    else xq.set(load16(a[j] + k), load16(a[j] + k + 16));
                    if constexpr (MODE == kBytes) sa = static_cast<const uint8_t*>(p.sa)[sa_row[j] + kb];
                    else s = load_scale(p.sa, sa_row[j] + kb, AE);
                } else {
                    quantize_frag<X, MODE>(raw[j], xq, sa);
                    s = exp_value(sa);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i][j] = block_product<MODE>(wq[i], xq, acc[i][j], sa, sb, s * fb);
            }
        };
        const int64_t whole = p.K / kBlock;
        int64_t kb = wave;
        for (; kb + (U - 1) * NW < whole; kb += U * NW) {
            u32x4 w[U][NT][2];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint8_t* q = b[i] + (kb + u * NW) * kBlock + 32 * g;
                    w[u][i][0] = load16(q);
                    w[u][i][1] = load16(q + 16);
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                Frag<MODE> wq[NT];
#pragma unroll
                for (int i = 0; i < NT; ++i) wq[i].set(w[u][i][0], w[u][i][1]);
                product(kb + u * NW, wq, std::false_type{});
            }
        }
        for (; kb < p.blocks; kb += NW) {
            Frag<MODE> wq[NT];
            const int64_t k = kb * kBlock + 32 * g;
            if (kb < whole) {
#pragma unroll
                for (int i = 0; i < NT; ++i) wq[i].set(load16(b[i] + k), load16(b[i] + k + 16));
                product(kb, wq, std::false_type{});
            } else {
#pragma unroll
                for (int i = 0; i < NT; ++i) wq[i].set(load_codes(b[i], k, p.K), load_codes(b[i], k + 16, p.K));
                product(kb, wq, std::true_type{});
            }
        }
    };
    std::true_type yes;
    std::false_type no;
    if constexpr (MODE == kBytes) {
        sums(yes, yes);
    } else if constexpr (!CODES) {   // A's scales are made here
        if (MODE == kWide && p.b_e8m0) sums(yes, yes);
        else sums(no, no);
    } else if (p.a_e8m0) {
        if (MODE == kWide && p.b_e8m0) sums(yes, yes);
        else sums(yes, no);
    } else {
        if (p.b_e8m0) sums(no, yes);
        else sums(no, no);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) red[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < NT * MT; t += NW) {
        floatx4 v[1][1] = {{red[0][t][lane]}};
#pragma unroll
        for (int w = 1; w < NW; ++w) v[0][0] += red[w][t][lane];
        store_tile<T>(p, m0 + 16 * (t % MT), n0 + 16 * (t / MT), v);
    }
}

// K = 0: act(bias), a thread to a 16 x 16 tile's lane.
template <class T>
__global__ __launch_bounds__(64)
void gemm8_empty_kernel(Params p) {
    const floatx4 zero[1][1] = {};
    const int64_t tiles_m = ceil_div(p.M, (int64_t)16), n = tiles_m * ceil_div(p.N, (int64_t)16);
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x)
        store_tile<T>(p, i % tiles_m * 16, i / tiles_m * 16, zero);
}

// Calls f with the way a result type and scale types call for.
template <class T, class F> int with_mode(const Params& p, F f) {
    using std::integral_constant;
    if constexpr (std::is_same_v<T, float>) return f(integral_constant<int, kWide>{});
    else if (p.a_e8m0 && p.b_e8m0) return f(integral_constant<int, kBytes>{});
    else return f(integral_constant<int, kFloats>{});
}

// Which kernel (us, scale bytes, bf16 results).
// Straight from global memory: up to 32 rows (16 x 4096 x 4096 6.9, by the ring of buffers
// 9.8), more while 128 x 128 tiles would be few and K is short (256 x 1024 x 1024 5.3, 5.6),
// and where the ring needs an alignment that is not there (64 x 4096 x 4001 29.3, by the
// 64 x 64 tiles of any alignment 31.5).
bool is_direct(int64_t M, int64_t N) {
    return M <= 64 || ceil_div(M, (int64_t)128) * ceil_div(N, (int64_t)128) < 64;
}
// The ring: 64 x 64 tiles up to two a CU.  64 x 1024 x 4096 9.8, straight from global memory
// 14.7; 128 x 4096 x 4016 11.4, straight 19.7, by 128 x 128 tiles 25.4; 512 x 4096 x 4096 15.8,
// by 128 x 128 tiles 25.2; 300 x 8192 x 4096 (640 tiles) 23.7 and 25.8 with scale bytes but
// 31.9 and 31.2 with floats, 46 and 45 for 32 bits.
bool is_ring(int64_t M, int64_t N, int64_t K) {
    return M > 32 && ceil_div(M, (int64_t)64) * ceil_div(N, (int64_t)64) <= 512 &&
           (K >= 2048 || !is_direct(M, N));
}
// 256 x 256 tiles when they fill most of the CUs: 200 of them (2560 x 5120 x 1024) 23.1,
// with 128 x 128 tiles 25.5; 128 of them (2048 x 4096 x 2048) 32.7 and 23.0.
bool is_large(int64_t M, int64_t N) {
    return ceil_div(M, (int64_t)256) * ceil_div(N, (int64_t)256) >= 200;
}
// x quantised by every workgroup for itself instead of by a kernel before: up to 16 rows of
// 4096, more rows of shorter length.  On the device 16 x 4096 x 4096 9.0 and 9.2, 16 x 1024 x
// 1024 3.9 and 5.6, 32 x 1024 x 1024 5.4 and 6.2, 64 x 4096 x 512 6.5 and 6.3 (but one launch
// and no workspace: calls from Python 8.9 and 14); 8 x 8192 x 8192 21.7 and 18.7, 17 x 4096 x
// 3840 11.4 and 8.8.  All of these are direct from codes too: the bits are the same.
bool quantizes_inside(int64_t M, int64_t K) {
    return M <= 64 && K <= 4096 && M * K <= (M <= 16 ? 65536 : 49152);
}

// The kernel of a product; `aligned`: rows of both operands begin at 16-byte addresses; `wide`:
// 32-bit results.
enum class Kernel { Empty, Direct, Ring, Tile128, Tile256, Any };
Kernel kernel_of(int64_t M, int64_t N, int64_t K, bool aligned, bool wide) {
    if (K == 0) return Kernel::Empty;
    aligned = aligned && K >= kBlock;
    if (aligned && is_ring(M, N, K)) return Kernel::Ring;
    if (is_direct(M, N)) return Kernel::Direct;
    if (!aligned) return Kernel::Any;
    return !wide && is_large(M, N) ? Kernel::Tile256 : Kernel::Tile128;
}

template <class T, class X>
int run_direct(const Params& p, const X* x, int64_t ldx, hipStream_t stream) {
    return with_mode<T>(p, [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        auto go = [&](auto mt, auto nt) {
            constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
            const int64_t grid = ceil_div(p.M, (int64_t)(16 * MT)) * ceil_div(p.N, (int64_t)(16 * NT));
            if (!grid_fits(grid, 64 * kDirectWaves))
                return set_error(CDX_ERR_UNSUPPORTED, "gemm8: too many output tiles");
            hipLaunchKernelGGL((gemm8_direct_kernel<T, MODE, MT, NT, X>), dim3((unsigned)grid),
                               dim3(64 * kDirectWaves), 0, stream, p, x, ldx);
            return hip_error(hipGetLastError(), "gemm8_direct_kernel launch");
        };
        using std::integral_constant;
        if (p.M <= 16) return go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
        if (p.M <= 32) return go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
        return go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    });
}

template <class T>
int run(const Params& p, hipStream_t stream) {
    const bool aligned = p.lda % 16 == 0 && p.ldb % 16 == 0 && ((uintptr_t)p.a | (uintptr_t)p.b) % 16 == 0 &&
                         p.lda <= kMaxLd && p.ldb <= kMaxLd;
    const Kernel kernel = kernel_of(p.M, p.N, p.K, aligned, std::is_same_v<T, float>);
    if (kernel == Kernel::Empty) {
        const int64_t g = ceil_div(p.M, (int64_t)16) * ceil_div(p.N, (int64_t)16);
        hipLaunchKernelGGL(gemm8_empty_kernel<T>, dim3((unsigned)(g < 65536 ? g : 65536)), dim3(64), 0,
                           stream, p);
        return hip_error(hipGetLastError(), "gemm8_empty_kernel launch");
    }
    const int64_t big = ceil_div(p.M, (int64_t)256) * ceil_div(p.N, (int64_t)256);
    const int64_t mid = ceil_div(p.M, (int64_t)128) * ceil_div(p.N, (int64_t)128);
    const int64_t grid = ceil_div(p.M, (int64_t)64) * ceil_div(p.N, (int64_t)64);
    if (!grid_fits(grid, 256)) return set_error(CDX_ERR_UNSUPPORTED, "gemm8: too many output tiles");
    if (kernel == Kernel::Ring) {
        return with_mode<T>(p, [&](auto mode) {
            hipLaunchKernelGGL((gemm8_ring_kernel<T, decltype(mode)::value>), dim3((unsigned)grid), dim3(256),
                               0, stream, p);
            return hip_error(hipGetLastError(), "gemm8_ring_kernel launch");
        });
    }
    if (kernel == Kernel::Direct) return run_direct<T>(p, static_cast<const uint8_t*>(nullptr), (int64_t)0, stream);
    return with_mode<T>(p, [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        if constexpr (MODE != kWide) {
            if (kernel == Kernel::Tile256) {
                hipLaunchKernelGGL((gemm8_tile_kernel<T, MODE, 256, 256, 2, 4>), dim3((unsigned)big),
                                   dim3(512), 0, stream, p);
                return hip_error(hipGetLastError(), "gemm8_tile_kernel launch");
            }
        }
        if (kernel == Kernel::Tile128)
            hipLaunchKernelGGL((gemm8_tile_kernel<T, MODE, 128, 128, 2, 2>), dim3((unsigned)mid),
                               dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL((gemm8_any_kernel<T, MODE>), dim3((unsigned)grid), dim3(256), 0, stream, p);
        return hip_error(hipGetLastError(), "gemm8 kernel launch");
    });
}

// Where a launch quantises x itself: codes, then scales behind them.
int64_t codes_ld(int64_t K) { return ceil_div(K, (int64_t)16) * 16; }
size_t codes_bytes(int64_t M, int64_t K) { return ((size_t)M * (size_t)codes_ld(K) + 255) / 256 * 256; }

}  // namespace

size_t gemm8_workspace(int64_t M, int64_t N, int64_t K, bool from_x) {
    (void)N;
    if (!from_x || M == 0 || K == 0 || quantizes_inside(M, K)) return 0;
    return codes_bytes(M, K) + (size_t)M * (size_t)ceil_div(K, (int64_t)kBlock) * 4;
}

const char* gemm8_kernel_name(int64_t M, int64_t N, int64_t K, bool aligned, bool wide, bool from_x) {
    if (from_x && K > 0 && quantizes_inside(M, K)) return "direct, quantises";
    static const char* const names[] = {"empty", "direct", "ring", "tile 128", "tile 256", "any"};
    return names[(int)kernel_of(M, N, K, aligned, wide)];
}

int launch_gemm8(const Gemm8Args& g, hipStream_t stream) {
    const int64_t blocks = ceil_div(g.K, (int64_t)kBlock);
    Params p{g.a.q, g.b.q, g.a.s, g.b.s, g.M, g.N, g.K, g.a.ldq, g.b.ldq, g.a.lds, g.b.lds, g.ldc,
             blocks, g.a.e8m0, g.b.e8m0, g.C, g.bias, g.epilogue};
    if (g.x && g.K > 0 && quantizes_inside(g.M, g.K)) {
        p.a_e8m0 = p.b_e8m0;   // (the way of the same product from codes)
        return with_dtype(g.cdtype, [&](auto t) {
            return with_dtype(g.xdtype, [&](auto xt) {
                using X = decltype(xt);
                return run_direct<decltype(t)>(p, static_cast<const X*>(g.x), g.ldx, stream);
            });
        });
    }
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
