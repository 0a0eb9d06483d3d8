// The kernels of a Linear layer in 16 bits, for the three products of a layer:
//   forward   y[m,n]  = sum_k x[m,k] w[n,k]       both operands' rows hold consecutive k
//   input     dx[m,n] = sum_k dz[m,k] w[k,n]      w's columns do
//   weight    dw[m,n] = sum_k dz[k,m] x[k,n]      both operands' columns do
//
// A step is 64 of k.  A tile's rows of 64 lie in LDS as eight 16-byte pieces, piece ^ (row / 2 & 7), so
// that the 16 rows that the hardware reads at a time are on all 64 banks; an operand whose columns hold
// k lies there as in memory, [k][extent], its 32-byte units exchanged by four bits of k, and
// ds_read_b64_tr_b16 gives each lane four k of its column.  Both layouts are exchanges of 16-byte pieces on
// the side of the global addresses, which go straight into LDS (16-byte rows) or through registers (any
// alignment, and the ragged end of k: zeros).
//
// B is the matrix instruction's first operand and A its second: a lane holds four consecutive n of one m.
//
// Sums are fp32 from the first product to the one rounding of a result; the gradient behind an activation,
// dz, is rounded to 16 bits, as the matrix instruction's operand: two of them, of its rounded value and of the
// rest, would double the products.  What that rounding gives is all of the gradients' distance from 32-bit slopes
// (8192 x 4096 x 4096 in bf16 2.6e-3 of their norm, 8e-5 where those are rounded too).  The bias gradient, which no
// matrix instruction forms then, is summed before it (linear16.hip).
#pragma once

#include "linear16.hpp"

namespace cdx {
namespace l16 {

using namespace b8;

typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;             // k a step
constexpr int64_t kMaxLd = 1 << 21;   // 256 rows within 32-bit byte offsets

struct Params {
    const uint16_t* a; const uint16_t* b;
    int64_t M, N, K, lda, ldb;
    int64_t chunk;                    // k a slice, whole steps
    Linear16Out out;
    float* col_sums;                  // fp32 column sums of A, slice s at col_sums + s * M,
    void* col_y;                      // or 16-bit ones
};

template <class T>
__device__ __forceinline__ floatx4 mfma(shortx8 b, shortx8 a, floatx4 c) {
    if constexpr (std::is_same_v<T, bf16>)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b),
                                                       __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b),
                                                      __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}

// The same with the sum kept in its registers: the compiler's own form gives each product a new place for
// its result, which 32 of them a wave do not leave room for.  What reads the sums otherwise has to call
// settle_sums first.
template <class T> __device__ __forceinline__ void mfma_in_place(shortx8 b, shortx8 a, floatx4& c) {
    if constexpr (std::is_same_v<T, bf16>)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(b), "v"(a));
    else
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(c) : "v"(b), "v"(a));
}

// Waits until the last products are written (a result is there 19 wait states after its instruction, at most).
template <int N, int M> __device__ __forceinline__ void settle_sums(floatx4 (&c)[N][M]) {
    asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) asm volatile("" : "+v"(c[i][j]));   // (reads come behind it)
}

// ---- an operand's tile of EXT rows (or columns) and one step in LDS ---------------------------

// What the 32-byte units of a row of k are exchanged by: rows 0 to 3 and 8 to 11 (4 to 7 and 12 to 15),
// which 32 lanes read together, differ in it and in the half of the banks that they begin at.
template <int EXT> __device__ __forceinline__ int unit_swap(int k) {
    return EXT == 64 ? (k >> 1 & 1) | (k >> 2 & 2) : (k & 3) | (k >> 1 & 4);
}

// Where LDS's 16-byte piece `at` of a tile comes from: element e of row r of what memory holds.
template <bool COLS, int EXT> __device__ __forceinline__ void piece_source(int at, int& r, int& e) {
    if constexpr (COLS) {
        r = at / (EXT / 8);
        const int pos = at % (EXT / 8);
        e = 8 * (((pos >> 1) ^ unit_swap<EXT>(r)) << 1 | (pos & 1));
    } else {
        r = at >> 3;
        e = 8 * ((at & 7) ^ (r >> 1 & 7));
    }
}

// A wave's F operands of the instruction, from the tile's 16 rows (columns) number `first` (a multiple of
// F) on: a lane has eight k (8 g + 0..7 of the step's half H) of row `l16`.
template <bool COLS, int EXT, int F> struct Reader {
    int at;
    __device__ __forceinline__ Reader(int lane, int first) {
        const int l16 = lane & 15, g = lane >> 4;
        if constexpr (COLS) {
            const int row = 8 * g + (l16 >> 2);
            at = row * (2 * EXT) + 32 * (first ^ unit_swap<EXT>(row)) + 8 * (l16 & 3);
        } else {
            at = first * 2048 + l16 * 128 + (g ^ (l16 >> 1)) * 16;
        }
    }
    template <int H> __device__ __forceinline__ void read(const uint8_t* tile, shortx8 (&f)[F]) const {
        int base = at;
        // (addresses are formed where they are used: kept over the loop, they would not fit the registers)
        if constexpr (COLS) asm volatile("" : "+v"(base));
#pragma unroll
        for (int i = 0; i < F; ++i) {
            if constexpr (COLS) {
                typedef __attribute__((address_space(3))) shortx4* P3;
                const uint8_t* p = tile + H * (64 * EXT) + (base ^ (32 * i));
                const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)p);
                const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)(p + 8 * EXT));
                f[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                f[i] = *reinterpret_cast<const shortx8*>(tile + i * 2048 + (base ^ (64 * H)));
            }
        }
    }
};

// A tile's way into LDS, EXT * 8 pieces by NT threads.
template <bool COLS, int EXT, int NT> struct Loader {
    static constexpr int LOADS = EXT * 8 / NT;
    static_assert(EXT * 8 % NT == 0, "whole rounds of loads");
    const uint16_t* p;     // the tile's first row (or column) at k = 0
    int64_t ld, step;      // elements between rows, and from one step to the next
    int extent;            // rows (columns) of the tile that exist
    uint32_t off[LOADS];   // bytes from the step's first element
    __device__ __forceinline__ Loader(const uint16_t* base, int64_t ld_, int64_t first, int64_t all)
        : p(base + (COLS ? first : first * ld_)), ld(ld_), step(COLS ? kStep * ld_ : kStep),
          extent(all - first < EXT ? (int)(all - first) : EXT) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            int r, e;
            piece_source<COLS, EXT>(i * NT + threadIdx.x, r, e);
            // rows past the last one read it again, and what they give is not stored
            if (COLS) e = e < extent ? e : (extent - 1) & ~7;
            else r = r < extent ? r : extent - 1;
            off[i] = 2 * ((uint32_t)r * (uint32_t)ld + (uint32_t)e);
        }
    }
    // One whole step straight into LDS.
    __device__ __forceinline__ void fetch(int64_t k, uint8_t* buf, int wave) const {
        typedef const __attribute__((address_space(1))) uint32_t* G;
        typedef const __attribute__((address_space(1))) uint8_t* G8;
        typedef __attribute__((address_space(3))) uint32_t* L;
        // (kept apart from the offsets: scalar base + 32-bit offset, one VGPR a load)
        uint64_t at = (uint64_t)(p + (COLS ? k * ld : k));
        asm("" : "+s"(at));
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            uint32_t o = off[i];
            asm("" : "+v"(o));
            __builtin_amdgcn_global_load_lds((G)((G8)at + o), (L)(buf + (i * NT + wave * 64) * 16), 16, 0, 0);
        }
    }
    // A step through registers: nothing past k_end or the tile's extent is read.
    struct Held { u32x4 v[LOADS]; };
    __device__ __forceinline__ void load(int64_t k, int64_t k_end, Held& held) const {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            int r, e;
            piece_source<COLS, EXT>(i * NT + threadIdx.x, r, e);
            const int64_t left = k_end - k;
            const int rows = COLS ? (left < kStep ? (int)left : kStep) : extent;
            const int cols = COLS ? extent : (left < kStep ? (int)left : kStep);
            const int n = r < rows ? cols - e : 0;
            const uint16_t* s = p + (COLS ? (k + r) * ld + e : (int64_t)r * ld + k + e);
            if (n >= 8) {
                held.v[i] = load16(s);
            } else {
                uint16_t t[8] = {};
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (j < n) t[j] = s[j];
                __builtin_memcpy(&held.v[i], t, 16);
            }
        }
    }
    __device__ __forceinline__ void store(const Held& held, uint8_t* buf) const {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            *reinterpret_cast<u32x4*>(buf + (i * NT + threadIdx.x) * 16) = held.v[i];
    }
};

// ---- activations -----------------------------------------------------------------------------

// The activation and grad times its slope.  ReLU lets NaN through, as the others do by themselves: a layer that
// turned NaN shows it.
template <class T, int ACT> __device__ __forceinline__ float layer_value(float v) {
    if constexpr (ACT == CDX_EPI_RELU) return v <= 0.0f ? 0.0f : v;
    else return act_value<T, ACT>(v, 0.0f);
}
template <class T, int ACT> __device__ __forceinline__ float layer_slope(float g, float v) {
    if constexpr (ACT == CDX_EPI_RELU) return v <= 0.0f ? 0.0f : g;
    else return act_slope<T, ACT>(g, v, 0.0f);
}

// ---- results ---------------------------------------------------------------------------------

// W sums of row m from column n on (the first `count` exist) through bias, activation and residual.
template <class T, int ACT, int W>
__device__ __forceinline__ void finish(const Linear16Out& o, int64_t m, int64_t n, int count,
                                       float (&v)[W], const float (&bias)[W]) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] += bias[j];
    if (o.z) store_n<W>(static_cast<T*>(o.z) + m * o.ldz + n, count, v);
    float r[W] = {};
    if (o.residual) load_n<W>(static_cast<const T*>(o.residual) + m * o.ldr + n, count, r);
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = layer_value<T, ACT>(v[j]);
    if (o.residual) {   // (adding a zero would turn -0 into 0)
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] += r[j];
    }
    store_n<W>(static_cast<T*>(o.y) + m * o.ldy + n, count, v);
}

template <class T, int W>
__device__ __forceinline__ void load_bias(const Linear16Out& o, int64_t n, int count, float (&b)[W]) {
#pragma unroll
    for (int j = 0; j < W; ++j) b[j] = 0.0f;
    if (!o.bias || count <= 0) return;
    if (o.bias_f32) load_n<W>(static_cast<const float*>(o.bias) + n, count, b);
    else load_n<W>(static_cast<const T*>(o.bias) + n, count, b);
}

// Calls f with the epilogue's code as a constant.
template <class F> __device__ __forceinline__ void with_epilogue(int act, F f) {
    using std::integral_constant;
    switch (act) {
        case CDX_EPI_RELU: f(integral_constant<int, CDX_EPI_RELU>{}); break;
        case CDX_EPI_GELU: f(integral_constant<int, CDX_EPI_GELU>{}); break;
        case CDX_EPI_SILU: f(integral_constant<int, CDX_EPI_SILU>{}); break;
        case CDX_EPI_SIGMOID: f(integral_constant<int, CDX_EPI_SIGMOID>{}); break;
        default: f(integral_constant<int, CDX_EPI_NONE>{}); break;
    }
}

// A workgroup's BM x BN sums through LDS (`buf`, ROWS rows of fp32 at a time), so that a thread has eight
// consecutive n of a row: whole 16-byte loads of the residual and stores of the results, and bias,
// activation and residual in fp32 before the one rounding.  Row r's 16-byte units lie at
// unit ^ 4 (r & 15).
template <class T, bool EPI, int BM, int BN, int WM, int WN, int ROWS>
__device__ __forceinline__ void store_tile(const Params& p, uint8_t* buf, int64_t m0, int64_t n0,
                                           int wm, int wn, const floatx4 (&acc)[BN / WN / 16][BM / WM / 16]) {
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16, NT = 64 * WM * WN, PARTS = BM / ROWS;
    constexpr int SWAP = BN / 16 - 1 < 15 ? BN / 16 - 1 : 15;   // (BN / 4 units)
    static_assert(PARTS % WM == 0 || WM % PARTS == 0, "a wave's rows lie in whole parts");
    constexpr int SPLIT = PARTS > WM ? PARTS / WM : 1;          // parts of a wave's rows
    constexpr int JP = FM / SPLIT;
    const int l16 = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    constexpr int CHUNKS = BN / 8;
    const int c = threadIdx.x % CHUNKS, r0 = threadIdx.x / CHUNKS;
    const int64_t n = n0 + 8 * c, left = p.N - n;
    const int count = left < 0 ? 0 : left > 8 ? 8 : (int)left;
    float bias[8];
    if constexpr (EPI) load_bias<T>(p.out, n, count, bias);
    float* sums = p.out.sums ? p.out.sums + (int64_t)blockIdx.y * p.M * p.N : nullptr;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        __syncthreads();
        const int first = part * ROWS;   // the tile's row that `buf` begins with
        if (wm * (BM / WM) < first + ROWS && (wm + 1) * (BM / WM) > first) {
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int jj = 0; jj < JP; ++jj) {
                    const int j = (SPLIT > 1 ? part % SPLIT * JP : 0) + jj;
                    const int r = wm * (BM / WM) + 16 * j + l16 - first;
                    const int unit = (wn * (BN / WN) / 4 + 4 * i + g) ^ (4 * (l16 & SWAP));
                    *reinterpret_cast<floatx4*>(buf + (r * (BN / 4) + unit) * 16) = acc[i][j];
                }
        }
        __syncthreads();
        const int64_t rest = p.M - m0 - first;
        const int rows = rest < ROWS ? (int)rest : ROWS;
        auto each = [&](auto sink) {
#pragma unroll 2
            for (int r = r0; r < rows; r += NT / CHUNKS) {
                float v[8];
                const int unit = (2 * c) ^ (4 * (r & SWAP));
                const floatx4* u = reinterpret_cast<const floatx4*>(buf) + r * (BN / 4) + unit;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = u[0][j];
                    v[4 + j] = u[1][j];
                }
                sink(m0 + first + r, v);
            }
        };
        if (count <= 0) continue;
        if (sums) {
            each([&](int64_t m, float (&v)[8]) { store_n<8>(sums + m * p.N + n, count, v); });
        } else if constexpr (EPI) {
            with_epilogue(p.out.act, [&](auto act) {
                each([&](int64_t m, float (&v)[8]) { finish<T, decltype(act)::value>(p.out, m, n, count, v, bias); });
            });
        } else {
            each([&](int64_t m, float (&v)[8]) {
                store_n<8>(static_cast<T*>(p.out.y) + m * p.out.ldy + n, count, v);
            });
        }
    }
}

// ---- the product -------------------------------------------------------------------------------

// A wave's products of a step, in halves of 32 k.  SUMS: the column sums of A as well, a lane's eight k of
// its column at a time (the vector unit has nothing else to do).  The workgroups of all tiles of B, and the WN
// waves that hold the same fragments of A, share the fragments, so that none has much more to do than the
// others (weight gradient of 8192 x 4096 x 4096 with all sums in the first tile's workgroups 233 us, so 215,
// without any 216).
template <class T, bool CA, bool CB, int BM, int BN, int WM, int WN, bool IN_PLACE = false> struct Wave {
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    static constexpr bool SUMS = CA && CB;
    static constexpr int FS = (FM + WN - 1) / WN;   // fragments whose sums a wave forms
    floatx4 acc[FN][FM] = {};
    float sums[SUMS ? FS : 1] = {};
    shortx8 fa[FM], fb[FN];
    const int wm, wn;
    int mine = 0;                                   // bit f: the sums of fragment wn FS + f are this wave's
    Reader<CA, BM, FM> ra;
    Reader<CB, BN, FN> rb;
    __device__ __forceinline__ Wave(const Params& p, int lane, int wave, int64_t n0)
        : wm(wave % WM), wn(wave / WM), ra(lane, wave % WM * FM), rb(lane, wave / WM * FN) {
        if constexpr (SUMS) {
            if (!p.col_sums && !p.col_y) return;
            const int64_t tiles = p.N > BN ? ceil_div(p.N, (int64_t)BN) : 1;
            const int every = tiles < 1024 ? (int)tiles : 1024, at = (int)(n0 / BN);
#pragma unroll
            for (int f = 0; f < FS; ++f)
                if (wn * FS + f < FM && (f * WM * WN + wave) % every == at) mine |= 1 << f;
        }
    }
    template <int H> __device__ __forceinline__ void read(const uint8_t* tile) {
        rb.template read<H>(tile + BM * 128, fb);
        ra.template read<H>(tile, fa);
    }
    __device__ __forceinline__ void multiply() {
        if constexpr (IN_PLACE) asm volatile("s_nop 1");   // (an operand that was moved rather than read is there)
#pragma unroll
        for (int i = 0; i < FN; ++i) {
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                if constexpr (IN_PLACE) mfma_in_place<T>(fb[i], fa[j], acc[i][j]);
                else acc[i][j] = mfma<T>(fb[i], fa[j], acc[i][j]);
            }
            if constexpr (SUMS)
                if (i == 0 && mine) add_sums();
        }
    }
    __device__ __forceinline__ void add_sums() {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            if (wn != j / FS || !(mine & (1 << j % FS))) continue;
            T e[8];
            __builtin_memcpy(e, &fa[j], 16);
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += (float)e[k];
            sums[j % FS] += s;
        }
    }
    __device__ __forceinline__ void settle() {
        if constexpr (IN_PLACE) settle_sums(acc);
    }
    // A column's sum lies in the four lanes that share it.
    __device__ __forceinline__ void store_sums(const Params& p, int64_t m0, int lane) const {
#pragma unroll
        for (int f = 0; f < FS; ++f) {
            if (!(mine & (1 << f))) continue;
            float v = sums[f];
            v += __shfl_xor(v, 16);
            v += __shfl_xor(v, 32);
            const int64_t m = m0 + 16 * (wm * FM + wn * FS + f) + (lane & 15);
            if (lane >= 16 || m >= p.M) continue;
            if (p.col_sums) p.col_sums[(int64_t)blockIdx.y * p.M + m] = v;
            else static_cast<T*>(p.col_y)[m] = (T)v;
        }
    }
};

// Which tile a workgroup takes: eight tiles of A's at a time, all of B's, neighbours on one XCD.
template <int BM, int BN> __device__ __forceinline__ void tile_of(const Params& p, int64_t& m0, int64_t& n0) {
    const int64_t tiles_m = ceil_div(p.M, (int64_t)BM);
    const int64_t tiles_n = p.N > 0 ? ceil_div(p.N, (int64_t)BN) : 1;
    int64_t id = xcd_tile(blockIdx.x, tiles_m * tiles_n);
    const int64_t first = id / (8 * tiles_n) * 8;
    const int64_t high = tiles_m - first < 8 ? tiles_m - first : 8;
    id -= first * tiles_n;
    m0 = (first + id % high) * BM;
    n0 = id / high * BN;
}

// The workgroup's k.
struct Slice {
    int64_t k0, k1, whole;             // whole: steps without a ragged end
    __device__ __forceinline__ explicit Slice(const Params& p) {
        k0 = (int64_t)blockIdx.y * p.chunk;
        k1 = k0 + p.chunk < p.K ? k0 + p.chunk : p.K;
        whole = k1 > k0 ? (k1 - k0) / kStep : 0;
    }
};

// Operands of any alignment: every step through registers into the LDS buffer that is not being read, the
// step after it on its way meanwhile; one barrier a step.  The loads' checks and the way through registers
// bound it: 4096 x 4096 x 4001 in 128 x 128 tiles of eight waves 183 to 203 us from card to card, 734 to 660 TFLOP/s (aligned operands
// of 4096, turns: 127).
template <class T, bool CA, bool CB, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN)
void linear16_any_kernel(Params p) {
    constexpr int NT = 64 * WM * WN, SIZE = (BM + BN) * 128;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SIZE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t m0, n0;
    tile_of<BM, BN>(p, m0, n0);
    const Slice sl(p);
    Loader<CA, BM, NT> la(p.a, p.lda, m0, p.M);
    Loader<CB, BN, NT> lb(p.b, p.ldb, n0, p.N);
    Wave<T, CA, CB, BM, BN, WM, WN> w(p, lane, wave, n0);
    typename Loader<CA, BM, NT>::Held ha;
    typename Loader<CB, BN, NT>::Held hb;
    auto load = [&](int64_t k) {
        if (k >= sl.k1) return;
        la.load(k, sl.k1, ha);
        lb.load(k, sl.k1, hb);
    };
    auto store = [&](uint8_t* buf) {
        la.store(ha, buf);
        lb.store(hb, buf + BM * 128);
    };
    load(sl.k0);
    if (sl.k0 < sl.k1) store(lds);
    load(sl.k0 + kStep);
    int buf = 0;
    for (int64_t k = sl.k0; k < sl.k1; k += kStep, buf ^= SIZE) {
        __syncthreads();   // this step's rows are in LDS, and the last step's are read
        if (k + kStep < sl.k1) {
            store(lds + (buf ^ SIZE));
            load(k + 2 * kStep);
        }
        w.template read<0>(lds + buf);
        w.multiply();
        w.template read<1>(lds + buf);
        w.multiply();
    }
    constexpr int ROWS = 2 * SIZE / (BN * 4) < BM ? 2 * SIZE / (BN * 4) : BM;
    store_tile<T, !CA && !CB, BM, BN, WM, WN, ROWS>(p, lds, m0, n0, w.wm, w.wn, w.acc);
    if constexpr (w.SUMS) w.store_sums(p, m0, lane);
}

// The ragged end of k through registers, and the results.
template <class T, bool CA, bool CB, int BM, int BN, int WM, int WN, class W, class LA, class LB>
__device__ __forceinline__ void finish_tile(const Params& p, const Slice& sl, W& w, const LA& la, const LB& lb,
                                            uint8_t* buf, int64_t m0, int64_t n0, int lane) {
    if (sl.k0 + sl.whole * kStep < sl.k1) {
        typename LA::Held ha;
        typename LB::Held hb;
        la.load(sl.k0 + sl.whole * kStep, sl.k1, ha);
        lb.load(sl.k0 + sl.whole * kStep, sl.k1, hb);
        __syncthreads();
        la.store(ha, buf);
        lb.store(hb, buf + BM * 128);
        __syncthreads();
        w.template read<0>(buf);
        w.multiply();
        w.template read<1>(buf);
        w.multiply();
    }
    w.settle();
    constexpr int FIT = (BM + BN) * 128 / (BN * 4);   // rows of sums that the buffer holds
    constexpr int ROWS = FIT >= BM ? BM : FIT >= BM / 2 ? BM / 2 : BM / 4;
    static_assert(ROWS <= FIT, "rows of sums fit the buffer");
    store_tile<T, !CA && !CB, BM, BN, WM, WN, ROWS>(p, buf, m0, n0, w.wm, w.wn, w.acc);
    if constexpr (W::SUMS) w.store_sums(p, m0, lane);
}

// Aligned operands, whole steps straight into LDS, D buffers of their own names (which tells the compiler
// that a step's reads need not wait for the later steps' loads): D - 1 steps are in flight, one
// barrier a step.  What bounds them, at 64 x 64 x 4 buffers: a step of four waves is short beside its barrier
// and the loads' way (one workgroup a CU, 1280 x 1280 x 1280: 10.2 us, 0.5 us a step; eight buffers
// are no faster), for which a CU does better with one of 128 x 64 and eight waves than with two of 64 x 64 (8192 x
// 256 x 784 10.4 us against 12.1); at 128 x 128: LDS reads, as many as matrix instructions have slots for (2048 x 2048 x
// 2048 with eight waves and four buffers, alone on a CU, 21.2 us, 810 TFLOP/s; two workgroups a CU with two
// buffers each hide each other's barriers, 2560 x 4608 x 1024 34 us, 710 TFLOP/s).
template <class T, bool CA, bool CB, int BM, int BN, int WM, int WN, int D>
__global__ __launch_bounds__(64 * WM * WN, 2)
void linear16_tile_kernel(Params p) {
    constexpr int NT = 64 * WM * WN, SIZE = (BM + BN) * 128;
    static_assert(D == 2 || D == 4, "two or four buffers");
    __shared__ __attribute__((aligned(1024))) uint8_t r0[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t r1[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t r2[D == 4 ? SIZE : 16];
    __shared__ __attribute__((aligned(1024))) uint8_t r3[D == 4 ? SIZE : 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t m0, n0;
    tile_of<BM, BN>(p, m0, n0);
    const Slice sl(p);
    const int64_t whole = sl.whole;
    Loader<CA, BM, NT> la(p.a, p.lda, m0, p.M);
    Loader<CB, BN, NT> lb(p.b, p.ldb, n0, p.N);
    constexpr int LOADS = Loader<CA, BM, NT>::LOADS + Loader<CB, BN, NT>::LOADS;
    Wave<T, CA, CB, BM, BN, WM, WN> w(p, lane, wave, n0);
    auto fetch = [&](int64_t s, uint8_t* buf) {
        // (past the last step that one again, which nobody reads: the waits count loads)
        s = s < whole ? s : whole - 1;
        la.fetch(sl.k0 + s * kStep, buf, wave);
        lb.fetch(sl.k0 + s * kStep, buf + BM * 128, wave);
    };
    auto step = [&](int64_t s, const uint8_t* now, uint8_t* last) {
        constexpr int N = (D - 2) * LOADS;
        // vmcnt(N) lgkmcnt(0): this step's rows are in LDS, and the last step's are read
        __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
        asm volatile("s_barrier" ::: "memory");
        fetch(s + D - 1, last);
        __builtin_amdgcn_sched_barrier(0);   // (the compiler would issue the loads between the last products)
        w.template read<0>(now);
        w.multiply();
        w.template read<1>(now);
        w.multiply();
    };
    if (whole > 0) {
        fetch(0, r0);
        if constexpr (D == 4) {
            fetch(1, r1);
            fetch(2, r2);
        }
        int64_t s = 0;
#pragma unroll 1
        for (; s + D <= whole; s += D) {
            step(s, r0, D == 4 ? r3 : r1);
            step(s + 1, r1, r0);
            if constexpr (D == 4) {
                step(s + 2, r2, r1);
                step(s + 3, r3, r2);
            }
        }
        if (s < whole) step(s, r0, D == 4 ? r3 : r1);
        if constexpr (D == 4) {
            if (s + 1 < whole) step(s + 1, r1, r0);
            if (s + 2 < whole) step(s + 2, r2, r1);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);   // nothing is on its way to LDS
    finish_tile<T, CA, CB, BM, BN, WM, WN>(p, sl, w, la, lb, r0, m0, n0, lane);
}

// The same with eight waves in two groups (a wave of each on every SIMD) that take turns: while one
// group's operands come out of LDS, the other multiplies, a barrier between the phases.  A step is four phases
// (read, multiply, read, multiply); the second group is a phase behind.  The next step's loads are
// issued in the first phase, when the step before is read to its end by both groups, and waited for before
// the barrier that ends the step for the first group.
//
// 256 x 256 is the widest tile whose sums (128 registers a lane) and operands stay in registers: a step's LDS
// reads are half of a 128 x 128 tile's for the same products.  Measured, bf16, 8192 x 4096 x 4096, from card
// to card: forward 207 to 234 us (1330 to 1175 TFLOP/s; a library product 174 to 198; with bias, residual, GELU and z 262),
// input gradient 204 to 222, weight gradient with bias sums 212 to 224; 4096 x 4096 x 4096 110 to 119.  The energy of LDS
// reads and matrix units bounds it: operands of zeros take 163 us (1690 TFLOP/s), and the clock is 2.4 GHz then,
// 1.9 to 2.2 with random ones, of whose cycles matrix instructions take 50 to 57 %.
template <class T, bool CA, bool CB>
__global__ __launch_bounds__(512, 2)
void linear16_turns_kernel(Params p) {
    constexpr int BM = 256, BN = 256, WM = 2, WN = 4, NT = 512, SIZE = (BM + BN) * 128;
    __shared__ __attribute__((aligned(1024))) uint8_t r0[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t r1[SIZE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t m0, n0;
    tile_of<BM, BN>(p, m0, n0);
    const Slice sl(p);
    const int64_t whole = sl.whole;
    Loader<CA, BM, NT> la(p.a, p.lda, m0, p.M);
    Loader<CB, BN, NT> lb(p.b, p.ldb, n0, p.N);
    Wave<T, CA, CB, BM, BN, WM, WN, true> w(p, lane, wave, n0);
    const bool second = wave >= 4;
    auto fetch = [&](int64_t s, uint8_t* buf) {
        s = s < whole ? s : whole - 1;   // (nobody reads it then)
        la.fetch(sl.k0 + s * kStep, buf, wave);
        lb.fetch(sl.k0 + s * kStep, buf + BM * 128, wave);
    };
    auto barrier = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&]() {
        __builtin_amdgcn_s_setprio(1);
        w.multiply();
        __builtin_amdgcn_s_setprio(0);
    };
    auto step = [&](int64_t s, uint8_t* now, uint8_t* next) {
        w.template read<0>(now);
        __builtin_amdgcn_sched_barrier(0);
        fetch(s + 1, next);
        barrier();
        multiply();
        barrier();
        w.template read<1>(now);
        // lgkmcnt(0): what was read is there before the other group may write over it; vmcnt(0)
        if (second) __builtin_amdgcn_s_waitcnt(0x0070);
        else __builtin_amdgcn_s_waitcnt(0xc07f);
        barrier();
        multiply();
        if (!second) __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
        barrier();
    };
    if (whole > 0) {
        fetch(0, r0);
        __builtin_amdgcn_s_waitcnt(0x0070);
        barrier();
        if (second) barrier();
        int64_t s = 0;
#pragma unroll 1
        for (; s + 2 <= whole; s += 2) {
            step(s, r0, r1);
            step(s + 1, r1, r0);
        }
        if (s < whole) step(s, r0, r1);
        if (!second) barrier();
    }
    __builtin_amdgcn_s_waitcnt(0x0070);   // nothing is on its way to LDS
    __syncthreads();
    finish_tile<T, CA, CB, BM, BN, WM, WN>(p, sl, w, la, lb, r0, m0, n0, lane);
}

// Few rows of x (both operands' rows hold k): operands from global memory straight into registers, any
// alignment, the inner size split over eight waves in chunks of 64, whose sums meet in LDS in the order
// of the waves.  A workgroup takes 16 columns and 16 MT rows; a wave has the weights of U chunks in
// flight.  The weights' way bounds it: 1 x 4096 x 4096 in bf16 6.6 us of a launch among others, 5.1 TB/s
// (37 x 1000 x 1200 in f16 4.5).
constexpr int kDirectWaves = 8;

template <class T, int MT>
__global__ __launch_bounds__(64 * kDirectWaves)
void linear16_direct_kernel(Params p) {
    constexpr int NW = kDirectWaves, U = 8 / MT;
    __shared__ floatx4 red[NW][MT][64];
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tiles_n = ceil_div(p.N, (int64_t)16);
    const int64_t n0 = blockIdx.x % tiles_n * 16, m0 = blockIdx.x / tiles_n * (16 * MT);
    // a lane's row of each operand tile (rows past the last read it again)
    const uint16_t* b = p.b + (n0 + l16 < p.N ? n0 + l16 : p.N - 1) * p.ldb + 8 * g;
    const uint16_t* a[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int64_t m = m0 + 16 * j + l16;
        a[j] = p.a + (m < p.M ? m : p.M - 1) * p.lda + 8 * g;
    }
    auto piece = [&](const uint16_t* s, int64_t k) {   // eight k from k + 8 g on, zeros past K
        const int64_t left = p.K - k - 8 * g;
        if (left >= 8) return load16(s + k);
        uint16_t t[8] = {};
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < left) t[j] = s[k + j];
        u32x4 v;
        __builtin_memcpy(&v, t, 16);
        return v;
    };
    floatx4 acc[MT] = {};
    auto multiply = [&](const u32x4 (&w)[2], const u32x4 (&x)[MT][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < MT; ++j)
                acc[j] = mfma<T>(__builtin_bit_cast(shortx8, w[h]), __builtin_bit_cast(shortx8, x[j][h]), acc[j]);
    };
    const int64_t whole = p.K / 64, chunks = ceil_div(p.K, (int64_t)64);
    int64_t c = wave;
    for (; c + (U - 1) * NW < whole; c += U * NW) {
        u32x4 w[U][2], x[U][MT][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[u][h] = load16(b + (c + u * NW) * 64 + 32 * h);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) x[u][j][h] = load16(a[j] + (c + u * NW) * 64 + 32 * h);
        __builtin_amdgcn_sched_barrier(0);   // (all of them on their way before the first is used)
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(w[u], x[u]);
    }
#pragma unroll 1
    for (; c < chunks; c += NW) {
        u32x4 w[2], x[MT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            w[h] = piece(b, c * 64 + 32 * h);
#pragma unroll
            for (int j = 0; j < MT; ++j) x[j][h] = piece(a[j], c * 64 + 32 * h);
        }
        multiply(w, x);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) red[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= MT) return;
    floatx4 sum = red[0][wave][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum += red[w][wave][lane];
    const int64_t m = m0 + 16 * wave + l16, n = n0 + 4 * g, left = p.N - n;
    const int count = left < 0 ? 0 : left > 4 ? 4 : (int)left;
    if (m >= p.M || count == 0) return;
    float bias[4], v[4] = {sum[0], sum[1], sum[2], sum[3]};
    load_bias<T>(p.out, n, count, bias);
    with_epilogue(p.out.act, [&](auto act) { finish<T, decltype(act)::value>(p.out, m, n, count, v, bias); });
}

// ---- launches ------------------------------------------------------------------------------------

enum class Kernel { Any, Any128, Ring64, Ring128, Tile128, Turns, Direct, Tall };
struct Plan { Kernel kernel; int64_t tiles; int slices; int64_t chunk; int mt = 1; };   // mt: Direct's MT

template <class F> int with_16(int dtype, F f) {
    return dtype == CDX_DTYPE_BF16 ? f(bf16{}) : f(f16{});
}

template <class T, bool CA, bool CB>
int run(const Params& p, const Plan& pl, hipStream_t stream) {
    const dim3 grid((unsigned)pl.tiles, (unsigned)pl.slices);
    switch (pl.kernel) {
        case Kernel::Turns:
            hipLaunchKernelGGL((linear16_turns_kernel<T, CA, CB>), grid, dim3(512), 0, stream, p);
            break;
        case Kernel::Tile128:
            hipLaunchKernelGGL((linear16_tile_kernel<T, CA, CB, 128, 128, 2, 2, 2>), grid, dim3(256), 0, stream, p);
            break;
        case Kernel::Ring128:
            hipLaunchKernelGGL((linear16_tile_kernel<T, CA, CB, 128, 128, 2, 4, 4>), grid, dim3(512), 0, stream, p);
            break;
        case Kernel::Ring64:
            hipLaunchKernelGGL((linear16_tile_kernel<T, CA, CB, 64, 64, 2, 2, 4>), grid, dim3(256), 0, stream, p);
            break;
        case Kernel::Tall:
            hipLaunchKernelGGL((linear16_tile_kernel<T, CA, CB, 128, 64, 4, 2, 4>), grid, dim3(512), 0, stream, p);
            break;
        case Kernel::Any128:
            hipLaunchKernelGGL((linear16_any_kernel<T, CA, CB, 128, 128, 2, 4>), grid, dim3(512), 0, stream, p);
            break;
        case Kernel::Any:
            hipLaunchKernelGGL((linear16_any_kernel<T, CA, CB, 64, 64, 2, 2>), grid, dim3(256), 0, stream, p);
            break;
        case Kernel::Direct:
            if constexpr (!CA && !CB) {
                const dim3 threads(64 * kDirectWaves);
                if (pl.mt == 1) hipLaunchKernelGGL((linear16_direct_kernel<T, 1>), grid, threads, 0, stream, p);
                else if (pl.mt == 2) hipLaunchKernelGGL((linear16_direct_kernel<T, 2>), grid, threads, 0, stream, p);
                else hipLaunchKernelGGL((linear16_direct_kernel<T, 4>), grid, threads, 0, stream, p);
            }
            break;
    }
    return hip_error(hipGetLastError(), "linear16 kernel launch");
}

// The products of one kind each (files of their own, which compile at the same time).
int run_forward(int dtype, const Params& p, const Plan& pl, hipStream_t stream);
int run_input(int dtype, const Params& p, const Plan& pl, hipStream_t stream);
int run_weight(int dtype, const Params& p, const Plan& pl, hipStream_t stream);

}  // namespace l16
}  // namespace cdx
