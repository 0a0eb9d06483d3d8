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

// A wave's F operands of the instruction, from the tile's 16 rows (columns) number `first` on: a lane
// has eight k (8 g + 0..7 of the step's half h) of row `l16`.
template <bool COLS, int EXT, int F> struct Reader {
    int at[COLS ? F : 2];
    __device__ __forceinline__ Reader(int lane, int first) {
        const int l16 = lane & 15, g = lane >> 4;
        if constexpr (COLS) {
            const int row = 8 * g + (l16 >> 2);
#pragma unroll
            for (int i = 0; i < F; ++i) {
                const int u = first + i, swap = unit_swap<EXT>(row);   // (the swap leaves u's high bits)
                at[i] = row * (2 * EXT) + 32 * (u ^ swap) + 8 * (l16 & 3);
            }
        } else {
            at[0] = first * 2048 + l16 * 128 + (g ^ (l16 >> 1)) * 16;
            at[1] = at[0] ^ 64;
        }
    }
    __device__ __forceinline__ shortx8 operator()(const uint8_t* tile, int i, int h) const {
        if constexpr (COLS) {
            typedef __attribute__((address_space(3))) shortx4* P3;
            const uint8_t* p = tile + h * (64 * EXT) + at[i];
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)p);
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)(p + 8 * EXT));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const shortx8*>(tile + i * 2048 + at[h]);
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

// ---- results ---------------------------------------------------------------------------------

// Eight sums of row m from column n on (the first `count` exist) through bias, activation and residual.
template <class T, int ACT>
__device__ __forceinline__ void finish8(const Linear16Out& o, int64_t m, int64_t n, int count,
                                        float (&v)[8], const float (&bias)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += bias[j];
    if (o.z) store_n<8>(static_cast<T*>(o.z) + m * o.ldz + n, count, v);
    float r[8] = {};
    if (o.residual) load_n<8>(static_cast<const T*>(o.residual) + m * o.ldr + n, count, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = act_value<T, ACT>(v[j], 0.0f);
    if (o.residual) {   // (adding a zero would turn -0 into 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
    }
    store_n<8>(static_cast<T*>(o.y) + m * o.ldy + n, count, v);
}

template <class T>
__device__ __forceinline__ void load_bias(const Linear16Out& o, int64_t n, int count, float (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.0f;
    if (!o.bias || count <= 0) return;
    if (o.bias_f32) load_n<8>(static_cast<const float*>(o.bias) + n, count, b);
    else load_n<8>(static_cast<const T*>(o.bias) + n, count, b);
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
                each([&](int64_t m, float (&v)[8]) { finish8<T, decltype(act)::value>(p.out, m, n, count, v, bias); });
            });
        } else {
            each([&](int64_t m, float (&v)[8]) {
                store_n<8>(static_cast<T*>(p.out.y) + m * p.out.ldy + n, count, v);
            });
        }
    }
}

// ---- the product -------------------------------------------------------------------------------

// A wave's products of a step, in halves of 32 k.  SUMS: the column sums of A as well, its product with
// ones, which the WN waves that hold the same fragments of A share.
template <class T, bool CA, bool CB, int BM, int BN, int WM, int WN> struct Wave {
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    static constexpr bool SUMS = CA && CB;
    static constexpr int FS = (FM + WN - 1) / WN;   // fragments whose sums a wave forms
    floatx4 acc[FN][FM] = {};
    floatx4 ones[SUMS ? FS : 1] = {};
    shortx8 fa[FM], fb[FN];
    const int wm, wn;
    const bool sums;
    Reader<CA, BM, FM> ra;
    Reader<CB, BN, FN> rb;
    __device__ __forceinline__ Wave(int lane, int wave, bool sums_)
        : wm(wave % WM), wn(wave / WM), sums(sums_), ra(lane, wave % WM * FM), rb(lane, wave / WM * FN) {}
    template <int H> __device__ __forceinline__ void read(const uint8_t* tile) {
#pragma unroll
        for (int i = 0; i < FN; ++i) fb[i] = rb(tile + BM * 128, i, H);
#pragma unroll
        for (int j = 0; j < FM; ++j) fa[j] = ra(tile, j, H);
    }
    __device__ __forceinline__ void multiply() {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = mfma<T>(fb[i], fa[j], acc[i][j]);
        if constexpr (SUMS) {
            if (sums) {
                const short one = std::is_same_v<T, bf16> ? 0x3f80 : 0x3c00;
                const shortx8 v = {one, one, one, one, one, one, one, one};
#pragma unroll
                for (int q = 0; q < WN; ++q) {
                    if (wn != q) continue;
#pragma unroll
                    for (int f = 0; f < FS; ++f)
                        if (q * FS + f < FM) ones[f] = mfma<T>(v, fa[q * FS + f], ones[f]);
                }
            }
        }
    }
    // The sums of column m0 + 16 j + lane of A, in every row of the product.
    __device__ __forceinline__ void store_sums(const Params& p, int64_t m0, int lane) const {
        if (!sums || lane >= 16) return;
#pragma unroll
        for (int f = 0; f < FS; ++f) {
            const int j = wn * FS + f;
            const int64_t m = m0 + 16 * (wm * FM + j) + lane;
            if (j >= FM || m >= p.M) continue;
            if (p.col_sums) p.col_sums[(int64_t)blockIdx.y * p.M + m] = ones[f][0];
            else static_cast<T*>(p.col_y)[m] = (T)ones[f][0];
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

// The workgroup's k, and whether it forms the column sums of A.
struct Slice {
    int64_t k0, k1, whole;             // whole: steps without a ragged end
    __device__ __forceinline__ explicit Slice(const Params& p) {
        k0 = (int64_t)blockIdx.y * p.chunk;
        k1 = k0 + p.chunk < p.K ? k0 + p.chunk : p.K;
        whole = k1 > k0 ? (k1 - k0) / kStep : 0;
    }
};
__device__ __forceinline__ bool forms_sums(const Params& p, int64_t n0) { return (p.col_sums || p.col_y) && n0 == 0; }

// Operands of any alignment: every step through registers, the next one's loads in flight while one is
// multiplied.
template <class T, bool CA, bool CB, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN)
void linear16_any_kernel(Params p) {
    constexpr int NT = 64 * WM * WN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[(BM + BN) * 128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t m0, n0;
    tile_of<BM, BN>(p, m0, n0);
    const Slice sl(p);
    Loader<CA, BM, NT> la(p.a, p.lda, m0, p.M);
    Loader<CB, BN, NT> lb(p.b, p.ldb, n0, p.N);
    Wave<T, CA, CB, BM, BN, WM, WN> w(lane, wave, forms_sums(p, n0));
    typename Loader<CA, BM, NT>::Held ha;
    typename Loader<CB, BN, NT>::Held hb;
    if (sl.k0 < sl.k1) {
        la.load(sl.k0, sl.k1, ha);
        lb.load(sl.k0, sl.k1, hb);
    }
    for (int64_t k = sl.k0; k < sl.k1; k += kStep) {
        __syncthreads();
        la.store(ha, lds);
        lb.store(hb, lds + BM * 128);
        __syncthreads();
        if (k + kStep < sl.k1) {
            la.load(k + kStep, sl.k1, ha);
            lb.load(k + kStep, sl.k1, hb);
        }
        w.template read<0>(lds);
        w.multiply();
        w.template read<1>(lds);
        w.multiply();
    }
    constexpr int ROWS = (BM + BN) * 128 / (BN * 4) < BM ? (BM + BN) * 128 / (BN * 4) : BM;
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
    constexpr int ROWS = (BM + BN) * 128 / (BN * 4) < BM ? (BM + BN) * 128 / (BN * 4) : BM;
    store_tile<T, !CA && !CB, BM, BN, WM, WN, ROWS>(p, buf, m0, n0, w.wm, w.wn, w.acc);
    if constexpr (W::SUMS) w.store_sums(p, m0, lane);
}

// Aligned operands, whole steps straight into LDS, D buffers of their own names (which tells the compiler
// that a step's reads need not wait for the later steps' loads): D - 1 steps are in flight, one
// barrier a step.
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
    Wave<T, CA, CB, BM, BN, WM, WN> w(lane, wave, forms_sums(p, n0));
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
    Wave<T, CA, CB, BM, BN, WM, WN> w(lane, wave, forms_sums(p, n0));
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

// ---- launches ------------------------------------------------------------------------------------

enum class Kernel { Any, Ring, Tile128, Turns };
struct Plan { Kernel kernel; int64_t tiles; int slices; int64_t chunk; };

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
        case Kernel::Ring:
            hipLaunchKernelGGL((linear16_tile_kernel<T, CA, CB, 64, 64, 2, 2, 4>), grid, dim3(256), 0, stream, p);
            break;
        case Kernel::Any:
            hipLaunchKernelGGL((linear16_any_kernel<T, CA, CB, 64, 64, 2, 2>), grid, dim3(256), 0, stream, p);
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
