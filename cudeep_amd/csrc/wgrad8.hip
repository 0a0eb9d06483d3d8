// The weight gradient of a Linear layer whose input was kept in 8 bits:
//   dw[n,k] = sum over m of dz[m,n] xh[m,k],   db[n] = sum over m of dz[m,n],
// xh = code * scale with a scale byte for each 128 columns of a row.
//
// xh is exact in bf16 (three fraction bits times a power of two), so it is one
// bf16 operand; dz is split into bf16 parts that hold it exactly: one part for
// bf16, two for f16 (11 bits), three for f32 (24 bits; below 2^-110 the last part
// may lose bits).  Every product is then exact in fp32 and the sums are fp32, so
// the gradient is that of the restored input with no rounding but the sums'.  Each part is an
// addition of its own to a sum: in fp32 64 x 250 x 333 is 1.1e-7 of the norm away from 64 bits, 8192 x
// 256 x 784 1.8e-7.
//
// Both operands have the sum's index m as their slow one.  Tiles lie in LDS as they
// do in memory, [m][n] and [m][k], and ds_read_b64_tr_b16 gives each lane the four m of
// its column: 16 lanes read 32 bytes of each of four rows, and a row's 32-byte
// units are exchanged so that the eight rows of 32 lanes lie on different banks.
// The next step's loads are in flight while a step is multiplied; two buffers, one
// barrier a step.  Few output tiles: m is split over workgroups, whose partials a second
// kernel adds in a fixed order.
//
// 8192 x 4096 x 4096: bf16 238 to 262 us, 1.1 PFLOP/s; f16 435, fp32 592 (two and three products
// each).  No unit is full (matrix slots 45 % busy, LDS 28, VALU 27, at 2.1 GHz): a step's loads,
// staging and products meet at its barrier.  8192 x 256 x 784 in fp32 24 and 6 for its partials,
// bound by traffic: its 448 workgroups read 73 MB past the L2s where the operands hold 15 (the
// tiles of a slice lie on all XCDs), and the partials are 26 MB written and read.
#include "block8.hpp"

namespace cdx {
namespace {

using namespace b8;

typedef short shortx4 __attribute__((ext_vector_type(4)));

template <class T> constexpr int kParts = std::is_same_v<T, float> ? 3 : std::is_same_v<T, f16> ? 2 : 1;

struct Params {
    const void* dz; int64_t lddz;
    const uint8_t* q; int64_t ldq;
    const uint8_t* s; int64_t lds;
    int64_t M, N, K;
    int64_t chunk;             // m per slice, a multiple of a step
    float* dw; float* db;      // slice z at dw + z * N * K, db + z * N
};

// The bf16 parts of eight values as four registers each: a part is the rest
// rounded to bf16, and the rest after it exact.  Values that round to an
// infinity are split apart from the others: infinities and NaN have no rest, and
// the largest finite ones begin with their leading bits instead.
template <int PARTS>
__device__ __forceinline__ void split_parts(const float (&v)[8], u32x4 (&out)[PARTS]) {
    float r[8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        r[j] = v[j];
        const uint32_t u = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
    const bool special = PARTS > 1 && top >= 0x7f7f8000u;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w = pack_bf16(r[2 * j], r[2 * j + 1]);
            if (q == 0 && special) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t u = __builtin_bit_cast(uint32_t, r[2 * j + h]);
                    const uint32_t mag = u & 0x7fffffffu;
                    if (mag >= 0x7f7f8000u && mag < 0x7f800000u)
                        w = h ? (w & 0xffffu) | (u & 0xffff0000u) : (w & 0xffff0000u) | (u >> 16);
                }
            }
            out[q][j] = w;
            if (q + 1 < PARTS) {
                r[2 * j] -= __builtin_bit_cast(float, w << 16);
                r[2 * j + 1] -= __builtin_bit_cast(float, w & 0xffff0000u);
            }
        }
        if (q == 0 && special) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(__builtin_fabsf(v[j]) < __builtin_inff())) r[j] = 0.0f;
        }
    }
}

// Eight codes times their scale as bf16 (exact).
__device__ __forceinline__ u32x4 restore_bf16(u32x2 w, float scale) {
    u32x4 o;
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, true));
    return o;
}

// Eight 16- or 32-bit values as loaded.
template <class T> struct Raw {
    u32x4 u[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = load16(reinterpret_cast<const char*>(p) + 16 * i);
    }
    __device__ __forceinline__ void load(const T* p, int n) {   // the first n, then zeros
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = u32x4{0u, 0u, 0u, 0u};
        if (n >= 8) {
            load(p);
        } else if (n > 0) {
            T e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = j < n ? p[j] : T(0);
            __builtin_memcpy(u, e, sizeof(e));
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        T e[8];
        __builtin_memcpy(e, u, sizeof(e));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)e[j];
    }
};

// What a row's 32-byte units are exchanged by: rows 0 to 3 and 8 to 11 (4 to 7 and 12 to
// 15), which 32 lanes read together, differ in it and in the half of the 64
// banks that they begin at (rows of 64 columns).
template <int COLS> __device__ __forceinline__ int unit_swap(int m) {
    return COLS == 64 ? (m >> 1 & 1) | (m >> 2 & 2) : (m & 3) | (m >> 1 & 4);
}

// BN x BK output tiles, WN x WK waves, MS (a multiple of 32) m a step.
template <class T, int BN, int BK, int WN, int WK, int MS>
__global__ __launch_bounds__(64 * WN * WK)
void wgrad8_kernel(Params p) {
    constexpr int PARTS = kParts<T>, NT = 64 * WN * WK;
    constexpr int FN = BN / WN / 16, FK = BK / WK / 16;
    __shared__ __attribute__((aligned(128))) uint16_t zs[2][PARTS][MS][BN];
    __shared__ __attribute__((aligned(128))) uint16_t xs[2][MS][BK];
    const int tid = threadIdx.x, l16 = tid & 15, g = (tid >> 4) & 3;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wk = wave / WN;
    const int64_t tiles_n = ceil_div(p.N, (int64_t)BN);
    // four tiles of n at a time, all of k: an XCD's tiles share more of dz (fp32 8192 x 4096 x
    // 4096 592 us, one column of tiles after the other 631; bf16 262 and 261)
    int64_t id = xcd_tile(blockIdx.x, gridDim.x);
    const int64_t tiles_k = gridDim.x / tiles_n, first = id / (4 * tiles_k) * 4;
    const int64_t wide = tiles_n - first < 4 ? tiles_n - first : 4;
    id -= first * tiles_k;
    const int64_t n0 = (first + id % wide) * BN, k0 = id / wide * BK;
    const int64_t m_begin = (int64_t)blockIdx.y * p.chunk;
    const int64_t m_end = m_begin + p.chunk < p.M ? m_begin + p.chunk : p.M;
    // a thread stages eight columns (zc, xc) of rows zr, zr + ZR, ... (xr, xr + XR, ...)
    constexpr int ZR = NT / (BN / 8), XR = NT / (BK / 8), ZI = MS / ZR, XI = MS / XR;
    static_assert(MS % ZR == 0 && MS % XR == 0 && ZR % 16 == 0 && XR % 16 == 0, "whole rounds of rows");
    const int zp = tid % (BN / 8), zr = tid / (BN / 8), zc = 8 * zp;
    const int xp = tid % (BK / 8), xr = tid / (BK / 8), xc = 8 * xp;
    const int zpos = 16 * (((zp >> 1) ^ unit_swap<BN>(zr)) << 1 | (zp & 1));   // bytes in an LDS row
    const int xpos = 16 * (((xp >> 1) ^ unit_swap<BK>(xr)) << 1 | (xp & 1));
    const int64_t z_left = p.N - n0 - zc, x_left = p.K - k0 - xc;
    const int zn = z_left < 0 ? 0 : z_left > 8 ? 8 : (int)z_left;
    const int xn = x_left < 0 ? 0 : x_left > 8 ? 8 : (int)x_left;
    const bool inner = n0 + BN <= p.N && k0 + BK <= p.K;
    const bool sums = p.db && k0 == 0;
    const T* zsrc = static_cast<const T*>(p.dz) + (m_begin + zr) * p.lddz + n0 + zc;
    const uint8_t* xsrc = p.q + (m_begin + xr) * p.ldq + k0 + xc;
    const uint8_t* ssrc = p.s + (m_begin + xr) * p.lds + (k0 + xc) / kBlock;
    const int64_t zstep = ZR * p.lddz, xstep = XR * p.ldq, sstep = XR * p.lds;
    Raw<T> zv[ZI];
    u32x2 xv[XI];
    uint32_t sv[XI];
    float bsum[8] = {};
    auto load = [&](int64_t m) {   // rows m .. m + MS - 1; advances the sources
        if (inner && m + MS <= m_end) {
#pragma unroll
            for (int i = 0; i < ZI; ++i) zv[i].load(zsrc + i * zstep);
#pragma unroll
            for (int i = 0; i < XI; ++i) {
                xv[i] = load8b(xsrc + i * xstep);
                sv[i] = ssrc[i * sstep];
            }
        } else {
#pragma unroll
            for (int i = 0; i < ZI; ++i) zv[i].load(zsrc + i * zstep, m + zr + i * ZR < m_end ? zn : 0);
#pragma unroll
            for (int i = 0; i < XI; ++i) {
                const int n = m + xr + i * XR < m_end ? xn : 0;
                u32x2 w = {0u, 0u};
                if (n == 8) {
                    w = load8b(xsrc + i * xstep);
                } else {
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (j < n) w[j >> 2] |= (uint32_t)xsrc[i * xstep + j] << (8 * (j & 3));
                }
                xv[i] = w;
                sv[i] = n > 0 ? ssrc[i * sstep] : 127;
            }
        }
        zsrc += ZI * zstep;
        xsrc += XI * xstep;
        ssrc += XI * sstep;
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < ZI; ++i) {
            float v[8];
            if (PARTS > 1 || sums) zv[i].get(v);
            u32x4 parts[PARTS];
            if constexpr (PARTS == 1) parts[0] = zv[i].u[0];
            else split_parts<PARTS>(v, parts);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
                *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(zs[buf][q][zr + i * ZR]) + zpos) = parts[q];
            if (sums) {
#pragma unroll
                for (int j = 0; j < 8; ++j) bsum[j] += v[j];
            }
        }
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            u32x2 w = xv[i];
            if (sv[i] == 255) w = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};   // a NaN scale: NaN codes
            *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(xs[buf][xr + i * XR]) + xpos) =
                restore_bf16(w, e8m0_value(sv[i]));
        }
    };
    // operand of lane (l16, g): column l16 of a unit, m = 8 g + 0..7 of 32, as two reads of
    // four rows; lane i of 16 points at row i / 4, columns 4 (i % 4)
    static_assert(BN == BK, "one set of unit offsets");
    constexpr int UNITS = BN == 64 ? 4 : 8;   // exchanged among each other
    const int row = 8 * g + (l16 >> 2);
    int unit[UNITS];
#pragma unroll
    for (int b = 0; b < UNITS; ++b) unit[b] = 32 * (b ^ unit_swap<BN>(row)) + 8 * (l16 & 3);
    auto operand = [&](const uint16_t* tile, int pitch, int u) {   // tile: row 0 of 32 m; unit u
        typedef __attribute__((address_space(3))) shortx4* P3;
        const char* at = reinterpret_cast<const char*>(tile) + row * pitch + u / UNITS * (32 * UNITS) + unit[u % UNITS];
        const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)at);
        const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)(at + 4 * pitch));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    floatx4 acc[FN][FK] = {};
    if (m_begin < m_end) {
        load(m_begin);
        stage(0);
        if (m_begin + MS < m_end) load(m_begin + MS);
    }
    // Half of the waves stage the next step before their products and half after them: a
    // SIMD's two waves are then at different work.
    const bool early = wave < WN * WK / 2;
    int buf = 0;
    for (int64_t m = m_begin; m < m_end; m += MS, buf ^= 1) {
        __syncthreads();   // this step's tiles are whole, and nobody reads the other buffer
        if (early && m + MS < m_end) {
            stage(buf ^ 1);
            if (m + 2 * MS < m_end) load(m + 2 * MS);
        }
#pragma unroll
        for (int h = 0; h < MS / 32; ++h) {
            bf16x8 xo[FK];
#pragma unroll
            for (int j = 0; j < FK; ++j) xo[j] = operand(xs[buf][32 * h], 2 * BK, wk * FK + j);
            // smallest parts first, as the larger ones then round their sum once; an
            // operand of dz is read ahead of the products of the one before it
            auto dz_operand = [&](int t) {   // t-th of PARTS * FN
                return operand(zs[buf][PARTS - 1 - t / FN][32 * h], 2 * BN, wn * FN + t % FN);
            };
            bf16x8 zo[2];
            zo[0] = dz_operand(0);
#pragma unroll
            for (int t = 0; t < PARTS * FN; ++t) {
                if (t + 1 < PARTS * FN) zo[(t + 1) & 1] = dz_operand(t + 1);
                __builtin_amdgcn_sched_barrier(0);   // (the compiler would read it after them)
#pragma unroll
                for (int j = 0; j < FK; ++j)
                    acc[t % FN][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(zo[t & 1], xo[j], acc[t % FN][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!early && m + MS < m_end) {
            stage(buf ^ 1);
            if (m + 2 * MS < m_end) load(m + 2 * MS);
        }
    }
    float* dw = p.dw + (int64_t)blockIdx.y * p.N * p.K;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t n = n0 + 16 * (wn * FN + i) + 4 * g + r;
            float* out = dw + n * p.K + k0 + 16 * wk * FK + l16;
#pragma unroll
            for (int j = 0; j < FK; ++j)
                if (n < p.N && k0 + 16 * (wk * FK + j) + l16 < p.K) out[16 * j] = acc[i][j][r];
        }
    if (sums) {
        // the staging threads' sums of a column, added in the order of their rows
        __syncthreads();
        float* red = reinterpret_cast<float*>(zs);
        static_assert(sizeof(zs) >= ZR * BN * sizeof(float), "room for the sums");
#pragma unroll
        for (int j = 0; j < 8; ++j) red[zr * BN + zc + j] = bsum[j];
        __syncthreads();
        for (int c = tid; c < BN; c += NT) {
            if (n0 + c >= p.N) break;
            float a = red[c];
            for (int i = 1; i < ZR; ++i) a += red[i * BN + c];
            p.db[(int64_t)blockIdx.y * p.N + n0 + c] = a;
        }
    }
}

// Partials of dw and of db (behind all of dw's), added in the order of the slices.
__global__ __launch_bounds__(256)
void wgrad8_sum_kernel(const float* __restrict__ part, int slices, int64_t nk, int64_t n_db,
                       float* __restrict__ dw, float* __restrict__ db) {
    const int64_t total = nk + n_db;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const bool is_db = i >= nk;
        const float* p = is_db ? part + slices * nk + (i - nk) : part + i;
        const int64_t step = is_db ? n_db : nk;
        float v = p[0];
        int s = 1;
        for (; s + 7 < slices; s += 8) {
            float t[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) t[u] = p[(s + u) * step];
#pragma unroll
            for (int u = 0; u < 8; ++u) v += t[u];
        }
        for (; s < slices; ++s) v += p[s * step];
        if (is_db) db[i - nk] = v;
        else dw[i] = v;
    }
}

// Tiles of 256, 128 or 64 by as many, and slices of m.
struct Plan { int side; int64_t tiles; int slices; int64_t chunk; };

constexpr int kMost = 64;   // m of the longest step

// (a layer without inputs still has its bias's column of tiles)
int64_t tiles_of(int64_t N, int64_t K, int side) {
    return ceil_div(N, (int64_t)side) * (K > 0 ? ceil_div(K, (int64_t)side) : 1);
}

// Sides (us, bf16 where nothing else is said): 256 where 256 workgroups get a tile or 1024 m
// and more each.  256 and 128: 8192 x 1024 x 4096 98 and 123, 16384 x 1024 x 1024 65 and 67, 256
// x 4096 x 4096 21.5 and 23.6; with 512 m each, 4096 x 2048 x 1024 47 and 42 (f16 62 and 66).
// 128 likewise where they get 192 m, or two tiles: 128 and 64, 4096 x 256 x 784 20.5 and 19.6,
// in fp32 22.9 and 25.9, 64 x 2048 x 4096 9.8 and 11.8; with less 2048 x 256 x 784 15.9 and
// 12.9, 512 x 1024 x 1024 13.0 and 9.3.
// Slices: one workgroup a CU of side 256, which fills LDS; two of the others (8192 x 256 x
// 784 23.7, with one 25.6, in fp32 31.1 and 33.7; 4096 x 768 x 768 23.5 and 22.2, in f16 28.9
// and 31.2), but one slice of as many tiles as CUs (1024 x 2048 x 2048 f16 36.8, two 42.5).
Plan plan_of(int64_t M, int64_t N, int64_t K) {
    int side = 64;
    const int64_t big = tiles_of(N, K, 256), mid = tiles_of(N, K, 128);
    const int64_t m = M < 1024 * 256 ? M : 1024 * 256;   // (their products stay in 64 bits)
    if (big >= 256 || big * m >= 1024 * 256) side = 256;
    else if (mid >= 512 || mid * m >= 192 * 256) side = 128;
    const int64_t tiles = tiles_of(N, K, side);
    int64_t s = tiles >= 256 ? 1 : (side == 256 ? 256 : 512) / tiles;
    if (s > M / 256) s = M / 256;
    if (s < 1) s = 1;
    const int64_t chunk = ceil_div(ceil_div(M, s), (int64_t)kMost) * kMost;
    return {side, tiles, (int)ceil_div(M, chunk), chunk};
}

template <class T>
int run(const Params& p, const Plan& pl, hipStream_t stream) {
    constexpr int MS = kParts<T> == 1 ? 64 : 32;   // (two steps of three parts fill LDS)
    const dim3 grid((unsigned)pl.tiles, (unsigned)pl.slices);
    if (pl.side == 256)
        hipLaunchKernelGGL((wgrad8_kernel<T, 256, 256, 2, 4, MS>), grid, dim3(512), 0, stream, p);
    else if (pl.side == 128)
        hipLaunchKernelGGL((wgrad8_kernel<T, 128, 128, 2, 4, MS>), grid, dim3(512), 0, stream, p);
    else
        hipLaunchKernelGGL((wgrad8_kernel<T, 64, 64, 2, 2, MS>), grid, dim3(256), 0, stream, p);
    return hip_error(hipGetLastError(), "wgrad8_kernel launch");
}

}  // namespace

size_t wgrad8_workspace(int64_t M, int64_t N, int64_t K, int dtype, bool bias) {
    (void)dtype;
    if (M == 0 || N == 0) return 0;
    const Plan pl = plan_of(M, N, K);
    return pl.slices > 1 ? (size_t)pl.slices * ((size_t)N * (size_t)K + (bias ? (size_t)N : 0)) * 4 : 0;
}

void wgrad8_plan(int64_t M, int64_t N, int64_t K, int* side, int* slices) {
    const Plan pl = plan_of(M, N, K);
    *side = pl.side;
    *slices = pl.slices;
}

int launch_wgrad8(const void* dz, int64_t lddz, int dtype, const Mat8& x, float* dw, float* db,
                  int64_t M, int64_t N, int64_t K, void* ws, hipStream_t stream) {
    const Plan pl = plan_of(M, N, K);
    if (!grid_fits(pl.tiles, 512)) return set_error(CDX_ERR_UNSUPPORTED, "wgrad8: too many output tiles");
    float* part = static_cast<float*>(ws);
    Params p{dz, lddz, x.q, x.ldq, static_cast<const uint8_t*>(x.s), x.lds, M, N, K, pl.chunk, dw, db};
    if (pl.slices > 1) {
        p.dw = part;
        p.db = db ? part + (int64_t)pl.slices * N * K : nullptr;
    }
    const int st = with_dtype(dtype, [&](auto t) { return run<decltype(t)>(p, pl, stream); });
    if (st || pl.slices == 1) return st;
    const int64_t grid = ceil_div(N * K + (db ? N : 0), (int64_t)256);
    hipLaunchKernelGGL(wgrad8_sum_kernel, dim3((unsigned)(grid < 65536 ? grid : 65536)), dim3(256), 0,
                       stream, part, pl.slices, N * K, db ? N : (int64_t)0, dw, db);
    return hip_error(hipGetLastError(), "wgrad8_sum_kernel launch");
}

}  // namespace cdx
