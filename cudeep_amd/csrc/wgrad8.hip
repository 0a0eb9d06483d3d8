// The weight gradient of a Linear layer whose input was kept in 8 bits:
//   dw[n,k] = sum over m of dz[m,n] xh[m,k],   db[n] = sum over m of dz[m,n],
// xh = code * scale with a scale byte for each 128 columns of a row.
//
// xh is exact in bf16 (three fraction bits times a power of two), so it is one
// bf16 operand; dz is split into bf16 parts that hold it exactly: one part for
// bf16, two for f16 (11 bits), three for f32 (24 bits; below 2^-110 the last part
// may lose bits).  Every product is then exact in fp32 and the sums are fp32, so
// the gradient is that of the restored input with no rounding but the sums'.
//
// Both operands have the sum's index m as their slow one.  Tiles are staged in
// LDS as they lie, [m][n] and [m][k], and ds_read_b64_tr_b16 gives each lane the
// four m of its column.  Few output tiles: m is split over workgroups, whose
// partials a second kernel adds in a fixed order.
#include "block8.hpp"

namespace cdx {
namespace {

using namespace b8;

typedef short shortx4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32;   // m per step: one v_mfma_f32_16x16x32_bf16

template <class T> constexpr int kParts = std::is_same_v<T, float> ? 3 : std::is_same_v<T, f16> ? 2 : 1;

struct Params {
    const void* dz; int64_t lddz;
    const uint8_t* q; int64_t ldq;
    const uint8_t* s; int64_t lds;
    int64_t M, N, K;
    int64_t chunk;             // m per slice, a multiple of kStep
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

// BN x BK output tiles, WN x WK waves.  LDS rows are padded by 32 bytes: the
// four rows that 16 lanes read together then fill all banks.
template <class T, int BN, int BK, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK)
void wgrad8_kernel(Params p) {
    constexpr int PARTS = kParts<T>, NT = 64 * WN * WK;
    constexpr int FN = BN / WN / 16, FK = BK / WK / 16;
    constexpr int PN = BN + 16, PK = BK + 16;   // LDS row lengths
    __shared__ __attribute__((aligned(16))) uint16_t zs[PARTS][kStep][PN];
    __shared__ __attribute__((aligned(16))) uint16_t xs[kStep][PK];
    const int tid = threadIdx.x, wave = tid >> 6, l16 = tid & 15, g = (tid >> 4) & 3;
    const int wn = wave % WN, wk = wave / WN;
    const int64_t tiles_n = ceil_div(p.N, (int64_t)BN);
    const int64_t n0 = (blockIdx.x % tiles_n) * BN, k0 = (blockIdx.x / tiles_n) * BK;
    const int64_t m_begin = (int64_t)blockIdx.y * p.chunk;
    const int64_t m_end = m_begin + p.chunk < p.M ? m_begin + p.chunk : p.M;
    // pieces of eight columns: a thread stages piece column zc (xc) of rows zr, zr + ZR, ...
    constexpr int ZR = NT / (BN / 8), XR = NT / (BK / 8);
    static_assert(kStep % ZR == 0 && kStep % XR == 0, "whole rows of pieces");
    const int zc = 8 * (tid % (BN / 8)), zr = tid / (BN / 8);
    const int xc = 8 * (tid % (BK / 8)), xr = tid / (BK / 8);
    const int64_t z_left = p.N - n0 - zc, x_left = p.K - k0 - xc;
    const int zn = z_left < 0 ? 0 : z_left > 8 ? 8 : (int)z_left;
    const int xn = x_left < 0 ? 0 : x_left > 8 ? 8 : (int)x_left;
    const bool sums = p.db && k0 == 0;
    float zv[kStep / ZR][8], bsum[8] = {};
    u32x2 xv[kStep / XR];
    float xscale[kStep / XR];
    auto load = [&](int64_t m) {
#pragma unroll
        for (int i = 0; i < kStep / ZR; ++i) {
            const int64_t r = m + zr + i * ZR;
            load_n<8>(static_cast<const T*>(p.dz) + r * p.lddz + n0 + zc, r < m_end ? zn : 0, zv[i]);
        }
#pragma unroll
        for (int i = 0; i < kStep / XR; ++i) {
            const int64_t r = m + xr + i * XR;
            const uint8_t* q = p.q + r * p.ldq + k0 + xc;
            u32x2 w = {0u, 0u};
            float sc = 1.0f;
            if (r < m_end && xn > 0) {
                uint32_t b = p.s[r * p.lds + (k0 + xc) / kBlock];
                sc = e8m0_value(b);
                if (xn == 8) {
                    w = load8b(q);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < xn) w[j >> 2] |= (uint32_t)q[j] << (8 * (j & 3));
                }
                if (b == 255) w = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};   // a NaN scale: NaN codes
            }
            xv[i] = w;
            xscale[i] = sc;
        }
    };
    floatx4 acc[FN][FK] = {};
    if (m_begin < m_end) load(m_begin);
    for (int64_t m = m_begin; m < m_end; m += kStep) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kStep / ZR; ++i) {
            u32x4 parts[PARTS];
            split_parts<PARTS>(zv[i], parts);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
                *reinterpret_cast<u32x4*>(&zs[q][zr + i * ZR][zc]) = parts[q];
            if (sums) {
#pragma unroll
                for (int j = 0; j < 8; ++j) bsum[j] += zv[i][j];
            }
        }
#pragma unroll
        for (int i = 0; i < kStep / XR; ++i)
            *reinterpret_cast<u32x4*>(&xs[xr + i * XR][xc]) = restore_bf16(xv[i], xscale[i]);
        __syncthreads();
        if (m + kStep < m_end) load(m + kStep);
        // operand of lane (l16, g): column l16, m = 8 g + 0..7, as two transposed
        // reads of four rows; lane i of 16 points at row i / 4, columns 4 (i % 4)
        const int row = 8 * g + (l16 >> 2), col = 4 * (l16 & 3);
        auto operand = [&](const uint16_t* base, int pitch) {
            typedef __attribute__((address_space(3))) shortx4* P3;
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)(base + row * pitch + col));
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P3)(base + (row + 4) * pitch + col));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        bf16x8 xo[FK];
#pragma unroll
        for (int j = 0; j < FK; ++j) xo[j] = operand(&xs[0][16 * (wk * FK + j)], PK);
        // smallest parts first, as the larger ones then round their sum once
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q)
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const bf16x8 zo = operand(&zs[q][0][16 * (wn * FN + i)], PN);
#pragma unroll
                for (int j = 0; j < FK; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(zo, xo[j], acc[i][j], 0, 0, 0);
            }
    }
    float* dw = p.dw + (int64_t)blockIdx.y * p.N * p.K;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t n = n0 + 16 * (wn * FN + i) + 4 * g + r;
#pragma unroll
            for (int j = 0; j < FK; ++j) {
                const int64_t k = k0 + 16 * (wk * FK + j) + l16;
                if (n < p.N && k < p.K) dw[n * p.K + k] = acc[i][j][r];
            }
        }
    if (sums) {
        // the staging threads' sums of a column, added in the order of their rows
        __shared__ float red[ZR][BN];
#pragma unroll
        for (int j = 0; j < 8; ++j) red[zr][zc + j] = bsum[j];
        __syncthreads();
        for (int c = tid; c < BN; c += NT) {
            if (n0 + c >= p.N) break;
            float a = red[0][c];
            for (int i = 1; i < ZR; ++i) a += red[i][c];
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

struct Plan { int64_t tiles; int slices; int64_t chunk; };

// Slices of m: enough workgroups for the 256 CUs, at least 256 m each.
Plan plan_of(int64_t M, int64_t N, int64_t K) {
    // (a layer without inputs still has its bias's column of tiles)
    const int64_t tiles = ceil_div(N, (int64_t)64) * (K > 0 ? ceil_div(K, (int64_t)64) : 1);
    int64_t s = tiles < 512 ? 512 / tiles : 1;
    if (s > M / 256) s = M / 256;
    if (s < 1) s = 1;
    const int64_t chunk = ceil_div(ceil_div(M, s), (int64_t)kStep) * kStep;
    return {tiles, (int)ceil_div(M, chunk), chunk};
}

}  // namespace

size_t wgrad8_workspace(int64_t M, int64_t N, int64_t K, int dtype, bool bias) {
    (void)dtype;
    if (M == 0 || N == 0) return 0;
    const Plan pl = plan_of(M, N, K);
    return pl.slices > 1 ? (size_t)pl.slices * ((size_t)N * (size_t)K + (bias ? (size_t)N : 0)) * 4 : 0;
}

int launch_wgrad8(const void* dz, int64_t lddz, int dtype, const Mat8& x, float* dw, float* db,
                  int64_t M, int64_t N, int64_t K, void* ws, hipStream_t stream) {
    const Plan pl = plan_of(M, N, K);
    if (pl.tiles >= (int64_t)1 << 31) return set_error(CDX_ERR_UNSUPPORTED, "wgrad8: too many output tiles");
    float* part = static_cast<float*>(ws);
    Params p{dz, lddz, x.q, x.ldq, static_cast<const uint8_t*>(x.s), x.lds, M, N, K, pl.chunk, dw, db};
    if (pl.slices > 1) {
        p.dw = part;
        p.db = db ? part + (int64_t)pl.slices * N * K : nullptr;
    }
    const int st = with_dtype(dtype, [&](auto t) {
        hipLaunchKernelGGL((wgrad8_kernel<decltype(t), 64, 64, 2, 2>),
                           dim3((unsigned)pl.tiles, (unsigned)pl.slices), dim3(256), 0, stream, p);
        return hip_error(hipGetLastError(), "wgrad8_kernel launch");
    });
    if (st || pl.slices == 1) return st;
    const int64_t grid = ceil_div(N * K + (db ? N : 0), (int64_t)256);
    hipLaunchKernelGGL(wgrad8_sum_kernel, dim3((unsigned)(grid < 65536 ? grid : 65536)), dim3(256), 0,
                       stream, part, pl.slices, N * K, db ? N : (int64_t)0, dw, db);
    return hip_error(hipGetLastError(), "wgrad8_sum_kernel launch");
}

}  // namespace cdx
