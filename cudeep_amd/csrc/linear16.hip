// A Linear layer in 16 bits: which kernel runs a product, the sums of its slices, and the slope of the
// activation.
#include "linear16_tile.hpp"

namespace cdx {
namespace {

using namespace l16;

// Sums of slices, added in their order, through the epilogue: a thread has eight n of a row.  Behind
// them the column sums.  Short and bound by its launch (256 x 784 in 4 slices 3.9 us).
template <class T, bool EPI>
__global__ __launch_bounds__(256)
void linear16_sum_kernel(Params p, const float* __restrict__ part, const float* __restrict__ col_part,
                         int slices) {
    const int64_t per_row = ceil_div(p.N, (int64_t)8), body = p.M * per_row;
    const int64_t total = body + (col_part ? p.M : 0);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        if (i >= body) {
            const int64_t m = i - body;
            float v = 0.0f;
            for (int s = 0; s < slices; ++s) v += col_part[s * p.M + m];
            if (p.col_sums) p.col_sums[m] = v;
            else static_cast<T*>(p.col_y)[m] = (T)v;
            continue;
        }
        const int64_t m = i / per_row, n = i % per_row * 8, left = p.N - n;
        const int count = left > 8 ? 8 : (int)left;
        float v[8];
        load_n<8>(part + m * p.N + n, count, v);
        for (int s = 1; s < slices; ++s) {
            float t[8];
            load_n<8>(part + (s * p.M + m) * p.N + n, count, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += t[j];
        }
        if (p.out.sums) {
            store_n<8>(p.out.sums + m * p.N + n, count, v);
        } else if constexpr (EPI) {
            float bias[8];
            load_bias<T>(p.out, n, count, bias);
            with_epilogue(p.out.act, [&](auto act) { finish<T, decltype(act)::value>(p.out, m, n, count, v, bias); });
        } else {
            store_n<8>(static_cast<T*>(p.out.y) + m * p.out.ldy + n, count, v);
        }
    }
}

// dz = grad act'(z), eight columns a thread, one pass that memory bounds (8192 x 4096 in bf16 36 us, 5.6 TB/s:
// some of z is in the caches).  PAST: grad and z pass the caches by
// (block8.hpp), so that dz is there for the products: a training step of 8192 x 4096 x 4096 727 us, 741
// without.  (grad, as the residual's gradient, may be read once more behind them: no slower for it.)
template <class T, int ACT, bool PAST>
__global__ __launch_bounds__(256)
void linear16_slope_kernel(const T* __restrict__ grad, int64_t ldg, const T* __restrict__ z, int64_t ldz,
                           T* __restrict__ dz, int64_t lddz, int64_t rows, int64_t cols) {
    const int64_t per_row = ceil_div(cols, (int64_t)8), total = rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row, c = i % per_row * 8, left = cols - c;
        const int count = left > 8 ? 8 : (int)left;
        float g[8], v[8];
        if (count == 8) {
            const u32x4 gu = load16_as<PAST>(grad + r * ldg + c), zu = load16_as<PAST>(z + r * ldz + c);
            T ge[8], ze[8];
            __builtin_memcpy(ge, &gu, 16);
            __builtin_memcpy(ze, &zu, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g[j] = (float)ge[j];
                v[j] = (float)ze[j];
            }
        } else {
            load_n<8>(grad + r * ldg + c, count, g);
            load_n<8>(z + r * ldz + c, count, v);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = layer_slope<T, ACT>(g[j], v[j]);
        store_n<8>(dz + r * lddz + c, count, v);
    }
}

// The same with the column sums of dz, which no matrix instruction needs in 16 bits: they are of the slopes'
// fp32 values, before dz is rounded.  A workgroup has 256 columns of `chunk` rows, a thread eight columns of every
// eighth row; its sums go to part[chunk's number], which the next kernel adds in their order.  Up to 32 rows are one part,
// the result itself (`whole`, or part in fp32; a backward pass of 16 x 4096 x 4096 31.2 us, with a second launch 32.9; but
// of 64 x 4096 x 1024 24.4 in one part, 23.3 in two).  8192 x 4096 with GELU
// in bf16 38.9 us and 1.4 for the parts (34.3 without sums), 8192 x 256 6.1 and 2.4 (5.5), 32768 x 512 19.6 and 4.6
// (19.3); a float32 bias gradient of 8192 rows is off by 1.5e-7 of its norm, by 1.7e-3 from the rounded dz.
constexpr int kSlopeCols = 256;

template <class T, int ACT, bool PAST>
__global__ __launch_bounds__(256)
void linear16_slope_sums_kernel(const T* __restrict__ grad, int64_t ldg, const T* __restrict__ z, int64_t ldz,
                                T* __restrict__ dz, int64_t lddz, int64_t rows, int64_t cols, int64_t chunk,
                                float* __restrict__ part, T* __restrict__ whole) {
    constexpr int U = 4, LANES = kSlopeCols / 8, STEP = 256 / LANES;
    __shared__ float red[STEP][kSlopeCols];
    const int lane = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
    const int64_t c = (int64_t)blockIdx.x * kSlopeCols + lane * 8, left = cols - c;
    const int count = left < 0 ? 0 : left > 8 ? 8 : (int)left;
    const int64_t first = (int64_t)blockIdx.y * chunk, last = first + chunk < rows ? first + chunk : rows;
    float sum[8] = {};
    auto use = [&](int64_t r, float (&g)[8], float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = layer_slope<T, ACT>(g[j], v[j]);
            // (an fp32 value of its own, as in the kernel above: multiplied and rounded to float16 in one instruction it
            // could end in another bit)
            asm("" : "+v"(v[j]));
            sum[j] += v[j];
        }
        store_n<8>(dz + r * lddz + c, count, v);
    };
    int64_t r = first + r0;
    if (count == 8) {
        for (; r + (U - 1) * STEP < last; r += U * STEP) {
            u32x4 gu[U], zu[U];   // (all of them on their way before the first is used)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                gu[u] = load16_as<PAST>(grad + (r + u * STEP) * ldg + c);
                zu[u] = load16_as<PAST>(z + (r + u * STEP) * ldz + c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                T ge[8], ze[8];
                __builtin_memcpy(ge, &gu[u], 16);
                __builtin_memcpy(ze, &zu[u], 16);
                float g[8], v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    g[j] = (float)ge[j];
                    v[j] = (float)ze[j];
                }
                use(r + u * STEP, g, v);
            }
        }
    }
    if (count > 0) {
        for (; r < last; r += STEP) {
            float g[8], v[8];
            load_n<8>(grad + r * ldg + c, count, g);
            load_n<8>(z + r * ldz + c, count, v);
            use(r, g, v);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) red[r0][lane * 8 + j] = sum[j];   // (columns past the last hold zeros)
    __syncthreads();
    const int64_t n = (int64_t)blockIdx.x * kSlopeCols + threadIdx.x;
    if (n >= cols) return;
    float v = red[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < STEP; ++i) v += red[i][threadIdx.x];
    if (whole) whole[n] = (T)v;
    else part[(int64_t)blockIdx.y * cols + n] = v;
}

// The parts' sums, in their order: 16 columns a workgroup, 16 threads a column.
template <class O>
__global__ __launch_bounds__(256)
void linear16_slope_join_kernel(const float* __restrict__ part, int parts, int64_t cols, O* __restrict__ out) {
    __shared__ float red[16][16];
    const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + lane;
    float v = 0.0f;
    if (n < cols) {
#pragma unroll 4
        for (int i = r0; i < parts; i += 16) v += part[i * cols + n];
    }
    red[r0][lane] = v;
    __syncthreads();
    if (r0 || n >= cols) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += red[i][lane];
    out[n] = (O)v;
}

// The rows of a part, and how many parts there are: enough workgroups for the chip, and few parts to add (backward
// pass of 32768 x 512 x 512 94.2 us; 1024 workgroups and 256 parts at most 96.2).
struct SlopeParts { int64_t chunk; int parts; };
SlopeParts slope_parts(int64_t rows, int64_t cols) {
    int64_t parts = 2048 / ceil_div(cols, (int64_t)kSlopeCols);
    if (parts > 512) parts = 512;
    if (parts < 1) parts = 1;
    const int64_t chunk = ceil_div(ceil_div(rows, parts), (int64_t)32) * 32;
    return {chunk, (int)ceil_div(rows, chunk)};
}

// (a layer without inputs still has its bias's column of tiles)
int64_t tiles_of(int64_t M, int64_t N, int rows, int cols) {
    return ceil_div(M, (int64_t)rows) * (N > 0 ? ceil_div(N, (int64_t)cols) : 1);
}
int64_t tiles_of(int64_t M, int64_t N, int side) { return tiles_of(M, N, side, side); }

Plan make_plan(Kernel kernel, int64_t M, int64_t N, int64_t K, int side, int64_t slices) {
    const int64_t tiles = kernel == Kernel::Tall ? tiles_of(M, N, 128, 64) : tiles_of(M, N, side);
    const int64_t chunk = ceil_div(ceil_div(K, slices), (int64_t)kStep) * kStep;
    return {kernel, tiles, K > 0 ? (int)ceil_div(K, chunk) : 1, chunk > 0 ? chunk : kStep};
}

Plan direct_plan(int64_t M, int64_t N, int mt) {
    return {Kernel::Direct, ceil_div(M, (int64_t)(16 * mt)) * ceil_div(N, (int64_t)16), 1, kStep, mt};
}

// Which kernel, and how many slices of k (all figures us, bf16, M x N x K; "input", "weight": of those
// products, else forward).  Slices are added by a launch of their own, so that they have to save more than
// that and their sums' traffic: 8 of ring 64 at most (256 x 256 x 16384 14.9, 16 of them 16.9), 16 of
// the others (weight 256 x 512 x 65536 on ring 128 48, 32 of them 56; unaligned 4 x 640 x 6575 15.1, 8 17.8).
Plan plan_of(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned) {
    aligned = aligned && K >= kStep && N > 0;   // (a whole step, and columns of B, to load straight into LDS)
    // Few rows, whose weights are read once: one launch with k split inside the workgroups, while these are no
    // more than the CUs (1 x 4096 x 4096 6.6, ring 64 in 4 slices 8.6; 128 x 1024 x 1024 5.0, ring 64 5.8; but
    // 16 x 8192 x 4096 18.9, ring 64 13.9) and k is short (1 x 2048 x 8192 12.0, ring 64 in 8 slices 9.9).
    // Operands of any alignment, which ring 64 does not take, up to 64 rows and, but for a single row, half that k
    // (1 x 4096 x 2049 9.7, any in 5 slices 12.0; 33 x 4096 x 1001 9.6, any in 2 11.7; 16 x 4096 x 2049 15.3, any in
    // 5 12.7; 64 x 4096 x 4001 50, any in 8 15.6; 65 x 4096 x 1001 15.9, any 13.0).
    if (kind == Linear16Kind::Forward && K > 0 && M <= (aligned ? 128 : 64) && K <= (aligned || M == 1 ? 4096 : 2048)) {
        const int64_t tiles_m = ceil_div(M, (int64_t)16), tiles_n = ceil_div(N, (int64_t)16);
        for (int mt = 1; mt <= (aligned ? 2 : 4); mt *= 2)
            if (ceil_div(tiles_m, (int64_t)mt) * tiles_n <= 256) return direct_plan(M, N, mt);
    }
    // slices for about `groups` workgroups, of `least` k and more, `most` of them
    auto cut = [&](int64_t tiles, int64_t groups, int64_t least, int64_t most) {
        int64_t s = groups / tiles;
        if (s > K / least) s = K / least;
        if (s > most) s = most;
        return s > 1 ? s : 1;
    };
    const int64_t t256 = tiles_of(M, N, 256), t128 = tiles_of(M, N, 128), t64 = tiles_of(M, N, 64);
    const int64_t long_k = K / 2048 < 256 ? K / 2048 : 256;
    const int64_t narrow = M < N ? M : N;       // the smaller side
    if (!aligned) {
        if (N == 0) return make_plan(Kernel::Any, M, N, K, 64, 1);
        // 128 x 128 tiles, where they fill more than half of the CUs or k is long enough for slices (4096 x 4096 x
        // 4001 183, 64 x 64 318; 2048 x 1280 x 1001 17.2, 64 x 64 19.7; 1336 x 1440 x 8001 in 3 slices 78, 64 x
        // 64 96; but 640 x 2048 x 1001 16.5, 64 x 64 13.5), and half of a tile does not lie outside (400000 x 64 x
        // 1024 199, 64 x 64 176)
        if (narrow > 64 && (t128 >= 140 || t128 * long_k >= 256))
            return make_plan(Kernel::Any128, M, N, K, 128, t128 >= 200 ? 1 : cut(t128, 512, 1024, 16));
        return make_plan(Kernel::Any, M, N, K, 64, t64 >= 200 ? 1 : cut(t64, 512, 384, 16));
    }
    // 256 x 256, for most of the CUs (2560 x 5120 x 1024 35.6, tile 128 38.8; 2560 x 4608 x 1024 37.5, tile 128
    // 34.0), by slices too (weight 1024 x 1024 x 65536 in 16 155, ring 128 in 4 177), where half of a tile does not
    // lie outside (128 x 128256 x 4096 255, tile 128 206; 192 x 65536 x 2048 74, tile 128 85)
    if (narrow > 128 && (t256 >= 200 || t256 * (long_k / 2) >= 256))
        return make_plan(Kernel::Turns, M, N, K, 256, cut(t256, 256, 4096, 256));
    // 128 x 128 tiles: two workgroups a CU share it where there is more than one (2048 x 2176 x 2048 32.3, ring 128
    // 36.7; 1 x 128256 x 4096 172, turns 246), else one has four buffers (2048 x 2048 x 2048 21.2, tile 128 26.4)
    if (t128 > 256) return make_plan(Kernel::Tile128, M, N, K, 128, 1);
    // fewer of them, with a long k, in three slices and more (1152 x 1152 x 8192 36, ring 64 46; weight 256 x 512 x
    // 65536 in 16 48, ring 64 55; but 2048 x 1024 x 4096 in 2 30.1, tall 24.2)
    if (t128 <= 85 && t128 * long_k >= 256)
        return make_plan(Kernel::Ring128, M, N, K, 128, cut(t128, 256, 2048, 16));
    // 128 x 64 where a CU would have more than one of 64 x 64 and has one of these (8192 x 256 x 784 10.4, ring 64
    // 12.1; 2048 x 1024 x 4096 24.2, ring 64 26.1; 1280 x 1280 x 1280 10.3, ring 64 10.6; but 1024 x 1024 x 1024
    // 8.3, ring 64 6.3, and 1408 x 1536 x 2048 24.5, ring 128 19.0)
    if (t64 > 256 && tiles_of(M, N, 128, 64) <= 256) return make_plan(Kernel::Tall, M, N, K, 64, 1);
    if (t64 > 256) return make_plan(Kernel::Ring128, M, N, K, 128, 1);
    return make_plan(Kernel::Ring64, M, N, K, 64, cut(t64, 256, 1024, 8));
}

// Calls f with an activation's code as a constant: those whose dz is rounded, and ReLU with them.
template <class F> int with_smooth_act(int act, F f) {
    using std::integral_constant;
    if (act == CDX_EPI_GELU) return f(integral_constant<int, CDX_EPI_GELU>{});
    if (act == CDX_EPI_SILU) return f(integral_constant<int, CDX_EPI_SILU>{});
    return f(integral_constant<int, CDX_EPI_SIGMOID>{});
}
template <class F> int with_layer_act(int act, F f) {
    return act == CDX_EPI_RELU ? f(std::integral_constant<int, CDX_EPI_RELU>{}) : with_smooth_act(act, f);
}

unsigned wide_grid(int64_t threads) {
    const int64_t g = ceil_div(threads, (int64_t)256);
    return (unsigned)(g < 65536 ? g : 65536);
}

int launch_plan(Linear16Kind kind, const Linear16Product& g, const Plan& pl, bool out_f32, void* col_y, void* ws,
                hipStream_t stream) {
    if (!grid_fits(pl.tiles, 512)) return set_error(CDX_ERR_UNSUPPORTED, "linear16: too many output tiles");
    Params p{static_cast<const uint16_t*>(g.a), static_cast<const uint16_t*>(g.b), g.M, g.N, g.K, g.lda,
             g.ldb, pl.chunk, g.out, nullptr, nullptr};
    if (out_f32) {
        p.out.sums = static_cast<float*>(g.out.y);
        p.col_sums = static_cast<float*>(col_y);
    } else {
        p.col_y = col_y;
    }
    Params part = p;
    float* sums = static_cast<float*>(ws);
    float* col_part = nullptr;
    if (pl.slices > 1) {
        part.out.sums = sums;
        if (col_y) col_part = part.col_sums = sums + (int64_t)pl.slices * g.M * g.N;
    }
    const int st = kind == Linear16Kind::Forward ? run_forward(g.dtype, part, pl, stream)
                   : kind == Linear16Kind::Input ? run_input(g.dtype, part, pl, stream)
                                                 : run_weight(g.dtype, part, pl, stream);
    if (st || pl.slices == 1) return st;
    return with_16(g.dtype, [&](auto t) {
        using T = decltype(t);
        const dim3 grid(wide_grid(g.M * ceil_div(g.N, (int64_t)8) + (col_y ? g.M : 0)));
        if (kind == Linear16Kind::Forward)
            hipLaunchKernelGGL((linear16_sum_kernel<T, true>), grid, dim3(256), 0, stream, p, sums, col_part, pl.slices);
        else
            hipLaunchKernelGGL((linear16_sum_kernel<T, false>), grid, dim3(256), 0, stream, p, sums, col_part, pl.slices);
        return hip_error(hipGetLastError(), "linear16_sum_kernel launch");
    });
}

}  // namespace

size_t linear16_workspace(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned, bool col_sums) {
    if (M == 0 || N == 0) return 0;
    const Plan pl = plan_of(kind, M, N, K, aligned);
    if (pl.slices == 1) return 0;
    return (size_t)pl.slices * ((size_t)M * (size_t)N + (col_sums ? (size_t)M : 0)) * 4;
}

size_t linear16_workspace(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool col_sums) {
    const size_t a = linear16_workspace(kind, M, N, K, false, col_sums);
    const size_t b = linear16_workspace(kind, M, N, K, true, col_sums);
    return a > b ? a : b;
}

bool linear16_aligned(Linear16Kind kind, int64_t M, int64_t N, const void* a, int64_t lda, const void* b, int64_t ldb) {
    const bool ca = kind == Linear16Kind::Weight, cb = kind != Linear16Kind::Forward;
    return lda % 8 == 0 && ldb % 8 == 0 && ((uintptr_t)a | (uintptr_t)b) % 16 == 0 && lda <= kMaxLd && ldb <= kMaxLd &&
           (!ca || M % 8 == 0) && (!cb || N % 8 == 0);
}

const char* linear16_kernel_name(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned,
                                 int* slices) {
    static const char* const names[] = {"any", "any 128", "ring 64", "ring 128", "tile 128", "turns", "direct", "tall"};
    const Plan pl = plan_of(kind, M, N, K, aligned);
    *slices = pl.slices;
    return names[(int)pl.kernel];
}

int launch_linear16(Linear16Kind kind, const Linear16Product& g, bool out_f32, void* col_y, void* ws,
                    hipStream_t stream) {
    const bool aligned = linear16_aligned(kind, g.M, g.N, g.a, g.lda, g.b, g.ldb);
    return launch_plan(kind, g, plan_of(kind, g.M, g.N, g.K, aligned), out_f32, col_y, ws, stream);
}

int launch_linear16_slope(const void* grad, int64_t ldg, const void* z, int64_t ldz, void* dz,
                          int64_t lddz, int64_t rows, int64_t cols, int dtype, int act,
                          hipStream_t stream) {
    return with_16(dtype, [&](auto t) {
        using T = decltype(t);
        return with_layer_act(act, [&](auto a) {
            const dim3 grid(wide_grid(rows * ceil_div(cols, (int64_t)8)));
            auto go = [&](auto past) {
                hipLaunchKernelGGL((linear16_slope_kernel<T, decltype(a)::value, decltype(past)::value>), grid,
                                   dim3(256), 0, stream, static_cast<const T*>(grad), ldg,
                                   static_cast<const T*>(z), ldz, static_cast<T*>(dz), lddz, rows, cols);
            };
            if (past_caches(rows, cols, dtype)) go(std::true_type{});
            else go(std::false_type{});
            return hip_error(hipGetLastError(), "linear16_slope_kernel launch");
        });
    });
}

size_t linear16_slope_sums_workspace(int64_t rows, int64_t cols) {
    if (rows == 0 || cols == 0) return 0;
    const int parts = slope_parts(rows, cols).parts;
    return parts > 1 ? (size_t)parts * (size_t)cols * sizeof(float) : 0;
}

int launch_linear16_slope_sums(const void* grad, int64_t ldg, const void* z, int64_t ldz, void* dz,
                               int64_t lddz, int64_t rows, int64_t cols, int dtype, int act, void* sums,
                               bool sums_f32, float* part, hipStream_t stream) {
    const SlopeParts sp = slope_parts(rows, cols);
    const int64_t strips = ceil_div(cols, (int64_t)kSlopeCols), joins = ceil_div(cols, (int64_t)16);
    if (!grid_fits(strips * sp.parts, 256) || !grid_fits(joins, 256))
        return set_error(CDX_ERR_UNSUPPORTED, "linear16: too many columns");
    if (sp.parts == 1 && sums_f32) part = static_cast<float*>(sums);
    return with_16(dtype, [&](auto t) {
        using T = decltype(t);
        T* whole = sp.parts == 1 && !sums_f32 ? static_cast<T*>(sums) : nullptr;
        const dim3 grid((unsigned)strips, (unsigned)sp.parts);
        auto run = [&](auto a, auto past) {
            hipLaunchKernelGGL((linear16_slope_sums_kernel<T, decltype(a)::value, decltype(past)::value>), grid,
                               dim3(256), 0, stream, static_cast<const T*>(grad), ldg, static_cast<const T*>(z),
                               ldz, static_cast<T*>(dz), lddz, rows, cols, sp.chunk, part, whole);
        };
        const bool past = past_caches(rows, cols, dtype);
        with_smooth_act(act, [&](auto a) {
            past ? run(a, std::true_type{}) : run(a, std::false_type{});
            return 0;
        });
        const int st = hip_error(hipGetLastError(), "linear16_slope_sums_kernel launch");
        if (st || sp.parts == 1) return st;
        if (sums_f32)
            hipLaunchKernelGGL(linear16_slope_join_kernel<float>, dim3((unsigned)joins), dim3(256), 0, stream, part,
                               sp.parts, cols, static_cast<float*>(sums));
        else
            hipLaunchKernelGGL(linear16_slope_join_kernel<T>, dim3((unsigned)joins), dim3(256), 0, stream, part,
                               sp.parts, cols, static_cast<T*>(sums));
        return hip_error(hipGetLastError(), "linear16_slope_join_kernel launch");
    });
}

}  // namespace cdx
