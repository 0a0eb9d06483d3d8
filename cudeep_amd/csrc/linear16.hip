// A Linear layer in 16 bits: which kernel runs a product, the sums of its slices, and the slope of the
// activation.
#include "linear16_tile.hpp"

namespace cdx {
namespace {

using namespace l16;

// Sums of slices, added in their order, through the epilogue: a thread has eight n of a row.  Behind
// them the column sums.
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

// dz = grad act'(z), eight columns a thread.  PAST: grad and z, which nobody reads again, pass the caches by
// (block8.hpp), so that dz is there for the products: a training step of 8192 x 4096 x 4096 727 us, 741
// without.
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
        for (int j = 0; j < 8; ++j) v[j] = act_slope<T, ACT>(g[j], v[j], 0.0f);
        store_n<8>(dz + r * lddz + c, count, v);
    }
}

// (a layer without inputs still has its bias's column of tiles)
int64_t tiles_of(int64_t M, int64_t N, int side) {
    return ceil_div(M, (int64_t)side) * (N > 0 ? ceil_div(N, (int64_t)side) : 1);
}

Plan make_plan(Kernel kernel, int64_t M, int64_t N, int64_t K, int side, int64_t slices) {
    const int64_t tiles = tiles_of(M, N, side);
    const int64_t chunk = ceil_div(ceil_div(K, slices), (int64_t)kStep) * kStep;
    return {kernel, tiles, K > 0 ? (int)ceil_div(K, chunk) : 1, chunk > 0 ? chunk : kStep};
}

Plan direct_plan(int64_t M, int64_t N, int mt) {
    return {Kernel::Direct, ceil_div(M, (int64_t)(16 * mt)) * ceil_div(N, (int64_t)16), 1, kStep, mt};
}

Plan plan_of(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned) {
    aligned = aligned && K >= kStep && N > 0;
    if (kind == Linear16Kind::Forward && K > 0 && M <= (aligned ? 128 : 64)) {
        const int64_t tiles_m = ceil_div(M, (int64_t)16), tiles_n = ceil_div(N, (int64_t)16);
        int mt = 1;
        while (mt < 4 && ceil_div(tiles_m, (int64_t)mt) * tiles_n > 256 && mt < tiles_m) mt *= 2;
        if (!aligned || (mt <= 2 && K <= 8192 && ceil_div(tiles_m, (int64_t)mt) * tiles_n <= (M <= 16 ? 512 : 256)))
            return direct_plan(M, N, mt);
    }
    // slices for about `groups` workgroups, of `least` k and more
    auto cut = [&](int64_t tiles, int64_t groups, int64_t least) {
        const int64_t s = groups / tiles;
        return s > K / least ? (K / least > 1 ? K / least : 1) : s > 1 ? s : 1;
    };
    // (without columns of B there is nothing to load straight into LDS)
    if (!aligned) {
        if (N == 0) return make_plan(Kernel::Any, M, N, K, 64, 1);
        const int64_t t128 = tiles_of(M, N, 128), t64 = tiles_of(M, N, 64);
        if (t128 >= 80) return make_plan(Kernel::Any128, M, N, K, 128, t128 >= 200 ? 1 : cut(t128, 512, 384));
        return make_plan(Kernel::Any, M, N, K, 64, t64 >= 200 ? 1 : cut(t64, 512, 384));
    }
    const int64_t t256 = tiles_of(M, N, 256), t128 = tiles_of(M, N, 128), t64 = tiles_of(M, N, 64);
    const int64_t long_k = K / 4096 < 256 ? K / 4096 : 256;
    if (t256 >= 200 || t256 * long_k >= 256) return make_plan(Kernel::Turns, M, N, K, 256, cut(t256, 256, 4096));
    if (t128 > 256) return make_plan(Kernel::Tile128, M, N, K, 128, 1);
    if (t128 >= 140 || t128 * long_k >= 256) return make_plan(Kernel::Ring128, M, N, K, 128, cut(t128, 256, 4096));
    return make_plan(Kernel::Ring64, M, N, K, 64, cut(t64, 256, 1024));
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

size_t linear16_workspace(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool col_sums) {
    if (M == 0 || N == 0) return 0;
    // (alignment may choose the kernel: the larger of both)
    size_t most = 0;
    for (int aligned = 0; aligned < 2; ++aligned) {
        const Plan pl = plan_of(kind, M, N, K, aligned);
        const size_t need = pl.slices > 1
            ? (size_t)pl.slices * ((size_t)M * (size_t)N + (col_sums ? (size_t)M : 0)) * 4 : 0;
        most = need > most ? need : most;
    }
    return most;
}

const char* linear16_kernel_name(Linear16Kind kind, int64_t M, int64_t N, int64_t K, bool aligned,
                                 int* slices) {
    static const char* const names[] = {"any", "any 128", "ring 64", "ring 128", "tile 128", "turns", "direct"};
    const Plan pl = plan_of(kind, M, N, K, aligned);
    *slices = pl.slices;
    return names[(int)pl.kernel];
}

int launch_linear16(Linear16Kind kind, const Linear16Product& g, bool out_f32, void* col_y, void* ws,
                    hipStream_t stream) {
    const bool ca = kind == Linear16Kind::Weight, cb = kind != Linear16Kind::Forward;
    const bool aligned = g.lda % 8 == 0 && g.ldb % 8 == 0 && ((uintptr_t)g.a | (uintptr_t)g.b) % 16 == 0 &&
                         g.lda <= kMaxLd && g.ldb <= kMaxLd && (!ca || g.M % 8 == 0) && (!cb || g.N % 8 == 0);
    return launch_plan(kind, g, plan_of(kind, g.M, g.N, g.K, aligned), out_f32, col_y, ws, stream);
}

int launch_linear16_slope(const void* grad, int64_t ldg, const void* z, int64_t ldz, void* dz,
                          int64_t lddz, int64_t rows, int64_t cols, int dtype, int act,
                          hipStream_t stream) {
    return with_16(dtype, [&](auto t) {
        using T = decltype(t);
        return with_act(act, [&](auto a) {
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

}  // namespace cdx
