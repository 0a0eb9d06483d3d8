// Layer norm over the last dimension, forward and backward:
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r,
//   y = xh w + b;
//   g = dy w, dx = r (g - mean(g) - xh mean(g xh)),
//   dw = sum over rows of dy xh, db = sum over rows of dy.
//
// A row stays in the registers of its threads (16 of a wave, a wave, 256 or
// 1024 threads, by its width), so x is read once and the variance is the mean
// of squared differences from the mean, not a difference of two large sums.
// All sums are fp32.  Rows beyond the registers (more than 32768 elements,
// backward 16384) are read again for each sum.
//
// A result may take the place of a row operand (y of x; dx of x or dy): a row is written by the
// threads that have read it, after the last sum that needs it, and the column sums of rows that are
// read twice come before dx.  These operands carry no __restrict__.
//
// Backward: workgroups walk the rows with a stride of the grid, the next row's
// loads in flight while this row's two sums are formed, and keep the columns'
// sums for dw and db in registers over all their rows; one row of partials per
// workgroup, added in a fixed order by a second kernel: no atomics, the same
// bits every time.
//
// Bound by memory where rows are many: 8192 x 4096 in bf16 forward 23.6 us, 5.7 TB/s (33 with
// operands that no cache holds), backward 46, 4.4 TB/s with the parameters' 4 us.  One row: 3.1
// us, a load, two barriers and a store.
#include <algorithm>

#include "block8.hpp"

namespace cdx {
namespace {

using namespace b8;

// A row's threads and 16-byte pieces per thread.
template <class T> constexpr int kVec = 16 / (int)sizeof(T);

// Sum over the TPR threads of a row, in all of them.  TPR > 64: through LDS,
// one barrier; `red` must not be written again before every thread has read it
// (callers alternate buffers).
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float (*red)[NV], int t) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = TPR == 16 ? sum16(v[i]) : sum64(v[i]);
    if constexpr (TPR > 64) {
        if ((t & 63) == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) red[t >> 6][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float s = red[0][i];
#pragma unroll
            for (int k = 1; k < TPR / 64; ++k) s += red[k][i];
            v[i] = s;
        }
    }
}

__device__ __forceinline__ int clip(int64_t n, int most) {
    return n < 0 ? 0 : n > most ? most : (int)n;
}

template <class T, class W, int TPR, int E>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256)
void layer_norm_kernel(const T* x, int64_t ldx, const W* __restrict__ w,
                       const W* __restrict__ b, T* y, int64_t ldy,
                       float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                       int64_t dim, float eps) {
    constexpr int V = kVec<T>, NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
    __shared__ float red[2][TPR > 64 ? TPR / 64 : 1][1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv = 1.0f / (float)dim;
    // (one row per workgroup where the row's threads meet at barriers)
    for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < rows; row += (int64_t)gridDim.x * RPB) {
        const T* xr = x + row * ldx;
        float v[E][V];
        int n[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t c = (int64_t)(e * TPR + t) * V;
            n[e] = clip(dim - c, V);
            load_n<V>(xr + c, n[e], v[e]);
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += v[e][j];
        row_sum<TPR, 1>(s, red[0], t);
        const float mu = s[0] * inv;
        float q[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = j < n[e] ? v[e][j] - mu : 0.0f;
                q[0] += d * d;
            }
        row_sum<TPR, 1>(q, red[1], t);
        const float r = 1.0f / sqrtf(q[0] * inv + eps);
        if (t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t c = (int64_t)(e * TPR + t) * V;
            float o[V], p[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = (v[e][j] - mu) * r;
            if (w) {
                load_n<V>(w + c, n[e], p);
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] *= p[j];
            }
            if (b) {
                load_n<V>(b + c, n[e], p);
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] += p[j];
            }
            store_n<V>(y + row * ldy + c, n[e], o);
        }
    }
}

// Rows of any width, read three times: 512 x 65536 in bf16 39 us, 3.4 TB/s of one reading.
template <class T, class W>
__global__ __launch_bounds__(1024)
void layer_norm_long_kernel(const T* x, int64_t ldx, const W* __restrict__ w,
                            const W* __restrict__ b, T* y, int64_t ldy,
                            float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                            int64_t dim, float eps) {
    constexpr int V = kVec<T>, TPR = 1024;
    __shared__ float red[2][TPR / 64][1];
    const int t = threadIdx.x;
    const float inv = 1.0f / (float)dim;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * ldx;
        float s[1] = {0.0f}, q[1] = {0.0f}, v[V], p[V];
        for (int64_t c = (int64_t)t * V; c < dim; c += TPR * V) {
            load_n<V>(xr + c, clip(dim - c, V), v);
            float part = 0.0f;   // sums of a piece first: a chain of dim / 8192 additions
#pragma unroll
            for (int j = 0; j < V; ++j) part += v[j];
            s[0] += part;
        }
        row_sum<TPR, 1>(s, red[0], t);
        const float mu = s[0] * inv;
        for (int64_t c = (int64_t)t * V; c < dim; c += TPR * V) {
            const int n = clip(dim - c, V);
            load_n<V>(xr + c, n, v);
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = j < n ? v[j] - mu : 0.0f;
                part += d * d;
            }
            q[0] += part;
        }
        row_sum<TPR, 1>(q, red[1], t);
        const float r = 1.0f / sqrtf(q[0] * inv + eps);
        if (t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
        for (int64_t c = (int64_t)t * V; c < dim; c += TPR * V) {
            const int n = clip(dim - c, V);
            load_n<V>(xr + c, n, v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (v[j] - mu) * r;
            if (w) {
                load_n<V>(w + c, n, p);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] *= p[j];
            }
            if (b) {
                load_n<V>(b + c, n, p);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] += p[j];
            }
            store_n<V>(y + row * ldy + c, n, v);
        }
    }
}

// A 16-byte piece of a row as loaded, zeros past its n elements.
template <class T> struct Piece {
    u32x4 u;
    __device__ __forceinline__ void load(const T* p, int n) {
        u = u32x4{0u, 0u, 0u, 0u};
        if (n == kVec<T>) {
            u = load16(p);
        } else if (n > 0) {
            T e[kVec<T>];
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) e[j] = j < n ? p[j] : T(0);
            __builtin_memcpy(&u, e, 16);
        }
    }
    __device__ __forceinline__ void get(float (&v)[kVec<T>]) const {
        T e[kVec<T>];
        __builtin_memcpy(e, &u, 16);
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j) v[j] = (float)e[j];
    }
};

template <int TPR> constexpr int kBwdThreads = TPR > 512 ? TPR : 512;

template <class T, class W, int TPR, int E, bool PARAMS>
__global__ __launch_bounds__(kBwdThreads<TPR>)
void layer_norm_backward_kernel(const T* dy, int64_t lddy, const T* x, int64_t ldx, const W* __restrict__ w,
                                const float* __restrict__ mean, const float* __restrict__ rstd,
                                T* dx, int64_t lddx, float* __restrict__ part,
                                int64_t rows, int64_t dim) {
    constexpr int V = kVec<T>, NT = kBwdThreads<TPR>, RPB = NT / TPR;
    __shared__ float red[2][RPB][TPR > 64 ? TPR / 64 : 1][2];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv = 1.0f / (float)dim;
    int n[E];
    // the weight stays in registers where 128 of them hold it too
    constexpr bool HOLD_W = TPR < 1024 || E * V < 16;
    W wv[HOLD_W ? E : 1][V];
    float dw[E][V], db[E][V];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int64_t c = (int64_t)(e * TPR + t) * V;
        n[e] = clip(dim - c, V);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            wv[HOLD_W ? e : 0][j] = W(1.0f);
            dw[e][j] = db[e][j] = 0.0f;
            if (HOLD_W && w && j < n[e]) wv[e][j] = w[c + j];
        }
    }
    // every thread of a workgroup takes the same number of turns (barriers);
    // past the last row nothing is loaded, added or stored.  The next row is on its way
    // while this one is summed, as loaded (registers hold it for 16-bit types, and for
    // fp32 up to 8 elements a thread).
    constexpr bool AHEAD = E * V <= 8 || (sizeof(T) == 2 && TPR < 1024);
    const int64_t step = (int64_t)gridDim.x * RPB;
    Piece<T> nx[AHEAD ? E : 1], ng[AHEAD ? E : 1];
    float nmu = 0.0f, nr = 0.0f;
    auto fetch = [&](int64_t row) {
        const bool live = row < rows;
        nmu = live ? mean[row] : 0.0f;
        nr = live ? rstd[row] : 0.0f;
#pragma unroll
        for (int e = 0; e < (AHEAD ? E : 0); ++e) {
            const int64_t c = (int64_t)(e * TPR + t) * V;
            nx[e].load(x + row * ldx + c, live ? n[e] : 0);
            ng[e].load(dy + row * lddy + c, live ? n[e] : 0);
        }
    };
    int phase = 0;
    fetch((int64_t)blockIdx.x * RPB + sub);
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < rows; base += step) {
        const int64_t row = base + sub;
        const bool live = row < rows;
        float xv[E][V], gv[E][V];
        const float mu = nmu, r = nr;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int m = live ? n[e] : 0;
            if constexpr (AHEAD) {
                nx[e].get(xv[e]);
                ng[e].get(gv[e]);
#pragma unroll
                for (int j = 0; j < V; ++j) xv[e][j] = j < m ? xv[e][j] : mu;
            } else {
                const int64_t c = (int64_t)(e * TPR + t) * V;
                load_n<V>(x + row * ldx + c, m, xv[e], mu);
                load_n<V>(dy + row * lddy + c, m, gv[e]);
            }
        }
        if (base + step < rows) fetch(row + step);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!HOLD_W && w) {
#pragma unroll
                for (int j = 0; j < V; ++j) wv[0][j] = j < n[e] ? w[(int64_t)(e * TPR + t) * V + j] : W(0.0f);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (xv[e][j] - mu) * r, d = gv[e][j];
                if constexpr (PARAMS) {
                    dw[e][j] += d * xh;
                    db[e][j] += d;
                }
                const float g = d * (float)wv[HOLD_W ? e : 0][j];
                s[0] += g;
                s[1] += g * xh;
                xv[e][j] = xh;
                gv[e][j] = g;
            }
        }
        row_sum<TPR, 2>(s, red[phase][sub], t);
        phase ^= 1;
        const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t c = (int64_t)(e * TPR + t) * V;
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = r * (gv[e][j] - c0 - xv[e][j] * c1);
            store_n<V>(dx + row * lddx + c, live ? n[e] : 0, o);
        }
    }
    if constexpr (PARAMS) {
        // the workgroup's rows side by side, added in order
        float* out = part + (int64_t)blockIdx.x * 2 * dim;
        if constexpr (RPB > 1) {
            __shared__ float sum[2][E * TPR * V];
            for (int k = 0; k < RPB; ++k) {
                if (sub == k) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const int c = (e * TPR + t) * V + j;
                            sum[0][c] = k ? sum[0][c] + dw[e][j] : dw[e][j];
                            sum[1][c] = k ? sum[1][c] + db[e][j] : db[e][j];
                        }
                }
                __syncthreads();
            }
            for (int64_t c = threadIdx.x; c < dim; c += NT) {
                out[c] = sum[0][c];
                out[dim + c] = sum[1][c];
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int64_t c = (int64_t)(e * TPR + t) * V + j;
                    if (j < n[e]) {
                        out[c] = dw[e][j];
                        out[dim + c] = db[e][j];
                    }
                }
        }
    }
}

// dx of rows of any width, x and dy read twice: with the parameters' sums 512 x 65536 in
// bf16 80 us, 2.5 TB/s of one reading.
template <class T, class W>
__global__ __launch_bounds__(1024)
void layer_norm_backward_long_kernel(const T* dy, int64_t lddy, const T* x, int64_t ldx,
                                     const W* __restrict__ w, const float* __restrict__ mean,
                                     const float* __restrict__ rstd, T* dx, int64_t lddx, int64_t rows, int64_t dim) {
    constexpr int V = kVec<T>, TPR = 1024;
    __shared__ float red[2][TPR / 64][2];
    const int t = threadIdx.x;
    const float inv = 1.0f / (float)dim;
    int phase = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx, *gr = dy + row * lddy;
        const float mu = mean[row], r = rstd[row];
        float s[2] = {0.0f, 0.0f}, xv[V], gv[V], wv[V];
        for (int64_t c = (int64_t)t * V; c < dim; c += TPR * V) {
            const int n = clip(dim - c, V);
            load_n<V>(xr + c, n, xv, mu);
            load_n<V>(gr + c, n, gv);
            if (w) load_n<V>(w + c, n, wv);
            float p0 = 0.0f, p1 = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g = w ? gv[j] * wv[j] : gv[j];
                p0 += g;
                p1 += g * ((xv[j] - mu) * r);
            }
            s[0] += p0;
            s[1] += p1;
        }
        row_sum<TPR, 2>(s, red[phase], t);
        phase ^= 1;
        const float c0 = s[0] * inv, c1 = s[1] * inv;
        for (int64_t c = (int64_t)t * V; c < dim; c += TPR * V) {
            const int n = clip(dim - c, V);
            load_n<V>(xr + c, n, xv, mu);
            load_n<V>(gr + c, n, gv);
            if (w) load_n<V>(w + c, n, wv);
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j)
                o[j] = r * ((w ? gv[j] * wv[j] : gv[j]) - c0 - (xv[j] - mu) * r * c1);
            store_n<V>(dx + row * lddx + c, n, o);
        }
    }
}

// Partials of dw and db of wide rows: 16 bytes of columns a thread, `chunk` rows.
template <class T>
__global__ __launch_bounds__(256)
void layer_norm_columns_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x,
                               int64_t ldx, const float* __restrict__ mean,
                               const float* __restrict__ rstd, float* __restrict__ part,
                               int64_t rows, int64_t dim, int64_t chunk) {
    constexpr int V = kVec<T>;
    const int64_t r0 = (int64_t)blockIdx.y * chunk;
    const int64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    for (int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; c < dim; c += (int64_t)gridDim.x * 256 * V) {
        const int n = clip(dim - c, V);
        float a[V] = {}, b[V] = {};
#pragma unroll 4
        for (int64_t row = r0; row < r1; ++row) {
            const float mu = mean[row], r = rstd[row];
            float xv[V], gv[V];
            load_n<V>(x + row * ldx + c, n, xv);
            load_n<V>(dy + row * lddy + c, n, gv);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                a[j] += gv[j] * ((xv[j] - mu) * r);
                b[j] += gv[j];
            }
        }
        float* out = part + (int64_t)blockIdx.y * 2 * dim + c;
        store_n<V>(out, n, a);
        store_n<V>(out + dim, n, b);
    }
}

// dw and db from `count` rows of partials [2][dim]: 64 columns by 16 lanes of
// rows a workgroup, eight loads in flight, the lanes' sums added in order.
template <class W>
__global__ __launch_bounds__(1024)
void layer_norm_params_kernel(const float* __restrict__ part, int count, int64_t dim,
                              W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float red[16][64];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < 2 * dim; c0 += (int64_t)gridDim.x * 64) {
        const int64_t c = c0 + tx;
        float a = 0.0f;
        if (c < 2 * dim) {
            const float* p = part + c;
            int k = ty;
            for (; k + 7 * 16 < count; k += 8 * 16) {
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = p[(int64_t)(k + 16 * u) * 2 * dim];
#pragma unroll
                for (int u = 0; u < 8; ++u) a += v[u];
            }
            for (; k < count; k += 16) a += p[(int64_t)k * 2 * dim];
        }
        red[ty][tx] = a;
        __syncthreads();
        if (ty == 0 && c < 2 * dim) {
            a = red[0][tx];
#pragma unroll
            for (int k = 1; k < 16; ++k) a += red[k][tx];
            if (c < dim) {
                if (dw) dw[c] = round_to<W>(a);
            } else if (db) {
                db[c - dim] = round_to<W>(a);
            }
        }
        __syncthreads();
    }
}

// The threads per row and 16-byte pieces per thread for a width: the fewest
// threads that hold it, with up to 32 elements each in the forward pass.  The
// backward one keeps five values of each and the next row: 8 elements (8192 x 4096
// in bf16: 47 us, with 16 of half the threads and no row ahead 63), 16 without sums.
template <class T, bool BWD, class F>
int with_shape(int64_t dim, F f) {
    constexpr int V = kVec<T>;
    using std::integral_constant;
#define CDX_LN_SHAPE(TPR, EL) \
    if (dim <= (int64_t)TPR * EL) return f(integral_constant<int, TPR>{}, integral_constant<int, EL / V>{})
    CDX_LN_SHAPE(16, 8);
    CDX_LN_SHAPE(64, 8);
    if constexpr (BWD) {
        CDX_LN_SHAPE(128, 8);
        CDX_LN_SHAPE(256, 8);
        CDX_LN_SHAPE(512, 8);
        CDX_LN_SHAPE(1024, 8);
        CDX_LN_SHAPE(1024, 16);
    } else {
        CDX_LN_SHAPE(64, 16);
        CDX_LN_SHAPE(64, 32);
        CDX_LN_SHAPE(256, 16);
        CDX_LN_SHAPE(256, 32);
        CDX_LN_SHAPE(1024, 16);
        CDX_LN_SHAPE(1024, 32);
    }
#undef CDX_LN_SHAPE
    return f(integral_constant<int, 0>{}, integral_constant<int, 0>{});
}

// Rows of partials: workgroups of the backward kernel, two per CU at most (one of
// 1024 threads).  Rows of more than 8192 elements keep no column sums, which would
// spill: a second pass over x and dy forms them, 32 rows at least each (2048 x 16384:
// 88 us in bf16 and 140 in fp32, with the sums kept 127 and 161).
constexpr int kBwdGroups = 512;

// Workgroups of a launch: the threads of one are counted in 32 bits.
constexpr int64_t kMostGroups = 1 << 20;

template <class T> int64_t partial_rows(int64_t rows, int64_t dim) {
    int64_t out = 0;
    (void)with_shape<T, true>(dim, [&](auto tpr, auto e) {
        constexpr int TPR = decltype(tpr)::value, EL = decltype(e)::value * kVec<T>;
        if constexpr (TPR == 0 || EL > 8) {
            out = std::min<int64_t>(ceil_div(rows, (int64_t)32), 128);
        } else {
            constexpr int NT = kBwdThreads<TPR>;
            out = std::min<int64_t>(ceil_div(rows, (int64_t)(NT / TPR)), NT > 512 ? kBwdGroups / 2 : kBwdGroups);
        }
        return 0;
    });
    return out;
}

template <class T, class W>
int forward_t(const T* x, int64_t ldx, const W* w, const W* b, T* y, int64_t ldy, float* mean,
              float* rstd, int64_t rows, int64_t dim, float eps, hipStream_t stream) {
    return with_shape<T, false>(dim, [&](auto tpr, auto e) {
        constexpr int TPR = decltype(tpr)::value, E = decltype(e)::value;
        if constexpr (TPR == 0) {
            const int64_t g = std::min(rows, kMostGroups);
            hipLaunchKernelGGL((layer_norm_long_kernel<T, W>), dim3((unsigned)g), dim3(1024), 0,
                               stream, x, ldx, w, b, y, ldy, mean, rstd, rows, dim, eps);
        } else {
            constexpr int NT = TPR > 256 ? TPR : 256;
            const int64_t g = std::min(ceil_div(rows, (int64_t)(NT / TPR)), kMostGroups);
            hipLaunchKernelGGL((layer_norm_kernel<T, W, TPR, E>), dim3((unsigned)g), dim3(NT), 0,
                               stream, x, ldx, w, b, y, ldy, mean, rstd, rows, dim, eps);
        }
        return hip_error(hipGetLastError(), "layer_norm_kernel launch");
    });
}

template <class T, class W>
int backward_t(const T* dy, int64_t lddy, const T* x, int64_t ldx, const W* w, const float* mean,
               const float* rstd, T* dx, int64_t lddx, W* dw, W* db, int64_t rows, int64_t dim,
               float* ws, hipStream_t stream) {
    const bool params = dw || db;
    const int64_t count = partial_rows<T>(rows, dim);
    int st = with_shape<T, true>(dim, [&](auto tpr, auto e) {
        constexpr int TPR = decltype(tpr)::value, E = decltype(e)::value;
        constexpr bool WIDE = TPR == 0 || E * kVec<T> > 8;   // column sums apart
        if constexpr (WIDE) {
            if (params) {   // (first: dx may be written over x or dy)
                hipLaunchKernelGGL((layer_norm_columns_kernel<T>),
                                   dim3((unsigned)std::min(ceil_div(dim, (int64_t)(256 * kVec<T>)), kMostGroups),
                                        (unsigned)count),
                                   dim3(256), 0, stream, dy, lddy, x, ldx, mean, rstd, ws, rows, dim,
                                   ceil_div(rows, count));
                const int st1 = hip_error(hipGetLastError(), "layer_norm_columns_kernel launch");
                if (st1) return st1;
            }
        }
        if constexpr (TPR == 0) {
            const int64_t g = std::min(rows, kMostGroups);
            hipLaunchKernelGGL((layer_norm_backward_long_kernel<T, W>), dim3((unsigned)g),
                               dim3(1024), 0, stream, dy, lddy, x, ldx, w, mean, rstd, dx, lddx,
                               rows, dim);
        } else {
            constexpr int NT = kBwdThreads<TPR>;
            constexpr int most = NT > 512 ? kBwdGroups / 2 : kBwdGroups;
            const dim3 grid((unsigned)std::min<int64_t>(ceil_div(rows, (int64_t)(NT / TPR)), most));
            if constexpr (!WIDE) {
                if (params) {
                    hipLaunchKernelGGL((layer_norm_backward_kernel<T, W, TPR, E, true>), grid,
                                       dim3(NT), 0, stream, dy, lddy, x, ldx, w, mean, rstd, dx,
                                       lddx, ws, rows, dim);
                    return hip_error(hipGetLastError(), "layer_norm_backward_kernel launch");
                }
            }
            hipLaunchKernelGGL((layer_norm_backward_kernel<T, W, TPR, E, false>), grid, dim3(NT), 0,
                               stream, dy, lddy, x, ldx, w, mean, rstd, dx, lddx, ws, rows, dim);
        }
        return hip_error(hipGetLastError(), "layer_norm_backward_kernel launch");
    });
    if (st || !params) return st;
    hipLaunchKernelGGL(layer_norm_params_kernel<W>,
                       dim3((unsigned)std::min(ceil_div(2 * dim, (int64_t)64), kMostGroups)), dim3(1024), 0, stream, ws, (int)count, dim, dw, db);
    return hip_error(hipGetLastError(), "layer_norm_params_kernel launch");
}

template <class T>
__global__ __launch_bounds__(256)
void zero_kernel(T* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = T(0);
}

// f(T value, W value) for the element and parameter types.
template <class F> int with_types(int dtype, int pdtype, F f) {
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if constexpr (!std::is_same_v<T, float>) {
            if (pdtype == dtype) return f(t, t);
        }
        return f(t, float{});
    });
}

}  // namespace

int launch_zero(void* p, int64_t n, int dtype, hipStream_t stream) {
    const int64_t g = ceil_div(n, (int64_t)256);
    const dim3 grid((unsigned)(g < 65536 ? g : 65536));
    if (dtype == CDX_DTYPE_F32)
        hipLaunchKernelGGL(zero_kernel<float>, grid, dim3(256), 0, stream, static_cast<float*>(p), n);
    else   // zero has the same bits in both 16-bit types
        hipLaunchKernelGGL(zero_kernel<uint16_t>, grid, dim3(256), 0, stream,
                           static_cast<uint16_t*>(p), n);
    return hip_error(hipGetLastError(), "zero_kernel launch");
}

int launch_layer_norm(const void* x, int64_t ldx, const void* w, const void* b, void* y,
                      int64_t ldy, float* mean, float* rstd, int64_t rows, int64_t dim, float eps,
                      int dtype, int pdtype, hipStream_t stream) {
    return with_types(dtype, pdtype, [&](auto t, auto p) {
        using T = decltype(t);
        using W = decltype(p);
        return forward_t(static_cast<const T*>(x), ldx, static_cast<const W*>(w),
                         static_cast<const W*>(b), static_cast<T*>(y), ldy, mean, rstd, rows, dim,
                         eps, stream);
    });
}

size_t layer_norm_partial_floats(int64_t rows, int64_t dim, int dtype) {
    int64_t n = 0;
    (void)with_dtype(dtype, [&](auto t) {
        n = partial_rows<decltype(t)>(rows, dim);
        return 0;
    });
    return (size_t)n * 2 * (size_t)dim;
}

int launch_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                               const void* w, const float* mean, const float* rstd, void* dx,
                               int64_t lddx, void* dw, void* db, int64_t rows, int64_t dim,
                               int dtype, int pdtype, float* ws, hipStream_t stream) {
    return with_types(dtype, pdtype, [&](auto t, auto p) {
        using T = decltype(t);
        using W = decltype(p);
        return backward_t(static_cast<const T*>(dy), lddy, static_cast<const T*>(x), ldx,
                          static_cast<const W*>(w), mean, rstd, static_cast<T*>(dx), lddx,
                          static_cast<W*>(dw), static_cast<W*>(db), rows, dim, ws, stream);
    });
}

}  // namespace cdx
