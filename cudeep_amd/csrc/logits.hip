// Rows of logits x over a vocabulary, at temperature T:
//   m = max x, S = sum exp((x - m) / T), L = log S, log softmax l = (x - m) / T - L, p = exp l;
//   the token's log probability l_t, the entropy H = -sum p l = L - sum p (x - m) / T;
//   gradient of g l_t + h H:  ((g [v = t] - g p) - h p (l + H)) / T;
//   distillation from a row's entries (i_k, v_k):  q = softmax(v / T),
//   loss = sum q (log q - l_{i_k}),  gradient w / T (p - sum over k with i_k = v of q_k).
//
// One pass forms m, S and sum exp(.) (x - m) together: a thread holds its own running maximum and
// rescales its sums when that grows, threads are joined in a fixed order.  Differences from the maximum
// are formed before they are scaled: (x - m) is exact or nearly so, where x / T and m / T rounded apart
// would lose |m| / T 2^-24.  The running maximum begins at the lowest finite value, so that masked
// logits (-infinity, or a type's lowest value) never meet infinity - infinity; a row of -infinity
// alone has S = 0, and L = -infinity says so.
#include "logits.hpp"

namespace cdx {
namespace {

using namespace b8;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kFar = -1e30f;       // a difference so large that its exponential is 0 at any temperature
constexpr int kUnroll = 4;           // 16-byte pieces of a thread in flight

template <class T> constexpr int kVec = 16 / (int)sizeof(T);

// The sums of some of a row's elements: m their maximum, s = sum e, t = sum e (x - m), e = exp((x - m) / T).
struct Part { float m, s, t; };

template <bool ENT> __device__ __forceinline__ void rescale(Part& a, float m, float c) {
    const float d = fmaxf(a.m - m, kFar), f = __builtin_amdgcn_exp2f(d * c);
    if constexpr (ENT) a.t = f * (a.t + a.s * d);
    a.s *= f;
    a.m = m;
}

template <bool ENT> __device__ __forceinline__ Part join(Part a, Part b, float c) {
    const float m = fmaxf(a.m, b.m);
    rescale<ENT>(a, m, c);
    rescale<ENT>(b, m, c);
    return {m, a.s + b.s, ENT ? a.t + b.t : 0.0f};
}

// Adds elements to the sums; the largest of them.
template <bool ENT, int N> __device__ __forceinline__ float take(Part& a, const float (&x)[N], float c) {
    float most = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) most = fmaxf(most, x[j]);
    const float m = fmaxf(a.m, most);
    rescale<ENT>(a, m, c);
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = x[j] - m, e = __builtin_amdgcn_exp2f(d * c);
        s += e;
        if constexpr (ENT) t += e * fmaxf(d, kFar);
    }
    a.s += s;
    if constexpr (ENT) a.t += t;
    return most;
}

// The join over a workgroup of NT threads, in all of them.
template <bool ENT, int NT> __device__ __forceinline__ Part join_all(Part a, float c, Part* red) {
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        const Part b{__shfl_xor(a.m, k), __shfl_xor(a.s, k), ENT ? __shfl_xor(a.t, k) : 0.0f};
        a = (threadIdx.x & k) ? join<ENT>(b, a, c) : join<ENT>(a, b, c);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    a = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) a = join<ENT>(a, red[w], c);
    return a;
}

// kUnroll pieces of a thread as loaded: piece u begins at element `at` + u * NT * kVec; elements from
// `end` on read as -infinity.
template <class T, int NT> struct Pieces {
    static constexpr int N = kUnroll * kVec<T>, STRIDE = NT * kVec<T>;
    u32x4 u[kUnroll];
    __device__ __forceinline__ void load(const T* x, int at) {
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) u[i] = load16(x + at + i * STRIDE);
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            T e[kVec<T>];
            __builtin_memcpy(e, &u[i], 16);
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) v[i * kVec<T> + j] = (float)e[j];
        }
    }
    __device__ __forceinline__ static void get_checked(const T* x, int at, int end, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int from = at + i * STRIDE, n = end - from;
            float w[kVec<T>];
            load_n<kVec<T>>(x + (n > 0 ? from : 0), n, w, -__builtin_inff());
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) v[i * kVec<T> + j] = w[j];
        }
    }
};

// The sums of elements begin .. end - 1, and, with TOP, the thread's largest value and the round it first
// lies in (-infinity and 0 where nothing is larger).
template <class T, int NT, bool ENT, bool TOP>
__device__ __forceinline__ Part scan(const T* x, int begin, int end, float c, float& best, int& round) {
    using P = Pieces<T, NT>;
    constexpr int ROUND = NT * P::N;
    Part a{kLowest, 0.0f, 0.0f};
    const int whole = (end - begin) / ROUND;
    const int at = begin + (int)threadIdx.x * kVec<T>;
    float v[P::N];
    best = -__builtin_inff();
    round = 0;
    auto use = [&](int r) {
        const float most = take<ENT>(a, v, c);
        if constexpr (TOP) {
            round = most > best ? r : round;
            best = fmaxf(best, most);
        }
    };
    if (whole > 0) {
        P now, next;
        now.load(x, at);
        for (int r = 0; r < whole; ++r) {
            if (r + 1 < whole) next.load(x, at + (r + 1) * ROUND);
            now.get(v);
            use(r);
            now = next;
        }
    }
    if (begin + whole * ROUND < end) {
        P::get_checked(x, at + whole * ROUND, end, v);
        use(whole);
    }
    return a;
}

// ---- the largest elements ---------------------------------------------------------------------

typedef unsigned long long u64;

// Orders by value, then the lowest index first; the two zeros are equal, NaN is above everything.
__device__ __forceinline__ u64 key_of(float x, int index) {
    uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    u = x != x ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return (u64)u << 32 | (uint32_t)~index;
}
__device__ __forceinline__ int key_index(u64 k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(u64 k) {
    const uint32_t u = (uint32_t)(k >> 32);
    if (u == 0xffffffffu) return __builtin_nanf("");
    return __builtin_bit_cast(float, u ^ (u >> 31 ? 0x80000000u : 0xffffffffu));
}

constexpr int kTopThreads = 256;
constexpr int kRoundKeys = kTopThreads * 8;             // at most, of one round of pieces
constexpr int kTopBuffer = kRoundKeys + 512;

struct TopShared {
    u64 keys[kTopBuffer];
    u64 best[kTopThreads];
    u64 threshold;
    int count, chosen, who[kMaxTop];
};

// Leaves the `k` largest of the first `count` keys in their order at the front (all threads call it).
// A key's place is the number of larger ones; keys differ, so that places do.
__device__ __forceinline__ int keep_largest(u64* keys, int count, int k) {
    constexpr int MOST = (kTopBuffer + kTopThreads - 1) / kTopThreads;
    u64 mine[MOST];
    int place[MOST];
    int n = 0;
    for (int i = threadIdx.x; i < count; i += kTopThreads, ++n) {
        const u64 key = keys[i];
        int larger = 0;
        for (int j = 0; j < count; ++j) larger += keys[j] > key;
        // (a static index: the arrays stay in registers)
#pragma unroll
        for (int s = 0; s < MOST; ++s)
            if (s == n) { mine[s] = key; place[s] = larger; }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < MOST; ++s)
        if (s < n && place[s] < k) keys[place[s]] = mine[s];
    __syncthreads();
    return count < k ? count : k;
}

// The k-th largest of the threads' keys (0 where fewer are there), by halving: the first wave holds all of
// them, four a lane.
__device__ __forceinline__ u64 kth_largest(const u64* best, int k) {
    const int lane = threadIdx.x & 63;
    u64 v[kTopThreads / 64];
#pragma unroll
    for (int i = 0; i < kTopThreads / 64; ++i) v[i] = best[lane + 64 * i];
    u64 at = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const u64 up = at | 1ull << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kTopThreads / 64; ++i) n += __popcll(__ballot(v[i] >= up));
        if (n >= k) at = up;
        if (n == k) break;
    }
    return at;
}

// The k largest of elements begin .. end - 1 at the front of sh.keys; how many there are.  `best`, `round`:
// the scan's.  Each thread's largest element is known; the k-th largest of those is a bound that the k
// largest elements of all reach, and they lie with the k threads whose own reach it: only those
// threads' elements are looked at again.
template <class T>
__device__ __forceinline__ int largest(const T* x, int begin, int end, int k, float best, int round, TopShared& sh) {
    using P = Pieces<T, kTopThreads>;
    constexpr int V = kVec<T>;
    const int tid = threadIdx.x;
    u64 mine = 0;
    // the first element of its round with that value
    const int at = begin + tid * V + round * (kTopThreads * P::N);
    if (at < end) {
        float v[P::N];
        P::get_checked(x, at, end, v);
#pragma unroll
        for (int j = P::N - 1; j >= 0; --j) {
            const int index = at + j / V * P::STRIDE + j % V;
            // (NaN alone: the first there is)
            if (index < end && (v[j] == best || (j == 0 && mine == 0))) mine = key_of(v[j], index);
        }
    }
    sh.best[tid] = mine;
    if (tid == 0) sh.count = sh.chosen = 0;
    __syncthreads();
    if (tid < 64) {
        const u64 t = kth_largest(sh.best, k);
        if (tid == 0) sh.threshold = t;
    }
    __syncthreads();
    u64 threshold = sh.threshold;
    if (mine && mine >= threshold) {
        const int i = atomicAdd(&sh.chosen, 1);
        if (i < kMaxTop) sh.who[i] = tid;
    }
    __syncthreads();
    const int chosen = sh.chosen < kMaxTop ? sh.chosen : kMaxTop;
    const int pieces = (int)(((int64_t)(end - begin) + kTopThreads * V - 1) / (kTopThreads * V));
    const int64_t items = (int64_t)chosen * pieces;
    for (int64_t first = 0; first < items; first += kTopThreads) {
        const int count = sh.count;
        __syncthreads();   // everybody has read the count
        if (count > kTopBuffer - kRoundKeys) {
            const int left = keep_largest(sh.keys, count, k);
            if (left == k) threshold = sh.keys[k - 1] > threshold ? sh.keys[k - 1] : threshold;
            if (tid == 0) sh.count = left;
            __syncthreads();
        }
        const int64_t i = first + tid;
        if (i < items) {
            const int from = begin + ((int)(i % pieces) * kTopThreads + sh.who[i / pieces]) * V, n = end - from;
            if (n > 0) {
                float v[V];
                load_n<V>(x + from, n, v);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const u64 key = key_of(v[j], from + j);
                    if (j < n && key >= threshold) {
                        const int slot = atomicAdd(&sh.count, 1);
                        if (slot < kTopBuffer) sh.keys[slot] = key;
                    }
                }
            }
        }
        __syncthreads();
    }
    return keep_largest(sh.keys, sh.count < kTopBuffer ? sh.count : kTopBuffer, k);
}

// ---- log probabilities --------------------------------------------------------------------------

struct LogprobParams {
    LogitRows r;
    const int64_t* targets;
    float* logprob; RowStats* stats; float* entropy;
    int top; float* top_logprob; int64_t* top_index;
    int parts, length;                 // a row's parts, elements each
    Part* part; u64* keys;             // [rows][parts], [rows][parts][top]
};

// (x - m) / T - L, -infinity in a row without a finite logit.
__device__ __forceinline__ float log_softmax(float x, RowStats s, float inv_t) {
    return s.l == -__builtin_inff() ? s.l : (x - s.m) * inv_t - s.l;
}

__device__ __forceinline__ float entropy_of(const Part& a, float l, float inv_t) {
    return a.s == 0.0f ? 0.0f : l - a.t / a.s * inv_t;
}

// What a row's sums give; one thread.
template <class T> __device__ __forceinline__ void finish_row(const LogprobParams& p, int64_t row, const Part& a, RowStats s) {
    const int64_t t = p.targets[row];
    float lp = 0.0f;
    if (t >= p.r.vocab) lp = __builtin_nanf("");
    else if (t >= 0) lp = log_softmax((float)static_cast<const T*>(p.r.x)[row * p.r.ldx + t], s, p.r.inv_t);
    p.logprob[row] = lp;
    p.stats[row] = s;
    if (p.entropy) p.entropy[row] = entropy_of(a, s.l, p.r.inv_t);
}

// A workgroup a row, or a part of one.
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(kTopThreads)
void logprob_kernel(LogprobParams p) {
    __shared__ Part red[kTopThreads / 64];
    __shared__ std::conditional_t<TOP, TopShared, char> sh;
    const int64_t row = blockIdx.x / p.parts;
    const int part = (int)(blockIdx.x % p.parts);
    const T* x = static_cast<const T*>(p.r.x) + row * p.r.ldx;
    const int begin = part * p.length;
    const int end = p.r.vocab - begin < p.length ? (int)p.r.vocab : begin + p.length;
    const float c = p.r.inv_t * kLog2e;
    float best;
    int round;
    Part a = scan<T, kTopThreads, ENT, TOP>(x, begin, end, c, best, round);
    a = join_all<ENT, kTopThreads>(a, c, red);
    if (p.parts > 1) {
        if (threadIdx.x == 0) p.part[row * p.parts + part] = a;
        if constexpr (TOP) {
            const int n = largest(x, begin, end, p.top, best, round, sh);
            if ((int)threadIdx.x < p.top)
                p.keys[(row * p.parts + part) * p.top + threadIdx.x] = (int)threadIdx.x < n ? sh.keys[threadIdx.x] : 0;
        }
        return;
    }
    const RowStats s{a.m, logf(a.s)};
    if (threadIdx.x == 0) finish_row<T>(p, row, a, s);
    if constexpr (TOP) {
        largest(x, begin, end, p.top, best, round, sh);
        if ((int)threadIdx.x < p.top) {
            const u64 key = sh.keys[threadIdx.x];
            p.top_logprob[row * p.top + threadIdx.x] = log_softmax(key_value(key), s, p.r.inv_t);
            p.top_index[row * p.top + threadIdx.x] = key_index(key);
        }
    }
}

// A row's parts together.
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(kTopThreads)
void logprob_join_kernel(LogprobParams p) {
    __shared__ Part red[kTopThreads / 64];
    __shared__ u64 keys[TOP ? kTopBuffer : 1];
    const int64_t row = blockIdx.x;
    const float c = p.r.inv_t * kLog2e;
    Part a{kLowest, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < p.parts; i += kTopThreads) a = join<ENT>(a, p.part[row * p.parts + i], c);
    a = join_all<ENT, kTopThreads>(a, c, red);
    const RowStats s{a.m, logf(a.s)};
    if (threadIdx.x == 0) finish_row<T>(p, row, a, s);
    if constexpr (TOP) {
        const int count = p.parts * p.top;   // at most kTopBuffer
        for (int i = threadIdx.x; i < count; i += kTopThreads) keys[i] = p.keys[row * count + i];
        __syncthreads();
        // (parts of fewer elements than `top` leave zeros, which are below every key)
        for (int i = threadIdx.x; i < count; i += kTopThreads)
            if (keys[i] == 0) keys[i] = i;   // small, and all different
        __syncthreads();
        keep_largest(keys, count, p.top);
        if ((int)threadIdx.x < p.top) {
            const u64 key = keys[threadIdx.x];
            p.top_logprob[row * p.top + threadIdx.x] = log_softmax(key_value(key), s, p.r.inv_t);
            p.top_index[row * p.top + threadIdx.x] = key_index(key);
        }
    }
}

// The gradient, element by element: a workgroup takes kBackward elements of a row.
constexpr int kBackwardThreads = 256;
template <class T> constexpr int kBackward = kBackwardThreads * kUnroll * kVec<T>;

template <class T>
__global__ __launch_bounds__(kBackwardThreads)
void logprob_backward_kernel(LogitRows r, const int64_t* __restrict__ targets, const RowStats* __restrict__ stats,
                             const float* __restrict__ g_lp, const float* __restrict__ entropy,
                             const float* __restrict__ g_h, T* grad, int64_t ldg, int parts) {
    constexpr int V = kVec<T>;
    const int64_t row = blockIdx.x / parts;
    const int64_t first = (int64_t)(blockIdx.x % parts) * kBackward<T>;
    const T* x = static_cast<const T*>(r.x) + row * r.ldx;
    T* out = grad + row * ldg;
    const RowStats s = stats[row];
    const int64_t t = targets[row];
    float g = g_lp ? g_lp[row] : 0.0f;
    if (t < 0) g = 0.0f;
    if (t >= r.vocab && g != 0.0f) g = __builtin_nanf("");
    const float h = g_h ? g_h[row] : 0.0f;
    // -g p - h p (l + H) = -p (h l + (h H + g))
    const float hs = h * r.inv_t, gs = g * r.inv_t, both = h != 0.0f ? (h * entropy[row] + g) * r.inv_t : gs;
    const bool none = (g == 0.0f && h == 0.0f) || s.l == -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t at = first + ((int64_t)i * kBackwardThreads + threadIdx.x) * V;
        const int64_t left = r.vocab - at;
        const int n = left < 0 ? 0 : left > V ? V : (int)left;
        if (n == 0) break;
        float v[V] = {};
        if (!none) {
            load_n<V>(x + at, n, v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float l = (v[j] - s.m) * r.inv_t - s.l, p = __builtin_amdgcn_exp2f(l * kLog2e);
                v[j] = -p * (hs * fmaxf(l, kFar) + both);
            }
            if (t >= at && t < at + V) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (t == at + j) v[j] += gs;
            }
        }
        store_n<V>(out + at, n, v);
    }
}

// ---- distillation ---------------------------------------------------------------------------------

constexpr int kDistillThreads = 1024;

struct DistillParams {
    DistillArgs a;
    int parts, length;
    Part* part; float* found;          // [rows][parts], [rows][count]: the logits at the entries
};

// A row's entries: index (-1: does not count), q and the logit there.
struct Entries {
    int index[kMaxEntries];
    float q[kMaxEntries], x[kMaxEntries];
};

__device__ __forceinline__ int entry_index(const DistillArgs& a, int64_t row, int k) {
    const int64_t i = a.index64 ? static_cast<const int64_t*>(a.index)[row * a.ldi + k]
                                : static_cast<const int32_t*>(a.index)[row * a.ldi + k];
    return i < 0 ? -1 : i < a.r.vocab ? (int)i : (int)kMaxVocab;   // (kMaxVocab: past the vocabulary)
}
__device__ __forceinline__ float entry_value(const DistillArgs& a, int64_t row, int k) {
    const int64_t at = row * a.ldt + k;
    if (a.teacher_dtype == CDX_DTYPE_F32) return static_cast<const float*>(a.teacher)[at];
    if (a.teacher_dtype == CDX_DTYPE_BF16) return (float)static_cast<const bf16*>(a.teacher)[at];
    return (float)static_cast<const f16*>(a.teacher)[at];
}

template <int NT, class F> __device__ __forceinline__ float reduce_all(float v, float* red, F f) {
#pragma unroll
    for (int k = 1; k < 64; k *= 2) v = f(v, __shfl_xor(v, k));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = f(v, red[w]);
    return v;
}

// q of the row's entries in e.q (whose e.index and e.x are there) and the loss; whether any counts.
template <int NT>
__device__ __forceinline__ bool entries_loss(const DistillArgs& a, int64_t row, RowStats s, Entries& e, float* red, float& loss) {
    const float inf = __builtin_inff();
    const int tid = threadIdx.x;
    float top = -inf;
    for (int k = tid; k < a.count; k += NT) {
        e.q[k] = e.index[k] < 0 ? -inf : entry_value(a, row, k);
        top = fmaxf(top, e.q[k]);
    }
    top = reduce_all<NT>(top, red, [](float u, float v) { return fmaxf(u, v); });
    float sum = 0.0f;
    bool nan = false;
    for (int k = tid; k < a.count; k += NT) {
        nan |= e.q[k] != e.q[k];
        if (top > -inf) sum += expf((e.q[k] - top) * a.r.inv_t);
    }
    sum = reduce_all<NT>(nan ? __builtin_nanf("") : sum, red, [](float u, float v) { return u + v; });
    const float log_sum = logf(sum);
    float part = 0.0f;
    for (int k = tid; k < a.count; k += NT) {
        const float lq = (e.q[k] - top) * a.r.inv_t - log_sum;
        float q = 0.0f;
        if (sum != 0.0f) q = sum != sum ? sum : expf(lq);
        e.q[k] = q;
        if (q != 0.0f) {
            const float l = e.index[k] == (int)kMaxVocab ? __builtin_nanf("") : log_softmax(e.x[k], s, a.r.inv_t);
            part += q * (lq - l);
        }
    }
    loss = reduce_all<NT>(part, red, [](float u, float v) { return u + v; });
    return sum != 0.0f;
}

// The gradient of elements begin .. end - 1; all threads call it, with the row's entries in LDS.
template <class T, int NT>
__device__ __forceinline__ void distill_grad(const DistillArgs& a, int64_t row, int begin, int end, RowStats s,
                                             bool some, float loss, const Entries& e) {
    constexpr int V = kVec<T>;
    const T* x = static_cast<const T*>(a.r.x) + row * a.r.ldx;
    T* out = static_cast<T*>(a.grad) + row * a.ldg;
    const float w = a.weight[row];
    const bool none = !some || w == 0.0f || s.l == -__builtin_inff();
    // (an index past the vocabulary shows in every element)
    const float f = loss != loss ? loss : w * a.r.inv_t;
    for (int at = begin + (int)threadIdx.x * V; at < end; at += NT * V) {
        const int n = end - at;
        float v[V] = {};
        if (!none) {
            load_n<V>(x + at, n, v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = f * __builtin_amdgcn_exp2f(((v[j] - s.m) * a.r.inv_t - s.l) * kLog2e);
        }
        store_n<V>(out + at, n, v);
    }
    if (none) return;
    __syncthreads();   // the entries' places are written above and once more below
    for (int k = threadIdx.x; k < a.count; k += NT) {
        const int i = e.index[k];
        if (i < begin || i >= end) continue;
        float q = 0.0f;   // of all entries of this index: each of them stores the same
        for (int j = 0; j < a.count; ++j) q += e.index[j] == i ? e.q[j] : 0.0f;
        out[i] = (T)(f * (__builtin_amdgcn_exp2f(((e.x[k] - s.m) * a.r.inv_t - s.l) * kLog2e) - q));
    }
}

// A workgroup a row: sums, entries, and the gradient, for which the row is read again.
template <class T, bool GRAD>
__global__ __launch_bounds__(kDistillThreads)
void distill_kernel(DistillParams p) {
    constexpr int NT = kDistillThreads;
    __shared__ Part red[NT / 64];
    __shared__ float redf[NT / 64];
    __shared__ Entries e;
    const DistillArgs& a = p.a;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.r.x) + row * a.r.ldx;
    const float c = a.r.inv_t * kLog2e;
    for (int k = threadIdx.x; k < a.count; k += NT) {
        const int i = entry_index(a, row, k);
        e.index[k] = i;
        e.x[k] = i >= 0 && i < a.r.vocab ? (float)x[i] : 0.0f;
    }
    float best;
    int round;
    Part s = scan<T, NT, false, false>(x, 0, (int)a.r.vocab, c, best, round);
    s = join_all<false, NT>(s, c, red);
    const RowStats st{s.m, logf(s.s)};
    float loss;
    const bool some = entries_loss<NT>(a, row, st, e, redf, loss);
    if (threadIdx.x == 0) a.loss[row] = loss;
    if constexpr (GRAD) {
        __syncthreads();
        distill_grad<T, NT>(a, row, 0, (int)a.r.vocab, st, some, loss, e);
    }
}

// A row in parts: their sums, and the logits at the entries that lie in them (the gradient may take their
// place).
template <class T>
__global__ __launch_bounds__(kDistillThreads)
void distill_part_kernel(DistillParams p) {
    constexpr int NT = kDistillThreads;
    __shared__ Part red[NT / 64];
    const DistillArgs& a = p.a;
    const int64_t row = blockIdx.x / p.parts;
    const int part = (int)(blockIdx.x % p.parts);
    const T* x = static_cast<const T*>(a.r.x) + row * a.r.ldx;
    const int begin = part * p.length;
    const int end = a.r.vocab - begin < p.length ? (int)a.r.vocab : begin + p.length;
    for (int k = threadIdx.x; k < a.count; k += NT) {
        const int i = entry_index(a, row, k);
        if (i >= begin && i < end) p.found[row * a.count + k] = (float)x[i];
    }
    const float c = a.r.inv_t * kLog2e;
    float best;
    int round;
    Part s = scan<T, NT, false, false>(x, begin, end, c, best, round);
    s = join_all<false, NT>(s, c, red);
    if (threadIdx.x == 0) p.part[row * p.parts + part] = s;
}

// The parts together: every workgroup for itself, then the gradient of its own part.  Without a gradient, one
// workgroup a row.
template <class T, bool GRAD>
__global__ __launch_bounds__(kDistillThreads)
void distill_join_kernel(DistillParams p) {
    constexpr int NT = kDistillThreads;
    __shared__ Part red[NT / 64];
    __shared__ float redf[NT / 64];
    __shared__ Entries e;
    const DistillArgs& a = p.a;
    const int64_t row = GRAD ? blockIdx.x / p.parts : blockIdx.x;
    const int part = GRAD ? (int)(blockIdx.x % p.parts) : 0;
    const float c = a.r.inv_t * kLog2e;
    for (int k = threadIdx.x; k < a.count; k += NT) {
        const int i = entry_index(a, row, k);
        e.index[k] = i;
        e.x[k] = i >= 0 && i < a.r.vocab ? p.found[row * a.count + k] : 0.0f;
    }
    Part s{kLowest, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < p.parts; i += NT) s = join<false>(s, p.part[row * p.parts + i], c);
    s = join_all<false, NT>(s, c, red);
    const RowStats st{s.m, logf(s.s)};
    float loss;
    const bool some = entries_loss<NT>(a, row, st, e, redf, loss);
    if (part == 0 && threadIdx.x == 0) a.loss[row] = loss;
    if constexpr (GRAD) {
        const int begin = part * p.length;
        const int end = a.r.vocab - begin < p.length ? (int)a.r.vocab : begin + p.length;
        __syncthreads();
        distill_grad<T, NT>(a, row, begin, end, st, some, loss, e);
    }
}

// ---- launches -----------------------------------------------------------------------------------

// How many parts of how many elements a row is cut into.
struct Cut { int parts, length; };

// `groups`: workgroups that are wanted; a part has at least `least` elements, and whole pieces.
Cut cut_of(int64_t rows, int64_t vocab, int64_t groups, int64_t least, int64_t most) {
    int64_t parts = rows > 0 ? groups / rows : 1;
    if (parts > vocab / least) parts = vocab / least;
    if (parts > most) parts = most;
    if (parts < 1) parts = 1;
    const int64_t length = ceil_div(ceil_div(vocab, parts), (int64_t)64) * 64;
    return {(int)ceil_div(vocab, length), (int)length};
}

Cut logprob_cut(int64_t rows, int64_t vocab, int top) {
    return cut_of(rows, vocab, 1024, 4096, top > 0 ? 1024 / top : 256);
}
Cut distill_cut(int64_t rows, int64_t vocab) { return cut_of(rows, vocab, 256, 8192, 256); }

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

template <class T>
int run_logprob(const LogprobParams& p, hipStream_t stream) {
    const int64_t groups = p.r.rows * p.parts;
    if (!grid_fits(groups, kTopThreads)) return set_error(CDX_ERR_UNSUPPORTED, "token_logprobs: too many rows");
    auto go = [&](auto ent, auto top) {
        constexpr bool ENT = decltype(ent)::value, TOP = decltype(top)::value;
        hipLaunchKernelGGL((logprob_kernel<T, ENT, TOP>), dim3((unsigned)groups), dim3(kTopThreads), 0, stream, p);
        int st = hip_error(hipGetLastError(), "logprob_kernel launch");
        if (st || p.parts == 1) return st;
        hipLaunchKernelGGL((logprob_join_kernel<T, ENT, TOP>), dim3((unsigned)p.r.rows), dim3(kTopThreads), 0, stream, p);
        return hip_error(hipGetLastError(), "logprob_join_kernel launch");
    };
    std::true_type yes;
    std::false_type no;
    if (p.entropy) return p.top ? go(yes, yes) : go(yes, no);
    return p.top ? go(no, yes) : go(no, no);
}

}  // namespace

size_t token_logprobs_workspace(int64_t rows, int64_t vocab, int dtype, int top) {
    (void)dtype;
    if (rows == 0) return 0;
    const Cut c = logprob_cut(rows, vocab, top);
    if (c.parts == 1) return 0;
    return round256((size_t)rows * c.parts * sizeof(Part)) + (size_t)rows * c.parts * top * sizeof(u64);
}

int token_logprobs_parts(int64_t rows, int64_t vocab, int dtype, int top) {
    (void)dtype;
    return logprob_cut(rows, vocab, top).parts;
}

int launch_token_logprobs(const TokenLogprobArgs& a, void* ws, hipStream_t stream) {
    const Cut c = logprob_cut(a.r.rows, a.r.vocab, a.top);
    LogprobParams p{a.r, a.targets, a.logprob, a.stats, a.entropy, a.top, a.top_logprob, a.top_index, c.parts,
                    c.length, static_cast<Part*>(ws), nullptr};
    if (c.parts > 1)
        p.keys = reinterpret_cast<u64*>(static_cast<uint8_t*>(ws) + round256((size_t)a.r.rows * c.parts * sizeof(Part)));
    return with_dtype(a.r.dtype, [&](auto t) { return run_logprob<decltype(t)>(p, stream); });
}

int launch_token_logprobs_backward(const LogitRows& r, const int64_t* targets, const RowStats* stats,
                                   const float* g, const float* entropy, const float* gh, void* grad,
                                   int64_t ldg, hipStream_t stream) {
    return with_dtype(r.dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t parts = ceil_div(r.vocab, (int64_t)kBackward<T>);
        if (!grid_fits(r.rows * parts, kBackwardThreads))
            return set_error(CDX_ERR_UNSUPPORTED, "token_logprobs_backward: too many elements");
        hipLaunchKernelGGL(logprob_backward_kernel<T>, dim3((unsigned)(r.rows * parts)), dim3(kBackwardThreads), 0,
                           stream, r, targets, stats, g, entropy, gh, static_cast<T*>(grad), ldg, (int)parts);
        return hip_error(hipGetLastError(), "logprob_backward_kernel launch");
    });
}

size_t distill_workspace(int64_t rows, int64_t vocab, int dtype, int count, bool grad) {
    (void)dtype; (void)grad;
    if (rows == 0) return 0;
    const Cut c = distill_cut(rows, vocab);
    if (c.parts == 1) return 0;
    return round256((size_t)rows * c.parts * sizeof(Part)) + (size_t)rows * count * sizeof(float);
}

int distill_parts(int64_t rows, int64_t vocab, int dtype, bool grad) {
    (void)dtype; (void)grad;
    return distill_cut(rows, vocab).parts;
}

int launch_distill(const DistillArgs& a, void* ws, hipStream_t stream) {
    const Cut c = distill_cut(a.r.rows, a.r.vocab);
    DistillParams p{a, c.parts, c.length, static_cast<Part*>(ws), nullptr};
    const int64_t groups = a.r.rows * c.parts;
    if (!grid_fits(groups, kDistillThreads)) return set_error(CDX_ERR_UNSUPPORTED, "distill_loss: too many rows");
    const dim3 rows((unsigned)a.r.rows), all((unsigned)groups), threads(kDistillThreads);
    if (c.parts > 1)
        p.found = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + round256((size_t)a.r.rows * c.parts * sizeof(Part)));
    return with_dtype(a.r.dtype, [&](auto t) {
        using T = decltype(t);
        if (c.parts == 1) {
            if (a.weight) hipLaunchKernelGGL((distill_kernel<T, true>), rows, threads, 0, stream, p);
            else hipLaunchKernelGGL((distill_kernel<T, false>), rows, threads, 0, stream, p);
            return hip_error(hipGetLastError(), "distill_kernel launch");
        }
        hipLaunchKernelGGL(distill_part_kernel<T>, all, threads, 0, stream, p);
        const int st = hip_error(hipGetLastError(), "distill_part_kernel launch");
        if (st) return st;
        if (a.weight) hipLaunchKernelGGL((distill_join_kernel<T, true>), all, threads, 0, stream, p);
        else hipLaunchKernelGGL((distill_join_kernel<T, false>), rows, threads, 0, stream, p);
        return hip_error(hipGetLastError(), "distill_join_kernel launch");
    });
}

}  // namespace cdx
