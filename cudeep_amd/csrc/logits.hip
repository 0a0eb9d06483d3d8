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
//
// Of gradients of 64 MB and more the logits are read for the last time past the caches, and those that the caches
// would not hold until the next product reads them are written past them too (enum Past): what
// those hold of rows that are read again stays there.
#include "logits.hpp"

namespace cdx {
namespace {

using namespace b8;

constexpr float kLog2e = 1.4426950408889634f;      // (as a float; the rest of the number beside it)
constexpr float kLog2eRest = (float)(1.4426950408889634 - (double)kLog2e);
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kFar = -1e20f;       // a difference so large that its exponential is 0 at any temperature, and
                                     // small enough that its products with sums and gradients are finite
constexpr int kUnroll = 4;           // 16-byte pieces of a thread in flight

template <class T> constexpr int kVec = 16 / (int)sizeof(T);

// The sums of some of a row's elements: m their maximum, s = sum e, t = sum e (x - m), e = exp((x - m) / T).
struct Part { float m, s, t; };

// A gradient's exp(y), of logits of T: the hardware's 2^(y log2 e), whose argument is off by up to |y| 2^-24; for fp32,
// whose results hold that, with the rest of the argument's rounding as a factor (exp(-85) is off by 63 2^-24 without
// it, by 8 at most with it).  The sums take the hardware's as it is: a row's roundings mostly cancel, and the constant's own is
// 1.3e-8 of a difference (log probabilities of 1021 x 50001 off by 5.3e-8 of their norm, in single torch operations by
// 6.5e-8; loss and gradient of 513 x 50001 by 1.0e-7 and 7.8e-8; the rest in the sums too would cost 108.7 us for 98.3).
template <class T> __device__ __forceinline__ float exp_of(float y) {
    const float h = y * kLog2e, r = __builtin_amdgcn_exp2f(h);
    if constexpr (!std::is_same_v<T, float>) return r;
    const float rest = __builtin_fmaf(y, kLog2eRest, __builtin_fmaf(y, kLog2e, -h));
    return r > 0.0f ? __builtin_fmaf(r, rest * kLn2, r) : r;   // (y of -infinity has no rest; NaN stays)
}

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

// The join over a workgroup of NT threads, in all of them: the waves' maxima and sums by lane rotations, the
// waves' parts by those of 16 lanes.
template <bool ENT, int NT> __device__ __forceinline__ Part join_all(Part a, float c, Part* red) {
    rescale<ENT>(a, max64(a.m), c);
    a.s = sum64(a.s);
    if constexpr (ENT) a.t = sum64(a.t);
    __syncthreads();   // (the last call's readers are done)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    const int w = threadIdx.x & 15;
    a = w < NT / 64 ? red[w] : Part{kLowest, 0.0f, 0.0f};
    rescale<ENT>(a, max16(a.m), c);
    a.s = sum16(a.s);
    if constexpr (ENT) a.t = sum16(a.t);
    return a;
}

// U pieces of 16 bytes of a thread as loaded: piece i is wanted from element `at` + i NT kVec on.  Where that
// would pass `end`, the row's last kVec elements are loaded instead and the wanted ones of them kept
// (mask), so that all loads are on their way together.
template <class T, int NT, int U> struct Pieces {
    static constexpr int V = kVec<T>, N = U * V, STRIDE = NT * V, ROUND = NT * N;
    u32x4 u[U];
    __device__ __forceinline__ void load(const T* x, int at, int end) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int from = at + i * STRIDE;
            u[i] = load16(x + (from < end - V ? from : end - V));
        }
    }
    __device__ __forceinline__ void get(int i, float (&v)[V]) const {
        T e[V];
        __builtin_memcpy(e, &u[i], 16);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)e[j];
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            float w[V];
            get(i, w);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i * V + j] = w[j];
        }
    }
    // -infinity in the place of the elements of piece i that belong to the piece before, or to none.
    __device__ __forceinline__ static void mask(int i, int at, int end, float (&v)[V]) {
        const int from = at + i * STRIDE, off = from - (end - V);   // the wanted ones begin at `off`
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < off ? -__builtin_inff() : v[j];
    }
    __device__ __forceinline__ static void mask(int at, int end, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            float w[V];
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = v[i * V + j];
            mask(i, at, end, w);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i * V + j] = w[j];
        }
    }
};

// A thread's largest value (-infinity where nothing is larger), the round that it first lies in and that
// round's pieces.
template <class T, int NT> struct Best { float value = -__builtin_inff(); int round = 0; Pieces<T, NT, kUnroll> held; };
struct NoBest {};

// The sums of elements begin .. end - 1, and, with a Best, that.
template <class T, int NT, bool ENT, class B>
__device__ __forceinline__ Part scan(const T* x, int begin, int end, float c, B& best) {
    using P = Pieces<T, NT, kUnroll>;
    Part a{kLowest, 0.0f, 0.0f};
    float v[P::N];
    P now, next;
    auto use = [&](int r) {
        const float most = take<ENT>(a, v, c);
        if constexpr (!std::is_same_v<B, NoBest>) {
            if (r == 0) best.held = now;
            if (most > best.value) {   // (seldom after the first rounds)
                best.value = most;
                best.round = r;
                best.held = now;
            }
        }
    };
    if (end - begin < P::V) {   // (less than one piece)
#pragma unroll
        for (int j = 0; j < P::N; ++j) {
            const int i = begin + j;
            v[j] = threadIdx.x == 0 && j < P::V && i < end ? (float)x[i] : -__builtin_inff();
        }
        take<ENT>(a, v, c);
        return a;
    }
    const int rounds = (end - begin + P::ROUND - 1) / P::ROUND, at = begin + (int)threadIdx.x * P::V;
    now.load(x, at, end);
    for (int r = 0; r + 1 < rounds; ++r) {
        next.load(x, at + (r + 1) * P::ROUND, end);
        now.get(v);
        use(r);
        now = next;
    }
    now.get(v);
    P::mask(at + (rounds - 1) * P::ROUND, end, v);
    use(rounds - 1);
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

constexpr int kGroups = 256;             // groups of neighbouring threads whose largest element is known, at most
constexpr int kSpare = 512;              // keys kept from one round of pieces to the next, at most

template <int NT> struct TopShared {
    static constexpr int ROUND = NT * 8, MOST = ROUND + kSpare;   // keys of one round of pieces, at most
    alignas(16) u64 keys[MOST];
    alignas(16) u64 best[kGroups];
    u64 threshold;
    int count, who[kMaxTop];
};

// How many of `count` keys (from a 16-byte address on) are larger.
__device__ __forceinline__ int larger_ones(const u64* keys, int count, u64 key) {
    typedef u64 u64x2 __attribute__((ext_vector_type(2)));
    int n = 0, j = 0;
#pragma unroll 1
    for (; j + 16 <= count; j += 16) {   // (eight reads on their way together)
        u64x2 k[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = *reinterpret_cast<const u64x2*>(keys + j + 2 * i);
#pragma unroll
        for (int i = 0; i < 8; ++i) n += (k[i][0] > key) + (k[i][1] > key);
    }
#pragma unroll 4
    for (; j < count; ++j) n += keys[j] > key;
    return n;
}

// Leaves the `k` largest of the first `count` keys, at most MOST, in their order at the front (all NT threads
// call it).  A key's place is the number of larger ones; keys differ, so that places do.
template <int NT, int MOST> __device__ __forceinline__ int keep_largest(u64* keys, int count, int k) {
    constexpr int EACH = (MOST + NT - 1) / NT;
    u64 mine[EACH];
    int place[EACH];
#pragma unroll
    for (int s = 0; s < EACH; ++s) {
        const int i = threadIdx.x + s * NT;
        place[s] = k;
        if (i < count) {
            mine[s] = keys[i];
            place[s] = larger_ones(keys, count, mine[s]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < EACH; ++s)
        if (place[s] < k) keys[place[s]] = mine[s];
    __syncthreads();
    return count < k ? count : k;
}

// The k largest of elements begin .. end - 1 at the front of sh.keys; how many there are.  Each group's
// largest element is known (`best`: the scan's); the k-th largest of those is a bound that the k
// largest elements of all reach, and they lie with the k groups whose own reach it: only those
// groups' elements are looked at again.
template <class T, int NT>
__device__ __forceinline__ int largest(const T* x, int begin, int end, int k, const Best<T, NT>& best, TopShared<NT>& sh) {
    using P = Pieces<T, NT, kUnroll>;
    using S = TopShared<NT>;
    constexpr int V = P::V;
    const int tid = threadIdx.x;
    const int pieces = (end - begin + P::STRIDE - 1) / P::STRIDE;   // of a thread
    // threads of a group: more for short rows and few wanted, where comparing the groups costs more than
    // looking at more elements (8192 rows of 4000, 5 of each: 256 groups 71 us, as below 41)
    int G = NT / kGroups;
    while (NT / G > 64 && NT / G >= 4 * k && (int64_t)k * pieces * 2 * G <= NT) G *= 2;
    u64 mine = 0;
    const int at = begin + tid * V + best.round * P::ROUND;
    if (end - begin < V) {
        for (int i = begin; tid == 0 && i < end; ++i) {
            const u64 key = key_of((float)x[i], i);
            mine = key > mine ? key : mine;
        }
    } else if (at < end) {
        // the first element of its round with that value (NaN alone: the first there is)
#pragma unroll
        for (int i = kUnroll - 1; i >= 0; --i) {
            const int from = at + i * P::STRIDE, first = from < end - V ? from : end - V;
            float v[V];
            best.held.get(i, v);
#pragma unroll
            for (int j = V - 1; j >= 0; --j)
                if (first + j >= from && v[j] == best.value) mine = key_of(v[j], first + j);
        }
        if (mine == 0) mine = key_of(__builtin_nanf(""), at);
    }
    for (int g = 1; g < G; g *= 2) {
        const u64 other = __shfl_xor(mine, g);
        mine = other > mine ? other : mine;
    }
    const int part = tid & (G - 1), groups = NT / G;
    if (part == 0) sh.best[tid / G] = mine;
    if (tid < kMaxTop) sh.who[tid] = -1;
    if (tid == 0) sh.count = 0, sh.threshold = 0;
    __syncthreads();
    // a group's place among them, each of its threads with a part of the comparisons
    int place = larger_ones(sh.best + part * (groups / G), groups / G, mine);
    for (int g = 1; g < G; g *= 2) place += __shfl_xor(place, g);
    if (part == 0 && mine && place < k) {
        sh.who[place] = tid;
        if (place == k - 1) sh.threshold = mine;
    }
    __syncthreads();
    u64 threshold = sh.threshold;   // (0 where fewer than k groups have elements)
    const int64_t items = (int64_t)k * pieces * G;
    for (int64_t first = 0; first < items; first += NT) {
        if (first > 0) {
            const int count = sh.count;
            __syncthreads();   // everybody has read the count
            if (count > kSpare) {
                const int left = keep_largest<NT, S::MOST>(sh.keys, count, k);
                if (left == k) threshold = sh.keys[k - 1] > threshold ? sh.keys[k - 1] : threshold;
                if (tid == 0) sh.count = left;
                __syncthreads();
            }
        }
        const int64_t i = first + tid;
        if (i < items) {
            const int q = (int)(i / G), who = sh.who[q / pieces];
            const int from = begin + q % pieces * P::STRIDE + (who + (int)(i & (G - 1))) * V, n = who < 0 ? 0 : end - from;
            if (n > 0) {
                float v[V];
                load_n<V>(x + from, n, v);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const u64 key = key_of(v[j], from + j);
                    if (j < n && key >= threshold) {
                        const int slot = atomicAdd(&sh.count, 1);
                        if (slot < S::MOST) sh.keys[slot] = key;
                    }
                }
            }
        }
        __syncthreads();
    }
    return keep_largest<NT, S::MOST>(sh.keys, sh.count < S::MOST ? sh.count : S::MOST, k);
}

// ---- log probabilities --------------------------------------------------------------------------

struct LogprobParams {
    LogitRows r;
    const int64_t* targets;
    float* logprob; float* stats; float* entropy;
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
    p.stats[row] = s.m;
    p.stats[p.r.rows + row] = s.l;
    if (p.entropy) p.entropy[row] = entropy_of(a, s.l, p.r.inv_t);
}

// A workgroup a row, or a part of one: the row is read once, with the next round's loads on their way, and
// memory bounds long batches (1021 x 50001 in fp32, with entropies, 37.3 us, 5.5 TB/s; 2048 x 131072 in
// bf16 with entropies and 8 alternatives 111.6, 4.8 TB/s).  A single row of 32000 in fp32 with 5 alternatives
// takes 8.0 us, most of them the chain of the alternatives.
template <class T, int NT, bool ENT, bool TOP>
__global__ __launch_bounds__(NT)
void logprob_kernel(LogprobParams p) {
    __shared__ Part red[NT / 64];
    __shared__ std::conditional_t<TOP, TopShared<NT>, char> sh;
    const int64_t row = blockIdx.x / p.parts;
    const int part = (int)(blockIdx.x % p.parts);
    const T* x = static_cast<const T*>(p.r.x) + row * p.r.ldx;
    const int begin = part * p.length;
    const int end = p.r.vocab - begin < p.length ? (int)p.r.vocab : begin + p.length;
    const float c = p.r.inv_t * kLog2e;
    std::conditional_t<TOP, Best<T, NT>, NoBest> best;
    Part a = scan<T, NT, ENT>(x, begin, end, c, best);
    a = join_all<ENT, NT>(a, c, red);
    if (p.parts > 1) {
        if (threadIdx.x == 0) p.part[row * p.parts + part] = a;
        if constexpr (TOP) {
            const int n = largest<T, NT>(x, begin, end, p.top, best, sh);
            if ((int)threadIdx.x < p.top)
                p.keys[(row * p.parts + part) * p.top + threadIdx.x] = (int)threadIdx.x < n ? sh.keys[threadIdx.x] : 0;
        }
        return;
    }
    const RowStats s{a.m, logf(a.s)};
    if (threadIdx.x == 0) finish_row<T>(p, row, a, s);
    if constexpr (TOP) {
        largest<T, NT>(x, begin, end, p.top, best, sh);
        if ((int)threadIdx.x < p.top) {
            const u64 key = sh.keys[threadIdx.x];
            p.top_logprob[row * p.top + threadIdx.x] = log_softmax(key_value(key), s, p.r.inv_t);
            p.top_index[row * p.top + threadIdx.x] = key_index(key);
        }
    }
}

constexpr int kJoinThreads = 256, kJoinKeys = 1024;   // (logprob_plan: parts * top is no more)

// A row's parts together.
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(kJoinThreads)
void logprob_join_kernel(LogprobParams p) {
    __shared__ Part red[kJoinThreads / 64];
    __shared__ __attribute__((aligned(16))) u64 keys[TOP ? kJoinKeys : 1];
    const int64_t row = blockIdx.x;
    const float c = p.r.inv_t * kLog2e;
    Part a{kLowest, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < p.parts; i += kJoinThreads) a = join<ENT>(a, p.part[row * p.parts + i], c);
    a = join_all<ENT, kJoinThreads>(a, c, red);
    const RowStats s{a.m, logf(a.s)};
    if (threadIdx.x == 0) finish_row<T>(p, row, a, s);
    if constexpr (TOP) {
        const int count = p.parts * p.top;
        for (int i = threadIdx.x; i < count; i += kJoinThreads) keys[i] = p.keys[row * count + i];
        __syncthreads();
        // (parts of fewer elements than `top` leave zeros, which are below every key)
        for (int i = threadIdx.x; i < count; i += kJoinThreads)
            if (keys[i] == 0) keys[i] = i;   // small, and all different
        __syncthreads();
        keep_largest<kJoinThreads, kJoinKeys>(keys, count, p.top);
        if ((int)threadIdx.x < p.top) {
            const u64 key = keys[threadIdx.x];
            p.top_logprob[row * p.top + threadIdx.x] = log_softmax(key_value(key), s, p.r.inv_t);
            p.top_index[row * p.top + threadIdx.x] = key_index(key);
        }
    }
}

// The gradient, element by element: a workgroup takes kBackward elements of a row.  Memory bounds it, 1021 x
// 50001 in fp32 61.9 us, 6.6 TB/s read and written (62.1 with the rows in reverse, which begins with those
// that were read last).
// What of a gradient passes the caches: nothing; its logits, read for the last time; both.  Measured with what reads
// the gradient next, a bf16 product of 50304 or 32000 logits with 1024 columns, us, nothing / logits / both:
//   bf16   48 MB 229.9 226.4 226.5 (in place 226.6 226.2 227.6)    64 MB 280.7 274.7 277.8 (270.5 270.2 272.4)
//         100 MB 448.8 440.5 478.6 (432.9 443.6 463.5)            160 MB 590.0 576.3 572.7 (554.1 570.0 572.3)
//         200 MB 766.4 759.8 750.0 (712.3 734.1 744.7)            400 MB 1422 1428 1398 (1416 1423 1400)
//   fp32, rounded to bf16 in between
//          63 MB 282.0 279.4 280.5 (277.7 279.5 276.3)            100 MB 353.2 348.4 355.0 (347.4 350.3 349.3)
//         129 MB 437.7 429.2 423.9 (424.8 426.7 423.2)            259 MB 793.6 789.9 763.2 (775.3 784.5 754.4)
// So both for fp32 from 64 MB on and for 16 bits from 200 MB on; below that, from 64 MB on, the logits alone (by itself, loss and gradient of 100 MB in bf16 57.5 54.5 52.2, of 513 x 50001 in fp32 66.1 with
// nothing, 48.8 with both).
enum class Past { None, Logits, Both };
Past gradient_past(const LogitRows& r) {
    if (!past_caches(r.rows, r.vocab, r.dtype)) return Past::None;
    return r.dtype == CDX_DTYPE_F32 || (double)r.rows * (double)r.vocab * 2 >= 200e6 ? Past::Both : Past::Logits;
}
// Calls f with it as a constant (Logits alone: 16 bits).
template <class T, class F> void with_past(Past past, F f) {
    using std::integral_constant;
    if (past == Past::Both) return f(integral_constant<Past, Past::Both>{});
    if constexpr (sizeof(T) == 2)
        if (past == Past::Logits) return f(integral_constant<Past, Past::Logits>{});
    f(integral_constant<Past, Past::None>{});
}

constexpr int kBackwardThreads = 256;
template <class T> constexpr int kBackward = kBackwardThreads * kUnroll * kVec<T>;

template <class T, Past PAST>
__global__ __launch_bounds__(kBackwardThreads)
void logprob_backward_kernel(LogitRows r, const int64_t* __restrict__ targets, const float* __restrict__ stats,
                             const float* __restrict__ g_lp, const float* __restrict__ entropy,
                             const float* __restrict__ g_h, T* grad, int64_t ldg, int parts) {
    constexpr int V = kVec<T>;
    const int64_t row = blockIdx.x / parts;
    const int64_t first = (int64_t)(blockIdx.x % parts) * kBackward<T>;
    const T* x = static_cast<const T*>(r.x) + row * r.ldx;
    T* out = grad + row * ldg;
    const RowStats s{stats[row], stats[r.rows + row]};
    const int64_t t = targets[row];
    float g = g_lp ? g_lp[row] : 0.0f;
    if (t < 0) g = 0.0f;
    if (t >= r.vocab && g != 0.0f) g = __builtin_nanf("");
    const float h = g_h ? g_h[row] : 0.0f;
    // -g p - h p (l + H) = -p (h l + (h H + g))
    const float hs = h * r.inv_t, gs = g * r.inv_t, both = h != 0.0f ? (h * entropy[row] + g) * r.inv_t : gs;
    const bool none = (g == 0.0f && h == 0.0f) || s.l == -__builtin_inff();
    auto gradient = [&](float (&v)[V], int64_t at) {
        if (none) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = 0.0f;
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float l = (v[j] - s.m) * r.inv_t - s.l, p = exp_of<T>(l);
            v[j] = -p * (hs * fmaxf(l, kFar) + both);
        }
        if (t >= at && t < at + V) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (t == at + j) v[j] += gs;
        }
    };
    const int64_t at0 = first + (int64_t)threadIdx.x * V;
    constexpr int64_t STRIDE = (int64_t)kBackwardThreads * V;
    if (at0 + (kUnroll - 1) * STRIDE + V <= r.vocab) {
        u32x4 u[kUnroll];
        if (!none) {   // (a row without a gradient is not read)
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) u[i] = load16_as<PAST != Past::None>(x + at0 + i * STRIDE);
        }
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            T e[V];
            float v[V];
            __builtin_memcpy(e, &u[i], 16);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (float)e[j];
            gradient(v, at0 + i * STRIDE);
            store16_as<PAST == Past::Both, T>(out + at0 + i * STRIDE, v);
        }
        return;
    }
    for (int64_t at = at0; at < r.vocab && at < first + kBackward<T>; at += STRIDE) {
        const int n = r.vocab - at < V ? (int)(r.vocab - at) : V;
        float v[V] = {};
        if (!none) load_n<V>(x + at, n, v);
        gradient(v, at);
        store_n<V>(out + at, n, v);
    }
}

// ---- distillation ---------------------------------------------------------------------------------

constexpr int kDistillThreads = 512;   // of a row's parts

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

// What a row's gradient needs: 0 everywhere (none), else f (exp(l) - q).
struct GradRow { RowStats s; float f, inv_t; bool none; };

__device__ __forceinline__ GradRow grad_row(const DistillArgs& a, int64_t row, RowStats s, bool some, float loss) {
    const float w = a.weight[row];
    // (an index past the vocabulary shows in every element)
    return {s, loss != loss ? loss : w * a.r.inv_t, a.r.inv_t, !some || w == 0.0f || s.l == -__builtin_inff()};
}

template <class T, int V> __device__ __forceinline__ void grad_values(const GradRow& g, float (&v)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        v[j] = g.none ? 0.0f : g.f * exp_of<T>((v[j] - g.s.m) * g.inv_t - g.s.l);
}

// Once the rest of the row is written, its entries that lie in begin .. end - 1, once more.
template <class T, int NT>
__device__ __forceinline__ void grad_entries(const DistillArgs& a, T* out, int begin, int end, const GradRow& g, const Entries& e) {
    if (g.none) return;
    __syncthreads();
    for (int k = threadIdx.x; k < a.count; k += NT) {
        const int i = e.index[k];
        if (i < begin || i >= end) continue;
        float q = 0.0f;   // of all entries of this index: each of them stores the same
        for (int j = 0; j < a.count; ++j) q += e.index[j] == i ? e.q[j] : 0.0f;
        out[i] = (T)(g.f * (exp_of<T>((e.x[k] - g.s.m) * g.inv_t - g.s.l) - q));
    }
}

// The gradient of elements begin .. end - 1, which are read again; all threads call it, with the row's entries
// in LDS.
template <class T, int NT, Past PAST>
__device__ __forceinline__ void distill_grad(const DistillArgs& a, int64_t row, int begin, int end, const GradRow& g, const Entries& e) {
    constexpr int V = kVec<T>, U = kUnroll;
    const T* x = static_cast<const T*>(a.r.x) + row * a.r.ldx;
    T* out = static_cast<T*>(a.grad) + row * a.ldg;
    int at = begin + (int)threadIdx.x * V;
    for (; at + ((U - 1) * NT + 1) * V <= end; at += U * NT * V) {
        u32x4 u[U];
#pragma unroll
        for (int i = 0; i < U; ++i) u[i] = load16_as<PAST != Past::None>(x + at + i * NT * V);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            T t[V];
            float v[V];
            __builtin_memcpy(t, &u[i], 16);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (float)t[j];
            grad_values<T>(g, v);
            store16_as<PAST == Past::Both, T>(out + at + i * NT * V, v);
        }
    }
    for (; at < end; at += NT * V) {
        const int n = end - at;
        float v[V] = {};
        if (!g.none) load_n<V>(x + at, n, v);
        grad_values<T>(g, v);
        store_n<V>(out + at, n, v);
    }
    grad_entries<T, NT>(a, out, begin, end, g, e);
}

// The indices of a row's entries, and the logits there.
template <class T, int NT>
__device__ __forceinline__ void load_entries(const DistillArgs& a, int64_t row, const T* x, Entries& e) {
    for (int k = threadIdx.x; k < a.count; k += NT) {
        const int i = entry_index(a, row, k);
        e.index[k] = i;
        e.x[k] = i >= 0 && i < a.r.vocab ? (float)x[i] : 0.0f;
    }
}

// A workgroup a row: sums, entries, and the gradient, for which the row is read again.  Memory bounds it:
// 4096 x 65536 in bf16 with 64 entries 232 us, in which 0.86 GB are read (0.54 are the logits) and 0.54
// written.  Rows kept in registers for the second reading do not fit (spills, 875 us against 247).
template <class T, int NT, bool GRAD, Past PAST>
__global__ __launch_bounds__(NT)
void distill_kernel(DistillArgs a) {
    __shared__ Part red[NT / 64];
    __shared__ float redf[NT / 64];
    __shared__ Entries e;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.r.x) + row * a.r.ldx;
    const float c = a.r.inv_t * kLog2e;
    load_entries<T, NT>(a, row, x, e);
    NoBest none;
    Part s = scan<T, NT, false>(x, 0, (int)a.r.vocab, c, none);
    s = join_all<false, NT>(s, c, red);
    const RowStats st{s.m, logf(s.s)};
    float loss;
    const bool some = entries_loss<NT>(a, row, st, e, redf, loss);
    if (threadIdx.x == 0) a.loss[row] = loss;
    if constexpr (GRAD) {
        __syncthreads();
        distill_grad<T, NT, PAST>(a, row, 0, (int)a.r.vocab, grad_row(a, row, st, some, loss), e);
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
    NoBest none;
    Part s = scan<T, NT, false>(x, begin, end, c, none);
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
        distill_grad<T, NT, Past::None>(a, row, begin, end, grad_row(a, row, st, some, loss), e);
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

struct LogprobPlan { Cut cut; int threads; };

int64_t row_bytes(int64_t vocab, int dtype) { return vocab * (dtype == CDX_DTYPE_F32 ? 4 : 2); }

// Few long rows are cut, which a second launch joins (1 x 131072 with 5 alternatives, bf16, in 8 parts 11.6 us,
// whole 16.5; 16 x 131072 6.2, whole 10.9; 1 x 65536 11.1 in 4, whole 11.5; 128 x 131072 17.6, whole 18.0).
// Threads of a row: 512 while a CU has one row (1 x 65536 with 5 alternatives 11.5 us, 256 threads 16.0; 128
// x 131072 18.0, 256 threads 20.8), else 256 (300 x 50001 10.7, 512 threads 12.7; 8192 x 4096 with 5
// alternatives 55, 512 threads 123), and 1024 where rows are long and only their sums wanted (1024 x 50001 in
// fp32 37.4, 256 threads 39.0; 1024 x 131072 55, 256 threads 57; but 600 x 64000 19.1, 256 threads 17.6).
// Parts do not depend on the type, which the workspace's query does not have.
LogprobPlan logprob_plan(int64_t rows, int64_t vocab, int top, int dtype) {
    Cut c{1, (int)vocab};
    if (rows < 128 && vocab > 65536) c = cut_of(rows, vocab, 512, 16384, top > 0 ? kJoinKeys / top : 256);
    if (rows < 256) return {c, 512};
    return {c, top == 0 && row_bytes(vocab, dtype) >= 150000 ? 1024 : 256};
}
struct DistillPlan { Cut cut; int threads; };

// The same with the gradient: parts from 65536 on (64 x 65536 with 64 entries, bf16, in 4 parts 14.0 us, whole
// 17.5; 64 x 131072 in 8 17.1, whole 25.4; 1 x 50001 in 4 13.4, whole 14.9, and without a gradient 16 x 32000
// in 2 8.0, whole 5.5).  Threads: a row that is read again should be in the caches still, and fewer rows are in
// flight with more threads each, but the entries cost them the same: 256 for rows of less than 48 KB (4096 x
// 8192, bf16, 31.9 us, 512 threads 51.9), 1024 from 128 KB on (513 x 50001 in fp32 50.9, 256 threads 54.2;
// 2048 x 64000, bf16, 117, 512 threads 120).
DistillPlan distill_plan(int64_t rows, int64_t vocab, int dtype) {
    if (rows < 128 && vocab >= 65536) return {cut_of(rows, vocab, 512, 16384, 256), kDistillThreads};
    const int64_t bytes = row_bytes(vocab, dtype);
    return {{1, (int)vocab}, rows < 512 ? 512 : bytes >= 128000 ? 1024 : bytes >= 48000 ? 512 : 256};
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

template <class T>
int run_logprob(const LogprobParams& p, int threads, hipStream_t stream) {
    const int64_t groups = p.r.rows * p.parts;
    auto go = [&](auto ent, auto top) {
        constexpr bool ENT = decltype(ent)::value, TOP = decltype(top)::value;
        auto run = [&](auto nt) {
            constexpr int NT = decltype(nt)::value;
            hipLaunchKernelGGL((logprob_kernel<T, NT, ENT, TOP>), dim3((unsigned)groups), dim3(NT), 0, stream, p);
        };
        constexpr int MOST = TOP ? 512 : 1024;   // (logprob_plan)
        if (threads == 256) run(std::integral_constant<int, 256>{});
        else if (threads == 512) run(std::integral_constant<int, 512>{});
        else run(std::integral_constant<int, MOST>{});
        int st = hip_error(hipGetLastError(), "logprob_kernel launch");
        if (st || p.parts == 1) return st;
        hipLaunchKernelGGL((logprob_join_kernel<T, ENT, TOP>), dim3((unsigned)p.r.rows), dim3(kJoinThreads), 0, stream, p);
        return hip_error(hipGetLastError(), "logprob_join_kernel launch");
    };
    std::true_type yes;
    std::false_type no;
    if (p.entropy) return p.top ? go(yes, yes) : go(yes, no);
    return p.top ? go(no, yes) : go(no, no);
}

template <class T>
int run_distill(const DistillParams& p, const DistillPlan& pl, hipStream_t stream) {
    const DistillArgs& a = p.a;
    const dim3 rows((unsigned)a.r.rows), all((unsigned)(a.r.rows * p.parts)), threads(kDistillThreads);
    if (p.parts == 1) {
        auto kind = [&](auto threads) {
            constexpr int NT = decltype(threads)::value;
            if (!a.weight) {
                hipLaunchKernelGGL((distill_kernel<T, NT, false, Past::None>), rows, dim3(NT), 0, stream, a);
                return;
            }
            with_past<T>(gradient_past(a.r), [&](auto past) {
                hipLaunchKernelGGL((distill_kernel<T, NT, true, decltype(past)::value>), rows, dim3(NT), 0, stream, a);
            });
        };
        if (pl.threads == 1024) kind(std::integral_constant<int, 1024>{});
        else if (pl.threads == 512) kind(std::integral_constant<int, 512>{});
        else kind(std::integral_constant<int, 256>{});
        return hip_error(hipGetLastError(), "distill_kernel launch");
    }
    hipLaunchKernelGGL(distill_part_kernel<T>, all, threads, 0, stream, p);
    const int st = hip_error(hipGetLastError(), "distill_part_kernel launch");
    if (st) return st;
    if (a.weight) hipLaunchKernelGGL((distill_join_kernel<T, true>), all, threads, 0, stream, p);
    else hipLaunchKernelGGL((distill_join_kernel<T, false>), rows, threads, 0, stream, p);
    return hip_error(hipGetLastError(), "distill_join_kernel launch");
}

int launch_distill_plan(const DistillArgs& a, const DistillPlan& pl, void* ws, hipStream_t stream) {
    DistillParams p{a, pl.cut.parts, pl.cut.length, static_cast<Part*>(ws), nullptr};
    if (p.parts > 1)
        p.found = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + round256((size_t)a.r.rows * p.parts * sizeof(Part)));
    return with_dtype(a.r.dtype, [&](auto t) { return run_distill<decltype(t)>(p, pl, stream); });
}

int launch_logprob_plan(const TokenLogprobArgs& a, const LogprobPlan& pl, void* ws, hipStream_t stream) {
    LogprobParams p{a.r, a.targets, a.logprob, a.stats, a.entropy, a.top, a.top_logprob, a.top_index, pl.cut.parts,
                    pl.cut.length, static_cast<Part*>(ws), nullptr};
    if (pl.cut.parts > 1)
        p.keys = reinterpret_cast<u64*>(static_cast<uint8_t*>(ws) + round256((size_t)a.r.rows * pl.cut.parts * sizeof(Part)));
    return with_dtype(a.r.dtype, [&](auto t) { return run_logprob<decltype(t)>(p, pl.threads, stream); });
}

}  // namespace

size_t token_logprobs_workspace(int64_t rows, int64_t vocab, int top) {
    if (rows == 0) return 0;
    const Cut c = logprob_plan(rows, vocab, top, CDX_DTYPE_F32).cut;
    if (c.parts == 1) return 0;
    return round256((size_t)rows * c.parts * sizeof(Part)) + (size_t)rows * c.parts * top * sizeof(u64);
}

int token_logprobs_parts(int64_t rows, int64_t vocab, int top) {
    return logprob_plan(rows, vocab, top, CDX_DTYPE_F32).cut.parts;
}

int token_logprobs_limits(const LogitRows& r, int top) {
    const LogprobPlan pl = logprob_plan(r.rows, r.vocab, top, r.dtype);
    if (grid_fits(r.rows * pl.cut.parts, pl.threads)) return CDX_OK;
    return set_error(CDX_ERR_UNSUPPORTED, "token_logprobs: too many rows");
}

int distill_limits(const LogitRows& r) {
    const DistillPlan pl = distill_plan(r.rows, r.vocab, r.dtype);
    if (grid_fits(r.rows * pl.cut.parts, pl.threads)) return CDX_OK;
    return set_error(CDX_ERR_UNSUPPORTED, "distill_loss: too many rows");
}

int launch_token_logprobs(const TokenLogprobArgs& a, void* ws, hipStream_t stream) {
    return launch_logprob_plan(a, logprob_plan(a.r.rows, a.r.vocab, a.top, a.r.dtype), ws, stream);
}

int launch_token_logprobs_backward(const LogitRows& r, const int64_t* targets, const float* stats,
                                   const float* g, const float* entropy, const float* gh, void* grad,
                                   int64_t ldg, hipStream_t stream) {
    return with_dtype(r.dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t parts = ceil_div(r.vocab, (int64_t)kBackward<T>);
        if (!grid_fits(r.rows * parts, kBackwardThreads))
            return set_error(CDX_ERR_UNSUPPORTED, "token_logprobs_backward: too many elements");
        const dim3 grid((unsigned)(r.rows * parts)), threads(kBackwardThreads);
        with_past<T>(gradient_past(r), [&](auto past) {
            hipLaunchKernelGGL((logprob_backward_kernel<T, decltype(past)::value>), grid, threads, 0, stream, r, targets,
                               stats, g, entropy, gh, static_cast<T*>(grad), ldg, (int)parts);
        });
        return hip_error(hipGetLastError(), "logprob_backward_kernel launch");
    });
}

size_t distill_workspace(int64_t rows, int64_t vocab, int dtype, int count) {
    if (rows == 0) return 0;
    const Cut c = distill_plan(rows, vocab, dtype).cut;
    if (c.parts == 1) return 0;
    return round256((size_t)rows * c.parts * sizeof(Part)) + (size_t)rows * count * sizeof(float);
}

int distill_parts(int64_t rows, int64_t vocab, int dtype) {
    return distill_plan(rows, vocab, dtype).cut.parts;
}

int gradient_past_caches(int64_t rows, int64_t vocab, int dtype) {
    return (int)gradient_past({nullptr, vocab, rows, vocab, dtype, 1.0f});
}

int launch_distill(const DistillArgs& a, void* ws, hipStream_t stream) {
    return launch_distill_plan(a, distill_plan(a.r.rows, a.r.vocab, a.r.dtype), ws, stream);
}

}  // namespace cdx
