// What reads a model's logits (logits.hip): log probabilities of given tokens with entropy and the
// likeliest alternatives, and distillation from a teacher's top logits.
#pragma once

#include "block8.hpp"

namespace cdx {

constexpr int kMaxTop = 64;            // alternatives of a row
constexpr int kMaxEntries = 1024;      // a teacher's entries of a row
constexpr int64_t kMaxVocab = ((int64_t)1 << 31) - ((int64_t)1 << 20);

struct LogitRows {
    const void* x; int64_t ldx;
    int64_t rows, vocab;
    int dtype;                         // CDX_DTYPE_F32, _F16 or _BF16
    float inv_t;                       // 1 / temperature
};

// The largest logit m of a row and L = log sum exp((x - m) / T): log softmax = (x - m) / T - L.
struct RowStats { float m, l; };

struct TokenLogprobArgs {
    LogitRows r;
    const int64_t* targets;
    float* logprob; float* stats;        // stats: m of all rows, then L
    float* entropy;                    // may be null
    int top; float* top_logprob; int64_t* top_index;
};
size_t token_logprobs_workspace(int64_t rows, int64_t vocab, int top);
int launch_token_logprobs(const TokenLogprobArgs& a, void* ws, hipStream_t stream);

// grad: may be the logits' own place.  g (null: none): the log probabilities' gradients; gh (null: none):
// the entropies'.
int launch_token_logprobs_backward(const LogitRows& r, const int64_t* targets, const float* stats,
                                   const float* g, const float* entropy, const float* gh, void* grad,
                                   int64_t ldg, hipStream_t stream);

struct DistillArgs {
    LogitRows r;
    const void* index; int64_t ldi; int index64;
    const void* teacher; int64_t ldt; int teacher_dtype;
    int count;
    float* loss;
    const float* weight;               // null: no gradient
    void* grad; int64_t ldg;
};
size_t distill_workspace(int64_t rows, int64_t vocab, int dtype, int count);
int launch_distill(const DistillArgs& a, void* ws, hipStream_t stream);

// Whether a launch holds that many rows (the entry points ask before they launch).
int token_logprobs_limits(const LogitRows& r, int top);
int distill_limits(const LogitRows& r);

// How many workgroups share a row (for tests that aim at one way or the other).
int token_logprobs_parts(int64_t rows, int64_t vocab, int top);
int distill_parts(int64_t rows, int64_t vocab, int dtype);
// What of a gradient passes the caches by: 0 nothing, 1 its logits, 2 both.
int gradient_past_caches(int64_t rows, int64_t vocab, int dtype);

}  // namespace cdx
