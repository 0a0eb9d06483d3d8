// extern "C" entry points of what reads a model's logits (declared in include/cudeep_amd.h).  Every
// argument is checked on the host before any launch, nothing throws, and scratch is the caller's
// workspace or allocated stream-ordered.
#include <cmath>

#include "capi_checks.hpp"
#include "logits.hpp"

using namespace cdx::checks;

namespace {

int check_logits(const char* fn, const void* x, int64_t ldx, int64_t rows, int64_t vocab, int dtype,
                 double temperature) {
    if (bad_dim(rows)) return bad(fn, "rows must be in [0, 2^40]");
    if (vocab < 1 || vocab > cdx::kMaxVocab) return bad(fn, "vocab must be in [1, 2^31 - 2^20]");
    if (!float_dtype(dtype)) return bad(fn, "dtype must be float32, float16 or bfloat16");
    if (!(temperature >= 1e-6 && temperature <= 1e6)) return bad(fn, "temperature must be in [1e-6, 1e6]");
    return check_matrix(fn, "logits", x, ldx, rows, vocab);
}

cdx::LogitRows logit_rows(const void* x, int64_t ldx, int64_t rows, int64_t vocab, int dtype, double temperature) {
    return {x, ldx, rows, vocab, dtype, (float)(1.0 / temperature)};
}

int check_gradient(const char* fn, const void* grad, int64_t ldg, const void* x, int64_t ldx, int64_t rows,
                   int64_t vocab, int dtype) {
    const int st = check_matrix(fn, "grad_logits", grad, ldg, rows, vocab);
    return st ? st : check_in_place(fn, "grad_logits and logits", {grad, ldg, rows, vocab, dtype},
                                    {x, ldx, rows, vocab, dtype});
}

// n values of `words` 4-byte words each as a row (none where p is NULL).
Span words_span(const void* p, int64_t n, int64_t words = 1) {
    return {p, n * words, 1, p ? n * words : 0, CDX_DTYPE_F32};
}

}  // namespace

extern "C" {

size_t cdx_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int top) {
    if (bad_dim(rows) || vocab < 1 || vocab > cdx::kMaxVocab || top < 0 || top > cdx::kMaxTop) return 0;
    return cdx::token_logprobs_workspace(rows, vocab, top);
}

int cdx_token_logprobs(const void* logits, int64_t ldx, int64_t rows, int64_t vocab, int dtype,
                       double temperature, const int64_t* targets, float* logprob, float* stats,
                       float* entropy, int top, float* top_logprob, int64_t* top_index,
                       void* workspace, size_t workspace_bytes, hipStream_t stream) {
    static const char fn[] = "cdx_token_logprobs";
    int st = check_logits(fn, logits, ldx, rows, vocab, dtype, temperature);
    if (!st) st = check_workspace(fn, workspace);
    if (st) return st;
    if (top < 0 || top > cdx::kMaxTop || top > vocab) return bad(fn, "top must be in [0, min(64, vocab)]");
    if (rows == 0) return CDX_OK;
    if (!targets || !logprob || !stats) return bad(fn, "targets, logprob or stats is NULL");
    if (top > 0 && (!top_logprob || !top_index)) return bad(fn, "top_logprob or top_index is NULL");
    const cdx::LogitRows r = logit_rows(logits, ldx, rows, vocab, dtype, temperature);
    st = cdx::token_logprobs_limits(r, top);
    if (st) return st;
    const NamedSpan reads[] = {{"logits", {logits, ldx, rows, vocab, dtype}}, {"targets", words_span(targets, rows, 2)}};
    const NamedSpan writes[] = {{"logprob", words_span(logprob, rows)}, {"stats", words_span(stats, rows, 2)},
                                {"entropy", words_span(entropy, rows)}, {"top_logprob", words_span(top ? top_logprob : nullptr, rows * top)},
                                {"top_index", words_span(top ? top_index : nullptr, rows * top, 2)}};
    st = check_results(fn, writes, reads);
    if (st) return st;
    cdx::TokenLogprobArgs a{r, targets, logprob, stats, entropy, top, top_logprob, top_index};
    return with_workspace(fn, cdx_token_logprobs_workspace_size(rows, vocab, top), workspace, workspace_bytes,
                          stream, [&](void* ws) { return cdx::launch_token_logprobs(a, ws, stream); });
}

int cdx_token_logprobs_backward(const float* grad_logprob, const void* logits, int64_t ldx, int64_t rows,
                                int64_t vocab, int dtype, double temperature, const int64_t* targets,
                                const float* stats, const float* entropy, const float* grad_entropy,
                                void* grad_logits, int64_t ldg, hipStream_t stream) {
    static const char fn[] = "cdx_token_logprobs_backward";
    int st = check_logits(fn, logits, ldx, rows, vocab, dtype, temperature);
    if (!st) st = check_gradient(fn, grad_logits, ldg, logits, ldx, rows, vocab, dtype);
    if (st || rows == 0) return st;
    if (!targets || !stats) return bad(fn, "targets or stats is NULL");
    if (grad_entropy && !entropy) return bad(fn, "grad_entropy needs entropy");
    // (several workgroups of a row read its values while others write theirs)
    const NamedSpan reads[] = {{"targets", words_span(targets, rows, 2)}, {"stats", words_span(stats, rows, 2)},
                               {"grad_logprob", words_span(grad_logprob, rows)},
                               {"entropy", words_span(grad_entropy ? entropy : nullptr, rows)},
                               {"grad_entropy", words_span(grad_entropy, rows)}};
    const NamedSpan writes[] = {{"grad_logits", {grad_logits, ldg, rows, vocab, dtype}}};
    st = check_results(fn, writes, reads);
    if (st) return st;
    return cdx::launch_token_logprobs_backward(logit_rows(logits, ldx, rows, vocab, dtype, temperature), targets,
                                               stats, grad_logprob,
                                               entropy, grad_entropy, grad_logits, ldg, stream);
}

size_t cdx_distill_loss_workspace_size(int64_t rows, int64_t vocab, int count) {
    if (bad_dim(rows) || vocab < 1 || vocab > cdx::kMaxVocab || count < 0 || count > cdx::kMaxEntries) return 0;
    return cdx::distill_workspace(rows, vocab, CDX_DTYPE_F32, count);
}

int cdx_distill_loss(const void* logits, int64_t ldx, int64_t rows, int64_t vocab, int dtype,
                     double temperature, const void* index, int64_t ldi, int index_bytes,
                     const void* teacher, int64_t ldt, int teacher_dtype, int count, float* loss,
                     const float* weight, void* grad_logits, int64_t ldg, void* workspace,
                     size_t workspace_bytes, hipStream_t stream) {
    static const char fn[] = "cdx_distill_loss";
    int st = check_logits(fn, logits, ldx, rows, vocab, dtype, temperature);
    if (!st) st = check_workspace(fn, workspace);
    if (st) return st;
    if (count < 0 || count > cdx::kMaxEntries) return bad(fn, "count must be in [0, 1024]");
    if (index_bytes != 4 && index_bytes != 8) return bad(fn, "index_bytes must be 4 or 8");
    if (!float_dtype(teacher_dtype)) return bad(fn, "teacher_dtype must be float32, float16 or bfloat16");
    st = check_matrix(fn, "index", index, ldi, rows, count);
    if (!st) st = check_matrix(fn, "teacher", teacher, ldt, rows, count);
    if (!st && weight) st = check_gradient(fn, grad_logits, ldg, logits, ldx, rows, vocab, dtype);
    if (st || rows == 0) return st;
    if (!loss) return bad(fn, "loss is NULL");
    const cdx::LogitRows r = logit_rows(logits, ldx, rows, vocab, dtype, temperature);
    st = cdx::distill_limits(r);
    if (st) return st;
    // (a row in parts is read by each of its workgroups, of which some write already)
    const int64_t words = index_bytes / 4;
    const NamedSpan entries[] = {{"index", {index, ldi * words, rows, count * words, CDX_DTYPE_F32}},
                                 {"teacher", {teacher, ldt, rows, count, teacher_dtype}}, {"weight", words_span(weight, rows)}};
    const NamedSpan writes[] = {{"loss", words_span(loss, rows)},
                                {"grad_logits", {grad_logits, ldg, rows, weight ? vocab : 0, dtype}}};
    st = check_results(fn, writes, entries);
    if (!st && overlap(writes[0].at, {logits, ldx, rows, vocab, dtype})) st = bad(fn, "loss and logits overlap");
    if (st) return st;
    cdx::DistillArgs a{r, index, ldi, index_bytes == 8,
                       teacher, ldt, teacher_dtype, count, loss, weight, grad_logits, ldg};
    return with_workspace(fn, cdx_distill_loss_workspace_size(rows, vocab, count), workspace, workspace_bytes,
                          stream, [&](void* ws) { return cdx::launch_distill(a, ws, stream); });
}

}  // extern "C"

// Internal: how many workgroups share a row (op 0: log probabilities with `top` alternatives; 1: distillation).
extern "C" int cdxi_logits_parts(int op, int64_t rows, int64_t vocab, int top) {
    return op ? cdx::distill_parts(rows, vocab, CDX_DTYPE_F32)
              : cdx::token_logprobs_parts(rows, vocab, top);
}

// Internal: what of a gradient of that size passes the caches by (0 nothing, 1 its logits, 2 both).
extern "C" int cdxi_logits_past_caches(int64_t rows, int64_t vocab, int dtype) {
    return cdx::gradient_past_caches(rows, vocab, dtype);
}
