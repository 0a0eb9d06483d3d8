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
    cdx::TokenLogprobArgs a{logit_rows(logits, ldx, rows, vocab, dtype, temperature), targets, logprob,
                            stats, entropy, top, top_logprob, top_index};
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
    cdx::DistillArgs a{logit_rows(logits, ldx, rows, vocab, dtype, temperature), index, ldi, index_bytes == 8,
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
