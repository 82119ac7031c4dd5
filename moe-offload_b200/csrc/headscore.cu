// Log-probabilities of given tokens, entropy and alternatives straight from hidden rows [T, H] and
// the LM head [V, H] (prompt scoring): the values of moe_lm_head_logits followed by
// moe_token_logprobs, four rows at a time through a [4, V] scratch.
#include "common.cuh"
#include "internal.h"

namespace {
constexpr int kRows = 4;               // rows per pass of the LM head
}

extern "C" size_t moe_head_logprobs_workspace_bytes(int T, int V, int n) {
    if (T <= 0 || V <= 0 || n < 0) return 0;
    return (size_t)(T < kRows ? T : kRows) * V * sizeof(float);
}

extern "C" int moe_head_logprobs(const void *head, int V, int H, const void *x, int T, const int32_t *targets, int n,
                                 float *logprob, float *entropy, int32_t *top_ids, float *top_logprobs,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = moe_logprobs_check("head logprobs", T, V, targets, n, logprob, entropy, top_ids, top_logprobs))
        return rc;
    if (!head || !x || H <= 0 || H % 8 || H > 8192)
        return moe_set_error(MOE_EINVAL, "head logprobs: head and x must be set, H=%d a multiple of 8 up to 8192", H);
    if ((reinterpret_cast<uintptr_t>(head) | reinterpret_cast<uintptr_t>(x)) & 15)
        return moe_set_error(MOE_EINVAL, "head logprobs: head and x must be 16-byte aligned");
    if (!workspace || workspace_bytes < moe_head_logprobs_workspace_bytes(T, V, n) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15))
        return moe_set_error(MOE_EINVAL, "head logprobs: a 16-byte aligned workspace of %zu bytes is needed",
                             moe_head_logprobs_workspace_bytes(T, V, n));
    float *logits = static_cast<float *>(workspace);
    const char *rows = static_cast<const char *>(x);
    for (int t = 0; t < T; t += kRows) {
        const int m = T - t < kRows ? T - t : kRows;
        int rc = moe_lm_head_logits(head, V, H, rows + (size_t)t * H * 2, m, logits, stream);
        if (rc != MOE_OK) return rc;
        rc = moe_token_logprobs_launch(logits, m, V, targets ? targets + t : nullptr, n, logprob ? logprob + t : nullptr,
                                       entropy + t, n ? top_ids + (size_t)t * n : nullptr,
                                       n ? top_logprobs + (size_t)t * n : nullptr, stream);
        if (rc != MOE_OK) return rc;
    }
    return MOE_OK;
}
