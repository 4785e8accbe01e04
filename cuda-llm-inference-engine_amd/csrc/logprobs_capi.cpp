// logprobs_capi.cpp — the extern "C" boundary of include/ie_logprobs.h: every
// check is made here, before any HIP call.
#include "ie_logprobs.h"

#include <hip/hip_runtime.h>

#include "logprobs.h"

extern "C" {

// Words that a row's part leaves for the join: its statistics, then k keys and
// k indices.
size_t ie_token_logprobs_workspace_bytes(int rows, int n, int k) {
    if (rows <= 0 || n <= 0 || k < 0 || n > IE_LOGPROBS_N_MAX || k > IE_LOGPROBS_TOP_MAX) return 0;
    const int parts = ie::logprobs_parts(rows, n, k);
    return parts > 1 ? (size_t)rows * parts * (8 + 2 * k) * sizeof(float) : 0;
}

int ie_token_logprobs(int rows, const float* logits, int row_stride, int n, const int* targets, int k,
                      float* logprobs, int* ranks, float* entropy, float* top_logprobs, int* top_idx,
                      float* workspace, size_t workspace_bytes, ie_stream_t stream) {
    using ie::fail;
    const char* fn = "token_logprobs";
    if (rows < 0 || n <= 0) return fail(IE_ERR_INVALID, "%s: bad sizes rows=%d n=%d", fn, rows, n);
    if (n > IE_LOGPROBS_N_MAX) return fail(IE_ERR_UNSUPPORTED, "%s: n=%d above %d", fn, n, IE_LOGPROBS_N_MAX);
    if (row_stride < n) return fail(IE_ERR_INVALID, "%s: row_stride=%d below n=%d", fn, row_stride, n);
    if (k < 0 || k > n || k > IE_LOGPROBS_TOP_MAX)
        return fail(IE_ERR_INVALID, "%s: k=%d outside [0, min(n=%d, %d)]", fn, k, n, IE_LOGPROBS_TOP_MAX);
    if (rows > (1 << 20)) return fail(IE_ERR_UNSUPPORTED, "%s: rows=%d above 2^20", fn, rows);
    if (rows == 0) return IE_OK;
    if (!logits || (k > 0 && (!top_logprobs || !top_idx)))
        return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if ((uintptr_t)logits % 4 || (uintptr_t)targets % 4)
        return fail(IE_ERR_INVALID, "%s: logits and targets must be 4-byte aligned", fn);
    const size_t need = ie_token_logprobs_workspace_bytes(rows, n, k);
    if (need) {
        if (!workspace) return fail(IE_ERR_INVALID, "%s: null workspace", fn);
        if ((uintptr_t)workspace % 8) return fail(IE_ERR_INVALID, "%s: workspace must be 8-byte aligned", fn);
        if (workspace_bytes < need)
            return fail(IE_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu", fn, workspace_bytes, need);
    }
    ie::LogprobsArgs a{rows, logits, row_stride, n, targets, k, logprobs, ranks, entropy, top_logprobs, top_idx, workspace};
    ie::launch_token_logprobs(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

}  // extern "C"
