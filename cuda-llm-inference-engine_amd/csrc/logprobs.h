// logprobs.h — launcher of the log-probability kernels (logprobs.hip;
// arguments validated by logprobs_capi.cpp).
#pragma once

#include "ie_internal.h"

namespace ie {

struct LogprobsArgs {
    int rows;
    const float* x;
    int ld;
    int n;
    const int* targets;
    int k;
    float* logprobs;
    int* ranks;
    float* entropy;
    float* top_logprobs;
    int* top_idx;
    float* ws;
};
// Parts that a row is cut into (above 1 the workspace joins them).
int logprobs_parts(int rows, int n, int k);
void launch_token_logprobs(const LogprobsArgs& a, hipStream_t s);

}  // namespace ie
