// logprobs.hip — log probabilities of given tokens, ranks, entropies and top
// alternatives (include/ie_logprobs.h), the plain kernel: one workgroup per
// row walks the row once for its maximum, once for its sums and once for each
// alternative.
#include <hip/hip_runtime.h>

#include <cmath>

#include "device_util.h"
#include "ie_logprobs.h"
#include "logprobs.h"

namespace ie {
namespace {

__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__global__ __launch_bounds__(256) void logprobs_kernel(LogprobsArgs a) {
    __shared__ float fs[3][4];
    __shared__ int is[4];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int r = blockIdx.x, n = a.n;
    const float* x = a.x + (size_t)r * a.ld;
    float m = -INFINITY;
    for (int i = tid; i < n; i += 256) m = max_of(m, x[i]);
    for (int o = 1; o < 64; o <<= 1) m = max_of(m, __shfl_xor(m, o, 64));
    if (lane == 0) fs[0][wid] = m;
    __syncthreads();
    m = max_of(max_of(fs[0][0], fs[0][1]), max_of(fs[0][2], fs[0][3]));
    __syncthreads();
    const int t = a.targets ? a.targets[r] : -1;
    const bool asked = t >= 0 && t < n;
    const float xt = asked ? x[t] : 0.0f;
    float e = 0.0f, w = 0.0f;
    int ahead = 0, tops = 0;
    const bool empty = m == -INFINITY;
    for (int i = tid; i < n; i += 256) {
        const float v = x[i], d = v - m;
        if (v == m && !empty)
            ++tops;
        else {
            const float ev = empty ? 0.0f : expf(d);
            e += ev;
            w += ev > 0.0f ? ev * d : 0.0f * ev;
        }
        ahead += v > xt || (v == xt && i < t);
    }
    float tf = (float)tops;
    for (int o = 1; o < 64; o <<= 1) {
        e += __shfl_xor(e, o, 64);
        w += __shfl_xor(w, o, 64);
        tf += __shfl_xor(tf, o, 64);
        ahead += __shfl_xor(ahead, o, 64);
    }
    if (lane == 0) {
        fs[0][wid] = e;
        fs[1][wid] = w;
        fs[2][wid] = tf;
        is[wid] = ahead;
    }
    __syncthreads();
    e = fs[0][0] + fs[0][1] + fs[0][2] + fs[0][3];
    w = fs[1][0] + fs[1][1] + fs[1][2] + fs[1][3];
    tf = fs[2][0] + fs[2][1] + fs[2][2] + fs[2][3];
    ahead = is[0] + is[1] + is[2] + is[3];
    // log sum exp(x - m) = log(1 + rest): the rest keeps its bits where one token has it all
    const float rest = empty ? 0.0f : e + (tf - 1.0f) + (m - m);
    const float L = log1pf(rest);
    if (tid == 0) {
        if (a.logprobs) a.logprobs[r] = !asked ? (t == -1 ? 0.0f : NAN) : empty ? -INFINITY : xt - m - L;
        if (a.ranks) a.ranks[r] = asked ? ahead + 1 : 0;
        if (a.entropy) a.entropy[r] = empty ? 0.0f : L - w / (1.0f + rest);
    }
    float pv = INFINITY;
    int pi = -1;
    for (int k = 0; k < a.k; ++k) {
        float bv = -INFINITY;
        int bi = n;
        for (int i = tid; i < n; i += 256) {
            const float v = x[i];
            const bool after = k == 0 || v < pv || (v == pv && i > pi);
            if (after && (bi == n || v > bv)) {
                bv = v;
                bi = i;
            }
        }
        for (int o = 1; o < 64; o <<= 1) {
            const float ov = __shfl_xor(bv, o, 64);
            const int oi = __shfl_xor(bi, o, 64);
            if (oi < n && (bi == n || ov > bv || (ov == bv && oi < bi))) {
                bv = ov;
                bi = oi;
            }
        }
        __syncthreads();
        if (lane == 0) {
            fs[0][wid] = bv;
            is[wid] = bi;
        }
        __syncthreads();
        bv = fs[0][0];
        bi = is[0];
        for (int v = 1; v < 4; ++v)
            if (is[v] < n && (bi == n || fs[0][v] > bv || (fs[0][v] == bv && is[v] < bi))) {
                bv = fs[0][v];
                bi = is[v];
            }
        pv = bv;
        pi = bi;
        if (tid == 0) {
            a.top_logprobs[(size_t)r * a.k + k] = empty ? -INFINITY : bv - m - L;
            a.top_idx[(size_t)r * a.k + k] = min(bi, n - 1);
        }
    }
}

}  // namespace

int logprobs_parts(int, int, int) { return 1; }

void launch_token_logprobs(const LogprobsArgs& a, hipStream_t s) { logprobs_kernel<<<a.rows, 256, 0, s>>>(a); }

}  // namespace ie
