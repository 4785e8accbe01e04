// kv8_attn.hip — attention over the 8-bit paged KV cache, the plain kernel:
// one workgroup per (sequence, token, query head) walks the keys 256 at a time
// (one key a thread for the scores, one channel a thread for the output) with
// a running maximum and sum.
#include <cmath>

#include "device_util.h"
#include "kv8.h"

namespace ie {
namespace {

template <int D>
__global__ __launch_bounds__(256) void kv8_attn_kernel(Kv8Attn a, float qscale) {
    __shared__ float q[D], p[256], red[4], part[256 / D][D];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    unsigned id = blockIdx.x;
    const int hq = (int)(id % (unsigned)a.H_q);
    id /= (unsigned)a.H_q;
    const int t = (int)(id % (unsigned)a.P), b = (int)(id / (unsigned)a.P);
    const int h = hq / (a.H_q / a.c.H), lg = a.c.bs_log2, bs = 1 << lg;
    const int n = a.lens ? min(a.lens[b], a.max_ctx) : a.start + t + 1;
    const float* qrow = a.Q + ((size_t)b * a.P + t) * a.q_ld + (size_t)hq * D;
    if (tid < D) q[tid] = qrow[tid] * qscale;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    const int c = tid % D, half = tid / D;
    for (int k0 = 0; k0 < n; k0 += 256) {
        __syncthreads();
        const int key = k0 + tid;
        float s = -INFINITY;
        if (key < n) {
            const size_t pair = (size_t)a.c.table[(size_t)b * a.c.nbps + (key >> lg)] * a.c.H + h;
            const int8_t* kr = a.c.k + (pair * bs + (key & (bs - 1))) * D;
            float acc = 0.0f;
            for (int i = 0; i < D; ++i) acc = fmaf((float)kr[i], q[i], acc);
            s = acc * a.c.ks[pair];
        }
        const float wm = wave_max(s);
        if (lane == 0) red[wid] = wm;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float pv = key < n ? exp2f(s - mn) : 0.0f;
        p[tid] = pv;
        const float ws = wave_sum(pv);
        __syncthreads();
        if (lane == 0) red[wid] = ws;
        __syncthreads();
        const float f = exp2f(m - mn);
        l = l * f + (red[0] + red[1] + red[2] + red[3]);
        o *= f;
        m = mn;
        for (int i = half; i < 256 && k0 + i < n; i += 256 / D) {
            const int kk = k0 + i;
            const size_t pair = (size_t)a.c.table[(size_t)b * a.c.nbps + (kk >> lg)] * a.c.H + h;
            const int r = kk & (bs - 1);
            const int8_t v = a.c.v[pair * bs * D + ((size_t)(r >> 4) * D + c) * 16 + (r & 15)];
            o = fmaf(p[i] * a.c.vs[pair], (float)v, o);
        }
    }
    part[half][c] = o;
    __syncthreads();
    if (tid < D) {
        float sum = 0.0f;
        for (int i = 0; i < 256 / D; ++i) sum += part[i][tid];
        a.O[((size_t)b * a.P + t) * a.H_q * D + (size_t)hq * D + tid] = n > 0 ? sum / l : 0.0f;
    }
}

void launch(const Kv8Attn& a, hipStream_t s) {
    const unsigned grid = (unsigned)a.B * a.P * a.H_q;
    const float qscale = (1.0f / sqrtf((float)a.c.d)) * 1.4426950408889634f;
    if (a.c.d == 64)
        kv8_attn_kernel<64><<<grid, 256, 0, s>>>(a, qscale);
    else
        kv8_attn_kernel<128><<<grid, 256, 0, s>>>(a, qscale);
}

}  // namespace

void launch_prefill_attn_kv8(const Kv8Attn& a, hipStream_t s) { launch(a, s); }

}  // namespace ie
