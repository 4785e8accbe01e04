// paged_attn.hip — attention over the paged cache with capped, biased and ranged
// scores, and of drafted trees (include/ie_paged.h).
#include "device_util.h"
#include "paged.h"

namespace ie {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t cache_row(const PageMap& m, const int* table, int p) {
    const int page = m.mul ? (int)(__umulhi((uint32_t)p, m.mul) >> m.shift) : p;
    return (uint32_t)table[page] * (uint32_t)m.block + (uint32_t)(p - page * m.block);
}

template <typename KV>
__device__ __forceinline__ float as_float(KV x) {
    if constexpr (sizeof(KV) == 4) return x;
    else return bf16_to_f32(x);
}

// A query row: token t of sequence b, its position and the keys it may see.
// Ranges: lo <= j < hi.  A tree: lo <= j < ctx, and ctx + u for u itself and its
// ancestors whose position is at least lo.
struct Row {
    int b, t, lo, hi, pos, ctx;
    bool live;
};

__device__ __forceinline__ int depth_of(const int* parents, int t) {
    int n = 0;
    for (int a = parents[t], c = t; a >= 0 && a < c; c = a, a = parents[a]) ++n;
    return n;
}

__device__ __forceinline__ Row row_at(const PagedAttn& a, int b, int t) {
    Row r;
    r.b = b;
    r.t = t;
    const int len = a.lens ? min(a.lens[b], a.P) : a.P;
    const int start = min(max(a.starts[b], 0), 1 << 30);
    r.live = t < len;
    r.lo = 0;
    if (a.parents) {
        r.ctx = min(start, a.max_ctx);
        r.pos = r.ctx + (r.live ? depth_of(a.parents + (size_t)b * a.P, t) : 0);
        r.hi = r.ctx + t + 1;
    } else {
        const size_t i = (size_t)b * a.P + t;
        r.pos = start + t;
        r.hi = min(min(start + len, a.max_ctx), a.end ? a.end[i] : r.pos + 1);
        if (a.first) r.lo = max(0, a.first[i]);
        r.ctx = 1 << 30;
    }
    if (a.window) r.lo = max(r.lo, r.pos - a.window + 1);
    return r;
}

// Whether a row sees key j of [lo, hi), and how far off it is.
__device__ __forceinline__ bool sees(const PagedAttn& a, const Row& r, int j, float& gap) {
    gap = fabsf((float)(r.pos - j));
    if (j < r.ctx) return j >= r.lo;
    const int* parents = a.parents + (size_t)r.b * a.P;
    const int u = j - r.ctx;
    int n = r.t, up = 0;
    while (n > u) {
        const int p = parents[n];
        n = p >= 0 && p < n ? p : -1;
        ++up;
    }
    gap = (float)up;
    return n == u && r.pos - up >= r.lo;
}

// A wave a row: a lane a key for the scores, two or one channel a lane for the
// sums.  Keys that are not seen are never multiplied.
template <int D, typename KV>
__global__ __launch_bounds__(256) void paged_row_kernel(PagedAttn a) {
    const int lane = threadIdx.x & 63;
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= a.B * a.P * a.H_q) return;
    const int h = row % a.H_q, bt = row / a.H_q;
    const Row r = row_at(a, bt / a.P, bt % a.P);
    if (!r.live) return;
    const int* table = a.pages.table + (size_t)r.b * a.pages.nbps;
    const size_t stride = (size_t)a.H_kv * D, at = (size_t)(h / (a.H_q / a.H_kv)) * D;
    const KV *K = static_cast<const KV*>(a.k) + at, *V = static_cast<const KV*>(a.v) + at;
    const float* q = a.Q + (size_t)row * D;
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    constexpr int N = D / 64;
    float m = -INFINITY, l = 0.0f, o[N] = {};
    for (int c0 = min(r.lo, r.ctx); c0 < r.hi; c0 += 64) {
        const int j = c0 + lane;
        float gap = 0.0f, s = -INFINITY;
        const bool seen = j < r.hi && sees(a, r, j, gap);
        uint32_t slot = 0;
        if (seen) {
            slot = cache_row(a.pages, table, j);
            const KV* k = K + slot * stride;
            float acc[4] = {};
            for (int e = 0; e < D; e += 4)
                for (int i = 0; i < 4; ++i) acc[i] = fmaf(q[e + i], as_float(k[e + i]), acc[i]);
            s = a.scale * ((acc[0] + acc[1]) + (acc[2] + acc[3]));
            if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
            if (a.slopes) s = fmaf(-slope, gap, s);
            s *= kLog2e;
        }
        const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.0f : mn;
        const float alpha = exp2_sm(m - mu), p = seen ? exp2_sm(s - mu) : 0.0f;
        l = fmaf(l, alpha, wave_sum(p));
        m = mn;
        for (int i = 0; i < N; ++i) o[i] *= alpha;
        for (uint64_t left = __ballot(seen); left; left &= left - 1) {
            const int k = __builtin_ctzll(left);
            const float w = __shfl(p, k);
            const KV* v = V + (uint32_t)__shfl((int)slot, k) * stride + lane * N;
            for (int i = 0; i < N; ++i) o[i] = fmaf(w, as_float(v[i]), o[i]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float* out = a.O + (size_t)row * D + lane * N;
    for (int i = 0; i < N; ++i) out[i] = o[i] * inv;
}

}  // namespace

int paged_attn_splits(int, int, int, int, int, int, int, int, int) { return 1; }

void launch_paged_attn(const PagedAttn& a, hipStream_t s) {
    const bool half = a.kv_dtype == IE_KV_BF16;
    const unsigned grid = (unsigned)(((long long)a.B * a.P * a.H_q + 3) / 4);
    auto* k = a.d == 64 ? (half ? paged_row_kernel<64, uint16_t> : paged_row_kernel<64, float>)
                        : (half ? paged_row_kernel<128, uint16_t> : paged_row_kernel<128, float>);
    k<<<grid, 256, 0, s>>>(a);
}

}  // namespace ie
