// logprobs.hip — log probabilities of given tokens, ranks, entropies and top
// alternatives (include/ie_logprobs.h).
//
// Mathematics.  With m = max x, d = x - m and one element of value m set aside:
// rest = sum of e^d over the others, so log sum e^x = m + log1p(rest), exact to
// its leading bits also where one token has nearly all (1 + rest would round
// the rest away); w = sum e^d d; log p_t = (x_t - m) - log1p(rest); entropy =
// log1p(rest) - w / (1 + rest).  Parts (m_p, rest_p, w_p) of a row join as
// e^(m_p - m) (1 + rest_p) and e^(m_p - m) (w_p + (m_p - m)(1 + rest_p)).
//
// One workgroup streams a row, or a part of it where there are few rows, once;
// nothing of it is kept but each thread's maximum and sums (rescaled a tile at a
// time), each wave's count of the elements ahead of the target, and each wave's
// candidates for the alternatives: a list in LDS of the elements at or above a
// lower bound of the row's k-th largest.  The bound is the least of what the
// waves say of themselves: each the ceil(k / waves)-th largest of its lanes'
// maxima so far, found one ballot a bit after tiles 1, 2, 4, .. (so k elements
// reach it; a wave that reads another's last word reads a lower bound all the
// same, and which elements are listed beyond the k best does not show).  Where a
// list fills up (equal elements) it is cut to its k best, searched for bit by
// bit, and the least of them is the bound.  After the first tile no wave waits
// for another before the row's end; then the lists are ranked by counting.
//
// Many rows are bound by HBM: 2048 x 50257, k = 20 91 us, 4.5 TB/s (a copy of 1 GiB
// moves 4.7 to 5.2); k = 0 77 us.  (With the row held in registers, 25 words a thread,
// 145 us: two rows a CU, which load and compute in step.)  Few rows are bound by
// one wave's instructions and waits (of a wave's 4.0 thousand issue slots with 64 rows,
// k = 5, 2.2 are waits and 1.1 instructions): 8 x 50257, k = 5 10.7 us, of them 4 the
// join's.  Six waves a SIMD at least: with eight, whose 78 scalar registers keep
// 57 more in vector lanes, 512 x 50257, k = 5 32.7 against 31.1 us, 2048, k = 20
// 88.6 against 91.4.  Two, six or eight words in flight a thread instead of four: 8 x
// 50257 11.5, 11.4, 12.2 against 10.9 us; 512 or 1024 threads a row gain nothing
// (8 rows in 8 parts 13.2 and 22.5 against 13.9 us, 2048 rows 126 and 323 against 92).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "device_util.h"
#include "ie_logprobs.h"
#include "logprobs.h"

namespace ie {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.92596298909e-8f;  // log2(e) in two parts
constexpr int kStats = 8;   // words of a part's statistics in the workspace
constexpr int kWide = 256;  // threads of a workgroup (64 for short rows)
constexpr int kMostParts = 16;
constexpr int kWords = 4;   // 16-byte words a thread has in flight: a tile
constexpr int kList = 512;  // candidates of a wave

// e^d, d <= 0, of what many elements share (a thread's, a wave's and a part's sums
// against the row's maximum): the exponent in two parts, so that its rounding
// (d 2^-24 of the result) and log2(e)'s own (1.3e-8 d) do not stay in all of them.
// An element's, and a thread's as its maximum moves, are exp2_sm(d * kLog2e): their
// roundings average out.  -log p under 50257 others lower by 78 to 82: off by 1.4e-7 at
// most, 2.3e-6 with all of them so; 8 x 50257, k = 5 10.75 against 10.6 us.
__device__ __forceinline__ float exp_of(float d) {
    d = fmaxf(d, -200.0f);  // (0 from -127 log 2 on)
    const float t = d * kLog2e, rest = fmaf(d, kLog2eRest, fmaf(d, kLog2e, -t));
    const float p = exp2_sm(t);
    return fmaf(p * 0.6931471805599453f, rest, p);
}

// Unsigned key with the order of the floats, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    uint32_t b = __float_as_uint(x);
    if (b == 0x80000000u) b = 0;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// Element of a workgroup's candidates: larger value first, then lower index.
__device__ __forceinline__ uint64_t packed(float v, int i) {
    return ((uint64_t)order_key(v) << 32) | (0xffffffffu - (uint32_t)i);
}

// Largest over the wave, in every lane; NaN stays.
__device__ __forceinline__ float wave_most(float v) {
    v = max_of(v, dpp_row_ror<8>(v));
    v = max_of(v, dpp_row_ror<4>(v));
    v = max_of(v, dpp_row_ror<2>(v));
    v = max_of(v, dpp_row_ror<1>(v));
    float a, b;
    pair16(v, a, b);
    v = max_of(a, b);
    pair32(v, a, b);
    return max_of(a, b);
}

// Candidates pk[0 .. cnt) ranked (all different), out(rank, packed) for the
// first k; 2^per threads share one.  pk[cnt] and pk[cnt + 1] are 0.
template <int T, typename Out>
__device__ __forceinline__ void rank_candidates(const uint64_t* pk, int cnt, int k, Out&& out) {
    int per = 0;
    while (per < 5 && (cnt << (per + 1)) <= T) ++per;
    const int sub = threadIdx.x & ((1 << per) - 1);
    for (int t = threadIdx.x >> per; t < cnt; t += T >> per) {
        const uint64_t mine = pk[t];
        int rank = 0;
#pragma unroll 4
        for (int u = 2 * sub; u < cnt; u += 2 << per) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(pk + u);
            rank += (int)(o.x > mine) + (int)(o.y > mine);
        }
        for (int o = 1; o < 1 << per; o <<= 1) rank += __shfl_xor(rank, o, 64);
        if (sub == 0 && rank < k) out(rank, mine);
    }
}

// A wave's candidates: list[0 .. cnt) in LDS, cnt uniform.
struct Candidates {
    uint64_t* list;
    int cnt = 0;
    float bound = -INFINITY;

    // Cut to the k largest; the least of them is the bound.
    __device__ __forceinline__ void cut(int k, int lane) {
        if (cnt <= k) return;
        constexpr int E = kList / 64;
        uint64_t e[E];
#pragma unroll
        for (int i = 0; i < E; ++i) e[i] = lane + 64 * i < cnt ? list[lane + 64 * i] : 0;
        // the k-th largest, bit by bit: the key, then the index's 19 bits
        // (n <= 2^19 keeps the 13 above them set)
        uint64_t b = 0;
        int kept = cnt;
        for (int bit = 63; bit >= 0 && kept != k; --bit) {
            if (bit == 31) {
                b |= 0xfff80000u;
                bit = 18;
            }
            const uint64_t c = b | (1ull << bit);
            int m = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) m += __popcll(__ballot(e[i] >= c));
            if (m >= k) {
                b = c;
                kept = m;
            }
        }
        cnt = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint64_t mask = __ballot(e[i] >= b && e[i] != 0);
            if (e[i] >= b && e[i] != 0) list[cnt + __popcll(mask & ((1ull << lane) - 1))] = e[i];
            cnt += __popcll(mask);
        }
        uint64_t least = ~0ull;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (e[i] >= b && e[i] != 0) least = min(least, e[i]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) least = min(least, (uint64_t)__shfl_xor((unsigned long long)least, o, 64));
        bound = fmaxf(bound, key_value((uint32_t)(least >> 32)));
    }

    // Adds the lanes' elements f of index i where `ok` and f reaches the bound;
    // there is room for 64 more.
    __device__ __forceinline__ void add(float f, int i, bool ok, int lane) {
        const uint64_t mask = __ballot(ok && f >= bound);
        if (mask == 0) return;  // uniform
        if (ok && f >= bound) list[cnt + __popcll(mask & ((1ull << lane) - 1))] = packed(f, i);
        cnt += __popcll(mask);
    }
};

// The need-th largest of the lanes' keys (need <= 64): exactly for the first few,
// by taking the largest away, otherwise its first 20 bits, one ballot a bit.
__device__ __forceinline__ uint32_t wave_bound(uint32_t key, int need) {
    if (need <= 4) {  // uniform
        uint32_t b = wave_umax(key);
        for (int found = __popcll(__ballot(key == b)); found < need; found += __popcll(__ballot(key == b))) {
            if (key >= b) key = 0;
            b = wave_umax(key);
        }
        return b;
    }
    uint32_t b = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t c = b | (1u << bit);
        if (__popcll(__ballot(key >= c)) >= need) b = c;
    }
    return b;
}

// blockIdx.x = row * parts + part.  The 16-byte words wholly inside the row are
// cut into parts; the at most three elements before the first of them go to
// threads of the first part, those behind the last to threads of the last, one
// each.  Places without an element hold -inf.
template <int T>
__global__ __launch_bounds__(T, 6) void logprobs_kernel(LogprobsArgs a, int parts, int words_per_part) {
    constexpr int W = T / 64;
    __shared__ __attribute__((aligned(16))) uint64_t pk[W * kList + 2];
    __shared__ float4 sh_s[W];  // a wave's maximum and sums
    __shared__ int2 sh_n[W];    // its count ahead of the target, its candidates
    __shared__ uint32_t sh_b[W];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = (int)(blockIdx.x / (unsigned)parts), part = (int)(blockIdx.x % (unsigned)parts);
    const int n = a.n, k = a.k;
    const float* x = a.x + (size_t)r * a.ld;
    const int head = min((int)(-((uintptr_t)x >> 2) & 3u), n);
    const int words = (n - head) / 4, w0 = min(part * words_per_part, words), w1 = min(w0 + words_per_part, words);
    const float4* base = reinterpret_cast<const float4*>(x + head);
    float4 v[kWords];
    auto load = [&](int c0) {
#pragma unroll
        for (int q = 0; q < kWords; ++q) v[q] = base[min(c0 + q * T + tid, w1 - 1)];
    };
    if (w0 < w1) load(w0);  // ahead of the target's two round trips
    const int t = a.targets ? a.targets[r] : -1;
    const bool asked = t >= 0 && t < n;
    const float xt = asked ? x[t] : 0.0f;
    int xi = INT_MAX;  // this thread's element outside the words
    if (part == 0 && tid < head) xi = tid;
    if (part == parts - 1 && tid >= head && tid < n - 4 * words) xi = 4 * words + tid;
    const float xv = xi < n ? x[xi] : -INFINITY;

    // Elements ahead of the target: at or above it before its word, above it
    // behind.  (v >= xt as v > the number before xt; nothing comes before -inf:
    // there the elements above it are counted, and those of them before it.)
    const uint32_t xb = __float_as_uint(xt);
    const bool lowest = xt == -INFINITY;
    const float before = lowest ? xt : (xb << 1) == 0 ? __uint_as_float(0x80000001u) : __uint_as_float(xt > 0.0f ? xb - 1 : xb + 1);
    const int tw = t >= head ? (t - head) >> 2 : -1;  // the target's word
    int ahead = __popcll(__ballot(xv > (xi < t ? before : xt))), above = __popcll(__ballot(lowest && xv > xt && xi < t));

    Candidates cand{pk + wid * kList};
    if (k > 0) cand.add(xv, xi, xi < n, lane);  // (at most six, listed before there is a bound)

    // Each thread's maximum m, and against it: tops elements equal to it, e = sum
    // e^d and w = sum e^d d of the others.
    float m = xv, e = 0.0f, w = 0.0f, tops = xv == -INFINITY ? 0.0f : 1.0f;
    const int need = (k + W - 1) / W;
    int tile = 0;
    for (int c0 = w0; c0 < w1; c0 += T * kWords, ++tile) {
        if (tile > 0) load(c0);
        if (c0 + T * kWords > w1) {  // uniform: the last tile
#pragma unroll
            for (int q = 0; q < kWords; ++q)
                if (c0 + q * T + tid >= w1) v[q] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
        float most[kWords], mn = m;
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
            most[q] = max_of(max_of(v[q].x, v[q].y), max_of(v[q].z, v[q].w));
            mn = max_of(mn, most[q]);
        }
        const float mm = mn == -INFINITY ? 0.0f : mn;
        {
            const float d = fmaxf(m - mm, -3.0e38f), f = exp2_sm(d * kLog2e), s = e + tops;
            const bool moved = mn != m;
            w = moved ? fmaf(s * f, d, w * f) : w;
            e = moved ? s * f : e;
            tops = moved ? 0.0f : tops;
            m = mn;
        }
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
            auto add = [&](float f) {
                const float d = fmaxf(f - mm, -3.0e38f);  // (finite: 0 times it is 0)
                const float ev = exp2_sm(d * kLog2e);
                const bool top = f == mn;
                e += top ? 0.0f : ev;  // (a small rest beside the maximum's own 1 keeps its bits)
                tops += top ? 1.0f : 0.0f;
                w = fmaf(ev, d, w);
            };
            add(v[q].x);
            add(v[q].y);
            add(v[q].z);
            add(v[q].w);
        }
#pragma unroll
        for (int q = 0; q < kWords; ++q) {  // (behind the sums, which do not wait for the target's logit)
            const float thr = c0 + q * T + tid < tw ? before : xt;
            ahead += __popcll(__ballot(v[q].x > thr)) + __popcll(__ballot(v[q].y > thr)) + __popcll(__ballot(v[q].z > thr)) +
                     __popcll(__ballot(v[q].w > thr));
            if (lowest && c0 + q * T <= tw) {  // uniform
                const bool in = c0 + q * T + tid < tw;
                above += __popcll(__ballot(in && v[q].x > xt)) + __popcll(__ballot(in && v[q].y > xt)) +
                         __popcll(__ballot(in && v[q].z > xt)) + __popcll(__ballot(in && v[q].w > xt));
            }
        }
        if (k == 0) continue;
        if (need <= 64) {
            if (tile == 0 || ((tile & (tile + 1)) == 0 && c0 + T * kWords < w1)) {  // uniform
                const uint32_t b = wave_bound(order_key(m), need);
                if (lane == 0) __hip_atomic_store(&sh_b[wid], b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (tile == 0) __syncthreads();
            }
            uint32_t b = ~0u;
#pragma unroll
            for (int i = 0; i < W; ++i) b = min(b, __hip_atomic_load(&sh_b[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            if (b > order_key(-INFINITY)) cand.bound = fmaxf(cand.bound, key_value(b));
        }
        int most_new = 0;
#pragma unroll
        for (int q = 0; q < kWords; ++q) most_new += 4 * __popcll(__ballot(most[q] >= cand.bound));
        if (most_new == 0) continue;
        if (cand.cnt + most_new <= kList) {
#pragma unroll
            for (int q = 0; q < kWords; ++q) {
                if (__ballot(most[q] >= cand.bound) == 0) continue;
                const int c = c0 + q * T + tid, i = 4 * c + head;
                cand.add(v[q].x, i, c < w1, lane);
                cand.add(v[q].y, i + 1, c < w1, lane);
                cand.add(v[q].z, i + 2, c < w1, lane);
                cand.add(v[q].w, i + 3, c < w1, lane);
            }
        } else {  // word by word, read again, with a cut wherever one might not fit
#pragma unroll 1
            for (int q = 0; q < kWords; ++q) {
                if (cand.cnt + 256 > kList) cand.cut(k, lane);
                const int c = c0 + q * T + tid, i = 4 * c + head;
                const float4 u = base[min(c, w1 - 1)];
                cand.add(u.x, i, c < w1, lane);
                cand.add(u.y, i + 1, c < w1, lane);
                cand.add(u.z, i + 2, c < w1, lane);
                cand.add(u.w, i + 3, c < w1, lane);
            }
        }
    }
    if (asked && tw >= w0 && tw < w1 && wid == 0)  // the target's own word
        for (int i = 4 * tw + head; i < t; ++i) {
            ahead += !lowest && x[i] == xt;
            above += lowest && x[i] > xt;
        }
    if (lowest) {  // equal ones before it: this part's elements before it that are not above it
        const int lo = 4 * w0 + head, hi = 4 * w1 + head;
        int mine = max(min(t, hi) - lo, 0);
        if (part == 0) mine += min(t, head);
        if (part == parts - 1) mine += max(t - (4 * words + head), 0);
        ahead += (wid == 0 ? mine : 0) - above;
    }
    if (cand.cnt > 128) cand.cut(k, lane);  // (k <= 128)

    // the threads' sums against the wave's maximum, then the waves' against the row's
    const float wm = wave_most(m);
    {
        const float d = fmaxf(m - (wm == -INFINITY ? 0.0f : wm), -3.0e38f), f = exp_of(d), s = e + tops;
        w = wave_sum(fmaf(s * f, d, w * f));
        e = wave_sum(m == wm ? e : s * f);
        tops = wave_sum(m == wm ? tops : 0.0f);
    }
    if (lane == 0) {
        sh_s[wid] = make_float4(wm, e, w, tops);
        sh_n[wid] = make_int2(ahead, cand.cnt);
    }
    __syncthreads();
    float rm = sh_s[0].x;
#pragma unroll
    for (int i = 1; i < W; ++i) rm = max_of(rm, sh_s[i].x);
    e = w = tops = 0.0f;
    ahead = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float4 o = sh_s[i];
        const float d = fmaxf(o.x - (rm == -INFINITY ? 0.0f : rm), -3.0e38f), f = exp_of(d), s = o.y + o.w;
        w += fmaf(s * f, d, o.z * f);
        e += o.x == rm ? o.y : s * f;
        tops += o.x == rm ? o.w : 0.0f;
        ahead += sh_n[i].x;
    }
    // What is only written to is read from the arguments here, so that the walk has
    // its scalar registers (with all of them held, 57 were kept in vector lanes).
    const __attribute__((address_space(4))) LogprobsArgs* z =
        (const __attribute__((address_space(4))) LogprobsArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(z));
    const bool empty = rm == -INFINITY;
    const float rest = empty ? 0.0f : e + (tops - 1.0f);
    float L = 0.0f;
    float* stats = z->ws + ((size_t)r * parts + part) * (kStats + 2 * k);
    if (parts == 1) {
        L = log1pf(rest) + (empty ? 0.0f : rm - rm);  // NaN for a row that holds NaN or +inf
        if (tid == 0) {
            if (z->logprobs) z->logprobs[r] = !asked ? (t == -1 ? 0.0f : NAN) : empty ? -INFINITY : xt - rm - L;
            if (z->ranks) z->ranks[r] = asked ? ahead + 1 : 0;
            if (z->entropy) z->entropy[r] = empty ? 0.0f : L - w / (1.0f + rest);
        }
    } else if (tid == 0) {
        stats[0] = rm;
        stats[1] = rest;
        stats[2] = w;
        stats[3] = __int_as_float(ahead);
        stats[4] = xt;
    }
    if (k == 0) return;

    auto out = [&](int rank, uint64_t p) {
        const float val = key_value((uint32_t)(p >> 32));
        const int idx = (int)(0xffffffffu - (uint32_t)p);
        if (parts == 1) {
            z->top_logprobs[(size_t)r * k + rank] = empty ? -INFINITY : val - rm - L;
            z->top_idx[(size_t)r * k + rank] = idx;
        } else {
            stats[kStats + rank] = val;
            stats[kStats + k + rank] = __int_as_float(idx);
        }
    };
    // the waves' lists one behind the other (each first read, then written lower)
    int cnt = 0, mine = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (i == wid) mine = cnt;
        cnt += sh_n[i].y;
    }
    if (W > 1) {
        uint64_t held[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 64 * i < cand.cnt) held[i] = cand.list[lane + 64 * i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 64 * i < cand.cnt) pk[mine + lane + 64 * i] = held[i];
    }
    if (tid < 2) pk[cnt + tid] = 0;
    // ranks that there is no element for: a part shorter than k, a row of NaN
    for (int i = tid; i < k; i += T)
        if (i >= cnt) {
            if (parts == 1) {
                z->top_logprobs[(size_t)r * k + i] = NAN;
                z->top_idx[(size_t)r * k + i] = i;
            } else {
                stats[kStats + i] = -INFINITY;
                stats[kStats + k + i] = __int_as_float(n);
            }
        }
    __syncthreads();
    rank_candidates<T>(pk, cnt, k, out);
}

// Joins a row's parts.
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobsArgs a, int parts) {
    __shared__ __attribute__((aligned(16))) uint64_t pk[kMostParts * IE_LOGPROBS_TOP_MAX + 2];
    const int r = blockIdx.x, tid = threadIdx.x, k = a.k, n = a.n;
    const int stride = kStats + 2 * k;
    const float* ws = a.ws + (size_t)r * parts * stride;
    const int t = a.targets ? a.targets[r] : -1;
    for (int i = tid; i < parts * k; i += 256) {
        const float* p = ws + (i / k) * stride + kStats + i % k;
        const int idx = __float_as_int(p[k]);
        pk[i] = idx < n ? packed(p[0], idx) : (uint64_t)(uint32_t)(i + 1);  // (a rank that its part has no element for: behind all)
    }
    if (tid < 2) pk[parts * k + tid] = 0;
    const bool asked = t >= 0 && t < n;
    const float xt = ws[4];
    float pm[kMostParts], pr[kMostParts], pw[kMostParts];
    int ahead = 0;
#pragma unroll
    for (int p = 0; p < kMostParts; ++p) {
        const float* st = ws + min(p, parts - 1) * stride;
        pm[p] = p < parts ? st[0] : -INFINITY;
        pr[p] = st[1];
        pw[p] = st[2];
        ahead += p < parts ? __float_as_int(st[3]) : 0;
    }
    float m = pm[0];
#pragma unroll
    for (int p = 1; p < kMostParts; ++p) m = max_of(m, pm[p]);
    const bool empty = m == -INFINITY;
    float rest = 0.0f, w = 0.0f;
    bool first = true;  // the first part that holds the maximum sets one element aside
#pragma unroll
    for (int p = 0; p < kMostParts; ++p) {
        const float d = fmaxf(pm[p] - m, -3.0e38f);  // (finite, as above)
        if (pm[p] == -INFINITY) continue;  // (nothing there; NaN is looked at below)
        const float f = exp_of(d);
        const bool it = d == 0.0f && first;
        first = first && !it;
        const float total = f + f * pr[p];
        rest += it ? pr[p] : total;
        w += f * pw[p] + d * total;  // (f before d: 0 times a number)
    }
    const float L = log1pf(rest) + (empty ? 0.0f : m - m);
    if (tid == 0) {
        if (a.logprobs) a.logprobs[r] = !asked ? (t == -1 ? 0.0f : NAN) : empty ? -INFINITY : xt - m - L;
        if (a.ranks) a.ranks[r] = asked ? ahead + 1 : 0;
        if (a.entropy) a.entropy[r] = empty ? 0.0f : L - w / (1.0f + rest);
    }
    if (k == 0) return;
    if (m != m) {  // uniform
        for (int i = tid; i < k; i += 256) {
            a.top_logprobs[(size_t)r * k + i] = NAN;
            a.top_idx[(size_t)r * k + i] = i;
        }
        return;
    }
    __syncthreads();
    rank_candidates<256>(pk, parts * k, k, [&](int rank, uint64_t p) {
        a.top_logprobs[(size_t)r * k + rank] = empty ? -INFINITY : key_value((uint32_t)(p >> 32)) - m - L;
        a.top_idx[(size_t)r * k + rank] = (int)(0xffffffffu - (uint32_t)p);
    });
}

// At most this many 16-byte words lie wholly inside a row of n.
int row_words(int n) { return std::max(n / 4, 1); }

}  // namespace

// A row's parts: up to five workgroups a CU, with as few tiles each as that allows
// and no more parts than those need, where at least four tiles of one workgroup are
// shared out (the second launch costs about four tiles' time) and the join ranks at
// most about 160 candidates.  50257 logits (13 tiles), k = 5: 8 rows 25.1 us in one
// part, 11.9 in 16, 10.8 in 13; 256 rows 29.8, 25.2 in 4, 24.5 in 5; 512 rows 35.4,
// 34.3 in 2; k = 20: 16 rows 30.5, 16.5 in 8, 21.3 in 16; 300 x 32001, k = 1 25.2,
// 22.9 in 3, 22.0 in 4.  64 x 8000, k = 5 (two tiles): 10.6, 12.0 in 2.
int logprobs_parts(int rows, int n, int k) {
    const int words = row_words(n);
    const int tiles = (words + kWide * kWords - 1) / (kWide * kWords);
    if (words < 4 * kWide * kWords - kWide) return 1;
    int p = std::min(1280 / rows, kMostParts);
    if (k > 0) p = std::min(p, 160 / k);
    p = std::max(p, 1);
    const int each = (tiles + p - 1) / p;
    return (tiles + each - 1) / each;
}

void launch_token_logprobs(const LogprobsArgs& a, hipStream_t s) {
    const int parts = logprobs_parts(a.rows, a.n, a.k);
    const int words = row_words(a.n), each = (words + parts - 1) / parts;
    const unsigned grid = (unsigned)a.rows * parts;
    if (each <= 64 * kWords)
        logprobs_kernel<64><<<grid, 64, 0, s>>>(a, parts, each);
    else
        logprobs_kernel<kWide><<<grid, kWide, 0, s>>>(a, parts, each);
    if (parts > 1) logprobs_join_kernel<<<a.rows, 256, 0, s>>>(a, parts);
}

}  // namespace ie
