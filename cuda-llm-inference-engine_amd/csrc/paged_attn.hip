// paged_attn.hip — attention over the paged cache with capped, biased and ranged
// scores, and of drafted trees (include/ie_paged.h).
//
// The rows of a (sequence, KV head) are its tokens times the query heads that share
// the KV head, row t * G + g, so a tile of rows reads a key once for all of them.
// Both products run on v_mfma_f32_32x32x16_bf16 with every fp32 operand as the sum of
// three bf16 (8 bits apiece, so the sum is the fp32 value): S^T = K Q^T, 32 keys x 32
// rows, leaves lane l (i = l % 32, h = l / 32) with row i and keys 8 (v / 4) + 4 h +
// v % 4, v < 16, of a block, so a softmax step is 16 values of the lane's own and one
// swap between the halves; the weights, split again, are as they lie the B operand of
// O^T += V^T P^T, whose A operand takes the same keys: 4 h .. 4 h + 3 and 8 + 4 h .. of
// each 16, read transposed from V's rows (ds_read_b64_tr_b16).  A bf16 cache is one
// part and takes three products, an fp32 cache six of the nine (the rest are below
// 2^-24).  Statistics and outputs are fp32.
#include <type_traits>

#include "device_util.h"
#include "paged.h"
#include "paged_plan.h"
#include "paged_walk.h"

namespace ie {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef __attribute__((address_space(3))) int8_t* lds_i8;

// 16 bytes a lane from global memory straight into LDS, 1 KiB from `to` on (uniform).  Written out because the
// compiler waits for such copies before any LDS read that follows; here the loop's own wait
// is where the stage is first read.  (m0 is the compiler's own: it sets it before each use, and has none here.)
__device__ __forceinline__ void copy16(const int8_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory");
}

// 4 bytes a lane, 256 from `to` on.
__device__ __forceinline__ void copy4(const int* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(to) : "memory");
}
// Waits until at most N of the wave's copies are under way (the oldest end first).
template <int N>
__device__ __forceinline__ void copies_left() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Waits for the wave's own reads and writes of LDS: what copies overwrite has been read, and what other waves read behind a
// barrier has been written.  (The compiler's wait for the latter is missing where a loop ends with the write and begins with
// the barrier.)
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int page_of(const PageMap& m, int p) {
    return m.mul ? (int)(__umulhi((uint32_t)p, m.mul) >> m.shift) : p;
}
__device__ __forceinline__ uint32_t cache_row(const PageMap& m, const int* table, int p) {
    const int page = page_of(m, p);
    return (uint32_t)table[page] * (uint32_t)m.block + (uint32_t)(p - page * m.block);
}

template <typename KV>
__device__ __forceinline__ float as_float(KV x) {
    if constexpr (sizeof(KV) == 4) return x;
    else return bf16_to_f32(x);
}

// The largest and smallest of non-negative ints over the wave.
__device__ __forceinline__ int wave_imax(int v) { return __builtin_amdgcn_readfirstlane((int)wave_umax((uint32_t)v)); }
__device__ __forceinline__ int wave_imin(int v) { return __builtin_amdgcn_readfirstlane((int)~wave_umax(~(uint32_t)v)); }

// ---- operands in three parts
__device__ __forceinline__ uint32_t round_pair(float x0, float x1) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x0, x1}), bf16x2));
}
__device__ __forceinline__ float low_of(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
// x0 and x1 as three parts each, the largest first, x0's in the low halves.
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t& a, uint32_t& b, uint32_t& c) {
    a = round_pair(x0, x1);
    const float r0 = x0 - low_of(a), r1 = x1 - high_of(a);
    b = round_pair(r0, r1);
    c = round_pair(r0 - low_of(b), r1 - high_of(b));
}
template <int N>
struct Parts {
    uint4 p[N];
};
__device__ __forceinline__ Parts<3> split8(const float* x) {
    Parts<3> r;
    split_pair(x[0], x[1], r.p[0].x, r.p[1].x, r.p[2].x);
    split_pair(x[2], x[3], r.p[0].y, r.p[1].y, r.p[2].y);
    split_pair(x[4], x[5], r.p[0].z, r.p[1].z, r.p[2].z);
    split_pair(x[6], x[7], r.p[0].w, r.p[1].w, r.p[2].w);
    return r;
}

// ---- the matrix instructions' shapes: M rows a wave (lane l: row i = l % M, group g = l / M)
// M = 32: v_mfma_f32_32x32x16_bf16; M = 16: v_mfma_f32_16x16x32_bf16.  A lane has 8 values of an operand, of channels (or
// keys' slots) 8 g on of each step; of a product AV values, its column the lane's row.  Of a block of 32 keys it ends
// with the scores of keys STEP (v / 4) + 4 g + v % 4, v < NS, whose weights p[8 k ..] are step k's operand of the
// second product.
template <int M>
struct Shape {
    static constexpr int AV = M * M / 64, TILES = 32 / M, NS = TILES * AV, STEP = M == 32 ? 8 : 16;
    static constexpr int KC = 512 / M;  // channels (keys) of a step
    typedef float Acc __attribute__((ext_vector_type(AV)));
    __device__ static __forceinline__ float rows_max(float x) {
        if constexpr (M == 16) x = max_xor16(x);
        return max_xor32(x);
    }
    __device__ static __forceinline__ float rows_sum(float x) {
        if constexpr (M == 16) x = sum_xor16(x);
        return sum_xor32(x);
    }
    // rows (bit i) that have a lane among `lanes`
    __device__ static __forceinline__ uint32_t rows_of(uint64_t lanes) {
        uint32_t x = (uint32_t)lanes | (uint32_t)(lanes >> 32);
        if constexpr (M == 16) x = (x | x >> 16) & 0xffffu;
        return x;
    }
};
__device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// c[t] += a[t] b, of a's N parts and b's three, the small products first; an accumulator's own are not back to back.
template <int N, int NT, typename Acc>
__device__ __forceinline__ void product(const Parts<N> (&a)[NT], const Parts<3>& b, Acc* c) {
    auto all = [&](int i, int j) {
#pragma unroll
        for (int t = 0; t < NT; ++t) c[t] = mfma(a[t].p[i], b.p[j], c[t]);
    };
    if constexpr (N == 3) {
        all(2, 0);
        all(0, 2);
        all(1, 1);
        all(1, 0);
    } else {
        all(0, 2);
    }
    all(0, 1);
    all(0, 0);
}

// ---- scores
// cap * tanh(x), cap with the factor to base 2.  Below 1 x (cap + y P(y)), y = x^2, P the polynomial nearest to
// cap (tanh(x) / x - 1) / y there (weighted least squares: 5.6e-9 of the value off, with fp32's
// steps and the cap's own 1.5e-7), below 0.55 one of degree 3 (3.8e-8, with fp32's steps 1.5e-7): nine instructions or six, which is all
// that a block takes whose scores lie there (2 x 2048 x 8 x 2 x 128 at scores below 0.4 of the cap 129.7 -> 126.0 us for the
// second; the kernel of one row, which waits for memory, has the first alone).  Above it 1 - 2 / (1 + e^2x), whose
// rounding is that of a value near 1; a block with one such score takes it for all (160 us).
struct Cap {
    float cap, p[7], low[4];
};
// The same value of every lane, in a scalar register.
__device__ __forceinline__ float uniform(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
__device__ __forceinline__ Cap cap_of(float cap) {
    const float c = cap * kLog2e;
    return {uniform(c),
            {uniform(c * -0.33333295583724976f), uniform(c * 0.13332344591617584f), uniform(c * -0.05387980118393898f),
             uniform(c * 0.021486656740307808f), uniform(c * -0.007946106605231762f), uniform(c * 0.0023013646714389324f),
             uniform(c * -0.00035845203092321754f)},
            {uniform(c * -0.3333294689655304f), uniform(c * 0.13320724666118622f), uniform(c * -0.05267181247472763f), uniform(c * 0.016437580808997154f)}};
}
__device__ __forceinline__ float capped_small(float x, const Cap& c) {
    const float y = x * x;
    float p = c.p[6];
#pragma unroll
    for (int i = 5; i >= 0; --i) p = fmaf(p, y, c.p[i]);
    return x * fmaf(p, y, c.cap);
}
__device__ __forceinline__ float capped_low(float x, const Cap& c) {
    const float y = x * x;
    float p = c.low[3];
#pragma unroll
    for (int i = 2; i >= 0; --i) p = fmaf(p, y, c.low[i]);
    return x * fmaf(p, y, c.cap);
}
__device__ __forceinline__ float capped(float x, const Cap& c) {
    const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * fabsf(x));
    const float big = c.cap * __builtin_copysignf(fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f), x);
    return fabsf(x) < 1.0f ? capped_small(x, c) : big;
}

// A head's slope to base 2 (0: none).  One that passes fp32 so is its largest: infinite it would make NaN of the
// distance 0, and any other distance takes all weight either way.
__device__ __forceinline__ float slope_of(const PagedAttn& a, int head) {
    if (!a.slopes) return 0.0f;
    const float x = a.slopes[head], y = x * kLog2e;
    return __builtin_isinf(y) && !__builtin_isinf(x) ? __builtin_copysignf(__FLT_MAX__, x) : y;
}

// What turns a product q.k into a score of base 2: the factor folded into q, and the distance's factor.
struct Scores {
    float q, slope;
};
__device__ __forceinline__ Scores scores_of(const PagedAttn& a, int head) {
    Scores s;
    s.q = a.cap > 0.0f ? a.scale / a.cap : a.scale * kLog2e;
    s.slope = slope_of(a, head);
    return s;
}

// ---- a tree's ancestors, by node: bit u of line[t] says that t sees node u, depth
// the number of its ancestors (inside or outside the window).
constexpr int kLine = IE_TREE_MAX / 32 + 1;  // (odd: 32 rows' words lie in different banks)
struct TreeLds {
    uint32_t line[IE_TREE_MAX][kLine];
    int depth[IE_TREE_MAX];
    int up[IE_TREE_MAX];
};
struct NoTree {};

// By pointer doubling: after round k a node has its 2^k nearest ancestors.  For any workgroup of at least IE_TREE_MAX
// threads, the first of which have a node each.
__device__ __forceinline__ void grow_tree(TreeLds& s, const int* parents, int T, int window) {
    const int t = threadIdx.x;
    const bool node = t < IE_TREE_MAX;
    constexpr int W = kLine - 1;
    uint32_t w[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = t >> 5 == k ? 1u << (t & 31) : 0u;
    int up = node && t < T ? parents[t] : -1;
    if (up >= t || up < 0) up = -1;
#pragma unroll 1
    for (int round = 0; round <= 8; ++round) {  // (2^8 ancestors at most)
        if (node) {
            s.up[t] = up;
#pragma unroll
            for (int k = 0; k < W; ++k) s.line[t][k] = w[k];
        }
        if (!__syncthreads_or(up >= 0)) break;
        if (up >= 0) {
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] |= s.line[up][k];
            up = s.up[up];
        }
        __syncthreads();
    }
    int deep = -1;
#pragma unroll
    for (int k = 0; k < W; ++k) deep += __builtin_popcount(w[k]);
    if (node) s.depth[t] = deep;
    __syncthreads();
    if (node && window > 0 && deep >= window) {
#pragma unroll
        for (int k = 0; k < W; ++k) {
            uint32_t keep = w[k];
            for (uint32_t left = w[k]; left; left &= left - 1) {
                const int u = __builtin_ctz(left);
                if (s.depth[32 * k + u] <= deep - window) keep &= ~(1u << u);
            }
            s.line[t][k] = keep;
        }
    }
    __syncthreads();
}

// ---- rows
// A row sees keys lo <= j < hi; of a tree's, j >= ctx only if its line has them.
struct Row {
    int t, head;  // of the sequence; query head
    int lo, hi, pos;
    bool live;
};

// Row r of a (sequence, KV head): its query.
template <int D>
__device__ __forceinline__ const float* query_row(const PagedAttn& a, int r, int b, int kvh) {
    const int G = a.H_q / a.H_kv, rc = min(r, a.P * G - 1), t = rc / G;
    return a.Q + (((size_t)b * a.P + t) * a.H_q + kvh * G + (rc - t * G)) * D;
}

template <bool TREE, typename Tree>
__device__ __forceinline__ Row row_of(const PagedAttn& a, const Tree& tree, int r, int b, int kvh, int start, int len) {
    const int G = a.H_q / a.H_kv;
    Row x;
    const int rc = min(r, a.P * G - 1);
    x.t = rc / G;
    x.head = kvh * G + (rc - x.t * G);
    x.live = r < a.P * G && x.t < len;
    x.lo = 0;
    if constexpr (TREE) {
        x.pos = start + tree.depth[x.t];
        x.hi = start + x.t + 1;
    } else {
        const size_t i = (size_t)b * a.P + x.t;
        x.pos = start + x.t;
        x.hi = max(0, min(min(start + len, a.max_ctx), a.end ? a.end[i] : x.pos + 1));
        if (a.first) x.lo = max(0, a.first[i]);
    }
    if (a.window) x.lo = max(x.lo, x.pos - a.window + 1);
    return x;
}

// The bits of a block of 32 keys from c0 on that a row sees.
template <bool TREE, typename Tree>
__device__ __forceinline__ uint32_t seen_bits(const Tree& tree, const Row& r, int c0, int ctx) {
    const int from = min(max(r.lo - c0, 0), 32), to = min(max(r.hi - c0, 0), 32);
    uint32_t bits = (uint32_t)((1ull << to) - 1) & (uint32_t)(~0ull << from);
    if constexpr (TREE) {
        const int o = c0 - ctx;  // node of the block's first key
        if (o > -32) {
            // nodes o .. o + 31; what lies before the tree counts as seen
            const int w = max(o, 0) >> 5, sh = max(o, 0) & 31;
            const uint32_t lo = w < kLine - 1 ? tree.line[r.t][w] : 0u, hi = w < kLine - 2 ? tree.line[r.t][w + 1] : 0u;
            uint32_t nodes = (uint32_t)((((uint64_t)hi << 32) | lo) >> sh);
            if (o < 0) nodes = (lo << -o) | ((1u << -o) - 1);
            // (a node's position is past ctx, so lo, which is about positions, cannot cut it here)
            const uint32_t before = o < 0 ? (1u << -o) - 1 : 0u;
            const uint32_t past = (uint32_t)((1ull << to) - 1);
            bits = (bits & before) | (nodes & past & ~before);
        }
    }
    return bits;
}

// ---- one row by one wave, a lane a key: what the matrix cores have no three-part
// form for (see attend's `bad`), over keys k0 .. k1 - 1.  Keys that the row does not
// see are not multiplied.  Leaves lane l with channels N l .. of the sum.
template <int D, typename KV, bool TREE, typename Tree>
__device__ __forceinline__ void exact_row(const PagedAttn& a, const Tree& tree, const Row& r, int b, int kvh, int ctx, int k0,
                                          int k1, float& m, float& l, float (&o)[D / 64]) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63;
    const int* table = a.pages.table + (size_t)b * a.pages.nbps;
    const size_t stride = (size_t)a.H_kv * D;
    const KV *K = static_cast<const KV*>(a.k) + (size_t)kvh * D, *V = static_cast<const KV*>(a.v) + (size_t)kvh * D;
    const float* q = a.Q + (((size_t)b * a.P + r.t) * a.H_q + r.head) * D;
    const float slope = slope_of(a, r.head);
    const Cap cap = cap_of(a.cap);
    k0 = max(k0, TREE ? min(r.lo, ctx) : r.lo);
    k1 = min(k1, r.hi);
    // The unit m is the largest score, and 2^32 more where that took a sum of large values past fp32 (2^30 keys at most).
    // Weights of 2^-94 are lost then: what they make of an infinite value is the first sum's.
    float before[N];
    for (int i = 0; i < N; ++i) before[i] = 0.0f;
#pragma unroll 1
    for (float room = 0.0f;; room = 32.0f) {
        float top = -INFINITY;
        m = -INFINITY;
        l = 0.0f;
        for (int i = 0; i < N; ++i) o[i] = 0.0f;
#pragma unroll 1
        for (int c0 = k0; c0 < k1; c0 += 64) {
            const int j = c0 + lane;
            const bool seen = j < k1 && (seen_bits<TREE>(tree, r, c0 + (lane & 32), ctx) >> (lane & 31) & 1);
            float s = -INFINITY;
            uint32_t slot = 0;
            if (seen) {
                slot = cache_row(a.pages, table, j);
                const KV* k = K + slot * stride;
                float acc[4] = {};
#pragma unroll 4
                for (int e = 0; e < D; e += 4)
                    for (int i = 0; i < 4; ++i) acc[i] = fmaf(q[e + i], as_float(k[e + i]), acc[i]);
                s = a.scale * ((acc[0] + acc[1]) + (acc[2] + acc[3]));
                s = a.cap > 0.0f ? capped(s / a.cap, cap) : s * kLog2e;
                int at = j;
                if constexpr (TREE) at = j < ctx ? j : ctx + tree.depth[j - ctx];
                if (a.slopes) s = fmaf(-slope, fabsf((float)(r.pos - at)), s);
            }
            top = fmaxf(top, wave_max(s));
            const float mn = top + room, mu = mn == -INFINITY ? 0.0f : mn;
            const float alpha = exp2_sm(m - mu), p = seen ? exp2_sm(s - mu) : 0.0f;
            l = fmaf(l, alpha, wave_sum(p));
            m = mn;
            for (int i = 0; i < N; ++i) o[i] *= alpha;
#pragma unroll 1
            for (uint64_t left = __ballot(seen); left; left &= left - 1) {
                const int k = __builtin_ctzll(left);
                const float w = __shfl(p, k);
                const KV* v = V + (uint32_t)__shfl((int)slot, k) * stride + lane * N;
                for (int i = 0; i < N; ++i) o[i] = fmaf(w, as_float(v[i]), o[i]);
            }
        }
        float bad = 0.0f;
        for (int i = 0; i < N; ++i) {
            if (o[i] != o[i] && __builtin_isinf(before[i])) o[i] = before[i];
            before[i] = o[i];
            bad = fmaf(o[i], 0.0f, bad);
        }
        if (room > 0.0f || !__ballot(!(bad == 0.0f))) return;
    }
}

// ---- what a wave keeps of its M rows
template <int D, int M>
struct State {
    using Sh = Shape<M>;
    static constexpr int NT = D / M;
    float m, l;              // the weights' unit, and a lane's own keys' sum of them
    typename Sh::Acc o[NT];  // o[t][v]: channel M t + 8 (v / 4) + 4 g + v % 4
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] = typename Sh::Acc{};
    }
    __device__ __forceinline__ void scale(float f) {
        l *= f;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] *= f;
    }
};

// What a wave's rows have in common: keys below all_lo or from all_hi on are not seen by all of them.
struct Limits {
    int lo, hi, all_lo, all_hi;
};
template <bool TREE>
__device__ __forceinline__ Limits limits_of(const Row& row, int ctx) {
    const bool some = row.live && row.lo < row.hi;
    Limits x;
    x.lo = wave_imin(some ? row.lo : 0x7fffffff);
    x.hi = wave_imax(some ? row.hi : 0);
    x.all_lo = wave_imax(row.live ? row.lo : 0);
    x.all_hi = wave_imin(row.live ? (TREE ? min(row.hi, ctx) : row.hi) : 0x7fffffff);
    return x;
}

// ---- gaps between rows' ranges (paged_walk.h)
// Only `first` and `end` can leave one: otherwise a token's keys begin no later than where the token's before it end.
template <bool TREE>
__device__ __forceinline__ bool has_ranges(const PagedAttn& a) {
    return !TREE && (a.first || a.end);
}

// Of a wave's M rows, row i in lane i: the lanes whose range begins a part and those whose range ends one; no gap: none.
struct Gaps {
    uint32_t begins, ends;
};
template <int M, bool TREE>
__device__ __forceinline__ Gaps gaps_of(const PagedAttn& a, const Row& row, const Limits& lim) {
    const Gaps none{0, 0};
    // (where all begin no later than any ends there is none: this is all that most tiles take)
    if (M == 1 || !has_ranges<TREE>(a) || lim.all_lo <= lim.all_hi) return none;
    const KeyRange mine{row.live ? row.lo : 0, row.live ? row.hi : 0};
    const int i = threadIdx.x & (M - 1);
    bool begin = mine.lo < mine.hi, end = begin;
#pragma unroll 1
    for (int j = 0; j < M; ++j) {
        const KeyRange other{__builtin_amdgcn_readlane(mine.lo, j), __builtin_amdgcn_readlane(mine.hi, j)};
        begin &= !hides_begin(mine, other, j < i);
        end &= !hides_end(mine, other, j < i);
    }
    constexpr uint32_t rows = (uint32_t)((1ull << M) - 1);
    const Gaps g{(uint32_t)__ballot(begin) & rows, (uint32_t)__ballot(end) & rows};
    return g.begins & (g.begins - 1) ? g : none;
}
// The key to look up at p.
__device__ __forceinline__ int seen_at(const Gaps& g, const Row& row, int p) {
    if (g.begins == 0) return p;
    int begin = -1, end = -1;
#pragma unroll 1
    for (uint32_t left = g.begins; left; left &= left - 1) {
        const int x = __builtin_amdgcn_readlane(row.lo, __builtin_ctz(left));
        if (x <= p) begin = max(begin, x);
    }
#pragma unroll 1
    for (uint32_t left = g.ends; left; left &= left - 1) {
        const int x = __builtin_amdgcn_readlane(row.hi, __builtin_ctz(left));
        if (x <= p) end = max(end, x);
    }
    return stand_in(p, begin, end);
}

// The same of a workgroup's N rows, by token, in LDS: where parts begin and end, in any order.
template <int N>
struct TileGaps {
    KeyRange range[N];
    int begin[N], end[N], count[2];
};
// Number of parts, 0 without a gap.  Called by the whole workgroup: `row` is the calling lane's, of token `token` of the
// tile's `tokens`, and `real` where the call has such a row.
template <int N>
__device__ __forceinline__ int find_gaps(TileGaps<N>& s, const Row& row, bool real, int token, int tokens) {
    const int t = threadIdx.x;
    if (real) s.range[token] = KeyRange{row.live ? row.lo : 0, row.live ? row.hi : 0};  // (a token's heads: the same)
    if (t < 2) s.count[t] = 0;
    __syncthreads();
    if (t < tokens) {
        const KeyRange mine = s.range[t];
        bool begin = mine.lo < mine.hi, end = begin;
#pragma unroll 1
        for (int j = 0; j < tokens; ++j) {
            const KeyRange other = s.range[j];
            begin &= !hides_begin(mine, other, j < t);
            end &= !hides_end(mine, other, j < t);
        }
        if (begin) s.begin[atomicAdd(&s.count[0], 1)] = mine.lo;
        if (end) s.end[atomicAdd(&s.count[1], 1)] = mine.hi;
    }
    __syncthreads();
    const int parts = __builtin_amdgcn_readfirstlane(s.count[0]);
    return parts > 1 ? parts : 0;
}
template <int N>
__device__ __forceinline__ int seen_at(const TileGaps<N>& s, int parts, int p) {
    if (parts == 0) return p;
    int begin = -1, end = -1;
#pragma unroll 1
    for (int k = 0; k < parts; ++k) {
        if (s.begin[k] <= p) begin = max(begin, s.begin[k]);
        if (s.end[k] <= p) end = max(end, s.end[k]);
    }
    return stand_in(p, begin, end);
}

// The products s of a block's keys from c0 on become their weights; st.o is scaled where their unit moves.
template <int D, int M, bool TREE, typename Tree>
__device__ __forceinline__ void weigh(const PagedAttn& a, const Tree& tree, const Row& row, const Limits& lim, float slope,
                                      const Cap& cap, int c0, int ctx, float (&s)[Shape<M>::NS], State<D, M>& st) {
    constexpr int NS = Shape<M>::NS, STEP = Shape<M>::STEP;
    const int g = (threadIdx.x & 63) / M;
    if (a.cap > 0.0f) {
        float most = 0.0f;
#pragma unroll
        for (int v = 0; v < NS; ++v) most = fmaxf(most, fabsf(s[v]));
        if (__ballot(!(most < 1.0f))) {
#pragma unroll
            for (int v = 0; v < NS; ++v) s[v] = capped(s[v], cap);
        } else if (!__ballot(!(most < 0.55f))) {
#pragma unroll
            for (int v = 0; v < NS; ++v) s[v] = capped_low(s[v], cap);
        } else {
#pragma unroll
            for (int v = 0; v < NS; ++v) s[v] = capped_small(s[v], cap);
        }
    }
    if (a.slopes) {
        if (TREE && c0 + 32 > ctx) {
            if constexpr (TREE) {
#pragma unroll
                for (int v = 0; v < NS; ++v) {
                    const int j = c0 + STEP * (v >> 2) + 4 * g + (v & 3);
                    const int at = j < ctx ? j : ctx + tree.depth[min(j - ctx, IE_TREE_MAX - 1)];
                    s[v] = fmaf(-slope, fabsf((float)(row.pos - at)), s[v]);
                }
            }
        } else {
            const int base = row.pos - c0 - 4 * g;
#pragma unroll
            for (int v = 0; v < NS; ++v) s[v] = fmaf(-slope, fabsf((float)(base - STEP * (v >> 2) - (v & 3))), s[v]);
        }
    }
    if (c0 < lim.all_lo || c0 + 32 > lim.all_hi) {
        const uint32_t bits = seen_bits<TREE>(tree, row, c0, ctx) >> (4 * g);
#pragma unroll
        for (int v = 0; v < NS; ++v)
            if (!(bits >> (STEP * (v >> 2) + (v & 3)) & 1)) s[v] = -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int v = 1; v < NS; ++v) top = fmaxf(top, s[v]);
    // The weights' unit m follows the largest score once that is 2^8 above it: up to there they only grow, and
    // fp32 holds them as well.  (With 32 rows a wave some row's largest grows in most blocks.)
    top = Shape<M>::rows_max(top);
    if (__ballot(top > st.m + 8.0f)) {
        const float mn = fmaxf(st.m, top);
        const float alpha = mn == -INFINITY ? 0.0f : exp2_sm(st.m - mn);
        st.m = mn;
        st.scale(alpha);
    }
    const float mu = st.m == -INFINITY ? 0.0f : st.m;  // no key yet: keep o, l at 0
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NS; ++v) {
        s[v] = exp2_sm(s[v] - mu);
        sum += s[v];
    }
    st.l += sum;
}

// A lane's share of its row of Q: channels KC s + 8 g on.
template <int D, int M>
struct RawQuery {
    static constexpr int KS = D / Shape<M>::KC;
    float4 x[KS][2];
};
template <int D, int M>
__device__ __forceinline__ RawQuery<D, M> load_query(const float* row, int g) {
    RawQuery<D, M> r;
#pragma unroll
    for (int s = 0; s < r.KS; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) r.x[s][k] = *reinterpret_cast<const float4*>(row + Shape<M>::KC * s + 8 * g + 4 * k);
    return r;
}
// Its parts, and whether one of the values has none that serve: one below 2^-98 once scaled, whose parts bf16 may
// not hold, or one from 2^64 on.
template <int D, int M>
__device__ __forceinline__ bool split_query(const float* row, const RawQuery<D, M>& r, float scale,
                                            Parts<3> (&q)[RawQuery<D, M>::KS]) {
    float least = INFINITY, most = 0.0f;
#pragma unroll
    for (int s = 0; s < r.KS; ++s) {
        float z[8] = {r.x[s][0].x, r.x[s][0].y, r.x[s][0].z, r.x[s][0].w, r.x[s][1].x, r.x[s][1].y, r.x[s][1].z, r.x[s][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            z[e] *= scale;
            least = fminf(least, fabsf(z[e]));
            most = fmaxf(most, fabsf(z[e]));
        }
        q[s] = split8(z);
    }
    bool bad = false;
    if (__ballot(!(least >= 0x1p-98f && most < 0x1p64f))) {  // (a zero anywhere among them, as of a padded head, is enough)
#pragma unroll 1
        for (int e = 0; e < D; ++e) {
            const float x = row[e], y = fabsf(x * scale);
            bad |= x != 0.0f && !(y >= 0x1p-98f && y < 0x1p64f);
        }
    }
    return bad;
}

// The rows of `again` (bit x: lane x's) one by one over keys k0 .. k1 - 1: outputs, or with splits partial sums.
template <int D, typename KV, bool TREE, typename Tree>
__device__ __forceinline__ void exact_rows(const PagedAttn& a, const Tree& tree, const Row& row, uint32_t again, int b, int kvh, int ctx,
                                           int split, int k0, int k1) {
    const int lane = threadIdx.x & 63;
    const size_t rows = (size_t)a.B * a.P * a.H_q;
#pragma unroll 1
    for (; again; again &= again - 1) {
        const int x = __builtin_ctz(again);
        Row r;
        r.t = __shfl(row.t, x);
        r.head = __shfl(row.head, x);
        r.lo = __shfl(row.lo, x);
        r.hi = __shfl(row.hi, x);
        r.pos = __shfl(row.pos, x);
        r.live = true;
        float rm, rl, ro[D / 64];
        exact_row<D, KV, TREE>(a, tree, r, b, kvh, ctx, k0, k1, rm, rl, ro);
        const size_t at = ((size_t)b * a.P + r.t) * a.H_q + r.head;
        float* out = a.O + at * D;
        float inv = 1.0f;
        if (a.splits == 1) {
            inv = rl == 0.0f ? 0.0f : 1.0f / rl;
        } else {
            out = a.ws + (split * rows + at) * D;
            if (lane == 0) *reinterpret_cast<float2*>(a.ws + a.splits * rows * D + 2 * (split * rows + at)) = make_float2(rm, rl);
        }
        for (int e = 0; e < D / 64; ++e) out[lane * (D / 64) + e] = ro[e] * inv;
    }
}

// Results of a wave's rows: outputs, or with splits partial sums.  Rows whose result is not finite, or whose query
// has no parts, again one by one over keys k0 .. k1 - 1.
template <int D, int M, typename KV, bool TREE, typename Tree>
__device__ __forceinline__ void finish(const PagedAttn& a, const Tree& tree, const Row& row, int b, int kvh, int ctx, int split,
                                       int k0, int k1, bool q_bad, const State<D, M>& st, float l) {
    constexpr int NT = D / M, AV = Shape<M>::AV;
    const int lane = threadIdx.x & 63, i = lane & (M - 1), g = lane / M;
    float bad = l * 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < AV; ++v) bad = fmaf(st.o[t][v], 0.0f, bad);
    const uint64_t lanes = __ballot(row.live && (q_bad || !(bad == 0.0f)));
    const uint32_t again = Shape<M>::rows_of(lanes);
    const size_t rows = (size_t)a.B * a.P * a.H_q, mine = ((size_t)b * a.P + row.t) * a.H_q + row.head;
    if (row.live && !(again >> i & 1)) {
        float* out;
        float inv = 1.0f;
        if (a.splits == 1) {
            inv = l > 0.0f ? 1.0f / l : 0.0f;
            out = a.O + mine * D;
        } else {
            out = a.ws + (split * rows + mine) * D;
            if (g == 0) *reinterpret_cast<float2*>(a.ws + a.splits * rows * D + 2 * (split * rows + mine)) = make_float2(st.m, l);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int v = 0; v < AV / 4; ++v)
                *reinterpret_cast<float4*>(out + M * t + 8 * v + 4 * g) =
                    make_float4(st.o[t][4 * v] * inv, st.o[t][4 * v + 1] * inv, st.o[t][4 * v + 2] * inv, st.o[t][4 * v + 3] * inv);
    }
    exact_rows<D, KV, TREE>(a, tree, row, again, b, kvh, ctx, split, k0, k1);
}

// Key groups' states through LDS into the first group's wave; `slot` numbers the others' and mine. Groups' waves
// with rows in common call this together; false: the wave is done.
template <int D, int M, int OTHERS>
__device__ __forceinline__ bool gather(int8_t* lds, int group, int per, int which, State<D, M>& st, float& l) {
    constexpr int NT = D / M, Q = Shape<M>::AV / 4, PER_LANE = D * M / 64;
    const int lane = threadIdx.x & 63;
    float4* mo = reinterpret_cast<float4*>(lds);
    float2* ml = reinterpret_cast<float2*>(lds + OTHERS * per * 64 * PER_LANE * 4);
    if (group > 0) {
        const int g = (group - 1) * per + which;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int v = 0; v < Q; ++v)
                mo[((g * NT + t) * Q + v) * 64 + lane] =
                    make_float4(st.o[t][4 * v], st.o[t][4 * v + 1], st.o[t][4 * v + 2], st.o[t][4 * v + 3]);
        ml[g * 64 + lane] = make_float2(st.m, l);
    }
    __syncthreads();
    if (group > 0) return false;
#pragma unroll 1
    for (int k = 0; k < OTHERS; ++k) {
        const int g = k * per + which;
        const float2 x = ml[g * 64 + lane];
        const float mn = fmaxf(st.m, x.x), mu = mn == -INFINITY ? 0.0f : mn;
        const float fa = exp2_sm(st.m - mu), fb = exp2_sm(x.x - mu);
        st.m = mn;
        l = l * fa + x.y * fb;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int v = 0; v < Q; ++v) {
                const float4 y = mo[((g * NT + t) * Q + v) * 64 + lane];
                st.o[t][4 * v] = st.o[t][4 * v] * fa + y.x * fb;
                st.o[t][4 * v + 1] = st.o[t][4 * v + 1] * fa + y.y * fb;
                st.o[t][4 * v + 2] = st.o[t][4 * v + 2] * fa + y.z * fb;
                st.o[t][4 * v + 3] = st.o[t][4 * v + 3] * fa + y.w * fb;
            }
    }
    return true;
}

// Which of the grid's workgroups this is: pair (sequence, KV head) u % pairs, so that a pair's tiles run on one
// XCD where pairs are a multiple of 8; then the tile, the last (a prompt's longest) first, then the split.  Up to 64
// sequences come by length, the longest first, so that what starts last is short (32 x 8 x 4 x 128 over 4096 to 8192 keys in
// two splits 154 us, unsorted 177).
//
// SHARED: two workgroups run on a CU.  Where one round of them fills more than half of the card the second half comes in
// reverse, so that a CU has a long one and a short one (2048 tokens x 8 x 128 58.1 -> 49.7 us; alone on its CU a
// workgroup has to come by length: 2048 x 16 x 128 in fp32 143 -> 200).
constexpr int kCus = 256;
struct Place {
    int b, kvh, tile, split, start, len;
};
template <bool TREE, bool SHARED>
__device__ __forceinline__ Place place_of(const PagedAttn& a, int tiles) {
    const int pairs = a.B * a.H_kv;
    int n = blockIdx.x;
    if (SHARED && n >= kCus && gridDim.x <= 2 * kCus) n = kCus + gridDim.x - 1 - n;
    const int u = n / pairs, pair = n - u * pairs;
    Place p;
    p.split = u / tiles;
    p.tile = tiles - 1 - (u - p.split * tiles);
    p.b = pair / a.H_kv;
    p.kvh = pair - p.b * a.H_kv;
    if (a.B > 1 && a.B <= 64) {
        const int k = threadIdx.x & 63;
        const int len = k < a.B ? a.starts[k] : -0x7fffffff;
        int rank = 0;
        for (int j = 0; j < a.B; ++j) {
            const int other = __builtin_amdgcn_readlane(len, j);
            rank += other > len || (other == len && j < k);
        }
        p.b = __builtin_ctzll(__ballot(k < a.B && rank == p.b));
    }
    p.start = min(max(a.starts[p.b], 0), TREE ? a.max_ctx : 1 << 30);
    p.len = a.lens ? min(a.lens[p.b], a.P) : a.P;
    return p;
}

// V's operand, channels M t on: keys k0 + 4 g .. + 3, and as many 8 (M = 32) or 16 on, of a block's bf16 rows.
template <typename T, int M>
__device__ __forceinline__ uint4 read_v(const int8_t* rows, int k0, int t) {
    // this lane's 8 bytes: key 4 g + (lane % 16) / 4, channels 4 (lane % 4) on of its 16 lanes' 16
    const int lane = threadIdx.x & 63, key = 4 * (lane / M) + (lane & 15) / 4;
    const int c = (M == 32 ? 4 * t + 2 * (lane >> 4 & 1) : 2 * t) + (lane >> 1 & 1);
    const int8_t* at = rows + key * T::ROW + 16 * (c ^ T::vswz(key)) + 8 * (lane & 1) + k0 * T::ROW;
    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at));
    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + (M == 32 ? 8 : 16) * T::ROW)));
    return make_uint4(x.x, x.y, y.x, y.y);
}

// ---- the tile kernel
// WR x WK waves: WR of them take 32 rows each, WK groups of them
// different keys.  A stage holds SK keys' K and V in LDS, NB blocks of 32 for each
// group of waves; rows past the tile's keys are its last key again.
template <int D, int NP, int WR, int WK_>
struct Tile {
    static constexpr int WK = WK_, W = WR * WK, THREADS = 64 * W;
    static constexpr bool SHARED = W == 4 && (D == 64 || (NP == 1 && WR == 4));  // two workgroups run on a CU
    static constexpr int NB = NP == 1 && WR == 4 ? 2 : 1;
    static constexpr int SK = 32 * NB * WK;
    static constexpr int ROW = 2 * D;          // bytes of a part's row
    static constexpr int PART = SK * ROW;      // of a stage's K or V
    static constexpr int STAGE = 2 * NP * PART;
    static constexpr int BUFS = NP == 1 ? 2 : 1;
    static constexpr int MERGE = (WK - 1) * WR * 64 * (D / 2 + 2) * 4;  // the other key groups' states
    static constexpr int LDS = BUFS * STAGE > MERGE ? BUFS * STAGE : MERGE;
    static constexpr int CH = ROW / 16;        // 16-byte chunks of a row
    // Chunk c of row r lies at c ^ swizzle: K's rows are read 32 at a time at one chunk, V's four at a
    // time at four chunks side by side; so each read touches every bank alike.
    __device__ static __forceinline__ int kswz(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
    __device__ static __forceinline__ int vswz(int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }
};

template <int D, int NP, int WR, int WK, bool TREE>
__global__ __launch_bounds__(64 * WR * WK, NP == 1 && WR == 4 ? 2 : 1) void paged_tile_kernel(PagedAttn a, int tiles) {
    using T = Tile<D, NP, WR, WK>;
    using KV = std::conditional_t<NP == 1, uint16_t, float>;
    using Tree = std::conditional_t<TREE, TreeLds, NoTree>;
    constexpr int NT = D / 32, KS = D / 16;
    __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS];
    __shared__ uint32_t slots[2][T::THREADS];  // a thread's each, SK of them keys of the stage
    __shared__ int bounds[T::W][4];
    __shared__ Tree tree;
    __shared__ std::conditional_t<TREE, NoTree, TileGaps<32 * WR>> gaps;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave % WR, kw = wave / WR;
    const Place at = place_of<TREE, T::SHARED>(a, tiles);
    const int b = at.b, kvh = at.kvh, ctx = at.start;
    const int r = at.tile * 32 * WR + rw * 32 + i;
    // the query first: it waits for nothing
    const float* q_row = query_row<D>(a, r, b, kvh);
    const RawQuery<D, 32> raw_q = load_query<D, 32>(q_row, h);
    if constexpr (TREE) grow_tree(tree, a.parents + (size_t)b * a.P, a.P, a.window);
    const Row row = row_of<TREE>(a, tree, r, b, kvh, at.start, at.len);
    const Limits lim = limits_of<TREE>(row, ctx);
    if (lane == 0) {
        bounds[wave][0] = lim.lo;
        bounds[wave][1] = lim.hi;
        bounds[wave][2] = lim.all_lo;
        bounds[wave][3] = lim.all_hi;
    }
    __syncthreads();
    int kbeg = 0x7fffffff, kend = 0;
#pragma unroll
    for (int w = 0; w < T::W; ++w) {
        kbeg = min(kbeg, bounds[w][0]);
        kend = max(kend, bounds[w][1]);
    }
    kend = __builtin_amdgcn_readfirstlane(kend);  // (scalars, and all that follows from them)
    kbeg = min(__builtin_amdgcn_readfirstlane(kbeg), kend);
    int parts = 0;
    if constexpr (!TREE) {
        if (has_ranges<TREE>(a)) {
            int lo = 0, hi = 0x7fffffff;
#pragma unroll
            for (int w = 0; w < T::W; ++w) {
                lo = max(lo, bounds[w][2]);
                hi = min(hi, bounds[w][3]);
            }
            // (as in gaps_of)
            if (__builtin_amdgcn_readfirstlane(lo) > __builtin_amdgcn_readfirstlane(hi)) {
                const int G = a.H_q / a.H_kv, r0 = at.tile * 32 * WR, t0 = r0 / G, t1 = (min(r0 + 32 * WR, a.P * G) - 1) / G;
                parts = find_gaps(gaps, row, r < a.P * G, row.t - t0, t1 - t0 + 1);
            }
        }
    }
    // this split's stages
    const int all = (kend - kbeg + T::SK - 1) / T::SK, per = (all + a.splits - 1) / a.splits;
    const int s0 = min(at.split * per, all), s1 = min(s0 + per, all);
    const int k0 = kbeg + s0 * T::SK, k1 = min(kbeg + s1 * T::SK, kend);

    const int* table = a.pages.table + (size_t)b * a.pages.nbps;
    const size_t row_bytes = (size_t)a.H_kv * D * sizeof(KV);
    const int8_t* kbase = reinterpret_cast<const int8_t*>(static_cast<const KV*>(a.k) + (size_t)kvh * D);
    const int8_t* vbase = reinterpret_cast<const int8_t*>(static_cast<const KV*>(a.v) + (size_t)kvh * D);
    auto pos_of = [&](int s) {  // of a stage's key tid
        const int p = min(kbeg + s * T::SK + tid, k1 - 1);
        if constexpr (TREE) return p;
        else return seen_at(gaps, parts, p);
    };
    // bf16: a stage's rows straight into LDS; a wave's load fills 1 KiB, its lanes' addresses are
    // permuted so that the chunks land swizzled.
    constexpr int RPL = 1024 / T::ROW, LOADS = T::SK / RPL / T::W;
    const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_i8)lds);
    // (a lane's rows are multiples of 16 apart, after which both swizzles repeat: one place in the row each)
    const int lane_row = wave * RPL + lane / T::CH;
    const int kcol = 16 * ((lane % T::CH) ^ T::kswz(lane_row)), vcol = 16 * ((lane % T::CH) ^ T::vswz(lane_row));
    auto copy = [&](int s, int buf) {
        if constexpr (NP == 1) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                const uint64_t at = slots[s & 1][lane_row + T::W * j * RPL] * row_bytes;
                const uint32_t to = lds_at + buf * T::STAGE + (wave + T::W * j) * 1024;
                copy16(kbase + (at + kcol), to);
                copy16(vbase + (at + vcol), to + T::PART);
            }
        }
    };
    // fp32: through registers, split on the way.
    constexpr int CPT = NP == 1 ? 1 : T::SK * T::CH / T::THREADS;  // chunks of eight values a thread
    float4 raw[2][CPT][2];
    auto load = [&](int s) {
        if constexpr (NP == 3) {
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
                const int id = tid + T::THREADS * j, r = id / T::CH, c = id % T::CH;
                const size_t at = slots[s & 1][r] * row_bytes + 32 * c;
                raw[0][j][0] = *reinterpret_cast<const float4*>(kbase + at);
                raw[0][j][1] = *reinterpret_cast<const float4*>(kbase + at + 16);
                raw[1][j][0] = *reinterpret_cast<const float4*>(vbase + at);
                raw[1][j][1] = *reinterpret_cast<const float4*>(vbase + at + 16);
            }
        }
    };
    auto store = [&] {
        if constexpr (NP == 3) {
#pragma unroll
            for (int j = 0; j < CPT; ++j) {
                const int id = tid + T::THREADS * j, r = id / T::CH, c = id % T::CH;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float4 p = raw[x][j][0], q = raw[x][j][1];
                    const float y[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
                    const Parts<3> parts = split8(y);
                    const int at = x * NP * T::PART + r * T::ROW + 16 * (c ^ (x ? T::vswz(r) : T::kswz(r)));
#pragma unroll
                    for (int n = 0; n < 3; ++n) *reinterpret_cast<uint4*>(lds + at + n * T::PART) = parts.p[n];
                }
            }
        }
    };

    if (s0 < s1) {
        slots[s0 & 1][tid] = cache_row(a.pages, table, pos_of(s0));
        slots[(s0 + 1) & 1][tid] = cache_row(a.pages, table, pos_of(s0 + 1));
    }
    __syncthreads();
    if (s0 < s1) {
        if constexpr (NP == 1) copy(s0, 0);
        else load(s0);
    }

    const Scores sc = scores_of(a, row.head);
    const Cap cap = cap_of(a.cap);
    Parts<3> q[KS];
    const bool q_bad = split_query<D, 32>(q_row, raw_q, sc.q, q);
    State<D, 32> st;
    st.clear();

    const int krow = i * T::ROW, kx = 16 * (h ^ T::kswz(i));  // chunk 2 s + h of key i
    auto attend = [&](const int8_t* stage, int blk, int c0) {
        const int8_t* kp = stage + blk * 32 * T::ROW;
        const int8_t* vp = stage + NP * T::PART + blk * 32 * T::ROW;
        __builtin_amdgcn_s_setprio(0);
        f32x16 sa[1] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            Parts<NP> x[1];
#pragma unroll
            for (int n = 0; n < NP; ++n) x[0].p[n] = *reinterpret_cast<const uint4*>(kp + n * T::PART + krow + (kx ^ (32 * k)));
            product<NP, 1>(x, q[k], sa);
        }
        __builtin_amdgcn_s_setprio(1);
        float p[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) p[v] = sa[0][v];
        weigh<D, 32, TREE>(a, tree, row, lim, sc.slope, cap, c0, ctx, p, st);
        __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Parts<3> w = split8(p + 8 * k);
#pragma unroll
            for (int t0 = 0; t0 < NT; t0 += 2) {
                Parts<NP> x[2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < NP; ++n) x[t].p[n] = read_v<T, 32>(vp + n * T::PART, 16 * k, t0 + t);
                product<NP, 2>(x, w, st.o + t0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };

#pragma unroll 1
    for (int s = s0; s < s1; ++s) {
        int buf = 0;
        lds_done();  // (slots of the last iteration)
        if constexpr (NP == 1) {
            buf = (s - s0) & 1;
            copies_left<0>();
            __syncthreads();  // stage s is there, and the other buffer read
            if (s + 1 < s1) copy(s + 1, buf ^ 1);
        } else {
            __syncthreads();  // the last stage has been read
            store();
            __syncthreads();
            if (s + 1 < s1) load(s + 1);
        }
        // The page of this thread's key of stage s + 2: asked for here, used behind the products.  By every
        // thread, and at the end too, where it is k1 - 1's: a register loaded or used under a condition makes
        // the compiler wait for the copies here.
        const int p2 = pos_of(s + 2), in2 = page_of(a.pages, p2);
        const uint32_t page = (uint32_t)table[in2], row2 = (uint32_t)(p2 - in2 * a.pages.block);
        const int8_t* stage = lds + buf * T::STAGE;
#pragma unroll 1
        for (int n = 0; n < T::NB; ++n) {
            const int blk = kw * T::NB + n, c0 = kbeg + s * T::SK + 32 * blk;
            if (c0 < lim.hi && c0 + 32 > lim.lo) attend(stage, blk, c0);
        }
        slots[s & 1][tid] = page * (uint32_t)a.pages.block + row2;
    }
    float l = sum_xor32(st.l);
    if constexpr (T::WK > 1) {
        __syncthreads();
        if (!gather<D, 32, T::WK - 1>(lds, kw, WR, rw, st, l)) return;
    }
    finish<D, 32, KV, TREE>(a, tree, row, b, kvh, ctx, at.split, k0, k1, q_bad, st, l);
}

// ---- the kernel for at most 32 rows
// Four or eight waves, all of the same 16 or 32 rows, take the keys' blocks of 32 in turn, each by itself: its K and V come into LDS
// of its own as they lie in the cache, DEEP blocks ahead, so the loop has no barrier and a block's products
// run beside the next ones' copies.  Of a bf16 cache K's and V's rows are operands as in the tile kernel; fp32 rows
// are split as they are read, V's a channel a lane (32 lanes read 128 bytes).  A page's number comes the same way,
// DEEP blocks ahead of its rows.
template <int D, int NP, int M>
struct Few {
    static constexpr int ROW = D * (NP == 1 ? 2 : 4);  // bytes of a row
    static constexpr int PART = 32 * ROW;              // of a block's K or V
    static constexpr int WAVES = M == 16 && PART <= 8192 ? 8 : 4;
    static constexpr int DEEP = WAVES * 4 * PART > 128 * 1024 ? 1 : 2;
    static constexpr int WAVE = 2 * DEEP * PART;
    static constexpr int COPIES = PART / 1024;         // a wave's copies of K or V
    static constexpr int MERGE = (WAVES - 1) * 64 * (D * M / 64 + 2) * 4;
    static constexpr int LDS = WAVES * WAVE;
    static constexpr int CH = ROW / 16;
    static_assert(LDS >= MERGE && 3 * COPIES + 2 < 63, "a wave's ring");
    // As Tile's; fp32 rows' chunks of four values, of which K's operand takes two; 16 rows' V is read eight keys at a
    // time at two chunks.
    __device__ static __forceinline__ int kswz(int r) {
        return NP == 3 ? (r & 7) << 1 : D == 128 ? r & 15 : (r >> 1) & 7;
    }
    __device__ static __forceinline__ int vswz(int r) {
        if (NP == 3) return 0;
        if (M == 16) return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
        return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
    }
};

template <int D, int NP, int M, bool TREE>
__global__ __launch_bounds__((64 * Few<D, NP, M>::WAVES), (Few<D, NP, M>::WAVES / 4)) void paged_few_kernel(PagedAttn a, int tiles) {
    using T = Few<D, NP, M>;
    using Sh = Shape<M>;
    using KV = std::conditional_t<NP == 1, uint16_t, float>;
    using Tree = std::conditional_t<TREE, TreeLds, NoTree>;
    constexpr int NT = D / M, KS = D / Sh::KC, DEEP = T::DEEP, C = T::COPIES, W = T::WAVES;
    __shared__ __attribute__((aligned(1024))) int8_t lds_all[T::LDS];
    __shared__ __attribute__((aligned(256))) int pages_all[W][2 * DEEP][64];  // pages of a block's keys
    __shared__ uint32_t slots_all[W][32];
    __shared__ Tree tree;
    const int lane = threadIdx.x & 63, i = lane & (M - 1), g = lane / M;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place at = place_of<TREE, false>(a, tiles);
    const int b = at.b, kvh = at.kvh, ctx = at.start;
    const int r = at.tile * M + i;
    const float* q_row = query_row<D>(a, r, b, kvh);
    RawQuery<D, M> raw_q = load_query<D, M>(q_row, g);
    if constexpr (TREE) grow_tree(tree, a.parents + (size_t)b * a.P, a.P, a.window);
    const Row row = row_of<TREE>(a, tree, r, b, kvh, at.start, at.len);
    const Limits lim = limits_of<TREE>(row, ctx);
    const int kbeg = min(lim.lo, lim.hi), kend = lim.hi;
    // this split's blocks, and this wave's: numbers wave, wave + W, ...
    const int all = (kend - kbeg + 127) / 128, per = (all + a.splits - 1) / a.splits;
    const int s0 = min(at.split * per, all), s1 = min(s0 + per, all);
    const int k0 = kbeg + s0 * 128, k1 = min(kbeg + s1 * 128, kend);
    const int n = ((k1 - k0 + 31) / 32 - wave + W - 1) / W;

    const int* table = a.pages.table + (size_t)b * a.pages.nbps;
    const size_t row_bytes = (size_t)a.H_kv * D * sizeof(KV);
    const int8_t* kbase = reinterpret_cast<const int8_t*>(static_cast<const KV*>(a.k) + (size_t)kvh * D);
    const int8_t* vbase = reinterpret_cast<const int8_t*>(static_cast<const KV*>(a.v) + (size_t)kvh * D);
    int8_t* const lds = lds_all + wave * T::WAVE;
    const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_i8)lds);
    const uint32_t pages_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_i8)(int8_t*)pages_all[wave]);
    uint32_t* const slots = slots_all[wave];
    auto first = [&](int j) { return k0 + 32 * (W * j + wave); };           // key of block j
    const Gaps gaps = gaps_of<M, TREE>(a, row, lim);
    auto pos_of = [&](int j) { return seen_at(gaps, row, min(first(j) + (lane & 31), k1 - 1)); };  // of this lane's key
    auto ask_pages = [&](int j) { copy4(table + page_of(a.pages, pos_of(j)), pages_at + (j & (2 * DEEP - 1)) * 256); };
    constexpr int RPC = 1024 / T::ROW;  // rows of a copy
    const int lane_row = lane / T::CH;
    auto col = [&](int j, bool v) {  // of this lane's 16 bytes in its row of copy j
        const int rr = lane_row + j * RPC;
        return 16 * ((lane % T::CH) ^ (v ? T::vswz(rr) : T::kswz(rr)));
    };
    // K of block j (its pages have come), and the pages of block j + DEEP
    auto ask_k = [&](int j) {
        const int p = pos_of(j), in = page_of(a.pages, p);
        const uint32_t page = (uint32_t)pages_all[wave][j & (2 * DEEP - 1)][lane & 31];
        slots[lane & 31] = page * (uint32_t)a.pages.block + (uint32_t)(p - in * a.pages.block);
        ask_pages(j + DEEP);
        lds_done();
#pragma unroll
        for (int c = 0; c < C; ++c)
            copy16(kbase + (slots[lane_row + c * RPC] * row_bytes + col(c, false)), lds_at + (j & (DEEP - 1)) * T::PART + c * 1024);
    };
    auto ask_v = [&](int j) {  // (after ask_k(j))
        lds_done();
#pragma unroll
        for (int c = 0; c < C; ++c)
            copy16(vbase + (slots[lane_row + c * RPC] * row_bytes + col(c, true)),
                   lds_at + (DEEP + (j & (DEEP - 1))) * T::PART + c * 1024);
    };

    if (n > 0) {
#pragma unroll
        for (int j = 0; j < DEEP; ++j) ask_pages(j);
    }
    // (the query is there before the copies start: the compiler's wait for it would be one for them)
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            asm volatile("" : "+v"(raw_q.x[s][k].x), "+v"(raw_q.x[s][k].y), "+v"(raw_q.x[s][k].z), "+v"(raw_q.x[s][k].w));
    const Scores sc = scores_of(a, row.head);
    const Cap cap = cap_of(a.cap);
    float slope = sc.slope;
    asm volatile("" : "+v"(slope));
    if (n > 0) {
        copies_left<0>();
        ask_k(0);
        ask_v(0);
        if (DEEP == 2 && n > 1) {
            ask_k(1);
            ask_v(1);
        }
    }
    Parts<3> q[KS];
    const bool q_bad = split_query<D, M>(q_row, raw_q, sc.q, q);
    State<D, M> st;
    st.clear();

#pragma unroll 1
    for (int j = 0; j < n; ++j) {
        // what may be under way while block j's K is read: V of j, and of j + 1 its successor's pages, K and V
        if (DEEP == 2 && j + 1 < n) copies_left<3 * C + 1>();
        else copies_left<C>();
        const int c0 = first(j);
        const int8_t* kp = lds + (j & (DEEP - 1)) * T::PART;
        const int8_t* vp = lds + (DEEP + (j & (DEEP - 1))) * T::PART;
        typename Sh::Acc sa[Sh::TILES] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            Parts<NP> x[Sh::TILES];
#pragma unroll
            for (int t = 0; t < Sh::TILES; ++t) {
                const int key = M * t + i;
                if constexpr (NP == 1) {
                    x[t].p[0] = *reinterpret_cast<const uint4*>(kp + key * T::ROW + 16 * ((Sh::KC / 8 * k + g) ^ T::kswz(key)));
                } else {
                    const int c = (Sh::KC / 4 * k + 2 * g) ^ T::kswz(key);
                    const float4 u = *reinterpret_cast<const float4*>(kp + key * T::ROW + 16 * c);
                    const float4 w = *reinterpret_cast<const float4*>(kp + key * T::ROW + 16 * (c + 1));
                    const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
                    x[t] = split8(y);
                }
            }
            product<NP, Sh::TILES>(x, q[k], sa);
        }
        if (j + DEEP < n) ask_k(j + DEEP);
        float p[Sh::NS];
#pragma unroll
        for (int v = 0; v < Sh::NS; ++v) p[v] = sa[v / Sh::AV][v % Sh::AV];
        weigh<D, M, TREE>(a, tree, row, lim, slope, cap, c0, ctx, p, st);
        // V of block j: behind it came K of j + DEEP and the pages behind that, and with two blocks under way the
        // same and V of j + 1
        if (j + DEEP < n) copies_left<DEEP == 2 ? 3 * C + 2 : C + 1>();
        else if (DEEP == 2 && j + 1 < n) copies_left<2 * C + 1>();
        else copies_left<0>();
#pragma unroll
        for (int k = 0; k < Sh::NS / 8; ++k) {
            const Parts<3> w = split8(p + 8 * k);
#pragma unroll
            for (int t0 = 0; t0 < NT; t0 += 2) {
                Parts<NP> x[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if constexpr (NP == 1) {
                        x[t].p[0] = read_v<T, M>(vp, 16 * k, t0 + t);
                    } else {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            y[e] = *reinterpret_cast<const float*>(vp + (16 * k + 4 * g + (e & 3) + Sh::STEP * (e >> 2)) * T::ROW +
                                                                   4 * (M * (t0 + t) + i));
                        x[t] = split8(y);
                    }
                }
                product<NP, 2>(x, w, st.o + t0);
            }
        }
        if (j + DEEP < n) ask_v(j + DEEP);
    }
    float l = Sh::rows_sum(st.l);
    copies_left<0>();
    __syncthreads();
    if (!gather<D, M, W - 1>(lds_all, wave, 1, 0, st, l)) return;
    finish<D, M, KV, TREE>(a, tree, row, b, kvh, ctx, at.split, k0, k1, q_bad, st, l);
}

// ---- the kernel for one row, or two of an fp32 cache: vector units
// At so few rows a matrix tile of 32 is mostly empty and its softmax costs as much as a full one's.  Here eight waves
// take the keys' batches in turn, in fp32 as they are: LPK lanes hold a key's row, 16 bytes each, so a copy
// brings KPI whole rows; a score is a lane's products summed over its LPK lanes, which then have the key's weight for
// their channels of V.  Each group of LPK lanes keeps its own unit, sum and output, joined at the end.  K and V come
// into LDS of the wave's own, 8 KiB each: the next batch's K while the weights are made, its V behind the products, its
// pages a batch earlier.  (Loaded into registers
// instead, four rows of 32 x 8 heads x 8192 x 128 bf16 took 450 us against 182: the loads' addresses and targets waited
// for one another's.)
template <int D, typename KV>
struct Lanes {
    static constexpr int E = 16 / (int)sizeof(KV);  // values a lane
    static constexpr int LPK = D / E;               // lanes a key
    static constexpr int KPI = 64 / LPK;            // keys a load
    static constexpr int U = 8;                     // copies of a batch's K or V
    static constexpr int PART = U * 1024;
    static constexpr int BK = U * KPI;              // its keys
};
// Sum over the N lanes that hold a key.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (N == 8) {
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, false));   // l ^ 1
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, false));   // l ^ 2
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xf, 0xf, false));  // 7 - l
        return v;
    } else if constexpr (N == 16) {
        return row16_sum(v);
    } else {
        return sum_xor16(row16_sum(v));
    }
}
// Over the groups of lanes that hold different keys.
template <int N>
__device__ __forceinline__ float groups_sum(float v) {
    if constexpr (N == 8) v += dpp_row_ror<8>(v);
    if constexpr (N <= 16) v = sum_xor16(v);
    return sum_xor32(v);
}
template <int N>
__device__ __forceinline__ float groups_max(float v) {
    if constexpr (N == 8) v = fmaxf(v, dpp_row_ror<8>(v));
    if constexpr (N <= 16) v = max_xor16(v);
    return max_xor32(v);
}
template <typename KV>
__device__ __forceinline__ void values(uint4 w, float (&x)[16 / sizeof(KV)]) {
    if constexpr (sizeof(KV) == 4) {
        x[0] = __builtin_bit_cast(float, w.x), x[1] = __builtin_bit_cast(float, w.y);
        x[2] = __builtin_bit_cast(float, w.z), x[3] = __builtin_bit_cast(float, w.w);
    } else {
        x[0] = low_of(w.x), x[1] = high_of(w.x), x[2] = low_of(w.y), x[3] = high_of(w.y);
        x[4] = low_of(w.z), x[5] = high_of(w.z), x[6] = low_of(w.w), x[7] = high_of(w.w);
    }
}

constexpr int kRowWaves = 8;
static_assert(64 * kRowWaves >= IE_TREE_MAX, "grow_tree has a thread a node");
template <int D, typename KV, int R, bool TREE>
__global__ __launch_bounds__(64 * kRowWaves, 2) void paged_row_kernel(PagedAttn a, int tiles) {
    using T = Lanes<D, KV>;
    using Tree = std::conditional_t<TREE, TreeLds, NoTree>;
    constexpr int E = T::E, U = T::U, W = kRowWaves;
    __shared__ Tree tree;
    __shared__ __attribute__((aligned(1024))) int8_t lds_all[W * 2 * T::PART];
    __shared__ __attribute__((aligned(256))) int pages_all[W][2][64];
    __shared__ uint32_t slots_all[W][64];
    __shared__ float sm_m[W][R], sm_l[W][R];
    static_assert(sizeof(lds_all) >= sizeof(float) * W * R * D, "the join");
    const int tid = threadIdx.x, lane = tid & 63, sub = lane % T::LPK, grp = lane / T::LPK;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at = place_of<TREE, false>(a, tiles);
    const int b = at.b, kvh = at.kvh, ctx = at.start;
    float q[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float* row = query_row<D>(a, at.tile * R + r, b, kvh) + E * sub;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(row + e);
            q[r][e] = x.x, q[r][e + 1] = x.y, q[r][e + 2] = x.z, q[r][e + 3] = x.w;
        }
    }
    if constexpr (TREE) grow_tree(tree, a.parents + (size_t)b * a.P, a.P, a.window);
    // a row's bounds in lane r, and in scalar registers
    const Row mine = row_of<TREE>(a, tree, at.tile * R + (lane & (R - 1)), b, kvh, at.start, at.len);
    const Limits lim = limits_of<TREE>(mine, ctx);
    Row rows[R];
    float slope[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        rows[r].t = __builtin_amdgcn_readlane(mine.t, r);
        rows[r].head = __builtin_amdgcn_readlane(mine.head, r);
        rows[r].lo = __builtin_amdgcn_readlane(mine.lo, r);
        rows[r].hi = __builtin_amdgcn_readlane(mine.hi, r);
        rows[r].pos = __builtin_amdgcn_readlane(mine.pos, r);
        slope[r] = slope_of(a, rows[r].head);
    }
    const int kbeg = min(lim.lo, lim.hi), kend = lim.hi;
    const int all = (kend - kbeg + 127) / 128, per = (all + a.splits - 1) / a.splits;
    const int s0 = min(at.split * per, all), s1 = min(s0 + per, all);
    const int k0 = kbeg + s0 * 128, k1 = min(kbeg + s1 * 128, kend);

    const int* table = a.pages.table + (size_t)b * a.pages.nbps;
    const size_t row_bytes = (size_t)a.H_kv * D * sizeof(KV);
    const int8_t* kbase = reinterpret_cast<const int8_t*>(static_cast<const KV*>(a.k) + (size_t)kvh * D) + 16 * sub;
    const int8_t* vbase = reinterpret_cast<const int8_t*>(static_cast<const KV*>(a.v) + (size_t)kvh * D) + 16 * sub;
    const Cap cap = cap_of(a.cap);
    const float factor = a.cap > 0.0f ? a.scale / a.cap : a.scale * kLog2e;

    float m[R], l[R], o[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = 0.0f;
    }
    // batch n of this wave: keys first(n) on
    auto first = [&](int n) { return k0 + T::BK * (W * n + wave); };
    const Gaps gaps = gaps_of<R, TREE>(a, mine, lim);
    auto pos_of = [&](int n) { return seen_at(gaps, mine, min(first(n) + (lane & (T::BK - 1)), k1 - 1)); };
    const int n1 = k1 > k0 ? ((k1 - k0 + T::BK - 1) / T::BK - wave + W - 1) / W : 0;
    int8_t* const lds = lds_all + wave * 2 * T::PART;
    const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_i8)lds);
    const uint32_t pages_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_i8)(int8_t*)pages_all[wave]);
    uint32_t* const slots = slots_all[wave];
    auto ask_pages = [&](int n) { copy4(table + page_of(a.pages, pos_of(n)), pages_at + (n & 1) * 256); };
    auto ask_k = [&](int n) {  // (its pages have come)
        const int p = pos_of(n);
        slots[lane] = (uint32_t)pages_all[wave][n & 1][lane] * (uint32_t)a.pages.block + (uint32_t)(p - page_of(a.pages, p) * a.pages.block);
        ask_pages(n + 1);
        lds_done();
#pragma unroll
        for (int u = 0; u < U; ++u) copy16(kbase + slots[u * T::KPI + grp] * row_bytes, lds_at + u * 1024);
    };
    auto ask_v = [&] {  // (after ask_k of the same batch)
        lds_done();
#pragma unroll
        for (int u = 0; u < U; ++u) copy16(vbase + slots[u * T::KPI + grp] * row_bytes, lds_at + T::PART + u * 1024);
    };
    if (n1 > 0) ask_pages(0);
#pragma unroll
    for (int r = 0; r < R; ++r) {  // (here before the copies start: a wait of the compiler's would be one for them)
        asm volatile("" : "+v"(slope[r]));
#pragma unroll
        for (int e = 0; e < E; ++e) asm volatile("" : "+v"(q[r][e]));
    }
    if (n1 > 0) {
        copies_left<0>();
        ask_k(0);
        ask_v();
    }
#pragma unroll 1
    for (int n = 0; n < n1; ++n) {
        const int c0 = first(n);
        float s[R][U];
        copies_left<U>();  // K of batch n; V of it may be under way
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[E];
            values<KV>(*reinterpret_cast<const uint4*>(lds + u * 1024 + 16 * lane), x);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d0 = q[r][0] * x[0], d1 = q[r][1] * x[1];
#pragma unroll
                for (int e = 2; e < E; e += 2) {
                    d0 = fmaf(q[r][e], x[e], d0);
                    d1 = fmaf(q[r][e + 1], x[e + 1], d1);
                }
                s[r][u] = lanes_sum<T::LPK>(d0 + d1) * factor;
            }
        }
        if (n + 1 < n1) ask_k(n + 1);
        const bool edge = c0 < lim.all_lo || c0 + T::BK > lim.all_hi;
        uint32_t seen[R];  // bit u: this lane's key of load u
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (a.cap > 0.0f) {
                float most = 0.0f;
#pragma unroll
                for (int u = 0; u < U; ++u) most = fmaxf(most, fabsf(s[r][u]));
                if (__ballot(!(most < 1.0f))) {
#pragma unroll
                    for (int u = 0; u < U; ++u) s[r][u] = capped(s[r][u], cap);
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u) s[r][u] = capped_small(s[r][u], cap);
                }
            }
            if (a.slopes) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    int j = c0 + u * T::KPI + grp;
                    if constexpr (TREE) j = j < ctx ? j : ctx + tree.depth[min(j - ctx, IE_TREE_MAX - 1)];
                    s[r][u] = fmaf(-slope[r], fabsf((float)(rows[r].pos - j)), s[r][u]);
                }
            }
            seen[r] = 0xffffffffu;
            if (edge) {
                seen[r] = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int j = c0 + u * T::KPI + grp;
                    bool in = j >= rows[r].lo && j < rows[r].hi;
                    if constexpr (TREE) {
                        const int x = min(max(j - ctx, 0), IE_TREE_MAX - 1);
                        if (j >= ctx) in = j < rows[r].hi && (tree.line[rows[r].t][x >> 5] >> (x & 31) & 1);
                    }
                    if (in) seen[r] |= 1u << u;
                    else s[r][u] = -INFINITY;
                }
            }
            float top = s[r][0];
#pragma unroll
            for (int u = 1; u < U; ++u) top = fmaxf(top, s[r][u]);
            if (__ballot(top > m[r] + 8.0f)) {  // (as weigh)
                const float mn = fmaxf(m[r], top), alpha = mn == -INFINITY ? 0.0f : exp2_sm(m[r] - mn);
                m[r] = mn;
                l[r] *= alpha;
#pragma unroll
                for (int e = 0; e < E; ++e) o[r][e] *= alpha;
            }
            const float mu = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[r][u] = exp2_sm(s[r][u] - mu);
                l[r] += s[r][u];
            }
        }
        if (n + 1 < n1) copies_left<U + 1>();  // V of batch n; behind it K of the next and the pages after that
        else copies_left<0>();
        const int8_t* vp = lds + T::PART + 16 * lane;
        if (edge) {  // (what a row does not see may be anything)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[E];
                values<KV>(*reinterpret_cast<const uint4*>(vp + u * 1024), x);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[r][e] = fmaf(s[r][u], seen[r] >> u & 1 ? x[e] : 0.0f, o[r][e]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[E];
                values<KV>(*reinterpret_cast<const uint4*>(vp + u * 1024), x);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[r][e] = fmaf(s[r][u], x[e], o[r][e]);
            }
        }
        if (n + 1 < n1) ask_v();
    }
    copies_left<0>();
    __syncthreads();  // (the waves' buffers serve the join)
    float (*sm_o)[R][D] = reinterpret_cast<float (*)[R][D]>(lds_all);
    // The wave's groups, then the waves.
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float mx = groups_max<T::LPK>(m[r]), f = mx == -INFINITY ? 0.0f : exp2_sm(m[r] - mx);
        const float sum = groups_sum<T::LPK>(l[r] * f);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = groups_sum<T::LPK>(o[r][e] * f);
        if (grp == 0) {
#pragma unroll
            for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(&sm_o[wave][r][E * sub + e]) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        }
        if (lane == 0) {
            sm_m[wave][r] = mx;
            sm_l[wave][r] = sum;
        }
    }
    __syncthreads();
    // The first wave: row r, channels c ..
    static_assert(R * D / 4 <= 64, "a wave has all rows' channels");
    if (wave > 0) return;
    const size_t total = (size_t)a.B * a.P * a.H_q;
    const int r = min(lane / (D / 4), R - 1), c = 4 * (lane % (D / 4));
    const Row row = row_of<TREE>(a, tree, at.tile * R + r, b, kvh, at.start, at.len);
    const bool on = lane < R * D / 4 && row.live;
    float mx = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) mx = fmaxf(mx, sm_m[w][r]);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float f = exp2_sm(sm_m[w][r] - mu);
        const float4 z = *reinterpret_cast<const float4*>(&sm_o[w][r][c]);
        sum = fmaf(f, sm_l[w][r], sum);
        y.x = fmaf(f, z.x, y.x), y.y = fmaf(f, z.y, y.y), y.z = fmaf(f, z.z, y.z), y.w = fmaf(f, z.w, y.w);
    }
    // A row that is not finite again by itself: weights of up to 2^8 may have taken sums of large values past fp32.
    const float bad = fmaf(sum, 0.0f, fmaf(y.x, 0.0f, fmaf(y.y, 0.0f, fmaf(y.z, 0.0f, y.w * 0.0f))));
    const uint64_t lanes = __ballot(on && !(bad == 0.0f));
    uint32_t again = 0;
#pragma unroll
    for (int x = 0; x < R; ++x)
        if (lanes >> (x * (D / 4)) & ((1ull << (D / 4)) - 1)) again |= 1u << x;
    if (on && !(again >> r & 1)) {
        const size_t to = ((size_t)b * a.P + row.t) * a.H_q + row.head;
        float* out = a.O + to * D;
        float inv = 1.0f;
        if (a.splits == 1) {
            inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        } else {
            out = a.ws + (at.split * total + to) * D;
            if (c == 0) *reinterpret_cast<float2*>(a.ws + a.splits * total * D + 2 * (at.split * total + to)) = make_float2(mx, sum);
        }
        *reinterpret_cast<float4*>(out + c) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    }
    exact_rows<D, KV, TREE>(a, tree, mine, again, b, kvh, ctx, at.split, k0, k1);
}

// O rows from their splits' partials: D / 4 lanes a row, SG times, each of which has every SG-th split; four splits'
// loads are under way at once, and with SG = 8 (more than four splits) the eight's sums meet in LDS (one sequence of
// 16000 keys, 8 x 4 x 128 in 16 splits: 31.0 us in all with a row's splits one after another, 20.3 so).
template <int D, int SG>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn a) {
    static_assert(IE_PAGED_MAX_SPLITS <= 128, "a row's parts and their rounding within 2^8");
    constexpr int L = D / 4, PER = 256 / (L * SG);
    const size_t rows = (size_t)a.B * a.P * a.H_q;
    const int c = threadIdx.x % L, sg = threadIdx.x / L % SG, local = threadIdx.x / (L * SG);
    const size_t r = (size_t)blockIdx.x * PER + local;
    const bool live = r < rows && !(a.lens && (int)(r / a.H_q % a.P) >= a.lens[r / a.H_q / a.P]);
    const float2* ml = reinterpret_cast<const float2*>(a.ws + a.splits * rows * D);
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // Parts count times 2^-8: as many as there can be, each finite, stay so together.
    auto add = [&](float xm, float xl, float4 y, float times) {  // (an empty part has xm = -inf, xl = 0 and no y)
        const float mn = fmaxf(m, xm), mu = mn == -INFINITY ? 0.0f : mn;
        const float fa = exp2_sm(m - mu), fb = exp2_sm(xm - mu) * times;
        m = mn;
        l = l * fa + xl * fb;
        o.x = o.x * fa + y.x * fb;
        o.y = o.y * fa + y.y * fb;
        o.z = o.z * fa + y.z * fb;
        o.w = o.w * fa + y.w * fb;
    };
    if (live) {
        for (int s0 = sg; s0 < a.splits; s0 += 4 * SG) {
            float2 x[4];
            float4 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int s = s0 + k * SG;
                x[k] = make_float2(-INFINITY, 0.0f);
                y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (s < a.splits) {
                    x[k] = ml[s * rows + r];
                    y[k] = reinterpret_cast<const float4*>(a.ws + (s * rows + r) * D)[c];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) add(x[k].x, x[k].y, y[k], 0x1p-8f);
        }
    }
    if constexpr (SG > 1) {
        __shared__ float4 so[256];
        __shared__ float2 sm[256];
        so[threadIdx.x] = o;
        sm[threadIdx.x] = make_float2(m, l);
        __syncthreads();
        if (sg > 0) return;
#pragma unroll
        for (int k = 1; k < SG; ++k) {
            const float2 x = sm[threadIdx.x + k * L];
            add(x.x, x.y, so[threadIdx.x + k * L], 1.0f);
        }
    }
    if (!live) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    reinterpret_cast<float4*>(a.O + r * D)[c] = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <int D, int NP, int ROWS, bool TREE, int WK = ROWS == 64 ? 2 : 1>
void launch_tile(const PagedAttn& a, hipStream_t s) {
    const int G = a.H_q / a.H_kv, tiles = (int)(((long long)a.P * G + ROWS - 1) / ROWS);
    const unsigned grid = (unsigned)((long long)a.B * a.H_kv * tiles * a.splits);
    using KV = std::conditional_t<NP == 1, uint16_t, float>;
    if constexpr (ROWS <= 2) paged_row_kernel<D, KV, ROWS, TREE><<<grid, 64 * kRowWaves, 0, s>>>(a, tiles);
    else if constexpr (ROWS <= 32) paged_few_kernel<D, NP, ROWS, TREE><<<grid, 64 * Few<D, NP, ROWS>::WAVES, 0, s>>>(a, tiles);
    else paged_tile_kernel<D, NP, ROWS / 32, WK, TREE><<<grid, 2 * ROWS * WK, 0, s>>>(a, tiles);
}

template <int D, int NP, bool TREE>
void launch_rows(const PagedAttn& a, hipStream_t s) {
    const PagedPlan p = paged_plan(a.B, a.P, a.H_q, a.H_kv, a.d, a.kv_dtype, a.parents ? a.max_ctx + a.P : a.max_ctx, a.window, a.splits);
    if (p.rows == 1) return launch_tile<D, NP, 1, TREE>(a, s);
    if constexpr (NP == 3) {
        if (p.rows == 2) return launch_tile<D, NP, 2, TREE>(a, s);
    } else {
        if (p.groups == 2) return launch_tile<D, NP, 128, TREE, 2>(a, s);
    }
    if (p.rows == 16) return launch_tile<D, NP, 16, TREE>(a, s);
    if (p.rows == 32) return launch_tile<D, NP, 32, TREE>(a, s);
    if (p.rows == 64) return launch_tile<D, NP, 64, TREE>(a, s);
    launch_tile<D, NP, 128, TREE>(a, s);
}

template <int D, int NP>
void launch_np(const PagedAttn& a, hipStream_t s) {
    if (a.parents) launch_rows<D, NP, true>(a, s);
    else launch_rows<D, NP, false>(a, s);
}

template <int D>
void launch_d(const PagedAttn& a, hipStream_t s) {
    if (a.kv_dtype == IE_KV_BF16) launch_np<D, 1>(a, s);
    else launch_np<D, 3>(a, s);
    if (a.splits > 1) {
        const long long rows = (long long)a.B * a.P * a.H_q;
        constexpr int per = 256 / (D / 4);  // rows of a workgroup, or an eighth of them
        // (with very many rows, whose grid of eighths would pass 2^32 threads, a row's splits have one group of lanes)
        if (a.splits <= 4 || rows > 1 << 20) paged_merge_kernel<D, 1><<<(unsigned)((rows + per - 1) / per), 256, 0, s>>>(a);
        else paged_merge_kernel<D, 8><<<(unsigned)((rows * 8 + per - 1) / per), 256, 0, s>>>(a);
    }
}

}  // namespace

int paged_attn_splits(int B, int P, int H_q, int H_kv, int d, int kv_dtype, int max_keys, int window, int asked) {
    return paged_plan(B, P, H_q, H_kv, d, kv_dtype, max_keys, window, asked).splits;
}

void launch_paged_attn(const PagedAttn& a, hipStream_t s) {
    if (a.d == 64) launch_d<64>(a, s);
    else launch_d<128>(a, s);
}

}  // namespace ie
