// kv8_prefill.hip — causal attention of a prompt chunk over the 8-bit paged KV
// cache (include/ie_kv8.h) on the half-precision matrix cores.
//
// Mathematics.  As kv8_decode.hip: o = sum_j w_j v_j / sum_j p_j, p_j =
// 2^(s_j - m), w_j = p_j vs_j over codes k_j, v_j.  A code is a half-precision
// number; the fp32 operands, a query row scaled to [2^14, 2^15) and the weights,
// are two of them each, x = hi + lo, 22 bits and more, with products summed in
// fp32 (v_mfma_f32_16x16x32_f16):
//   S^T = K q^T   A = 16 keys x 32 channels, B = 16 query rows
//   O^T = V^T w^T A = 16 channels x 32 keys, B = the same rows' weights
// A tile is 64 keys, four 16-token groups.  Row 4 q + r of product t of S^T is
// key 16 q + 4 t + r, so a lane receives the scores of 16 keys of one group
// (whose page has one scale) and one row, and they are, in order, its B
// operand's keys of the second product: no value crosses lanes between the two.
// A row of the kernel is (token, query head of the KV head), token-major: the
// heads that share K and V share its staging.
//
// The running maximum m and the weights' unit move only when a weight would
// pass the unit (set to 8 times the largest of a tile), or a scale 2^126 units
// (which costs 4 x 512 x 12 x 64 12.5 -> 12.7 us, and without which it is infinite where its
// weight is not); then the output is rescaled.  Weights more than 29 powers of two
// below the unit lose bits.
//
// Two forms.  block: four waves of 16 NC rows each walk the tiles together;
// wave w brings group w of the next tile (global bytes in registers during the
// current one, then converted into the other half of LDS), one barrier a tile;
// of two such teams each takes every other tile and they merge at the end.
// split: the rows of a workgroup are 16, its waves take every NW-th tile of its
// part of the context on their own, straight from the cache, and merge in LDS in
// wave order.  Either takes a context in parts, joined in a second launch.
//
// The block form is bound by the matrix cores and the vector units together: 1 x
// 4096 x (8 x 4) x 128 230 us on one card, 261 on a slower one: 597 and 526 TFLOP/s
// of attention, twice that of half-precision products (a large library product in
// bf16 reaches 1108 to 1121), matrix cores busy 48%, vector units 46% of the 230.
// Two waves share a SIMD there, and with the one that has its scores put first
// (s_setprio) from the weights to the end of the second product the two take turns,
// one with each unit: without, 264 and 283 us.  (With four waves a SIMD, d = 64, it costs 3%, and is left out.)  Where a
// launch puts two blocks on some CUs, the shortest go beside the longest: 1 x 2048 x
// (8 x 4) x 128 96 -> 91 us, 4 x 640 x 12 x 64 15.6 -> 14.1.  With one tile in flight
// or two it is the same, so not by memory.  The split form is bound by its conversions
// of K and V (320 of 606 vector instructions a tile at d = 128).
#include <algorithm>
#include <cmath>

#include "device_util.h"
#include "kv8.h"

namespace ie {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __fp16 fp16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;  // keys
constexpr int NW = 4;      // waves of the split form's workgroup

// Four codes as half-precision numbers: the byte plus 128 in the low bits of
// 1024.0's pattern is 1024 + byte + 128, exactly.
__device__ __forceinline__ void halves(uint32_t w, uint32_t& a, uint32_t& b) {
    const uint32_t u = w ^ 0x80808080u;
    const half2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
    b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
}
// Eight codes (two words) as an operand.
__device__ __forceinline__ u32x4 halves8(uint32_t w0, uint32_t w1) {
    u32x4 r;
    uint32_t a, b;
    halves(w0, a, b);
    r[0] = a; r[1] = b;
    halves(w1, a, b);
    r[2] = a; r[3] = b;
    return r;
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// One lane's share of 16 query rows: row lane & 15, channels [8 (lane / 16), + 8)
// of each 32 (ORDER 0), or 16 (lane / 16) + 8 (s & 1) of each 64 (ORDER 1: the
// order in which 16-byte words of a cache row come).
template <int D, int ORDER>
struct Query {
    u32x4 hi[D / 32], lo[D / 32];
    float scale;  // of the products with codes, log2(e) / sqrt(d) included; NaN for a row that is not finite
    int lim;      // keys that the row sees

    __device__ __forceinline__ void load(const Kv8Attn& a, int b, int h, int G, int row, float qscale) {
        const int lane = threadIdx.x & 63, kg = lane >> 4;
        const int t = row / G, g = row - t * G;
        lim = a.start + t + 1;
        const float* p = a.Q + ((size_t)b * a.P + t) * a.q_ld + ((size_t)h * G + g) * D;
        float x[D / 32][8];
        uint32_t mx = 0;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const float4* p4 = reinterpret_cast<const float4*>(p + (ORDER == 0 ? 32 * s + 8 * kg : 64 * (s / 2) + 16 * kg + 8 * (s & 1)));
            const float4 u = p4[0], v = p4[1];
            x[s][0] = u.x; x[s][1] = u.y; x[s][2] = u.z; x[s][3] = u.w;
            x[s][4] = v.x; x[s][5] = v.y; x[s][6] = v.z; x[s][7] = v.w;
        }
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = max(mx, __builtin_bit_cast(uint32_t, x[s][e]) & 0x7fffffffu);
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
        const int e = max((int)(mx >> 23), 15);  // both factors stay normal numbers
        const float up = pow2(min(268 - e, 253));
        scale = e == 255 ? __builtin_nanf("") : pow2(max(e - 14, 1)) * qscale;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            half8_t vh, vl;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[s][i] * up;
                vh[i] = (_Float16)y;
                vl[i] = (_Float16)(y - (float)vh[i]);
            }
            hi[s] = __builtin_bit_cast(u32x4, vh);
            lo[s] = __builtin_bit_cast(u32x4, vl);
        }
    }
};

template <int D>
struct State {
    float m, l;
    int ub;  // biased exponent of the weights' unit: o is in units
    f32x4 o[D / 16];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
        ub = 127;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
};

// Scores (products with codes) of one tile to weights: the lane's 16 keys as
// the two halves of its operand.  key0: the first of them; edge (uniform): some
// row of the wave does not see all 64 keys.
template <int D>
__device__ __forceinline__ void weights(const f32x4 (&acc)[4], float sw, float vscale, int key0, int lim, bool edge,
                                        State<D>& st, u32x4 (&hi)[2], u32x4 (&lo)[2]) {
    float top;
    if (edge) {
        asm volatile("");  // a branch, not selects in every tile
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (key0 + i < lim) top = max_of(top, acc[i >> 2][i & 3]);
    } else {
        top = acc[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = max_of(top, acc[i >> 2][i & 3]);
    }
    top = top == -INFINITY ? top : top * sw;
    // log2 of the lane's largest weight, rounded up, against m; and a scale has to be a
    // number of units that fp32 holds (so as if no weight were less than 2^-111 of it)
    float vexp = (float)(biased_exp(vscale) - 126);
    const float ahead = top - st.m;
    bool moved = fmaxf(fmaxf(ahead, -111.0f) + (vexp - (float)(st.ub - 127)), ahead - 70.0f) > 15.0f;
    if (__ballot(moved) != 0) {  // uniform
        if (key0 >= lim) {  // (a page that the row sees nothing of)
            moved = false;
            vexp = -126.0f;
        }
        moved = max_xor32(max_xor16(moved ? 1.0f : 0.0f)) > 0.0f;  // over the row
        const float rtop = max_xor32(max_xor16(top));
        const float mn = moved ? fmaxf(st.m, rtop) : st.m;
        const float f = moved ? exp2_sm(st.m - mn) : 1.0f;
        const float wm = max_xor32(max_xor16(top - mn + vexp));
        // 8 times the tile's largest weight, not below the unit that the output has so far
        // (which may be of far larger values: o moves by at most a factor of 2), and not
        // below 2^-126 of the tile's largest scale (of which no weight is less)
        const float most = max_xor32(max_xor16(vexp));
        const float unit = fmaxf(fmaxf(ceilf(wm) + (127.0f + 3.0f - 15.0f), ceilf((float)st.ub + (st.m - mn))), most + 1.0f);
        const int ub = moved ? (int)fminf(fmaxf(unit, 1.0f), 224.0f) : st.ub;
        const float fo = f * pow2(127 + min(max(st.ub - ub, -126), 127));
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st.o[j] *= fo;
        st.l *= f;
        st.m = mn;
        st.ub = ub;
    }
    const float m = st.m;
    float wc = vscale * pow2(254 - st.ub);
    float p[16], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = exp2_sm(fmaf(acc[i >> 2][i & 3], sw, -m));
    if (edge) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = key0 + i < lim ? p[i] : 0.0f;
        wc = key0 < lim ? wc : 0.0f;  // (a page that the row sees nothing of may have a scale that is not finite)
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        sum += p[i];
        sum += p[i + 1];
        const float w0 = p[i] * wc, w1 = p[i + 1] * wc;
        const fp16x2_t h = __builtin_amdgcn_cvt_pkrtz(w0, w1);
        hi[i / 8][i / 2 % 4] = __builtin_bit_cast(uint32_t, h);
        lo[i / 8][i / 2 % 4] = __builtin_bit_cast(
            uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], -1.0f, w0), fmaf((float)h[1], -1.0f, w1)));
    }
    st.l += sum;
}

// Where a 16-byte word of K lies in LDS: (32-channel step s, 8-channel part kg)
// rows of 64 keys by (t, m = 4 q + r), m exchanged so that neither the staging's
// writes (m & 3 and the channel vary) nor the products' reads (m varies) meet in
// a bank.
__device__ __forceinline__ int k_word(int s, int kg, int t, int m) {
    return (s * 4 + kg) * 64 + t * 16 + (m ^ (((t ^ (2 * s + (kg >> 1))) & 3) << 2));
}

// blockIdx.x = (row blocks, last first) * (B * H) + (sequence, KV head), but see
// below; CUT: that * splits + split, and partial results to the workspace.
template <int D, int NC, int TM, bool CUT>
__global__ __launch_bounds__(256 * TM, D == 64 ? 4 : 2) void kv8_prefill_block_kernel(Kv8Attn a, int blocks, float qscale) {
    constexpr int S = D / 32, J = D / 16, CH = D / 64, ROWS = 64 * NC;
    // the teams' halves of K and V; at the end the other teams' outputs
    __shared__ u32x4 sh_kv[TM][2][2][8 * D];
    __shared__ float2 sh_s[TM][2][4];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int team = TM == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int H = a.c.H, G = a.H_q / H;
    const int splits = CUT ? a.splits : 1, split = CUT ? (int)(blockIdx.x % (unsigned)splits) : 0;
    unsigned id = CUT ? blockIdx.x / (unsigned)splits : blockIdx.x;
    if constexpr (!CUT && (D == 64 || NC == 2)) {
        // Two workgroups fit a CU: where those from 256 on are second ones of a CU, the
        // shortest of them join the longest of the first.  (Bits 0 to 2, the XCD, stay.)
        const unsigned full = gridDim.x & ~7u;
        if (gridDim.x <= 512 && id >= 256 && id < full) id = 256 + full - 8 - (id & ~7u) + (id & 7u);
    }
    const unsigned bh = id % (unsigned)(a.B * H);
    const int blk = blocks - 1 - (int)(id / (unsigned)(a.B * H));
    const int h = (int)(bh % (unsigned)H), b = (int)(bh / (unsigned)H);
    const int rows = a.P * G, row0 = blk * ROWS;
    const int n = a.start + min(row0 + ROWS - 1, rows - 1) / G + 1;  // keys that the block sees
    const int all = (n + kTile - 1) / kTile, last = (n - 1) >> 4;
    const int t0 = CUT ? (int)((unsigned)all * split / (unsigned)splits) : 0;
    const int tiles = CUT ? (int)((unsigned)all * (split + 1) / (unsigned)splits) : all;  // (the end of this part)
    const int lgg = a.c.bs_log2 - 4, gmask = (1 << lgg) - 1;
    const int* table = a.c.table + (size_t)b * a.c.nbps;

    // group wid of a tile: its words in registers, its page's scales
    u32x4 kr[CH], vr[CH];
    float ks, vs;
    auto entry = [&](int tile) { return table[min(4 * tile + wid, last) >> lgg]; };
    auto fetch = [&](int tile, int page) {
        const size_t pair = (size_t)page * H + h;
        const size_t at = ((pair << lgg) + (min(4 * tile + wid, last) & gmask)) * (16 * D) + lane * 16;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            kr[i] = *reinterpret_cast<const u32x4*>(a.c.k + at + i * 1024);
            vr[i] = *reinterpret_cast<const u32x4*>(a.c.v + at + i * 1024);
        }
        ks = a.c.ks[pair];
        vs = a.c.vs[pair];
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = lane + 64 * i, key = id / (D / 16), c = id % (D / 16);
            const int s = c >> 1, kg = (c & 1) * 2, t = key >> 2, m = 4 * wid + (key & 3);
            sh_kv[team][buf][0][k_word(s, kg, t, m)] = halves8(kr[i][0], kr[i][1]);
            sh_kv[team][buf][0][k_word(s, kg + 1, t, m)] = halves8(kr[i][2], kr[i][3]);
            sh_kv[team][buf][1][(2 * wid) * D + id] = halves8(vr[i][0], vr[i][1]);
            sh_kv[team][buf][1][(2 * wid + 1) * D + id] = halves8(vr[i][2], vr[i][3]);
        }
        // a scale that is not finite makes every score of its page NaN
        if (lane == 0) sh_s[team][buf][wid] = make_float2(ks + ((ks - ks) + (vs - vs)), vs);
    };
    // the i-th tile of this team (past the last one: the last again)
    auto nth = [&](int i) { return max(min(t0 + team + i * TM, tiles - 1), 0); };
    int page = entry(nth(0));
    fetch(nth(0), page);
    page = entry(nth(1));

    const int wrow = row0 + wid * 16 * NC;  // the wave's first row
    Query<D, 0> q[NC];
    State<D> st[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        q[c].load(a, b, h, G, min(wrow + 16 * c + (lane & 15), rows - 1), qscale);
        st[c].clear();
    }
    const int wmin = a.start + min(wrow, rows - 1) / G + 1, wmax = a.start + min(wrow + 16 * NC - 1, rows - 1) / G + 1;
    const bool any = wrow < rows;
    const int q4 = lane >> 4, m16 = lane & 15;
    stage(0);
    __syncthreads();
    const int rounds = (tiles - t0 + TM - 1) / TM;  // (every wave makes every round: the barriers are the workgroup's)
    for (int i = 0; i < rounds; ++i) {
        const int tile = t0 + team + i * TM, buf = i & 1;
        if (i + 1 < rounds) {
            fetch(nth(i + 1), page);
            page = entry(nth(i + 2));
        }
        if (any && tile < tiles && tile * kTile < wmax) {  // uniform over the wave
            f32x4 acc[NC][4];
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                u32x4 k[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) k[t] = sh_kv[team][buf][0][k_word(s, q4, t, m16)];
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[c][t] = mfma(k[t], q[c].lo[s], acc[c][t]);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[c][t] = mfma(k[t], q[c].hi[s], acc[c][t]);
            }
            if (NC == 2) __builtin_amdgcn_s_setprio(1);
            const float2 sc = sh_s[team][buf][q4];
            const bool edge = (tile + 1) * kTile > wmin;
            u32x4 hi[NC][2], lo[NC][2];
#pragma unroll
            for (int c = 0; c < NC; ++c)
                weights<D>(acc[c], q[c].scale * sc.x, sc.y, tile * kTile + 16 * q4, q[c].lim, edge, st[c], hi[c], lo[c]);
            if (NC == 2) __builtin_amdgcn_s_setprio(1);  // (again: nothing is moved across; without it 243.2 against 241.4 us)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                u32x4 v[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) v[u] = sh_kv[team][buf][1][(2 * q4 + u) * D + 16 * j + m16];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int c = 0; c < NC; ++c) st[c].o[j] = mfma(v[u], lo[c][u], st[c].o[j]);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int c = 0; c < NC; ++c) st[c].o[j] = mfma(v[u], hi[c][u], st[c].o[j]);
            }
            if (NC == 2) __builtin_amdgcn_s_setprio(0);
        }
        if (i + 1 < rounds) stage(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) st[c].l = sum_xor32(sum_xor16(st[c].l));
    if constexpr (TM == 2) {  // team 1's sums join team 0's
        float4* sh = reinterpret_cast<float4*>(sh_kv) + (size_t)wid * NC * (J + 1) * 64 + lane;
        if (team == 1) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    sh[(c * (J + 1) + j) * 64] = make_float4(st[c].o[j][0], st[c].o[j][1], st[c].o[j][2], st[c].o[j][3]);
                sh[(c * (J + 1) + J) * 64] = make_float4(st[c].m, st[c].l, pow2(st[c].ub), 0.f);
            }
        }
        __syncthreads();
        if (team == 1) return;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float4 other = sh[(c * (J + 1) + J) * 64];
            const float mm = fmaxf(st[c].m, other.x);
            // a team without keys (m = -inf, o = l = 0) counts for nothing; NaN stays
            const float f0 = st[c].l == 0.0f ? 0.0f : exp2_sm(st[c].m - mm), f1 = other.y == 0.0f ? 0.0f : exp2_sm(other.x - mm);
            st[c].l = st[c].l * f0 + other.y * f1;
            const float u0 = f0 * pow2(st[c].ub), u1 = f1 * other.z;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float4 o = sh[(c * (J + 1) + j) * 64];
                st[c].o[j] = st[c].o[j] * u0 + f32x4{o.x, o.y, o.z, o.w} * u1;
            }
            st[c].ub = 127;
            st[c].m = mm;
        }
    }
    if constexpr (CUT) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int row = wrow + 16 * c + m16;
            if (row < rows) {
                const float f = pow2(st[c].ub);
                float* out = a.ws + ((((size_t)b * a.P + row / G) * a.H_q + (size_t)h * G + row % G) * splits + split) * (D + 2);
#pragma unroll
                for (int j = 0; j < J; ++j) {  // (8-byte aligned)
                    *reinterpret_cast<float2*>(out + 16 * j + 4 * q4) = make_float2(st[c].o[j][0] * f, st[c].o[j][1] * f);
                    *reinterpret_cast<float2*>(out + 16 * j + 4 * q4 + 2) = make_float2(st[c].o[j][2] * f, st[c].o[j][3] * f);
                }
                if (q4 == 0) *reinterpret_cast<float2*>(out + D) = make_float2(st[c].m, st[c].l);
            }
        }
        return;
    }
    // lane: row lane & 15 of each 16, channels 16 j + 4 q4 + r
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int row = wrow + 16 * c + m16;
        if (row < rows) {
            const float f = pow2(st[c].ub) / st[c].l;
            float* out = a.O + (((size_t)b * a.P + row / G) * a.H_q + (size_t)h * G + row % G) * D + 4 * q4;
#pragma unroll
            for (int j = 0; j < J; ++j)
                *reinterpret_cast<float4*>(out + 16 * j) =
                    make_float4(st[c].o[j][0] * f, st[c].o[j][1] * f, st[c].o[j][2] * f, st[c].o[j][3] * f);
        }
    }
}

// blockIdx.x = ((row blocks of 16, last first) * (B * H) + (sequence, KV head)) * splits + split
template <int D>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : 2) void kv8_prefill_split_kernel(Kv8Attn a, int blocks, float qscale) {
    constexpr int S = D / 32, J = D / 16, KB = D / 64;
    __shared__ float sh_o[NW][16][D];
    __shared__ float sh_m[NW][16], sh_l[NW][16];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int H = a.c.H, G = a.H_q / H;
    const int split = (int)(blockIdx.x % (unsigned)a.splits);
    const unsigned id = blockIdx.x / (unsigned)a.splits, bh = id % (unsigned)(a.B * H);
    const int blk = blocks - 1 - (int)(id / (unsigned)(a.B * H));
    const int h = (int)(bh % (unsigned)H), b = (int)(bh / (unsigned)H);
    const int rows = a.P * G, row0 = blk * 16;
    const int n = a.start + min(row0 + 15, rows - 1) / G + 1;  // keys that the block sees
    const int nmin = a.start + row0 / G + 1;
    const int tiles = (n + kTile - 1) / kTile, last = (n - 1) >> 4;
    const int lgg = a.c.bs_log2 - 4, gmask = (1 << lgg) - 1;
    const int* table = a.c.table + (size_t)b * a.c.nbps;
    const int q4 = lane >> 4, m16 = lane & 15, gk = m16 >> 2;

    State<D> st;
    st.clear();
    const int t0 = (int)((unsigned)tiles * split / (unsigned)a.splits), t1 = (int)((unsigned)tiles * (split + 1) / (unsigned)a.splits);
    int tile = t0 + wid;
    if (tile < t1) {  // uniform over the wave
        u32x4 kw[4][KB], vw[J];
        float ks, vs;
        auto entry = [&](int t, int g) { return table[min(4 * t + g, last) >> lgg]; };
        int pk = entry(tile, gk), pv = entry(tile, q4);
        Query<D, 1> q;
        q.load(a, b, h, G, min(row0 + m16, rows - 1), qscale);
        size_t at_k, at_v, at_s;
        auto place = [&](int t) {
            const size_t pairk = (size_t)pk * H + h, pairv = (size_t)pv * H + h;
            at_k = ((pairk << lgg) + (min(4 * t + gk, last) & gmask)) * (16 * D) + (m16 & 3) * D + q4 * 16;
            at_v = ((pairv << lgg) + (min(4 * t + q4, last) & gmask)) * (16 * D) + m16 * 16;
            at_s = pairv;
        };
        auto load_k = [&]() {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    kw[t][kb] = *reinterpret_cast<const u32x4*>(a.c.k + at_k + t * 4 * D + kb * 64);
            ks = a.c.ks[at_s];
            vs = a.c.vs[at_s];
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < J; ++j) vw[j] = *reinterpret_cast<const u32x4*>(a.c.v + at_v + j * 256);
        };
        place(tile);
        load_k();
        load_v();
        int next = min(tile + NW, t1 - 1);
        pk = entry(next, gk);
        pv = entry(next, q4);
        for (;;) {
            f32x4 acc[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const u32x4 k = halves8(kw[t][s / 2][2 * (s & 1)], kw[t][s / 2][2 * (s & 1) + 1]);
                    acc[t] = mfma(k, q.lo[s], acc[t]);
                    acc[t] = mfma(k, q.hi[s], acc[t]);
                }
            const float kscale = ks + ((ks - ks) + (vs - vs)), vscale = vs;
            place(next);
            load_k();
            next = min(tile + 2 * NW, t1 - 1);
            pk = entry(next, gk);
            pv = entry(next, q4);
            u32x4 hi[2], lo[2];
            weights<D>(acc, q.scale * kscale, vscale, tile * kTile + 16 * q4, q.lim, (tile + 1) * kTile > nmin, st, hi, lo);
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x4 v = halves8(vw[j][2 * u], vw[j][2 * u + 1]);
                    st.o[j] = mfma(v, lo[u], st.o[j]);
                    st.o[j] = mfma(v, hi[u], st.o[j]);
                }
            load_v();
            tile += NW;
            if (tile >= t1) break;
        }
    }
    const float unit = pow2(st.ub);
#pragma unroll
    for (int j = 0; j < J; ++j)
        *reinterpret_cast<float4*>(&sh_o[wid][m16][16 * j + 4 * q4]) =
            make_float4(st.o[j][0] * unit, st.o[j][1] * unit, st.o[j][2] * unit, st.o[j][3] * unit);
    const float lt = sum_xor32(sum_xor16(st.l));
    if (q4 == 0) {
        sh_m[wid][m16] = st.m;
        sh_l[wid][m16] = lt;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * D; i += 64 * NW) {
        const int r = i / D, dim = i % D, row = row0 + r;
        if (row >= rows) break;
        float mm = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sh_m[w][r]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float lw = sh_l[w][r], f = lw == 0.0f ? 0.0f : exp2_sm(sh_m[w][r] - mm);  // a wave without keys; NaN stays
            l = fmaf(lw, f, l);
            o = fmaf(sh_o[w][r][dim], f, o);
        }
        const size_t at = ((size_t)b * a.P + row / G) * a.H_q + (size_t)h * G + row % G;
        if (a.splits == 1) {
            a.O[at * D + dim] = o / l;
        } else {
            float* ws = a.ws + (at * a.splits + split) * (D + 2);
            ws[dim] = o;
            if (dim == 0) {
                ws[D] = mm;
                ws[D + 1] = l;
            }
        }
    }
}

int row_blocks(int P, int G, int rows) { return (int)(((long long)P * G + rows - 1) / rows); }

// The form of a call and the parts of its contexts.  A row is a token x query head
// of a KV head; g16, g64, g128 are the workgroups of that many rows.
//
// Contexts in one piece:
//   Up to 32 rows a KV head leave most of the block form's without work: 64 x 4 x 16
//     x 128 behind 1000 41.9 us in the split form against 101, 16 x 8 x (16 x 4) x 128
//     (32 rows) 24.3 against 26.3; 48 rows 34.3 against 27.6.
//   Below g64 = 128 the block form leaves CUs idle, and the split form's 16-row
//     workgroups fill them: 1 x 512 x 12 x 64 (96) 7.9 against 10.2 us.  From 128 the
//     split form has several a CU, which cost more than the block form's walk where
//     that is short: 1 x 384 x (8 x 4) x 128 (192, 6 tiles) 20.5 against 13.2, 2 x 640
//     x 12 x 64 (240, 10 tiles) 13.6 against 12.7, but 2 x 512 x 8 x 128 (128, 8
//     tiles) 13.9 against 15.4, 1 x 1536 x 8 x 128 (192, 24 tiles) 28.6 against 34.
//     From 256 the block form is ahead: 2 x 256 x (8 x 4) x 128 (256) 22 against 12.3.
//   Below 1024 two teams of four waves share a block's tiles: 4 x 512 x 12 x 64 (384)
//     12.8 against 16.2 us on one team; from there on one team: 4 x 1000 x (8 x 4) x
//     64 (2016) 52.5 against 60.3 us, and at d = 128 with 32 rows a wave, which read K
//     and V from LDS half as often: 1 x 4096 x (8 x 4) x 128 264 against 314 us (at d
//     = 64 57 against 52.5).
//
// Cut contexts (their parts joined by a second launch):
//   The split form up to g16 = 128, for about a workgroup a CU: 1 x 16 x (8 x 4) x 128
//     behind 4000 13.0 us against 29 in one piece.
//   Up to 208 (the split form uncut leaves CUs idle, and cut has some with two): two
//     teams, a block a CU (two at d = 64): 1 x 77 x (8 x 4) x 128 behind 4001 (160) 26.2
//     in six parts against 29.8, at d = 64 17.6 against 19.8.
//   From 256 on, behind a context of the chunk's length at least and for parts of 8
//     to 10 tiles or more.  d = 128: 32 rows a wave, two blocks a CU: 1 x 300 x (8 x 4)
//     behind 4000 55.2 in six parts against 74.7 uncut, 1 x 512 77.8 against 85.7, 1 x
//     1000 behind 8000 245 against 316 (behind 1000, 1 x 512 in four parts 39.7 against
//     35.1); with more blocks than 256 two rounds of them: 1 x 1200 behind 4000 183
//     against 253, 1 x 8192 x 8 behind none 254 against 332.  Where those parts would
//     be too short, two teams: 1 x 150 behind 4000 36.6 against 50.3.  d = 64: two teams
//     for at least four parts, 1 x 512 x 12 behind 4000 29.7 against 34.1, else one: 1
//     x 1500 x 12 behind 4000 74.8 against 94.9, 1 x 400 x (8 x 4) 47.5 against 57.7.
//   Left in one piece, and not measured cut: 209 to 256, and lengths for which the
//     fixed number of parts above would give parts that are too short, though fewer
//     parts would not (8 x 4 heads behind 4000: 105 to 144 tokens at d = 64, 105 to 128
//     at d = 128).
enum Form { kRows16, kTwoTeams, kOneTeam };
struct Plan {
    Form form;
    int splits;
};

Plan plan(int B, int P, int G, int H_kv, int d, int max_ctx, bool cut) {
    const long long bh = (long long)B * H_kv;
    const int n16 = row_blocks(P, G, 16), n128 = row_blocks(P, G, 128), tiles = (max_ctx + kTile - 1) / kTile;
    const long long g16 = n16 * bh, g64 = row_blocks(P, G, 64) * bh, g128 = n128 * bh;
    if (n16 <= 2 || g16 <= 128) {
        const int each = (tiles + NW - 1) / NW;  // a tile at least for each wave
        const int s = cut ? (int)std::min<long long>({256 / g16, each, IE_KV8_MAX_SPLITS}) : 1;
        return {kRows16, std::max(s, 1)};
    }
    if (cut) {
        const bool behind = max_ctx - P >= P;
        if (d == 128 && g16 > 256 && g128 <= 512 && 4ll * P * G >= 3 * 128ll * n128 && (behind || g128 > 256)) {
            const int s = (int)((g128 <= 256 ? 512 : 1024) / g128);
            if (s >= 2 && 8 * s <= tiles) return {kOneTeam, s};
        }
        if (behind && (g16 <= 208 || (d == 128 && g16 > 256))) {
            const int s = (int)std::min<long long>((d == 128 ? 256 : 512) / g64, tiles / 10);
            if (s >= 2) return {kTwoTeams, s};
        } else if (behind && g16 > 256) {
            const int two = (int)(512 / g64), one = g64 <= 448 ? (int)(1024 / g64) : 1;
            if (two >= 4 && 10 * two <= tiles) return {kTwoTeams, two};
            if (one >= 2 && 10 * one <= tiles) return {kOneTeam, one};
        }
    }
    if (g64 < 128 || (g64 < 256 && g64 < 24ll * tiles)) return {kRows16, 1};
    return {g64 < 1024 ? kTwoTeams : kOneTeam, 1};
}

template <int D>
void launch(const Kv8Attn& a, hipStream_t s) {
    const float qscale = (1.0f / sqrtf((float)D)) * 1.4426950408889634f;
    const int G = a.H_q / a.c.H, n16 = row_blocks(a.P, G, 16), n64 = row_blocks(a.P, G, 64), n128 = row_blocks(a.P, G, 128);
    const unsigned bh = (unsigned)a.B * a.c.H, parts = bh * a.splits;
    const Form form = plan(a.B, a.P, G, a.c.H, D, a.max_ctx, a.splits > 1).form;
    constexpr int NC = D == 64 ? 1 : 2;  // of one team
    const int n = D == 64 ? n64 : n128;
    if (form == kRows16)
        kv8_prefill_split_kernel<D><<<n16 * parts, 64 * NW, 0, s>>>(a, n16, qscale);
    else if (form == kTwoTeams && a.splits == 1)
        kv8_prefill_block_kernel<D, 1, 2, false><<<n64 * bh, 512, 0, s>>>(a, n64, qscale);
    else if (form == kTwoTeams)
        kv8_prefill_block_kernel<D, 1, 2, true><<<n64 * parts, 512, 0, s>>>(a, n64, qscale);
    else if (a.splits == 1)
        kv8_prefill_block_kernel<D, NC, 1, false><<<n * bh, 256, 0, s>>>(a, n, qscale);
    else
        kv8_prefill_block_kernel<D, NC, 1, true><<<n * parts, 256, 0, s>>>(a, n, qscale);
    if (a.splits > 1) launch_kv8_merge(D, a.B * a.P * a.H_q, a.splits, a.ws, a.O, s);
}

}  // namespace

int kv8_prefill_splits(int B, int P, int H_q, int H_kv, int d, int max_ctx) {
    return plan(B, P, H_q / H_kv, H_kv, d, max_ctx, true).splits;
}

int launch_prefill_attn_kv8(const Kv8Attn& a, hipStream_t s) {
    if (a.splits < 1 || a.splits > IE_KV8_MAX_SPLITS || (a.splits > 1 && !a.ws))
        return fail(IE_ERR_INVALID, "prefill_attn_kv8: %d splits, workspace %p", a.splits, (void*)a.ws);
    if (a.c.d == 64)
        launch<64>(a, s);
    else
        launch<128>(a, s);
    return IE_OK;
}

}  // namespace ie
