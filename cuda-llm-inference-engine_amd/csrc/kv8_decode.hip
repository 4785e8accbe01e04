// kv8_decode.hip — split-K decode attention over the 8-bit paged KV cache
// (include/ie_kv8.h), on the int8 matrix cores with the cache's bytes as they
// lie: no conversion of K or V, no LDS in the walk.
//
// Mathematics.  o = sum_j w_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j =
// log2(e) / sqrt(d) * ks_j (q . k_j), w_j = p_j vs_j; k_j, v_j are codes, ks_j,
// vs_j their page's scales.  Both products take one fp32 operand to int8
// exactly enough: a 30-bit fixed-point number (relative to the row's largest
// magnitude, so its steps are 2^-30 of that) is four signed digits of 8 bits,
// x = sum_i 256^i x_i, whose products with codes add up exactly in int32.  The
// four digits of up to four query heads are the 16 columns of
// v_mfma_i32_16x16x64_i8:
//   S^T = K q^T   A = 16 keys x 64 channels (16 bytes a lane straight from the
//                 page), B = the queries' digits, once per launch in registers
//   O^T = V^T w^T A = 16 channels x 64 keys (16 bytes a lane straight from the
//                 page: V lies with a channel's 16 tokens side by side), B = the
//                 weights' digits
// A tile is 64 keys, four 16-token groups; row 4 q + r of product t of S^T is
// key 16 q + 4 t + r, so the lane that receives scores (rows 4 q .. 4 q + 3 of
// column n, t = 0..3) holds the 16 keys of group q of column n, which are the 16
// bytes of its own B operand of the second product: each lane adds its column's
// digits over the quad (two DPP adds), takes the exponential and keeps its own
// digit's bytes.  Softmax work is done by the four lanes of a quad alike.
//
// The running maximum m and the weights' unit W are moved only when a weight
// would pass W (first set to 8 times the largest weight of a tile): until then
// the second product accumulates in its int32 registers, which hold 2^17 keys.
// Where it must, they are added to fp32 sums and m and W set anew (rebase).
//
// A wave walks tiles of its workgroup's range for 4 NT query heads; a tile's K
// is requested when the previous one's scores are done, its V when the previous
// one's output is, its table entries one tile earlier.  A workgroup is one
// (sequence, KV head, split) with up to 4 NT HT query heads; its waves merge in
// LDS in wave order, the splits in a second launch in split order.
//
// Bound by the bytes in flight: a wave's tile is 8 KB (d = 64) or 16 KB, and
// the fp32 sums lie in LDS so that three waves a SIMD fit (four at d = 64, two
// with eight heads a wave).  32 x (8 x 4) x 8192 x 128 95 us, 5.7 TB/s; with the
// sums in registers 102.  Eight heads on one wave (NT = 2) read the tile once: 2 x
// (8 x 8) x 40000 x 128 45.3 against 46.0 us on two waves of four heads each.
// Eight or sixteen waves a workgroup are never ahead (8 x 12 x 1024 x 64: 9.5 us
// with 4 waves, 10.0 with 8, 11.0 with 16).
#include <algorithm>
#include <cmath>

#include "device_util.h"
#include "kv8_rule.h"

// The lanes of a quad take different digits of one number, so they must come to
// the same bits: no product is fused into the quad's sums (which would round one
// of two addends, another one in each lane).
#pragma clang fp contract(off)

namespace ie {
namespace {

constexpr int kTile = 64;  // keys
constexpr int NW = 4;      // waves a workgroup

template <int CTRL>
__device__ __forceinline__ float dpp_quad(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// Sum over the four lanes of a quad, in every lane.
__device__ __forceinline__ float quad_sum(float v) {
    v += dpp_quad<0xB1>(v);  // lanes 1, 0, 3, 2
    v += dpp_quad<0x4E>(v);  // lanes 2, 3, 0, 1
    return v;
}
// Biased digits: byte i of the result is the signed digit i of x plus 128.
__device__ __forceinline__ uint32_t biased_digits(int x) { return (uint32_t)x + 0x80808080u; }

// Byte b of four words as one word (sel = b in each byte position, see v_perm).
__device__ __forceinline__ uint32_t gather_bytes(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t sel) {
    // sel picks byte b of the second operand into byte 0 and of the first into byte 1
    const uint32_t lo = __builtin_amdgcn_perm(x1, x0, sel), hi = __builtin_amdgcn_perm(x3, x2, sel);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// One wave: sequence b's new row of K or of V, head h, at position pos of its
// cache.  A page that grows is rare, so what it holds is read only then.
template <int D>
__device__ __forceinline__ void append_row(const Kv8Attn& a, bool is_v, int b, int h, int pos) {
    constexpr int C = D / 64;  // channels a lane
    const int lane = threadIdx.x & 63, bs = 1 << a.c.bs_log2, r = pos & (bs - 1);
    const float* src = (is_v ? a.V : a.K) + (size_t)b * a.kv_ld + (size_t)h * D + C * lane;
    float x[C];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        x[i] = src[i];
        mx = max(mx, fbits(x[i]) & 0x7fffffffu);
    }
    const size_t pair = (size_t)a.c.table[(size_t)b * a.c.nbps + (pos >> a.c.bs_log2)] * a.c.H + h;
    int8_t* codes = (is_v ? a.c.v : a.c.k) + pair * ((size_t)bs * D);
    float* scale_at = (is_v ? a.c.vs : a.c.ks) + pair;
    const float had = r > 0 ? *scale_at : 0.0f;
    const PageScale page(wave_umax(mx), r, had);
    const bool keep = a.undo.at != nullptr;  // uniform
    const size_t entry = ((size_t)b * 2 + is_v) * a.c.H + h;
    if (keep && lane == 0) a.undo.at[entry] = page.grew ? pos : -1;
    if (page.grew) {  // uniform
        if (keep && lane == 0) a.undo.scale[entry] = had;
        uint32_t* words = reinterpret_cast<uint32_t*>(codes);
        uint32_t* kept = a.undo.codes + entry * (bs * D / 4);
        for (int i0 = lane; i0 < bs * D / 4; i0 += 4 * 64) {  // (a page is 256 words at least)
            uint32_t was[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (first_row(i0 + 64 * u, is_v, D) < r) was[u] = words[i0 + 64 * u];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + 64 * u, row = first_row(i, is_v, D);
                if (row >= r) continue;
                if (keep) kept[i] = was[u];
                int q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    q[e] = byte_of(was[u], e);
                    if (!is_v || row + e < r) q[e] = code((float)q[e] * page.move);
                }
                words[i] = pack4(q[0], q[1], q[2], q[3]);
            }
        }
        __threadfence_block();  // before the row's bytes, which may lie in those words
    }
    if (lane == 0 && (r == 0 || page.grew)) *scale_at = page.scale;
#pragma unroll
    for (int i = 0; i < C; ++i)
        codes[is_v ? ((size_t)(r >> 4) * D + C * lane + i) * 16 + (r & 15) : (size_t)r * D + C * lane + i] = (int8_t)code(x[i] * page.inv);
}

// blockIdx.x = ((b * H + h) * groups + head group) * splits + split.  APPEND (one
// workgroup a sequence and KV head): the sequence's new row first.
template <int D, int NT, int HT, bool APPEND>
__global__ __launch_bounds__(64 * NW, D == 64 ? (NT == 1 ? 4 : 3) : (NT == 1 ? 3 : 2)) void kv8_decode_kernel(Kv8Attn a, int groups, float qscale) {
    constexpr int KB = D / 64, JB = D / 16, HEADS = 4 * NT * HT;
    constexpr int TW = NW / HT;  // waves that share a set of heads
    __shared__ float sh_o[NW][4 * NT][D];
    __shared__ float sh_m[NW][4 * NT], sh_l[NW][4 * NT];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, ht = wid % HT, tw = wid / HT;
    unsigned id = blockIdx.x;
    const int split = (int)(id % (unsigned)a.splits);
    id /= (unsigned)a.splits;
    const int hg = (int)(id % (unsigned)groups);
    id /= (unsigned)groups;
    const int H = a.c.H, h = (int)(id % (unsigned)H), b = (int)(id / (unsigned)H);
    const int G = a.H_q / H, g0 = hg * HEADS, gn = min(HEADS, G - g0);
    int n;
    if (APPEND) {
        const int pos = a.positions[b];
        const bool in = pos >= 0 && pos < (long long)a.c.nbps << a.c.bs_log2;  // (else the sequence is left out)
        if (wid < 2 && in) append_row<D>(a, wid == 1, b, h, pos);
        __syncthreads();
        n = in ? min(pos, a.max_ctx - 1) + 1 : 0;
    } else {
        n = max(0, min(a.lens[b], a.max_ctx));
    }
    const int tiles = (n + kTile - 1) / kTile;
    const int t0 = (int)((unsigned)tiles * split / (unsigned)a.splits), t1 = (int)((unsigned)tiles * (split + 1) / (unsigned)a.splits);

    const int col = lane & 15, q4 = lane >> 4, digit = lane & 3;
    const int lgg = a.c.bs_log2 - 4;  // 16-token groups a page, log2
    const int* table = a.c.table + (size_t)b * a.c.nbps;
    const int last = (n - 1) >> 4;  // the context's last group
    const int gk = (lane >> 2) & 3, gv = q4;
    // K operand: key row 4 t + (lane & 3) of group gk, bytes 64 kb + 16 q4
    const int k_off = (lane & 3) * D + q4 * 16;
    // V operand: channel 16 j + col of group gv
    const int v_off = col * 16;

    struct Where {
        size_t k, v, s;  // byte offsets of the lane's K and V groups, index of its scales
    };
    auto entry = [&](int tile, int g) { return table[min(4 * tile + g, last) >> lgg]; };
    auto place = [&](int tile, int pk, int pv) {
        const int mask = (1 << lgg) - 1;
        const size_t pairk = (size_t)pk * H + h, pairv = (size_t)pv * H + h;
        Where w;
        w.k = ((pairk << lgg) + (min(4 * tile + gk, last) & mask)) * (16 * D) + k_off;
        w.v = ((pairv << lgg) + (min(4 * tile + gv, last) & mask)) * (16 * D) + v_off;
        w.s = pairv;
        return w;
    };

    float m[NT], l[NT];
    int ub[NT];  // biased exponent of W * 2^-30
    i32x4 acc[NT][JB];
    // The fp32 sums, digits joined: rarely touched, so in LDS.  Lane (col, q4)
    // with digit 0 has channels 16 j + 4 q4 .. + 3 of head col / 4.
    auto sums = [&](int c, int j) { return reinterpret_cast<float4*>(&sh_o[wid][4 * c + (col >> 2)][16 * j + 4 * q4]); };
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.0f;
        ub[c] = 127 - 30;
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            acc[c][j] = i32x4{0, 0, 0, 0};
            if (digit == 0) *sums(c, j) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    // sums = (sums + acc) * f
    auto flush = [&](int c, float f) {
        const float f0 = pow2(ub[c]) * pow2(127 + 8 * digit);
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = quad_sum((float)acc[c][j][r] * f0);
            if (digit == 0) {
                const float4 was = *sums(c, j);
                *sums(c, j) = make_float4((was.x + o[0]) * f, (was.y + o[1]) * f, (was.z + o[2]) * f, (was.w + o[3]) * f);
            }
        }
    };
    const float digit_w = pow2(127 + 8 * digit);  // 256^digit
    const uint32_t sel = (uint32_t)digit * 0x0101u + 0x0400u;

    int tile = t0 + tw;
    if (tile < t1) {  // uniform over the wave
        // The queries' channels 64 kb + 16 q4 .. + 15 of head col / 4 of each
        // column tile, requested ahead of the table entries' round trip.
        float x[NT][KB][16];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const int g = min(g0 + 4 * (ht * NT + c) + (col >> 2), G - 1);
            const float* qp = a.Q + (size_t)b * a.q_ld + ((size_t)h * G + g) * D + q4 * 16;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 f = *reinterpret_cast<const float4*>(qp + kb * 64 + 4 * i);
                    x[c][kb][4 * i] = f.x; x[c][kb][4 * i + 1] = f.y; x[c][kb][4 * i + 2] = f.z; x[c][kb][4 * i + 3] = f.w;
                }
        }
        i32x4 kw[4][KB], vw[JB];
        float ks, vs;
        Where w = place(tile, entry(tile, gk), entry(tile, gv));
        auto load_k = [&]() {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    kw[t][kb] = *reinterpret_cast<const i32x4*>(a.c.k + w.k + t * 4 * D + kb * 64);
            ks = a.c.ks[w.s];
            vs = a.c.vs[w.s];
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < JB; ++j) vw[j] = *reinterpret_cast<const i32x4*>(a.c.v + w.v + j * 256);
        };
        load_k();
        load_v();
        int next = min(tile + TW, t1 - 1);
        int pk = entry(next, gk), pv = entry(next, gv);

        // Their digits: lane (col, q4) holds digit `digit`.
        i32x4 qd[NT][KB];
        float qw[NT];  // what a score's digit counts
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            uint32_t mx = 0;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = max(mx, __builtin_bit_cast(uint32_t, x[c][kb][i]) & 0x7fffffffu);
            mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
            mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
            const int e = max((int)(mx >> 23), 30);  // both factors stay normal numbers
            const float up = pow2(min(283 - e, 253));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t dg[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) dg[k] = biased_digits((int)rintf(x[c][kb][4 * i + k] * up));
                    qd[c][kb][i] = (int)(gather_bytes(dg[0], dg[1], dg[2], dg[3], sel) ^ 0x80808080u);
                }
            qw[c] = e == 255 ? __builtin_nanf("") : pow2(max(e - 29, 1)) * digit_w;
        }

        int since = 0;
        for (;;) {
            const bool more = tile + TW < t1;
            i32x4 s[NT][4];
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    s[c][t] = i32x4{0, 0, 0, 0};
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
                        s[c][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kw[t][kb], qd[c][kb], s[c][t], 0, 0, 0);
                }
            // a scale that is not finite makes every score of its page NaN
            const float kscale = (ks + ((ks - ks) + (vs - vs))) * qscale, vscale = vs;
            const int seen = n - tile * kTile - 16 * q4;  // keys of this lane's group within the context
            w = place(next, pk, pv);
            load_k();
            next = min(tile + 2 * TW, t1 - 1);
            pk = entry(next, gk);
            pv = entry(next, gv);

#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const float sw = qw[c] * kscale;
                float sc[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = quad_sum((float)s[c][i >> 2][i & 3] * sw);
                if (tile * kTile + kTile > n) {  // uniform: the context's last tile
#pragma unroll
                    for (int i = 0; i < 16; ++i) sc[i] = i < seen ? sc[i] : -INFINITY;
                }
                float top = sc[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[i]);
                // log2 of the lane's largest weight, rounded up, against m
                const float vexp = (float)(biased_exp(vscale) - 126);
                bool moved = fmaxf(top - m[c] + vexp - (float)(ub[c] - 127), top - m[c] - 70.0f) > 30.0f;
                if (__ballot(moved) != 0 || since == 1024) {  // uniform
                    moved = max_xor32(max_xor16(moved ? 1.0f : 0.0f)) > 0.0f;  // over the column
                    const float ctop = max_xor32(max_xor16(top));
                    const float mn = moved ? fmaxf(m[c], ctop) : m[c];
                    const float f = moved ? exp2_sm(m[c] - mn) : 1.0f;
                    if (since > 0) {
                        flush(c, f);
#pragma unroll
                        for (int j = 0; j < JB; ++j) acc[c][j] = i32x4{0, 0, 0, 0};
                    }
                    l[c] *= f;
                    m[c] = mn;
                    // W = 8 times the power of two above the tile's largest weight
                    const float wm = max_xor32(max_xor16(top - mn + vexp));
                    if (moved) ub[c] = (int)fminf(fmaxf(ceilf(wm) + (127.0f + 3.0f - 30.0f), 1.0f), 224.0f);
                }
                float p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = exp2_sm(sc[i] - m[c]);
                float wc = vscale * pow2(254 - ub[c]);
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += p[i];
                l[c] += sum;
                if (__ballot(wc == INFINITY) != 0) {  // uniform; a scale more than 2^127 times W's: its weights in two steps
                    asm volatile("");
                    const bool over = wc == INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[i] *= over ? vscale : 1.0f;
                    wc = over ? pow2(254 - ub[c]) : wc;
                }
                i32x4 wd;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    uint32_t dg[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) dg[r] = biased_digits((int)(p[4 * t + r] * wc));
                    wd[t] = (int)(gather_bytes(dg[0], dg[1], dg[2], dg[3], sel) ^ 0x80808080u);
                }
#pragma unroll
                for (int j = 0; j < JB; ++j)
                    acc[c][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vw[j], wd, acc[c][j], 0, 0, 0);
            }
            load_v();
            since = since == 1024 ? 1 : since + 1;
            if (!more) break;
            tile += TW;
        }
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        flush(c, 1.0f);
        const float lt = sum_xor32(sum_xor16(l[c]));
        if (digit == 0 && q4 == 0) {
            sh_m[wid][4 * c + (col >> 2)] = m[c];
            sh_l[wid][4 * c + (col >> 2)] = lt;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gn * D; i += 64 * NW) {
        const int g = i / D, dim = i % D, gw = g % (4 * NT), w0 = g / (4 * NT);
        float mm = -INFINITY;
#pragma unroll
        for (int w = w0; w < NW; w += HT) mm = fmaxf(mm, sh_m[w][gw]);
        float o = 0.0f, lt = 0.0f;
#pragma unroll
        for (int w = w0; w < NW; w += HT) {
            const float lw = sh_l[w][gw];
            const float f = lw == 0.0f ? 0.0f : exp2_sm(sh_m[w][gw] - mm);  // a wave without keys; NaN stays
            lt = fmaf(lw, f, lt);
            o = fmaf(sh_o[w][gw][dim], f, o);
        }
        const size_t row = (size_t)b * a.H_q + (size_t)h * G + g0 + g;
        if (a.splits == 1) {
            a.O[row * D + dim] = lt == 0.0f ? 0.0f : o / lt;
        } else {
            float* ws = a.ws + (row * a.splits + split) * (D + 2);
            ws[dim] = o;
            if (dim == 0) {
                ws[D] = mm;
                ws[D + 1] = lt;
            }
        }
    }
}

// Joins the splits of one (sequence, query head): a workgroup's wave w has
// splits w, w + 4, .., all of whose rows are requested at once; then the waves'
// sums in wave order.  D threads a wave are D / 64 channels a lane.
template <int D>
__global__ __launch_bounds__(256) void kv8_merge_kernel(int S, const float* __restrict__ ws, float* __restrict__ O) {
    constexpr int C = D / 64, MOST = IE_KV8_MAX_SPLITS / 4;
    __shared__ float sh[4][D];
    const int row = blockIdx.x, wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float* w = ws + (size_t)row * S * (D + 2);
    const int sl = min(lane, S - 1);
    const float ms = w[(size_t)sl * (D + 2) + D];
    float ls = w[(size_t)sl * (D + 2) + D + 1];
    float x[MOST][C];
#pragma unroll
    for (int u = 0; u < MOST; ++u)
        if (wid + 4 * u < S)  // uniform
#pragma unroll
            for (int i = 0; i < C; ++i) x[u][i] = w[(size_t)(wid + 4 * u) * (D + 2) + 64 * i + lane];
    if (lane >= S) ls = 0.0f;
    const float mm = wave_max(ls == 0.0f ? -INFINITY : ms);
    const float f = ls == 0.0f ? 0.0f : exp2_sm(ms - mm);
    const float l = wave_sum(ls * f);
    float o[C];
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = 0.0f;
#pragma unroll
    for (int u = 0; u < MOST; ++u)
        if (wid + 4 * u < S) {
            const float fu = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), wid + 4 * u));
#pragma unroll
            for (int i = 0; i < C; ++i) o[i] = fmaf(x[u][i], fu, o[i]);
        }
#pragma unroll
    for (int i = 0; i < C; ++i) sh[wid][64 * i + lane] = o[i];
    __syncthreads();
    if (threadIdx.x < D) {
        const float sum = sh[0][threadIdx.x] + sh[1][threadIdx.x] + sh[2][threadIdx.x] + sh[3][threadIdx.x];
        O[(size_t)row * D + threadIdx.x] = l == 0.0f ? 0.0f : sum / l;
    }
}

// The same for at most MOST splits: a wave a row, without LDS.  With MOST 2 to 8 it
// takes 0.6 us less (1 x 12 x 64, ctx 2048 in eight splits 6.05 against 6.65 in all;
// 6144 rows of two 12.5 against 16.5); with 16, one wave's loads, 9.2 against 9.0.
template <int D, int MOST>
__global__ __launch_bounds__(256) void kv8_merge_few_kernel(int rows, int S, const float* __restrict__ ws, float* __restrict__ O) {
    constexpr int C = D / 64;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows) return;
    const float* w = ws + (size_t)row * S * (D + 2);
    float x[MOST][C], m[MOST], l[MOST];
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
        const float* p = w + min(u, S - 1) * (D + 2);
#pragma unroll
        for (int i = 0; i < C; ++i) x[u][i] = p[64 * i + lane];
        m[u] = p[D];
        l[u] = u < S ? p[D + 1] : 0.0f;
    }
    float mm = -INFINITY, lt = 0.0f, o[C];
#pragma unroll
    for (int u = 0; u < MOST; ++u) mm = l[u] == 0.0f ? mm : fmaxf(mm, m[u]);
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = 0.0f;
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
        const float f = l[u] == 0.0f ? 0.0f : exp2_sm(m[u] - mm);
        lt = fmaf(l[u], f, lt);
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = fmaf(x[u][i], f, o[i]);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) O[(size_t)row * D + 64 * i + lane] = lt == 0.0f ? 0.0f : o[i] / lt;
}

template <int D>
void merge(int rows, int splits, const float* ws, float* O, hipStream_t s) {
    const unsigned few = (unsigned)(rows + 3) / 4;
    if (splits <= 2)
        kv8_merge_few_kernel<D, 2><<<few, 256, 0, s>>>(rows, splits, ws, O);
    else if (splits <= 4)
        kv8_merge_few_kernel<D, 4><<<few, 256, 0, s>>>(rows, splits, ws, O);
    else if (splits <= 8)
        kv8_merge_few_kernel<D, 8><<<few, 256, 0, s>>>(rows, splits, ws, O);
    else
        kv8_merge_kernel<D><<<rows, 256, 0, s>>>(splits, ws, O);
}

template <int D>
void launch(const Kv8Attn& a, hipStream_t s) {
    const int G = a.H_q / a.c.H;
    const float qscale = (1.0f / sqrtf((float)D)) * 1.4426950408889634f;
    const int heads = G <= 4 ? 4 : G <= 8 ? 8 : 16, groups = (G + heads - 1) / heads;
    const unsigned grid = (unsigned)a.B * a.c.H * groups * a.splits;
    if (a.positions)
        kv8_decode_kernel<D, 1, 1, true><<<grid, 64 * NW, 0, s>>>(a, groups, qscale);
    else if (heads == 4)
        kv8_decode_kernel<D, 1, 1, false><<<grid, 64 * NW, 0, s>>>(a, groups, qscale);
    else if (heads == 8)
        kv8_decode_kernel<D, 2, 1, false><<<grid, 64 * NW, 0, s>>>(a, groups, qscale);
    else
        kv8_decode_kernel<D, 2, 2, false><<<grid, 64 * NW, 0, s>>>(a, groups, qscale);
    if (a.splits > 1) launch_kv8_merge(D, a.B * a.H_q, a.splits, a.ws, a.O, s);
}

}  // namespace

void launch_kv8_merge(int d, int rows, int splits, const float* ws, float* O, hipStream_t s) {
    if (d == 64)
        merge<64>(rows, splits, ws, O, s);
    else
        merge<128>(rows, splits, ws, O, s);
}

int launch_decode_attn_kv8(const Kv8Attn& a, hipStream_t s) {
    if (a.splits < 1 || a.splits > IE_KV8_MAX_SPLITS || (a.splits > 1 && !a.ws))
        return fail(IE_ERR_INVALID, "decode_attn_kv8: %d splits, workspace %p", a.splits, (void*)a.ws);
    if (a.positions && (a.splits > 1 || a.H_q > 4 * a.c.H))
        return fail(IE_ERR_INVALID, "decode_attn_kv8: no append with %d splits, %d heads on %d", a.splits, a.H_q, a.c.H);
    if (a.c.d == 64)
        launch<64>(a, s);
    else
        launch<128>(a, s);
    return IE_OK;
}

}  // namespace ie
