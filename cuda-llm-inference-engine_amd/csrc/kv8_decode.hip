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
// A wave walks tiles of its workgroup's range; a tile's K is requested when the
// previous one's scores are done, its V when the previous one's output is, its
// table entries one tile earlier.  A workgroup is one (sequence, KV head, split)
// with up to 4 NT query heads; its waves merge in LDS in wave order, the splits
// in a second launch in split order.
#include <algorithm>
#include <cmath>

#include "device_util.h"
#include "kv8.h"

namespace ie {
namespace {

constexpr int kTile = 64;  // keys

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
__device__ __forceinline__ float pow2(int biased) { return __builtin_bit_cast(float, (uint32_t)biased << 23); }
__device__ __forceinline__ int biased_exp(float v) { return (int)((__builtin_bit_cast(uint32_t, v) >> 23) & 255u); }
// Biased digits: byte i of the result is the signed digit i of x plus 128.
__device__ __forceinline__ uint32_t biased_digits(int x) { return (uint32_t)x + 0x80808080u; }

// Byte b of four words as one word (sel = b in each byte position, see v_perm).
__device__ __forceinline__ uint32_t gather_bytes(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t sel) {
    // sel picks byte b of the second operand into byte 0 and of the first into byte 1
    const uint32_t lo = __builtin_amdgcn_perm(x1, x0, sel), hi = __builtin_amdgcn_perm(x3, x2, sel);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// blockIdx.x = ((b * H + h) * groups + head group) * splits + split
template <int D, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void kv8_decode_kernel(Kv8Attn a, int groups, float qscale) {
    constexpr int KB = D / 64, JB = D / 16, HEADS = 4 * NT;
    __shared__ float sh_o[NW][HEADS][D];
    __shared__ float sh_m[NW][HEADS], sh_l[NW][HEADS];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    unsigned id = blockIdx.x;
    const int split = (int)(id % (unsigned)a.splits);
    id /= (unsigned)a.splits;
    const int hg = (int)(id % (unsigned)groups);
    id /= (unsigned)groups;
    const int H = a.c.H, h = (int)(id % (unsigned)H), b = (int)(id / (unsigned)H);
    const int G = a.H_q / H, g0 = hg * HEADS, gn = min(HEADS, G - g0);
    const int n = max(0, min(a.lens[b], a.max_ctx));
    const int tiles = (n + kTile - 1) / kTile;
    const int t0 = (int)((long long)tiles * split / a.splits), t1 = (int)((long long)tiles * (split + 1) / a.splits);

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
    float of[NT][JB][4];
    i32x4 acc[NT][JB];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.0f;
        ub[c] = 127 - 30;
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            acc[c][j] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < 4; ++r) of[c][j][r] = 0.0f;
        }
    }
    const float digit_w = pow2(127 + 8 * digit);  // 256^digit
    const uint32_t sel = (uint32_t)digit * 0x0101u + 0x0400u;

    int tile = t0 + wid;
    if (tile < t1) {  // uniform over the wave
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
        int next = min(tile + NW, t1 - 1);
        int pk = entry(next, gk), pv = entry(next, gv);

        // The queries' digits: lane (col, q4) holds digit `digit` of channels
        // 64 kb + 16 q4 .. + 15 of head col / 4 of each column tile.
        i32x4 qd[NT][KB];
        float qw[NT];  // what a score's digit counts
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const int g = min(g0 + 4 * c + (col >> 2), G - 1);
            const float* qp = a.Q + (size_t)b * a.q_ld + ((size_t)h * G + g) * D + q4 * 16;
            float x[KB][16];
            uint32_t mx = 0;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 f = *reinterpret_cast<const float4*>(qp + kb * 64 + 4 * i);
                    x[kb][4 * i] = f.x; x[kb][4 * i + 1] = f.y; x[kb][4 * i + 2] = f.z; x[kb][4 * i + 3] = f.w;
                }
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = max(mx, __builtin_bit_cast(uint32_t, x[kb][i]) & 0x7fffffffu);
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
                    for (int k = 0; k < 4; ++k) dg[k] = biased_digits((int)rintf(x[kb][4 * i + k] * up));
                    qd[c][kb][i] = (int)(gather_bytes(dg[0], dg[1], dg[2], dg[3], sel) ^ 0x80808080u);
                }
            qw[c] = e == 255 ? __builtin_nanf("") : pow2(max(e - 29, 1)) * digit_w;
        }

        int since = 0;
        for (;;) {
            const bool more = tile + NW < t1;
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
            next = min(tile + 2 * NW, t1 - 1);
            pk = entry(next, gk);
            pv = entry(next, gv);

#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const float sw = qw[c] * kscale;
                float p[16];
                auto weights = [&](float mm) {
                    const float off = -0.25f * mm;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        p[i] = exp2_sm(quad_sum(fmaf((float)s[c][i >> 2][i & 3], sw, off)));
                    if (tile * kTile + kTile > n) {  // uniform: the context's last tile
#pragma unroll
                        for (int i = 0; i < 16; ++i) p[i] = i < seen ? p[i] : 0.0f;
                    }
                };
                weights(m[c]);
                float pm = p[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) pm = fmaxf(pm, p[i]);
                // past W, or near fp32's end although its page's scale is small
                bool moved = fmaxf(pm * (vscale * pow2(254 - ub[c])), pm * 0x1p-70f) > 0x1p30f;
                if (__ballot(moved) != 0 || since == 1024) {  // uniform
                    const float f0 = pow2(ub[c]) * digit_w;
                    moved = max_xor32(max_xor16(moved ? 1.0f : 0.0f)) > 0.0f;  // over the column
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float sc = quad_sum((float)s[c][i >> 2][i & 3] * sw);
                        if (i < seen) top = fmaxf(top, sc);
                    }
                    top = max_xor32(max_xor16(top));
                    const float mn = moved ? fmaxf(m[c], top) : m[c];
                    const float f = moved ? exp2_sm(m[c] - mn) : 1.0f;
#pragma unroll
                    for (int j = 0; j < JB; ++j) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) of[c][j][r] = fmaf((float)acc[c][j][r], f0, of[c][j][r]) * f;
                        acc[c][j] = i32x4{0, 0, 0, 0};
                    }
                    l[c] *= f;
                    m[c] = mn;
                    weights(mn);
                    pm = p[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) pm = fmaxf(pm, p[i]);
                    const float wm = max_xor32(max_xor16(pm * vscale));
                    // W = 8 times the power of two above the tile's largest weight
                    if (moved) ub[c] = min(max(biased_exp(wm) + 4 - 30, 1), 224);
                }
                const float wc = vscale * pow2(254 - ub[c]);
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += p[i];
                l[c] += sum;
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
            tile += NW;
        }
    }
    // fp32 sums, digits joined: lane (col, q4) holds channels 16 j + 4 q4 + r of head col / 4
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const float f0 = pow2(ub[c]) * digit_w;
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            float4 o;
            o.x = quad_sum(fmaf((float)acc[c][j][0], f0, of[c][j][0]));
            o.y = quad_sum(fmaf((float)acc[c][j][1], f0, of[c][j][1]));
            o.z = quad_sum(fmaf((float)acc[c][j][2], f0, of[c][j][2]));
            o.w = quad_sum(fmaf((float)acc[c][j][3], f0, of[c][j][3]));
            if (digit == 0) *reinterpret_cast<float4*>(&sh_o[wid][4 * c + (col >> 2)][16 * j + 4 * q4]) = o;
        }
        const float lt = sum_xor32(sum_xor16(l[c]));
        if (digit == 0 && q4 == 0) {
            sh_m[wid][4 * c + (col >> 2)] = m[c];
            sh_l[wid][4 * c + (col >> 2)] = lt;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gn * D; i += 64 * NW) {
        const int g = i / D, dim = i % D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sh_m[w][g]);
        float o = 0.0f, lt = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float lw = sh_l[w][g];
            const float f = lw == 0.0f ? 0.0f : exp2_sm(sh_m[w][g] - mm);  // a wave without keys; NaN stays
            lt = fmaf(lw, f, lt);
            o = fmaf(sh_o[w][g][dim], f, o);
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

// Joins the splits of one (sequence, query head) with one wave, in split order.
template <int D>
__global__ __launch_bounds__(256) void kv8_merge_kernel(int rows, int S, const float* __restrict__ ws,
                                                        float* __restrict__ O) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows) return;
    const float* w = ws + (size_t)row * S * (D + 2);
    const int sl = min(lane, S - 1);
    const float ms = w[(size_t)sl * (D + 2) + D], ls = lane < S ? w[(size_t)sl * (D + 2) + D + 1] : 0.0f;
    const float mm = wave_max(ls == 0.0f ? -INFINITY : ms);
    const float f = ls == 0.0f ? 0.0f : exp2_sm(ms - mm);
    const float l = wave_sum(ls * f);
    float o[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] = 0.0f;
    for (int s0 = 0; s0 < S; s0 += 8) {
        float x[8][D / 64];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) x[u][i] = w[(size_t)min(s0 + u, S - 1) * (D + 2) + 64 * i + lane];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float fu = __shfl(f, (s0 + u) & 63, 64);  // 0 past the last split
#pragma unroll
            for (int i = 0; i < D / 64; ++i) o[i] = fmaf(x[u][i], s0 + u < S ? fu : 0.0f, o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) O[(size_t)row * D + 64 * i + lane] = l == 0.0f ? 0.0f : o[i] / l;
}

template <int D>
void launch(const Kv8Attn& a, hipStream_t s) {
    const int G = a.H_q / a.c.H;
    const float qscale = (1.0f / sqrtf((float)D)) * 1.4426950408889634f;
    const int heads = G <= 4 ? 4 : 8, groups = (G + heads - 1) / heads;
    const unsigned grid = (unsigned)a.B * a.c.H * groups * a.splits;
    if (G <= 4)
        kv8_decode_kernel<D, 1, 4><<<grid, 256, 0, s>>>(a, groups, qscale);
    else
        kv8_decode_kernel<D, 2, 4><<<grid, 256, 0, s>>>(a, groups, qscale);
    if (a.splits > 1)
        kv8_merge_kernel<D><<<(a.B * a.H_q + 3) / 4, 256, 0, s>>>(a.B * a.H_q, a.splits, a.ws, a.O);
}

}  // namespace

void launch_decode_attn_kv8(const Kv8Attn& a, hipStream_t s) {
    if (a.c.d == 64)
        launch<64>(a, s);
    else
        launch<128>(a, s);
}

}  // namespace ie
