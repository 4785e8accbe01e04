// kv8_cache.hip — rows into and out of the 8-bit paged KV cache
// (include/ie_kv8.h has the layout and the rule that scales follow).
//
// A page of one head is cut into tiles of 16 tokens x 64 channels, one wave (or T
// tiles of one wave) each.  Lane l holds tokens 4 (l / 16) .. + 3, channels 4 (l %
// 16) .. + 3: fp32 rows move as 256 contiguous bytes for each of four rows an
// instruction, K codes as one word (4 channels) a row, V codes as one word (4
// tokens) a channel.  A workgroup holds all tiles of one (sequence, page, head)
// of K or of V in registers, so the page's maximum, its codes and (where the
// scale had to grow) the earlier rows' new codes come from one pass over the data.
//
// Bound by HBM: 4 x 2000 rows of 8 x 128, K and V (65.5 MB in, 16.4 out) written in
// 17.3 us, 4.7 TB/s, and read back in 15.0, 5.5 TB/s (a copy of 1 GiB moves 4.7 to 5.2).
// The maximum goes over the wave by DPP and lane swaps: by six LDS permutes, with
// 16-byte words of codes a lane (64-byte pieces of fp32 rows an instruction), the
// write took 25.5 us and the read 20.8.
#include <algorithm>

#include "device_util.h"
#include "kv8_rule.h"

namespace ie {
namespace {

// Word j of a lane's four in tile t of a page: K row 4 (lane / 16) + j, V channel
// 4 (lane % 16) + j.
template <int D>
__device__ __forceinline__ int word_of(int t, bool is_v, int lane, int j) {
    constexpr int HALVES = D / 64;
    const int c = t % HALVES * 64 + 4 * (lane & 15), r = 4 * (lane >> 4);
    return t / HALVES * (4 * D) + (is_v ? (c + j) * 4 + r / 4 : ((r + j) * D + c) / 4);
}

// blockIdx.x = (b * npages + page) * H + h of K, then the same of V (K and V side by
// side, two streams in and two out at once, took 18.7 us where this takes 17.3)
template <int D, int T>
__global__ __launch_bounds__(1024) void kv8_write_kernel(Kv8Write a, int npages) {
    constexpr int HALVES = D / 64;
    __shared__ uint32_t wave_mx[16];
    __shared__ float had_sh;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
    unsigned id = blockIdx.x;
    const bool is_v = id >= gridDim.x / 2;
    if (is_v) id -= gridDim.x / 2;
    const int h = (int)(id % (unsigned)a.c.H);
    id /= (unsigned)a.c.H;
    const int j = (int)(id % (unsigned)npages), b = (int)(id / (unsigned)npages);
    const int lg = a.c.bs_log2, bs = 1 << lg;
    const int start = a.positions ? a.positions[b] : a.start;
    if (a.positions) {  // uniform
        const bool in = start >= 0 && start < (long long)a.c.nbps << lg;
        if (a.ctx_lens && h == 0 && !is_v && threadIdx.x == 0) a.ctx_lens[b] = in ? start + 1 : 0;
        if (!in) return;
    }
    const int lp = (start >> lg) + j, page0 = lp << lg;
    const int r0 = max(start - page0, 0), r1 = min(start + a.P - page0, bs);  // rows written here
    const size_t pair = (size_t)a.c.table[(size_t)b * a.c.nbps + lp] * a.c.H + h;
    uint32_t* codes = reinterpret_cast<uint32_t*>((is_v ? a.c.v : a.c.k) + pair * ((size_t)bs * D));
    float* scale_at = (is_v ? a.c.vs : a.c.ks) + pair;
    const float* src = (is_v ? a.V : a.K) + (size_t)b * a.P * a.ld + (size_t)h * D;

    float x[T][4][4];  // [row][channel]
    uint32_t was[T][4];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int t = wid * T + i, row0 = (t / HALVES) * 16, c0 = (t % HALVES) * 64;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + 4 * (lane >> 4) + r;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row >= r0 && row < r1)
                v = *reinterpret_cast<const float4*>(src + (size_t)(page0 + row - start) * a.ld + c0 + 4 * (lane & 15));
            x[i][r][0] = v.x; x[i][r][1] = v.y; x[i][r][2] = v.z; x[i][r][3] = v.w;
        }
        // the bytes beside the written ones; a tile without those is read only if the scale grows
        if ((row0 < r0 || row0 + 16 > r1) && row0 + 16 > r0 && row0 < r1)
#pragma unroll
            for (int k = 0; k < 4; ++k) was[i][k] = codes[word_of<D>(t, is_v, lane, k)];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) mx = max(mx, fbits(x[i][r][c]) & 0x7fffffffu);
    }
    mx = wave_umax(mx);
    // One wave reads the old scale, so that it is read before it is replaced.
    if (wid == 0 && lane == 0) had_sh = r0 > 0 ? *scale_at : 0.0f;
    if (lane == 0) wave_mx[wid] = mx;
    __syncthreads();
    for (int w = 0; w < nw; ++w) mx = max(mx, wave_mx[w]);
    const PageScale page(mx, r0, had_sh);
    const bool grew = page.grew;
    const float inv = page.inv, move = page.move;
    if (threadIdx.x == 0 && (r0 == 0 || grew)) *scale_at = page.scale;
    const bool keep = a.undo.at != nullptr;  // uniform
    const size_t entry = ((size_t)b * 2 + is_v) * a.c.H + h;
    if (keep && threadIdx.x == 0) {
        a.undo.at[entry] = grew ? start : -1;
        a.undo.scale[entry] = had_sh;
    }
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int t = wid * T + i, row0 = (t / HALVES) * 16;
        if (row0 >= r1 || (row0 + 16 <= r0 && !grew)) continue;  // nothing of this tile changes (uniform)
        const bool whole = row0 >= r0 && row0 + 16 <= r1;
        if (row0 + 16 <= r0)
#pragma unroll
            for (int k = 0; k < 4; ++k) was[i][k] = codes[word_of<D>(t, is_v, lane, k)];
        if (keep && grew && row0 < r0)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                a.undo.codes[entry * ((size_t)bs * D / 4) + word_of<D>(t, is_v, lane, k)] = was[i][k];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            int q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = is_v ? e : k, row = row0 + 4 * (lane >> 4) + r;
                q[e] = code((is_v ? x[i][e][k] : x[i][k][e]) * inv);
                if (!whole) {
                    const int old = byte_of(was[i][k], e);
                    q[e] = row < r0 ? (grew ? code((float)old * move) : old) : row < r1 ? q[e] : old;
                }
            }
            codes[word_of<D>(t, is_v, lane, k)] = pack4(q[0], q[1], q[2], q[3]);
        }
    }
}

// One wave per (sequence, K or V, head), blockIdx.x: the words that hold rows before
// the undone one, and the page's scale.
__global__ __launch_bounds__(64) void kv8_undo_kernel(int pos, Kv8Cache c, Kv8Undo u) {
    const size_t entry = blockIdx.x;
    const int h = (int)(entry % (unsigned)c.H), is_v = (int)(entry / (unsigned)c.H) & 1, b = (int)(entry / (2u * (unsigned)c.H));
    if (u.at[entry] != pos) return;  // uniform
    const int bs = 1 << c.bs_log2, r = pos & (bs - 1), words = bs * c.d / 4;
    const size_t pair = (size_t)c.table[(size_t)b * c.nbps + (pos >> c.bs_log2)] * c.H + h;
    uint32_t* codes = reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + pair * ((size_t)bs * c.d));
    for (int i = threadIdx.x; i < words; i += 64)
        if (first_row(i, is_v, c.d) < r) codes[i] = u.codes[entry * words + i];
    if (threadIdx.x == 0) (is_v ? c.vs : c.ks)[pair] = u.scale[entry];
}

// One wave per (sequence, 16-token group, head, 64 channels) of K and of V.
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8Read a, int groups, unsigned waves) {
    constexpr int HALVES = D / 64;
    const int lane = threadIdx.x & 63;
    unsigned id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= waves) return;
    const int half = (int)(id % HALVES);
    id /= HALVES;
    const int h = (int)(id % (unsigned)a.c.H);
    id /= (unsigned)a.c.H;
    const int g = (int)(id % (unsigned)groups), b = (int)(id / (unsigned)groups);
    const int lg = a.c.bs_log2, H = a.c.H;
    const long long start = a.starts[b];
    const long long first = ((start >> 4) + g) * 16;  // the group's first position
    const long long end = start + a.n;
    if (first >= end) return;
    long long lim = (long long)a.c.nbps << lg;
    if (a.lens) lim = min(lim, (long long)a.lens[b]);
    uint32_t kw[4] = {0, 0, 0, 0}, vw[4] = {0, 0, 0, 0};
    float ks = 0.0f, vs = 0.0f;
    if (first >= 0 && first < lim) {
        const size_t pair = (size_t)a.c.table[(size_t)b * a.c.nbps + (first >> lg)] * H + h;
        const size_t at = pair * ((size_t)D << lg) + (size_t)(first & ((1 << lg) - 1)) * D;
        const uint32_t* kc = reinterpret_cast<const uint32_t*>(a.c.k + at);
        const uint32_t* vc = reinterpret_cast<const uint32_t*>(a.c.v + at);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            kw[k] = kc[word_of<D>(half, false, lane, k)];
            vw[k] = vc[word_of<D>(half, true, lane, k)];
        }
        ks = a.c.ks[pair];
        vs = a.c.vs[pair];
    }
    const size_t row_n = (size_t)H * D;
    const size_t base = (size_t)b * a.n * row_n + (size_t)h * D + half * 64 + 4 * (lane & 15);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const long long pos = first + 4 * (lane >> 4) + r;
        if (pos < start || pos >= end) continue;
        const bool in = pos < lim;
        const size_t at = base + (size_t)(pos - start) * row_n;
        // (a row behind the limit is zero whatever its page's scale is)
        auto value = [&](int q, float s) { return in ? (float)q * s : 0.0f; };
        *reinterpret_cast<float4*>(a.K + at) = make_float4(value(byte_of(kw[r], 0), ks), value(byte_of(kw[r], 1), ks),
                                                           value(byte_of(kw[r], 2), ks), value(byte_of(kw[r], 3), ks));
        *reinterpret_cast<float4*>(a.V + at) = make_float4(value(byte_of(vw[0], r), vs), value(byte_of(vw[1], r), vs),
                                                           value(byte_of(vw[2], r), vs), value(byte_of(vw[3], r), vs));
    }
}

template <int D>
void launch_write(const Kv8Write& a, hipStream_t s) {
    const int lg = a.c.bs_log2;
    const int npages = a.positions ? 1 : (int)(((long long)a.start + a.P - 1) >> lg) - (a.start >> lg) + 1;
    const int tiles = (1 << lg) / 16 * (D / 64);
    const unsigned grid = (unsigned)a.B * npages * a.c.H * 2;
    if (tiles <= 16)
        kv8_write_kernel<D, 1><<<grid, 64 * tiles, 0, s>>>(a, npages);
    else
        kv8_write_kernel<D, 2><<<grid, 32 * tiles, 0, s>>>(a, npages);
}

}  // namespace

void launch_kv8_write(const Kv8Write& a, hipStream_t s) {
    if (a.c.d == 64)
        launch_write<64>(a, s);
    else
        launch_write<128>(a, s);
}

void launch_kv8_read(const Kv8Read& a, hipStream_t s) {
    const int groups = (a.n + 14) / 16 + 1;  // groups that n rows from any start can touch
    const unsigned waves = (unsigned)a.B * groups * a.c.H * (a.c.d / 64);
    const unsigned grid = (waves + 3) / 4;
    if (a.c.d == 64)
        kv8_read_kernel<64><<<grid, 256, 0, s>>>(a, groups, waves);
    else
        kv8_read_kernel<128><<<grid, 256, 0, s>>>(a, groups, waves);
}

void launch_kv8_undo(int B, int pos, const Kv8Cache& c, const Kv8Undo& u, hipStream_t s) {
    if (B > 0) kv8_undo_kernel<<<(unsigned)B * 2 * c.H, 64, 0, s>>>(pos, c, u);
}

}  // namespace ie
