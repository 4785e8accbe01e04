// kv8_cache.hip — rows into and out of the 8-bit paged KV cache
// (include/ie_kv8.h has the layout and the rule that scales follow).
//
// A page of one head is cut into tiles of 16 tokens x 64 channels, one wave
// (or T tiles of one wave) each, so a tile's codes are 1 KB that the wave
// stores as one 16-byte word a lane:
//   K tile (rows of d bytes): lane l holds token l / 4, channels 16 (l % 4) ..
//   V tile ([channel][16 tokens]): lane l holds channel l of all 16 tokens
// and the fp32 rows are read as 64 contiguous bytes a lane (K) or 256 a wave
// (V).  A workgroup holds all tiles of one (sequence, page, head) of K or of
// V in registers, so the page's maximum, its codes and (where the scale had to
// grow) the earlier rows' new codes come from one pass over the data.
#include <algorithm>

#include "device_util.h"
#include "kv8.h"

namespace ie {
namespace {

constexpr float kFloor = 0x1p-100f;  // least scale (1 / scale stays finite)

__device__ __forceinline__ uint32_t fbits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float bitsf(uint32_t x) { return __builtin_bit_cast(float, x); }
// Larger of two values >= +0, where NaN is the largest.
__device__ __forceinline__ float max_nan(float a, float b) { return bitsf(max(fbits(a), fbits(b))); }
// rint as an int; NaN gives 0.  |x| <= 127 * (1 + 2^-22) here: need / scale <= 1.
__device__ __forceinline__ int code(float x) { return (int)rintf(x); }
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}
__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A lane's 16-byte word of tile t of a page.
template <int D>
__device__ __forceinline__ int word_of(int t, bool is_v, int lane) {
    constexpr int HALVES = D / 64;
    const int c0 = t % HALVES * 64;
    return t / HALVES * D + (is_v ? c0 + lane : (lane >> 2) * (D / 16) + c0 / 16 + (lane & 3));
}

// blockIdx.x = ((b * npages + page) * H + h) * 2 + (K or V)
template <int D, int T>
__global__ __launch_bounds__(1024) void kv8_write_kernel(Kv8Write a, int npages) {
    constexpr int HALVES = D / 64;
    __shared__ uint32_t wave_mx[16];
    __shared__ float had_sh;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
    unsigned id = blockIdx.x;
    const bool is_v = id & 1;
    id >>= 1;
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
    int8_t* codes = (is_v ? a.c.v : a.c.k) + pair * ((size_t)bs * D);
    float* scale_at = (is_v ? a.c.vs : a.c.ks) + pair;
    const float* src = (is_v ? a.V : a.K) + (size_t)b * a.P * a.ld + (size_t)h * D;

    float x[T][16];
    u32x4 was[T];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int t = wid * T + i, row0 = (t / HALVES) * 16, c0 = (t % HALVES) * 64;
        if (is_v) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = row0 + r;
                x[i][r] = row >= r0 && row < r1 ? src[(size_t)(page0 + row - start) * a.ld + c0 + lane] : 0.0f;
            }
        } else {
            const int row = row0 + (lane >> 2);
            const bool fresh = row >= r0 && row < r1;
            const float4* p = reinterpret_cast<const float4*>(src + (size_t)(fresh ? page0 + row - start : 0) * a.ld +
                                                              c0 + (lane & 3) * 16);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 v = fresh ? p[q] : make_float4(0.f, 0.f, 0.f, 0.f);
                x[i][4 * q] = v.x; x[i][4 * q + 1] = v.y; x[i][4 * q + 2] = v.z; x[i][4 * q + 3] = v.w;
            }
        }
        // the bytes that this call does not write anew
        if (row0 < r0 || row0 + 16 > r1) was[i] = reinterpret_cast<const u32x4*>(codes)[word_of<D>(t, is_v, lane)];
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = max(mx, fbits(x[i][e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    // One wave reads the old scale, so that it is read before it is replaced.
    if (wid == 0 && lane == 0) had_sh = r0 > 0 ? *scale_at : 0.0f;
    if (lane == 0) wave_mx[wid] = mx;
    __syncthreads();
    for (int w = 0; w < nw; ++w) mx = max(mx, wave_mx[w]);
    const float had = had_sh;
    const float need = max_nan(bitsf(mx) / 127.0f, kFloor);
    const float scale = r0 == 0 ? need : need <= had ? had : max_nan(need, 1.25f * had);
    const float inv = 1.0f / scale;
    const bool grew = r0 > 0 && !(scale == had);
    const float move = had * inv;
    if (threadIdx.x == 0 && (r0 == 0 || grew)) *scale_at = scale;
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int t = wid * T + i, row0 = (t / HALVES) * 16;
        if (row0 >= r1 || (row0 + 16 <= r0 && !grew)) continue;  // nothing of this tile changes (uniform)
        u32x4 out;
        const bool whole = row0 >= r0 && row0 + 16 <= r1;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            int q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = row0 + (is_v ? 4 * w + e : lane >> 2);
                q[e] = code(x[i][4 * w + e] * inv);
                if (!whole) {
                    const int old = byte_of(was[i][w], e);
                    q[e] = row < r0 ? (grew ? code((float)old * move) : old) : row < r1 ? q[e] : old;
                }
            }
            out[w] = pack4(q[0], q[1], q[2], q[3]);
        }
        reinterpret_cast<u32x4*>(codes)[word_of<D>(t, is_v, lane)] = out;
    }
}

// One wave per (sequence, 16-token group, head, 64 channels) of K and of V.
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8Read a, int groups, unsigned waves) {
    constexpr int HALVES = D / 64;
    const int lane = threadIdx.x & 63;
    unsigned id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= waves) return;
    const int c0 = (int)(id % HALVES) * 64;
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
    u32x4 kw = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
    float ks = 0.0f, vs = 0.0f;
    if (first >= 0 && first < lim) {
        const size_t pair = (size_t)a.c.table[(size_t)b * a.c.nbps + (first >> lg)] * H + h;
        const size_t at = pair * ((size_t)D << lg) + (size_t)(first & ((1 << lg) - 1)) * D;
        kw = reinterpret_cast<const u32x4*>(a.c.k + at)[word_of<D>(c0 / 64, false, lane)];
        vw = reinterpret_cast<const u32x4*>(a.c.v + at)[word_of<D>(c0 / 64, true, lane)];
        ks = a.c.ks[pair];
        vs = a.c.vs[pair];
    }
    const size_t row_n = (size_t)H * D;
    const size_t base = (size_t)b * a.n * row_n + (size_t)h * D + c0;
    {
        const long long pos = first + (lane >> 2);
        if (pos >= start && pos < end) {
            float4* dst = reinterpret_cast<float4*>(a.K + base + (size_t)(pos - start) * row_n + (lane & 3) * 16);
            const float s = pos < lim ? ks : 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t w = pos < lim ? kw[q] : 0;
                dst[q] = make_float4((float)byte_of(w, 0) * s, (float)byte_of(w, 1) * s, (float)byte_of(w, 2) * s,
                                     (float)byte_of(w, 3) * s);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long pos = first + r;
        if (pos >= start && pos < end)
            a.V[base + (size_t)(pos - start) * row_n + lane] = pos < lim ? (float)byte_of(vw[r / 4], r % 4) * vs : 0.0f;
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

}  // namespace ie
