// paged_cache.hip — rows into the paged cache with their rotation, and rows of
// an accepted path moved together (include/ie_paged.h).
#include <algorithm>

#include "device_util.h"
#include "paged.h"

namespace ie {
namespace {

// Page and row of position p, as the cache's row number.
__device__ __forceinline__ uint32_t cache_row(const PageMap& m, const int* table, int p) {
    const int page = m.mul ? (int)(__umulhi((uint32_t)p, m.mul) >> m.shift) : p;
    return (uint32_t)table[page] * (uint32_t)m.block + (uint32_t)(p - page * m.block);
}

// cos and sin of pos * freq.  The product has 31 + 24 bits and the turns' rest is
// taken from it in 64 bits; the rest as an fp32 number and what that leaves,
// whose first order is added: without it a rest near half a turn is off by 2^-25 of
// a turn, 1.9e-7, three times what the functions themselves are.
__device__ __forceinline__ float2 turn(long long pos, float freq) {
    const double turns = (double)pos * (double)freq * 0.15915494309189535;
    const double rest = turns - rint(turns);
    const float hi = (float)rest, lo = (float)(rest - (double)hi) * 6.2831853f;
    float s, c;
    sincospif(2.0f * hi, &s, &c);
    return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
}
__device__ __forceinline__ void rotate(float& x, float& y, float2 cs) {
    const float a = x;
    x = fmaf(a, cs.x, -(y * cs.y));
    y = fmaf(y, cs.x, a * cs.y);
}

template <typename KV>
__device__ __forceinline__ void put4(KV* p, float4 v) {
    if constexpr (sizeof(KV) == 4)
        *reinterpret_cast<float4*>(p) = v;
    else
        *reinterpret_cast<ushort4*>(p) =
            make_ushort4(f32_to_bf16_rne(v.x), f32_to_bf16_rne(v.y), f32_to_bf16_rne(v.z), f32_to_bf16_rne(v.w));
}
template <typename KV>
__device__ __forceinline__ void put1(KV* p, float v) {
    if constexpr (sizeof(KV) == 4)
        *p = v;
    else
        *p = f32_to_bf16_rne(v);
}

// A row (b, t): which it is and where it goes.
struct RowOf {
    int b;
    bool live, stored;
    long long pos;  // of its angles
    int at;         // in the cache
};
__device__ __forceinline__ RowOf row_of(const RopeWrite& a, int row) {
    RowOf r;
    r.b = row / a.P;
    const int t = row - r.b * a.P;
    r.live = !a.lens || t < a.lens[r.b];
    const long long at = (long long)a.starts[r.b] + t;
    r.stored = at >= 0 && at < (long long)a.pages.nbps * a.pages.block;
    r.at = r.stored ? (int)at : 0;
    r.pos = a.positions ? a.positions[row] : at;
    return r;
}

// TOK rows to a workgroup (blockDim.x / units of them, one where a row has more
// units than threads; then gridDim.y workgroups share it).  A unit is eight channels
// of a head: a rotated pair of fours (i .., i + rot / 2 ..), eight side by side where
// pairs are interleaved, and eight side by side behind the rotated ones and of V.
// The row's angles are computed once a workgroup, for all of its heads, while the
// first unit's channels arrive.  Bound by HBM: reads 4 bytes a value, writes 4 of Q
// and 2 or 4 of K and V.
template <typename KV>
__global__ __launch_bounds__(256) void rope_write_kernel(RopeWrite a, int units, int tok) {
    __shared__ float2 cs[512];  // (tok * rot / 2: a row has at least d / 4 units)
    const int half = a.rot / 2, per = a.d / 8, rows = a.B * a.P;
    const int lt = tok > 1 ? threadIdx.x / units : 0;
    const int row = blockIdx.x * tok + lt;
    int u = tok > 1 ? threadIdx.x - lt * units : blockIdx.y * 256 + threadIdx.x;
    const bool mine = lt < tok && row < rows;
    RowOf r{};
    if (mine) r = row_of(a, row);
    const size_t q_src = (size_t)row * a.q_ld, kv_src = (size_t)row * a.kv_ld;

    float4 x, y;
    int head = 0, c = 0, c2 = 0;
    auto fetch = [&] {
        head = u / per;
        const int w = u - head * per;
        const bool pair = !a.interleaved && head < a.H_q + a.H_kv && 4 * w < half;
        // (fours of the first half stand for both halves, so the rest begins at rot)
        c = pair ? 4 * w : 8 * w;
        c2 = pair ? c + half : c + 4;
        const float* p = head < a.H_q ? a.Q + q_src + (size_t)head * a.d
                         : head < a.H_q + a.H_kv ? a.K + kv_src + (size_t)(head - a.H_q) * a.d
                                                 : a.V + kv_src + (size_t)(head - a.H_q - a.H_kv) * a.d;
        x = *reinterpret_cast<const float4*>(p + c);
        y = *reinterpret_cast<const float4*>(p + c2);
    };
    const bool go = mine && r.live && u < units;
    if (go) fetch();
    for (int i = threadIdx.x; i < tok * half; i += 256) {
        const int rr = blockIdx.x * tok + i / half;
        if (rr < rows) {
            const RowOf o = row_of(a, rr);
            cs[i] = turn(o.pos, a.freq[i % half]);
        }
    }
    __syncthreads();
    if (!go) return;
    const float2* t = cs + lt * half;
    const size_t slot = r.stored ? cache_row(a.pages, a.pages.table + (size_t)r.b * a.pages.nbps, r.at) : 0;
    for (;;) {
        if (head < a.H_q + a.H_kv && c < a.rot) {
            if (a.interleaved) {
                rotate(x.x, x.y, t[c / 2]);
                rotate(x.z, x.w, t[c / 2 + 1]);
                rotate(y.x, y.y, t[c / 2 + 2]);
                rotate(y.z, y.w, t[c / 2 + 3]);
            } else if (c < half) {
                rotate(x.x, y.x, t[c]);
                rotate(x.y, y.y, t[c + 1]);
                rotate(x.z, y.z, t[c + 2]);
                rotate(x.w, y.w, t[c + 3]);
            }
        }
        if (head < a.H_q) {
            float* o = a.out + ((size_t)row * a.H_q + head) * a.d;
            *reinterpret_cast<float4*>(o + c) = x;
            *reinterpret_cast<float4*>(o + c2) = y;
        } else if (r.stored) {
            const bool key = head < a.H_q + a.H_kv;
            KV* o = static_cast<KV*>(key ? a.k : a.v) + (slot * a.H_kv + (head - a.H_q - (key ? 0 : a.H_kv))) * a.d;
            put4(o + c, x);
            put4(o + c2, y);
        }
        if (tok > 1) return;
        u += gridDim.y * 256;
        if (u >= units) return;
        fetch();
    }
}

// Any rot: a thread takes a value and its partner.
template <typename KV>
__global__ __launch_bounds__(256) void rope_write_any_kernel(RopeWrite a) {
    const int row = blockIdx.x, half = a.rot / 2;
    const RowOf r = row_of(a, row);
    if (!r.live) return;
    const size_t q_src = (size_t)row * a.q_ld, kv_src = (size_t)row * a.kv_ld;
    const size_t slot = r.stored ? cache_row(a.pages, a.pages.table + (size_t)r.b * a.pages.nbps, r.at) : 0;
    // of a head: its pairs, then the values behind them; V: its values
    const int turned = half + (a.d - a.rot), n = (a.H_q + a.H_kv) * turned + a.H_kv * a.d;
    for (int u = blockIdx.y * 256 + threadIdx.x; u < n; u += gridDim.y * 256) {
        const int of_v = u - (a.H_q + a.H_kv) * turned;
        if (of_v >= 0) {
            if (r.stored) put1(static_cast<KV*>(a.v) + slot * a.H_kv * a.d + of_v, a.V[kv_src + of_v]);
            continue;
        }
        const int head = u / turned, i = u - head * turned;
        const bool pair = i < half;
        const int c = pair ? (a.interleaved ? 2 * i : i) : i + half, c2 = a.interleaved ? c + 1 : c + half;
        const float* p = head < a.H_q ? a.Q + q_src + (size_t)head * a.d : a.K + kv_src + (size_t)(head - a.H_q) * a.d;
        float x = p[c], y = pair ? p[c2] : 0.0f;
        if (pair) rotate(x, y, turn(r.pos, a.freq[i]));
        if (head < a.H_q) {
            float* o = a.out + ((size_t)row * a.H_q + head) * a.d;
            o[c] = x;
            if (pair) o[c2] = y;
        } else if (r.stored) {
            KV* o = static_cast<KV*>(a.k) + (slot * a.H_kv + (head - a.H_q)) * a.d;
            put1(o + c, x);
            if (pair) put1(o + c2, y);
        }
    }
}

// A workgroup for a (sequence, layer): K's 16-byte chunks of a row and V's behind them, a thread the same one of every
// row, in the path's order.  An entry's row lies at or behind the place it goes to, and every later entry's behind
// that place, so in order no row is overwritten before it is read; eight are read ahead of eight writes.  Bound by the
// chain count, path, table, row, not by the bytes: a wave looks up 64 entries side by side (one after another, four
// rows ahead of four writes: 32 x 32 layers of 8 x 128 bf16 30.2 us, so XXX).
constexpr int kLayers = 64;
struct KeepArgs {
    void* cache[2][kLayers];
    PageMap pages;
    int most, chunks;
    const int *ctx, *paths, *counts;
};
__global__ __launch_bounds__(256) void kv_keep_kernel(KeepArgs a) {
    __shared__ uint32_t from[64], to[64];
    __shared__ int valid;
    const int b = blockIdx.y, lane = threadIdx.x & 63;
    const int* table = a.pages.table + (size_t)b * a.pages.nbps;
    const int* path = a.paths + (size_t)b * a.most;
    const int ctx = a.ctx[b], n = min(a.counts[b], a.most);
    const long long end = (long long)a.pages.nbps * a.pages.block;
    if (ctx < 0) return;
    for (int j0 = 0; j0 < n; j0 += 64) {
        if (threadIdx.x < 64) {
            const int j = j0 + lane, p = j < n ? path[j] : -1, before = j > 0 && j < n ? path[j - 1] : -1;
            const bool ok = p > before && (long long)ctx + p < end;
            const uint64_t bad = ~__ballot(ok);
            const int count = bad ? __builtin_ctzll(bad) : 64;  // (the path ends at the first that is not)
            if (lane < count) {
                from[lane] = cache_row(a.pages, table, ctx + p);
                to[lane] = cache_row(a.pages, table, ctx + j);
            }
            if (lane == 0) valid = count;
        }
        __syncthreads();
        const int count = valid;
        for (int c = threadIdx.x; c < 2 * a.chunks; c += 256) {
            const bool v = c >= a.chunks;
            uint4* cache = static_cast<uint4*>(a.cache[v][blockIdx.x]) + (v ? c - a.chunks : c);
            for (int k0 = 0; k0 < count; k0 += 8) {
                uint4 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k0 + k < count && from[k0 + k] != to[k0 + k]) x[k] = cache[(size_t)from[k0 + k] * a.chunks];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k0 + k < count && from[k0 + k] != to[k0 + k]) cache[(size_t)to[k0 + k] * a.chunks] = x[k];
            }
        }
        if (count < 64) return;
        __syncthreads();
    }
}

}  // namespace

void launch_rope_write(const RopeWrite& a, hipStream_t s) {
    const bool half = a.kv_dtype == IE_KV_BF16;
    const int rows = a.B * a.P;
    // fours of a pair stay whole, and what is not rotated is whole eights
    if (a.rot % 8 == 0) {
        const int units = (a.H_q + 2 * a.H_kv) * a.d / 8;
        const int tok = std::max(1, 256 / units);
        const dim3 grid((unsigned)((rows + tok - 1) / tok), tok > 1 ? 1u : (unsigned)std::min(65535, (units + 255) / 256));
        auto* k = half ? rope_write_kernel<uint16_t> : rope_write_kernel<float>;
        k<<<grid, 256, 0, s>>>(a, units, tok);
    } else {
        const long long n = (long long)(a.H_q + 2 * a.H_kv) * a.d;
        auto* k = half ? rope_write_any_kernel<uint16_t> : rope_write_any_kernel<float>;
        k<<<dim3((unsigned)rows, (unsigned)std::min(65535ll, (n + 255) / 256)), 256, 0, s>>>(a);
    }
}

void launch_kv_keep(const KeepRows& a, hipStream_t s) {
    for (int l0 = 0; l0 < a.layers; l0 += kLayers) {
        const int n = std::min(kLayers, a.layers - l0);
        KeepArgs k{};
        for (int l = 0; l < n; ++l) {
            k.cache[0][l] = a.k[l0 + l];
            k.cache[1][l] = a.v[l0 + l];
        }
        k.pages = a.pages;
        k.most = a.most;
        k.chunks = a.row_bytes / 16;
        k.ctx = a.ctx;
        k.paths = a.paths;
        k.counts = a.counts;
        kv_keep_kernel<<<dim3((unsigned)n, (unsigned)a.B), 256, 0, s>>>(k);
    }
}

}  // namespace ie
