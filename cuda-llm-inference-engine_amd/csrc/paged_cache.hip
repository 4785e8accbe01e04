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

// cos and sin of pos * freq.  The product has up to 31 + 24 bits, more than a double: its rounding, exact by
// fma, and the rest of 1 / 2 pi go along, so the turns' rest is right to 2^-50 of a turn as far as a position
// times a frequency has whole turns to take off (2^50).  The rest as an fp32 number and what that leaves,
// whose first order is added: without it a rest near half a turn is off by 2^-25 of
// a turn, 1.9e-7, three times what the functions themselves are.
__device__ __forceinline__ float2 turn(long long pos, float freq) {
    constexpr double per = 0x1.45f306dc9c883p-3, more = -0x1.6b01ec5417056p-57;  // 1 / 2 pi
    const double p = (double)pos * (double)freq, low = fma((double)pos, (double)freq, -p);
    const double rest = fma(p, per, -rint(p * per)) + fma(p, more, low * per);
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

// VEC values side by side: sources, which are read once, past the caches (4 x 2000 rows of 48 x 128 38.3 -> 32.9 us).
template <int VEC>
struct Values {
    float v[VEC];
};
template <int VEC>
__device__ __forceinline__ Values<VEC> get(const float* p) {
    typedef float Raw __attribute__((ext_vector_type(VEC)));
    Values<VEC> r;
    if constexpr (VEC == 1) {
        r.v[0] = __builtin_nontemporal_load(p);
    } else {
        const Raw x = __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p));
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = x[i];
    }
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, const Values<VEC>& x) {
    T y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if constexpr (sizeof(T) == 4) y[i] = x.v[i];
        else y[i] = f32_to_bf16_rne(x.v[i]);
    }
    struct alignas(sizeof(T) * VEC) Whole {
        T v[VEC];
    };
    *reinterpret_cast<Whole*>(p) = __builtin_bit_cast(Whole, y);
}

constexpr int kUnits = 3;  // of a thread, where there are rows enough
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

// A unit is 2 VEC channels of a head: rotated pairs, VEC of the first half (i ..) and theirs of the second (i + rot / 2
// ..), or side by side where pairs are interleaved, behind the rotated ones and of V.  VEC is 4 where rot is a multiple of 8,
// 2 of 4, else 1.  `tok` rows to a workgroup where a row has few units, else gridDim.y workgroups to a row, and N units
// to a thread.  A row's angles are computed once a workgroup, for all of its heads, while the units' channels arrive.
// Bound by HBM: reads 4 bytes a value, writes 4 of Q and 2 or 4 of K and V; four ragged sequences of at most 2000 rows
// of (32 + 16) x 128 into bf16 pages (150 MB) take 36 us, 4.2 TB/s, with one unit a thread 43.
template <typename KV, int VEC, int N>
__global__ __launch_bounds__(256) void rope_write_kernel(RopeWrite a, int units, int tok) {
    __shared__ float2 cs[512];  // (tok * rot / 2: a row has at least d / VEC units)
    const int half = a.rot / 2, per = a.d / (2 * VEC), rows = a.B * a.P;
    const int lt = tok > 1 ? threadIdx.x / units : 0;
    const int row = blockIdx.x * tok + lt;
    const int u0 = tok > 1 ? threadIdx.x - lt * units : blockIdx.y * (256 * N) + threadIdx.x;
    const bool mine = lt < tok && row < rows;
    RowOf r{};
    if (mine) r = row_of(a, row);
    const size_t q_src = (size_t)row * a.q_ld, kv_src = (size_t)row * a.kv_ld;
    const bool go = mine && r.live;

    Values<VEC> x[N], y[N];
    int head[N], c[N], c2[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int u = u0 + 256 * n;
        head[n] = u / per;
        const int w = u - head[n] * per;
        const bool pair = !a.interleaved && head[n] < a.H_q + a.H_kv && VEC * w < half;
        // (a unit of pairs stands for both halves, so the rest begins at rot)
        c[n] = pair ? VEC * w : 2 * VEC * w;
        c2[n] = pair ? c[n] + half : c[n] + VEC;
        if (go && u < units) {
            const float* p = head[n] < a.H_q ? a.Q + q_src + (size_t)head[n] * a.d
                             : head[n] < a.H_q + a.H_kv ? a.K + kv_src + (size_t)(head[n] - a.H_q) * a.d
                                                        : a.V + kv_src + (size_t)(head[n] - a.H_q - a.H_kv) * a.d;
            x[n] = get<VEC>(p + c[n]);
            y[n] = get<VEC>(p + c2[n]);
        }
    }
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
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (u0 + 256 * n >= units) return;
        const int h = head[n], i = c[n];
        if (h < a.H_q + a.H_kv && i < a.rot) {
            if (a.interleaved) {
                float z[2 * VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) z[e] = x[n].v[e], z[VEC + e] = y[n].v[e];
#pragma unroll
                for (int e = 0; e < VEC; ++e) rotate(z[2 * e], z[2 * e + 1], t[i / 2 + e]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[n].v[e] = z[e], y[n].v[e] = z[VEC + e];
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) rotate(x[n].v[e], y[n].v[e], t[i + e]);
            }
        }
        if (h < a.H_q) {
            float* o = a.out + ((size_t)row * a.H_q + h) * a.d;
            put(o + i, x[n]);
            put(o + c2[n], y[n]);
        } else if (r.stored) {
            const bool key = h < a.H_q + a.H_kv;
            KV* o = static_cast<KV*>(key ? a.k : a.v) + (slot * a.H_kv + (h - a.H_q - (key ? 0 : a.H_kv))) * a.d;
            put(o + i, x[n]);
            put(o + c2[n], y[n]);
        }
    }
}

template <typename KV, int VEC>
void launch_rope(const RopeWrite& a, hipStream_t s) {
    const long long units = (long long)(a.H_q + 2 * a.H_kv) * a.d / (2 * VEC);
    const int rows = a.B * a.P, tok = (int)std::max(1ll, 256 / units);
    // several units a thread where there are rows enough (a decode step's few are spread over more workgroups), and where
    // a row has more than a grid's second size times them
    const bool many = (rows >= 512 && units > 256) || units > 256ll * 65535;
    const int each = many ? 256 * kUnits : 256;
    const dim3 grid((unsigned)((rows + tok - 1) / tok), tok > 1 ? 1u : (unsigned)((units + each - 1) / each));
    auto* k = many ? rope_write_kernel<KV, VEC, kUnits> : rope_write_kernel<KV, VEC, 1>;
    k<<<grid, 256, 0, s>>>(a, (int)units, tok);
}

// A workgroup for a (sequence, layer): K's 16-byte chunks of a row and V's behind them, a thread the same one of every
// row, in the path's order.  An entry's row lies at or behind the place it goes to, and every later entry's behind
// that place, so in order no row is overwritten before it is read; eight are read ahead of eight writes.  Bound by the
// chain count, path, table, row, not by the bytes: a wave looks up 64 entries side by side (one after another, four
// rows ahead of four writes: 32 x 32 layers of 8 x 128 bf16 30.8 us, so 18.2).
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
    auto go = [&](auto kv) {
        using KV = decltype(kv);
        if (a.rot % 8 == 0) launch_rope<KV, 4>(a, s);
        else if (a.rot % 4 == 0) launch_rope<KV, 2>(a, s);
        else launch_rope<KV, 1>(a, s);
    };
    if (a.kv_dtype == IE_KV_BF16) go(uint16_t{});
    else go(float{});
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
