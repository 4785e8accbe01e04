// paged_capi.cpp — the extern "C" boundary of include/ie_paged.h: every check
// is made here, before any HIP call.
#include <hip/hip_runtime.h>

#include <cmath>
#include <initializer_list>

#include "paged.h"

namespace {
using ie::fail;

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
bool words(std::initializer_list<const void*> p) {
    for (const void* x : p)
        if (!aligned(x, 4)) return false;
    return true;
}
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

// Workgroups of a launch; a grid's threads must stay below 2^32.
constexpr long long kMaxGroups = 1ll << 21;
// Longest context: positions and their tiles' ends stay within an int.
constexpr long long kMaxContext = 1ll << 30;

int check_layout(const char* fn, int B, int H_kv, int d, int kv_dtype, int block_size, int nbps) {
    if (B < 0 || H_kv <= 0 || d <= 0 || nbps < 0)
        return fail(IE_ERR_INVALID, "%s: bad sizes B=%d heads=%d d=%d num_blocks_per_seq=%d", fn, B, H_kv, d, nbps);
    if (d != 64 && d != 128) return fail(IE_ERR_UNSUPPORTED, "%s: head dim %d not in {64,128}", fn, d);
    if (block_size <= 0) return fail(IE_ERR_INVALID, "%s: block_size=%d", fn, block_size);
    if (kv_dtype != IE_KV_F32 && kv_dtype != IE_KV_BF16)
        return fail(IE_ERR_INVALID, "%s: unknown kv_dtype %d", fn, kv_dtype);
    if ((long long)H_kv * d > 1ll << 24) return fail(IE_ERR_UNSUPPORTED, "%s: rows of more than 2^24 values", fn);
    return IE_OK;
}

int check_cache(const char* fn, const void* k, const void* v, const int* table) {
    if (!k || !v || !table) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(table, 4))
        return fail(IE_ERR_INVALID, "%s: the caches must be 16-byte aligned", fn);
    return IE_OK;
}

// Workgroups of 32 rows of an attention call, before splits; past kMaxGroups where they are too many.
long long row_groups(int B, int P, int H_q, int H_kv) {
    const long long n = ((long long)P * (H_q / H_kv) + 31) / 32;
    if (n > kMaxGroups || n * H_kv > kMaxGroups) return kMaxGroups + 1;
    return n * H_kv * B;  // (below 2^53)
}

// What both attentions check; keys: positions that a sequence may hold.
int check_attn(const char* fn, ie::PagedAttn& a, long long keys, int block_size, int nbps, float* workspace,
               size_t workspace_bytes, int num_splits) {
    int st = check_layout(fn, a.B, a.H_kv, a.d, a.kv_dtype, block_size, nbps);
    if (st != IE_OK) return st;
    if (a.H_q <= 0 || a.H_q % a.H_kv)
        return fail(IE_ERR_INVALID, "%s: H_q=%d not a multiple of H_kv=%d", fn, a.H_q, a.H_kv);
    if (a.P < 0 || a.max_ctx < 0 || a.window < 0)
        return fail(IE_ERR_INVALID, "%s: %d tokens, max_context_len=%d, window=%d", fn, a.P, a.max_ctx, a.window);
    if (keys > (long long)nbps * block_size)
        return fail(IE_ERR_INVALID, "%s: %lld positions do not fit %d blocks of %d", fn, keys, nbps, block_size);
    if (keys > kMaxContext) return fail(IE_ERR_UNSUPPORTED, "%s: positions past 2^30", fn);
    if (!std::isfinite(a.scale) || !std::isfinite(a.cap) || a.scale < 0 || a.cap < 0)
        return fail(IE_ERR_INVALID, "%s: scale=%g cap=%g", fn, (double)a.scale, (double)a.cap);
    if (a.B == 0 || a.P == 0) return IE_OK;
    const long long groups = row_groups(a.B, a.P, a.H_q, a.H_kv);
    if (groups > kMaxGroups)
        return fail(IE_ERR_UNSUPPORTED, "%s: grid too large (ceil(tokens x heads / 32) x KV heads x B > 2^21)", fn);
    if (!a.Q || !a.O || !a.starts) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(a.Q, 16) || !aligned(a.O, 16))
        return fail(IE_ERR_INVALID, "%s: Q and O must be 16-byte aligned", fn);
    if (!words({a.starts, a.lens, a.first, a.end, a.parents, a.slopes}))
        return fail(IE_ERR_INVALID, "%s: an array of ints or floats is not 4-byte aligned", fn);
    const size_t bytes = (size_t)a.B * a.P * a.H_q * a.d * sizeof(float);
    if (overlap(a.Q, bytes, a.O, bytes)) return fail(IE_ERR_INVALID, "%s: O overlaps Q", fn);
    if (keys > 0 && (st = check_cache(fn, a.k, a.v, a.pages.table)) != IE_OK) return st;
    if (a.scale == 0.0f) a.scale = 1.0f / sqrtf((float)a.d);
    // cap tanh(s / cap) is s to fp32 where |s| < 2^-12 cap; from 2^80 on a cap is none (folded into the queries it would
    // bring their values below what three bf16 parts hold, and times log2(e) the largest pass fp32).
    if (a.cap >= 0x1p80f) a.cap = 0;
    // The factor of a product q.k, to base 2 where there is no cap
    const float factor = a.cap > 0 ? a.scale / a.cap : a.scale * 1.4426950408889634f;
    if (!std::isfinite(factor) || (a.cap > 0 && factor < 0x1p-126f))
        return fail(IE_ERR_INVALID, "%s: scale=%g and cap=%g leave fp32's normal range", fn, (double)a.scale, (double)a.cap);
    a.splits = workspace ? ie_paged_attn_num_splits(a.B, a.P, a.H_q, a.H_kv, a.d, a.kv_dtype, (int)keys, a.window, num_splits) : 1;
    if (!workspace && num_splits > 1 &&
        ie_paged_attn_num_splits(a.B, a.P, a.H_q, a.H_kv, a.d, a.kv_dtype, (int)keys, a.window, num_splits) > 1)
        return fail(IE_ERR_INVALID, "%s: null workspace with %d splits", fn, num_splits);
    if (a.splits > 1) {
        const size_t need = ie_paged_attn_workspace_bytes(a.B, a.P, a.H_q, a.d, a.splits);
        if (!aligned(workspace, 16)) return fail(IE_ERR_INVALID, "%s: workspace must be 16-byte aligned", fn);
        if (workspace_bytes < need)
            return fail(IE_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu for %d splits", fn, workspace_bytes, need, a.splits);
        if (overlap(workspace, need, a.Q, bytes) || overlap(workspace, need, a.O, bytes))
            return fail(IE_ERR_INVALID, "%s: workspace overlaps Q or O", fn);
        a.ws = workspace;
    }
    return IE_OK;
}
}  // namespace

extern "C" {

int ie_rope_kv_write(int B, int P, const float* Q_src, const float* K_src, const float* V_src, int q_stride,
                     int kv_stride, int H_q, int H_kv, int d, int rot_dim, int interleaved, const float* inv_freq, const int* starts,
                     const int* lens, const int* positions, float* Q_out, void* k_cache, void* v_cache, int kv_dtype,
                     const int* block_table, int num_blocks_per_seq, int block_size, ie_stream_t stream) {
    const char* fn = "rope_kv_write";
    int st = check_layout(fn, B, H_kv, d, kv_dtype, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (P < 0 || H_q < 0) return fail(IE_ERR_INVALID, "%s: P=%d H_q=%d", fn, P, H_q);
    if (rot_dim < 0 || rot_dim > d || rot_dim % 2)
        return fail(IE_ERR_INVALID, "%s: rot_dim=%d is odd or outside 0 .. %d", fn, rot_dim, d);
    const long long q_row = (long long)H_q * d, kv_row = (long long)H_kv * d;
    if (q_row > 1ll << 24) return fail(IE_ERR_UNSUPPORTED, "%s: rows of more than 2^24 values", fn);
    if ((H_q > 0 && (q_stride < q_row || q_stride % 4)) || kv_stride < kv_row || kv_stride % 4)
        return fail(IE_ERR_INVALID, "%s: q_stride=%d or kv_stride=%d is below a row (%lld, %lld floats) or no multiple of 4", fn,
                    q_stride, kv_stride, q_row, kv_row);
    if ((long long)num_blocks_per_seq * block_size > kMaxContext)
        return fail(IE_ERR_UNSUPPORTED, "%s: positions past 2^30", fn);
    if (B == 0 || P == 0) return IE_OK;
    if ((long long)B * P > kMaxGroups) return fail(IE_ERR_UNSUPPORTED, "%s: B x P above 2^21 rows", fn);
    if (!K_src || !V_src || !starts || (H_q > 0 && (!Q_src || !Q_out)) || (rot_dim > 0 && !inv_freq))
        return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(Q_src, 16) || !aligned(K_src, 16) || !aligned(V_src, 16) || !aligned(Q_out, 16))
        return fail(IE_ERR_INVALID, "%s: Q_src, K_src, V_src and Q_out must be 16-byte aligned", fn);
    if (!words({inv_freq, starts, lens, positions}))
        return fail(IE_ERR_INVALID, "%s: an array of ints or floats is not 4-byte aligned", fn);
    if ((st = check_cache(fn, k_cache, v_cache, block_table)) != IE_OK) return st;
    const size_t n = (size_t)B * P, out = n * q_row * sizeof(float);
    const size_t q_bytes = ((n - 1) * q_stride + q_row) * sizeof(float), kv_bytes = ((n - 1) * kv_stride + kv_row) * sizeof(float);
    if (H_q > 0 && (overlap(Q_out, out, Q_src, q_bytes) || overlap(Q_out, out, K_src, kv_bytes) ||
                    overlap(Q_out, out, V_src, kv_bytes)))
        return fail(IE_ERR_INVALID, "%s: Q_out overlaps an input", fn);
    ie::RopeWrite a{};
    a.B = B; a.P = P; a.H_q = H_q; a.H_kv = H_kv; a.d = d; a.rot = rot_dim; a.interleaved = interleaved != 0;
    a.Q = Q_src; a.K = K_src; a.V = V_src; a.q_ld = q_stride; a.kv_ld = kv_stride; a.freq = inv_freq;
    a.starts = starts; a.lens = lens; a.positions = positions; a.out = Q_out; a.k = k_cache; a.v = v_cache;
    a.kv_dtype = kv_dtype; a.pages = ie::page_map(block_table, num_blocks_per_seq, block_size);
    ie::launch_rope_write(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

int ie_paged_attn_num_splits(int B, int P, int H_q, int H_kv, int d, int kv_dtype, int max_keys, int window,
                             int num_splits) {
    if (B <= 0 || P <= 0 || H_kv <= 0 || H_q <= 0 || H_q % H_kv || (d != 64 && d != 128) || max_keys <= 0 ||
        (kv_dtype != IE_KV_F32 && kv_dtype != IE_KV_BF16) || window < 0)
        return 1;
    const long long groups = row_groups(B, P, H_q, H_kv);
    if (groups > kMaxGroups) return 1;
    const int s = ie::paged_attn_splits(B, P, H_q, H_kv, d, kv_dtype, max_keys, window, num_splits);
    const long long most = kMaxGroups / groups;
    return s < most ? s : (int)most;
}

size_t ie_paged_attn_workspace_bytes(int B, int P, int H_q, int d, int num_splits) {
    if (B <= 0 || P <= 0 || H_q <= 0 || d <= 0 || num_splits <= 1) return 0;
    return (size_t)B * P * H_q * num_splits * (d + 2) * sizeof(float);
}

int ie_paged_attn(int B, int P, int H_q, int H_kv, int d, const float* Q, const void* k_cache, const void* v_cache,
                  int kv_dtype, const int* block_table, int num_blocks_per_seq, int block_size, const int* starts,
                  const int* lens, int max_context_len, const int* first, const int* end, int window, float scale,
                  float cap, const float* slopes, float* O, float* workspace, size_t workspace_bytes, int num_splits,
                  ie_stream_t stream) {
    const char* fn = "paged_attn";
    ie::PagedAttn a{};
    a.B = B; a.P = P; a.H_q = H_q; a.H_kv = H_kv; a.d = d; a.Q = Q; a.k = k_cache; a.v = v_cache; a.kv_dtype = kv_dtype;
    if (block_size > 0) a.pages = ie::page_map(block_table, num_blocks_per_seq, block_size);
    a.starts = starts; a.lens = lens; a.max_ctx = max_context_len; a.first = first; a.end = end; a.window = window;
    a.scale = scale; a.cap = cap; a.slopes = slopes; a.O = O;
    const int st = check_attn(fn, a, max_context_len, block_size, num_blocks_per_seq, workspace, workspace_bytes, num_splits);
    if (st != IE_OK || B == 0 || P == 0) return st;
    ie::launch_paged_attn(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

int ie_tree_attn(int B, int T, int H_q, int H_kv, int d, const float* Q, const void* k_cache, const void* v_cache,
                 int kv_dtype, const int* block_table, int num_blocks_per_seq, int block_size, const int* context_lens,
                 const int* lens, const int* parents, int max_context_len, int window, float scale, float cap,
                 const float* slopes, float* O, float* workspace, size_t workspace_bytes, int num_splits,
                 ie_stream_t stream) {
    const char* fn = "tree_attn";
    if (T > IE_TREE_MAX) return fail(IE_ERR_UNSUPPORTED, "%s: %d nodes, at most %d", fn, T, IE_TREE_MAX);
    ie::PagedAttn a{};
    a.B = B; a.P = T; a.H_q = H_q; a.H_kv = H_kv; a.d = d; a.Q = Q; a.k = k_cache; a.v = v_cache; a.kv_dtype = kv_dtype;
    if (block_size > 0) a.pages = ie::page_map(block_table, num_blocks_per_seq, block_size);
    a.starts = context_lens; a.lens = lens; a.max_ctx = max_context_len; a.parents = parents; a.window = window;
    a.scale = scale; a.cap = cap; a.slopes = slopes; a.O = O;
    const int st = check_attn(fn, a, (long long)max_context_len + T, block_size, num_blocks_per_seq, workspace, workspace_bytes,
                              num_splits);
    if (st != IE_OK || B == 0 || T == 0) return st;
    if (!parents) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    ie::launch_paged_attn(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

int ie_kv_cache_keep(int B, int max_count, int n_layers, void* const* k_caches, void* const* v_caches, int kv_dtype,
                     const int* block_table, int num_blocks_per_seq, int block_size, int n_heads, int d_head,
                     const int* context_lens, const int* paths, const int* counts, ie_stream_t stream) {
    const char* fn = "kv_cache_keep";
    int st = check_layout(fn, B, n_heads, d_head, kv_dtype, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (max_count < 0 || n_layers < 0) return fail(IE_ERR_INVALID, "%s: max_count=%d n_layers=%d", fn, max_count, n_layers);
    if ((long long)num_blocks_per_seq * block_size > kMaxContext)
        return fail(IE_ERR_UNSUPPORTED, "%s: positions past 2^30", fn);
    if (B > 65535) return fail(IE_ERR_UNSUPPORTED, "%s: more than 65535 sequences", fn);
    if (B == 0 || max_count == 0 || n_layers == 0) return IE_OK;
    if (!k_caches || !v_caches || !context_lens || !paths || !counts) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!words({context_lens, paths, counts}))
        return fail(IE_ERR_INVALID, "%s: an array of ints is not 4-byte aligned", fn);
    for (int l = 0; l < n_layers; ++l)
        if ((st = check_cache(fn, k_caches[l], v_caches[l], block_table)) != IE_OK) return st;
    ie::KeepRows a{};
    a.B = B; a.most = max_count; a.layers = n_layers; a.k = k_caches; a.v = v_caches;
    a.pages = ie::page_map(block_table, num_blocks_per_seq, block_size);
    a.row_bytes = n_heads * d_head * (kv_dtype == IE_KV_BF16 ? 2 : 4);
    a.ctx = context_lens; a.paths = paths; a.counts = counts;
    ie::launch_kv_keep(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

}  // extern "C"
