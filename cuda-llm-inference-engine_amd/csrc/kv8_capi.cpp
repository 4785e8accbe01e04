// kv8_capi.cpp — the extern "C" boundary of the 8-bit KV cache
// (include/ie_kv8.h): every check is made here, before any HIP call.
#include <hip/hip_runtime.h>

#include "kv8.h"

namespace {
using ie::fail;

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Workgroups of a launch; a grid's threads must stay below 2^32.
constexpr long long kMaxGroups = 1ll << 21;
// Pages x heads of a write: two workgroups of up to 1024 threads each.
constexpr long long kMaxWritten = 1ll << 20;
// Longest context: positions and their tiles' ends stay within an int.
constexpr long long kMaxContext = 1ll << 30;

int check_layout(const char* fn, int B, int H_kv, int d, int block_size, int nbps) {
    if (B < 0 || H_kv <= 0 || d <= 0 || nbps < 0)
        return fail(IE_ERR_INVALID, "%s: bad sizes B=%d heads=%d d=%d num_blocks_per_seq=%d", fn, B, H_kv, d, nbps);
    if (d != 64 && d != 128) return fail(IE_ERR_UNSUPPORTED, "%s: head dim %d not in {64,128}", fn, d);
    if (block_size <= 0) return fail(IE_ERR_INVALID, "%s: block_size=%d", fn, block_size);
    if (block_size < 16 || block_size > 256 || (block_size & (block_size - 1)))
        return fail(IE_ERR_UNSUPPORTED, "%s: block_size %d not in {16,32,64,128,256}", fn, block_size);
    return IE_OK;
}

int check_cache(const char* fn, const void* k, const void* v, const float* ks, const float* vs, const int* table) {
    if (!k || !v || !ks || !vs || !table) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(ks, 4) || !aligned(vs, 4) || !aligned(table, 4))
        return fail(IE_ERR_INVALID, "%s: the caches must be 16-byte aligned", fn);
    return IE_OK;
}

ie::Kv8Cache cache(const void* k, const void* v, const float* ks, const float* vs, const int* table, int nbps, int H,
                   int d, int block_size) {
    ie::Kv8Cache c{};
    c.k = static_cast<int8_t*>(const_cast<void*>(k));
    c.v = static_cast<int8_t*>(const_cast<void*>(v));
    c.ks = const_cast<float*>(ks);
    c.vs = const_cast<float*>(vs);
    c.table = table;
    c.nbps = nbps;
    c.H = H;
    c.d = d;
    c.bs_log2 = __builtin_ctz((unsigned)block_size);
    return c;
}

int check_source(const char* fn, const float* K, const float* V, int src_stride, int n_heads, int d_head) {
    if (src_stride < (long long)n_heads * d_head || src_stride % 4)
        return fail(IE_ERR_INVALID, "%s: src_stride=%d is below n_heads * d_head = %lld or no multiple of 4", fn,
                    src_stride, (long long)n_heads * d_head);
    if (!K || !V) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(K, 16) || !aligned(V, 16)) return fail(IE_ERR_INVALID, "%s: K_src and V_src must be 16-byte aligned", fn);
    return IE_OK;
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

int check_attn(const char* fn, int H_q, int H_kv, int d, long long rows, const float* Q, const float* O) {
    if (!Q || !O) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(Q, 16) || !aligned(O, 16)) return fail(IE_ERR_INVALID, "%s: Q and O must be 16-byte aligned", fn);
    const size_t bytes = (size_t)rows * H_q * d * sizeof(float);
    if (overlap(Q, bytes, O, bytes)) return fail(IE_ERR_INVALID, "%s: O overlaps Q", fn);
    return IE_OK;
}

// A prompt's workgroups of 16 tokens (each product is below 2^63).
bool too_many(int B, int P, int H_q) {
    const long long n = (long long)((P + 15) / 16) * H_q;
    return n > kMaxGroups || n * B > kMaxGroups;
}
}  // namespace

extern "C" {

int ie_kv8_cache_write(int B, int P, const float* K_src, const float* V_src, int src_stride, void* k_cache,
                       void* v_cache, float* k_scales, float* v_scales, const int* block_table,
                       int num_blocks_per_seq, int start_pos, int n_heads, int d_head, int block_size,
                       ie_stream_t stream) {
    const char* fn = "kv8_cache_write";
    int st = check_layout(fn, B, n_heads, d_head, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (P < 0 || start_pos < 0) return fail(IE_ERR_INVALID, "%s: P=%d start_pos=%d", fn, P, start_pos);
    if ((long long)start_pos + P > (long long)num_blocks_per_seq * block_size)
        return fail(IE_ERR_INVALID, "%s: positions up to %lld do not fit %d blocks of %d", fn, (long long)start_pos + P,
                    num_blocks_per_seq, block_size);
    if ((long long)start_pos + P > kMaxContext) return fail(IE_ERR_UNSUPPORTED, "%s: positions past 2^30", fn);
    if (B == 0 || P == 0) return IE_OK;
    if ((st = check_source(fn, K_src, V_src, src_stride, n_heads, d_head)) != IE_OK) return st;
    if ((st = check_cache(fn, k_cache, v_cache, k_scales, v_scales, block_table)) != IE_OK) return st;
    const long long pages = ((long long)start_pos + P - 1) / block_size - start_pos / block_size + 1;
    if (pages * n_heads > kMaxWritten || pages * n_heads * B > kMaxWritten)
        return fail(IE_ERR_UNSUPPORTED, "%s: more than 2^20 pages x heads in one call", fn);
    ie::Kv8Write a{};
    a.B = B; a.P = P; a.K = K_src; a.V = V_src; a.ld = src_stride;
    a.c = cache(k_cache, v_cache, k_scales, v_scales, block_table, num_blocks_per_seq, n_heads, d_head, block_size);
    a.start = start_pos;
    ie::launch_kv8_write(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

int ie_kv8_cache_append_batch(int B, const float* K_src, const float* V_src, int src_stride, void* k_cache,
                              void* v_cache, float* k_scales, float* v_scales, const int* block_table,
                              int num_blocks_per_seq, const int* positions, int n_heads, int d_head, int block_size,
                              ie_stream_t stream) {
    const char* fn = "kv8_cache_append_batch";
    int st = check_layout(fn, B, n_heads, d_head, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (B == 0) return IE_OK;
    if ((st = check_source(fn, K_src, V_src, src_stride, n_heads, d_head)) != IE_OK) return st;
    if ((st = check_cache(fn, k_cache, v_cache, k_scales, v_scales, block_table)) != IE_OK) return st;
    if (!positions) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if ((long long)B * n_heads > kMaxWritten) return fail(IE_ERR_UNSUPPORTED, "%s: B x n_heads above 2^20", fn);
    ie::Kv8Write a{};
    a.B = B; a.P = 1; a.K = K_src; a.V = V_src; a.ld = src_stride;
    a.c = cache(k_cache, v_cache, k_scales, v_scales, block_table, num_blocks_per_seq, n_heads, d_head, block_size);
    a.positions = positions;
    ie::launch_kv8_write(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

int ie_kv8_cache_read(int B, int n, const int* starts, const int* context_lens, const void* k_cache,
                      const void* v_cache, const float* k_scales, const float* v_scales, const int* block_table,
                      int num_blocks_per_seq, int n_heads, int d_head, int block_size, float* K_dst, float* V_dst,
                      ie_stream_t stream) {
    const char* fn = "kv8_cache_read";
    int st = check_layout(fn, B, n_heads, d_head, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (n < 0) return fail(IE_ERR_INVALID, "%s: n=%d", fn, n);
    if (B == 0 || n == 0) return IE_OK;
    if ((st = check_cache(fn, k_cache, v_cache, k_scales, v_scales, block_table)) != IE_OK) return st;
    if (!starts || !K_dst || !V_dst) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned(K_dst, 16) || !aligned(V_dst, 16)) return fail(IE_ERR_INVALID, "%s: K_dst and V_dst must be 16-byte aligned", fn);
    const long long groups = (long long)n / 16 + 2;  // 16-token groups that n rows can touch
    if (groups * n_heads > kMaxGroups || groups * n_heads * B > kMaxGroups)
        return fail(IE_ERR_UNSUPPORTED, "%s: more than 2^21 groups of 16 rows x heads in one call", fn);
    ie::Kv8Read a{};
    a.B = B; a.n = n; a.starts = starts; a.lens = context_lens;
    a.c = cache(k_cache, v_cache, k_scales, v_scales, block_table, num_blocks_per_seq, n_heads, d_head, block_size);
    a.K = K_dst; a.V = V_dst;
    ie::launch_kv8_read(a, (hipStream_t)stream);
    return ie::check_launch(fn);
}

int ie_decode_kv8_num_splits(int B, int H_q, int H_kv, int d, int max_context_len, int num_splits) {
    if (B <= 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv || max_context_len <= 0) return 1;
    const int tiles = (int)(((long long)max_context_len + 63) / 64);
    int s = num_splits;
    if (s <= 0) {
        // A workgroup a CU, and a tile at least for each of its four waves; one
        // split where more would spare a wave few tiles (about 0.7 us each at
        // d = 64, 1.3 at 128, against the merge and its launch and, past 64
        // workgroups, the memory they share): 1 x 12 x 64, ctx 1024 6.2 us in one and
        // 6.1 in four, 2048 8.9 and 6.1 in eight; 8 x 12 x 64, ctx 2048 9.5 in one and
        // in two, ctx 8000 26.3, 20.5 in two, 25.2 in three; 1 x (8 x 4) x 128, ctx 1000
        // 9.5 and 8.2 in four.
        const int G = H_q / H_kv, heads = G <= 4 ? 4 : G <= 8 ? 8 : 16;
        const long long units = (long long)B * H_kv * ((G + heads - 1) / heads);
        const int each = (tiles + 3) / 4;
        s = (int)(256 / units);
        s = s < 1 ? 1 : s > each ? each : s;
        const int worth = (d <= 64 ? 4 : 3) * (units > 64 ? 2 : 1);
        if (each - (each + s - 1) / s < worth) s = 1;
    }
    if (s > IE_KV8_MAX_SPLITS) s = IE_KV8_MAX_SPLITS;
    return s < tiles ? s : tiles;
}

int ie_decode_attn_kv8(int B, int H_q, int H_kv, int d, const float* Q, const void* k_cache, const void* v_cache,
                       const float* k_scales, const float* v_scales, const int* block_table, const int* context_lens,
                       int max_context_len, int block_size, int num_blocks_per_seq, float* O, float* workspace,
                       size_t workspace_bytes, int num_splits, ie_stream_t stream) {
    const char* fn = "decode_attn_kv8";
    int st = check_layout(fn, B, H_kv, d, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (H_q <= 0 || H_q % H_kv) return fail(IE_ERR_INVALID, "%s: H_q=%d not a multiple of H_kv=%d", fn, H_q, H_kv);
    if (max_context_len < 0) return fail(IE_ERR_INVALID, "%s: max_context_len=%d", fn, max_context_len);
    if (max_context_len > (long long)num_blocks_per_seq * block_size)
        return fail(IE_ERR_INVALID, "%s: max_context_len=%d does not fit %d blocks of %d", fn, max_context_len,
                    num_blocks_per_seq, block_size);
    if (max_context_len > kMaxContext) return fail(IE_ERR_UNSUPPORTED, "%s: max_context_len past 2^30", fn);
    if (B == 0) return IE_OK;
    if ((long long)B * H_q > kMaxGroups) return fail(IE_ERR_UNSUPPORTED, "%s: B x H_q above 2^21", fn);
    if ((st = check_attn(fn, H_q, H_kv, d, B, Q, O)) != IE_OK) return st;
    if (!context_lens) return fail(IE_ERR_INVALID, "%s: null pointer", fn);
    if (max_context_len > 0 && (st = check_cache(fn, k_cache, v_cache, k_scales, v_scales, block_table)) != IE_OK) return st;
    const int S = ie_decode_kv8_num_splits(B, H_q, H_kv, d, max_context_len, num_splits);
    if ((long long)B * H_q * S > kMaxGroups)
        return fail(IE_ERR_UNSUPPORTED, "%s: B x H_q x splits above 2^21", fn);
    if (S > 1) {
        const size_t need = ie_decode_attn_workspace_bytes(B, H_q, d, S);
        if (!workspace) return fail(IE_ERR_INVALID, "%s: null workspace with %d splits", fn, S);
        if (!aligned(workspace, 4)) return fail(IE_ERR_INVALID, "%s: workspace must be 4-byte aligned", fn);
        if (workspace_bytes < need)
            return fail(IE_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu for %d splits", fn, workspace_bytes, need, S);
    }
    ie::Kv8Attn a{};
    a.B = B; a.P = 1; a.H_q = H_q; a.Q = Q; a.q_ld = H_q * d;
    a.c = cache(k_cache, v_cache, k_scales, v_scales, block_table, num_blocks_per_seq, H_kv, d, block_size);
    a.lens = context_lens; a.max_ctx = max_context_len; a.O = O; a.ws = workspace; a.splits = S;
    st = ie::launch_decode_attn_kv8(a, (hipStream_t)stream);
    return st != IE_OK ? st : ie::check_launch(fn);
}

size_t ie_prefill_kv8_workspace_bytes(int B, int P, int H_q, int H_kv, int d, int start_pos) {
    if (B <= 0 || P <= 0 || H_kv <= 0 || H_q <= 0 || H_q % H_kv || (d != 64 && d != 128) || start_pos < 0 ||
        (long long)start_pos + P > kMaxContext || too_many(B, P, H_q))
        return 0;
    const int S = ie::kv8_prefill_splits(B, P, H_q, H_kv, d, start_pos + P);
    return S > 1 ? (size_t)B * P * H_q * S * (d + 2) * sizeof(float) : 0;
}

int ie_prefill_attn_kv8(int B, int P, int H_q, int H_kv, int d, const float* Q, const void* k_cache,
                        const void* v_cache, const float* k_scales, const float* v_scales, const int* block_table,
                        int num_blocks_per_seq, int block_size, int start_pos, float* O, float* workspace,
                        size_t workspace_bytes, ie_stream_t stream) {
    const char* fn = "prefill_attn_kv8";
    int st = check_layout(fn, B, H_kv, d, block_size, num_blocks_per_seq);
    if (st != IE_OK) return st;
    if (P < 0 || start_pos < 0) return fail(IE_ERR_INVALID, "%s: P=%d start_pos=%d", fn, P, start_pos);
    if (H_q <= 0 || H_q % H_kv) return fail(IE_ERR_INVALID, "%s: H_q=%d not a multiple of H_kv=%d", fn, H_q, H_kv);
    if ((long long)start_pos + P > (long long)num_blocks_per_seq * block_size)
        return fail(IE_ERR_INVALID, "%s: positions up to %lld do not fit %d blocks of %d", fn, (long long)start_pos + P,
                    num_blocks_per_seq, block_size);
    if ((long long)start_pos + P > kMaxContext) return fail(IE_ERR_UNSUPPORTED, "%s: positions past 2^30", fn);
    if (B == 0 || P == 0) return IE_OK;
    if (too_many(B, P, H_q))
        return fail(IE_ERR_UNSUPPORTED, "%s: grid too large (ceil(P/16) x H_q x B > 2^21)", fn);
    if ((st = check_attn(fn, H_q, H_kv, d, (long long)B * P, Q, O)) != IE_OK) return st;
    if ((st = check_cache(fn, k_cache, v_cache, k_scales, v_scales, block_table)) != IE_OK) return st;
    ie::Kv8Attn a{};
    a.B = B; a.P = P; a.H_q = H_q; a.Q = Q; a.q_ld = H_q * d;
    a.c = cache(k_cache, v_cache, k_scales, v_scales, block_table, num_blocks_per_seq, H_kv, d, block_size);
    a.start = start_pos; a.max_ctx = start_pos + P; a.O = O;
    a.splits = workspace ? ie::kv8_prefill_splits(B, P, H_q, H_kv, d, start_pos + P) : 1;
    if (a.splits > 1) {
        const size_t need = ie_prefill_kv8_workspace_bytes(B, P, H_q, H_kv, d, start_pos);
        if (!aligned(workspace, 8)) return fail(IE_ERR_INVALID, "%s: workspace must be 8-byte aligned", fn);
        if (workspace_bytes < need)
            return fail(IE_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu for %d splits", fn, workspace_bytes, need, a.splits);
        a.ws = workspace;
    }
    st = ie::launch_prefill_attn_kv8(a, (hipStream_t)stream);
    return st != IE_OK ? st : ie::check_launch(fn);
}

}  // extern "C"
