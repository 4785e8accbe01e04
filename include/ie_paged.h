/*
 * ie_paged.h — C ABI of what rotary models and drafted tokens need around the
 * paged KV cache: rows rotated by their positions on the way into it,
 * attention over it whose scores are capped, fall off with distance or are
 * kept to ranges of keys, attention of a tree of drafted tokens, and the rows
 * of an accepted path moved together.  Plain C; conventions as ie_amd.h
 * (device pointers, sizes and a stream, an ie_status back, ie_last_error() for
 * the message, arguments checked on the host before any HIP call, nothing
 * allocated, asynchronous on the given stream).  The reference has plain
 * causal attention and learned positions only (src/gpt2_engine.cu:321-346,
 * 484-493); these have no counterpart there.
 *
 * The caches are ie_amd.h's: K and V [num_blocks][block_size][H_kv][d] in
 * kv_dtype (IE_KV_F32, IE_KV_BF16), 16-byte aligned, any block_size; position
 * p of sequence b is row p % block_size of page
 * block_table[b][p / block_size], block_table [B, num_blocks_per_seq].  d in
 * {64, 128}.  A table entry is read only where the call writes or a query of
 * it may see a key, and what lies behind a sequence's last position is never
 * used.  No output overlaps an input or another output.
 *
 * A workspace serves one call at a time: calls that may run at once (on two
 * streams, from two replayed graphs) take one each.
 */
#ifndef IE_PAGED_H
#define IE_PAGED_H

#include "ie_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rotates Q and K and writes K and V: row (b, t), t < lens[b], of Q_src [.., H_q,
 * d] lies at (b * P + t) * q_stride floats, of K_src and V_src [.., H_kv, d] at (b * P
 * + t) * kv_stride (the rows of a QKV projection serve as they lie; multiples of 4,
 * at least a row), and goes to cache position starts[b] + t.  Its angles
 * are a_i = pos * inv_freq[i], i < rot_dim / 2, pos = positions[b * P + t]
 * (positions NULL: starts[b] + t), less their full turns to 2^-50 of one (up to
 * 2^50 of them); channels (x, y) = (i, i + rot_dim / 2), or (2 i, 2 i + 1) where
 * interleaved is not 0, become (x cos - y sin, y cos + x sin).  Channels from
 * rot_dim on (even, 0 .. d) pass as they are, as does V.  K and V are rounded to
 * the cache's type once; Q_out [B, P, H_q, d] is fp32 (H_q may be 0: no Q).  lens
 * NULL: P rows each (values past P count as P).  Rows from lens[b] on are
 * left out: neither the cache nor Q_out has them; a row whose cache position is
 * negative or past its table's row has Q_out alone.  inv_freq [rot_dim / 2],
 * starts and lens [B] and positions [B, P] are device arrays.  No two rows of a
 * call go to the same row of the cache (sequences that share a page write past it). */
int ie_rope_kv_write(int B, int P, const float* Q_src, const float* K_src, const float* V_src, int q_stride,
                     int kv_stride, int H_q, int H_kv, int d, int rot_dim, int interleaved, const float* inv_freq, const int* starts,
                     const int* lens, const int* positions, float* Q_out, void* k_cache, void* v_cache, int kv_dtype,
                     const int* block_table, int num_blocks_per_seq, int block_size, ie_stream_t stream);

/* Most splits of a tile's keys that the two attentions take. */
#define IE_PAGED_MAX_SPLITS 64
/* Split count of an attention call over max_keys keys at most (ie_paged_attn:
 * max_context_len, ie_tree_attn: max_context_len + T; with a window, no more
 * than window + P are walked).  num_splits > 0 is clamped to [1,
 * IE_PAGED_MAX_SPLITS] and to the keys' blocks; num_splits <= 0 chooses. */
int ie_paged_attn_num_splits(int B, int P, int H_q, int H_kv, int d, int kv_dtype, int max_keys, int window,
                             int num_splits);
/* Bytes of workspace for that many splits: 0 for 1. */
size_t ie_paged_attn_workspace_bytes(int B, int P, int H_q, int d, int num_splits);

/* Attention of lens[b] <= P query tokens of each sequence over its cache: prompts,
 * chunks and single tokens.  Token t of sequence b is at position pos = starts[b]
 * + t; its sequence holds n = min(starts[b] + lens[b], max_context_len) positions
 * (negative starts count as 0; lens NULL: P, values past P count as P).  It sees
 * the keys j of
 *   max(0, first[b, t], pos - window + 1) <= j < min(n, end[b, t]),
 * where first (NULL: 0) and end (NULL: pos + 1, causal) are int32 [B, P] and
 * window 0 is none: first at a document's beginning keeps documents packed into
 * a row apart, end = max(prefix, pos + 1) lets a prefix see itself whole.  With
 * h the query head, G = H_q / H_kv, the score of key j is
 *   s = scale * (q . K[j, h / G])          (scale 0: 1 / sqrt(d))
 *   s = cap * tanh(s / cap)                (cap 0, or from 2^80 on: none)
 *   s = s - slopes[h] * |pos - j|          (slopes [H_q] fp32, NULL: none)
 * and O [B, P, H_q, d] = sum_j softmax(s)_j V[j, h / G].  A query that sees no
 * key, or none above minus infinity, gives zeros; rows from lens[b] on are left as they were.  Q, O fp32,
 * token-major; starts [B] and lens [B] are device int32.  Values at keys that a
 * query does not see never reach it, infinite and NaN ones included; one
 * that it sees makes what fp32 arithmetic makes of it.  Refused are a scale that
 * passes fp32 times log2(e) and a scale / cap outside its normal range.
 * A NULL workspace stands for num_splits = 1; otherwise workspace_bytes must
 * cover ie_paged_attn_workspace_bytes of ie_paged_attn_num_splits' count.  A
 * repeated call repeats its bits; those of a token may depend on the chunk and
 * batch it came in. */
int ie_paged_attn(int B, int P, int H_q, int H_kv, int d, const float* Q, const void* k_cache, const void* v_cache,
                  int kv_dtype, const int* block_table, int num_blocks_per_seq, int block_size, const int* starts,
                  const int* lens, int max_context_len, const int* first, const int* end, int window, float scale,
                  float cap, const float* slopes, float* O, float* workspace, size_t workspace_bytes, int num_splits,
                  ie_stream_t stream);

/* Most drafted tokens of a sequence. */
#define IE_TREE_MAX 256
/* Attention of a tree of drafted tokens: node t < lens[b] (NULL: T) of sequence b
 * has its rows at cache position context_lens[b] + t and follows node
 * parents[b, t] < t (int32 [B, T]; one that is no earlier node counts as -1, the
 * context's last token).  It sees the first context_lens[b] positions, its
 * ancestors and itself, inside the window; its position, and that of a drafted
 * key, is context_lens[b] + the number of its ancestors.  Scores, outputs, rows
 * left out and workspace as ie_paged_attn's (P = T).  context_lens (taken as 0 ..
 * max_context_len) and lens are device int32 [B];
 * max_context_len + T <= num_blocks_per_seq * block_size; T <= IE_TREE_MAX. */
int ie_tree_attn(int B, int T, int H_q, int H_kv, int d, const float* Q, const void* k_cache, const void* v_cache,
                 int kv_dtype, const int* block_table, int num_blocks_per_seq, int block_size, const int* context_lens,
                 const int* lens, const int* parents, int max_context_len, int window, float scale, float cap,
                 const float* slopes, float* O, float* workspace, size_t workspace_bytes, int num_splits,
                 ie_stream_t stream);

/* The rows of an accepted path together: in every one of n_layers caches (host
 * arrays of device pointers), row context_lens[b] + paths[b, j] of sequence b
 * moves to context_lens[b] + j, j = 0 .. counts[b] - 1 (paths int32 [B, max_count],
 * counts and context_lens int32 [B], device; counts past max_count count as it).
 * A path ascends; it ends before an entry that is not above the one before it
 * (the first: not below 0) or whose row is past the table's.  No cache stands
 * twice among them.  Rows behind the moved ones keep their bytes and count as dropped.  No page that a path moves
 * rows into may be shared. */
int ie_kv_cache_keep(int B, int max_count, int n_layers, void* const* k_caches, void* const* v_caches, int kv_dtype,
                     const int* block_table, int num_blocks_per_seq, int block_size, int n_heads, int d_head,
                     const int* context_lens, const int* paths, const int* counts, ie_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
