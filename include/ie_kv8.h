/*
 * ie_kv8.h — C ABI of the paged KV cache held in 8 bits: its writes, its read
 * and the attention over it.  Plain C; conventions as ie_amd.h (device
 * pointers, sizes and a stream, an ie_status back, ie_last_error() for the
 * message, arguments checked on the host before any HIP call, nothing
 * allocated, asynchronous on the given stream).  The reference keeps its cache
 * in fp32 (src/gpt2_engine.cu:321-346); this cache has no counterpart there.
 *
 * Layout, for num_blocks pages of block_size tokens (16, 32, 64, 128 or 256),
 * n_heads key/value heads of d_head channels (64 or 128):
 *   k_cache  int8  [num_blocks][n_heads][block_size][d_head]
 *   v_cache  int8  [num_blocks][n_heads][block_size / 16][d_head][16]
 *            (the 16 tokens of a group side by side for each channel)
 *   k_scales, v_scales  fp32 [num_blocks][n_heads]
 * A value is code * scale, codes in [-127, 127].  Nothing needs initialising:
 * a page's scale and codes are written before they are read.  Token `pos` of
 * sequence b is row pos % block_size of page
 * block_table[b][pos / block_size]; a table entry is read only where the
 * sequence has tokens there.  Pages that several sequences share (a common
 * prefix) may be read at will and written by none.
 *
 * Scales follow the rows of their page, in fp32:
 *   need = max|x| / 127 over the page's rows written by one call (>= 2^-100);
 *   a call that writes the page's row 0 starts the page anew: scale = need;
 *   a later call keeps the scale if it is at least need; otherwise it becomes
 *   max(need, 1.25 * scale), and the rows before the written ones keep their
 *   place with codes rint(code * (scale_old * (1 / scale_new))).
 * New codes are rint(x * (1 / scale)).  A value written with its page is off
 * by at most half a scale; one whose page grew under it by at most 2.5 scales
 * (0.5 / (1 - 1/1.25)), however often it grew.  Rows behind the written ones
 * keep their bytes and count as dropped.  A non-finite value makes its page's
 * scale non-finite until the page starts anew, and attention of a query that
 * sees a token of the page returns NaN.
 *
 * A workspace serves one call at a time: calls that may run at once (on two
 * streams, from two replayed graphs) take one each.  No output overlaps an input.
 */
#ifndef IE_KV8_H
#define IE_KV8_H

#include "ie_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache type of GPT2EngineOptions::kv_dtype and ie_engine_create for this
 * cache (the entry points of ie_amd.h take IE_KV_F32 and IE_KV_BF16 only). */
#define IE_KV_I8 2

/* Writes P rows of each of B sequences at positions start_pos ..
 * start_pos + P - 1.  K_src / V_src hold row (b, t) at (b * P + t) *
 * src_stride, n_heads * d_head floats each (src_stride >= n_heads * d_head, a
 * multiple of 4: the rows of a QKV projection serve as they lie).  block_table
 * [B, num_blocks_per_seq]; start_pos + P <= num_blocks_per_seq * block_size.
 * No page may be written for two sequences in one call. */
int ie_kv8_cache_write(int B, int P, const float* K_src, const float* V_src, int src_stride,
                       void* k_cache, void* v_cache, float* k_scales, float* v_scales,
                       const int* block_table, int num_blocks_per_seq, int start_pos,
                       int n_heads, int d_head, int block_size, ie_stream_t stream);

/* Batched decode append: row b of K_src / V_src (at b * src_stride) goes to
 * position positions[b] (device int32) of sequence b.  A sequence whose
 * position is negative or past its table's row is left out. */
int ie_kv8_cache_append_batch(int B, const float* K_src, const float* V_src, int src_stride,
                              void* k_cache, void* v_cache, float* k_scales, float* v_scales,
                              const int* block_table, int num_blocks_per_seq, const int* positions,
                              int n_heads, int d_head, int block_size, ie_stream_t stream);

/* The cached values back as fp32: row t of sequence b, t < n, is position
 * starts[b] + t (starts: device int32 [B]); K_dst / V_dst [B, n, n_heads,
 * d_head].  Positions at or past context_lens[b] (device int32 [B]; NULL: no
 * such limit), negative ones and ones past the table's row give zeros. */
int ie_kv8_cache_read(int B, int n, const int* starts, const int* context_lens,
                      const void* k_cache, const void* v_cache, const float* k_scales,
                      const float* v_scales, const int* block_table, int num_blocks_per_seq,
                      int n_heads, int d_head, int block_size, float* K_dst, float* V_dst,
                      ie_stream_t stream);

/* Most splits of a sequence's context that ie_decode_attn_kv8 takes. */
#define IE_KV8_MAX_SPLITS 64
/* Split count of a call: num_splits > 0 is clamped to [1, IE_KV8_MAX_SPLITS]
 * and to the context's 64-token tiles; num_splits <= 0 chooses. */
int ie_decode_kv8_num_splits(int B, int H_q, int H_kv, int d, int max_context_len, int num_splits);

/* Decode attention for one query token per sequence, as ie_decode_attn:
 * Q, O [B, H_q, d] fp32, d in {64, 128}, H_q any multiple of H_kv; attends to
 * the first context_lens[b] (device int32, taken as at most max_context_len)
 * positions; an empty context gives zeros.  workspace_bytes must cover
 * ie_decode_attn_workspace_bytes(B, H_q, d, splits) of
 * ie_decode_kv8_num_splits' count where that is above 1 (else the workspace
 * may be NULL).  A repeated call repeats its bits.  O must not overlap Q. */
int ie_decode_attn_kv8(int B, int H_q, int H_kv, int d, const float* Q, const void* k_cache,
                       const void* v_cache, const float* k_scales, const float* v_scales,
                       const int* block_table, const int* context_lens, int max_context_len,
                       int block_size, int num_blocks_per_seq, float* O, float* workspace,
                       size_t workspace_bytes, int num_splits, ie_stream_t stream);

/* Bytes of workspace with which ie_prefill_attn_kv8 can split the context of a
 * call of this size (rows that do not fill the GPU, behind a long one); 0 where
 * it would not. */
size_t ie_prefill_kv8_workspace_bytes(int B, int P, int H_q, int H_kv, int d, int start_pos);

/* Causal attention of a prompt chunk over the cache, as ie_prefill_attn: Q, O
 * [B, P, H_q, d] fp32, token t of each sequence at position start_pos + t, its
 * rows cached already; it attends to positions 0 .. start_pos + t.  H_q any
 * multiple of H_kv, d in {64, 128}.  O must not overlap Q.  With a workspace
 * NULL the context is not split; otherwise workspace_bytes must cover
 * ie_prefill_kv8_workspace_bytes of the call.  A repeated call repeats its
 * bits; those of a token may depend on the chunk and batch it came in. */
int ie_prefill_attn_kv8(int B, int P, int H_q, int H_kv, int d, const float* Q, const void* k_cache,
                        const void* v_cache, const float* k_scales, const float* v_scales,
                        const int* block_table, int num_blocks_per_seq, int block_size,
                        int start_pos, float* O, float* workspace, size_t workspace_bytes,
                        ie_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
