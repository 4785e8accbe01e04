// kv8.h — the 8-bit paged KV cache: launchers (arguments validated by
// kv8_capi.cpp) and what its kernels share.  Layout: include/ie_kv8.h.  The two
// attention launchers return a status: they refuse what no kernel is there for
// (parts without a workspace, an append with parts or many heads).
#pragma once

#include "ie_internal.h"
#include "ie_kv8.h"

namespace ie {

struct Kv8Cache {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    const int* table;  // [B, nbps]
    int nbps;
    int H;             // key/value heads
    int d;
    int bs_log2;       // pages of 1 << bs_log2 tokens
};

// What an append of one token a sequence changed of the rows before it, so that the
// step can be undone: for each (sequence, K or V, head), at index (b * 2 + is_v) *
// heads + h, the position whose append made the page's scale grow (-1: the last one
// did not), the scale before it and the page's words before it.  Null: not kept.
struct Kv8Undo {
    int* at;
    float* scale;
    uint32_t* codes;  // block_size * d / 4 words each
};

// Rows of B sequences into the cache (kv8_cache.hip): P each from start on, or
// with positions one each at positions[b].
struct Kv8Write {
    int B, P;
    const float* K;
    const float* V;
    int ld;
    Kv8Cache c;
    int start;
    const int* positions;
    int* ctx_lens;  // with positions: ctx_lens[b] = positions[b] + 1 (may be null)
    Kv8Undo undo;   // with positions
};
void launch_kv8_write(const Kv8Write& a, hipStream_t s);
// The rows before position pos of B sequences as they were before the append at pos,
// which has to be the last one that kept this undo.  The row itself counts as dropped.
void launch_kv8_undo(int B, int pos, const Kv8Cache& c, const Kv8Undo& u, hipStream_t s);

struct Kv8Read {
    int B, n;
    const int* starts;
    const int* lens;
    Kv8Cache c;
    float* K;
    float* V;
};
void launch_kv8_read(const Kv8Read& a, hipStream_t s);

// Attention of B x P query tokens over the cache; token t of sequence b sees
// its first min(lens[b], max_ctx) positions (decode, P = 1), or with lens null
// the first start + t + 1 (prompt).  Q row (b, t) at (b * P + t) * q_ld.
struct Kv8Attn {
    int B, P, H_q;
    const float* Q;
    int q_ld;
    Kv8Cache c;
    const int* lens;
    int max_ctx;
    int start;
    float* O;  // [B, P, H_q, d]
    float* ws;
    int splits;
    // Decode with at most 4 query heads a KV head in one split may append first:
    // K and V rows b * kv_ld to positions[b] (a sequence whose position is negative or
    // past its table's row is left out, its output zero), attention over the first
    // min(positions[b] + 1, max_ctx) (lens unused).  positions null: attention alone.
    const float* K;
    const float* V;
    int kv_ld;
    const int* positions;
    Kv8Undo undo;  // with positions
};
int launch_decode_attn_kv8(const Kv8Attn& a, hipStream_t s);  // kv8_decode.hip
// O rows [rows, d] from their splits' partials ws [rows, splits, d + 2]: sums, m, l (kv8_decode.hip).
void launch_kv8_merge(int d, int rows, int splits, const float* ws, float* O, hipStream_t s);
// Splits of the context that launch_prefill_attn_kv8 works with best (above 1 it needs the workspace).
int kv8_prefill_splits(int B, int P, int H_q, int H_kv, int d, int max_ctx);
int launch_prefill_attn_kv8(const Kv8Attn& a, hipStream_t s);  // kv8_prefill.hip

}  // namespace ie
