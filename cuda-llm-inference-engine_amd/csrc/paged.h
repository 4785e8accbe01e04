// paged.h — launchers behind include/ie_paged.h (arguments validated by
// paged_capi.cpp).
#pragma once

#include "ie_internal.h"
#include "ie_paged.h"

namespace ie {

// Positions to pages: any block size by one multiplication.  For n < 2^31, n /
// block = (n * mul) >> (32 + shift) with mul = ceil(2^(32 + shift) / block),
// shift = ceil(log2 block) - 1 (0 for a block of 1): mul < 2^32, and its excess e <
// block gives an error of n e / 2^(32 + shift) / block < 1 / block.  A block of 1
// would need mul = 2^32: it has mul = 0, which stands for n itself.
struct PageMap {
    const int* table;  // [B, nbps]
    int nbps, block;
    uint32_t mul;
    int shift;
};
inline PageMap page_map(const int* table, int nbps, int block) {
    PageMap p{table, nbps, block, 0, 0};
    if (block > 1) {
        p.shift = 31 - __builtin_clz((unsigned)(block - 1));
        p.mul = (uint32_t)(((1ull << (32 + p.shift)) + block - 1) / block);
    }
    return p;
}

struct RopeWrite {
    int B, P, H_q, H_kv, d, rot, interleaved;
    const float *Q, *K, *V;
    int q_ld, kv_ld;  // floats from row to row
    const float* freq;
    const int *starts, *lens, *positions;
    float* out;
    void *k, *v;
    int kv_dtype;
    PageMap pages;
};
void launch_rope_write(const RopeWrite& a, hipStream_t s);

struct KeepRows {
    int B, most, layers;
    void* const* k;
    void* const* v;
    PageMap pages;
    int row_bytes;
    const int *ctx, *paths, *counts;
};
void launch_kv_keep(const KeepRows& a, hipStream_t s);

// Attention of B x P query tokens: ranges of keys, or with parents a tree
// (starts are then the contexts' lengths, P the nodes).
struct PagedAttn {
    int B, P, H_q, H_kv, d;
    const float* Q;
    const void *k, *v;
    int kv_dtype;
    PageMap pages;
    const int *starts, *lens;
    int max_ctx;  // of starts + lens, or of the context before a tree
    const int *first, *end;
    const int* parents;
    int window;
    float scale, cap;
    const float* slopes;
    float* O;
    float* ws;
    int splits;
};
void launch_paged_attn(const PagedAttn& a, hipStream_t s);
// The split count that a launch works with: `asked`, or a choice where it is <= 0.
int paged_attn_splits(int B, int P, int H_q, int H_kv, int d, int kv_dtype, int max_keys, int window, int asked);

}  // namespace ie
