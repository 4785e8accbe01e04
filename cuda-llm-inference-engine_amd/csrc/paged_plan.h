// paged_plan.h — which kernel of paged_attn.hip a call takes, and in how many
// splits of its keys (host code only).
#pragma once

#include <cmath>

#include "ie_paged.h"

namespace ie {

// Which kernel, and how many splits: the least estimated time.  A form has tiles of 1 or 2 rows (paged_row_kernel),
// 16 or 32 (paged_few_kernel), 64 or 128 (paged_tile_kernel); a workgroup of it takes `start` us and `rate` us for every
// 1000 keys, measured with 8 workgroups on the card (8 KV heads over 512 and 2560 keys), `loaded` with one or two on every
// CU (32 and 64 sequences; the smallest forms, whose keys come from HBM then: prompts of 1000 tokens).
struct PagedForm {
    int rows;
    float start, rate, loaded;
    int groups = 1;  // of waves with keys of their own, of 128 rows
};
constexpr int kPagedForms = 5;
constexpr PagedForm kPagedTiles[2][2][kPagedForms] = {
    // fp32, d 64 and 128
    {{{16, 5.7f, 10.5f, 12.0f}, {32, 5.8f, 19.9f, 22.0f}, {64, 5.2f, 36.1f, 39.5f}, {128, 5.8f, 53.0f, 53.0f}, {}},
     {{16, 5.7f, 29.3f, 33.0f}, {32, 8.4f, 34.3f, 40.0f}, {64, 8.2f, 62.2f, 76.0f}, {128, 7.9f, 104.0f, 112.0f}, {}}},
    // bf16
    {{{16, 5.7f, 4.4f, 5.5f}, {32, 5.9f, 9.8f, 10.2f}, {64, 5.9f, 18.3f, 18.6f}, {128, 5.7f, 27.0f, 27.0f}, {128, 7.4f, 18.4f, 27.0f, 2}},
     {{16, 7.5f, 6.6f, 8.8f}, {32, 8.8f, 15.5f, 18.0f}, {64, 8.1f, 25.4f, 32.3f}, {128, 7.9f, 41.0f, 42.5f}, {128, 11.0f, 28.8f, 46.4f, 2}}}};
// One row, and two of an fp32 cache, have no other form (us, 8 KV heads, one sequence of 2000 keys; 32 of 4000; against 16
// rows'): fp32 d 64 one 15.8 and 26.9; 92.2 and 96.7, two 20.9 and 26.8; 94.4 and 96.7, four 30.8 and 27.0; 98.9 and
// 96.4, d 128 two 41.7 and 65.6; 185 and 186, four 63.7 and 65.6; 192 and 186; bf16 d 64 one 11.4 and 14.3; 46.1 and
// 47.7, two 15.3 and 14.3; 49.0 and 47.9, d 128 one 19.5 and 19.6; 93.3 and 94.0, two 25.7 and 19.8; 96.3 and 94.1.
constexpr PagedForm kPagedRows[2][2][2] = {{{{1, 4.7f, 5.6f, 5.6f}, {2, 5.5f, 7.8f, 7.8f}}, {{1, 4.7f, 13.8f, 13.8f}, {2, 5.5f, 18.5f, 18.5f}}},
                                 {{{1, 4.7f, 3.3f, 3.3f}, {}}, {{1, 4.7f, 7.3f, 7.3f}, {}}}};

struct PagedPlan {
    int rows, groups, splits;
};
// asked > 0: the best form for that many splits (clamped); else the best of both.
inline PagedPlan paged_plan(int B, int P, int H_q, int H_kv, int d, int kv_dtype, int max_keys, int window, int asked) {
    const int half = kv_dtype == IE_KV_BF16, wide = d == 128;
    const double rows = (double)P * (H_q / H_kv), pairs = (double)B * H_kv;
    const double walked = window && (long long)window + P < max_keys ? (double)window + P : max_keys;
    const int stages = (int)((walked + 127) / 128), most = stages < IE_PAGED_MAX_SPLITS ? stages : IE_PAGED_MAX_SPLITS;
    const bool few = rows <= (half ? 1 : 2);
    const PagedForm* forms = few ? &kPagedRows[half][wide][(int)rows - 1] : kPagedTiles[half][wide];
    PagedPlan best{forms[0].rows, 1, 1};
    double least = INFINITY;
    for (int f = 0; f < (few ? 1 : kPagedForms); ++f) {
        const PagedForm& x = forms[f];
        if (!x.rows || (f > 0 && rows <= x.rows / 2)) continue;  // (not a tile that the next smaller one holds)
        const double tiles = (double)(((long long)rows + x.rows - 1) / x.rows), groups = tiles * pairs;
        const int last = asked > 0 && asked < most ? asked : most < 1 ? 1 : most;
        for (int n = asked > 0 ? last : 1; n <= last; ++n) {
            const double a_cu = groups * n / 256;
            // 1000 keys of a workgroup where all CUs read their own from HBM (5.5 TB/s); tiles of a pair share theirs
            const double memory = 1000.0 * 2 * d * (half ? 2 : 4) / (5.5e6 / 256) / tiles * (a_cu < 1 ? a_cu : 1);
            // Workgroups of like length come in whole rounds; a causal prompt's tiles see half of its own keys on average.
            // A batch's sequences are taken to hold four fifths of the longest's keys: no call says how many they hold (alike
            // ones, 32 of 8192, take two splits for it: 192 us, in one 186).  0.6 of a round and of a start are as rough.
            const bool alike = walked >= 2.0 * P;
            const double seen = (alike ? walked - (P - 1) / 2.0 : walked > P ? walked - P / 2.0 : walked / 2) * (B > 1 ? 0.8 : 1);
            const double load = a_cu * seen / walked, own = x.rate + (x.loaded - x.rate) * (load < 1 ? load : 1);
            const double rate = (own > memory ? own : memory) / 1000 / n;
            const double rounds = a_cu <= 1 ? a_cu : alike ? std::ceil(a_cu) : a_cu + 0.6;
            const double start = x.rows >= 64 && x.groups == 1 ? 0.6 * x.start : x.start;  // (several of those share a CU)
            const double longest = x.start + walked * rate, work = rounds * (start + seen * rate);
            double t = longest > work ? longest : work;
            if (n > 1) t += 5 + rows * pairs * n * (d + 2) * 8 / 4e6;  // the join: a launch, partial results out and back
            if (t < least) {
                least = t;
                best = {x.rows, x.groups, n};
            }
        }
    }
    return best;
}

}  // namespace ie
