// kv8_rule.h — how values become codes of the 8-bit KV cache and how a page's
// scale follows its rows (include/ie_kv8.h), for the kernels that write it.
#pragma once

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

// Word i of a page's codes: 4 channels of a row of K, 4 tokens of a channel of V; its (first) row.
__device__ __forceinline__ int first_row(int i, bool is_v, int d) {
    return is_v ? i / (4 * d) * 16 + i % 4 * 4 : i / (d / 4);
}

// The scale of a page after a call that writes rows from r0 on, whose largest
// magnitude has the bits mx; had: the scale before (read only where r0 > 0).
struct PageScale {
    float scale, inv;
    bool grew;   // rows before r0 become code * move
    float move;
    __device__ __forceinline__ PageScale(uint32_t mx, int r0, float had) {
        const float need = max_nan(bitsf(mx) / 127.0f, kFloor);
        scale = r0 == 0 ? need : need <= had ? had : max_nan(need, 1.25f * had);
        inv = 1.0f / scale;
        grew = r0 > 0 && !(scale == had);
        move = had * inv;
    }
};

}  // namespace
}  // namespace ie
