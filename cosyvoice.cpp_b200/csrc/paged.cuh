// paged.cuh -- pages of 8-bit codes: formats, places, rounding.
//
// A block is 16 positions x 64 values of one head, 1024 codes and one f32 scale.  Keys lie position by position: lane
// (g, t) = (lane / 4, lane % 4) of a warp finds 16 neighbouring values of a key in one 16-byte load, its part of four
// k-steps of an m16n8k16 product (the order of values in a dot product is free).  Values lie in the order of the other
// product's operand: 16 bytes are 4 tiles of 8 dims x 4 positions of one lane, so no byte has to change lanes.  Two
// 16-byte loads a lane and tensor are a whole block either way.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace cvattn {
namespace paged {

constexpr int kD = 64;
constexpr int kBlock = CVATTN_PAGE_BLOCK;       // positions
constexpr int kBlockBytes = kBlock * kD;
constexpr int kI8 = CVATTN_PAGE_I8, kE4M3 = CVATTN_PAGE_E4M3;

template <int F> constexpr float kMostCode = F == kI8 ? 127.0f : 448.0f;

// e4m3 to f32, exactly (0x7f, 0xff: NaN).
__device__ __forceinline__ float e4m3_value(uint32_t b) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)b));
    return h2f((uint16_t)r);
}
template <int F> __device__ __forceinline__ float code_value(uint32_t b) {
    if constexpr (F == kI8) return (float)((int)b - 128);
    return e4m3_value(b);
}

__device__ __forceinline__ uint32_t to_e4m3(float x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(x));
    return r & 0xffu;
}

// The code nearest to num / den (ties to even), y being that quotient to 2^-22: roundings of y from just below and just
// above agree unless the quotient is next to a border between two codes; then it is formed in 64 bits.
template <int F>
__device__ __forceinline__ uint32_t nearest_code(float y, double num, double den) {
    constexpr float lo = 1.0f - 0x1p-21f, hi = 1.0f + 0x1p-21f;
    if constexpr (F == kI8) {
        y = fminf(fmaxf(y, -127.0f), 127.0f);
        const float a = rintf(y * lo), b = rintf(y * hi);
        float c = a;
        if (a != b) c = fminf(fmaxf((float)rint(num / den), -127.0f), 127.0f);
        return (uint32_t)((int)c + 128);
    } else {
        const uint32_t a = to_e4m3(y * lo), b = to_e4m3(y * hi);
        if (a == b) return a;
        const double q = fabs(num / den), mid = 0.5 * ((double)fabsf(e4m3_value(a)) + (double)fabsf(e4m3_value(b)));
        if (q == mid) return a & 1u ? b : a;
        return q < mid ? a : b;  // (b is the larger magnitude)
    }
}

// Scale of a block from the largest finite magnitude of its values.
template <int F> __device__ __forceinline__ float scale_of(float amax) {
    const float s = __fdiv_rn(amax, kMostCode<F>);
    return s < 0x1p-126f ? 0.0f : s;
}

// Entry of a table: the page, or -1 where it is out of range.
__device__ __forceinline__ int page_of(const int32_t* row, int entry, int n_pages) {
    const int p = row[entry];
    return (uint32_t)p < (uint32_t)n_pages ? p : -1;
}

}  // namespace paged
}  // namespace cvattn
