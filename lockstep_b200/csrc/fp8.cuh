// What the FP8 quantizers and the FP8 products share: the block scale, and the row slots of
// ragged groups.
//
// A block is 128 values along the axis a product sums over (128 x 128 for weights).  Its scale
// is the smallest power of two s with amax <= 448 s, at least 2^-126 (so that it and its
// reciprocal are normal numbers), 1 for a block of zeros; amax runs over the finite values.
// Division by s is exact, so the only rounding is the one to E4M3 (nearest, ties to even).
#pragma once

#include "common.cuh"

namespace ls {

constexpr int kFp8MaxGroups = 1024;     // offsets and tile prefixes of all groups fit in shared memory

// Row slots of ragged groups.  Group g holds rows [lo, hi) = [offsets[g], offsets[g + 1]); its
// rows are cut into tiles of 128 from its first row on, and tile i of group g has slot
//   lo / 128 + g + i.
// Slots of different groups never collide (lo / 128 + g + ceil((hi - lo) / 128) <= hi / 128 + g + 1),
// a slot needs no prefix sum over the groups, and there are rows / 128 + groups of them.
// Offsets outside [0, rows] or out of order are clamped, so that every access stays in bounds.
inline int64_t fp8_slots(int64_t rows, int64_t groups) { return rows / 128 + groups; }

// The next GEMM's tensor maps are functions of these.
inline int64_t fp8_sf_tiles(int64_t rows, int64_t blocks) { return ((rows + 127) / 128) * ((blocks + 3) / 4); }

#ifdef __CUDACC__
__device__ __forceinline__ int group_lo(const int *offsets, int g, int rows) { return min(max(offsets[g], 0), rows); }
__device__ __forceinline__ int group_hi(const int *offsets, int g, int rows, int lo)
{
    return min(max(offsets[g + 1], lo), rows);
}

// E8M0 byte of the block scale from the bits of amax (finite, sign cleared).  448 = 1.75 * 2^8:
// mantissas up to .11 keep the exponent - 8, larger ones take the next.
__device__ __forceinline__ uint32_t fp8_e8m0(uint32_t amax_bits)
{
    if (amax_bits == 0u) return 127u;
    return uint32_t(max(int((amax_bits + 0x1FFFFFu) >> 23) - 8, 1));
}
__device__ __forceinline__ float fp8_inv_scale(uint32_t e8m0) { return __uint_as_float((254u - e8m0) << 23); }

// Four floats -> four E4M3 codes, the first in the low byte.  |q| <= 448 or NaN.
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d)
{
    uint32_t out;
    asm("{\n.reg .b16 lo, hi;\n"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
        "mov.b32 %0, {lo, hi};\n}\n" : "=r"(out) : "f"(a), "f"(b), "f"(c), "f"(d));
    return out;
}
#endif

}  // namespace ls
