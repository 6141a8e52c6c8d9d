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
// Programmatic dependent launch: every FP8 kernel may be set up under the tail of the kernel before
// it and lets the next one do the same; it touches memory only after this.
__device__ __forceinline__ void begin_dependent_launch()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    LS_CUDA(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
    return LS_OK;
}

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
constexpr uint32_t kAbs = 0x7FFFFFFFu;

// Values are kept as the 32-bit words they were loaded in: one fp32 value, or two bf16 values.
// bf16 pairs are handled two at a time: NaN-propagating maxima of magnitudes that need no masking of
// signs, and a packed multiplication by the reciprocal scale, which is exact (a power of two; results
// below bf16's range are far below E4M3's).
template <typename T> struct Word {
    static constexpr bool PAIR = sizeof(T) == 2;
    // the larger magnitude (per half), NaN if either is one; the result's sign means nothing
    static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b)
    {
        uint32_t m;
        if constexpr (PAIR) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
        else asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
        return m;
    }
    // fp32 bits of the (larger half's) magnitude
    static __device__ __forceinline__ uint32_t fold(uint32_t m)
    {
        return PAIR ? max(m & 0x7FFF0000u, (m << 16) & kAbs) : m & kAbs;
    }
    // the reciprocal scale as a word that multiplies (both halves of) a word
    static __device__ __forceinline__ uint32_t inv(uint32_t e8m0)
    {
        return PAIR ? ((254u - e8m0) << 7) * 0x00010001u : (254u - e8m0) << 23;
    }
    // E4M3 codes of two words of pairs, or four words, times their reciprocal scales
    static __device__ __forceinline__ uint32_t codes(const uint32_t *w, const uint32_t *inv)
    {
        if constexpr (PAIR) {
            uint32_t q[2];
#pragma unroll
            for (int i = 0; i < 2; i++) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(q[i]) : "r"(w[i]), "r"(inv[i]));
            return cvt_e4m3x4(__uint_as_float(q[0] << 16), __uint_as_float(q[0] & 0xFFFF0000u),
                              __uint_as_float(q[1] << 16), __uint_as_float(q[1] & 0xFFFF0000u));
        } else {
            return cvt_e4m3x4(__uint_as_float(w[0]) * __uint_as_float(inv[0]), __uint_as_float(w[1]) * __uint_as_float(inv[1]),
                              __uint_as_float(w[2]) * __uint_as_float(inv[2]), __uint_as_float(w[3]) * __uint_as_float(inv[3]));
        }
    }
    // sets a non-finite value to zero and flags it: bit 0 the low half (or the value), bit 1 the high half
    static __device__ __forceinline__ uint32_t drop_special(uint32_t &w)
    {
        uint32_t flags = 0;
        if constexpr (PAIR) {
            if ((w & 0x7F80u) == 0x7F80u) flags |= 1u, w &= 0xFFFF0000u;
            if ((w & 0x7F800000u) == 0x7F800000u) flags |= 2u, w &= 0xFFFFu;
        } else if ((w & kAbs) >= kBitsInf) {
            flags = 1u, w = 0u;
        }
        return flags;
    }
};

// WORDS words of consecutive values from x, of which the first `left` values exist (zeros after them)
template <int WORDS, typename T>
__device__ __forceinline__ void load_ragged(const T *x, int left, uint32_t *w)
{
    if (sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(x) & 3) == 0) {     // pairs on word boundaries
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            w[i] = 0u;
            if (2 * i + 1 < left) w[i] = reinterpret_cast<const uint32_t *>(x)[i];
            else if (2 * i < left) w[i] = reinterpret_cast<const uint16_t *>(x)[2 * i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
        if constexpr (sizeof(T) == 2) {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(x);
            const uint32_t lo = 2 * i < left ? h[2 * i] : 0u, hi = 2 * i + 1 < left ? h[2 * i + 1] : 0u;
            w[i] = lo | (hi << 16);
        } else {
            w[i] = i < left ? __float_as_uint(x[i]) : 0u;
        }
    }
}

__device__ __forceinline__ int64_t fp8_sf_tiles_dev(int rows, int blocks) { return int64_t((rows + 127) / 128) * ((blocks + 3) / 4); }
#endif

// y = q(x) w^T for a few rows in one launch (fp8_skinny.cu); arguments as ls_fp8_linear, checked by it
bool fp8_skinny_fits(int64_t rows, int64_t N, int64_t K, int64_t groups);       // groups = 0: dense
int fp8_skinny_linear(const void *x, int dtype, int64_t rows, int64_t K, const uint8_t *codes, int64_t ld, const uint8_t *sf, int64_t N,
                      void *y, int out_dtype, const int *offsets, int64_t groups, int zero_tail, cudaStream_t st);

}  // namespace ls
