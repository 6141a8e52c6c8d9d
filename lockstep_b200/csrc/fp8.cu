// FP8 quantizers: bf16 / fp32 -> E4M3 codes with one power-of-two scale per block of 128, the
// scales written straight to the tensor-core scale-factor layout (the MXFP4 one: tiles of 128
// rows x 4 blocks).  Codes keep the orientation of the input in every form: the products read
// an operand whose blocks run down its columns as an MN-major one, so nothing is transposed.
// All three are HBM-bound: the input once, one byte per code out.
#include <algorithm>

#include <cuda_fp8.h>

#include "fp8.cuh"

namespace ls {
namespace {

constexpr uint32_t kAbs = 0x7FFFFFFFu;

// bits of |v|, 0 for an infinity or a NaN
__device__ __forceinline__ uint32_t finite_abs(float v)
{
    const uint32_t a = __float_as_uint(v) & kAbs;
    return a < kBitsInf ? a : 0u;
}
// E4M3 has no infinity: both kinds of non-finite value are stored as its NaN
__device__ __forceinline__ float finite_or_nan(float v)
{
    return (__float_as_uint(v) & kAbs) < kBitsInf ? v : __uint_as_float(0x7FC00000u);
}

// N consecutive values from x[0 .. N), of which the first `left` exist (zeros after them).
template <int N, bool VEC, typename T>
__device__ __forceinline__ void load_values(const T *x, int left, float (&v)[N])
{
    if constexpr (VEC) {
        if (left <= 0) {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = 0.0f;
            return;
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < N / 8; h++) {
                const uint4 u = ld_stream(reinterpret_cast<const uint4 *>(x) + h);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[8 * h + 2 * i] = __uint_as_float(w[i] << 16);
                    v[8 * h + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < N / 4; h++) {
                const uint4 u = ld_stream(reinterpret_cast<const uint4 *>(x) + h);
                v[4 * h] = __uint_as_float(u.x), v[4 * h + 1] = __uint_as_float(u.y);
                v[4 * h + 2] = __uint_as_float(u.z), v[4 * h + 3] = __uint_as_float(u.w);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = 0.0f;
            if (i < left) {
                if constexpr (sizeof(T) == 2) v[i] = __bfloat162float(x[i]);
                else v[i] = x[i];
            }
        }
    }
}

// ---- blocks along the rows of a dense tensor -----------------------------------------------
// One warp takes 512 consecutive values of a row = 4 blocks = one scale word; 8 lanes share a block.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
fp8_rows_kernel(const T *__restrict__ x, int64_t rows, int K, uint8_t *__restrict__ codes, int64_t ld,
                float *__restrict__ scale, uint8_t *__restrict__ sf)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int chunks = (K + 511) / 512, blocks = (K + 127) / 128;
    const int64_t total = rows * chunks, step = int64_t(gridDim.x) * 8;
    for (int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); i < total; i += step) {
        const int64_t row = i / chunks;
        const int chunk = int(i - row * chunks), col = chunk * 512 + lane * 16;
        float v[16];
        load_values<16, VEC>(x + row * K + col, K - col, v);
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) amax = max(amax, __float_as_uint(v[j]) & kAbs);
        if (__any_sync(0xFFFFFFFFu, amax >= kBitsInf)) {
            amax = 0;
#pragma unroll
            for (int j = 0; j < 16; j++) amax = max(amax, finite_abs(v[j])), v[j] = finite_or_nan(v[j]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
        const uint32_t e8 = fp8_e8m0(amax);
        const float inv = fp8_inv_scale(e8);
        if (col < K) {
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                c[j] = cvt_e4m3x4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
            *reinterpret_cast<uint4 *>(codes + row * ld + col) = make_uint4(c[0], c[1], c[2], c[3]);
        }
        if (scale && (lane & 7) == 0 && col < K) scale[row * blocks + col / 128] = __uint_as_float(e8 << 23);
        if (sf) {
            const uint32_t b1 = __shfl_down_sync(0xFFFFFFFFu, e8, 8), b2 = __shfl_down_sync(0xFFFFFFFFu, e8, 16),
                           b3 = __shfl_down_sync(0xFFFFFFFFu, e8, 24);
            if (lane == 0)
                *reinterpret_cast<uint32_t *>(sf + sf_offset(uint32_t(row), uint32_t(chunk * 4), uint32_t(chunks))) =
                    e8 | (b1 << 8) | (b2 << 16) | (b3 << 24);
        }
    }
}

// ---- tiles of 128 x 128 ---------------------------------------------------------------------
// One CTA holds a tile in registers: lane l of warp w has columns 8 (l % 16) .. + 7 of rows
// 16 w + l / 16 + 2 i.  kRows: blocks along the rows; kCols: blocks down the columns (kRows | kCols
// from one read); kWeight: one block for the whole tile, its scale to both scale layouts.
enum { kRows = 1, kCols = 2, kWeight = 4 };

struct TileArgs {
    int rows, cols;                 // of one matrix
    const int *offsets;             // ragged row groups, or NULL
    int groups;
    int slots;                      // row tiles of one matrix (rows / 128 + groups with offsets)
    uint8_t *codes;                 // row-wise (or weight) codes, pitch ld, in the input's row order
    int64_t ld;
    float *scale;                   // kWeight: [matrix, row block, column block], or NULL
    uint8_t *sf;                    // rows = slot rows, blocks along the columns
    uint8_t *codes_t;               // column-wise codes, pitch ld; groups: rows in slot order, zeros after a group's last
    uint8_t *sf_t;                  // rows = columns of x, blocks = row slots
};

// Slot t -> its group, first row and row count (0: no such tile).  Called by a whole warp.
__device__ __forceinline__ void slot_rows(const TileArgs &p, int t, int lane, int &row0, int &n)
{
    int below = 0;                                          // groups whose first slot is at or before t
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        const bool at = g < p.groups && group_lo(p.offsets, g, p.rows) / 128 + g <= t;
        below += __popc(__ballot_sync(0xFFFFFFFFu, at));
    }
    const int g = max(below - 1, 0);
    const int lo = group_lo(p.offsets, g, p.rows), hi = group_hi(p.offsets, g, p.rows, lo);
    const int i = t - (lo / 128 + g);
    row0 = lo + 128 * max(i, 0);
    n = i < 0 ? 0 : max(0, min(128, hi - row0));
}

template <typename T, bool VEC, int MODE>
__global__ void __launch_bounds__(256)
fp8_tile_kernel(const T *__restrict__ x, const TileArgs p)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t colmax[8][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kb = (p.cols + 127) / 128, kt = (kb + 3) / 4;
    const int t = int(blockIdx.x / unsigned(kb)), cb = int(blockIdx.x - unsigned(t) * unsigned(kb));    // row slot, column block
    int row0 = 128 * t, n = min(128, p.rows - row0);
    if (!(MODE & kWeight) && p.offsets) slot_rows(p, t, lane, row0, n);
    if (n <= 0) return;                                     // uniform over the CTA
    const int64_t matrix = blockIdx.y;                      // 0 unless kWeight
    const T *xm = x + matrix * p.rows * p.cols;
    const int col = cb * 128 + 8 * (lane & 15), r0 = 16 * warp + (lane >> 4);

    float v[8][8];
    uint32_t amax_all = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + 2 * i;
        load_values<8, VEC>(xm + int64_t(row0 + r) * p.cols + col, r < n ? p.cols - col : 0, v[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) amax_all = max(amax_all, __float_as_uint(v[i][j]) & kAbs);
    }
    const bool special = __any_sync(0xFFFFFFFFu, amax_all >= kBitsInf);
    // From here on non-finite values are NaN, and `mag` counts them as 0.
    auto mag = [&](float f) { return special ? finite_abs(f) : __float_as_uint(f) & kAbs; };
    if (special) {
        amax_all = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = finite_or_nan(v[i][j]), amax_all = max(amax_all, finite_abs(v[i][j]));
    }

    if constexpr (MODE & kWeight) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) amax_all = max(amax_all, __shfl_xor_sync(0xFFFFFFFFu, amax_all, o));
        if (lane == 0) colmax[0][warp] = amax_all;
        __syncthreads();
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) m = max(m, colmax[0][w]);
        const uint32_t e8 = fp8_e8m0(m);
        const float inv = fp8_inv_scale(e8);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = r0 + 2 * i;
            if (r < n && col < p.cols)
                *reinterpret_cast<uint2 *>(p.codes + (matrix * p.rows + row0 + r) * p.ld + col) =
                    make_uint2(cvt_e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                               cvt_e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
        }
        const int nb = (p.rows + 127) / 128, nt = (nb + 3) / 4;
        if (threadIdx.x == 0 && p.scale) p.scale[(matrix * nb + t) * kb + cb] = __uint_as_float(e8 << 23);
        if (threadIdx.x < 128) {
            if (p.sf) p.sf[matrix * nb * kt * 512 + sf_offset(uint32_t(128 * t + threadIdx.x), uint32_t(cb), uint32_t(kt))] = uint8_t(e8);
            if (p.sf_t) p.sf_t[matrix * kb * nt * 512 + sf_offset(uint32_t(128 * cb + threadIdx.x), uint32_t(t), uint32_t(nt))] = uint8_t(e8);
        }
        return;
    }

    if constexpr (MODE & kRows) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = r0 + 2 * i;
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) m = max(m, mag(v[i][j]));
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const uint32_t e8 = fp8_e8m0(m);
            const float inv = fp8_inv_scale(e8);
            if (r < n) {
                if (col < p.cols)
                    *reinterpret_cast<uint2 *>(p.codes + int64_t(row0 + r) * p.ld + col) =
                        make_uint2(cvt_e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                                   cvt_e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
                if ((lane & 15) == 0) {
                    if (p.sf) p.sf[sf_offset(uint32_t(128 * t + r), uint32_t(cb), uint32_t(kt))] = uint8_t(e8);
                    if (p.scale) p.scale[int64_t(row0 + r) * kb + cb] = __uint_as_float(e8 << 23);
                }
            }
        }
    }
    if constexpr (MODE & kCols) {
        uint32_t m[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            m[j] = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) m[j] = max(m[j], mag(v[i][j]));
            m[j] = max(m[j], __shfl_xor_sync(0xFFFFFFFFu, m[j], 16));
        }
        if (lane < 16) {
#pragma unroll
            for (int j = 0; j < 8; j++) colmax[warp][8 * lane + j] = m[j];
        }
        __syncthreads();
        float inv[8];
        uint32_t e8[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t a = 0;
#pragma unroll
            for (int w = 0; w < 8; w++) a = max(a, colmax[w][8 * (lane & 15) + j]);
            e8[j] = fp8_e8m0(a);
            inv[j] = fp8_inv_scale(e8[j]);
        }
        // Groups: the tile goes to its slot's rows, all 128 of them, so that the product over a
        // group's rows runs in whole blocks (the values past the group are zeros).
        const int64_t out0 = p.offsets ? 128ll * t : row0;
        const int out_n = p.offsets ? 128 : n;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = r0 + 2 * i;
            if (r < out_n && col < p.cols)
                *reinterpret_cast<uint2 *>(p.codes_t + (out0 + r) * p.ld + col) =
                    make_uint2(cvt_e4m3x4(v[i][0] * inv[0], v[i][1] * inv[1], v[i][2] * inv[2], v[i][3] * inv[3]),
                               cvt_e4m3x4(v[i][4] * inv[4], v[i][5] * inv[5], v[i][6] * inv[6], v[i][7] * inv[7]));
        }
        if (warp == 0 && lane < 16) {
            const int st = (p.slots + 3) / 4;
#pragma unroll
            for (int j = 0; j < 8; j++) p.sf_t[sf_offset(uint32_t(col + j), uint32_t(t), uint32_t(st))] = uint8_t(e8[j]);
        }
    }
}

// codes * scale, one scale per 128 values of a row
template <typename T>
__global__ void __launch_bounds__(256)
fp8_dequantize_kernel(const uint8_t *__restrict__ codes, int64_t ld, const float *__restrict__ scale, int64_t rows, int K,
                      int row_block, T *__restrict__ out)
{
    const int blocks = (K + 127) / 128;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
        for (int c = blockIdx.x * 256 + threadIdx.x; c < K; c += gridDim.x * 256) {
            __half_raw h = __nv_cvt_fp8_to_halfraw(codes[row * ld + c], __NV_E4M3);
            const float v = __half2float(__half(h)) * scale[(row / row_block) * blocks + c / 128];
            if constexpr (sizeof(T) == 2) out[row * K + c] = __float2bfloat16_rn(v);
            else out[row * K + c] = v;
        }
}

int check_quantize(const void *x, int dtype, int64_t rows, int64_t K, int64_t ld)
{
    if (int rc = check_device()) return rc;
    if (dtype != LS_F32 && dtype != LS_BF16) return fail(LS_EINVAL, "unsupported input dtype %d", dtype);
    if (rows < 0 || K < 0 || rows > (1 << 30) || K > (1 << 30)) return fail(LS_EINVAL, "dimension out of range");
    if (ld < K || ld % 16 != 0) return fail(LS_EINVAL, "row pitch %lld of the codes: a multiple of 16, at least %lld", (long long)ld, (long long)K);
    if (rows && K && !x) return fail(LS_EINVAL, "null pointer");
    return LS_OK;
}

int check_groups(const int *offsets, int64_t groups)
{
    if (offsets && (groups < 1 || groups > kFp8MaxGroups))
        return fail(LS_EINVAL, "groups=%lld must be 1..%d", (long long)groups, kFp8MaxGroups);
    return LS_OK;
}

// 16-byte loads of whole runs of `run` values
bool vectorizes(const void *x, int dtype, int64_t K, int run)
{
    return aligned16(x) && K % run == 0 && (K * (dtype == LS_BF16 ? 2 : 4)) % 16 == 0;
}

template <int MODE>
int launch_tiles(const void *x, int dtype, const TileArgs &p, int64_t matrices, cudaStream_t st)
{
    const int64_t tiles = int64_t((p.cols + 127) / 128) * p.slots;
    if (tiles > 0x7FFFFFFFll) return fail(LS_EINVAL, "too many tiles of 128 x 128");
    const dim3 grid{unsigned(tiles), unsigned(matrices), 1};
    const bool vec = vectorizes(x, dtype, p.cols, 8);
    if (dtype == LS_BF16) {
        if (vec) fp8_tile_kernel<__nv_bfloat16, true, MODE><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16 *>(x), p);
        else fp8_tile_kernel<__nv_bfloat16, false, MODE><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16 *>(x), p);
    } else {
        if (vec) fp8_tile_kernel<float, true, MODE><<<grid, 256, 0, st>>>(static_cast<const float *>(x), p);
        else fp8_tile_kernel<float, false, MODE><<<grid, 256, 0, st>>>(static_cast<const float *>(x), p);
    }
    LS_LAUNCH_CHECK("fp8_tile_kernel");
    return LS_OK;
}

}  // namespace
}  // namespace ls

using namespace ls;

extern "C" int64_t ls_fp8_sf_bytes(int64_t rows, int64_t K) { return fp8_sf_tiles(rows, (K + 127) / 128) * 512; }
extern "C" int64_t ls_fp8_slots(int64_t rows, int64_t groups) { return groups > 0 ? fp8_slots(rows, groups) : (rows + 127) / 128; }

extern "C" int ls_quantize_fp8(const void *x, int dtype, int64_t rows, int64_t K, const int *offsets, int64_t groups,
                               uint8_t *codes, int64_t ld, float *scale, uint8_t *sf, void *stream)
{
    if (int rc = check_quantize(x, dtype, rows, K, ld)) return rc;
    if (int rc = check_groups(offsets, groups)) return rc;
    if (rows == 0 || K == 0) return LS_OK;
    if (!codes) return fail(LS_EINVAL, "null pointer");
    if (!aligned16(codes) || !aligned16(sf) || !aligned16(scale)) return fail(LS_EALIGN, "codes and scales must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (offsets) {
        TileArgs p{int(rows), int(K), offsets, int(groups), int(fp8_slots(rows, groups)), codes, ld, scale, sf, nullptr, nullptr};
        return launch_tiles<kRows>(x, dtype, p, 1, st);
    }
    const int64_t warps = rows * ((K + 511) / 512), want = (warps + 7) / 8, most = int64_t(sm_count()) * 16;
    const unsigned grid = unsigned(want < most ? want : most);
    const bool vec = vectorizes(x, dtype, K, 16);
    if (dtype == LS_BF16) {
        const __nv_bfloat16 *xb = static_cast<const __nv_bfloat16 *>(x);
        if (vec) fp8_rows_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(xb, rows, int(K), codes, ld, scale, sf);
        else fp8_rows_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(xb, rows, int(K), codes, ld, scale, sf);
    } else {
        const float *xf = static_cast<const float *>(x);
        if (vec) fp8_rows_kernel<float, true><<<grid, 256, 0, st>>>(xf, rows, int(K), codes, ld, scale, sf);
        else fp8_rows_kernel<float, false><<<grid, 256, 0, st>>>(xf, rows, int(K), codes, ld, scale, sf);
    }
    LS_LAUNCH_CHECK("fp8_rows_kernel");
    return LS_OK;
}

extern "C" int ls_quantize_fp8_both(const void *x, int dtype, int64_t rows, int64_t K, const int *offsets, int64_t groups,
                                    uint8_t *codes, uint8_t *sf, uint8_t *codes_t, uint8_t *sf_t, int64_t ld, void *stream)
{
    if (int rc = check_quantize(x, dtype, rows, K, ld)) return rc;
    if (int rc = check_groups(offsets, groups)) return rc;
    if (rows == 0 || K == 0) return LS_OK;
    if (!codes_t || !sf_t || (codes == nullptr) != (sf == nullptr)) return fail(LS_EINVAL, "null pointer");
    if (!aligned16(codes) || !aligned16(sf) || !aligned16(codes_t) || !aligned16(sf_t))
        return fail(LS_EALIGN, "codes and scales must be 16-byte aligned");
    const int64_t slots = offsets ? fp8_slots(rows, groups) : (rows + 127) / 128;
    TileArgs p{int(rows), int(K), offsets, int(groups), int(slots), codes, ld, nullptr, sf, codes_t, sf_t};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!codes) return launch_tiles<kCols>(x, dtype, p, 1, st);
    return launch_tiles<kRows | kCols>(x, dtype, p, 1, st);
}

extern "C" int ls_quantize_fp8_weight(const void *w, int dtype, int64_t matrices, int64_t N, int64_t K, uint8_t *codes,
                                      int64_t ld, float *scale, uint8_t *sf, uint8_t *sf_t, void *stream)
{
    if (int rc = check_quantize(w, dtype, N, K, ld)) return rc;
    if (matrices < 0 || matrices > kFp8MaxGroups) return fail(LS_EINVAL, "matrices=%lld must be 0..%d", (long long)matrices, kFp8MaxGroups);
    if (matrices == 0 || N == 0 || K == 0) return LS_OK;
    if (!codes) return fail(LS_EINVAL, "null pointer");
    if (!aligned16(codes) || !aligned16(sf) || !aligned16(sf_t) || !aligned16(scale))
        return fail(LS_EALIGN, "codes and scales must be 16-byte aligned");
    TileArgs p{int(N), int(K), nullptr, 0, int((N + 127) / 128), codes, ld, scale, sf, nullptr, sf_t};
    return launch_tiles<kWeight>(w, dtype, p, matrices, static_cast<cudaStream_t>(stream));
}

extern "C" int ls_dequantize_fp8(const uint8_t *codes, int64_t ld, const float *scale, int64_t rows, int64_t K,
                                 int row_block, void *out, int out_dtype, void *stream)
{
    if (int rc = check_device()) return rc;
    if (out_dtype != LS_F32 && out_dtype != LS_BF16) return fail(LS_EINVAL, "unsupported output dtype %d", out_dtype);
    if (rows < 0 || K < 0 || K > (1 << 30) || ld < K || row_block < 1) return fail(LS_EINVAL, "bad shape");
    if (rows == 0 || K == 0) return LS_OK;
    if (!codes || !scale || !out) return fail(LS_EINVAL, "null pointer");
    const dim3 grid{unsigned(std::min<int64_t>((K + 255) / 256, 64)), unsigned(std::min<int64_t>(rows, 65535)), 1};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (out_dtype == LS_BF16)
        fp8_dequantize_kernel<<<grid, 256, 0, st>>>(codes, ld, scale, rows, int(K), row_block, static_cast<__nv_bfloat16 *>(out));
    else
        fp8_dequantize_kernel<<<grid, 256, 0, st>>>(codes, ld, scale, rows, int(K), row_block, static_cast<float *>(out));
    LS_LAUNCH_CHECK("fp8_dequantize_kernel");
    return LS_OK;
}
