// Accumulator registers -> row-major output, shared by the GEMM kernels' epilogues.
#pragma once

#include "common.cuh"

namespace ls {

// 4 x 4 transpose of 16-byte items inside each group of four lanes: afterwards item k of
// lane 4g + j is what lane 4g + k held as item j.
__device__ __forceinline__ void transpose4(uint4 (&it)[4], int lane)
{
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const bool up = (lane >> b) & 1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i & (1 << b)) continue;
            const int hi = i | (1 << b);
            uint4 send = up ? it[i] : it[hi], recv;
            recv.x = __shfl_xor_sync(0xFFFFFFFFu, send.x, 1 << b);
            recv.y = __shfl_xor_sync(0xFFFFFFFFu, send.y, 1 << b);
            recv.z = __shfl_xor_sync(0xFFFFFFFFu, send.z, 1 << b);
            recv.w = __shfl_xor_sync(0xFFFFFFFFu, send.w, 1 << b);
            if (up) it[i] = recv;
            else it[hi] = recv;
        }
    }
}

// Ragged edge of the output (N not a multiple of the vector width, or the last columns of
// a tile): element-wise stores from a private copy of the chunk.  Kept out of line, and fed
// from a copy, so that neither its loop nor its run-time index touches the epilogue's
// accumulator registers (a run-time index into them would move them to local memory) or
// its code size (a tile's epilogue runs once per tile; short tiles pay for every
// instruction fetched).
static __device__ __noinline__ void store_tail_impl(void *dst, bool bf16, int n, const uint32_t *v)
{
    if (bf16)
        for (int j = 0; j < n; j++) static_cast<__nv_bfloat16 *>(dst)[j] = __float2bfloat16_rn(__uint_as_float(v[j]));
    else
        for (int j = 0; j < n; j++) static_cast<float *>(dst)[j] = __uint_as_float(v[j]);
}
__device__ __forceinline__ void store_tail(void *dst, bool bf16, int n, const uint32_t (&r)[32])
{
    uint32_t v[32];
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = r[j];
    store_tail_impl(dst, bf16, n, v);
}

// Stores one accumulator chunk: lane l of the warp holds the 32 consecutive outputs
// (columns col0 .. col0 + 31) of row row0 + l.  Called by the whole warp.  Storing each
// lane's own row would touch 32 rows per instruction (one 16-byte piece each); the
// pieces are transposed inside groups of four lanes first, so that four adjacent lanes
// write 64 contiguous bytes of one row and an instruction touches 8 rows.
__device__ __forceinline__ void store_chunk(int row_end, int N, void *cbase, bool bf16, int row0, int lane, int col0,
                                            const uint32_t (&r)[32])
{
    if (row0 >= row_end || col0 >= N) return;                       // uniform over the warp
    const int row = row0 + lane;
    const int trow = row0 + (lane & ~3), tq = lane & 3;            // first row / piece of this lane after a transpose
    if (bf16) {
        __nv_bfloat16 *base = static_cast<__nv_bfloat16 *>(cbase);
        if (col0 + 32 <= N && (N & 7) == 0) {
            uint4 it[4];
#pragma unroll
            for (int v = 0; v < 4; v++) {
                uint32_t *ow = &it[v].x;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(r[8 * v + 2 * j]),
                                                             __uint_as_float(r[8 * v + 2 * j + 1]));
                    ow[j] = *reinterpret_cast<uint32_t *>(&h);
                }
            }
            transpose4(it, lane);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (trow + k < row_end)
                    *reinterpret_cast<uint4 *>(base + int64_t(trow + k) * N + col0 + 8 * tq) = it[k];
        } else if (row < row_end) {
            store_tail(base + int64_t(row) * N + col0, true, min(32, N - col0), r);
        }
    } else {
        float *base = static_cast<float *>(cbase);
        if (col0 + 32 <= N && (N & 3) == 0) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint4 it[4];
#pragma unroll
                for (int v = 0; v < 4; v++)
                    it[v] = make_uint4(r[16 * h + 4 * v], r[16 * h + 4 * v + 1], r[16 * h + 4 * v + 2], r[16 * h + 4 * v + 3]);
                transpose4(it, lane);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (trow + k < row_end)
                        *reinterpret_cast<uint4 *>(base + int64_t(trow + k) * N + col0 + 16 * h + 4 * tq) = it[k];
            }
        } else if (row < row_end) {
            store_tail(base + int64_t(row) * N + col0, false, min(32, N - col0), r);
        }
    }
}

}  // namespace ls
