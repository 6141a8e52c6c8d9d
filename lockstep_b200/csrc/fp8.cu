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

// E4M3 has no infinity: non-finite values, whose codes were stored as zeros, become its NaN.
// Byte stores out of line, so that the ordinary path carries none of it.
__device__ __noinline__ void store_nans(uint8_t *dst, uint32_t flags)
{
    for (; flags; flags &= flags - 1) dst[__ffs(flags) - 1] = 0x7F;
}

// 32 bytes in one instruction: two 16-byte loads of a lane would fetch every 32-byte sector twice.
// once: the tensor is too large to stay in L2 and its lines are the first to leave (33.2 -> 32.4 us for
// 16384 x 4096 bf16 rows; a small tensor is read 0.2 us faster without, and in the tiles of both forms
// below the same hint costs 5 %).
__device__ __forceinline__ void ld_stream32(const void *p, uint32_t *w, bool once)
{
    if (once)
        asm volatile("ld.global.nc.L1::no_allocate.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
    else
        asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}

// ---- ragged groups ------------------------------------------------------------------------
// The clamped offsets (groups + 1 of them) in shared memory.  Called by the whole CTA.
__device__ __forceinline__ void load_bounds(int *bounds, const int *offsets, int groups, int rows)
{
    for (int g = threadIdx.x; g <= groups; g += blockDim.x) bounds[g] = group_lo(offsets, g, rows);
    __syncthreads();
}
// Row of x -> its slot row, -1 if it belongs to no group.  Called by a whole warp with one row.
__device__ __forceinline__ int slot_row(const int *bounds, int groups, int row)
{
    const int lane = threadIdx.x & 31;
    int before = 0;                                         // groups that start at or before the row
    for (int g0 = 0; g0 < groups; g0 += 32)
        before += __popc(__ballot_sync(0xFFFFFFFFu, g0 + lane < groups && bounds[min(g0 + lane, groups)] <= row));
    const int g = before - 1;
    if (g < 0 || row >= bounds[g + 1]) return -1;
    return (bounds[g] / 128 + g) * 128 + row - bounds[g];
}
// Slot t -> its first row and row count (0: no such tile).  Called by a whole warp.
__device__ __forceinline__ void slot_rows(const int *bounds, int groups, int t, int &row0, int &n)
{
    const int lane = threadIdx.x & 31;
    int before = 0;                                         // groups whose first slot is at or before t
    for (int g0 = 0; g0 < groups; g0 += 32) {
        const int g = g0 + lane;
        before += __popc(__ballot_sync(0xFFFFFFFFu, g < groups && (uint32_t(bounds[min(g, groups)]) >> 7) + g <= t));
    }
    const int g = max(before - 1, 0);
    const int i = t - (bounds[g] / 128 + g);
    row0 = bounds[g] + 128 * max(i, 0);
    n = i < 0 ? 0 : max(0, min(128, bounds[g + 1] - row0));
}

// ---- blocks along the rows -----------------------------------------------
// One warp takes 512 consecutive values of a row = 4 blocks = one scale word; 8 lanes share a block.
// Rows that do not start on 32-byte boundaries are read element by element, lane by lane along the
// row, and turned into 16 values per lane through shared memory (each lane's run padded by 16 bytes
// against bank conflicts).
template <typename T> constexpr int kTurn = 32 * (16 + 16 / int(sizeof(T)));

template <typename T, bool VEC>
__device__ __forceinline__ void load_chunk(const T *row, int chunk, int K, T *turn, bool once, uint32_t (&w)[8 * sizeof(T) / 2])
{
    constexpr int WORDS = 8 * sizeof(T) / 2;
    const int lane = threadIdx.x & 31;
    if constexpr (VEC) {
        const int col = chunk * 512 + lane * 16;
#pragma unroll
        for (int h = 0; h < WORDS / 8; h++) {
            if (col < K) ld_stream32(row + col + 32 / int(sizeof(T)) * h, w + 8 * h, once);
            else
                for (int i = 0; i < 8; i++) w[8 * h + i] = 0u;
        }
    } else {
        constexpr int RUN = 16 + 16 / int(sizeof(T));
        T v[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int col = chunk * 512 + 32 * j + lane;
            v[j] = col < K ? row[col] : T(0.0f);
        }
        __syncwarp();                                       // the turn buffer has been read
#pragma unroll
        for (int j = 0; j < 16; j++) turn[(2 * j + (lane >> 4)) * RUN + (lane & 15)] = v[j];
        __syncwarp();
#pragma unroll
        for (int h = 0; h < WORDS / 4; h++) {
            const uint4 q = reinterpret_cast<const uint4 *>(turn + lane * RUN)[h];
            w[4 * h] = q.x, w[4 * h + 1] = q.y, w[4 * h + 2] = q.z, w[4 * h + 3] = q.w;
        }
    }
}

template <typename T>
__device__ __forceinline__ void quantize_chunk(uint32_t (&w)[8 * sizeof(T) / 2], int64_t row, int64_t sf_row, int chunk, int K,
                                               int chunks, uint8_t *codes, int64_t ld, float *scale, uint8_t *sf)
{
    if (sf_row < 0) return;                                 // a row of no group
    using W = Word<T>;
    constexpr int WORDS = 8 * sizeof(T) / 2, PER = WORDS / 4;
    const int lane = threadIdx.x & 31, col = chunk * 512 + lane * 16;
    auto largest = [&]() {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < WORDS; i++) m = W::max_of(m, w[i]);
        return W::fold(m);
    };
    uint32_t amax = largest(), flags = 0;
    const bool special = __any_sync(0xFFFFFFFFu, amax >= kBitsInf);
    if (special) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) flags |= W::drop_special(w[i]) << (i * 16 / WORDS);
        amax = largest();
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const uint32_t e8 = fp8_e8m0(amax), s = W::inv(e8);
    if (col < K) {
        const uint32_t inv[4] = {s, s, s, s};
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; j++) c[j] = W::codes(w + PER * j, inv);
        *reinterpret_cast<uint4 *>(codes + row * ld + col) = make_uint4(c[0], c[1], c[2], c[3]);
        if (special) store_nans(codes + row * ld + col, flags);
        if (scale && (lane & 7) == 0) scale[row * ((K + 127) / 128) + col / 128] = __uint_as_float(e8 << 23);
    }
    if (sf) {
        // the four blocks' bytes as one word: lanes 0, 8, 16, 24 put theirs in place
        const uint32_t word = __reduce_or_sync(0xFFFFFFFFu, e8 << (lane & 24));
        if (lane == 0)
            *reinterpret_cast<uint32_t *>(sf + sf_offset(uint32_t(sf_row), uint32_t(chunk * 4), uint32_t(chunks))) = word;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 4)
fp8_rows_kernel(const T *__restrict__ x, int64_t rows, int K, const int *__restrict__ offsets, int groups,
                uint8_t *__restrict__ codes, int64_t ld, float *__restrict__ scale, uint8_t *__restrict__ sf, bool once)
{
    begin_dependent_launch();
    __shared__ int bounds[kFp8MaxGroups + 1];
    if (offsets) load_bounds(bounds, offsets, groups, int(rows));
    const int chunks = (K + 511) / 512;
    // chunk number of this warp, and its step, as (row, chunk of the row)
    const int64_t first = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5), step = int64_t(gridDim.x) * 8;
    int64_t row = first / chunks;
    int chunk = int(first - row * chunks);
    const int64_t row_step = step / chunks;
    const int chunk_step = int(step - row_step * chunks);
    auto advance = [&]() {
        row += row_step, chunk += chunk_step;
        if (chunk >= chunks) chunk -= chunks, row++;
    };
    __shared__ alignas(16) T turns[VEC ? 1 : 8][VEC ? 1 : kTurn<T>];
    T *turn = turns[VEC ? 0 : threadIdx.x >> 5];
    // two chunks at a time: the second one's load is in flight while the first is reduced
    while (row < rows) {
        uint32_t a[8 * sizeof(T) / 2], b[8 * sizeof(T) / 2];
        const int64_t row_a = row;
        const int chunk_a = chunk;
        load_chunk<T, VEC>(x + row * K, chunk, K, turn, once, a);
        advance();
        const int64_t row_b = row;
        const int chunk_b = chunk;
        load_chunk<T, VEC>(x + row * K, chunk, row < rows ? K : 0, turn, once, b);
        advance();
        const int64_t at_a = offsets ? slot_row(bounds, groups, int(row_a)) : row_a;
        quantize_chunk<T>(a, row_a, at_a, chunk_a, K, chunks, codes, ld, scale, sf);
        if (row_b < rows) {
            const int64_t at_b = offsets ? slot_row(bounds, groups, int(row_b)) : row_b;
            quantize_chunk<T>(b, row_b, at_b, chunk_b, K, chunks, codes, ld, scale, sf);
        }
    }
}

// ---- tiles of 128 x 128 ---------------------------------------------------------------------
// kRows: blocks along the rows; kCols: blocks down the columns (kRows | kCols from one read);
// kWeight: one block for the whole tile, its scale to both scale layouts.
//
// Persistent CTAs; a thread owns 8 columns of R rows of a tile (bf16: 8 rows, 256 threads, three CTAs per
// SM; fp32: 4 rows, 512 threads, two): lane l of warp w has columns 8 (l % 16) .. + 7 of rows
// 2 R w + l / 16 + 2 i.  bf16: each thread copies its own 16-byte pieces of the next tiles to shared
// memory ahead of time (cp.async, waited for by itself: the ring needs no barrier), so loads stay in
// flight while a tile is reduced.  16384 x 4096 in both forms: 51.4 us = 5.2 TB/s (205 us with the tile in
// registers and no ring, 52.7 with 4 rows per thread); bound by memory with one stream in and two out:
// without the conversions, the barriers or the scale bytes it takes 2 % less.  fp32 tiles are loaded straight to registers (a ring of them leaves room for one CTA per SM:
// 99 us against 55 for 8192 x 8192 weights).
// Non-finite values (rare) are set to zero for the maxima and patched into the codes afterwards.
enum { kRows = 1, kCols = 2, kWeight = 4 };

struct TileArgs {
    int rows, cols;                 // of one matrix
    const int *offsets;             // ragged row groups, or NULL
    int groups;
    int slots;                      // row tiles of one matrix (rows / 128 + groups with offsets)
    int matrices;                   // kWeight
    uint8_t *codes;                 // row-wise (or weight) codes, pitch ld, in the input's row order
    int64_t ld;
    float *scale;                   // kWeight: [matrix, row block, column block], or NULL
    uint8_t *sf;                    // rows = slot rows, blocks along the columns
    uint8_t *codes_t;               // column-wise codes, pitch ld; groups: rows in slot order, zeros after a group's last
    uint8_t *sf_t;                  // rows = columns of x, blocks = row slots
};

// A thread's R x 8 values: bf16 as 4 words per row, fp32 as 8.
template <typename T> struct Piece {
    using W = Word<T>;
    static constexpr int WORDS = sizeof(T) == 2 ? 4 : 8, CHUNKS = WORDS / 4;
    static constexpr int R = sizeof(T) == 2 ? 8 : 4, THREADS = 2048 / R;
    uint32_t u[R][WORDS];
    __device__ __forceinline__ float value(int i, int j) const
    {
        if constexpr (sizeof(T) == 2) return __uint_as_float(j & 1 ? u[i][j >> 1] & 0xFFFF0000u : u[i][j >> 1] << 16);
        else return __uint_as_float(u[i][j]);
    }
    // sets non-finite values to zero; bit 8 i + j: value (i, j) was one
    __device__ __forceinline__ uint64_t drop_special()
    {
        uint64_t flags = 0;
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int w = 0; w < WORDS; w++) flags |= uint64_t(W::drop_special(u[i][w])) << (8 * i + 8 / WORDS * w);
        return flags;
    }
    // fp32 bits of the largest magnitude of row i
    __device__ __forceinline__ uint32_t row_max(int i) const
    {
        uint32_t m = u[i][0];
#pragma unroll
        for (int w = 1; w < WORDS; w++) m = W::max_of(m, u[i][w]);
        return W::fold(m);
    }
    // largest magnitudes of the R rows in word w: one (fp32) or two (bf16) columns
    __device__ __forceinline__ uint32_t col_max(int w) const
    {
        uint32_t m = u[0][w];
#pragma unroll
        for (int i = 1; i < R; i++) m = W::max_of(m, u[i][w]);
        return m;
    }
};

constexpr int kRing = 2;                                    // tiles of the ring: 64 KB, three CTAs per SM
constexpr int kRingBytes = kRing * 128 * 128 * 2;

template <typename T, bool VEC, int MODE>
__global__ void __launch_bounds__(Piece<T>::THREADS, sizeof(T) == 2 ? 3 : 2)
fp8_tile_kernel(const T *__restrict__ x, const TileArgs p)
{
    begin_dependent_launch();
    using P = Piece<T>;
    using W = Word<T>;
    constexpr int D = kRing, CH = P::CHUNKS, R = P::R, WARPS = P::THREADS / 32;
    constexpr bool RING = VEC && sizeof(T) == 2;
    extern __shared__ uint4 ring[];                        // [D][R rows][CH][thread]
    __shared__ uint32_t colpart[WARPS][16 * P::WORDS];        // per warp: the columns' maxima (or, kWeight, one maximum)
    __shared__ alignas(16) float colinv[128];              // reciprocal scales of the columns
    __shared__ int bounds[MODE & kWeight ? 1 : kFp8MaxGroups + 1];
    if (!(MODE & kWeight) && p.offsets) load_bounds(bounds, p.offsets, p.groups, p.rows);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kb = (p.cols + 127) / 128, kt = (kb + 3) / 4;
    const int total = kb * p.slots * (MODE & kWeight ? p.matrices : 1);
    const int r0 = 2 * R * warp + (lane >> 4), c0 = 8 * (lane & 15);

    // Tiles are walked with the grid's stride; a cursor keeps a tile's row slot and column block.
    struct Cursor { int tile, rest, cb; };                  // rest: row slot (kWeight: of all matrices)
    const int rest_step = int(gridDim.x) / kb, cb_step = int(gridDim.x) - rest_step * kb;
    auto advance = [&](Cursor &c) {
        c.tile += gridDim.x, c.rest += rest_step, c.cb += cb_step;
        if (c.cb >= kb) c.cb -= kb, c.rest++;
    };
    __shared__ int2 found[P::THREADS / 32][D];              // per warp: rows of the tiles in the ring
    auto place = [&](const Cursor &c, int &t, int64_t &matrix, int &row0, int &n) {
        matrix = MODE & kWeight ? c.rest / p.slots : 0;
        t = MODE & kWeight ? c.rest - int(matrix) * p.slots : c.rest;
        if (!(MODE & kWeight) && p.offsets) slot_rows(bounds, p.groups, t, row0, n);
        else row0 = 128 * t, n = min(128, p.rows - row0);
    };
    auto fetch = [&](const Cursor &c, int stage) {          // one commit group per call, empty past the last tile
        if (RING && c.tile < total) {
            int t, row0, n;
            int64_t matrix;
            place(c, t, matrix, row0, n);
            if (!(MODE & kWeight) && p.offsets && lane == 0) found[warp][stage] = make_int2(row0, n);   // (searched for once)
            const int col = c.cb * 128 + c0;
            const T *src = x + (matrix * p.rows + row0 + r0) * p.cols + col;
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int h = 0; h < CH; h++) {
                    const bool in = r0 + 2 * i < n && col + 8 / CH * h < p.cols;
                    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[((stage * R + i) * CH + h) * P::THREADS + tid]));
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 ::"r"(dst), "l"(in ? src + int64_t(2 * i) * p.cols + 8 / CH * h : x), "r"(in ? 16 : 0) : "memory");
                }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    Cursor now{int(blockIdx.x), int(blockIdx.x) / kb, int(blockIdx.x) % kb}, ahead = now;
#pragma unroll
    for (int d = 0; d < D; d++) {
        fetch(ahead, d);
        advance(ahead);
    }
    int stage = 0;
    for (; now.tile < total; advance(now)) {
        const int cb = now.cb;
        int t, row0, n;
        int64_t matrix;
        if (RING && !(MODE & kWeight) && p.offsets) {
            __syncwarp();
            t = now.rest, matrix = 0, row0 = found[warp][stage].x, n = found[warp][stage].y;
        } else {
            place(now, t, matrix, row0, n);
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
        P v;
        const int col = cb * 128 + c0;
        if constexpr (VEC) {
            const T *src = x + (matrix * p.rows + row0) * p.cols + col;
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int h = 0; h < CH; h++) {
                    uint4 q = make_uint4(0, 0, 0, 0);
                    if (RING) q = ring[((stage * R + i) * CH + h) * P::THREADS + tid];
                    else if (r0 + 2 * i < n && col + 8 / CH * h < p.cols)
                        q = ld_stream(reinterpret_cast<const uint4 *>(src + int64_t(r0 + 2 * i) * p.cols + 8 / CH * h));
                    v.u[i][4 * h] = q.x, v.u[i][4 * h + 1] = q.y, v.u[i][4 * h + 2] = q.z, v.u[i][4 * h + 3] = q.w;
                }
        } else {
#pragma unroll
            for (int i = 0; i < R; i++)
                load_ragged<P::WORDS>(x + (matrix * p.rows + row0 + r0 + 2 * i) * p.cols + col, r0 + 2 * i < n ? p.cols - col : 0, v.u[i]);
        }
        uint32_t m[R], most = 0;
#pragma unroll
        for (int i = 0; i < R; i++) m[i] = v.row_max(i), most = max(most, m[i]);
        // every value has been used, so the loads above are done: refill their place in the ring
        if (RING) {
            fetch(ahead, stage);
            advance(ahead);
        }
        stage = stage + 1 == D ? 0 : stage + 1;
        if (n <= 0) continue;                               // a slot without rows; uniform over the CTA
        uint64_t flags = 0;
        const bool special = __any_sync(0xFFFFFFFFu, most >= kBitsInf);
        if (special) {
            flags = v.drop_special();
            most = 0;
#pragma unroll
            for (int i = 0; i < R; i++) m[i] = v.row_max(i), most = max(most, m[i]);
        }
        auto put = [&](uint8_t *dst, int i, uint32_t lo, uint32_t hi) {
            *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
            if (special) store_nans(dst, uint32_t(flags >> (8 * i)) & 0xFFu);
        };

        if constexpr (MODE & kWeight) {
            uint32_t a = __reduce_max_sync(0xFFFFFFFFu, most);
            if (lane == 0) colpart[warp][0] = a;
            __syncthreads();
            a = __reduce_max_sync(0xFFFFFFFFu, colpart[lane % WARPS][0]);
            const uint32_t e8 = fp8_e8m0(a);
#pragma unroll
            for (int i = 0; i < R; i++) {
                const uint32_t s = W::inv(e8), inv[4] = {s, s, s, s};
                if (r0 + 2 * i < n && col < p.cols)
                    put(p.codes + (matrix * p.rows + row0 + r0 + 2 * i) * p.ld + col, i, W::codes(v.u[i], inv), W::codes(v.u[i] + P::WORDS / 2, inv));
            }
            const int nb = p.slots, nt = (nb + 3) / 4;
            if (tid == 0 && p.scale) p.scale[(matrix * nb + t) * kb + cb] = __uint_as_float(e8 << 23);
            if (tid < 128) {
                if (p.sf) p.sf[matrix * nb * kt * 512 + sf_offset(uint32_t(128 * t + tid), uint32_t(cb), uint32_t(kt))] = uint8_t(e8);
                if (p.sf_t) p.sf_t[matrix * kb * nt * 512 + sf_offset(uint32_t(128 * cb + tid), uint32_t(t), uint32_t(nt))] = uint8_t(e8);
            }
            __syncthreads();                                // colpart is written again for the next tile
            continue;
        }

        constexpr int SHARE = 16 / R;                       // lanes that end up with the same row
        uint32_t row_e8 = 0;
        if constexpr (MODE & kCols) {
#pragma unroll
            for (int w = 0; w < P::WORDS; w++) {
                uint32_t a = v.col_max(w);
                a = W::max_of(a, __shfl_xor_sync(0xFFFFFFFFu, a, 16));
                if (lane < 16) colpart[warp][P::WORDS * lane + w] = a;
            }
        }
        if constexpr (MODE & kRows) {
            // Maxima of the R rows over 16 lanes: exchanges that halve what a lane keeps (its row is then the
            // upper log2 R of its four lane bits), plain steps for the other bits, and the scales
            // sent back: 16 shuffles instead of 32 for eight rows.
#pragma unroll
            for (int h = R / 2, o = 8; h > 0; h /= 2, o /= 2) {
                const bool up = lane & o;
#pragma unroll
                for (int k = 0; k < h; k++) {
                    const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, up ? m[k] : m[k + h], o);
                    m[k] = max(up ? m[k + h] : m[k], got);
                }
            }
            uint32_t z = m[0];
#pragma unroll
            for (int o = SHARE / 2; o > 0; o /= 2) z = max(z, __shfl_xor_sync(0xFFFFFFFFu, z, o));
            row_e8 = fp8_e8m0(z);
            const int mine = r0 + 2 * ((lane & 15) / SHARE);
            if (lane % SHARE == 0 && mine < n) p.sf[sf_offset(uint32_t(128 * t + mine), uint32_t(cb), uint32_t(kt))] = uint8_t(row_e8);
        }
        float inv[8];                                       // of this thread's columns
        if constexpr (MODE & kCols) {
            __syncthreads();
            if (tid < 16 * P::WORDS) {                      // one word of columns per thread
                uint32_t a = 0;
#pragma unroll
                for (int w = 0; w < WARPS; w++) a = W::max_of(a, colpart[w][tid]);
                const int st = (p.slots + 3) / 4;
#pragma unroll
                for (int h = 0; h < 8 / P::WORDS; h++) {
                    const int c = 8 / P::WORDS * tid + h;
                    const uint32_t e8 = fp8_e8m0(P::WORDS == 8 ? a & kAbs : h ? a & 0x7FFF0000u : (a << 16) & kAbs);
                    colinv[c] = fp8_inv_scale(e8);
                    p.sf_t[sf_offset(uint32_t(cb * 128 + c), uint32_t(t), uint32_t(st))] = uint8_t(e8);
                }
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float4 f = reinterpret_cast<const float4 *>(colinv)[2 * (lane & 15) + h];
                inv[4 * h] = f.x, inv[4 * h + 1] = f.y, inv[4 * h + 2] = f.z, inv[4 * h + 3] = f.w;
            }
        }
        // Both forms of a row from one unpacking to fp32.  Groups: the column-wise tile goes to its
        // slot's rows, all 128 of them, so that the product over a group's rows runs in whole blocks (the
        // values past the group are zeros).
        const int64_t out0 = p.offsets ? 128ll * t : row0;
        const int out_n = p.offsets ? 128 : n;
#pragma unroll
        for (int i = 0; i < R; i++) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = v.value(i, j);
            const int r = r0 + 2 * i;
            if constexpr (MODE & kRows) {
                const float s = fp8_inv_scale(__shfl_sync(0xFFFFFFFFu, row_e8, (lane & 16) | (i * SHARE)));
                if (r < n && col < p.cols)
                    put(p.codes + int64_t(row0 + r) * p.ld + col, i,
                        cvt_e4m3x4(f[0] * s, f[1] * s, f[2] * s, f[3] * s), cvt_e4m3x4(f[4] * s, f[5] * s, f[6] * s, f[7] * s));
            }
            if constexpr (MODE & kCols)
                if (r < out_n && col < p.cols)
                    put(p.codes_t + (out0 + r) * p.ld + col, i, cvt_e4m3x4(f[0] * inv[0], f[1] * inv[1], f[2] * inv[2], f[3] * inv[3]),
                        cvt_e4m3x4(f[4] * inv[4], f[5] * inv[5], f[6] * inv[6], f[7] * inv[7]));
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

// rows made of whole runs of `run` values, each on a boundary of its size
bool vectorizes(const void *x, int dtype, int64_t K, int run)
{
    const uintptr_t bytes = std::min<uintptr_t>(32, uintptr_t(run) * (dtype == LS_BF16 ? 2 : 4));
    return reinterpret_cast<uintptr_t>(x) % bytes == 0 && K % run == 0;
}

template <typename T, bool VEC, int MODE>
int launch_tile_kernel(const void *x, const TileArgs &p, int64_t tiles, cudaStream_t st)
{
    constexpr int ring = VEC && sizeof(T) == 2 ? kRingBytes : 0;
    static bool attr_set[64] = {};
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    {
        std::lock_guard<std::mutex> lk(state_mutex());
        if (!attr_set[dev]) {
            LS_CUDA(cudaFuncSetAttribute(fp8_tile_kernel<T, VEC, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, ring));
            attr_set[dev] = true;
        }
    }
    const int64_t most = int64_t(sm_count()) * (sizeof(T) == 2 ? 3 : 2);
    return launch_dependent(fp8_tile_kernel<T, VEC, MODE>, dim3(unsigned(std::min(tiles, most))), Piece<T>::THREADS, ring, st,
                            static_cast<const T *>(x), p);
}

template <typename T, bool VEC>
int launch_rows(const void *x, int64_t rows, int64_t K, const int *offsets, int64_t groups, uint8_t *codes, int64_t ld, float *scale,
                uint8_t *sf, unsigned grid, cudaStream_t st)
{
    return launch_dependent(fp8_rows_kernel<T, VEC>, dim3(grid), 256, 0, st, static_cast<const T *>(x), rows, int(K), offsets, int(groups),
                            codes, ld, scale, sf, rows * K * int64_t(sizeof(T)) > int64_t(64) << 20);
}

template <int MODE>
int launch_tiles(const void *x, int dtype, const TileArgs &p, cudaStream_t st)
{
    const int64_t tiles = int64_t((p.cols + 127) / 128) * p.slots * p.matrices;
    if (tiles > 0x3FFFFFFFll) return fail(LS_EINVAL, "too many tiles of 128 x 128");
    const bool vec = vectorizes(x, dtype, p.cols, dtype == LS_BF16 ? 8 : 4);
    if (dtype == LS_BF16)
        return vec ? launch_tile_kernel<__nv_bfloat16, true, MODE>(x, p, tiles, st) : launch_tile_kernel<__nv_bfloat16, false, MODE>(x, p, tiles, st);
    return vec ? launch_tile_kernel<float, true, MODE>(x, p, tiles, st) : launch_tile_kernel<float, false, MODE>(x, p, tiles, st);
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
    const int64_t warps = rows * ((K + 511) / 512), want = (warps + 7) / 8, most = int64_t(sm_count()) * 4;
    const unsigned grid = unsigned(want < most ? want : most);
    const bool vec = vectorizes(x, dtype, K, 16);
    if (dtype == LS_BF16)
        return vec ? launch_rows<__nv_bfloat16, true>(x, rows, K, offsets, groups, codes, ld, scale, sf, grid, st)
                   : launch_rows<__nv_bfloat16, false>(x, rows, K, offsets, groups, codes, ld, scale, sf, grid, st);
    return vec ? launch_rows<float, true>(x, rows, K, offsets, groups, codes, ld, scale, sf, grid, st)
               : launch_rows<float, false>(x, rows, K, offsets, groups, codes, ld, scale, sf, grid, st);
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
    TileArgs p{int(rows), int(K), offsets, int(groups), int(slots), 1, codes, ld, nullptr, sf, codes_t, sf_t};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!codes) return launch_tiles<kCols>(x, dtype, p, st);
    return launch_tiles<kRows | kCols>(x, dtype, p, st);
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
    TileArgs p{int(N), int(K), nullptr, 0, int((N + 127) / 128), int(matrices), codes, ld, scale, sf, nullptr, sf_t};
    return launch_tiles<kWeight>(w, dtype, p, static_cast<cudaStream_t>(stream));
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
