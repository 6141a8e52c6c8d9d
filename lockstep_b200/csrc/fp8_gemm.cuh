// FP8 products with one scale per block of 128, dense and grouped by ragged row groups, on the
// 5th-generation tensor cores (kind::mxf8f6f4, E4M3 operands, fp32 accumulators in tensor memory).
//
// The block scales are powers of two (UE8M0 bytes), so the tensor core applies them itself: an
// MMA covers 32 values of K and takes one scale byte per row, the four MMAs of a block of 128
// name the same byte.  One 512-byte scale tile (128 rows x 4 blocks) lasts 512 values of K, so
// the scale copies cost a quarter of what they cost the MXFP4 product.
//
// Three forms of one kernel (A is the operand of the output's rows, B of its columns):
//   NT  C = A[M, K] B[N, K]^T      forward                      A, B K-major
//   NN  C = A[M, K] B[K, N]        gradient of the input        B MN-major
//   TN  C = A[K, M]^T B[K, N]      gradient of the weight       A, B MN-major
// so every operand is read as the quantizers wrote it; nothing is transposed in memory.
// Grouped: NT and NN cut A's rows by `offsets` and take B[g]; TN cuts K (rows in slot order, see
// fp8.cuh) and writes C[g].
//
// Roles of a CTA: warp 0 TMA producer, warp 1 MMA issuer, warps 2-9 epilogue.  CTAS = 2: a pair
// of CTAs works on 256 x 256 tiles with cta_group::2 MMAs, each staging its own 128 rows of A and
// its own half of B.  The tiles are handed out statically to a persistent grid.
#pragma once

#include <cuda.h>
#include <algorithm>
#include <atomic>

#include "epilogue.cuh"
#include "fp8.cuh"
#include "ptx.cuh"

namespace ls {

enum Form { NT = 0, NN = 1, TN = 2 };
constexpr int kMaxSplits = 4;           // CTAs of a cluster that share the K loop of a tile

struct Fp8Params {
    void *c;
    int M, N, K;                   // of the whole product: M counts the rows of all groups (NT, NN), K those of TN
    int out_bf16;
    const int *offsets;            // NULL: one group
    int groups;
    int zero_tail;                 // NT, NN: rows that belong to no group are set to zero
    int sfa_kt, sfb_kt;            // scale tiles along K per 128 rows of A / columns of B
    int sfb_rt;                    // NT, NN: 128-column scale tiles of one group's B
    int a_bytes;                   // what one load of an A tile delivers
    int splits;                    // dense, single CTAs: CTAs per tile, each with its part of K (1: no split)
    int *err;
};
struct Fp8Maps { CUtensorMap a, b, sfa, sfb, c; };

namespace {

constexpr int kThreads = 320;
constexpr int kTmemCols = 512;
constexpr int kBlock = 128;             // values of K per stage = per scale block
constexpr int kSegment = 32;            // blocks per accumulation chain of the LONG kernels

constexpr int kStagingWords = 512;      // one epilogue warp's staging area: 16 rows of 128 bytes

template <int CTAS, int BN>
struct Fp8Cfg {
    static_assert(CTAS == 1 || BN == 256, "pairs work on 256-column tiles");
    static constexpr int BCOLS = BN / CTAS;                // columns of B staged by one CTA
    static constexpr int A_BYTES = 128 * kBlock;
    static constexpr int B_BYTES = BCOLS * kBlock;
    static constexpr int SFB_TILES = BN >= 128 ? BN / 128 : 1;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2048;       // 512 B of A's scales, 512 SFB_TILES of B's
    static constexpr int STAGES = BN == 64 ? 7 : CTAS == 2 || BN == 128 ? 6 : 4;
    static constexpr int OVL = BN == 256 ? 32 : 0;         // columns that the two accumulators share
    static constexpr int ACC1 = BN - OVL;
    static constexpr int SFA_COL = 2 * BN - OVL, SFB_COL = SFA_COL + 4;
    static_assert(SFB_COL + 4 * SFB_TILES <= kTmemCols, "tensor memory overflow");
    static constexpr int STAGING = STAGES * STAGE_BYTES;   // of the epilogue warps; then barriers, the groups' tile prefix
    static constexpr int TAIL = STAGING + 8 * kStagingWords * 4;
    // K split over a cluster of up to kMaxSplits CTAs: the others' sums of a tile lie over the stages of the first
    static constexpr int PART_BYTES = 128 * BN * 4;
    static constexpr int LIST = TAIL + 256;
    static constexpr int SMEM = LIST + 4 * (kFp8MaxGroups + 4) + 1024;
    static_assert(STAGING % 1024 == 0, "swizzled tiles start on 1024-byte boundaries");
    static_assert(SMEM <= 227 * 1024, "shared memory overflow");
};

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_ctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// 16 lanes write the 32 columns of one row: lane j holds elements 2 j and 2 j + 1 in `word`, dst is
// element 2 j.  odd: the row starts on an odd element, so the aligned pairs are elements 2 j + 1 and
// 2 j + 2, and the first and the last element go alone.
__device__ __forceinline__ void store_pair(uint16_t *dst, uint32_t word, bool odd, int j, int left, bool in)
{
    const uint32_t next = odd ? __shfl_down_sync(0xFFFFFFFFu, word, 1, 16) : 0u;
    const uint32_t pair = odd ? __funnelshift_r(word, next, 16) : word;
    const int first = 2 * j + odd;
    if (!in) return;
    if (first + 1 < left) *reinterpret_cast<uint32_t *>(dst + odd) = pair;
    else if (first < left) dst[odd] = uint16_t(pair);
    if (odd && j == 0) dst[0] = uint16_t(word);
}

// Stores a chunk as store_chunk does, for rows that do not start on 16-byte boundaries and for the
// ragged last columns, through shared memory: element stores straight from the accumulator layout
// touch 32 rows per instruction.  bf16: 16 lanes write the 32 columns of a row as aligned pairs.
// fp32: 16 columns at a time, 16 lanes a row.
__device__ __forceinline__ void store_ragged(uint32_t *stage, int row_end, int N, void *cbase, bool bf16, int row0, int lane, int col0,
                                             const uint32_t (&r)[32])
{
    if (row0 >= row_end || col0 >= N) return;                      // uniform over the warp
    const int j = lane & 15, up = lane & 16;                       // rows i (lanes 0-15) and i + 16: different banks
    const int left = min(N - col0, 32), rows = row_end - row0 - up;
    const int64_t at = int64_t(row0 + up) * N + col0;
    if (lane == 0) ptx::bulk_wait_read();                          // a store_rows before has read the area
    // Row k is 16 words at 16 k, its four 16-byte pieces permuted by (k / 2) % 4: eight lanes then write
    // different banks, and reading row up + i the permutation is a constant of the unrolled loop.
    uint4 *put = reinterpret_cast<uint4 *>(stage) + 4 * lane;
    const int turn = (lane >> 1) & 3;
    const uint32_t *from[4];
#pragma unroll
    for (int c = 0; c < 4; c++) from[c] = stage + 16 * up + (((j >> 2) ^ c) << 2) + (j & 3);
    auto row = [&](int i) { return from[(i >> 1) & 3][16 * i]; };
    if (bf16) {
        __syncwarp();                                              // the staging area has been read
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(r[8 * c + 2 * i]), __uint_as_float(r[8 * c + 2 * i + 1]));
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
            put[c ^ turn] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        uint16_t *dst = static_cast<uint16_t *>(cbase) + at + 2 * j;
        if (!(N & 1)) {                                            // every row starts on a pair
            const bool in = 2 * j < left;
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (in && i < rows) *reinterpret_cast<uint32_t *>(dst + i * int64_t(N)) = row(i);
            return;
        }
        // every other row starts on a pair (the same ones in both halves of the warp)
        if (row0 & 1) {
#pragma unroll
            for (int i = 0; i < 16; i++) store_pair(dst + i * int64_t(N), row(i), (i & 1) == 0, j, left, i < rows);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) store_pair(dst + i * int64_t(N), row(i), (i & 1) != 0, j, left, i < rows);
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (16 * h >= left) return;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; c++)
            put[c ^ turn] = make_uint4(r[16 * h + 4 * c], r[16 * h + 4 * c + 1], r[16 * h + 4 * c + 2], r[16 * h + 4 * c + 3]);
        __syncwarp();
        uint32_t *dst = static_cast<uint32_t *>(cbase) + at + 16 * h + j;
        const bool in = 16 * h + j < left;
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (in && i < rows) dst[i * int64_t(N)] = row(i);
    }
}

// Stores 32 rows of 128 bytes (64 bf16 or 32 fp32 columns; lane l holds row l as 32 words) by TMA through
// the warp's staging area, 16 rows at a time: whole lines, and no address arithmetic or shuffles
// per piece.  Columns past the tensor are clipped; the caller sees to it that all rows may be stored.
__device__ __forceinline__ void store_rows(uint32_t stage, const CUtensorMap *map, int lane, int col0, int row0, int g, const uint32_t (&w)[32])
{
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (lane == 0) ptx::bulk_wait_read();                      // the store before has read the area
        __syncwarp();
        if ((lane >> 4) == h) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                             ::"r"(stage + (lane & 15) * 128 + ((j ^ (lane & 7)) << 4)), "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3]) : "memory");
            ptx::fence_async_shared();
        }
        __syncwarp();
        if (lane == 0) ptx::tma_store_3d(map, stage, col0, row0 + 16 * h, g);
    }
}

// The parts of a tile's K loop meet in the cluster's shared memory, over the stages, which are free once
// every CTA's MMAs are done.  The epilogue warps of one number share a piece of the tile; one of them,
// a different CTA's for each number, adds the others' parts to its own in their order.  Called by the epilogue warps of all
// CTAs, each with its part in `sum` (the other warps take part in the two cluster barriers); true for the
// warp that has the result.  live: the piece has rows to store.
template <int CH>
__device__ __forceinline__ bool join(uint32_t smem_base, const uint8_t *gen_base, int warp, int lane, int part, int splits, bool live,
                                     float (&sum)[CH][32])
{
    const int owner = warp % splits;
    auto place = [&](int of) { return uint32_t(((of < owner ? of : of - 1) * 8 + warp) * CH * 4096 + lane * 4); };
    __syncwarp();
    cluster_sync();
    if (part != owner && live) {
        const uint32_t to = ptx::map_to_cta(smem_base + place(part), uint32_t(owner));
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 32; i++)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + c * 4096 + i * 128), "f"(sum[c][i]) : "memory");
    }
    __syncwarp();
    cluster_sync();
    if (part != owner || !live) return false;
    for (int of = 0; of < splits; of++) {
        if (of == owner) continue;
        const float *from = reinterpret_cast<const float *>(gen_base + place(of));
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 32; i++) sum[c][i] += from[c * 1024 + i * 32];
    }
    return true;
}

// One output tile of the CTA (pair): everything the three roles need.
struct Item {
    int g;                         // group
    int row0, row_end;             // this CTA's first output row, and the end of the rows it may store
    int n0;                        // first output column
    int k0;                        // first block of K of this CTA
    int kb0, nkb;                  // blocks of K: scale index of the first, count
    int slot;                      // this CTA's row tile in A's scale buffer
};

// LONG: sums of more than kSegment blocks in fp32 output.  The tensor core's accumulator drops what does
// not fit as it adds, always in one direction, so the error of one chain grows with its length (relative
// to 64 bits: 3.4e-7 after 2048 values of K, 3.6e-6 after 16384).  The K loop is cut into segments of
// kSegment blocks, each a chain of its own, that the epilogue adds in registers: 2.2e-7 after 16384
// (torch's fp32 product: 3.6e-7) in 54 us for 4096 x 1024 outputs; segments half as long give 1.2e-7
// in 57 us, one chain takes 51 us.
template <int CTAS, int BN, int FORM, bool LONG, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                const __grid_constant__ CUtensorMap tm_c, const Fp8Params p)
{
    using C = Fp8Cfg<CTAS, BN>;
    constexpr bool A_MN = FORM == TN, B_MN = FORM != NT;
    static_assert(!SPLIT || (CTAS == 1 && (kMaxSplits - 1) * C::PART_BYTES <= C::STAGING), "partial sums overflow the stages");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *gen_base = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t bar_base = smem_base + C::TAIL;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (C::STAGES + s); };
    // One "full" barrier per accumulator: with accumulators that share nothing, two tiles can be
    // finished while a slow epilogue warp still stores the one before them, and a single barrier
    // would be two phases ahead of it.
    const uint32_t acc_full_bar = bar_base + 8u * (2 * C::STAGES);
    const uint32_t acc_free_bar = acc_full_bar + 16u;      // two of them when the accumulators share nothing
    const uint32_t tmem_slot = acc_free_bar + 16u;
    volatile uint32_t *tmem_slot_p = reinterpret_cast<volatile uint32_t *>(gen_base + C::TAIL + 8 * (2 * C::STAGES + 4));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot_p + 1);
    int *list_pre = reinterpret_cast<int *>(gen_base + C::LIST);       // [groups + 1] tiles (of 128 CTAS rows) before a group

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = CTAS == 2 ? cluster_ctarank() : 0u;
    const int splits = SPLIT ? p.splits : 1, part = SPLIT ? int(cluster_ctarank()) : 0;
    const int worker = blockIdx.x / (CTAS * splits), workers = gridDim.x / (CTAS * splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(acc_full_bar, 1);
        ptx::mbar_init(acc_full_bar + 8u, 1);
        ptx::mbar_init(acc_free_bar, 8 * CTAS);
        ptx::mbar_init(acc_free_bar + 8u, 8 * CTAS);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tm_a);
        ptx::prefetch_tmap(&tm_b);
        ptx::prefetch_tmap(&tm_sfa);
        ptx::prefetch_tmap(&tm_sfb);
        // The first tiles of a dense forward product's weight start towards L2 while the kernel before
        // (the quantizer of A) still runs.  Only a hint: L2 stays coherent with whoever writes them.
        if (FORM == NT && !p.offsets) {
            const int n0 = worker / ((p.M + 128 * CTAS - 1) / (128 * CTAS)) * BN + int(cta) * C::BCOLS;
            const int k0 = SPLIT ? part * (((p.K + kBlock - 1) / kBlock + splits - 1) / splits) : 0;
            for (int k = k0; k < k0 + C::STAGES && k * kBlock < p.K && n0 < p.N; k++)
#pragma unroll
                for (int b = 0; b < (C::BCOLS + 127) / 128; b++) ptx::tma_prefetch_3d(&tm_b, k * kBlock, n0 + 128 * b, 0);
        }
    }
    if (warp == 1) {
        ptx::tmem_alloc<CTAS>(tmem_slot, kTmemCols);
        ptx::tmem_relinquish<CTAS>();
    }
    // (every thread waits here: rows of no group are stored without a load)
    begin_dependent_launch();
    if (warp == 2 && p.offsets) {
        const int rows = FORM == TN ? p.K : p.M;
        int before = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            const int g = g0 + lane;
            int lo = rows, hi = rows;
            if (g < p.groups) lo = group_lo(p.offsets, g, rows), hi = group_hi(p.offsets, g, rows, lo);
            const int own = (hi - lo + 128 * CTAS - 1) / (128 * CTAS);
            int sum = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                if (lane >= o) sum += v;
            }
            if (g < p.groups) {
                list_pre[g] = before + sum - own;
                if (g == p.groups - 1) list_pre[p.groups] = before + sum;
            }
            before = min(before + __shfl_sync(0xFFFFFFFFu, sum, 31), 1 << 30);     // (only offsets out of order reach the limit)
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();                          // both CTAs' barriers exist before any remote arrive
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot_p;

    // ---- the list of tiles, the same for every role
    // (more tiles than ordered offsets can have would be those of overlapping groups: no sense, and no bound)
    const int m_tiles = FORM == TN || !p.offsets ? (p.M + 128 * CTAS - 1) / (128 * CTAS)
                                                 : min(list_pre[p.groups], p.M / (128 * CTAS) + p.groups);
    const int n_tiles = (p.N + BN - 1) / BN;
    const int items = m_tiles * n_tiles * (FORM == TN ? p.groups : 1);
    auto item_of = [&](int t) {
        Item it;
        if (FORM == TN) {
            const int mt = t % m_tiles, rest = t / m_tiles;
            it.n0 = rest % n_tiles * BN;
            it.g = rest / n_tiles;
            it.row0 = mt * 128 * CTAS + 128 * int(cta);
            it.row_end = p.M;
            it.slot = mt * CTAS + int(cta);
            const int lo = p.offsets ? group_lo(p.offsets, it.g, p.K) : 0;
            const int hi = p.offsets ? group_hi(p.offsets, it.g, p.K, lo) : p.K;
            it.kb0 = p.offsets ? lo / 128 + it.g : 0;
            it.nkb = (hi - lo + kBlock - 1) / kBlock;
        } else {
            // Group after group (a group's rows and weight are then used up while they are in L2), rows
            // of tiles inside a column of tiles.
            it.g = 0;
            int lo = 0, hi = p.M, i = t, mine = m_tiles;
            if (p.offsets) {
                int a = 0, b = p.groups - 1;                // last group whose tiles start at or before t
                const int column = t / n_tiles;
                while (a < b) {
                    const int m = (a + b + 1) >> 1;
                    if (list_pre[m] <= column) a = m;
                    else b = m - 1;
                }
                it.g = a;
                lo = group_lo(p.offsets, a, p.M), hi = group_hi(p.offsets, a, p.M, lo);
                i = t - list_pre[a] * n_tiles, mine = list_pre[a + 1] - list_pre[a];
            }
            const int nt = i / mine;
            i -= nt * mine;
            it.n0 = nt * BN;
            it.row0 = lo + (i * CTAS + int(cta)) * 128;
            it.row_end = hi;
            it.slot = (p.offsets ? lo / 128 + it.g : 0) + i * CTAS + int(cta);
            it.kb0 = 0;
            it.nkb = (p.K + kBlock - 1) / kBlock;
        }
        it.k0 = 0;
        if (SPLIT) {                                        // dense: every part has blocks (the host sees to it)
            const int per = (it.nkb + splits - 1) / splits;
            it.k0 = part * per;
            it.kb0 += it.k0;
            it.nkb = min(it.nkb, it.k0 + per) - it.k0;
        }
        return it;
    };

    if (warp == 0) {
        // ------------------------------------------------------------ producer (every CTA)
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = worker; t < items && ok; t += workers) {
                const Item it = item_of(t);
                const int sfb0 = (FORM == TN ? 0 : it.g * p.sfb_rt) + it.n0 / 128;
                // the second CTA of a pair whose group ended in the first one's rows multiplies zeros (rows behind
                // the tensor), not the next group's rows: that takes less power
                const int row_a = CTAS == 2 && FORM != TN && it.row0 >= it.row_end ? p.M : it.row0;
                for (int k = 0; k < it.nkb; k++) {
                    if (!(ok = ptx::mbar_wait(empty_bar(s), ph ^ 1, abort_flag))) break;
                    const int kb = it.kb0 + k;
                    const bool scales = k == 0 || (kb & 3) == 0;        // a scale tile lasts four blocks
                    const uint32_t st = smem_base + s * C::STAGE_BYTES;
                    // CTAS = 2: every load of either CTA completes on CTA 0's barrier
                    const uint32_t bar = CTAS == 2 ? ptx::map_to_cta(full_bar(s), 0) : full_bar(s);
                    if (cta == 0)
                        ptx::mbar_expect_tx(full_bar(s), CTAS * (p.a_bytes + C::B_BYTES + (scales ? 512u * (1 + C::SFB_TILES) : 0u)));
                    if (A_MN) ptx::tma_load_3d<CTAS>(st, &tm_a, it.row0, kb * kBlock, 0, bar);
                    else ptx::tma_load_3d<CTAS>(st, &tm_a, (it.k0 + k) * kBlock, row_a, 0, bar);
                    const uint32_t stb = st + C::A_BYTES;
                    const int nb0 = it.n0 + int(cta) * C::BCOLS;
#pragma unroll
                    for (int b = 0; b < (C::BCOLS + 127) / 128; b++) {
                        if (!B_MN) ptx::tma_load_3d<CTAS>(stb + b * 128 * kBlock, &tm_b, (it.k0 + k) * kBlock, nb0 + 128 * b, it.g, bar);
                        else if (FORM == NN) ptx::tma_load_3d<CTAS>(stb + b * 128 * kBlock, &tm_b, nb0 + 128 * b, (it.k0 + k) * kBlock, it.g, bar);
                        else ptx::tma_load_3d<CTAS>(stb + b * 128 * kBlock, &tm_b, nb0 + 128 * b, kb * kBlock, 0, bar);
                    }
                    if (scales) {
                        const uint32_t stf = stb + C::B_BYTES;
                        ptx::tma_load_3d<CTAS>(stf, &tm_sfa, 0, it.slot * p.sfa_kt + (kb >> 2), 0, bar);
#pragma unroll
                        for (int b = 0; b < C::SFB_TILES; b++)
                            ptx::tma_load_3d<CTAS>(stf + 512 * (1 + b), &tm_sfb, 0, (sfb0 + b) * p.sfb_kt + (kb >> 2), 0, bar);
                    }
                    if (++s == C::STAGES) s = 0, ph ^= 1;
                }
            }
            for (int i = 0; i < C::STAGES && ok; i++) {     // wait until the MMA side is done with every stage
                ok = ptx::mbar_wait(empty_bar(s), ph ^ 1, abort_flag);
                if (++s == C::STAGES) s = 0, ph ^= 1;
            }
        }
    } else if (warp == 1 && cta == 0) {
        // ------------------------------------------------------------ MMA issuer (CTA 0 of a pair)
        if (ptx::elect_one()) {
            constexpr uint32_t idesc = ptx::idesc_mxf8(128 * CTAS, BN, A_MN, B_MN);
            const uint64_t adesc0 = A_MN ? ptx::desc_sw128_mn(smem_base, 128 * kBlock) : ptx::desc_sw128(smem_base);
            const uint64_t bdesc0 = B_MN ? ptx::desc_sw128_mn(smem_base + C::A_BYTES, 128 * kBlock) : ptx::desc_sw128(smem_base + C::A_BYTES);
            const uint64_t sfdesc0 = ptx::desc_sf(smem_base + C::A_BYTES + C::B_BYTES);
            constexpr uint32_t A_STEP = A_MN ? 32 * 128 / 16 : 2, B_STEP = B_MN ? 32 * 128 / 16 : 2;   // 32 values of K
            const uint32_t sfa_t = tmem_base + C::SFA_COL, sfb_t = tmem_base + C::SFB_COL;
            int s = 0, lt = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = worker; t < items && ok; t += workers) {
                const Item it = item_of(t);
                // a 64-column tile uses one half of a 128-row scale tile: rows 32 c .. + 31 sit in column c
                const uint32_t sfb_sub = BN >= 128 ? 0u : uint32_t(it.n0 & 127) / 32u;
                // (an empty group's weight gradient has no blocks: no sum to take)
                for (int k0 = 0; k0 < it.nkb && ok; k0 += LONG ? kSegment : it.nkb, lt++) {
                    if (C::OVL > 0) {
                        // the sum before this one has been read out of the columns the two accumulators share
                        if (lt > 0 && !(ok = ptx::mbar_wait(acc_free_bar, (lt - 1) & 1, abort_flag))) break;
                    } else {
                        // this accumulator's previous sum (two back) has been read out
                        if (lt > 1 && !(ok = ptx::mbar_wait(acc_free_bar + 8u * (lt & 1), ((lt >> 1) - 1) & 1, abort_flag))) break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t acc = tmem_base + ((lt & 1) ? C::ACC1 : 0);
                    const int k1 = LONG ? min(k0 + kSegment, it.nkb) : it.nkb;
                    for (int k = k0; k < k1; k++) {
                        if (!(ok = ptx::mbar_wait(full_bar(s), ph, abort_flag))) break;
                        ptx::tc_fence_after();
                        const int kb = it.kb0 + k;
                        const uint32_t st16 = uint32_t(s) * (C::STAGE_BYTES >> 4);
                        if (k == 0 || (kb & 3) == 0) {
#pragma unroll
                            for (int b = 0; b < 1 + C::SFB_TILES; b++) ptx::tmem_cp_sf<CTAS>(sfa_t + 4 * b, sfdesc0 + st16 + 32 * b);
                        }
                        const uint32_t id = uint32_t(kb & 3);   // byte of the scale column
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            ptx::mma_mxf8<CTAS>(acc, adesc0 + st16 + A_STEP * j, bdesc0 + st16 + B_STEP * j, idesc | (id << 29) | (id << 4),
                                                sfa_t + (id << 30), sfb_t + sfb_sub + (id << 30), (k == k0 && j == 0) ? 0u : 1u);
                        if (CTAS == 2) ptx::tc_commit_pair(empty_bar(s), 3);
                        else ptx::tc_commit(empty_bar(s));
                        if (++s == C::STAGES) s = 0, ph ^= 1;
                    }
                    if (ok) {
                        if (CTAS == 2) ptx::tc_commit_pair(acc_full_bar + 8u * (lt & 1), 3);
                        else ptx::tc_commit(acc_full_bar + 8u * (lt & 1));
                    }
                }
            }
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------------ epilogue (every CTA)
        // Warp w reads the tensor-memory lanes of quarter w % 4 and one half of the tile's columns.
        const int q = warp & 3, half = (warp - 2) >> 2;
        const bool bf16 = p.out_bf16 != 0;
        uint32_t *stage = reinterpret_cast<uint32_t *>(gen_base + C::STAGING) + (warp - 2) * kStagingWords;
        const bool vec = p.N % (bf16 ? 8 : 4) == 0;
        const uint32_t stage_addr = smem_base + C::STAGING + (warp - 2) * kStagingWords * 4;
        int lt = 0;
        bool ok = true;
        for (int t = worker; t < items && ok; t += workers) {
            const Item it = item_of(t);
            constexpr int CH = BN / 64;                     // chunks of 32 columns per warp
            uint8_t *dst = static_cast<uint8_t *>(p.c) + (FORM == TN ? int64_t(it.g) * p.M * p.N * (bf16 ? 2 : 4) : 0);
            const int row = it.row0 + 32 * q;
            const bool tma = BN >= 128 && vec && row + 32 <= it.row_end;           // uniform over the warp
            const int zc = FORM == TN ? it.g : 0;
            auto emit = [&](int c, const uint32_t (&r)[32]) {
                const int col0 = it.n0 + 32 * c;
                if (!vec) store_ragged(stage, it.row_end, p.N, dst, bf16, row, lane, col0, r);
                else if (!tma || bf16) store_chunk(it.row_end, p.N, dst, bf16, row, lane, col0, r);
                else if (col0 < p.N) store_rows(stage_addr, &tm_c, lane, col0, row, zc, r);
            };
            if (it.nkb == 0) {
                uint32_t z[32];
#pragma unroll
                for (int i = 0; i < 32; i++) z[i] = 0u;
#pragma unroll 1
                for (int i = 0; i < CH; i++) emit(CH * half + i, z);
                continue;
            }
            auto release = [&]() {
                ptx::tc_fence_before();
                __syncwarp();
                const uint32_t bar = acc_free_bar + (C::OVL > 0 ? 0u : 8u * (lt & 1));
                if (lane == 0) {
                    if (CTAS == 2) ptx::mbar_arrive_cluster(bar, 0);
                    else ptx::mbar_arrive(bar);
                }
            };
            // The 32 columns shared by the accumulators are the last chunk of accumulator 0 and the
            // first of accumulator 1: their owners read them first and then let the next sum's MMAs
            // start; the other warps do so at once.  Without shared columns a warp frees its
            // accumulator when its last load has landed.
            if constexpr (LONG) {
                float sum[CH][32];
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int i = 0; i < 32; i++) sum[c][i] = 0.0f;
                for (int k0 = 0; k0 < it.nkb && ok; k0 += kSegment, lt++) {
                    if (!(ok = ptx::mbar_wait(acc_full_bar + 8u * (lt & 1), (lt >> 1) & 1, abort_flag))) break;
                    ptx::tc_fence_after();
                    const uint32_t acc = tmem_base + ((lt & 1) ? C::ACC1 : 0) + (uint32_t(32 * q) << 16) + 32 * CH * half;
                    const bool last_first = C::OVL > 0 && !(lt & 1) && half == 1, owner = C::OVL > 0 && ((lt & 1) ? half == 0 : half == 1);
                    auto add = [&](int c, float (&to)[32]) {
                        uint32_t r[32];
                        ptx::tmem_ld32(acc + 32 * c, r);
                        ptx::tmem_ld_wait(r);
#pragma unroll
                        for (int i = 0; i < 32; i++) to[i] += __uint_as_float(r[i]);
                    };
                    if (C::OVL > 0 && !owner) release();
                    if (last_first) add(CH - 1, sum[CH - 1]), release();
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        if (c < CH - 1 || !last_first) add(c, sum[c]);
                        if (c == 0 && owner && !last_first) release();
                    }
                    if (C::OVL == 0) release();
                }
                if constexpr (SPLIT)
                    if (!join<CH>(smem_base, gen_base, warp - 2, lane, part, splits, row < it.row_end, sum)) continue;
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    uint32_t r[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) r[i] = __float_as_uint(sum[c][i]);
                    emit(CH * half + c, r);
                }
                continue;
            }
            if constexpr (SPLIT) {
                {                                           // one tile per CTA: nobody waits for this accumulator
                    float sum[CH][32];
                    ok = ptx::mbar_wait(acc_full_bar, 0, abort_flag);
                    ptx::tc_fence_after();
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        uint32_t r[32];
                        ptx::tmem_ld32(tmem_base + (uint32_t(32 * q) << 16) + 32 * (CH * half + c), r);
                        ptx::tmem_ld_wait(r);
#pragma unroll
                        for (int i = 0; i < 32; i++) sum[c][i] = __uint_as_float(r[i]);
                    }
                    if (!join<CH>(smem_base, gen_base, warp - 2, lane, part, splits, row < it.row_end, sum) || !ok) continue;
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        uint32_t r[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) r[i] = __float_as_uint(sum[c][i]);
                        emit(CH * half + c, r);
                    }
                    continue;
                }
            }
            if (!(ok = ptx::mbar_wait(acc_full_bar + 8u * (lt & 1), (lt >> 1) & 1, abort_flag))) break;
            ptx::tc_fence_after();
            const uint32_t acc = tmem_base + ((lt & 1) ? C::ACC1 : 0) + (uint32_t(32 * q) << 16);
            const bool owner = C::OVL > 0 && ((lt & 1) ? half == 0 : half == 1);
            if (C::OVL > 0 && !owner) release();
            uint32_t ra[32], rb[32];
            if constexpr (CH == 1) {
                ptx::tmem_ld32(acc + 32 * half, ra);
                ptx::tmem_ld_wait(ra);
                release();
                emit(half, ra);
            } else if (!vec) {
                // chunk after chunk; the next one's load is in flight while this one is stored
                const int start = owner && !(lt & 1) ? CH - 1 : 0;
                auto chunk = [&](int i) { return CH * half + (C::OVL > 0 ? ((start + i) & (CH - 1)) : i); };
                ptx::tmem_ld32(acc + 32 * chunk(0), ra);
#pragma unroll 1
                for (int i = 0; i < CH; i += 2) {
                    ptx::tmem_ld_wait(ra);
                    ptx::tmem_ld32(acc + 32 * chunk(i + 1), rb);
                    if (i == 0 && owner) release();
                    store_ragged(stage, it.row_end, p.N, dst, bf16, row, lane, it.n0 + 32 * chunk(i), ra);
                    ptx::tmem_ld_wait(rb);
                    if (i + 2 < CH) ptx::tmem_ld32(acc + 32 * chunk(i + 2), ra);
                    else if (C::OVL == 0) release();
                    store_ragged(stage, it.row_end, p.N, dst, bf16, row, lane, it.n0 + 32 * chunk(i + 1), rb);
                }
            } else {
                // pairs of chunks (64 bf16 columns are whole lines), the one with the shared columns first
                const int first = owner && !(lt & 1) ? CH / 2 - 1 : 0;
#pragma unroll 1
                for (int i = 0; i < CH / 2; i++) {
                    const int c = CH * half + 2 * (first ^ i), col0 = it.n0 + 32 * c;
                    ptx::tmem_ld32(acc + 32 * c, ra);
                    ptx::tmem_ld32(acc + 32 * c + 32, rb);
                    ptx::tmem_ld_wait(ra);
                    ptx::tmem_ld_wait(rb);
                    if (i == 0 && owner) release();
                    if (C::OVL == 0 && i == CH / 2 - 1) release();
                    if (!tma) {
                        store_chunk(it.row_end, p.N, dst, bf16, row, lane, col0, ra);
                        store_chunk(it.row_end, p.N, dst, bf16, row, lane, col0 + 32, rb);
                    } else if (!bf16) {
                        if (col0 < p.N) store_rows(stage_addr, &tm_c, lane, col0, row, zc, ra);
                        if (col0 + 32 < p.N) store_rows(stage_addr, &tm_c, lane, col0 + 32, row, zc, rb);
                    } else if (col0 < p.N) {
                        uint32_t w[32];
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(ra[2 * k]), __uint_as_float(ra[2 * k + 1]));
                            const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(rb[2 * k]), __uint_as_float(rb[2 * k + 1]));
                            w[k] = *reinterpret_cast<const uint32_t *>(&x), w[16 + k] = *reinterpret_cast<const uint32_t *>(&y);
                        }
                        store_rows(stage_addr, &tm_c, lane, col0, row, zc, w);
                    }
                }
            }
            lt++;
        }
        if (lane == 0) ptx::bulk_wait_all();                // (none of its own: returns at once)
        if (FORM != TN && p.offsets && p.zero_tail) {       // rows behind the last group
            const int64_t bytes = int64_t(p.N) * (bf16 ? 2 : 4);
            uint8_t *dst = static_cast<uint8_t *>(p.c);
            const int first = group_hi(p.offsets, p.groups - 1, p.M, group_lo(p.offsets, p.groups - 1, p.M));
            for (int r = first + blockIdx.x * 8 + warp - 2; r < p.M; r += gridDim.x * 8) {
                uint8_t *line = dst + r * bytes;
                if (bytes % 16 == 0)
                    for (int64_t i = lane; i < bytes / 16; i += 32) reinterpret_cast<uint4 *>(line)[i] = make_uint4(0, 0, 0, 0);
                else
                    for (int64_t i = lane; i < bytes / 2; i += 32) reinterpret_cast<uint16_t *>(line)[i] = 0;
            }
        }
    }

    if (SPLIT && warp < 2) {                                // the other side of join()
        __syncwarp();
        cluster_sync();
        cluster_sync();
    }

    // ---------------------------------------------------------------- teardown
    if (*abort_flag) {
        for (int i = 0; i < 4096; i++) __nanosleep(256);    // copies and MMAs in flight land before memory is released
        if (threadIdx.x == 0) atomicExch(p.err, 1);
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (CTAS == 2 || SPLIT) cluster_sync();        // no CTA leaves while another may still signal or write to it
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<CTAS>(tmem_base, kTmemCols);
    }
}

// ---- launches ---------------------------------------------------------------------
template <int CTAS, int BN, int FORM, bool LONG, bool SPLIT>
int launch(const Fp8Maps &m, const Fp8Params &p, int64_t most_tiles, cudaStream_t st)
{
    using C = Fp8Cfg<CTAS, BN>;
    static int resident[64] = {};                           // CTAs (pairs) of this kernel that fit at once, per device
    const unsigned cluster = unsigned(CTAS * p.splits);
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    std::unique_lock<std::mutex> lk(state_mutex());
    if (!resident[dev]) {
        LS_CUDA(cudaFuncSetAttribute(fp8_gemm_kernel<CTAS, BN, FORM, LONG, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        int n = sm_count();
        if (CTAS == 2) {
            cfg.gridDim = dim3(unsigned(sm_count() & ~1), 1, 1);
            cfg.attrs = at + 1, cfg.numAttrs = 1;
            LS_CUDA(cudaOccupancyMaxActiveClusters(&n, fp8_gemm_kernel<CTAS, BN, FORM, LONG, SPLIT>, &cfg));
            if (n < 1) return fail(LS_ECUDA, "no CTA pair of the FP8 product fits on this device");
        }
        resident[dev] = n;
    }
    // (a K split has one tile per cluster, and needs no two clusters at once)
    const int64_t workers = p.splits > 1 ? most_tiles : std::max<int64_t>(1, std::min<int64_t>(most_tiles, resident[dev]));
    lk.unlock();
    cfg.gridDim = dim3(unsigned(cluster * workers), 1, 1);
    cfg.attrs = at, cfg.numAttrs = cluster > 1 ? 2 : 1;
    LS_CUDA(cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<CTAS, BN, FORM, LONG, SPLIT>, m.a, m.b, m.sfa, m.sfb, m.c, p));
    return LS_OK;
}

// The kernel that fp8_gemm.cu chose for one form: pairs, or single CTAs with tiles of `bn` columns.
template <int FORM>
int launch_form(bool pair, int bn, bool many, const Fp8Maps &m, const Fp8Params &p, int64_t items, cudaStream_t st)
{
#define LS_FP8_LAUNCH(C, B, S) \
    return many ? launch<C, B, FORM, true, S>(m, p, items, st) : launch<C, B, FORM, false, S>(m, p, items, st)
    if (pair) LS_FP8_LAUNCH(2, 256, false);
    if (bn == 256) LS_FP8_LAUNCH(1, 256, false);
    if constexpr (FORM == NT) {
        if (bn == 64 && p.splits > 1) LS_FP8_LAUNCH(1, 64, true);
        if (bn == 64) LS_FP8_LAUNCH(1, 64, false);
    }
    if (p.splits > 1) LS_FP8_LAUNCH(1, 128, true);
    LS_FP8_LAUNCH(1, 128, false);
#undef LS_FP8_LAUNCH
}

}  // namespace

// one translation unit per form
int fp8_launch_nt(bool pair, int bn, bool many, const Fp8Maps &m, const Fp8Params &p, int64_t items, cudaStream_t st);
int fp8_launch_nn(bool pair, int bn, bool many, const Fp8Maps &m, const Fp8Params &p, int64_t items, cudaStream_t st);
int fp8_launch_tn(bool pair, int bn, bool many, const Fp8Maps &m, const Fp8Params &p, int64_t items, cudaStream_t st);
int fp8_cluster_room(int size);         // clusters of `size` single CTAs that run at once on the current device (0: unknown)

}  // namespace ls
