// The FP8 linear layer for a handful of rows (one decoded token, or a few per expert): y = q(x) w^T
// in one launch, x quantized on the fly.
//
// Bound by the weight stream (one byte per weight) and, below that, by latency: at 4096 x 4096 the
// stream is 2.6 us.  A CTA of 8 warps takes up to 8 tiles of 16 output columns (as many as leave three
// CTAs per SM: what a CTA does once, finding its group and quantizing x, is then paid less often);
// its warps take every eighth of the tiles' blocks of 128 along K, and every lane copies its own 16-byte pieces of the warp's next four blocks to shared
// memory (cp.async: 64 KB per CTA in flight, no barrier between warps; loads to registers four blocks
// ahead waited for one another and reached half the rate).  While the first blocks are on their
// way, the CTA quantizes its rows of x to shared memory.
// The codes become f16 (exact) for mma.sync.m16n8k16, whose n = 8 columns are the rows of x: the
// tensor work is a few per cent of the stream's time either way, and tcgen05 would add the set-up of
// tensor memory, barriers and tensor maps to a kernel of a few microseconds.  A lane's 16-byte
// piece of a weight row is 16 consecutive k, so the k order inside a block is permuted alike for
// both operands.  Each block's sum (K = 128) leaves the MMA chain and is scaled and added in fp32;
// the warps' sums are added in a fixed order.
#include <algorithm>

#include <cuda_fp16.h>

#include "fp8.cuh"

namespace ls {
namespace {

constexpr int kWarps = 8, kRowsPerPass = 8, kAhead = 4, kMaxTiles = 8;

struct SkinnyArgs {
    int rows, K, N;
    const uint8_t *codes;           // [groups, N, K], pitch ld
    int64_t ld;
    const uint8_t *sf;              // scale tiles of the weights, group after group
    void *out;
    int out_bf16;
    const int *offsets;             // ragged groups, or NULL
    int groups, zero_tail;
    int tiles;                      // of 16 columns per CTA
};

// four E4M3 codes -> two f16 pairs
__device__ __forceinline__ void to_half(uint32_t codes, uint32_t &lo, uint32_t &hi)
{
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi) : "r"(codes));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, 3)
fp8_skinny_kernel(const T *__restrict__ x, const SkinnyArgs p)
{
    using W = Word<T>;
    constexpr int WORDS = 16 * int(sizeof(T)) / 4;          // words of 16 values
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * 16 * p.tiles, tiles = min(p.tiles, (p.N - n0 + 15) / 16);
    // A dense weight's rows start towards L2 while the kernel before still runs (only a hint: L2 stays
    // coherent with whoever writes them): the lines of the first two blocks of every warp.
    if (!p.offsets)
        for (int i = threadIdx.x; i < 16 * 2 * kWarps; i += 32 * kWarps) {
            const int r = n0 + i / (2 * kWarps), k = i % (2 * kWarps) * 128;
            if (r < p.N && k < p.K) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.codes + int64_t(r) * p.ld + k));
        }
    begin_dependent_launch();
    const int kb_count = (p.K + 127) / 128, kt = (kb_count + 3) / 4;

    int group = 0, lo = 0, hi = p.rows;
    if (p.offsets) {
        // this CTA's group: number blockIdx.y of those that have rows
        int want = blockIdx.y;
        group = -1;
        for (int g0 = 0; g0 < p.groups && group < 0; g0 += 32) {
            const int i = g0 + lane;
            int a = 0, b = 0;
            if (i < p.groups) a = group_lo(p.offsets, i, p.rows), b = group_hi(p.offsets, i, p.rows, a);
            uint32_t mask = __ballot_sync(0xFFFFFFFFu, b > a);
            if (want < __popc(mask)) {
                for (; want > 0; want--) mask &= mask - 1;
                const int at = __ffs(mask) - 1;
                group = g0 + at, lo = __shfl_sync(0xFFFFFFFFu, a, at), hi = __shfl_sync(0xFFFFFFFFu, b, at);
            } else {
                want -= __popc(mask);
            }
        }
        if (blockIdx.y == 0 && p.zero_tail) {               // rows behind the last group
            const int a = group_lo(p.offsets, p.groups - 1, p.rows), first = group_hi(p.offsets, p.groups - 1, p.rows, a);
            const int width = min(16 * tiles, p.N - n0);
            for (int i = threadIdx.x; i < (p.rows - first) * width; i += 32 * kWarps) {
                const int r = i / width;
                const int64_t at = int64_t(first + r) * p.N + n0 + i - r * width;
                if (p.out_bf16) static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(0.0f);
                else static_cast<float *>(p.out)[at] = 0.0f;
            }
        }
        if (group < 0) return;                              // uniform over the CTA
    }
    const uint8_t *codes = p.codes + int64_t(group) * p.N * p.ld;
    // Shared memory: the ring of weight pieces; x as f16 values of its codes, rows 16 bytes apart modulo
    // 128 (the eight lanes of a 16-byte access then cover all banks); x's block scales; the scale bytes
    // of the weight rows; the warps' sums.
    extern __shared__ uint4 smem[];
    uint4 *ring = smem;                                     // [kAhead][4 pieces][thread]
    const int ldx = kb_count * 128 + 8;
    __half *xs = reinterpret_cast<__half *>(smem + kAhead * 4 * 32 * kWarps);
    float *xscale = reinterpret_cast<float *>(xs + min(kRowsPerPass, p.rows) * ldx);
    uint32_t *wscale = reinterpret_cast<uint32_t *>(xscale + min(kRowsPerPass, p.rows) * kb_count);     // [16 tiles][kt] words
    float *sums = reinterpret_cast<float *>(wscale + 16 * p.tiles * kt);                                // [warp][tile][row][column]
    const int sums_warp = p.tiles * 16 * kRowsPerPass;
    // A warp's place in the list of (tile, block), which it walks in steps of kWarps
    struct Place { int tile, kb; };
    auto advance = [&](Place &a) {
        for (a.kb += kWarps; a.kb >= kb_count; a.kb -= kb_count) a.tile++;
    };
    Place first{0, warp};
    for (; first.kb >= kb_count; first.kb -= kb_count) first.tile++;
    auto fetch = [&](const Place &a, int stage) {           // one commit group per call
        if (a.tile < tiles) {
            // columns past N repeat the last and are not stored
            const uint8_t *rows2[2] = {codes + int64_t(min(n0 + 16 * a.tile + g, p.N - 1)) * p.ld,
                                       codes + int64_t(min(n0 + 16 * a.tile + g + 8, p.N - 1)) * p.ld};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = a.kb * 128 + 64 * (i & 1) + 16 * c;
                const int left = min(max(p.K - k, 0), 16);  // bytes behind the row's end are not read, but zeros
                const uint8_t *src = rows2[i >> 1] + (left > 0 ? k : 0);
                const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[(stage * 4 + i) * 32 * kWarps + threadIdx.x]));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(left) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const uint8_t *sf = p.sf + int64_t(group) * fp8_sf_tiles_dev(p.N, kb_count) * 512;

    for (int r0 = lo; r0 < hi; r0 += kRowsPerPass) {
        const int n = min(kRowsPerPass, hi - r0);
        Place now = first, ahead = first;
#pragma unroll
        for (int d = 0; d < kAhead; d++) {
            fetch(ahead, d);
            advance(ahead);
        }
        for (int i = lane; i < sums_warp; i += 32) sums[warp * sums_warp + i] = 0.0f;
        for (int i = threadIdx.x; i < 16 * tiles * kt; i += 32 * kWarps) {
            const int r = i / kt, t = i - r * kt;
            wscale[i] = *reinterpret_cast<const uint32_t *>(sf + sf_offset(uint32_t(min(n0 + r, p.N - 1)), uint32_t(4 * t), uint32_t(kt)));
        }

        const int chunks = (p.K + 511) / 512;               // a warp takes 512 values of a row, eight lanes a block
        for (int i = warp; i < n * chunks; i += kWarps) {
            const int r = i / chunks, col = (i - r * chunks) * 512 + lane * 16;
            const T *src = x + int64_t(r0 + r) * p.K + col;
            uint32_t v[WORDS];
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < WORDS / 4; j++) {
                    const uint4 q = p.K - col > j * 16 / int(sizeof(T)) ? __ldg(reinterpret_cast<const uint4 *>(src) + j) : make_uint4(0, 0, 0, 0);
                    v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
                }
            } else {
                load_ragged<WORDS>(src, p.K - col, v);
            }
            auto largest = [&]() {
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < WORDS; j++) m = W::max_of(m, v[j]);
                return W::fold(m);
            };
            uint32_t m = largest(), flags = 0;
            const bool special = __any_sync(0xFFFFFFFFu, m >= kBitsInf);
            if (special) {
#pragma unroll
                for (int j = 0; j < WORDS; j++) flags |= W::drop_special(v[j]) << (16 / WORDS * j);
                m = largest();
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const uint32_t e8 = fp8_e8m0(m), inv1 = W::inv(e8);
            if (col < kb_count * 128) {
                const uint32_t inv[4] = {inv1, inv1, inv1, inv1};
                uint32_t h[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t q = W::codes(v + WORDS / 4 * j, inv);
                    if (special) q |= ((((flags >> (4 * j)) & 15u) * 0x00204081u) & 0x01010101u) * 0x7Fu;       // NaN codes
                    to_half(q, h[2 * j], h[2 * j + 1]);
                }
                uint4 *dst = reinterpret_cast<uint4 *>(xs + r * ldx + col);
                dst[0] = make_uint4(h[0], h[1], h[2], h[3]), dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
                if ((lane & 7) == 0) xscale[r * kb_count + col / 128] = __uint_as_float(e8 << 23);
            }
        }
        __syncthreads();
        // This lane's row of x as the B operand (k along the lane's pieces), and the scales of the two
        // rows whose sums it holds; rows that do not exist are zeros.
        const bool have = g < n, have0 = 2 * c < n, have1 = 2 * c + 1 < n;
        const __half *xg = xs + (have ? g : 0) * ldx + 16 * c;
        const float *sc0 = xscale + (have0 ? 2 * c : 0) * kb_count, *sc1 = xscale + (have1 ? 2 * c + 1 : 0) * kb_count;
        float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float *mine = sums + warp * sums_warp + 32 * c + g;        // rows 2 c and 2 c + 1, columns g and g + 8
        int stage = 0;
        while (now.tile < tiles) {
            const int kb = now.kb, tile = now.tile;
            const uint8_t *wsc_a = reinterpret_cast<const uint8_t *>(wscale + (16 * tile + g) * kt), *wsc_b = wsc_a + 32 * kt;
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
            float acc[2][4] = {};                           // two chains, to wait half as long
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint4 b[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (have) {
                    b[0] = reinterpret_cast<const uint4 *>(xg + kb * 128 + 64 * h)[0];
                    b[1] = reinterpret_cast<const uint4 *>(xg + kb * 128 + 64 * h)[1];
                }
                const uint4 wa = ring[(stage * 4 + h) * 32 * kWarps + threadIdx.x], wb = ring[(stage * 4 + 2 + h) * 32 * kWarps + threadIdx.x];
                const uint32_t bw[8] = {b[0].x, b[0].y, b[0].z, b[0].w, b[1].x, b[1].y, b[1].z, b[1].w};
                const uint32_t ca[4] = {wa.x, wa.y, wa.z, wa.w}, cb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t a0, a1, a2, a3;
                    to_half(ca[j], a0, a2);
                    to_half(cb[j], a1, a3);
                    mma_f16(acc[j & 1], a0, a1, a2, a3, bw[2 * j], bw[2 * j + 1]);
                }
            }
            const float s_a = __uint_as_float(uint32_t(wsc_a[kb]) << 23), s_b = __uint_as_float(uint32_t(wsc_b[kb]) << 23);
            const float s0 = sc0[kb], s1 = sc1[kb];
            total[0] += (acc[0][0] + acc[1][0]) * s_a * s0, total[1] += (acc[0][1] + acc[1][1]) * s_a * s1;
            total[2] += (acc[0][2] + acc[1][2]) * s_b * s0, total[3] += (acc[0][3] + acc[1][3]) * s_b * s1;
            fetch(ahead, stage);                            // the pieces have been used: refill their place
            advance(ahead);
            stage = stage + 1 == kAhead ? 0 : stage + 1;
            advance(now);
            if (now.tile != tile) {                         // this warp's share of the tile is done
                float *to = mine + tile * 16 * kRowsPerPass;
                to[0] = total[0], to[16] = total[1], to[8] = total[2], to[24] = total[3];
                total[0] = total[1] = total[2] = total[3] = 0.0f;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tiles * 16 * kRowsPerPass; i += 32 * kWarps) {
            float v = sums[i];
#pragma unroll
            for (int w = 1; w < kWarps; w++) v += sums[w * sums_warp + i];
            const int r = r0 + ((i >> 4) & (kRowsPerPass - 1)), col = n0 + 16 * (i / (16 * kRowsPerPass)) + (i & 15);
            if (r < hi && col < p.N) {
                if (p.out_bf16) static_cast<__nv_bfloat16 *>(p.out)[int64_t(r) * p.N + col] = __float2bfloat16_rn(v);
                else static_cast<float *>(p.out)[int64_t(r) * p.N + col] = v;
            }
        }
        __syncthreads();                                    // the next pass overwrites x and the sums
    }
}

constexpr int kRingBytes = kAhead * 4 * 32 * kWarps * 16, kMaxX = 72 * 1024;
constexpr int kMaxSmem = 200 * 1024;

size_t x_bytes(int64_t rows, int64_t K)
{
    const size_t n = rows < kRowsPerPass ? rows : kRowsPerPass, kb = (K + 127) / 128;
    return n * ((kb * 128 + 8) * 2 + kb * 4);
}
size_t tile_bytes(int64_t K) { return 16 * ((K + 511) / 512) * 4 + kWarps * 16 * kRowsPerPass * 4; }

template <typename T, bool VEC>
int launch(const void *x, const SkinnyArgs &p, cudaStream_t st)
{
    static bool attr_set[64] = {};
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    {
        std::lock_guard<std::mutex> lk(state_mutex());
        if (!attr_set[dev]) {
            LS_CUDA(cudaFuncSetAttribute(fp8_skinny_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
            attr_set[dev] = true;
        }
    }
    const dim3 grid(unsigned((p.N + 16 * p.tiles - 1) / (16 * p.tiles)), unsigned(p.offsets ? std::min(p.groups, p.rows) : 1), 1);
    return launch_dependent(fp8_skinny_kernel<T, VEC>, grid, 32 * kWarps, kRingBytes + x_bytes(p.rows, p.K) + p.tiles * tile_bytes(p.K), st,
                            static_cast<const T *>(x), p);
}

}  // namespace

// Whether this form is the faster one.  It wins while latency counts: one row takes 6.5 us at 4096 x
// 4096 (quantizer and tcgen05 product 11.0), 16.1 at 8192 x 8192 (18.3), 55 at 16384 x 16384 (48.6);
// eight rows 6.5 at K = 2048, N = 4096 (8.8) and 16.3 at N = 16384 (11.6): the more rows, the more of
// a CTA's time goes into quantizing x, which every CTA does.  Per expert: eight of 1024 x 1024 4.5
// us (6.9), four of 4096 x 1024 8.9 (7.7).
bool fp8_skinny_fits(int64_t rows, int64_t N, int64_t K, int64_t groups)
{
    if (x_bytes(rows, K) > kMaxX) return false;
    if (groups == 0) return rows <= kRowsPerPass && rows * N * K <= int64_t(128) << 20;
    return rows <= 4 * kRowsPerPass && std::min(groups, rows) * N * K <= int64_t(12) << 20;
}

// y = q(x) w^T for a few rows; arguments as ls_fp8_linear, checked by it.
int fp8_skinny_linear(const void *x, int dtype, int64_t rows, int64_t K, const uint8_t *codes, int64_t ld, const uint8_t *sf, int64_t N,
                      void *y, int out_dtype, const int *offsets, int64_t groups, int zero_tail, cudaStream_t st)
{
    // tiles per CTA: what leaves as many CTAs per SM as x leaves room for, three at most
    const int64_t units = (N + 15) / 16 * (offsets ? std::min(groups, rows) : 1);
    const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(3, 220 * 1024 / (kRingBytes + x_bytes(rows, K) + tile_bytes(K))));
    int64_t tiles = std::min<int64_t>({units / (per_sm * sm_count()) + 1, kMaxTiles, (N + 15) / 16});
    while (tiles > 1 && (kRingBytes + x_bytes(rows, K) + tiles * tile_bytes(K)) * per_sm > 224 * 1024) tiles--;
    const SkinnyArgs p{int(rows), int(K), int(N), codes, ld, sf, y, out_dtype == LS_BF16, offsets, int(groups), zero_tail, int(tiles)};
    const bool vec = aligned16(x) && K * (dtype == LS_BF16 ? 2 : 4) % 16 == 0;
    if (dtype == LS_BF16) return vec ? launch<__nv_bfloat16, true>(x, p, st) : launch<__nv_bfloat16, false>(x, p, st);
    return vec ? launch<float, true>(x, p, st) : launch<float, false>(x, p, st);
}

}  // namespace ls
