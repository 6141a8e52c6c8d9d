// Host side of the FP8 products: tensor maps, the choice of kernel, the entry points.  The kernels are in
// fp8_gemm.cuh, compiled once per form.
#include <algorithm>
#include <atomic>

#include "fp8_gemm.cuh"

namespace ls {
namespace {

struct MapSpec {
    const void *base;
    int64_t inner, rows, depth;    // elements, rows, matrices
    int64_t pitch;                 // bytes between rows
    int box_inner, box_rows;
    MapType type;
    bool operator==(const MapSpec &o) const
    {
        return base == o.base && inner == o.inner && rows == o.rows && depth == o.depth && pitch == o.pitch &&
               box_inner == o.box_inner && box_rows == o.box_rows && type == o.type;
    }
};

// Encoded tensor maps are pure functions of their specification: a direct-mapped cache per host
// thread saves the driver's encoding for operands that come back (weights, recycled buffers).
int make_map(CUtensorMap *m, const MapSpec &k)
{
    struct Slot { MapSpec key; CUtensorMap map; bool used; };
    static thread_local Slot slots[256] = {};
    uint64_t h = (reinterpret_cast<uintptr_t>(k.base) >> 4) ^ uint64_t(k.rows) * 0x9E3779B97F4A7C15ull ^
                 uint64_t(k.inner) * 0xC2B2AE3D27D4EB4Full ^ uint64_t(k.depth * 131 + k.pitch * 31 + k.box_rows * 7 + k.type);
    h ^= h >> 29;
    Slot &slot = slots[h % 256];
    if (!slot.used || !(slot.key == k)) {
        if (int rc = encode_map_3d(&slot.map, k.base, k.inner, k.rows, k.depth, k.pitch, k.box_inner, k.box_rows, k.type)) {
            slot.used = false;
            return rc;
        }
        slot.key = k, slot.used = true;
    }
    *m = slot.map;
    return LS_OK;
}

std::atomic<int> g_variant{0};          // 0 = choose by size; else see ls_fp8_gemm_set_variant

int fp8_gemm(int form, const uint8_t *a, int64_t lda, const uint8_t *b, int64_t ldb, const uint8_t *sfa, const uint8_t *sfb,
             void *c, int out_dtype, int64_t M, int64_t N, int64_t K, const int *offsets, int64_t groups, int zero_tail,
             void *stream)
{
    if (int rc = check_device()) return rc;
    if (form < NT || form > TN) return fail(LS_EINVAL, "form must be 0 (NT), 1 (NN) or 2 (TN)");
    if (out_dtype != LS_F32 && out_dtype != LS_BF16) return fail(LS_EINVAL, "unsupported output dtype %d", out_dtype);
    if (M < 0 || N < 0 || K < 0 || M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) return fail(LS_EINVAL, "dimension out of range");
    if (groups < 1 || groups > kFp8MaxGroups) return fail(LS_EINVAL, "groups=%lld must be 1..%d", (long long)groups, kFp8MaxGroups);
    if (groups > 1 && !offsets) return fail(LS_EINVAL, "several groups need offsets");
    if (M == 0 || N == 0) return LS_OK;
    if (!c) return fail(LS_EINVAL, "null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (K == 0) {                                           // empty sums
        if (offsets && form != TN && !zero_tail) return fail(LS_EINVAL, "K must be positive where rows of no group are kept");
        LS_CUDA(cudaMemsetAsync(c, 0, size_t(form == TN ? groups : 1) * M * N * (out_dtype == LS_BF16 ? 2 : 4), st));
        return LS_OK;
    }
    if (!a || !b || !sfa || !sfb) return fail(LS_EINVAL, "null pointer");
    if (!aligned16(a) || !aligned16(b) || !aligned16(sfa) || !aligned16(sfb) || !aligned16(c))
        return fail(LS_EALIGN, "operands, scale buffers and outputs must be 16-byte aligned");
    const int64_t a_inner = form == TN ? M : K, b_inner = form == NT ? K : N;
    if (lda < a_inner || ldb < b_inner || lda % 16 || ldb % 16)
        return fail(LS_EINVAL, "row pitches must be multiples of 16 and cover a row (lda=%lld, ldb=%lld)", (long long)lda, (long long)ldb);
    int *err = error_word();
    if (!err) return fail(LS_ECUDA, "the device error word is not available");

    // Rows (M) or K that the operands hold: with groups the TN operands are in slot order.
    const int64_t slots = offsets ? fp8_slots(form == TN ? K : M, groups) : ((form == TN ? K : M) + 127) / 128;
    const int64_t a_rows = form == TN ? (offsets ? slots * 128 : K) : M;
    const int64_t b_rows = form == NT ? N : form == NN ? K : a_rows;
    const int64_t depth = form == TN ? 1 : groups;
    const int64_t kblocks = form == TN ? slots : (K + 127) / 128;
    Fp8Params p{};
    p.c = c, p.M = int(M), p.N = int(N), p.K = int(K);
    p.out_bf16 = out_dtype == LS_BF16;
    p.offsets = offsets, p.groups = int(groups), p.zero_tail = zero_tail;
    p.sfa_kt = p.sfb_kt = int((kblocks + 3) / 4);
    p.sfb_rt = int((N + 127) / 128);
    p.err = err;

    // Which kernel: the one with the smallest product of rounds over the SMs and cycles per block of K.
    // A pair's 256 x 256 tile takes the tensor cores' 512 cycles.  The tiles of single CTAs are bound by
    // shared memory, which is written and read once per staged byte at 128 bytes per cycle: 128 x 256
    // 768, 128 x 128 512, 128 x 64 (K-major B only) 384.  Among equals the smaller tile, whose epilogue is
    // shorter (2048 x 1024 over 4999 rows: 12.6 us against 17.0 of the pair's).  A ragged group ends in
    // half a tile on average.  With few rows per group the second CTA of a pair idles: no pairs there.
    const int variant = g_variant.load(std::memory_order_relaxed), sms = sm_count();
    p.splits = 1;
    const bool by_rows = form != TN && offsets;
    auto tiles = [&](int64_t rows, int64_t cols, int64_t part) {       // part / 2 of a tile more per group
        const int64_t m = by_rows ? M / rows + (part * groups + 1) / 2 : (M + rows - 1) / rows;
        return m * ((N + cols - 1) / cols) * (form == TN ? groups : 1);
    };
    // K split: the CTAs of a cluster take parts of a dense tile's K loop, while all clusters run at once (74 of
    // two, 45 of three, 33 of four CTAs: the SMs of a cluster are neighbours); their sums meet in shared
    // memory, which takes about 3500 + 400 cycles per part with 64 columns and 3000 + 1500 with 128.  A
    // split is taken where it promises a sixth or more.  16 rows, 16384 -> 2048: 27.6 -> 12.8 us; weight
    // gradient of 512 x 512 over 16384 rows: 30.5 -> 14.9; 16 rows, 4096 -> 4096: 9.4 -> 8.9.
    const int64_t nkb = (K + kBlock - 1) / kBlock;
    bool pair = variant == 2;
    int bn = variant == 4 || variant == 2 ? 256 : variant == 3 && form == NT ? 64 : 128;
    if (variant == 5) p.splits = int(std::min<int64_t>(kMaxSplits, nkb));
    if (variant == 0) {
        int64_t best = -1;
        auto consider = [&](bool p2, int cols, int64_t cycles, int splits) {
            const int64_t workers = p2 ? sms / 2 : sms, n = tiles(p2 ? 256 : 128, cols, 1) * splits;
            if (splits > 1 && (offsets || n > int64_t(splits) * fp8_cluster_room(splits) || nkb < splits)) return;
            int64_t cost = cycles * ((nkb + splits - 1) / splits);
            if (splits == 1) cost *= (n + workers - 1) / workers;
            else cost = (cost + (cols == 64 ? 3500 + 400 * splits : 3000 + 1500 * splits)) * 7 / 6;
            if (best < 0 || cost < best) best = cost, pair = p2, bn = cols, p.splits = splits;
        };
        for (int splits = 1; splits <= kMaxSplits; splits++) {
            if (form == NT) consider(false, 64, 384, splits);
            consider(false, 128, 512, splits);
        }
        consider(false, 256, 768, 1);
        if (M > (by_rows ? 128 * groups : 128)) consider(true, 256, 512, 1);
    }
    if (offsets || pair || bn == 256 || tiles(128, bn, 2) > (1 << 28)) p.splits = 1;
    if (p.splits > 1) p.splits = int((nkb + (nkb + p.splits - 1) / p.splits - 1) / ((nkb + p.splits - 1) / p.splits));    // no empty part
    const int64_t items = tiles(pair ? 256 : 128, bn, 2);
    if (items > 0x7FFFFFFFll) return fail(LS_EINVAL, "too many output tiles");
    const int64_t a_tiles = fp8_sf_tiles(form == TN ? M : slots * 128, kblocks);
    const int64_t b_tiles = fp8_sf_tiles(N, kblocks) * depth;
    // Filling what lies outside a tensor is slow (a tile whose 128 columns are partly outside takes almost
    // twice as long), so along M and N the maps reach into the rows' padding: those sums are not stored.
    // Along K the extent is exact: behind it the operands read as zeros.
    const int64_t a_extent = form == TN ? std::min(lda, (M + 127) / 128 * 128) : K;
    const int64_t b_extent = form == NT ? K : std::min(ldb, (N + 127) / 128 * 128);
    CUtensorMap ta, tb, tsa, tsb;
    // With fewer rows than a tile the box of A is no taller than they need: rows outside the tensor
    // cost more than rows inside it (one row, 4096 x 4096: 14.7 us with 128-row boxes).  The rest of
    // the stage keeps what shared memory held; an output row depends on its own row of A only.
    int a_box = 128;
    if (form != TN)
        for (a_box = 16; a_box < M && a_box < 128; a_box *= 2) {}
    p.a_bytes = a_box * kBlock;
    if (int rc = make_map(&ta, {a, a_extent, a_rows, 1, lda, 128, a_box, kMapBytes})) return rc;
    if (int rc = make_map(&tb, {b, b_extent, b_rows, depth, ldb, 128, form == NT && bn == 64 ? 64 : 128, kMapBytes})) return rc;
    if (int rc = make_map(&tsa, {sfa, 128, a_tiles, 1, 512, 128, 1, kMapWords})) return rc;
    if (int rc = make_map(&tsb, {sfb, 128, b_tiles, 1, 512, 128, 1, kMapWords})) return rc;
    // C, stored in boxes of 16 rows x 128 bytes; rows that do not start on 16-byte boundaries have no map
    CUtensorMap tc = ta;
    const int64_t es = p.out_bf16 ? 2 : 4;
    if (N * es % 16 == 0)
        if (int rc = make_map(&tc, {c, N, M, form == TN ? groups : 1, N * es, int(128 / es), 16, p.out_bf16 ? kMapBf16 : kMapF32})) return rc;
    const bool many = out_dtype == LS_F32 && kblocks > kSegment;
    const Fp8Maps maps{ta, tb, tsa, tsb, tc};
    const auto run = form == NT ? fp8_launch_nt : form == NN ? fp8_launch_nn : fp8_launch_tn;
    return run(pair, bn, many, maps, p, items, st);
}

}  // namespace
}  // namespace ls

using namespace ls;

extern "C" int ls_fp8_gemm(int form, const uint8_t *a, int64_t lda, const uint8_t *b, int64_t ldb, const uint8_t *sfa,
                           const uint8_t *sfb, void *c, int out_dtype, int64_t M, int64_t N, int64_t K, void *stream)
{
    return fp8_gemm(form, a, lda, b, ldb, sfa, sfb, c, out_dtype, M, N, K, nullptr, 1, 0, stream);
}

extern "C" int ls_fp8_gemm_grouped(int form, const uint8_t *a, int64_t lda, const uint8_t *b, int64_t ldb, const uint8_t *sfa,
                                   const uint8_t *sfb, void *c, int out_dtype, int64_t M, int64_t N, int64_t K,
                                   const int *offsets, int64_t groups, int zero_tail, void *stream)
{
    if (!offsets) return fail(LS_EINVAL, "null pointer");
    return fp8_gemm(form, a, lda, b, ldb, sfa, sfb, c, out_dtype, M, N, K, offsets, groups, zero_tail, stream);
}

extern "C" int ls_fp8_gemm_set_variant(int variant)
{
    if (variant < 0 || variant > 5) return fail(LS_EINVAL, "variant must be 0..5");
    g_variant.store(variant, std::memory_order_relaxed);
    return LS_OK;
}
