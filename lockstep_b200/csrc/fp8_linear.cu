// The FP8 linear layer as one call per direction: the quantizers and products of fp8.cu and
// fp8_gemm.cu in order on one stream, their operands in two buffers of the caller (`work`, free
// again when the call's kernels are done, and `saved`, kept for the backward pass).  A serving call
// is a few microseconds of device time; separate calls with a buffer for every operand cost 25 us
// of host time per linear, this form about half.
#include <atomic>

#include "fp8.cuh"

namespace ls {
namespace {

std::atomic<int> g_no_skinny{0};

struct Shape {
    int64_t rows, N, K;
    const int *offsets;
    int64_t groups;                // 1 without offsets
    int64_t matrices() const { return groups; }
    int64_t slot_rows() const { return offsets ? 128 * fp8_slots(rows, groups) : rows; }
};
int64_t pitch(int64_t n) { return (n + 127) / 128 * 128; }     // whole lines: see _pitch in fp8.py
int64_t sf_bytes(int64_t rows, int64_t K) { return ls_fp8_sf_bytes(rows, K); }

// Hands out 128-byte aligned pieces of a buffer; with a null buffer it only counts.
struct Carver {
    uint8_t *base;
    int64_t at = 0;
    uint8_t *take(int64_t bytes)
    {
        uint8_t *p = base ? base + at : nullptr;
        at += (bytes + 127) / 128 * 128;
        return p;
    }
};
enum { kGradX = 1, kGradW = 2 };

struct RowOperand { uint8_t *codes, *sf; };
RowOperand take_rows(Carver &c, const Shape &s, int64_t width)
{
    RowOperand r;
    r.codes = c.take(s.rows * pitch(width)), r.sf = c.take(sf_bytes(s.slot_rows(), width));
    return r;
}
RowOperand take_cols(Carver &c, const Shape &s, int64_t width)
{
    RowOperand r;
    r.codes = c.take(s.slot_rows() * pitch(width)), r.sf = c.take(sf_bytes(width, s.slot_rows()));
    return r;
}

// what the backward pass needs: x column-wise for gw, the weight's codes and transposed scales for gx
struct Saved { RowOperand x, w; };
Saved take_saved(Carver &c, const Shape &s, int grads)
{
    Saved v{};
    if (grads & kGradW) v.x = take_cols(c, s, s.K);
    if (grads & kGradX) v.w.codes = c.take(s.matrices() * s.N * pitch(s.K)), v.w.sf = c.take(s.matrices() * sf_bytes(s.K, s.N));
    return v;
}
struct Forward { RowOperand x; uint8_t *w_codes, *w_sf; };
Forward take_forward(Carver &c, const Shape &s, int grads)
{
    Forward f;
    f.x = take_rows(c, s, s.K);
    f.w_sf = c.take(s.matrices() * sf_bytes(s.N, s.K));
    f.w_codes = grads & kGradX ? nullptr : c.take(s.matrices() * s.N * pitch(s.K));
    return f;
}
struct Backward { RowOperand g, gt; };
Backward take_backward(Carver &c, const Shape &s, int grads)
{
    Backward b{};
    if (grads & kGradX) b.g = take_rows(c, s, s.N);
    if (grads & kGradW) b.gt = take_cols(c, s, s.N);
    return b;
}

// A few rows (per group) go through a kernel that needs no buffer.
bool few_rows(const Shape &s)
{
    return s.K > 0 && fp8_skinny_fits(s.rows, s.N, s.K, s.offsets ? s.groups : 0) && !g_no_skinny.load(std::memory_order_relaxed);
}

int check_shape(const Shape &s, int grads)
{
    if (int rc = check_device()) return rc;
    if (s.rows < 0 || s.N < 0 || s.K < 0 || s.rows > (1 << 30) || s.N > (1 << 30) || s.K > (1 << 30)) return fail(LS_EINVAL, "dimension out of range");
    if (s.groups < 1 || s.groups > kFp8MaxGroups) return fail(LS_EINVAL, "groups=%lld must be 1..%d", (long long)s.groups, kFp8MaxGroups);
    if (s.groups > 1 && !s.offsets) return fail(LS_EINVAL, "several groups need offsets");
    if (grads & ~(kGradX | kGradW)) return fail(LS_EINVAL, "unknown gradient flags %d", grads);
    return LS_OK;
}
int check_buffer(const void *p, const char *what)
{
    if (!p) return fail(LS_EINVAL, "%s is null", what);
    return aligned16(p) ? LS_OK : fail(LS_EALIGN, "%s must be 16-byte aligned", what);
}

int product(int form, const uint8_t *a, int64_t lda, const uint8_t *b, int64_t ldb, const uint8_t *sfa, const uint8_t *sfb, void *c,
            int dtype, int64_t M, int64_t N, int64_t K, const Shape &s, int zero_tail, void *stream)
{
    if (s.offsets)
        return ls_fp8_gemm_grouped(form, a, lda, b, ldb, sfa, sfb, c, dtype, M, N, K, s.offsets, s.groups, zero_tail, stream);
    return ls_fp8_gemm(form, a, lda, b, ldb, sfa, sfb, c, dtype, M, N, K, stream);
}

}  // namespace
}  // namespace ls

using namespace ls;

extern "C" int64_t ls_fp8_linear_bytes(int what, int64_t rows, int64_t N, int64_t K, int64_t groups, int grads)
{
    static const int some_offsets = 0;                      // only whether there are offsets counts here
    const Shape s{rows, N, K, groups > 0 ? &some_offsets : nullptr, groups > 0 ? groups : 1};
    Carver c{nullptr};
    switch (what) {
    case LS_FP8_SERVE:
        if (!few_rows(s)) take_rows(c, s, K);
        break;
    case LS_FP8_FORWARD: take_forward(c, s, grads); break;
    case LS_FP8_SAVED: take_saved(c, s, grads); break;
    case LS_FP8_BACKWARD: take_backward(c, s, grads); break;
    default: return -1;
    }
    return c.at;
}

extern "C" int ls_fp8_linear(const void *x, int dtype, int64_t rows, int64_t K, const uint8_t *w_codes, int64_t ldw,
                             const uint8_t *w_sf, int64_t N, void *y, int out_dtype, const int *offsets, int64_t groups,
                             int zero_tail, void *work, void *stream)
{
    const Shape s{rows, N, K, offsets, groups};
    if (int rc = check_shape(s, 0)) return rc;
    if (rows == 0 || N == 0) return LS_OK;
    if (dtype != LS_F32 && dtype != LS_BF16) return fail(LS_EINVAL, "unsupported input dtype %d", dtype);
    if (out_dtype != LS_F32 && out_dtype != LS_BF16) return fail(LS_EINVAL, "unsupported output dtype %d", out_dtype);
    if (int rc = check_buffer(y, "y")) return rc;
    // A few rows (per group): one launch that reads the weights once and quantizes x on the fly.
    if (few_rows(s)) {
        if (!x) return fail(LS_EINVAL, "x is null");
        if (int rc = check_buffer(w_codes, "w_codes")) return rc;
        if (int rc = check_buffer(w_sf, "w_sf")) return rc;
        if (ldw < K || ldw % 16) return fail(LS_EINVAL, "row pitch %lld of the weight's codes", (long long)ldw);
        return fp8_skinny_linear(x, dtype, rows, K, w_codes, ldw, w_sf, N, y, out_dtype, offsets, groups, zero_tail, static_cast<cudaStream_t>(stream));
    }
    if (int rc = check_buffer(work, "work")) return rc;
    Carver c{static_cast<uint8_t *>(work)};
    const RowOperand q = take_rows(c, s, K);
    if (int rc = ls_quantize_fp8(x, dtype, rows, K, offsets, groups, q.codes, pitch(K), nullptr, q.sf, stream)) return rc;
    return product(0, q.codes, pitch(K), w_codes, ldw, q.sf, w_sf, y, out_dtype, rows, N, K, s, zero_tail, stream);
}

extern "C" int ls_fp8_linear_forward(const void *x, int dtype, const void *w, int w_dtype, int64_t rows, int64_t N, int64_t K,
                                     const int *offsets, int64_t groups, int grads, void *y, void *saved, void *work, void *stream)
{
    const Shape s{rows, N, K, offsets, groups};
    if (int rc = check_shape(s, grads)) return rc;
    if (int rc = check_buffer(work, "work")) return rc;
    if (grads)
        if (int rc = check_buffer(saved, "saved")) return rc;
    Carver cw{static_cast<uint8_t *>(work)}, cs{static_cast<uint8_t *>(saved)};
    const Forward f = take_forward(cw, s, grads);
    const Saved keep = take_saved(cs, s, grads);
    uint8_t *wc = grads & kGradX ? keep.w.codes : f.w_codes;
    if (int rc = ls_quantize_fp8_weight(w, w_dtype, s.matrices(), N, K, wc, pitch(K), nullptr, f.w_sf, keep.w.sf, stream)) return rc;
    int rc = grads & kGradW ? ls_quantize_fp8_both(x, dtype, rows, K, offsets, groups, f.x.codes, f.x.sf, keep.x.codes, keep.x.sf, pitch(K), stream)
                            : ls_quantize_fp8(x, dtype, rows, K, offsets, groups, f.x.codes, pitch(K), nullptr, f.x.sf, stream);
    if (rc) return rc;
    return product(0, f.x.codes, pitch(K), wc, pitch(K), f.x.sf, f.w_sf, y, dtype, rows, N, K, s, 1, stream);
}

extern "C" int ls_fp8_linear_backward(const void *gy, int dtype, int64_t rows, int64_t N, int64_t K, const int *offsets, int64_t groups,
                                      int grads, const void *saved, void *gx, int gx_dtype, void *gw, int gw_dtype, void *work,
                                      void *stream)
{
    const Shape s{rows, N, K, offsets, groups};
    if (int rc = check_shape(s, grads)) return rc;
    if (!grads) return LS_OK;
    if (int rc = check_buffer(work, "work")) return rc;
    if (int rc = check_buffer(saved, "saved")) return rc;
    Carver cw{static_cast<uint8_t *>(work)}, cs{static_cast<uint8_t *>(const_cast<void *>(saved))};
    const Backward b = take_backward(cw, s, grads);
    const Saved keep = take_saved(cs, s, grads);
    int rc = grads & kGradW ? ls_quantize_fp8_both(gy, dtype, rows, N, offsets, groups, b.g.codes, b.g.sf, b.gt.codes, b.gt.sf, pitch(N), stream)
                            : ls_quantize_fp8(gy, dtype, rows, N, offsets, groups, b.g.codes, pitch(N), nullptr, b.g.sf, stream);
    if (rc) return rc;
    if (grads & kGradX) {
        rc = product(1, b.g.codes, pitch(N), keep.w.codes, pitch(K), b.g.sf, keep.w.sf, gx, gx_dtype, rows, K, N, s, 1, stream);
        if (rc) return rc;
    }
    if (grads & kGradW)
        return product(2, b.gt.codes, pitch(N), keep.x.codes, pitch(K), b.gt.sf, keep.x.sf, gw, gw_dtype, N, K, rows, s, 0, stream);
    return LS_OK;
}

extern "C" int ls_fp8_linear_set_skinny(int on)
{
    g_no_skinny.store(on ? 0 : 1, std::memory_order_relaxed);
    return LS_OK;
}
