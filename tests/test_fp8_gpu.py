"""FP8 block-128 quantizers and products against the 64-bit oracle.

Tolerances.  Codes and scales are exact.  Every product of two E4M3 values with power-of-two scales is
exact in fp32; a sum of K of them in the tensor core's fp32 accumulator loses at most one unit in the
last place (2^-23) of the partial sums' bound S = sum |a||b| per addition, K 2^-23 S in all; rounding
the result to the output type loses half a step (2^-8 bf16, 2^-24 fp32) of the value."""

import numpy as np
import pytest
import torch

from oracle import fp8_ref as ref

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _data(*shape, seed=0, dtype=torch.bfloat16, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, device="cuda", generator=g)
    x = x * torch.exp(spread * torch.randn(*shape[:-1], 1, device="cuda", generator=g))
    return x.to(dtype)


def _close(got, a, b, what):
    """got against a @ b (doubles) within the derived bound."""
    want, bound = a @ b, a.abs() @ b.abs()
    tol = HALF_STEP[got.dtype] * want.abs() + (a.shape[1] + 1) * 2.0 ** -23 * bound + 1e-300
    off = ((got.double() - want).abs() / tol).max().item() if got.numel() else 0.0
    assert off <= 1.0, f"{what}: {off:.2f} times the bound"


def _status():
    from lockstep_b200 import mxfp4_gemm
    mxfp4_gemm.gemm_status()


# ---------------------------------------------------------------- quantizers
QSHAPES = [(1, 128), (1, 1), (3, 100), (7, 16), (128, 128), (129, 512), (200, 1000), (333, 1111), (64, 2048), (257, 640)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", QSHAPES)
def test_row_quantizer_exact(rows, K, dtype):
    from lockstep_b200 import fp8
    x = _data(rows, K, seed=rows + K, dtype=dtype, spread=6.0)
    codes, scale = fp8.quantize_fp8(x)
    q, s = ref.quantize(x, (1, 128))
    assert codes.shape == x.shape and codes.dtype == torch.float8_e4m3fn
    assert torch.equal(codes.double(), q)
    assert torch.equal(scale.double().repeat_interleave(128, 1)[:, :K], s)
    assert torch.equal(fp8.dequantize_fp8(codes, scale).double(), q * s)
    packed, sf = fp8.quantize_fp8_packed(x)
    assert torch.equal(packed.view(torch.uint8), codes.view(torch.uint8))
    want = fp8.scales_to_sf(scale)
    used = fp8.scales_to_sf(torch.ones_like(scale)) > 0
    assert torch.equal(sf[used], want[used])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", QSHAPES)
def test_both_forms_exact(rows, K, dtype):
    from lockstep_b200 import fp8
    x = _data(rows, K, seed=rows * 3 + K, dtype=dtype, spread=4.0)
    codes, sf, codes_t, sf_t = fp8.quantize_fp8_both(x)
    rc, rsf = fp8.quantize_fp8_packed(x)
    assert torch.equal(codes.view(torch.uint8), rc.view(torch.uint8))
    used = fp8.scales_to_sf(torch.ones(rows, -(-K // 128), device="cuda")) > 0
    assert torch.equal(sf[used], rsf[used])
    q, s = ref.quantize(x, (128, 1))
    assert torch.equal(codes_t.double(), q)
    used = fp8.scales_to_sf(torch.ones(K, -(-rows // 128), device="cuda")) > 0
    assert torch.equal(sf_t[used], fp8.scales_to_sf(s[::128].t().float())[used])
    only = fp8.quantize_fp8_both(x, rows_too=False)
    assert only[0] is None and only[1] is None and torch.equal(only[2].view(torch.uint8), codes_t.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(128, 128), (1, 1), (130, 1000), (3, 200, 300), (2, 256, 512)])
def test_weight_quantizer_exact(shape, dtype):
    from lockstep_b200 import fp8
    w = _data(*shape, seed=sum(shape), dtype=dtype, spread=2.0)
    codes, sf, sf_t, scale = fp8.quantize_fp8_weight(w, want_scale=True)
    spans = (1,) * (len(shape) - 2) + (128, 128)
    q, s = ref.quantize(w, spans)
    N, K = shape[-2:]
    assert torch.equal(codes.double(), q)
    assert torch.equal(scale.double(), s[..., ::128, ::128])
    used = fp8.scales_to_sf(torch.ones_like(scale), N) > 0
    assert torch.equal(sf.view(used.shape)[used], fp8.scales_to_sf(scale, N)[used])
    st = scale.transpose(-1, -2).contiguous()
    used = fp8.scales_to_sf(torch.ones_like(st), K) > 0
    assert torch.equal(sf_t.view(used.shape)[used], fp8.scales_to_sf(st, K)[used])
    assert torch.equal(fp8.dequantize_fp8(codes, scale).double(), q * s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_special_values(dtype):
    from lockstep_b200 import fp8
    x = torch.zeros(9, 384, device="cuda")
    x[1, 5] = float("inf")
    x[2, 130], x[2, 131] = float("nan"), 3.0
    x[3, :] = 448.0                                            # scale exactly 1
    x[4, 7] = 450.0                                            # above 448 in both types: scale 2
    x[5, 0], x[5, 1] = -0.0, 1e-30
    x[6, 300] = torch.finfo(torch.float32).max if dtype == torch.float32 else torch.finfo(torch.bfloat16).max
    x[7, 200] = 1e-39                                          # below the smallest scale's reach: scale 2^-126
    x[8] = torch.linspace(-448, 448, 384, device="cuda")       # every binade of the format, ties among them
    x = x.to(dtype)
    q, s = ref.quantize(x, (1, 128))
    codes, scale = fp8.quantize_fp8(x)
    assert torch.equal(codes.double().nan_to_num(999.0), q.nan_to_num(999.0))
    assert torch.equal(scale.double().repeat_interleave(128, 1), s)
    c, _, ct, _ = fp8.quantize_fp8_both(x)
    assert torch.equal(c.double().nan_to_num(999.0), q.nan_to_num(999.0))
    assert torch.equal(ct.double().nan_to_num(999.0), ref.quantize(x, (128, 1))[0].nan_to_num(999.0))
    wc, _, _ = fp8.quantize_fp8_weight(x)
    assert torch.equal(wc.double().nan_to_num(999.0), ref.quantize(x, (128, 128))[0].nan_to_num(999.0))


# ---------------------------------------------------------------- products
def _variant(v):
    from lockstep_b200._lib import check, lib
    check(lib().ls_fp8_gemm_set_variant(v))


@pytest.fixture(params=[0, 1, 2, 3, 4, 5])
def variant(request):
    _variant(request.param)
    yield request.param
    _variant(0)


GSHAPES = [(128, 128, 128), (1, 128, 128), (128, 128, 512), (130, 136, 200), (17, 8, 1), (256, 256, 640), (300, 513, 1000),
           (1, 1111, 4096), (513, 257, 129), (700, 384, 1536)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", GSHAPES)
def test_forward_product(M, N, K, out, variant):
    from lockstep_b200 import fp8
    x, w = _data(M, K, seed=1), _data(N, K, seed=2, dtype=torch.float32)
    xc, xsf = fp8.quantize_fp8_packed(x)
    wc, wsf, _ = fp8.quantize_fp8_weight(w)
    c = fp8.fp8_gemm(xc, wc, xsf, wsf, out)
    _status()
    assert c.shape == (M, N) and c.dtype == out
    _close(c, *ref.forward(x, w), f"NT {M}x{N}x{K}")


@pytest.mark.parametrize("M,N,K", GSHAPES)
def test_input_gradient_product(M, N, K, variant):
    from lockstep_b200 import fp8
    gy, w = _data(M, K, seed=3), _data(K, N, seed=4)
    gc, gsf = fp8.quantize_fp8_packed(gy)
    wc, _, wsf_t = fp8.quantize_fp8_weight(w)
    c = fp8.fp8_gemm_nn(gc, wc, gsf, wsf_t, torch.float32)
    _status()
    _close(c, *ref.grad_input(gy, w), f"NN {M}x{N}x{K}")


@pytest.mark.parametrize("M,N,K", GSHAPES)
def test_weight_gradient_product(M, N, K, variant):
    from lockstep_b200 import fp8
    gy, x = _data(K, M, seed=5), _data(K, N, seed=6)
    _, _, gct, gsf_t = fp8.quantize_fp8_both(gy)
    _, _, xct, xsf_t = fp8.quantize_fp8_both(x)
    c = fp8.fp8_gemm_tn(gct, xct, gsf_t, xsf_t)
    _status()
    assert c.dtype == torch.float32
    _close(c, *ref.grad_weight(gy, x), f"TN {M}x{N}x{K}")


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(5000, 2040, 300), (4600, 2041, 260), (260, 9000, 5000)])
def test_many_tiles_per_cta(M, N, K, out, variant):
    # several tiles, and for fp32 several accumulation chains, pass through every accumulator of a CTA
    from lockstep_b200 import fp8
    x, w = _data(M, K, seed=1), _data(N, K, seed=2)
    xc, xsf = fp8.quantize_fp8_packed(x)
    wc, wsf, _ = fp8.quantize_fp8_weight(w)
    _close(fp8.fp8_gemm(xc, wc, xsf, wsf, out), *ref.forward(x, w), f"NT {M}x{N}x{K}")
    w = _data(K, N, seed=3)
    wc, _, wsf_t = fp8.quantize_fp8_weight(w)
    _close(fp8.fp8_gemm_nn(xc, wc, xsf, wsf_t, out), *ref.grad_input(x, w), f"NN {M}x{N}x{K}")
    gy, v = _data(K, M, seed=4), _data(K, N, seed=5)
    _, _, gct, gsf_t = fp8.quantize_fp8_both(gy)
    _, _, vct, vsf_t = fp8.quantize_fp8_both(v)
    _close(fp8.fp8_gemm_tn(gct, vct, gsf_t, vsf_t, out), *ref.grad_weight(gy, v), f"TN {M}x{N}x{K}")
    _status()


def test_long_sums_are_as_exact_as_short_ones(variant):
    # fp32 output: the K loop is cut into chains of 4096 values, each with an error e relative to its sum;
    # the sum of m of them has at most m e |chain| ~ sqrt(m) e |sum| if all errors point one way.  (One
    # chain of 20000 has (20000 / 4096)^1.5 times the absolute error of one of 4096, twice the bound.)
    from lockstep_b200 import fp8
    errs = {}
    for K in (4096, 20000):
        gy, x = _data(K, 300, seed=5, spread=0.0), _data(K, 264, seed=6, spread=0.0)
        _, _, gct, gsf_t = fp8.quantize_fp8_both(gy)
        _, _, xct, xsf_t = fp8.quantize_fp8_both(x)
        a, b = ref.grad_weight(gy, x)
        want = a @ b
        tn = fp8.fp8_gemm_tn(gct, xct, gsf_t, xsf_t)
        _close(tn, a, b, f"TN {K}")
        errs[K] = ((tn.double() - want).norm() / want.norm()).item()
        xc, xsf = fp8.quantize_fp8_packed(gy.t().contiguous())
        wc, wsf, wsf_t = fp8.quantize_fp8_weight(x.t().contiguous())
        _close(fp8.fp8_gemm(xc, wc, xsf, wsf, torch.float32), *ref.forward(gy.t(), x.t()), f"NT {K}")
        wc, _, wsf_t = fp8.quantize_fp8_weight(x)
        _close(fp8.fp8_gemm_nn(xc, wc, xsf, wsf_t, torch.float32), *ref.grad_input(gy.t(), x), f"NN {K}")
    _status()
    assert errs[20000] <= np.sqrt(20000 / 4096) * errs[4096] + 2.0 ** -24, errs


# ---------------------------------------------------------------- grouped
MANY = [0, 1, 3, 130, 0, 0, 2, 40] * 128                      # 1024 groups
GROUPS = [[128], [0], [5, 0, 0, 300, 1, 0], [128, 128, 256], [1] * 40, [129, 127, 2, 640, 0, 33], [0, 0, 7], [1000, 3]]


def _offsets(sizes, dtype=torch.int32):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=dtype, device="cuda")


def test_as_many_groups_as_there_may_be():
    from lockstep_b200 import fp8, fp8_linear
    G, T, K, N = len(MANY), sum(MANY) + 5, 128, 72
    x, gy, w = _data(T, K, seed=7), _data(T, N, seed=8), _data(G, N, K, seed=9)
    off = _offsets(MANY)
    xi, wi = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fp8_linear.grouped_linear(xi, wi, off)
    y.backward(gy)
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    assert torch.equal(fp8_linear.grouped_linear_quantized(x, codes, sf, off), y)
    _status()
    bounds = off.tolist()
    for g in list(range(0, 24)) + list(range(1000, 1024)):
        r = slice(bounds[g], bounds[g + 1])
        if bounds[g] == bounds[g + 1]:
            assert (wi.grad[g] == 0).all()
            continue
        _close(y.detach()[r], *ref.forward(x[r], w[g]), f"y of group {g}")
        _close(xi.grad[r], *ref.grad_input(gy[r], w[g]), f"gx of group {g}")
        _close(wi.grad[g], *ref.grad_weight(gy[r], x[r]), f"gw of group {g}")
    assert (y[bounds[-1]:] == 0).all() and (xi.grad[bounds[-1]:] == 0).all()
    few = fp8_linear.grouped_linear_quantized(x[:20], codes, sf, off.clamp_max(20))
    _close(few[1:4], *ref.forward(x[1:4], w[2]), "group 2 of a few rows")


@pytest.mark.parametrize("N,K", [(128, 128), (264, 1000), (513, 200)])
@pytest.mark.parametrize("sizes", GROUPS, ids=lambda s: "-".join(map(str, s[:6])))
@pytest.mark.parametrize("tail", [0, 70])
def test_grouped_products(sizes, N, K, tail, variant):
    from lockstep_b200 import fp8
    G, T = len(sizes), sum(sizes) + tail
    x, gy = _data(T, K, seed=7), _data(T, N, seed=8)
    w = _data(G, N, K, seed=9)
    off = _offsets(sizes, torch.int64 if tail else torch.int32)
    wc, wsf, wsf_t = fp8.quantize_fp8_weight(w)
    xc, xsf, xct, xsf_t = fp8.quantize_fp8_both(x, off)
    gc, gsf, gct, gsf_t = fp8.quantize_fp8_both(gy, off)
    y = fp8.fp8_gemm_grouped(xc, wc, xsf, wsf, off, torch.float32)
    gx = fp8.fp8_gemm_grouped_nn(gc, wc, gsf, wsf_t, off)
    gw = fp8.fp8_gemm_grouped_tn(gct, xct, gsf_t, xsf_t, off, T)
    kept = torch.full((T, N), 7.0, device="cuda")
    fp8.fp8_gemm_grouped(xc, wc, xsf, wsf, off, torch.float32, out=kept)
    _status()
    at = 0
    for g, n in enumerate(sizes):
        rows = slice(at, at + n)
        at += n
        if n == 0:
            assert (gw[g] == 0).all()
            continue
        _close(y[rows], *ref.forward(x[rows], w[g]), f"y of group {g}")
        _close(gx[rows], *ref.grad_input(gy[rows], w[g]), f"gx of group {g}")
        _close(gw[g], *ref.grad_weight(gy[rows], x[rows]), f"gw of group {g}")
    assert (y[at:] == 0).all() and (gx[at:] == 0).all()
    assert torch.equal(kept[:at], y[:at]) and (kept[at:] == 7.0).all()


# ---------------------------------------------------------------- layers
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K,N", [(1, 128, 128), (257, 200, 131), (640, 1000, 512)])
def test_linear_and_gradients(T, K, N, dtype, wdtype):
    from lockstep_b200 import fp8, fp8_linear
    x, gy = _data(T, K, seed=11, dtype=dtype), _data(T, N, seed=12, dtype=dtype)
    w = _data(N, K, seed=13, dtype=wdtype)
    xi, wi = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fp8_linear.linear(xi, wi)
    y.backward(gy)
    _status()
    assert y.dtype == dtype and xi.grad.dtype == dtype and wi.grad.dtype == wdtype
    _close(y.detach(), *ref.forward(x, w), "y")
    _close(xi.grad, *ref.grad_input(gy, w), "gx")
    _close(wi.grad, *ref.grad_weight(gy, x), "gw")
    # one gradient at a time, without gradients, and from quantized weights: the same bits
    a = torch.autograd.grad(fp8_linear.linear(xi, w), xi, gy)[0]
    b = torch.autograd.grad(fp8_linear.linear(x, wi), wi, gy)[0]
    assert torch.equal(a, xi.grad) and torch.equal(b, wi.grad)
    assert torch.equal(fp8_linear.linear(x, w), y)
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    served = fp8_linear.linear_quantized(x, codes, sf)
    _close(served, *ref.forward(x, w), "served y")
    assert T <= 8 or torch.equal(served, y)                    # a few rows go through another kernel, with sums in another order
    x3 = x.view(1, T, 1, K)
    assert torch.equal(fp8_linear.linear_quantized(x3, codes, sf), served.view(1, T, 1, N))
    assert torch.equal(fp8_linear.linear(x3, w), y.view(1, T, 1, N))


@pytest.mark.parametrize("sizes,tail", [([5, 0, 300, 1], 9), ([0, 0], 3), ([128, 256], 0)])
def test_grouped_linear_and_gradients(sizes, tail):
    from lockstep_b200 import fp8, fp8_linear
    T, G, K, N = sum(sizes) + tail, len(sizes), 200, 136
    x, gy = _data(T, K, seed=14), _data(T, N, seed=15)
    layer = fp8_linear.FP8GroupedLinear(G, K, N).cuda()
    off = _offsets(sizes)
    xi = x.clone().requires_grad_()
    y = layer(xi, off)
    y.backward(gy)
    _status()
    at, w = 0, layer.weight.detach()
    for g, n in enumerate(sizes):
        rows = slice(at, at + n)
        at += n
        if n == 0:
            assert (layer.weight.grad[g] == 0).all()
            continue
        _close(y.detach()[rows], *ref.forward(x[rows], w[g]), "y")
        _close(xi.grad[rows], *ref.grad_input(gy[rows], w[g]), "gx")
        _close(layer.weight.grad[g], *ref.grad_weight(gy[rows], x[rows]), "gw")
    assert (y[at:] == 0).all() and (xi.grad[at:] == 0).all()
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    if T > 32:
        assert torch.equal(fp8_linear.grouped_linear_quantized(x, codes, sf, off), y)
    kept = torch.full((T, N), 3.0, device="cuda", dtype=x.dtype)
    assert fp8_linear.grouped_linear_quantized(x, codes, sf, off, out=kept) is kept
    assert torch.equal(kept[:at], fp8_linear.grouped_linear_quantized(x, codes, sf, off)[:at]) and (kept[at:] == 3.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 7, 8])
@pytest.mark.parametrize("K,N", [(128, 16), (1, 1), (1000, 130), (1111, 17), (4096, 256), (5000, 40)])
def test_few_rows(T, K, N, dtype):
    from lockstep_b200 import fp8, fp8_linear
    x, w = _data(T, K, seed=16, dtype=dtype, spread=3.0), _data(N, K, seed=17)
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    for out in (torch.bfloat16, torch.float32):
        _close(fp8_linear.linear_quantized(x, codes, sf, out), *ref.forward(x, w), f"{T} rows, {out}")
    if T > 1:
        x[1, K // 2], x[0, K - 1] = float("inf"), float("nan")
        y = fp8_linear.linear_quantized(x, codes, sf)
        assert y[:2].isnan().all() and y[2:].isfinite().all()


@pytest.mark.parametrize("sizes,tail", [([1], 0), ([0, 3, 0, 0, 9, 1], 2), ([0] * 40 + [1, 0, 17], 0), ([1] * 32, 0), ([0, 0], 5)])
@pytest.mark.parametrize("K,N", [(256, 64), (1000, 33)])
def test_few_rows_grouped(sizes, tail, K, N):
    from lockstep_b200 import fp8, fp8_linear
    T, G = sum(sizes) + tail, len(sizes)
    x, w = _data(T, K, seed=18), _data(G, N, K, seed=19)
    off = _offsets(sizes)
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    y = fp8_linear.grouped_linear_quantized(x, codes, sf, off, torch.float32)
    kept = fp8_linear.grouped_linear_quantized(x, codes, sf, off, torch.float32, out=torch.full((T, N), 7.0, device="cuda"))
    at = 0
    for g, n in enumerate(sizes):
        if n:
            _close(y[at:at + n], *ref.forward(x[at:at + n], w[g]), f"group {g}")
        at += n
    assert (y[at:] == 0).all() and torch.equal(kept[:at], y[:at]) and (kept[at:] == 7.0).all()


# ---------------------------------------------------------------- refusals
def test_python_refusals():
    from lockstep_b200 import fp8, fp8_linear
    x, w = _data(64, 256), _data(128, 256)
    xc, xsf = fp8.quantize_fp8_packed(x)
    wc, wsf, wsf_t = fp8.quantize_fp8_weight(w)
    w3, w3sf, _ = fp8.quantize_fp8_weight(w[None])
    off = _offsets([64])
    bad = [lambda: fp8.fp8_gemm(xc, wc, wsf, wsf[:-1]),                     # scale buffers of the wrong size or type
           lambda: fp8.fp8_gemm(xc, wc, xsf.float(), wsf),
           lambda: fp8.fp8_gemm(xc, wc[:, :128], xsf, wsf),                 # K differs
           lambda: fp8.fp8_gemm(xc[None], wc, xsf, wsf),
           lambda: fp8.fp8_gemm_grouped(xc, wc, xsf, wsf, off),             # a matrix where a stack is needed
           lambda: fp8.fp8_gemm_grouped(xc, w3, xsf, w3sf, _offsets([30, 34])),
           lambda: fp8.fp8_gemm_grouped_tn(xc, xc, xsf, xsf, off, 64),      # not in slot order
           lambda: fp8.fp8_gemm(xc, wc, xsf, wsf, out=torch.empty(64, 127, device="cuda", dtype=torch.bfloat16)),
           lambda: fp8.fp8_gemm(xc, wc, xsf, wsf, torch.float32, out=torch.empty(64, 128, device="cuda", dtype=torch.bfloat16)),
           lambda: fp8.quantize_fp8_both(x[None]), lambda: fp8.quantize_fp8_weight(x[0]),
           lambda: fp8.quantize_fp8_packed(x, torch.zeros(1026, dtype=torch.int32, device="cuda")),
           lambda: fp8.quantize_fp8_packed(x, torch.zeros(1, dtype=torch.int32, device="cuda")),
           lambda: fp8.quantize_fp8_packed(x[None], off),
           lambda: fp8.dequantize_fp8(xc, torch.ones(64, 3, device="cuda")),
           lambda: fp8_linear.linear_quantized(x, wc, wsf[1:]),
           lambda: fp8_linear.grouped_linear(x, w[None], _offsets([30, 34]))]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was not refused")
    for call in (lambda: fp8.quantize_fp8_packed(x, off.float()), lambda: fp8.fp8_gemm(x, wc, xsf, wsf),
                 lambda: fp8.fp8_gemm(xc, wc, xsf, wsf, torch.float16), lambda: fp8_linear.linear(x.half(), w)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: fp8.fp8_gemm(xc, wc.cpu(), xsf, wsf), lambda: fp8.quantize_fp8_packed(x, off.cpu())):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    y = fp8_linear.linear(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError):                                       # no second derivative
        g = torch.autograd.grad(y, y.grad_fn.next_functions[0][0].variable, torch.ones_like(y), create_graph=True)[0]
        g.sum().backward()


def test_abi_refusals():
    from lockstep_b200._lib import lib, ptr, stream
    L, buf = lib(), torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p, odd = ptr(buf), buf[8:].data_ptr()
    off = _offsets([4])
    EINVAL, EALIGN = -1, -2

    def gemm(form=0, a=p, lda=128, b=p, ldb=128, sfa=p, sfb=p, c=p, dt=0, M=4, N=4, K=128):
        return L.ls_fp8_gemm(form, a, lda, b, ldb, sfa, sfb, c, dt, M, N, K, stream())
    assert gemm(form=3) == gemm(dt=5) == gemm(M=-1) == gemm(K=1 << 31) == EINVAL
    assert gemm(a=None) == gemm(b=None) == gemm(sfa=None) == gemm(sfb=None) == gemm(c=None) == EINVAL
    assert gemm(lda=127) == gemm(ldb=120) == gemm(lda=136) == EINVAL
    assert gemm(a=odd) == gemm(b=odd) == gemm(c=odd) == gemm(sfa=odd) == EALIGN
    assert gemm(M=0) == gemm(N=0, c=None) == 0                              # nothing to do
    grouped = lambda off_, G: L.ls_fp8_gemm_grouped(0, p, 128, p, 128, p, p, p, 0, 4, 4, 128, off_, G, 0, stream())
    assert grouped(None, 1) == grouped(ptr(off), 0) == grouped(ptr(off), 1025) == EINVAL

    def quant(x=p, dt=0, rows=4, K=128, off_=None, G=0, codes=p, ld=128, scale=None, sf=p):
        return L.ls_quantize_fp8(x, dt, rows, K, off_, G, codes, ld, scale, sf, stream())
    assert quant(dt=2) == quant(x=None) == quant(codes=None) == quant(ld=120) == quant(rows=-1) == EINVAL
    assert quant(off_=ptr(off), G=0) == quant(off_=ptr(off), G=2000) == EINVAL
    assert quant(codes=odd) == quant(sf=odd) == EALIGN
    both = lambda **k: L.ls_quantize_fp8_both(p, 0, 4, 128, None, 0, k.get("c", p), k.get("s", p), k.get("ct", p), k.get("st", p), 128, stream())
    assert both(c=None) == both(ct=None) == both(st=None) == EINVAL and both(ct=odd) == EALIGN
    assert L.ls_quantize_fp8_weight(p, 0, 1025, 4, 128, p, 128, None, p, p, stream()) == EINVAL
    serve = lambda **k: L.ls_fp8_linear(k.get("x", p), k.get("dt", 0), k.get("rows", 20), 128, k.get("w", p), k.get("ldw", 128), p, 4, k.get("y", p),
                                        0, None, k.get("G", 1), 0, k.get("work", p), stream())
    assert serve(work=None) == serve(y=None) == serve(dt=7) == serve(G=0) == serve(G=3) == EINVAL
    assert serve(rows=2, x=None) == serve(rows=2, ldw=100) == serve(rows=2, w=None) == EINVAL and serve(rows=2, w=odd) == EALIGN
    assert L.ls_fp8_linear_forward(p, 0, p, 0, 4, 4, 128, None, 1, 3, p, None, p, stream()) == EINVAL       # nowhere to keep
    assert L.ls_fp8_linear_forward(p, 0, p, 0, 4, 4, 128, None, 1, 4, p, p, p, stream()) == EINVAL
    assert L.ls_fp8_gemm_grouped(0, p, 128, p, 128, p, p, p, 0, 4, 4, 0, ptr(off), 1, 0, stream()) == EINVAL
    assert L.ls_fp8_gemm_set_variant(6) == EINVAL
    torch.cuda.synchronize()


# ---------------------------------------------------------------- how tensors come
def test_strides_offsets_and_alignment():
    from lockstep_b200 import fp8, fp8_linear
    base = _data(260, 700, seed=20)
    w = _data(130, 256, seed=21)
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    want = lambda x: fp8_linear.linear_quantized(x.contiguous(), codes, sf)
    for x in (base[:, 3:259], base[::2, 100:356], base[1:, :256], base.t()[100:356, :200].t()):
        assert torch.equal(fp8_linear.linear_quantized(x, codes, sf), want(x))
    # weights at any pitch and alignment
    x = base[:50, :256].contiguous()
    wide = torch.zeros(130, 300, dtype=torch.uint8, device="cuda")
    for at in (0, 16, 5):
        wide[:, at:at + 256] = codes.view(torch.uint8)
        view = wide.view(torch.float8_e4m3fn)[:, at:at + 256]
        assert torch.equal(fp8_linear.linear_quantized(x, view, sf), want(x))
        assert torch.equal(fp8_linear.linear_quantized(x[:2], view, sf), want(x[:2]))
    flat = torch.empty(130 * 256 + 7, dtype=torch.uint8, device="cuda")[7:]
    flat.view(130, 256).copy_(codes.view(torch.uint8))
    assert torch.equal(fp8_linear.linear_quantized(x, flat.view(130, 256), sf), want(x))
    # a gradient that is an expanded view
    xi = x.clone().requires_grad_()
    fp8_linear.linear(xi, w).sum().backward()
    ones = torch.ones(50, 130, device="cuda", dtype=torch.bfloat16)
    _close(xi.grad, *ref.grad_input(ones, w), "gradient of a sum")
    # the same weight twice in one graph: its gradients add up
    wi = w.float().requires_grad_()
    (fp8_linear.linear(x, wi) + fp8_linear.linear(x, wi)).backward(ones)
    one = torch.autograd.grad(fp8_linear.linear(x, wi), wi, ones)[0]
    assert torch.equal(wi.grad, one + one)


@pytest.mark.parametrize("T,K,N,G", [(0, 64, 64, 0), (5, 64, 0, 0), (5, 0, 64, 0), (0, 64, 64, 3), (6, 0, 32, 2)])
def test_empty_sizes(T, K, N, G):
    from lockstep_b200 import fp8_linear
    x = torch.zeros(T, K, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros(*([G] if G else []), N, K, device="cuda", requires_grad=True)
    off = _offsets([T // 2, T - T // 2] + [0] * (G - 2)) if G else None
    y = fp8_linear.grouped_linear(x, w, off) if G else fp8_linear.linear(x, w)
    assert y.shape == (T, N) and (y == 0).all()
    y.backward(torch.ones_like(y))
    assert x.grad.shape == x.shape and (x.grad == 0).all() and w.grad.shape == w.shape and (w.grad == 0).all()


def test_offsets_out_of_order_stay_in_bounds():
    # unspecified values, but nothing outside the outputs and no failed wait
    from lockstep_b200 import fp8, fp8_linear
    T, K, N = 300, 200, 136
    x, gy = _data(T, K, seed=22), _data(T, N, seed=23)
    for vals in ([0, 200, 100, 300], [50, -7, 1 << 30, 20], [-5, -5, -5, -5], [300, 300, 300, 300], [7, 7, 7, 400]):
        off = torch.tensor(vals, dtype=torch.int32, device="cuda")
        w = _data(3, N, K, seed=24).requires_grad_()
        guard = torch.full((T + 64, N), 7.0, device="cuda", dtype=torch.bfloat16)
        codes, sf, _ = fp8.quantize_fp8_weight(w.detach())
        fp8_linear.grouped_linear_quantized(x, codes, sf, off, out=guard[32:32 + T])
        fp8_linear.grouped_linear_quantized(x[:9], codes, sf, off)
        xi = x.clone().requires_grad_()
        fp8_linear.grouped_linear(xi, w, off).backward(gy)
        _status()
        assert (guard[:32] == 7.0).all() and (guard[32 + T:] == 7.0).all()


@pytest.mark.parametrize("M,N", [(300, 513), (7, 130), (129, 64)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_nothing_is_stored_outside_the_output(M, N, out, variant):
    from lockstep_b200 import fp8
    x, w = _data(M, 300, seed=25), _data(N, 300, seed=26)
    xc, xsf = fp8.quantize_fp8_packed(x)
    wc, wsf, _ = fp8.quantize_fp8_weight(w)
    flat = torch.full((M * N + 256,), 7.0, device="cuda", dtype=out)
    c = fp8.fp8_gemm(xc, wc, xsf, wsf, out, out=flat[128:128 + M * N].view(M, N))
    _close(c, *ref.forward(x, w), "C")
    assert (flat[:128] == 7.0).all() and (flat[128 + M * N:] == 7.0).all()


def test_a_nan_stays_in_its_rows():
    from lockstep_b200 import fp8, fp8_linear
    x, w = _data(300, 400, seed=27), _data(200, 400, seed=28)
    x[17, 3], x[299, 399] = float("nan"), float("-inf")
    y = fp8_linear.linear(x, w)
    rows = torch.zeros(300, dtype=torch.bool, device="cuda")
    rows[17] = rows[299] = True
    assert y[rows].isnan().all() and y[~rows].isfinite().all()
    w[5, 0] = float("nan")
    y = fp8_linear.linear(x, w)
    assert y[:, 5].isnan().all() and y[~rows][:, [c for c in range(200) if c != 5]].isfinite().all()


def test_more_than_2_to_31_values():
    from lockstep_b200 import fp8
    rows, K, N = 66000, 33024, 32                              # 2.18e9 values
    x = torch.empty(rows, K, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w = _data(N, K, seed=29)
    codes, sf = fp8.quantize_fp8_packed(x)
    wc, wsf, _ = fp8.quantize_fp8_weight(w)
    y = fp8.fp8_gemm(codes, wc, sf, wsf, torch.float32)
    _status()
    for r in (0, 40000, 65409, rows - 1):
        q, _ = ref.quantize(x[r:r + 1], (1, 128))
        assert torch.equal(codes[r:r + 1].double(), q)
        _close(y[r:r + 1], *ref.forward(x[r:r + 1], w), f"row {r}")
    _, _, codes_t, sf_t = fp8.quantize_fp8_both(x, rows_too=False)
    q, _ = ref.quantize(x[65920:66000, :300], (128, 1))
    assert torch.equal(codes_t[65920:, :300].double(), q)


# ---------------------------------------------------------------- streams, graphs, threads
def test_on_another_stream_and_captured():
    from lockstep_b200 import fp8, fp8_linear
    w = _data(3, 264, 400, seed=30)
    codes, sf, _ = fp8.quantize_fp8_weight(w)
    dense = (codes[0], sf[0].contiguous())
    runs = {T: (_data(T, 400, seed=31), _offsets([T // 3, 0, T - T // 3])) for T in (3, 200)}
    calls = [lambda x, o: fp8_linear.linear_quantized(x, *dense), lambda x, o: fp8_linear.grouped_linear_quantized(x, codes, sf, o)]
    want = {(T, i): f(*a) for T, a in runs.items() for i, f in enumerate(calls)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = {(T, i): f(*a) for T, a in runs.items() for i, f in enumerate(calls)}
    side.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    # two graphs of the same calls, replayed in turn and at once, on inputs changed in place
    graphs = []
    for _ in range(2):
        ins = {T: (x.clone(), o.clone()) for T, (x, o) in runs.items()}
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = {(T, i): f(*ins[T]) for T in runs for i, f in enumerate(calls)}
        graphs.append((g, ins, outs))
    other = {T: (_data(T, 400, seed=32), _offsets([1, T - 2, 1])) for T in runs}
    for T in runs:
        for a, b in zip(graphs[1][1][T], other[T]):
            a.copy_(b)
    torch.cuda.synchronize()
    s0, s1 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s0):
            graphs[0][0].replay()
        with torch.cuda.stream(s1):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    _status()
    assert all(torch.equal(graphs[0][2][k], want[k]) for k in want)
    assert all(torch.equal(graphs[1][2][k], calls[k[1]](*other[k[0]])) for k in want)


def test_training_step_captured():
    from lockstep_b200 import fp8_linear
    x, gy = _data(200, 256, seed=33), _data(200, 136, seed=34)
    off = _offsets([50, 0, 150])
    layer = fp8_linear.FP8GroupedLinear(3, 256, 136).cuda()
    xi = x.clone().requires_grad_()
    ref_grads = [t.clone() for t in torch.autograd.grad(layer(xi, off), (xi, layer.weight), gy)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    leaf, weight = x.clone().requires_grad_(), layer.weight.detach().clone().requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(fp8_linear.grouped_linear(leaf, weight, off), (leaf, weight), gy)
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(g, stream=s):
        got = torch.autograd.grad(fp8_linear.grouped_linear(leaf, weight, off), (leaf, weight), gy)
    for t in got:
        t.zero_()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref_grads[0]) and torch.equal(got[1], ref_grads[1])


def test_nothing_is_kept_without_gradients():
    from lockstep_b200 import fp8_linear
    rows, K, N = 4096, 2048, 256
    x, w = _data(rows, K, seed=35).requires_grad_(), _data(N, K, seed=36).requires_grad_()
    off = _offsets([1000, rows - 1000])
    wg = torch.stack([w.detach(), -w.detach()]).requires_grad_()
    for f, experts in ((lambda: fp8_linear.linear(x, w), 1), (lambda: fp8_linear.grouped_linear(x, wg, off), 2)):
        want = f()
        kept = want.detach().clone()
        del want
        for mode in (torch.no_grad, torch.inference_mode):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            with mode():
                y = f()
            torch.cuda.synchronize()
            peak = torch.cuda.max_memory_allocated() - before
            # one byte per value, the scales (a 32nd of that at most) and the output; half of x's codes again is too much
            values = (rows + experts * 128) * K + experts * N * K
            assert peak < values * 33 // 32 + y.numel() * y.element_size() + rows * K // 2, (peak, values)
            assert torch.equal(y, kept)
            del y


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    code = ("import torch\nfrom lockstep_b200 import fp8, fp8_linear\n"
            "x = torch.randn(40, 256, device='cuda').bfloat16(); w = torch.randn(64, 256, device='cuda')\n"
            "torch.cuda.synchronize(); g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n    c, s, _ = fp8.quantize_fp8_weight(w); y = fp8_linear.linear_quantized(x, c, s)\n"
            "g.replay(); torch.cuda.synchronize(); c, s, _ = fp8.quantize_fp8_weight(w)\n"
            "assert torch.equal(y, fp8_linear.linear_quantized(x, c, s)); print('ok')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]


def test_host_threads_at_once():
    import threading
    from lockstep_b200 import fp8, fp8_linear
    shapes = [(40 + 50 * i, 256 + 64 * i, 136 + 8 * i) for i in range(4)]
    data = [(_data(T, K, seed=i), fp8.quantize_fp8_weight(_data(N, K, seed=40 + i))) for i, (T, K, N) in enumerate(shapes)]
    want = [fp8_linear.linear_quantized(x, w[0], w[1]) for x, w in data]
    torch.cuda.synchronize()
    fails = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    y = fp8_linear.linear_quantized(data[i][0], data[i][1][0], data[i][1][1])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    fails.append(i)
        except Exception as e:                                             # noqa: BLE001
            fails.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not fails, fails


# ---------------------------------------------------------------- together, as a model has them
def test_gradients_against_differences():
    # linear functionals of y: d/de <c, f(x + e d)> by the operator's own formula; the quantizer is a
    # staircase, so differences are taken of the unquantized product and must agree with the FP8
    # gradient within the rounding of its operands (2^-4 relative each, random signs)
    from lockstep_b200 import fp8_linear
    x, w, gy = _data(256, 384, seed=35, dtype=torch.float32, spread=0.0), _data(128, 384, seed=36, dtype=torch.float32, spread=0.0), \
        _data(256, 128, seed=37, dtype=torch.float32, spread=0.0)
    xi, wi = x.clone().requires_grad_(), w.clone().requires_grad_()
    fp8_linear.linear(xi, wi).backward(gy)
    f = lambda a, b: (gy.double() * (a @ b.t())).sum()
    for got, at in ((xi.grad, 0), (wi.grad, 1)):
        args = [x.double(), w.double()]
        d = got.double()                                       # the steepest direction: no cancellation
        e = 1e-6
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + e * d, args[at] - e * d
        slope = (f(*up) - f(*down)) / (2 * e)
        assert abs(slope / (d * d).sum() - 1) <= 2.0 ** -4


def test_experts_as_a_model_runs_them():
    # routing -> sort -> grouped up projection -> gelu -> grouped down projection -> unsort, forward and
    # backward, against the same composition of the oracle's products, step by step
    from lockstep_b200 import fp8_linear
    T, G, D, H = 700, 5, 256, 384
    x, gy = _data(T, D, seed=38, spread=0.3), _data(T, D, seed=39, spread=0.3)
    up, down = fp8_linear.FP8GroupedLinear(G, D, H).cuda(), fp8_linear.FP8GroupedLinear(G, H, D).cuda()
    expert = torch.randint(0, G, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    expert[expert == 2] = 3                                    # an expert without rows
    order = torch.argsort(expert, stable=True)
    off = torch.cat([torch.zeros(1, device="cuda", dtype=torch.long), torch.bincount(expert, minlength=G).cumsum(0)])
    xi = x.clone().requires_grad_()
    h = up(xi[order], off)
    a = torch.nn.functional.gelu(h)
    a.retain_grad(), h.retain_grad()
    y = down(a, off)
    out = torch.zeros_like(y).index_copy(0, order, y)
    out.backward(gy)
    _status()
    bounds = off.tolist()
    gs = gy[order]
    for g in range(G):
        r = slice(bounds[g], bounds[g + 1])
        if bounds[g] == bounds[g + 1]:
            assert (up.weight.grad[g] == 0).all() and (down.weight.grad[g] == 0).all()
            continue
        _close(h.detach()[r], *ref.forward(x[order][r], up.weight.detach()[g]), "up")
        _close(y.detach()[r], *ref.forward(a.detach()[r], down.weight.detach()[g]), "down")
        _close(a.grad[r], *ref.grad_input(gs[r], down.weight.detach()[g]), "grad of the activation")
        _close(down.weight.grad[g], *ref.grad_weight(gs[r], a.detach()[r]), "grad of down")
        _close(up.weight.grad[g], *ref.grad_weight(h.grad[r], x[order][r]), "grad of up")


def test_decoder_steps_with_fp8_projections():
    # runs, every parameter gets a finite gradient, and the projections' gradients are the operator's
    import train_bench
    t = train_bench.Trainer("fp8", layers=2, width=256, heads=4, context=128, batch=4, vocab=512)
    lin = t.model.blocks[0].attn.proj
    seen = {}
    lin.register_forward_hook(lambda m, i, o: (seen.update(x=i[0].detach()), o.register_hook(lambda g: seen.update(gy=g)))[0] and None)
    t.step()
    t.flat.zero_()
    with torch.autocast("cuda", torch.bfloat16):
        loss = t.model(t.x, t.y)
    loss.backward()
    t.close()
    _status()
    assert torch.isfinite(loss) and all(p.grad.isfinite().all() for p in t.params)
    gy, x = seen["gy"].reshape(-1, 256), seen["x"].reshape(-1, 256).bfloat16()
    _close(lin.weight.grad, *ref.grad_weight(gy, x), "projection weight")
