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


@pytest.fixture(params=[0, 1, 2, 3, 4])
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


def test_long_sums_are_as_exact_as_short_ones(variant):
    # fp32 output: the K loop is cut into chains of 2048 values, each with an error e relative to its sum;
    # the sum of m of them has at most m e |chain| ~ sqrt(m) e |sum| if all errors point one way.  A single
    # chain of 20000 has (20000 / 2048)^1.5 times the absolute error of one of 2048.
    from lockstep_b200 import fp8
    errs = {}
    for K in (2048, 20000):
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
    assert errs[20000] <= np.sqrt(20000 / 2048) * errs[2048] + 2.0 ** -24, errs


# ---------------------------------------------------------------- grouped
GROUPS = [[128], [0], [5, 0, 0, 300, 1, 0], [128, 128, 256], [1] * 40, [129, 127, 2, 640, 0, 33], [0, 0, 7], [1000, 3]]


def _offsets(sizes, dtype=torch.int32):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=dtype, device="cuda")


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
