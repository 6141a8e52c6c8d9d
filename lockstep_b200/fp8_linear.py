"""(extension) Linear layers in FP8 with one scale per block of 128, dense and grouped by expert.

The 8-bit counterpart of fp4_linear.py.  Forward, input gradient and weight gradient are FP8
products, each operand quantized along the axis its product sums over:

    y  = q(x) q(w)^T          activations: blocks of 128 along the features
    gx = q(gy) q(w)           weights: blocks of 128 x 128, the same codes in both products
    gw = q(gy)^T q(x)         blocks of 128 tokens

x and gy are read once each (both forms leave one kernel); what is kept for the backward pass is
one byte per value.  Grouped: the rows of x are sorted by expert, `offsets` (see fp8.py) says
where each expert's rows start, and the weight is [experts, out, in].

There is no CPU path.
"""

import torch
import torch.nn as nn

from . import fp8


def _check(x, w, dims):
    if w.dim() != dims:
        raise ValueError(f"weight must be {dims}-dimensional, got shape {tuple(w.shape)}")
    if x.shape[-1] != w.shape[-1]:
        raise ValueError(f"input of width {x.shape[-1]} for a weight of shape {tuple(w.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {x.dtype}")


class _FP8Matmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        wc, wsf, wsf_t = fp8.quantize_fp8_weight(w)
        if ctx.needs_input_grad[1]:
            xc, xsf, xct, xsf_t = fp8.quantize_fp8_both(x, offsets)
        else:
            (xc, xsf), xct, xsf_t = fp8.quantize_fp8_packed(x, offsets), None, None
        keep_w = ctx.needs_input_grad[0]
        ctx.save_for_backward(offsets, xct, xsf_t, wc if keep_w else None, wsf_t if keep_w else None)
        ctx.rows, ctx.dtypes = x.shape[0], (x.dtype, w.dtype)
        if offsets is None:
            return fp8.fp8_gemm(xc, wc, xsf, wsf, x.dtype)
        return fp8.fp8_gemm_grouped(xc, wc, xsf, wsf, offsets, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        offsets, xct, xsf_t, wc, wsf_t = ctx.saved_tensors
        x_dtype, w_dtype = ctx.dtypes
        need_x, need_w = ctx.needs_input_grad[:2]
        gx = gw = None
        if need_w:
            gc, gsf, gct, gsf_t = fp8.quantize_fp8_both(gy, offsets, rows_too=need_x)
        elif need_x:
            gc, gsf = fp8.quantize_fp8_packed(gy, offsets)
        out_w = w_dtype if w_dtype in (torch.float32, torch.bfloat16) else torch.float32
        if offsets is None:
            gx = fp8.fp8_gemm_nn(gc, wc, gsf, wsf_t, x_dtype) if need_x else None
            gw = fp8.fp8_gemm_tn(gct, xct, gsf_t, xsf_t, out_w) if need_w else None
        else:
            gx = fp8.fp8_gemm_grouped_nn(gc, wc, gsf, wsf_t, offsets, x_dtype) if need_x else None
            gw = fp8.fp8_gemm_grouped_tn(gct, xct, gsf_t, xsf_t, offsets, ctx.rows, out_w) if need_w else None
        return gx, (gw.to(w_dtype) if need_w else None), None


def linear(x, weight):
    """x [..., in] (bf16 or fp32), weight [out, in] -> [..., out] in x's dtype, with FP8 gradients."""
    _check(x, weight, 2)
    y = _FP8Matmul.apply(x.reshape(-1, x.shape[-1]), weight, None)
    return y.view(*x.shape[:-1], weight.shape[0])


def linear_quantized(x, codes, sf, out_dtype=None):
    """linear(x, w) for a weight quantized beforehand (codes and sf of fp8.quantize_fp8_weight); no gradients."""
    _check(x, codes, 2)
    xc, xsf = fp8.quantize_fp8_packed(x.reshape(-1, x.shape[-1]))
    return fp8.fp8_gemm(xc, codes, xsf, sf, out_dtype or x.dtype).view(*x.shape[:-1], codes.shape[0])


def grouped_linear(x, weight, offsets):
    """x [rows, in] sorted by expert, weight [experts, out, in] -> [rows, out] in x's dtype, with FP8
    gradients.  Rows of no expert give zeros, also in their gradient."""
    _check(x, weight, 3)
    if x.dim() != 2:
        raise ValueError(f"rows sorted by expert are two-dimensional, got shape {tuple(x.shape)}")
    return _FP8Matmul.apply(x, weight, offsets)


def grouped_linear_quantized(x, codes, sf, offsets, out_dtype=None, out=None):
    """grouped_linear for weights quantized beforehand; no gradients.  With `out` the rows of no
    expert are left as they were."""
    _check(x, codes, 3)
    if x.dim() != 2:
        raise ValueError(f"rows sorted by expert are two-dimensional, got shape {tuple(x.shape)}")
    xc, xsf = fp8.quantize_fp8_packed(x, offsets)
    return fp8.fp8_gemm_grouped(xc, codes, xsf, sf, offsets, out_dtype or x.dtype, out)


class FP8Linear(nn.Linear):
    """nn.Linear whose three products run in FP8 (bias unsupported)."""

    def __init__(self, fan_in, fan_out, bias=False):
        assert not bias, "FP8Linear has no bias"
        super().__init__(fan_in, fan_out, bias=False)

    def forward(self, x):
        dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
        with torch.autocast("cuda", enabled=False):
            return linear(x.to(dt), self.weight)


class FP8GroupedLinear(nn.Module):
    """One FP8Linear per expert over rows sorted by expert: weight [experts, fan_out, fan_in]."""

    def __init__(self, experts, fan_in, fan_out):
        super().__init__()
        self.experts, self.fan_in, self.fan_out = experts, fan_in, fan_out
        self.weight = nn.Parameter(torch.empty(experts, fan_out, fan_in))
        for w in self.weight:                                # as nn.Linear initialises each of them
            nn.init.kaiming_uniform_(w, a=5 ** 0.5)

    def forward(self, x, offsets):
        dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
        with torch.autocast("cuda", enabled=False):
            return grouped_linear(x.to(dt), self.weight, offsets)
