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

import functools

import torch
import torch.nn as nn

from . import _lib, fp8
from ._lib import check, lib, on_device_of

_SERVE, _FORWARD, _SAVED, _BACKWARD = range(4)
_GRAD_X, _GRAD_W = 1, 2


def _check(x, w, dims):
    if w.dim() != dims:
        raise AssertionError(f"weight must be {dims}-dimensional, got shape {tuple(w.shape)}")
    if x.shape[-1] != w.shape[-1]:
        raise AssertionError(f"input of width {x.shape[-1]} for a weight of shape {tuple(w.shape)}")
    if x.dtype not in fp8._DTYPE:
        raise TypeError(f"unsupported dtype {x.dtype}")


@functools.lru_cache(maxsize=4096)
def _buffer_bytes(what, rows, N, K, groups, grads):
    return int(lib().ls_fp8_linear_bytes(what, rows, N, K, groups, grads))


@functools.lru_cache(maxsize=4096)
def _training_bytes(rows, N, K, groups, grads):
    """Buffers of a forward pass, kept for the backward pass, of a backward pass."""
    return tuple(max(16, _buffer_bytes(what, rows, N, K, groups, grads)) for what in (_FORWARD, _SAVED, _BACKWARD))


class _FP8Matmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, recording):
        # recording: the caller's grad mode; without it nothing is prepared for a backward pass
        with on_device_of(x, w, offsets):
            off, G = (None, 0) if offsets is None else fp8._groups(offsets)
            if off is not None and w.shape[0] != G:
                raise AssertionError(f"{w.shape[0]} experts for offsets of {G} groups")
            xi, wi = fp8._aligned(x), fp8._input(w, w.dim())
            (rows, K), N = xi.shape, w.shape[-2]
            need = ctx.needs_input_grad
            grads = (_GRAD_X if need[0] else 0) | (_GRAD_W if need[1] else 0) if recording else 0
            work_bytes, saved_bytes, back_bytes = _training_bytes(rows, N, K, G, grads)
            y = xi.new_empty((rows, N))
            work = xi.new_empty((work_bytes,), dtype=torch.uint8)
            saved = xi.new_empty((saved_bytes,), dtype=torch.uint8) if grads else None
            check(lib().ls_fp8_linear_forward(xi.data_ptr(), fp8._DTYPE[xi.dtype], wi.data_ptr(), fp8._DTYPE[wi.dtype], rows, N, K,
                                              fp8._ptr(off), G or 1, grads, y.data_ptr(), fp8._ptr(saved), work.data_ptr(), fp8._stream(xi)))
            ctx.save_for_backward(saved, off)
            ctx.what = (rows, N, K, G, grads, x.dtype, w.dtype, w.shape, back_bytes)
            return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        saved, off = ctx.saved_tensors
        rows, N, K, G, grads, x_dtype, w_dtype, w_shape, back_bytes = ctx.what
        with on_device_of(gy, saved, off):
            gy = fp8._input(gy)
            gx = gy.new_empty((rows, K), dtype=x_dtype) if grads & _GRAD_X else None
            gw = gy.new_empty(w_shape, dtype=w_dtype if w_dtype in fp8._DTYPE else torch.float32) if grads & _GRAD_W else None
            work = gy.new_empty((back_bytes,), dtype=torch.uint8)
            check(lib().ls_fp8_linear_backward(gy.data_ptr(), fp8._DTYPE[gy.dtype], rows, N, K, fp8._ptr(off), G or 1, grads,
                                               saved.data_ptr(), fp8._ptr(gx), fp8._DTYPE[x_dtype], fp8._ptr(gw),
                                               _lib.LS_F32 if gw is None else fp8._DTYPE[gw.dtype], work.data_ptr(), fp8._stream(gy)))
            return gx, (gw if gw is None or gw.dtype == w_dtype else gw.to(w_dtype)), None, None


def linear(x, weight):
    """x [..., in] (bf16 or fp32), weight [out, in] -> [..., out] in x's dtype, with FP8 gradients."""
    _check(x, weight, 2)
    if x.dim() == 2:
        return _FP8Matmul.apply(x, weight, None, torch.is_grad_enabled())
    return _FP8Matmul.apply(x.reshape(-1, x.shape[-1]), weight, None, torch.is_grad_enabled()).view(*x.shape[:-1], weight.shape[0])


def grouped_linear(x, weight, offsets):
    """x [rows, in] sorted by expert, weight [experts, out, in] -> [rows, out] in x's dtype, with FP8
    gradients.  Rows of no expert give zeros, also in their gradient."""
    _check(x, weight, 3)
    if x.dim() != 2:
        raise AssertionError(f"rows sorted by expert are two-dimensional, got shape {tuple(x.shape)}")
    if offsets is None:
        raise AssertionError("offsets are needed")
    return _FP8Matmul.apply(x, weight, offsets, torch.is_grad_enabled())


# One token's linear is a few microseconds on the device, so these two keep to what the call needs;
# whatever is not the ordinary case goes through the same helpers as everywhere else.
def _serve(x, codes, sf, offsets, out_dtype, out):
    with on_device_of(x, codes, sf, offsets, out):
        off, G = (None, 0) if offsets is None else fp8._groups(offsets)
        if off is not None and codes.shape[0] != G:
            raise AssertionError(f"{codes.shape[0]} experts for offsets of {G} groups")
        if not x.is_contiguous() or x.data_ptr() % 32:
            x = fp8._aligned(x)
        rows, K = x.shape
        N = codes.shape[-2]
        codes, ld = fp8._pitched(codes)
        sf = fp8._sf(sf, (G or 1) * fp8.sf_bytes(N, K), "sf")
        if out_dtype is None:
            out_dtype = x.dtype
        code = fp8._out_code(out_dtype)
        y = x.new_empty((rows, N), dtype=out_dtype) if out is None else fp8._given(out, (rows, N), out_dtype)
        size = _buffer_bytes(_SERVE, rows, N, K, G, 0)
        work = x.new_empty((size,), dtype=torch.uint8) if size else None       # (a few rows need no buffer)
        check(lib().ls_fp8_linear(x.data_ptr(), fp8._DTYPE[x.dtype], rows, K, codes.data_ptr(), ld, sf.data_ptr(), N, y.data_ptr(), code,
                                  fp8._ptr(off), G or 1, 1 if out is None else 0, fp8._ptr(work), fp8._stream(x)))
        return y


def linear_quantized(x, codes, sf, out_dtype=None):
    """linear(x, w) for a weight quantized beforehand (codes and sf of fp8.quantize_fp8_weight); no gradients."""
    _check(x, codes, 2)
    if x.dim() == 2:
        return _serve(x, codes, sf, None, out_dtype, None)
    return _serve(x.reshape(-1, x.shape[-1]), codes, sf, None, out_dtype, None).view(*x.shape[:-1], codes.shape[0])


def grouped_linear_quantized(x, codes, sf, offsets, out_dtype=None, out=None):
    """grouped_linear for weights quantized beforehand; no gradients.  With `out` the rows of no
    expert are left as they were."""
    _check(x, codes, 3)
    if x.dim() != 2:
        raise AssertionError(f"rows sorted by expert are two-dimensional, got shape {tuple(x.shape)}")
    if offsets is None:
        raise AssertionError("offsets are needed")
    return _serve(x, codes, sf, offsets, out_dtype, out)


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
