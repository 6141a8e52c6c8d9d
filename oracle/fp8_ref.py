"""64-bit restatement of the FP8 block-128 format and of the linear layers on it (test infrastructure).

scale = smallest power of two s with amax <= 448 s over the block's finite values, at least 2^-126,
1 for a block of zeros; value = E4M3(x / s) s, nearest with ties to even; non-finite -> NaN."""

import torch

BLOCK = 128


def e4m3(q):
    """Nearest E4M3 value of doubles with |q| <= 448 (ties to even); NaN stays NaN."""
    e = torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)                                    # 3 fraction bits; subnormals have the step of 2^-6
    return torch.round(q / step) * step


def scale_of(amax):
    """Powers of two (float64) from block maxima (float64, finite)."""
    m, e = torch.frexp(amax)                                    # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-126)
    s = torch.exp2(e.double())
    return torch.where(amax > 0, s, torch.ones_like(s))


def quantize(x, spans):
    """x -> (code values, scales with x's shape), one scale per block of spans[i] along axis i."""
    x = x.double()
    q, s = torch.empty_like(x), torch.empty_like(x)
    padded = [-(-n // b) * b for n, b in zip(x.shape, spans)]
    full = torch.zeros(padded, dtype=torch.float64, device=x.device)
    full[tuple(slice(n) for n in x.shape)] = x
    shape = [v for n, b in zip(padded, spans) for v in (n // b, b)]
    blocks = full.view(shape)
    finite = torch.where(blocks.isfinite(), blocks.abs(), torch.zeros((), dtype=torch.float64, device=x.device))
    sc = scale_of(finite.amax(tuple(range(1, 2 * len(spans), 2)), keepdim=True)) if x.numel() else blocks
    codes = torch.where(blocks.isfinite(), e4m3(torch.where(blocks.isfinite(), blocks, 0.0) / sc), torch.nan)
    at = tuple(slice(n) for n in x.shape)
    q = codes.reshape(padded)[at]
    s = sc.expand(shape).reshape(padded)[at]
    return q, s


def fq(x, *spans):
    q, s = quantize(x, spans)
    return q * s


def forward(x, w):
    return fq(x, 1, BLOCK), fq(w, BLOCK, BLOCK).t()


def grad_input(gy, w):
    return fq(gy, 1, BLOCK), fq(w, BLOCK, BLOCK)


def grad_weight(gy, x):
    return fq(gy, BLOCK, 1).t(), fq(x, BLOCK, 1)
