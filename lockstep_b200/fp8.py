"""(extension) FP8 values with one power-of-two scale per block of 128: quantizers and products.

lockstep's codec and products are 4-bit; this module is the 8-bit step above them for layers
and gradients that do not survive E2M1.  Codes are E4M3.  A block is 128 values along the axis a
product sums over, and 128 x 128 for weights (so that a weight and its transpose have the same
codes); its scale is the smallest power of two s with max|x| <= 448 s, at least 2^-126, and 1
for a block of zeros.  The scales being powers of two, division by them is exact and the tensor
cores apply them (`tcgen05.mma.kind::mxf8f6f4.block_scale`).  The maximum runs over the finite
values; infinities and NaNs become E4M3's NaN.

Sizes are free: a ragged end is a short block.  Codes are float8_e4m3fn tensors whose row pitch
is a multiple of 16 bytes (a view of a wider buffer where the row length is not); `sf` buffers
hold the scale bytes in the tensor-core layout of fp4.py.

Ragged groups (rows sorted by expert): `offsets` is a CUDA tensor of groups + 1 integers, rows
offsets[g] .. offsets[g + 1] belong to group g.  Nothing reads it on the host.  Groups may be
empty; rows behind offsets[-1] belong to nobody.  A tensor quantized with offsets goes to the
grouped products with the same offsets.
"""

import torch

from . import _lib
from ._lib import aligned, check, lib, on_device_of, ptr, stream

FP8_MAX = 448.0
BLOCK = 128
MAX_GROUPS = 1024
_CODES = torch.float8_e4m3fn


def sf_bytes(rows: int, K: int) -> int:
    """Size of the scale-factor buffer of a [rows, K] operand with blocks along K."""
    return int(lib().ls_fp8_sf_bytes(rows, K))


def slots(rows: int, groups: int) -> int:
    """Row tiles of 128 that a tensor of `rows` rows in `groups` ragged groups may take (see ls_fp8_slots)."""
    return int(lib().ls_fp8_slots(rows, groups))


def _input(x, dims=2):
    if x.dim() != dims:
        raise ValueError(f"expected a {dims}-dimensional tensor, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        x = x.float()
    return aligned(x)


def _codes(lead, rows, K, device):
    pitch = -(-K // 16) * 16
    return torch.empty((*lead, rows, pitch), dtype=_CODES, device=device)[..., :K]


def _pitched(codes):
    """(codes, row pitch) as the products read them: rows 16-byte aligned, matrices back to back."""
    if codes.dtype == torch.uint8:
        codes = codes.view(_CODES)
    if codes.dtype != _CODES:
        raise TypeError(f"codes must be float8_e4m3fn (or their bytes), got {codes.dtype}")
    *lead, rows, K = codes.shape
    ld = codes.stride(-2) if rows > 1 else max(codes.stride(-2), -(-K // 16) * 16)
    if rows == 1 and ld % 16:
        ld = -(-K // 16) * 16
    ok = (K <= 1 or codes.stride(-1) == 1) and ld >= K and ld % 16 == 0 and codes.data_ptr() % 16 == 0
    if lead and lead[0] > 1:
        ok = ok and codes.stride(0) == rows * ld
    if not ok:
        fresh = _codes(lead, rows, K, codes.device)
        fresh.view(torch.uint8).copy_(codes.view(torch.uint8)) if codes.stride(-1) == 1 or K <= 1 else \
            fresh.view(torch.uint8).copy_(codes.contiguous().view(torch.uint8))
        codes, ld = fresh, fresh.stride(-2) if rows > 1 else -(-K // 16) * 16
    return codes, ld


def _groups(offsets, device):
    """(int32 offsets, number of groups)."""
    if offsets.dim() != 1 or offsets.numel() < 2 or offsets.numel() > MAX_GROUPS + 1:
        raise ValueError(f"offsets: groups + 1 values, 1 to {MAX_GROUPS} groups; got shape {tuple(offsets.shape)}")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    return offsets.to(torch.int32).contiguous(), offsets.numel() - 1


def _quantize_rows(x, offsets, want_scale, want_sf):
    with on_device_of(x, offsets):
        *lead, K = x.shape
        x = _input(x.reshape(-1, K) if x.dim() != 2 else x)
        rows = x.shape[0]
        off, G = (None, 0) if offsets is None else _groups(offsets, x.device)
        codes = _codes((), rows, K, x.device)
        scale = torch.empty((rows, -(-K // BLOCK)), dtype=torch.float32, device=x.device) if want_scale else None
        sf_rows = rows if off is None else BLOCK * slots(rows, G)
        sf = torch.empty(sf_bytes(sf_rows, K), dtype=torch.uint8, device=x.device) if want_sf else None
        check(lib().ls_quantize_fp8(ptr(x), _lib.dtype_code(x.dtype), rows, K, ptr(off), G, ptr(codes), -(-K // 16) * 16,
                                    ptr(scale), ptr(sf), stream()))
        if len(lead) != 1:
            codes = codes.view(*lead, K) if codes.is_contiguous() else codes.unflatten(0, lead)
            scale = None if scale is None else scale.view(*lead, -1)
        return codes, scale, sf


def quantize_fp8(x: torch.Tensor):
    """x [..., K] -> (codes [..., K], scale fp32 [..., ceil(K / 128)]), blocks along the last dim."""
    codes, scale, _ = _quantize_rows(x, None, True, False)
    return codes, scale


def quantize_fp8_packed(x: torch.Tensor, offsets: torch.Tensor = None):
    """x [..., K] -> (codes, sf): what the products take as their row operand.  With offsets
    (x two-dimensional), the codes keep x's row order and sf is in slot order."""
    if offsets is not None and x.dim() != 2:
        raise ValueError("a grouped tensor is two-dimensional")
    codes, _, sf = _quantize_rows(x, offsets, False, True)
    return codes, sf


def quantize_fp8_both(x: torch.Tensor, offsets: torch.Tensor = None, rows_too: bool = True):
    """x [rows, K] -> (codes, sf, codes_t, sf_t) from one read: blocks along the rows, and blocks of
    128 rows down the columns for a product that sums over rows.  codes_t has x's orientation; with
    offsets its rows are in slot order, zeros behind a group's last row.  rows_too=False leaves
    the first two out (None)."""
    with on_device_of(x, offsets):
        x = _input(x)
        rows, K = x.shape
        off, G = (None, 0) if offsets is None else _groups(offsets, x.device)
        sf_rows = rows if off is None else BLOCK * slots(rows, G)
        codes = _codes((), rows, K, x.device) if rows_too else None
        sf = torch.empty(sf_bytes(sf_rows, K), dtype=torch.uint8, device=x.device) if rows_too else None
        codes_t = _codes((), sf_rows, K, x.device)
        sf_t = torch.empty(sf_bytes(K, sf_rows), dtype=torch.uint8, device=x.device)
        check(lib().ls_quantize_fp8_both(ptr(x), _lib.dtype_code(x.dtype), rows, K, ptr(off), G, ptr(codes), ptr(sf),
                                         ptr(codes_t), ptr(sf_t), -(-K // 16) * 16, stream()))
        return codes, sf, codes_t, sf_t


def quantize_fp8_weight(w: torch.Tensor, want_scale: bool = False):
    """w [N, K] or [groups, N, K] -> (codes, sf, sf_t[, scale fp32 [..., N / 128, K / 128]]) with one
    scale per 128 x 128; sf serves products over K, sf_t (the transpose's) products over N."""
    with on_device_of(w):
        w = _input(w, w.dim() if w.dim() in (2, 3) else 2)
        *lead, N, K = w.shape
        G = lead[0] if lead else 1
        if G > MAX_GROUPS:
            raise ValueError(f"at most {MAX_GROUPS} matrices, got {G}")
        codes = _codes(lead, N, K, w.device)
        sf = torch.empty((*lead, sf_bytes(N, K)), dtype=torch.uint8, device=w.device)
        sf_t = torch.empty((*lead, sf_bytes(K, N)), dtype=torch.uint8, device=w.device)
        scale = torch.empty((*lead, -(-N // BLOCK), -(-K // BLOCK)), dtype=torch.float32, device=w.device) if want_scale else None
        check(lib().ls_quantize_fp8_weight(ptr(w), _lib.dtype_code(w.dtype), G, N, K, ptr(codes), -(-K // 16) * 16, ptr(scale),
                                           ptr(sf), ptr(sf_t), stream()))
        return (codes, sf, sf_t, scale) if want_scale else (codes, sf, sf_t)


def dequantize_fp8(codes: torch.Tensor, scale: torch.Tensor, out_dtype=torch.float32):
    """codes * scale.  scale [..., ceil(K / 128)] of quantize_fp8, or [..., N / 128, K / 128] of
    quantize_fp8_weight (told apart by its next-to-last size)."""
    with on_device_of(codes, scale):
        *lead, rows, K = codes.shape if codes.dim() > 1 else (1, *codes.shape)
        kb = -(-K // BLOCK)
        row_block = 1 if scale.shape == (*codes.shape[:-1], kb) else BLOCK
        if row_block == BLOCK and scale.shape != (*lead, -(-rows // BLOCK), kb):
            raise ValueError(f"scale shape {tuple(scale.shape)} does not fit codes {tuple(codes.shape)}")
        out = torch.empty(codes.shape, dtype=out_dtype, device=codes.device)
        scale = aligned(scale.float())
        if row_block == 1:
            codes, ld = _pitched(codes.reshape(-1, K))
            check(lib().ls_dequantize_fp8(ptr(codes), ld, ptr(scale), codes.shape[0], K, 1, ptr(out), _lib.dtype_code(out_dtype), stream()))
            return out
        for c, s, o in zip(codes.reshape(-1, rows, K), scale.reshape(-1, -(-rows // BLOCK), kb), out.view(-1, rows, K)):
            c, ld = _pitched(c)
            check(lib().ls_dequantize_fp8(ptr(c), ld, ptr(s), rows, K, BLOCK, ptr(o), _lib.dtype_code(out_dtype), stream()))
        return out


def scales_to_sf(scale: torch.Tensor, rows: int = None):
    """fp32 power-of-two scales -> sf bytes: [rows, K / 128], or with `rows` given one scale per
    128 x 128 ([..., rows / 128, K / 128], as a checkpoint may hold them).  A verification and
    loading helper in torch operations, not a fast path."""
    with on_device_of(scale):
        e = (scale.float().contiguous().view(torch.int32) >> 23).to(torch.uint8)
        if rows is not None:
            e = e.repeat_interleave(BLOCK, dim=-2)[..., :rows, :]
        *lead, n, kb = e.shape
        rt, kt = -(-n // BLOCK), -(-kb // 4)
        full = torch.zeros((*lead, rt * BLOCK, kt * 4), dtype=torch.uint8, device=e.device)
        full[..., :n, :kb] = e
        d = len(lead)
        full = full.view(*lead, rt, 4, 32, kt, 4).permute(*range(d), d, d + 3, d + 2, d + 1, d + 4)
        return full.reshape(*lead, -1)


# ---------------------------------------------------------------- products
_NT, _NN, _TN = 0, 1, 2


def _sf(sf, matrices, rows, K, what):
    want = matrices * sf_bytes(rows, K)
    if sf.dtype != torch.uint8 or sf.numel() != want:
        raise ValueError(f"{what}: a scale-factor buffer of {want} bytes is needed, got {sf.numel()} of {sf.dtype}")
    return aligned(sf)


def _product(form, a, b, a_sf, b_sf, out_dtype, out, offsets, rows):
    with on_device_of(a, b, a_sf, b_sf, offsets, out):
        if a.dim() != 2 or b.dim() != (2 if offsets is None or form == _TN else 3):
            raise ValueError(f"operand shapes {tuple(a.shape)} and {tuple(b.shape)}")
        off, G = (None, 1) if offsets is None else _groups(offsets, a.device)
        if form == _TN:
            held, M = a.shape
            N = b.shape[1]
            K = held if off is None else rows
            tiles = -(-held // BLOCK) * BLOCK if off is None else BLOCK * slots(K, G)
            if b.shape[0] != held or (off is not None and held != tiles):
                raise ValueError(f"operands with {a.shape[0]} and {b.shape[0]} rows"
                                 + ("" if off is None else f", {tiles} needed for {K} rows in {G} groups"))
            a_sf, b_sf = _sf(a_sf, 1, M, tiles, "a_sf"), _sf(b_sf, 1, N, tiles, "b_sf")
            shape = (M, N) if off is None else (G, M, N)
        else:
            M, K = a.shape
            N, Kb = b.shape[-2:] if form == _NT else b.shape[-1:-3:-1]
            if Kb != K or (off is not None and b.shape[0] != G):
                raise ValueError(f"operand shapes {tuple(a.shape)} and {tuple(b.shape)} do not fit" + ("" if off is None else f" {G} groups"))
            a_sf = _sf(a_sf, 1, M if off is None else BLOCK * slots(M, G), K, "a_sf")
            b_sf = _sf(b_sf, G, N, K, "b_sf")
            shape = (M, N)
        (a, lda), (b, ldb) = _pitched(a), _pitched(b)
        if out is None:
            c = torch.empty(shape, dtype=out_dtype, device=a.device)
        else:
            if out.shape != shape or out.dtype != out_dtype or not out.is_contiguous() or out.data_ptr() % 16:
                raise ValueError(f"out must be a contiguous, 16-byte aligned {tuple(shape)} tensor of {out_dtype}")
            c = out
        args = (form, ptr(a), lda, ptr(b), ldb, ptr(a_sf), ptr(b_sf), ptr(c), _lib.dtype_code(out_dtype), M, N, K)
        if off is None:
            check(lib().ls_fp8_gemm(*args, stream()))
        else:
            check(lib().ls_fp8_gemm_grouped(*args, ptr(off), G, 1 if out is None else 0, stream()))
        return c


def fp8_gemm(a, b, a_sf, b_sf, out_dtype=torch.bfloat16, out=None):
    """C = A @ B.T: a [M, K] and b [N, K] codes with their sf; the forward product.  bf16 or fp32."""
    return _product(_NT, a, b, a_sf, b_sf, out_dtype, out, None, None)


def fp8_gemm_nn(a, b, a_sf, b_sf_t, out_dtype=torch.bfloat16, out=None):
    """C = A @ B: a [M, K] codes, b [K, N] codes of quantize_fp8_weight and its sf_t; the input gradient."""
    return _product(_NN, a, b, a_sf, b_sf_t, out_dtype, out, None, None)


def fp8_gemm_tn(a_t, b_t, a_sf_t, b_sf_t, out_dtype=torch.float32, out=None):
    """C = A.T @ B over the rows of a_t [rows, M] and b_t [rows, N], the column-wise forms of
    quantize_fp8_both; the weight gradient."""
    return _product(_TN, a_t, b_t, a_sf_t, b_sf_t, out_dtype, out, None, None)


def fp8_gemm_grouped(a, b, a_sf, b_sf, offsets, out_dtype=torch.bfloat16, out=None):
    """C[r] = A[r] @ B[g].T for the rows r of every group g: a [rows, K], b [groups, N, K].  Rows of
    no group are zeros, or with `out` left as they were."""
    return _product(_NT, a, b, a_sf, b_sf, out_dtype, out, offsets, None)


def fp8_gemm_grouped_nn(a, b, a_sf, b_sf_t, offsets, out_dtype=torch.bfloat16, out=None):
    """C[r] = A[r] @ B[g]: a [rows, K], b [groups, K, N] with its sf_t."""
    return _product(_NN, a, b, a_sf, b_sf_t, out_dtype, out, offsets, None)


def fp8_gemm_grouped_tn(a_t, b_t, a_sf_t, b_sf_t, offsets, rows, out_dtype=torch.float32, out=None):
    """C[g] = A[rows of g].T @ B[rows of g]: the column-wise forms of two tensors with `rows` rows
    quantized with these offsets.  [groups, M, N]; zeros for an empty group."""
    return _product(_TN, a_t, b_t, a_sf_t, b_sf_t, out_dtype, out, offsets, rows)
