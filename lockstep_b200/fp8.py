"""(extension) FP8 values with one power-of-two scale per block of 128: quantizers and products.

lockstep's codec and products are 4-bit; this module is the 8-bit step above them for layers
and gradients that do not survive E2M1.  Codes are E4M3.  A block is 128 values along the axis a
product sums over, and 128 x 128 for weights (so that a weight and its transpose have the same
codes); its scale is the smallest power of two s with max|x| <= 448 s, at least 2^-126, and 1
for a block of zeros.  The scales being powers of two, division by them is exact and the tensor
cores apply them (`tcgen05.mma.kind::mxf8f6f4.block_scale`).  The maximum runs over the finite
values; infinities and NaNs become E4M3's NaN.

Sizes are free: a ragged end is a short block.  Codes are float8_e4m3fn tensors; the quantizers lay
rows out at a pitch of whole 128-byte lines (a view of a wider buffer where the row length is none),
the products take any pitch that is a multiple of 16 bytes and copy others.  `sf` buffers hold the
scale bytes in the tensor-core layout of fp4.py.

Ragged groups (rows sorted by expert): `offsets` is a CUDA tensor of groups + 1 integers, rows
offsets[g] .. offsets[g + 1] belong to group g.  Nothing reads it on the host.  Groups may be
empty; rows behind offsets[-1] belong to nobody.  A tensor quantized with offsets goes to the
grouped products with the same offsets.
"""

import torch

from . import _lib
from ._lib import check, lib, on_device_of

FP8_MAX = 448.0
BLOCK = 128
MAX_GROUPS = 1024
_CODES = torch.float8_e4m3fn


# Serving calls take microseconds, and so do the host's own steps: pointers go to ctypes as plain
# integers, and sizes are computed here.
def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream if _raw_stream is None else _raw_stream(t.get_device())


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_DTYPE = {torch.float32: _lib.LS_F32, torch.bfloat16: _lib.LS_BF16}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _aligned(t):
    return t if t.is_contiguous() and t.data_ptr() % 32 == 0 else _lib.aligned(t, 32)


def _out_code(dtype):
    code = _DTYPE.get(dtype)
    return _lib.dtype_code(dtype) if code is None else code       # raises for the others


def sf_bytes(rows: int, K: int) -> int:
    """Size of the scale-factor buffer of a [rows, K] operand with blocks along K."""
    return ((rows + 127) // 128) * ((K + 511) // 512) * 512


def slots(rows: int, groups: int) -> int:
    """Row tiles of 128 that a tensor of `rows` rows in `groups` ragged groups may take (see ls_fp8_slots)."""
    return rows // 128 + groups


def _input(x, dims=2):
    if x.dim() != dims:
        raise AssertionError(f"expected a {dims}-dimensional tensor, got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPE:
        x = x.float()
    return _aligned(x)


def _pitch(K):
    # whole 128-byte lines: rows that start inside one cost a tensor copy twice the traffic (a weight
    # gradient of 4999 rows: 22.5 us at a pitch of 2064 and 1008 bytes, 12.6 at 2048 and 1024)
    return (K + 127) // 128 * 128


def _codes(lead, rows, K, device):
    if K % 128 == 0:
        return torch.empty((*lead, rows, K), dtype=_CODES, device=device)
    return torch.empty((*lead, rows, _pitch(K)), dtype=_CODES, device=device)[..., :K]


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _pitched(codes):
    """(codes, row pitch) as the products read them: rows 16-byte aligned, matrices back to back."""
    if codes.dtype is _CODES and codes.is_contiguous() and codes.shape[-1] % 16 == 0 and codes.data_ptr() % 16 == 0:
        return codes, codes.shape[-1]
    if codes.dtype != _CODES:
        if codes.dtype != torch.uint8:
            raise TypeError(f"codes must be float8_e4m3fn (or their bytes), got {codes.dtype}")
        codes = codes.view(_CODES)
    rows, K = codes.shape[-2:]
    ld = codes.stride(-2)
    if rows == 1 and (ld < K or ld % 16):                     # the pitch of a single row is free
        ld = _pitch(K) if codes.dim() == 2 else 0
    if (codes.stride(-1) == 1 or K <= 1) and ld >= K and ld % 16 == 0 and codes.data_ptr() % 16 == 0 and \
            (codes.dim() == 2 or codes.shape[0] <= 1 or codes.stride(0) == rows * ld) and \
            (ld == K or codes.untyped_storage().nbytes() >= codes.storage_offset() + codes.numel() // K * ld):
        return codes, ld
    # (the last test: the products may read the padding of the last row)
    fresh = _codes(codes.shape[:-2], rows, K, codes.device)
    fresh.view(torch.uint8).copy_(codes.view(torch.uint8))
    return fresh, _pitch(K)


def _groups(offsets):
    """(int32 offsets, number of groups)."""
    if offsets is None:
        return None, 0
    if offsets.dim() != 1 or not 2 <= offsets.shape[0] <= MAX_GROUPS + 1:
        raise AssertionError(f"offsets: groups + 1 values, 1 to {MAX_GROUPS} groups; got shape {tuple(offsets.shape)}")
    if offsets.dtype != torch.int32:
        if offsets.dtype != torch.int64:
            raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
        offsets = offsets.to(torch.int32)
    return offsets.contiguous(), offsets.shape[0] - 1


def _quantize_rows(x, offsets, want_scale, want_sf):
    with on_device_of(x, offsets):
        shape = x.shape
        K = shape[-1]
        x = _input(x if len(shape) == 2 else x.reshape(-1, K))
        rows, dev = x.shape[0], x.device
        off, G = _groups(offsets)
        codes = _codes((), rows, K, dev)
        scale = torch.empty((rows, -(-K // BLOCK)), dtype=torch.float32, device=dev) if want_scale else None
        sf = _bytes(sf_bytes(rows if off is None else BLOCK * slots(rows, G), K), dev) if want_sf else None
        check(lib().ls_quantize_fp8(x.data_ptr(), _DTYPE[x.dtype], rows, K, _ptr(off), G, codes.data_ptr(), _pitch(K),
                                    _ptr(scale), _ptr(sf), _stream(x)))
        if len(shape) != 2:
            codes = codes.view(shape) if codes.is_contiguous() else codes.unflatten(0, shape[:-1]) if len(shape) > 2 else codes[0]
            scale = None if scale is None else scale.view(*shape[:-1], -1)
        return codes, scale, sf


def quantize_fp8(x: torch.Tensor):
    """x [..., K] -> (codes [..., K], scale fp32 [..., ceil(K / 128)]), blocks along the last dim."""
    codes, scale, _ = _quantize_rows(x, None, True, False)
    return codes, scale


def quantize_fp8_packed(x: torch.Tensor, offsets: torch.Tensor = None):
    """x [..., K] -> (codes, sf): what the products take as their row operand.  With offsets
    (x two-dimensional), the codes keep x's row order and sf is in slot order."""
    if offsets is not None and x.dim() != 2:
        raise AssertionError("a grouped tensor is two-dimensional")
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
        dev = x.device
        off, G = _groups(offsets)
        sf_rows = rows if off is None else BLOCK * slots(rows, G)
        codes = _codes((), rows, K, dev) if rows_too else None
        sf = _bytes(sf_bytes(sf_rows, K), dev) if rows_too else None
        codes_t = _codes((), sf_rows, K, dev)
        sf_t = _bytes(sf_bytes(K, sf_rows), dev)
        check(lib().ls_quantize_fp8_both(x.data_ptr(), _DTYPE[x.dtype], rows, K, _ptr(off), G, _ptr(codes), _ptr(sf),
                                         codes_t.data_ptr(), sf_t.data_ptr(), _pitch(K), _stream(x)))
        return codes, sf, codes_t, sf_t


def quantize_fp8_weight(w: torch.Tensor, want_scale: bool = False):
    """w [N, K] or [groups, N, K] -> (codes, sf, sf_t[, scale fp32 [..., N / 128, K / 128]]) with one
    scale per 128 x 128; sf serves products over K, sf_t (the transpose's) products over N."""
    with on_device_of(w):
        w = _input(w, 3 if w.dim() == 3 else 2)
        *lead, N, K = w.shape
        G, dev = lead[0] if lead else 1, w.device
        if G > MAX_GROUPS:
            raise AssertionError(f"at most {MAX_GROUPS} matrices, got {G}")
        codes = _codes(lead, N, K, dev)
        sf, sf_t = _bytes((*lead, sf_bytes(N, K)), dev), _bytes((*lead, sf_bytes(K, N)), dev)
        scale = torch.empty((*lead, -(-N // BLOCK), -(-K // BLOCK)), dtype=torch.float32, device=dev) if want_scale else None
        check(lib().ls_quantize_fp8_weight(w.data_ptr(), _DTYPE[w.dtype], G, N, K, codes.data_ptr(), _pitch(K), _ptr(scale),
                                           sf.data_ptr(), sf_t.data_ptr(), _stream(w)))
        return (codes, sf, sf_t, scale) if want_scale else (codes, sf, sf_t)


def dequantize_fp8(codes: torch.Tensor, scale: torch.Tensor, out_dtype=torch.float32):
    """codes * scale.  scale [..., ceil(K / 128)] of quantize_fp8, or [..., N / 128, K / 128] of
    quantize_fp8_weight (told apart by its next-to-last size)."""
    with on_device_of(codes, scale):
        *lead, rows, K = codes.shape if codes.dim() > 1 else (1, *codes.shape)
        kb = -(-K // BLOCK)
        row_block = 1 if scale.shape == (*codes.shape[:-1], kb) else BLOCK
        if row_block == BLOCK and scale.shape != (*lead, -(-rows // BLOCK), kb):
            raise AssertionError(f"scale shape {tuple(scale.shape)} does not fit codes {tuple(codes.shape)}")
        out = torch.empty(codes.shape, dtype=out_dtype, device=codes.device)
        scale = _aligned(scale.float())

        def one(c, s, o):
            c, ld = _pitched(c)
            check(lib().ls_dequantize_fp8(c.data_ptr(), ld, s.data_ptr(), *c.shape, row_block, o.data_ptr(), _out_code(out_dtype), _stream(o)))
        if row_block == 1:
            one(codes.reshape(-1, K), scale, out)
        else:
            for c, s, o in zip(codes.reshape(-1, rows, K), scale.reshape(-1, -(-rows // BLOCK), kb), out.view(-1, rows, K)):
                one(c, s, o)
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


def _sf(sf, want, what):
    if sf.dtype != torch.uint8 or sf.numel() != want:
        raise AssertionError(f"{what}: a scale-factor buffer of {want} bytes is needed, got {sf.numel()} of {sf.dtype}")
    return _aligned(sf)


def _given(out, shape, dtype):
    if out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise AssertionError(f"out must be a contiguous, 16-byte aligned {tuple(shape)} tensor of {dtype}")
    return out


def _product(form, a, b, a_sf, b_sf, out_dtype, out, offsets, rows):
    with on_device_of(a, b, a_sf, b_sf, offsets, out):
        if a.dim() != 2 or b.dim() != (2 if offsets is None or form == _TN else 3):
            raise AssertionError(f"operand shapes {tuple(a.shape)} and {tuple(b.shape)}")
        off, G = _groups(offsets) if offsets is not None else (None, 1)
        if form == _TN:
            held, M = a.shape
            N = b.shape[1]
            K = held if off is None else rows
            tiles = -(-held // BLOCK) * BLOCK if off is None else BLOCK * slots(K, G)
            if b.shape[0] != held or (off is not None and held != tiles):
                raise AssertionError(f"operands with {a.shape[0]} and {b.shape[0]} rows"
                                 + ("" if off is None else f", {tiles} needed for {K} rows in {G} groups"))
            a_sf, b_sf = _sf(a_sf, sf_bytes(M, tiles), "a_sf"), _sf(b_sf, sf_bytes(N, tiles), "b_sf")
            shape = (M, N) if off is None else (G, M, N)
        else:
            M, K = a.shape
            N, Kb = b.shape[-2:] if form == _NT else b.shape[-1:-3:-1]
            if Kb != K or (off is not None and b.shape[0] != G):
                raise AssertionError(f"operand shapes {tuple(a.shape)} and {tuple(b.shape)} do not fit" + ("" if off is None else f" {G} groups"))
            a_sf = _sf(a_sf, sf_bytes(M if off is None else BLOCK * slots(M, G), K), "a_sf")
            b_sf = _sf(b_sf, G * sf_bytes(N, K), "b_sf")
            shape = (M, N)
        (a, lda), (b, ldb) = _pitched(a), _pitched(b)
        code = _out_code(out_dtype)
        c = torch.empty(shape, dtype=out_dtype, device=a.device) if out is None else _given(out, shape, out_dtype)
        if off is None:
            check(lib().ls_fp8_gemm(form, a.data_ptr(), lda, b.data_ptr(), ldb, a_sf.data_ptr(), b_sf.data_ptr(), c.data_ptr(), code,
                                    M, N, K, _stream(a)))
        else:
            check(lib().ls_fp8_gemm_grouped(form, a.data_ptr(), lda, b.data_ptr(), ldb, a_sf.data_ptr(), b_sf.data_ptr(), c.data_ptr(),
                                            code, M, N, K, off.data_ptr(), G, 1 if out is None else 0, _stream(a)))
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
