"""The FP8 operators' cases: linear layers whose products run on E4M3 values with one power-of-two scale per
block of 128, dense and grouped by expert, for serving (weights quantized once) and for training (forward, input
gradient and weight gradient), and the quantizer alone.

Definition.  A block's scale is the smallest power of two s with max|x| <= 448 s over its finite values, at least
2^-126, and 1 for a block of zeros; its codes are x / s rounded to E4M3 (ties to even).  Activations and gradients
have blocks of 128 values along the axis that the product sums over, weights blocks of 128 x 128; a ragged end is a
short block.
    y  = deq(q_K(x)) deq(q(w))^T            x [T, K], w [N, K]
    gx = deq(q_N(gy)) deq(q(w))
    gw = deq(q_T(gy))^T deq(q_T(x))
Grouped: rows offsets[g] .. offsets[g + 1] of x belong to expert g and its weight w[g]; q_T's blocks start at each
group's first row; rows behind offsets[G] belong to nobody and come out as zeros.
"""

import math

import torch

own = False

BLOCK = 128
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one token through a square projection: latency and the weight stream
        {"name": "linear_one_token", "kind": "linear", "T": 1, "K": 4096, "N": 4096, "dtype": "bf16"},
        # a small decode batch against a weight larger than the L2 cache
        {"name": "linear_decode_16", "kind": "linear", "T": 16, "K": 16384, "N": 16384, "dtype": "bf16"},
        # no size a multiple of anything, fp32 in and out
        {"name": "linear_odd_f32", "kind": "linear", "T": 333, "K": 1000, "N": 1111, "dtype": "f32"},
        # prefill or evaluation: two batches of 4096 rows against one square weight
        {"name": "linear_prefill", "kind": "linear", "T": 8192, "K": 8192, "N": 8192, "dtype": "bf16"},
        # the feed-forward input projection of the training harness (width 1024, 16 x 1024 tokens), fp32 master weights
        {"name": "train_ffn", "kind": "train", "T": 16384, "K": 1024, "N": 4096, "dtype": "bf16", "wdtype": "f32"},
        # a training step on a ragged batch with bf16 weights
        {"name": "train_odd", "kind": "train", "T": 4999, "K": 1000, "N": 2050, "dtype": "bf16", "wdtype": "bf16"},
        # the quantizer alone: a large activation, and a ragged fp32 tensor
        {"name": "quantize_rows", "kind": "quantize", "T": 16384, "K": 4096, "dtype": "bf16"},
        {"name": "quantize_odd_f32", "kind": "quantize", "T": 5003, "K": 1111, "dtype": "f32"},
        # decode through 32 experts, most of them empty
        {"name": "grouped_decode", "kind": "grouped", "T": 16, "K": 1024, "N": 4096, "G": 32, "skew": 0.0, "tail": 0, "dtype": "bf16"},
        # ragged groups, odd sizes, rows behind the last group (a padded batch)
        {"name": "grouped_odd", "kind": "grouped", "T": 3001, "K": 1016, "N": 1111, "G": 13, "skew": 1.0, "tail": 57, "dtype": "f32"},
        # prefill through 16 experts
        {"name": "grouped_prefill", "kind": "grouped", "T": 16384, "K": 4096, "N": 4096, "G": 16, "skew": 0.5, "tail": 0, "dtype": "bf16"},
        # the training harness' feed-forward projection as 8 experts: forward and both gradients
        {"name": "grouped_train", "kind": "grouped_train", "T": 16384, "K": 1024, "N": 4096, "G": 8, "skew": 0.5, "tail": 0,
         "dtype": "bf16", "wdtype": "f32"},
    ]


def draw(rng):
    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        step = rng.choice([1, 8, 16, 128])
        return max(lo, min(hi, n if n < step else n // step * step))

    kind = rng.choice(["linear", "linear", "train", "quantize", "grouped", "grouped", "grouped_train"])
    case = {"kind": kind, "T": size(1, 16384), "K": size(64, 8192), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "quantize":
        return case
    case["N"] = size(64, 8192)
    if kind.startswith("grouped"):
        case |= {"G": rng.choice([1, 2, 5, 8, 13, 16, 32, 64]), "skew": rng.choice([0.0, 0.5, 1.0]),
                 "tail": rng.choice([0, 0, 1, 100])}
        case["K"], case["N"] = min(case["K"], 4096), min(case["N"], 4096)
        case["T"] = max(case["T"], case["tail"] + 1)                  # at least one row belongs to a group
    if kind.endswith("train"):
        case["wdtype"] = rng.choice(["f32", "bf16"])
        case["T"] = max(case["T"], 128)
    while work(case)["flops"] > 1.0e12:                               # no more than linear_prefill
        case["T"] = max(case["T"] // 2, case.get("tail", 0) + 1)
    return case


# ---------------------------------------------------------------- inputs
def _sizes(case, seed):
    """Rows of each expert: a softmax of normal logits (skew 0: uniform routing), the rest by lot."""
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    rows = case["T"] - case["tail"]
    p = torch.softmax(case["skew"] * torch.randn(case["G"], generator=g), 0).clamp_max(max(4.0 / case["G"], 1e-9))
    pick = torch.multinomial(p, max(rows, 1), replacement=True, generator=g)[:rows]
    return torch.bincount(pick, minlength=case["G"]).tolist()


def _pitched(codes):
    """The same values with rows that start on multiples of 16 bytes, as the quantizer lays them out."""
    *lead, N, K = codes.shape
    buf = torch.zeros(*lead, N, -(-K // 16) * 16, dtype=torch.uint8, device=codes.device)
    buf[..., :K] = codes.view(torch.uint8)
    return buf.view(torch.float8_e4m3fn)[..., :K]


def _tiled(exponents):
    """Scale bytes [..., rows, kb] in tiles of 128 rows x 4 blocks: row r of a tile at (r % 32) * 16 + (r / 32) * 4 + kb % 4."""
    *lead, rows, kb = exponents.shape
    rt, kt = -(-rows // 128), -(-kb // 4)
    full = torch.zeros(*lead, rt * 128, kt * 4, dtype=torch.uint8, device=exponents.device)
    full[..., :rows, :kb] = exponents
    n = len(lead)
    return full.view(*lead, rt, 4, 32, kt, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).contiguous().view(*lead, -1)


def prepare(case, seed):
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, K = case["T"], case["K"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    # activations: tokens of different magnitude and a few outlier channels
    x = normal(T, K) * torch.exp(0.5 * normal(T, 1))
    x = (x * torch.where(torch.rand(K, device="cuda", generator=g) < 0.01, 20.0, 1.0)).to(dt)
    state = {"kind": case["kind"], "x": x}
    if case["kind"] == "quantize":
        return state
    N = case["N"]
    lead = (case["G"],) if "G" in case else ()
    w = normal(*lead, N, K) * 0.02
    if "G" in case:
        sizes = _sizes(case, seed)
        state["offsets"] = torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
        state["most"] = max(sizes)
    if case["kind"].endswith("train"):
        state["x"].requires_grad_(True)
        state["w"] = w.to(_DTYPES[case["wdtype"]]).requires_grad_(True)
        # gradients are small and heavy-tailed
        state["gy"] = (1e-3 * normal(T, N) * torch.exp(normal(T, 1))).to(dt)
        return state
    # a serving program keeps its weights quantized: E4M3 values, the scales, and the scales in the products' layout
    codes, scale = _quantize_weight(w)
    state["codes"] = _pitched(codes)
    state["scale"] = scale
    exponents = (torch.log2(scale) + 127).to(torch.uint8)
    state["sf"] = _tiled(exponents.repeat_interleave(BLOCK, dim=-2)[..., :N, :])
    return state


# ---------------------------------------------------------------- plain form, 32 bits
def _scale(amax):
    """Smallest power of two s with amax <= 448 s, at least 2^-126; 1 for zeros."""
    mantissa, exponent = torch.frexp(amax)                            # amax = mantissa 2^exponent, 0.5 <= mantissa < 1
    e = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)          # 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(amax), e.clamp_min(-126))
    return torch.where(amax > 0, s, torch.ones_like(s))


def _blocks(x, dim):
    """x in fp32 with axis `dim` padded to whole blocks and split in two: [..., blocks, 128, ...]."""
    n = x.shape[dim]
    nb = max(1, -(-n // BLOCK))
    pad = [0] * (2 * x.dim())
    pad[2 * (x.dim() - 1 - (dim % x.dim())) + 1] = nb * BLOCK - n
    x = torch.nn.functional.pad(x.float(), pad)
    dim = dim % x.dim()
    return x.view(*x.shape[:dim], nb, BLOCK, *x.shape[dim + 1:])


def _quantize(x, dim):
    """(E4M3 codes shaped as x, scales with one value per block of 128 along `dim`)."""
    dim = dim % x.dim()
    b = _blocks(x, dim)
    s = _scale(b.abs().amax(dim + 1))
    q = (b / s.unsqueeze(dim + 1)).to(torch.float8_e4m3fn).view(torch.uint8)
    q = q.flatten(dim, dim + 1).narrow(dim, 0, x.shape[dim]).contiguous().view(torch.float8_e4m3fn)
    return q, s


def _quantize_weight(w):
    """(codes shaped as w, scales [..., N / 128, K / 128])."""
    b = _blocks(_blocks(w, -1), -3)                                   # [..., nb, 128, kb, 128]
    s = _scale(b.abs().amax((-3, -1)))
    q = (b / s[..., :, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    q = q.flatten(-2, -1).flatten(-3, -2)[..., :w.shape[-2], :w.shape[-1]].contiguous().view(torch.float8_e4m3fn)
    return q, s


def _values(codes, scale, *dims):
    """codes * scale with the scales repeated over their blocks along `dims`."""
    for d in dims:
        scale = scale.repeat_interleave(BLOCK, dim=d).narrow(d, 0, codes.shape[d])
    return codes.float() * scale


def _fq(x, dim):
    return _values(*_quantize(x, dim), dim)


def _fq_weight(w):
    return _values(*_quantize_weight(w), -2, -1)


def _places(offsets, T):
    """For every row its group, its place in the group, and whether it has one."""
    at = torch.arange(T, device=offsets.device)
    group = torch.searchsorted(offsets.long(), at, right=True) - 1
    inside = group < offsets.numel() - 1
    group = torch.where(inside, group, torch.zeros_like(group))
    return group, at - offsets.long()[group], inside


def _spread(x, places, G, rows):
    """Rows of x [T, D] in fp32 laid out as [G, rows, D], zeros elsewhere."""
    group, at, inside = places
    out = torch.zeros(G, rows, x.shape[1], dtype=torch.float32, device=x.device)
    out[group[inside], at[inside]] = x.float()[inside]
    return out


def _collect(y, places):
    group, at, inside = places
    at = torch.where(inside, at, torch.zeros_like(at))
    return torch.where(inside[:, None], y[group, at], torch.zeros((), device=y.device))


def run(state):
    kind, x = state["kind"], state["x"]
    if own:
        from lockstep_b200 import fp8, fp8_linear
        if kind == "quantize":
            return fp8.quantize_fp8(x)
        if kind == "linear":
            return fp8_linear.linear_quantized(x, state["codes"], state["sf"])
        if kind == "grouped":
            return fp8_linear.grouped_linear_quantized(x, state["codes"], state["sf"], state["offsets"])
        if kind == "train":
            y = fp8_linear.linear(x, state["w"])
        else:
            y = fp8_linear.grouped_linear(x, state["w"], state["offsets"])
        return (y.detach(), *torch.autograd.grad(y, (x, state["w"]), state["gy"]))
    with torch.no_grad():
        if kind == "quantize":
            return _quantize(x, -1)
        if kind == "linear":
            return (_fq(x, -1) @ _values(state["codes"], state["scale"], -2, -1).t()).to(x.dtype)
        if kind == "train":
            w, gy = state["w"], state["gy"]
            wq = _fq_weight(w)
            return ((_fq(x, -1) @ wq.t()).to(x.dtype), (_fq(gy, -1) @ wq).to(x.dtype),
                    (_fq(gy, 0).t() @ _fq(x, 0)).to(w.dtype))
        T, rows = x.shape[0], max(1, state["most"])
        places = _places(state["offsets"], T)
        if kind == "grouped":
            w = _values(state["codes"], state["scale"], -2, -1)
            return _collect(torch.bmm(_spread(_fq(x, -1), places, w.shape[0], rows), w.transpose(1, 2)), places).to(x.dtype)
        w, gy = state["w"], state["gy"]
        G, wq = w.shape[0], _fq_weight(w)
        y = _collect(torch.bmm(_spread(_fq(x, -1), places, G, rows), wq.transpose(1, 2)), places)
        gx = _collect(torch.bmm(_spread(_fq(gy, -1), places, G, rows), wq), places)
        gw = torch.bmm(_fq(_spread(gy, places, G, rows), 1).transpose(1, 2), _fq(_spread(x, places, G, rows), 1))
        return y.to(x.dtype), gx.to(x.dtype), gw.to(w.dtype)


# ---------------------------------------------------------------- floor
def work(case):
    T, K, N = case["T"], case["K"], case.get("N", 0)
    xb = 2 if case["dtype"] == "bf16" else 4
    scales = lambda n: -(-n // BLOCK)
    if case["kind"] == "quantize":
        return {"bytes": T * K * (xb + 1) + 4 * T * scales(K), "flops": 2 * T * K}
    G = case.get("G", 1)
    rows = T - case.get("tail", 0)
    if case["kind"].endswith("train"):
        wb = 2 if case["wdtype"] == "bf16" else 4
        return {"bytes": 2 * T * K * xb + 2 * T * N * xb + 2 * G * N * K * wb, "flops": 6 * rows * N * K}
    live = min(G, rows) if G > 1 else 1                               # experts whose weights are read, at most
    return {"bytes": T * K * xb + T * N * xb + live * (N * K + N * scales(K)), "flops": 2 * rows * N * K}


# ---------------------------------------------------------------- 64 bits, from the definition
def _e4m3(q):
    """Nearest E4M3 value of a double with |q| <= 448, ties to even: 3 fraction bits, exponents from -6."""
    e = torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(q / step) * step


def _pow2_scale(amax):
    e = torch.ceil(torch.log2(amax / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e)      # log2's rounding next to a power of two
    e = torch.where(448.0 * torch.exp2(e) < amax, e + 1, e)
    return torch.where(amax > 0, torch.exp2(e.clamp_min(-126)), torch.ones_like(amax))


def _rounded64(x, *spans):
    """x in doubles, quantized and put back, one scale per block of spans[i] along axis i (1: each index its own)."""
    x = x.double()
    shape = x.shape
    whole = [-(-n // s) * s for n, s in zip(shape, spans)]
    out = torch.zeros(whole, dtype=torch.float64, device=x.device)
    out[tuple(slice(0, n) for n in shape)] = x
    split = [v for n, s in zip(whole, spans) for v in (n // s, s)]
    b = out.view(split)
    s = _pow2_scale(b.abs().amax(tuple(range(1, 2 * len(spans), 2)), keepdim=True))
    v = (_e4m3(b / s) * s).reshape(whole)
    return v[tuple(slice(0, n) for n in shape)], s


def exact(case, seed):
    state = prepare(case, seed)
    kind, x = state["kind"], state["x"].detach()
    if kind == "quantize":
        v, s = _rounded64(x, 1, BLOCK)
        s = s.reshape(x.shape[0], -1)
        return v / s.repeat_interleave(BLOCK, 1)[:, :x.shape[1]], s
    xk = _rounded64(x, 1, BLOCK)[0]
    if kind == "linear":
        s = state["scale"].double().repeat_interleave(BLOCK, 0)[:case["N"]].repeat_interleave(BLOCK, 1)[:, :case["K"]]
        return xk @ (state["codes"].to(torch.float64) * s).t()
    if kind == "train":
        w, gy = state["w"].detach(), state["gy"]
        wq = _rounded64(w, BLOCK, BLOCK)[0]
        return (xk @ wq.t(), _rounded64(gy, 1, BLOCK)[0] @ wq,
                _rounded64(gy, BLOCK, 1)[0].t() @ _rounded64(x, BLOCK, 1)[0])
    off = state["offsets"].tolist()
    y = torch.zeros(case["T"], case["N"], dtype=torch.float64, device=x.device)
    if kind == "grouped":
        for g, (lo, hi) in enumerate(zip(off, off[1:])):
            s = state["scale"][g].double().repeat_interleave(BLOCK, 0)[:case["N"]].repeat_interleave(BLOCK, 1)[:, :case["K"]]
            y[lo:hi] = xk[lo:hi] @ (state["codes"][g].to(torch.float64) * s).t()
        return y
    w, gy = state["w"].detach(), state["gy"]
    gx = torch.zeros(case["T"], case["K"], dtype=torch.float64, device=x.device)
    gw = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for g, (lo, hi) in enumerate(zip(off, off[1:])):
        if hi > lo:
            wq = _rounded64(w[g], BLOCK, BLOCK)[0]
            y[lo:hi] = xk[lo:hi] @ wq.t()
            gx[lo:hi] = _rounded64(gy[lo:hi], 1, BLOCK)[0] @ wq
            gw[g] = _rounded64(gy[lo:hi], BLOCK, 1)[0].t() @ _rounded64(x[lo:hi], BLOCK, 1)[0]
    return y, gx, gw
