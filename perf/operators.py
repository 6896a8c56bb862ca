"""Timed calls of the operators for mixtures of experts and for 4-bit weights.

A case is one call (or the two calls that belong together) at one size:

  * "grouped": products of ragged groups of tokens with their expert's weights
    (wgb_gemm_grouped), forward (weights stored out x in) and input gradient
    (the same weights read the other way);
  * "weight_grad": each expert's weight gradient from its own tokens
    (wgb_gemm_grouped_k);
  * "quantize": to MXFP4 (blocks of 32, a power of two each, E2M1 codes) and
    back (wgb_mxfp4_quantize, wgb_mxfp4_dequantize);
  * "mx_product": tokens quantised to MXFP4 and multiplied with MXFP4 weights,
    one matrix (wgb_mxfp4_gemm) or one per expert (wgb_mxfp4_gemm_grouped).

Tensors are row-major here, which is the library's column-major frame read the
other way: a tensor of shape (n, ld) is a matrix of n columns.
"""
import math

import torch

own = False  # False: the plain form in torch; True: the library's kernels

F32, F16, BF16 = "f32", "f16", "bf16"
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
SIZE = {F32: 4, F16: 2, BF16: 2}


# ---- the cases -----------------------------------------------------------------


def listed():
    return [
        # One decoding step of 64 token-expert pairs over 64 experts: each active expert's weights are read for
        # about one token.
        {"name": "grouped_tokens", "op": "grouped", "t": BF16, "ot": BF16, "groups": 64, "m": 2048, "n": 64, "k": 1024, "trans": 1, "pad": 0, "skew": 0.0},
        # The forward product of a training batch of 16384 token-expert pairs over 16 experts.
        {"name": "grouped_forward", "op": "grouped", "t": BF16, "ot": BF16, "groups": 16, "m": 8192, "n": 16384, "k": 4096, "trans": 1, "pad": 0, "skew": 0.3},
        # The gradient of a layer's input: the same weights, contiguous along the output this time.
        {"name": "grouped_input_grad", "op": "grouped", "t": F16, "ot": F16, "groups": 8, "m": 2048, "n": 8192, "k": 4096, "trans": 0, "pad": 0, "skew": 0.3},
        # Single precision at odd sizes: what a user of sgemm has in hand.
        {"name": "grouped_odd_f32", "op": "grouped", "t": F32, "ot": F32, "groups": 5, "m": 1000, "n": 1537, "k": 777, "trans": 1, "pad": 0, "skew": 0.6},
        # The weight gradients of a training batch, kept in 32 bits for the optimizer.
        {"name": "weight_grad", "op": "weight_grad", "t": BF16, "ot": F32, "groups": 8, "m": 4096, "n": 8192, "k": 2048, "pad": 0, "skew": 0.3},
        # A small batch with uneven groups, most of them shorter than a tile.
        {"name": "weight_grad_small", "op": "weight_grad", "t": F16, "ot": F16, "groups": 12, "m": 1032, "n": 1111, "k": 520, "pad": 0, "skew": 1.0},
        # The activations of a few tokens to 4 bits and back: latency counts.
        {"name": "quantize_tokens", "op": "quantize", "t": BF16, "k": 4096, "n": 17, "trans": 0, "pad": 0},
        # A large weight matrix, quantised along its strided axis (the operand of the other product of training).
        {"name": "quantize_weights", "op": "quantize", "t": BF16, "k": 8192, "n": 16384, "trans": 1, "pad": 0},
        # One token through one layer of 4-bit weights.
        {"name": "mx_token", "op": "mx_product", "ot": BF16, "groups": 0, "m": 8192, "n": 1, "k": 4096, "skew": 0.0},
        # A prompt through one layer of 4-bit weights.
        {"name": "mx_prompt", "op": "mx_product", "ot": BF16, "groups": 0, "m": 8192, "n": 4096, "k": 8192, "skew": 0.0},
        # One decoding step over 4-bit experts.
        {"name": "mx_grouped_tokens", "op": "mx_product", "ot": BF16, "groups": 64, "m": 4096, "n": 96, "k": 2048, "skew": 0.3},
        # A batch of prompts over 4-bit experts.
        {"name": "mx_grouped_prompt", "op": "mx_product", "ot": BF16, "groups": 16, "m": 4096, "n": 16384, "k": 4096, "skew": 0.3},
    ]


def _log(rng, lo, hi, step=8):
    """A whole number from lo to hi, spread over the logarithm; three of four rounded to multiples of `step` where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.75 and v >= 2 * step:
        v = v // step * step
    v = max(lo, min(hi, v))
    return v + 8 if v == 3072 else v


def draw(rng):
    op = rng.choice(["grouped", "grouped", "weight_grad", "quantize", "mx_product", "mx_product"])
    if op == "quantize":
        return {"op": op, "t": rng.choice([F32, F16, BF16]), "k": _log(rng, 256, 8192), "n": _log(rng, 1, 16384),
                "trans": rng.randrange(2), "pad": rng.choice([0, 0, 1, 8])}
    c = {"op": op}
    if op != "mx_product":
        c["t"] = rng.choice([BF16, BF16, F16, F32])
    c["ot"] = F32 if c.get("t") == F32 else rng.choice([BF16, F32]) if c.get("t") == BF16 else F16 if "t" in c else rng.choice([BF16, F32])
    single = c.get("t") == F32
    c["groups"] = rng.choice([1, 3, 8, 16, 64])
    if op == "mx_product" and rng.random() < 0.4:
        c["groups"] = 0
    c.update(m=_log(rng, 256, 2048 if single else 8192), n=_log(rng, 1, 4096 if single else 16384), k=_log(rng, 256, 2048 if single else 4096))
    if op == "grouped":
        c["trans"] = rng.randrange(2)
    if op != "mx_product":
        c["pad"] = rng.choice([0, 0, 0, 1, 8])
    c["skew"] = rng.choice([0.0, 0.3, 1.0]) if c["groups"] > 1 else 0.0
    while max(1, c["groups"]) * c["m"] * c["k"] > 16 * 8192 * 4096 or _padded(c) > 3 * 16384 * 8192 * 4096:
        c["m"] = (c["m"] + 1) // 2
    return c


def _padded(c):
    """About the multiplications of the plain form, which pads every group to the longest."""
    return c["m"] * c["n"] * c["k"] * (1.0 + 3.0 * c["skew"])


def work(c):
    op = c["op"]
    if op == "quantize":
        n = c["n"] * c["k"]
        return {"bytes": 2 * n * (SIZE[c["t"]] + 17 / 32), "flops": 2 * n}
    m, n, k, groups = c["m"], c["n"], c["k"], max(1, c["groups"])
    # the weights of experts that get no token need not be read: of evenly drawn ones so many get some
    active = groups * (1.0 - (1.0 - 1.0 / groups) ** n)
    flops = 2 * m * n * k
    if op == "grouped":
        return {"bytes": (active * m * k + n * k) * SIZE[c["t"]] + n * m * SIZE[c["ot"]], "flops": flops}
    if op == "weight_grad":
        return {"bytes": n * (m + k) * SIZE[c["t"]] + groups * m * k * SIZE[c["ot"]], "flops": flops}
    return {"bytes": active * m * k * 17 / 32 + n * k * 2 + n * m * SIZE[c["ot"]], "flops": flops}


# ---- inputs ----------------------------------------------------------------------


def _sizes(c, seed):
    """Tokens of each expert: drawn with the unequal chances that a router gives them."""
    g = torch.Generator().manual_seed(int(seed) + 77)
    chance = torch.softmax(torch.randn(c["groups"], generator=g) * c["skew"], 0)
    return torch.bincount(torch.multinomial(chance, c["n"], replacement=True, generator=g), minlength=c["groups"])


def prepare(c, seed):
    s = {"case": dict(c)}
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = c["op"]

    def normal(*shape, scale=1.0, t=BF16, pad=0):
        full = shape[:-1] + (shape[-1] + pad,)
        return torch.empty(full, dtype=TORCH[t], device="cuda").normal_(0.0, scale, generator=g)

    if op == "quantize":
        k, n = c["k"], c["n"]
        s["X"] = normal(k, n, t=c["t"], pad=c["pad"]) if c["trans"] else normal(n, k, t=c["t"], pad=c["pad"])
        _room(s, "X", n, k)
        s["out"] = torch.empty(n, k, dtype=TORCH[c["t"]], device="cuda")
        torch.cuda.synchronize()
        return s
    m, n, k, groups = c["m"], c["n"], c["k"], c["groups"]
    if groups:
        sizes = _sizes(c, seed)
        s["longest"] = max(1, int(sizes.max()))
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).cuda()
    if op == "mx_product":
        s["X"] = normal(n, k)
        weights = normal(max(1, groups) * m, k, scale=k ** -0.5)
        s["codes"], s["scales"] = _pack(weights)
        _room(s, "X", n, k)
        s["C"] = torch.empty(n, m, dtype=TORCH[c["ot"]], device="cuda")
    elif op == "grouped":
        s["A"] = normal(groups, m, k, scale=k ** -0.5, t=c["t"], pad=c["pad"]) if c["trans"] else normal(
            groups, k, m, scale=k ** -0.5, t=c["t"], pad=c["pad"])
        s["B"] = normal(n, k, t=c["t"], pad=c["pad"])
        s["C"] = torch.empty(n, m, dtype=TORCH[c["ot"]], device="cuda")
    else:
        s["A"] = normal(n, m, t=c["t"], pad=c["pad"])
        s["B"] = normal(n, k, t=c["t"], pad=c["pad"])
        s["C"] = torch.empty(groups, k, m, dtype=TORCH[c["ot"]], device="cuda")
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    return s


def _stride(k):
    """Elements between the columns of a matrix in MXFP4: whole runs of 128."""
    return (k + 127) // 128 * 128


def _room(s, name, n, k):
    """Buffers for the quantised form of an operand, kept as a program keeps them."""
    ld = _stride(k)
    s[name + "_codes"] = torch.empty(n, ld // 2, dtype=torch.uint8, device="cuda")
    s[name + "_scales"] = torch.empty(n, ld // 32, dtype=torch.uint8, device="cuda")


# ---- the plain form ----------------------------------------------------------------


def _scaled(x):
    """Blocks of 32 of a matrix (rows x k) divided by their power of two, and its exponent."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    # frexp's mantissa is in [0.5, 1): floor(log2 amax) is its exponent less one
    e = torch.frexp(x.abs().amax(2))[1] - 3
    e = torch.where(x.abs().amax(2) == 0, -127, e.clamp(min=-127))
    return torch.ldexp(x, -e[:, :, None]), e


def _rounded(v):
    """To the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code."""
    step = 0.5 * (1.0 + (v.abs() >= 2).float() + 2.0 * (v.abs() >= 4).float())
    return ((v / step).round() * step).clamp(-6.0, 6.0)


def _values(x):
    """The values that the MXFP4 form of x stands for."""
    v, e = _scaled(x)
    return torch.ldexp(_rounded(v), e[:, :, None]).view(x.shape[0], -1)[:, : x.shape[1]]


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pack(x):
    """Codes (two a byte, the first in the low half) and scales, each column in whole runs of 128 elements."""
    rows, k = x.shape
    levels = torch.tensor(_LEVELS, device=x.device)
    codes = torch.zeros(rows, _stride(k) // 2, dtype=torch.uint8, device=x.device)
    scales = torch.zeros(rows, _stride(k) // 32, dtype=torch.uint8, device=x.device)
    v, e = _scaled(x)
    q = _rounded(v).view(rows, -1)
    q = (torch.searchsorted(levels, q.abs(), out_int32=True) + 8 * (q < 0)).to(torch.uint8)
    codes[:, : q.shape[1] // 2] = q[:, 0::2] + 16 * q[:, 1::2]
    scales[:, : e.shape[1]] = (e + 127).to(torch.uint8)
    return codes, scales


def _unpack(codes, scales, k):
    """The values of a packed matrix, in 32 bits."""
    levels = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=codes.device)
    q = torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1)
    v = levels[q.int()].view(codes.shape[0], -1, 32)
    return torch.ldexp(v, scales.int()[:, :, None] - 127).view(codes.shape[0], -1)[:, :k]


def _places(offsets, longest, n):
    """For each group its tokens' places, padded to the longest, and which of them are tokens of the group."""
    at = offsets[:-1, None] + torch.arange(longest, device=offsets.device)
    return at.clamp(max=n - 1), at < offsets[1:, None]


def _back(padded, offsets, n):
    """The tokens' rows of a padded product, in their own order."""
    token = torch.arange(n, device=offsets.device)
    group = torch.searchsorted(offsets[1:], token, right=True)
    return padded[group, token - offsets[group]]


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "quantize":
        x = s["X"][:, : c["n"]].t() if c["trans"] else s["X"][:, : c["k"]]
        return _values(x).to(TORCH[c["t"]])
    m, n, k = c["m"], c["n"], c["k"]
    dtype = TORCH[c["ot"]]
    if op == "weight_grad":
        at, valid = _places(s["offsets"], s["longest"], n)
        a = s["A"][:, :m].float()[at] * valid[:, :, None]
        b = s["B"][:, :k].float()[at]
        return torch.bmm(b.transpose(1, 2), a).to(dtype)
    if op == "mx_product":
        x = _values(s["X"])
        w = _unpack(s["codes"], s["scales"], k)
        if not c["groups"]:
            return (x @ w.t()).to(dtype)
        w = w.view(c["groups"], m, k).transpose(1, 2)
    else:
        x = s["B"][:, :k].float()
        w = s["A"][:, :, :k].float().transpose(1, 2) if c["trans"] else s["A"][:, :, :m].float()
    at, _ = _places(s["offsets"], s["longest"], n)
    return _back(torch.bmm(x[at], w), s["offsets"], n).to(dtype)


# ---- the library's form ------------------------------------------------------------

_ctx = None


def _context():
    """The device handle that a program opens once and keeps."""
    global _ctx
    if _ctx is None:
        import wgblas_amd

        _ctx = wgblas_amd.Context(0)
    return _ctx


def _kernels(s):
    import wgblas_amd as wg

    ctx, c, op = _context(), s["case"], s["case"]["op"]
    kind = {F32: wg.F32, F16: wg.F16, BF16: wg.BF16}

    def at(name):
        return s[name].data_ptr()

    if op == "quantize":
        k, n, ld = c["k"], c["n"], _stride(c["k"])
        ctx.mxfp4_quantize(kind[c["t"]], c["trans"], k, n, at("X"), s["X"].shape[1], at("X_codes"), at("X_scales"), ld)
        ctx.mxfp4_dequantize(kind[c["t"]], k, n, at("X_codes"), at("X_scales"), ld, at("out"), k)
        return s["out"]
    m, n, k, groups = c["m"], c["n"], c["k"], c["groups"]
    ot = kind[c["ot"]]
    if op == "grouped":
        lda = s["A"].shape[2]
        ctx.gemm_grouped(kind[c["t"]], c["trans"], groups, m, n, k, 1.0, at("A"), lda, s["A"].shape[1] * lda,
                         at("B"), s["B"].shape[1], at("offsets"), 0.0, at("C"), m, ot)
    elif op == "weight_grad":
        ctx.gemm_grouped_k(kind[c["t"]], groups, m, k, n, 1.0, at("A"), s["A"].shape[1], at("B"), s["B"].shape[1],
                           at("offsets"), 0.0, at("C"), m, m * k, ot)
    else:
        ld = _stride(k)
        ctx.mxfp4_quantize(wg.BF16, 0, k, n, at("X"), k, at("X_codes"), at("X_scales"), ld)
        if groups:
            ctx.mxfp4_gemm_grouped(groups, m, n, k, 1.0, at("codes"), at("scales"), ld, m * ld, at("X_codes"),
                                   at("X_scales"), ld, at("offsets"), 0.0, at("C"), m, ot)
        else:
            ctx.mxfp4_gemm(m, n, k, 1.0, at("codes"), at("scales"), ld, at("X_codes"), at("X_scales"), ld, 0.0,
                           at("C"), m, ot)
    return s["C"]


def run(s):
    return _kernels(s) if own else _plain(s)


# ---- the definition in 64 bits -----------------------------------------------------


def _exact_mx(x):
    """What the MXFP4 form of a matrix (rows x k) stands for: each block's power of two from its largest magnitude,
    each value to the nearest code by the thresholds between them, ties to the even code."""
    rows, k = x.shape
    x = x.double()
    full = torch.zeros(rows, (k + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    full[:, :k] = x
    blocks = full.view(rows, -1, 32)
    top = blocks.abs().amax(2, keepdim=True)
    scale = torch.exp2((torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 2.0).clamp(min=-127.0))
    v = (blocks / scale).abs()
    q = torch.zeros_like(v)
    for upper, level, low in ((0.25, 0.5, 0.0), (0.75, 1.0, 0.5), (1.25, 1.5, 1.0), (1.75, 2.0, 1.5), (2.5, 3.0, 2.0),
                              (3.5, 4.0, 3.0), (5.0, 6.0, 4.0)):
        # the upper neighbour also takes the tie where its code is the even one (1, 2 and 4)
        above = v >= upper if level in (1.0, 2.0, 4.0) else v > upper
        q = torch.where(above, level, q)
    return (torch.sign(blocks) * q * scale).view(rows, -1)[:, :k]


def _exact_unpacked(codes, scales, k):
    """The value of each code from its sign, exponent and mantissa bits."""
    rows = codes.shape[0]
    both = torch.empty(rows, codes.shape[1] * 2, dtype=torch.int64, device=codes.device)
    both[:, 0::2] = codes.long() % 16
    both[:, 1::2] = codes.long() // 16
    sign, e, half = 1 - 2 * (both // 8), (both // 2) % 4, both % 2
    v = sign * torch.where(e == 0, 0.5 * half, (1.0 + 0.5 * half) * torch.exp2((e - 1).double()))
    power = torch.exp2(scales.double() - 127.0).repeat_interleave(32, dim=1)
    return (v * power)[:, :k]


def exact(c, seed):
    s = prepare(c, seed)
    op = c["op"]
    if op == "quantize":
        return _exact_mx(s["X"][:, : c["n"]].t() if c["trans"] else s["X"][:, : c["k"]])
    m, n, k, groups = c["m"], c["n"], c["k"], c["groups"]
    if op == "mx_product":
        x = _exact_mx(s["X"])
        if not groups:
            return x @ _exact_unpacked(s["codes"], s["scales"], k).t()
    offsets = s["offsets"].tolist()
    out = torch.zeros((groups, k, m) if op == "weight_grad" else (n, m), dtype=torch.float64, device="cuda")
    for g in range(groups):
        lo, hi = offsets[g], offsets[g + 1]
        if lo == hi:
            continue
        if op == "weight_grad":
            out[g] = s["B"][lo:hi, :k].double().t() @ s["A"][lo:hi, :m].double()
        elif op == "mx_product":
            w = _exact_unpacked(s["codes"][g * m : (g + 1) * m], s["scales"][g * m : (g + 1) * m], k)
            out[lo:hi] = x[lo:hi] @ w.t()
        else:
            w = s["A"][g, :, :k].double().t() if c["trans"] else s["A"][g, :, :m].double()
            out[lo:hi] = s["B"][lo:hi, :k].double() @ w
    return out
