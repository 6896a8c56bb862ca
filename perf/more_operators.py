"""Timed calls of the operators that route tokens to experts and multiply in 8-bit floating point.

A case is one call (or the calls that belong together) at one size:

  * "route": scores, the choice of experts and their weights (wgb_route), and the tokens' places in the order by
    expert (wgb_route_order);
  * "route_grad": the gradient of the weights back to the router's logits (wgb_route_grad);
  * "rows": tokens copied to their experts' columns (wgb_route_gather) and the experts' results added up for each token
    (wgb_route_combine); with "grad" the gradients of both (wgb_route_combine_grad, and wgb_route_combine without
    weights);
  * "fp8_quantize": to 8 bits with a scale for each block of 128 and back (wgb_fp8_quantize, wgb_fp8_dequantize);
  * "fp8_product": tokens quantised and multiplied with 8-bit weights, one matrix (wgb_fp8_gemm) or one per expert
    (wgb_fp8_gemm_grouped); "block" 1 is the weight gradient, both operands quantised along the tokens.

Tensors are row-major here, which is the library's column-major frame read the other way: a tensor of shape (n, ld) is a
matrix of n columns.
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
        # One decoding step of 16 sequences through a router of 64 experts: latency counts.
        {"name": "route_tokens", "op": "route", "t": F32, "n": 16, "experts": 64, "topk": 8, "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "best": 1, "renorm": 1, "scale": 1.0, "pad": 0, "empty": 0.0},
        # A batch of prompts through a router with a bias for balance and groups of experts.
        {"name": "route_prompt", "op": "route", "t": F32, "n": 16384, "experts": 256, "topk": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "best": 2, "renorm": 1, "scale": 2.5, "pad": 0, "empty": 0.0},
        # 16-bit logits at odd sizes; some tokens are padding and have no expert left.
        {"name": "route_odd", "op": "route", "t": BF16, "n": 4097, "experts": 60, "topk": 6, "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "best": 1, "renorm": 0, "scale": 1.0, "pad": 3, "empty": 0.1},
        # The router's gradient in a training step: every expert's logit has one, through the softmax.
        {"name": "route_grad", "op": "route_grad", "t": F32, "n": 16384, "experts": 128, "topk": 8, "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "best": 1, "renorm": 0, "scale": 1.0, "pad": 0, "empty": 0.0},
        # One decoding step's tokens to their experts and back.
        {"name": "rows_tokens", "op": "rows", "t": BF16, "n": 32, "d": 4096, "topk": 8, "experts": 64, "grad": False, "pad": 0},
        # The gradients of both for a training batch.
        {"name": "rows_grad", "op": "rows", "t": BF16, "n": 8192, "d": 2048, "topk": 6, "experts": 64, "grad": True, "pad": 0},
        # The activations of a prompt to 8 bits and back.
        {"name": "fp8_quantize_tokens", "op": "fp8_quantize", "t": BF16, "k": 4096, "n": 4097, "trans": 0, "block": 1, "pad": 0},
        # A weight matrix in square blocks.
        {"name": "fp8_quantize_weights", "op": "fp8_quantize", "t": F32, "k": 8192, "n": 4096, "trans": 0, "block": 128, "pad": 0},
        # A prompt through one layer of 8-bit weights.
        {"name": "fp8_prompt", "op": "fp8_product", "ot": BF16, "groups": 0, "m": 8192, "n": 4096, "k": 8192, "trans": 1, "block": 128, "skew": 0.0},
        # One decoding step over 8-bit experts.
        {"name": "fp8_grouped_tokens", "op": "fp8_product", "ot": BF16, "groups": 64, "m": 4096, "n": 96, "k": 2048, "trans": 1, "block": 128, "skew": 0.3},
        # The gradient of the experts' input in training: the same weights read the other way.
        {"name": "fp8_grouped_input_grad", "op": "fp8_product", "ot": BF16, "groups": 16, "m": 4096, "n": 16384, "k": 2048, "trans": 0, "block": 128, "skew": 0.3},
        # The weight gradient of one layer, summed over a batch of tokens.
        {"name": "fp8_weight_grad", "op": "fp8_product", "ot": F32, "groups": 0, "m": 4096, "n": 2048, "k": 16384, "trans": 1, "block": 1, "skew": 0.0},
    ]


def _log(rng, lo, hi, step=8):
    """A whole number from lo to hi, spread over the logarithm; three of four rounded to multiples of `step` where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.75 and v >= 2 * step:
        v = v // step * step
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["route", "route", "route_grad", "rows", "rows", "fp8_quantize", "fp8_product", "fp8_product", "fp8_product"])
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 4, 8])
        per = rng.choice([2, 7, 8, 16, 32, 33]) if groups > 1 else 1
        experts = groups * per if groups > 1 else _log(rng, 8, 384)
        top_groups = rng.randint(1, groups)
        topk = min(rng.choice([1, 2, 4, 6, 8]), top_groups * per if groups > 1 else experts)
        scoring = rng.choice(["softmax", "sigmoid"])
        bias = scoring == "sigmoid" and rng.random() < 0.7
        return {"op": op, "t": rng.choice([F32, F32, BF16, F16]), "n": _log(rng, 1, 16384), "experts": experts, "topk": topk,
                "scoring": scoring, "bias": bias, "groups": groups, "top_groups": top_groups, "best": rng.choice([1, 2]),
                "renorm": rng.randrange(2), "scale": rng.choice([1.0, 2.5]), "pad": rng.choice([0, 0, 1, 4]),
                "empty": rng.choice([0.0, 0.0, 0.1])}
    if op == "rows":
        c = {"op": op, "t": rng.choice([BF16, BF16, F16, F32]), "n": _log(rng, 1, 8192), "d": _log(rng, 64, 4096),
             "topk": rng.choice([1, 2, 4, 6, 8]), "experts": rng.choice([8, 64, 256]), "grad": rng.random() < 0.5,
             "pad": rng.choice([0, 0, 1, 8])}
        while c["n"] * c["d"] * c["topk"] * SIZE[c["t"]] > 8192 * 4096 * 4 * 2:
            c["n"] = (c["n"] + 1) // 2
        return c
    if op == "fp8_quantize":
        return {"op": op, "t": rng.choice([F32, F16, BF16]), "k": _log(rng, 128, 8192), "n": _log(rng, 1, 8192),
                "trans": rng.randrange(2), "block": rng.choice([1, 1, 128]), "pad": rng.choice([0, 0, 1, 8])}
    c = {"op": op, "ot": rng.choice([BF16, BF16, F16, F32]), "groups": rng.choice([0, 0, 3, 8, 64]),
         "m": _log(rng, 256, 8192), "n": _log(rng, 1, 16384), "k": _log(rng, 128, 8192), "trans": rng.randrange(2), "block": 128}
    if c["groups"] == 0 and rng.random() < 0.4:
        c.update(trans=1, block=1)
    c["skew"] = rng.choice([0.0, 0.3, 1.0]) if c["groups"] > 1 else 0.0
    while max(1, c["groups"]) * c["m"] * c["k"] > 16 * 4096 * 4096 or _padded(c) > 8192 * 4096 * 8192:
        c["m"] = (c["m"] + 1) // 2
    return c


def _padded(c):
    """About the multiplications of the plain form, which pads every group to the longest."""
    return c["m"] * c["n"] * c["k"] * (1.0 + 3.0 * c["skew"])


def work(c):
    op = c["op"]
    if op in ("route", "route_grad"):
        n, experts, topk = c["n"], c["experts"], c["topk"]
        size = SIZE[c["t"]]
        if op == "route":  # logits; ids, weights, places and pairs of four bytes each; offsets
            return {"bytes": n * experts * size + 16 * n * topk + 8 * (experts + 1), "flops": 8 * n * experts}
        return {"bytes": 2 * n * experts * size + 8 * n * topk, "flops": 8 * n * experts}
    if op == "rows":
        one, all_ = c["n"] * c["d"] * SIZE[c["t"]], c["n"] * c["topk"] * c["d"] * SIZE[c["t"]]
        pairs = 8 * c["n"] * c["topk"]
        if c["grad"]:  # dC, Y and the columns' gradients read, those of Y and X written
            return {"bytes": 2 * one + 3 * all_ + 2 * pairs, "flops": 4 * c["n"] * c["topk"] * c["d"]}
        return {"bytes": 2 * one + 2 * all_ + 2 * pairs, "flops": 2 * c["n"] * c["topk"] * c["d"]}
    if op == "fp8_quantize":
        n = c["n"] * c["k"]
        return {"bytes": 2 * n * (SIZE[c["t"]] + 1 + 4 / (128 * c["block"])), "flops": 2 * n}
    m, n, k, groups = c["m"], c["n"], c["k"], max(1, c["groups"])
    # the weights of experts that get no token need not be read: of evenly drawn ones so many get some
    active = groups * (1.0 - (1.0 - 1.0 / groups) ** n)
    weights = m * k * 2 if c["block"] == 1 else active * m * k
    return {"bytes": weights + n * k * 2 + n * m * SIZE[c["ot"]], "flops": 2 * m * n * k}


# ---- inputs ----------------------------------------------------------------------


def _sizes(c, seed):
    """Tokens of each expert: drawn with the unequal chances that a router gives them."""
    g = torch.Generator().manual_seed(int(seed) + 77)
    chance = torch.softmax(torch.randn(c["groups"], generator=g) * c["skew"], 0)
    return torch.bincount(torch.multinomial(chance, c["n"], replacement=True, generator=g), minlength=c["groups"])


def _blocks(n):
    return (n + 127) // 128


def _weights(groups, rows, length, normal):
    """8-bit weights in square blocks as a checkpoint has them: any scale, codes (groups, rows, whole runs of 128) and
    scales (groups, blocks along a row, blocks of rows)."""
    ld, high = 128 * _blocks(length), 128 * _blocks(rows)
    codes = torch.zeros(groups, rows, ld, dtype=torch.uint8, device="cuda")
    scales = torch.empty(groups, ld // 128, high // 128, device="cuda")
    for g in range(groups):
        w = torch.zeros(high, ld, device="cuda")
        w[:rows, :length] = normal(rows, length, scale=length ** -0.5, t=F32)
        w = w.view(high // 128, 128, ld // 128, 128)
        s = (w.abs().amax((1, 3)) / 448.0).clamp(min=1e-12)
        codes[g] = (w / s[:, None, :, None]).clamp(-448.0, 448.0).view(high, ld)[:rows].to(torch.float8_e4m3fn).view(torch.uint8)
        scales[g] = s.t()
    return codes, scales


def prepare(c, seed):
    s = {"case": dict(c)}
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = c["op"]

    def normal(*shape, scale=1.0, t=BF16, pad=0):
        full = shape[:-1] + (shape[-1] + pad,)
        return torch.empty(full, dtype=TORCH[t], device="cuda").normal_(0.0, scale, generator=g)

    def empty(*shape, t=torch.int32):
        return torch.empty(shape, dtype=t, device="cuda")

    n, topk = c["n"], c.get("topk")
    if op in ("route", "route_grad"):
        experts = c["experts"]
        s["logits"] = normal(n, experts, scale=1.5, t=c["t"], pad=c["pad"])
        gone = torch.rand(n, device="cuda", generator=g) < c["empty"]
        s["logits"][gone] = -math.inf
        s["bias"] = normal(experts, scale=0.05, t=F32) if c["bias"] else None
        s["ids"], s["weights"] = empty(n, topk), empty(n, topk, t=torch.float32)
        if op == "route":
            s["offsets"], s["places"], s["pairs"] = empty(experts + 1, t=torch.int64), empty(n, topk), empty(n * topk)
        else:  # the choice that the forward pass made, and what came back for its weights
            s["ids"] = _choose(s)[1]
            s["dweights"] = normal(n, topk, t=F32)
            s["dlogits"] = empty(n, experts, t=TORCH[c["t"]])
    elif op == "rows":
        d, t = c["d"], TORCH[c["t"]]
        chance = torch.rand(n, c["experts"], device="cuda", generator=g)
        ids = chance.argsort(1)[:, :topk].reshape(-1)
        s["places"] = empty(n, topk)
        s["places"].view(-1)[torch.argsort(ids, stable=True)] = torch.arange(n * topk, dtype=torch.int32, device="cuda")
        w = torch.rand(n, topk, device="cuda", generator=g) + 0.1
        s["weights"] = w / w.sum(1, keepdim=True)
        s["X"], s["Y"] = normal(n, d, t=c["t"], pad=c["pad"]), normal(n * topk, d, t=c["t"])
        s["out"], s["rows_out"] = empty(n, d, t=t), empty(n * topk, d, t=t)
        if c["grad"]:
            s["dY"], s["dweights"] = empty(n * topk, d, t=t), empty(n, topk, t=torch.float32)
            s["drows"] = normal(n * topk, d, t=c["t"])
    elif op == "fp8_quantize":
        k = c["k"]
        s["X"] = normal(k, n, t=c["t"], pad=c["pad"]) if c["trans"] else normal(n, k, t=c["t"], pad=c["pad"])
        _room(s, "X", n, k, c["block"])
        s["out"] = empty(n, k, t=TORCH[c["t"]])
    else:
        m, k, groups = c["m"], c["k"], c["groups"]
        if groups:
            sizes = _sizes(c, seed)
            s["longest"] = max(1, int(sizes.max()))
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).cuda()
        if c["block"] == 1:  # k is the tokens: two activations, neither of which lies along it
            s["X"], s["dY"] = normal(k, n), normal(k, m)
            _room(s, "dY", m, k, 1)
        else:
            s["X"] = normal(n, k)
            s["codes"], s["scales"] = _weights(max(1, groups), m if c["trans"] else k, k if c["trans"] else m, normal)
        _room(s, "X", n, k, 1)
        s["C"] = empty(n, m, t=TORCH[c["ot"]])
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    return s


def _room(s, name, n, k, block):
    """Buffers for the quantised form of an operand, kept as a program keeps them."""
    s[name + "_codes"] = torch.empty(n, 128 * _blocks(k), dtype=torch.uint8, device="cuda")
    s[name + "_scales"] = torch.empty(_blocks(k), (n + block - 1) // block, dtype=torch.float32, device="cuda")


# ---- the plain form ----------------------------------------------------------------


def _scores(s):
    """Scores of the experts in 64 bits: values next to each other decide the choice."""
    c = s["case"]
    x = s["logits"][:, : c["experts"]].double()
    if c["scoring"] == "sigmoid":
        return 1.0 / (1.0 + (-x).exp())
    top = x.amax(1, keepdim=True)
    e = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    return e / e.sum(1, keepdim=True).clamp(min=1e-300)


def _choose(s):
    """(scores, ids): the experts in the order of their choice values, -1 where none is left."""
    c = s["case"]
    n, experts, topk = c["n"], c["experts"], c["topk"]
    p = _scores(s)
    choice = torch.where(s["logits"][:, :experts] == -math.inf, -math.inf, p)
    if s["bias"] is not None:
        choice = choice + s["bias"].double()
    if c["groups"] > 1:
        grouped = choice.view(n, c["groups"], -1)
        best = grouped.sort(dim=2, descending=True)[0][:, :, : c["best"]].sum(2)
        group = best.sort(dim=1, descending=True, stable=True)[1][:, : c["top_groups"]]
        keep = torch.zeros(n, c["groups"], dtype=torch.bool, device=p.device).scatter_(1, group, True)
        choice = torch.where(keep[:, :, None], grouped, -math.inf).reshape(n, experts)
    value, ids = choice.sort(dim=1, descending=True, stable=True)
    ids = torch.where(value == -math.inf, -1, ids)
    return p, ids[:, :topk].to(torch.int32).contiguous()


def _chosen(s, p, ids):
    """Scores of the chosen experts (0 where there is none) and their sum."""
    got = torch.where(ids < 0, 0.0, p.gather(1, ids.clamp(min=0).long()))
    return got, got.sum(1, keepdim=True)


def _plain_route(s):
    c = s["case"]
    p, ids = _choose(s)
    w, total = _chosen(s, p, ids)
    if c["renorm"]:
        w = w / torch.where(total == 0, 1.0, total)
    # stable order by expert, the pairs without one at the end
    flat = torch.where(ids < 0, c["experts"], ids).view(-1)
    order = flat.argsort(stable=True)
    count = torch.bincount(flat, minlength=c["experts"] + 1)[: c["experts"]]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=flat.device), count.cumsum(0)])
    at = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    places = torch.empty_like(at)
    places[order] = at
    places = torch.where(ids < 0, -1, places.view(ids.shape))
    pairs = torch.where(at < offsets[-1], order, -1).to(torch.int32)
    return ids, (w * c["scale"]).float(), offsets, places, pairs


def _plain_route_grad(s):
    c, ids = s["case"], s["ids"]
    p = _scores(s)
    got, total = _chosen(s, p, ids)
    d = torch.where(ids < 0, 0.0, s["dweights"].double()) * c["scale"]
    if c["renorm"]:
        total = torch.where(total == 0, 1.0, total)
        d = (d - (d * got).sum(1, keepdim=True) / total) / total
    d = torch.where(ids < 0, 0.0, d)
    d = torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0).long(), d)
    if c["scoring"] == "sigmoid":
        grad = d * p * (1.0 - p)
    else:
        grad = p * (d - (d * p).sum(1, keepdim=True))
    return grad.to(TORCH[c["t"]])


def _plain_rows(s):
    c = s["case"]
    n, d, topk = c["n"], c["d"], c["topk"]
    dtype = TORCH[c["t"]]
    at = s["places"].long()
    x = s["X"][:, :d].float()
    w = s["weights"][:, :, None]
    if c["grad"]:  # X is the gradient of the combined result
        dweights = (s["Y"].float()[at] * x[:, None, :]).sum(2)
        dy = torch.empty(n * topk, d, device=x.device)
        dy[at.view(-1)] = (w * x[:, None, :]).view(-1, d)
        return dy.to(dtype), dweights, s["drows"].float()[at].sum(1).to(dtype)
    rows = torch.empty(n * topk, d, device=x.device)
    rows[at.view(-1)] = x.repeat_interleave(topk, 0)
    return rows.to(dtype), (s["Y"].float()[at] * w).sum(1).to(dtype)


def _e4m3(v):
    """To the nearest 8-bit float with 4 bits of exponent, ties to even; |v| <= 448."""
    e = (torch.frexp(v)[1] - 1).clamp(min=-6)
    return torch.ldexp(torch.ldexp(v, 3 - e).round(), e - 3).clamp(-448.0, 448.0)


def _values(x, block):
    """The values that the quantised form of x (rows x k, blocks of `block` rows by 128) stands for."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -rows % block))
    x = x.view(-1, block, x.shape[1] // 128, 128)
    f, e = torch.frexp(x.abs().amax((1, 3), keepdim=True))
    # the least power of two that brings f 2^e to 448 = 0.875 2^9 or less
    e = torch.where(f == 0, -126, (e - 9 + (f > 0.875)).clamp(min=-126))
    return torch.ldexp(_e4m3(torch.ldexp(x, -e)), e).reshape(-1, x.shape[2] * 128)[:rows, :k]


def _unpack(codes, scales, rows, length):
    """Weights of one expert (rows x length) in 32 bits."""
    v = codes.view(torch.float8_e4m3fn).float()
    s = scales.t().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)
    return (v * s)[:, :length]


def _places(offsets, longest, n):
    """For each group its tokens' places, padded to the longest."""
    at = offsets[:-1, None] + torch.arange(longest, device=offsets.device)
    return at.clamp(max=n - 1)


def _back(padded, offsets, n):
    """The tokens' rows of a padded product, in their own order."""
    token = torch.arange(n, device=offsets.device)
    group = torch.searchsorted(offsets[1:], token, right=True)
    return padded[group, token - offsets[group]]


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "route":
        return _plain_route(s)
    if op == "route_grad":
        return _plain_route_grad(s)
    if op == "rows":
        return _plain_rows(s)
    k, n = c["k"], c["n"]
    if op == "fp8_quantize":
        x = s["X"][:, :n].t() if c["trans"] else s["X"][:, :k]
        return _values(x, c["block"]).to(TORCH[c["t"]])
    m, groups, dtype = c["m"], c["groups"], TORCH[c["ot"]]
    if c["block"] == 1:
        return (_values(s["X"].t(), 1) @ _values(s["dY"].t(), 1).t()).to(dtype)
    x = _values(s["X"], 1)
    rows, length = (m, k) if c["trans"] else (k, m)
    w = torch.stack([_unpack(a, b, rows, length) for a, b in zip(s["codes"], s["scales"])])
    w = w.transpose(1, 2) if c["trans"] else w
    if not groups:
        return (x @ w[0]).to(dtype)
    at = _places(s["offsets"], s["longest"], n)
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
        return None if s[name] is None else s[name].data_ptr()

    n = c["n"]
    if op in ("route", "route_grad"):
        experts, topk, t = c["experts"], c["topk"], kind[c["t"]]
        scoring = wg.SIGMOID if c["scoring"] == "sigmoid" else wg.SOFTMAX
        ld = s["logits"].shape[1]
        if op == "route":
            ctx.route(t, scoring, experts, n, topk, at("logits"), ld, at("bias"), c["groups"], c["top_groups"], c["best"],
                      c["renorm"], c["scale"], at("ids"), at("weights"))
            ctx.route_order(experts, n, topk, at("ids"), at("offsets"), at("places"), at("pairs"))
            return s["ids"], s["weights"], s["offsets"], s["places"], s["pairs"]
        ctx.route_grad(t, scoring, experts, n, topk, at("logits"), ld, at("ids"), c["renorm"], c["scale"], at("dweights"),
                       at("dlogits"), experts)
        return s["dlogits"]
    if op == "rows":
        d, topk, t, ld = c["d"], c["topk"], kind[c["t"]], s["X"].shape[1]
        if c["grad"]:
            ctx.route_combine_grad(t, d, n, topk, at("X"), ld, at("Y"), d, at("places"), at("weights"), at("dY"), d,
                                   at("dweights"))
            ctx.route_combine(t, d, n, topk, at("drows"), d, at("places"), None, 0.0, at("out"), d)
            return s["dY"], s["dweights"], s["out"]
        ctx.route_gather(t, d, n, topk, at("X"), ld, at("places"), None, at("rows_out"), d)
        ctx.route_combine(t, d, n, topk, at("Y"), d, at("places"), at("weights"), 0.0, at("out"), d)
        return s["rows_out"], s["out"]
    k = c["k"]
    ld = 128 * _blocks(k)
    if op == "fp8_quantize":
        columns = s["X_scales"].shape[1]
        ctx.fp8_quantize(kind[c["t"]], c["trans"], c["block"], k, n, at("X"), s["X"].shape[1], at("X_codes"), ld,
                         at("X_scales"), columns)
        ctx.fp8_dequantize(kind[c["t"]], c["block"], k, n, at("X_codes"), ld, at("X_scales"), columns, at("out"), k)
        return s["out"]
    m, groups, ot = c["m"], c["groups"], kind[c["ot"]]
    if c["block"] == 1:
        ctx.fp8_quantize(wg.BF16, wg.TRANS, 1, k, n, at("X"), n, at("X_codes"), ld, at("X_scales"), n)
        ctx.fp8_quantize(wg.BF16, wg.TRANS, 1, k, m, at("dY"), m, at("dY_codes"), ld, at("dY_scales"), m)
        ctx.fp8_gemm(wg.TRANS, m, n, k, 1.0, at("dY_codes"), ld, 1, at("dY_scales"), m, at("X_codes"), ld, at("X_scales"), n,
                     0.0, at("C"), m, ot)
        return s["C"]
    ctx.fp8_quantize(wg.BF16, wg.NO_TRANS, 1, k, n, at("X"), k, at("X_codes"), ld, at("X_scales"), n)
    _, rows, lda = s["codes"].shape
    along, across = s["scales"].shape[1:]
    if groups:
        ctx.fp8_gemm_grouped(c["trans"], groups, m, n, k, 1.0, at("codes"), lda, rows * lda, 128, at("scales"), across,
                             along * across, at("X_codes"), ld, at("X_scales"), n, at("offsets"), 0.0, at("C"), m, ot)
    else:
        ctx.fp8_gemm(c["trans"], m, n, k, 1.0, at("codes"), lda, 128, at("scales"), across, at("X_codes"), ld,
                     at("X_scales"), n, 0.0, at("C"), m, ot)
    return s["C"]


def run(s):
    return _kernels(s) if own else _plain(s)


# ---- the definition in 64 bits -----------------------------------------------------


def _exact_route(s):
    """Scores by the logarithm of their sum; the choice one expert after the other, the first of the largest."""
    c = s["case"]
    n, experts, topk = c["n"], c["experts"], c["topk"]
    x = s["logits"][:, :experts].double()
    empty = torch.isneginf(x).all(1, keepdim=True)
    if c["scoring"] == "sigmoid":
        p = torch.sigmoid(x)
    else:
        p = torch.exp(x - torch.where(empty, 0.0, torch.logsumexp(x, 1, keepdim=True)))
    choice = p.masked_fill(torch.isneginf(x), -math.inf)
    if s["bias"] is not None:
        choice = choice + s["bias"].double()

    def first_largest(v, count):
        """Places of the `count` largest of each row, the lowest place of equal ones."""
        v, out = v.clone(), []
        place = torch.arange(v.shape[1], device=v.device)
        for _ in range(count):
            top = v.amax(1, keepdim=True)
            at = torch.where(v == top, place, v.shape[1]).amin(1, keepdim=True)
            out.append(torch.where(torch.isneginf(top), -1, at))
            v.scatter_(1, at, -math.inf)
        return torch.cat(out, 1)

    if c["groups"] > 1:
        per = experts // c["groups"]
        score = torch.topk(choice.view(n, c["groups"], per), min(per, c["best"]), dim=2)[0].sum(2)
        group = first_largest(score, c["top_groups"])
        member = torch.arange(experts, device=x.device) // per
        keep = (member[None, :, None] == group[:, None, :]).any(2)
        choice = choice.masked_fill(~keep, -math.inf)
    ids = first_largest(choice, topk)
    w = torch.where(ids < 0, 0.0, p.gather(1, ids.clamp(min=0)))
    return p, ids, w


def _exact_order(ids, experts):
    """Places by counting: the pairs of lower experts, and the earlier ones of the same."""
    flat = ids.reshape(-1).cpu()
    offsets, places = torch.zeros(experts + 1, dtype=torch.int64), torch.full((flat.numel(),), -1, dtype=torch.int64)
    pairs = torch.full((flat.numel(),), -1, dtype=torch.int64)
    for e in range(experts):
        mine = torch.nonzero(flat == e).view(-1)
        offsets[e + 1] = offsets[e] + len(mine)
        places[mine] = torch.arange(int(offsets[e]), int(offsets[e + 1]))
        pairs[int(offsets[e]) : int(offsets[e + 1])] = mine
    return offsets.cuda(), places.view(ids.shape).cuda(), pairs.cuda()


def _exact_e4m3():
    """The magnitudes of all codes from their exponent and mantissa bits (the last code is NaN)."""
    code = torch.arange(127, device="cuda")
    e, f = code // 8, (code % 8).double()
    return torch.where(e == 0, f * 2.0 ** -9, (1.0 + f / 8.0) * torch.exp2(e.double() - 7.0))


def _exact_values(x, block):
    """What the quantised form of x stands for: each block's scale, each value to the nearest magnitude by the middles
    between them, a middle to the even code."""
    rows, k = x.shape
    full = torch.zeros((rows + block - 1) // block * block, 128 * _blocks(k), dtype=torch.float64, device=x.device)
    full[:rows, :k] = x.double()
    tiles = full.view(full.shape[0] // block, block, -1, 128)
    top = tiles.abs().amax((1, 3), keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 448.0)).clamp(min=-126.0))
    v = tiles / scale
    levels = _exact_e4m3()
    middles = (levels[:-1] + levels[1:]) / 2
    low = torch.searchsorted(middles, v.abs().contiguous())  # middles below |v|: a tie stays at the lower code
    tie = (low < 126) & (v.abs() == middles[low.clamp(max=125)]) & (low % 2 == 1)
    q = levels[torch.where(tie, low + 1, low)] * torch.sign(v)
    return (q * scale).reshape(full.shape)[:rows, :k]


def _exact_weights(codes, scales, rows, length):
    """Weights of one expert from sign and magnitude bits and the block that each belongs to."""
    v = torch.cat([_exact_e4m3(), torch.full((1,), math.nan, dtype=torch.float64, device="cuda")])[codes.long() % 128]
    v = torch.where(codes >= 128, -v, v)[:, :length]
    r = torch.arange(rows, device="cuda") // 128
    q = torch.arange(length, device="cuda") // 128
    return v * scales.double()[q[None, :], r[:, None]]


def exact(c, seed):
    s = prepare(c, seed)
    op = c["op"]
    if op == "route":
        _, ids, w = _exact_route(s)
        if c["renorm"]:
            total = w.sum(1, keepdim=True)
            w = torch.where(total == 0, 0.0, w / total)
        return (ids, w * c["scale"]) + _exact_order(ids, c["experts"])
    if op == "route_grad":
        p, _, _ = _exact_route(s)
        ids = s["ids"].long()
        # the weights' Jacobian applied to what came back, one place after the other
        w = torch.where(ids < 0, 0.0, p.gather(1, ids.clamp(min=0)))
        dw = torch.where(ids < 0, 0.0, s["dweights"].double())
        total = w.sum(1, keepdim=True)
        total = torch.where(total == 0, 1.0, total)
        dp = torch.zeros_like(p)
        for j in range(c["topk"]):
            d = dw[:, j : j + 1]
            if c["renorm"]:
                d = d / total - (dw * w).sum(1, keepdim=True) / total ** 2
            dp.scatter_add_(1, ids[:, j : j + 1].clamp(min=0), torch.where(ids[:, j : j + 1] < 0, 0.0, c["scale"] * d))
        if c["scoring"] == "sigmoid":
            x = s["logits"][:, : c["experts"]].double()
            return dp * torch.sigmoid(x) * torch.sigmoid(-x)
        return p * dp - p * (p * dp).sum(1, keepdim=True)
    if op == "rows":
        n, d, topk = c["n"], c["d"], c["topk"]
        x, w = s["X"][:, :d].double(), s["weights"].double()
        pair = torch.empty(n * topk, dtype=torch.int64, device="cuda")
        pair[s["places"].long().view(-1)] = torch.arange(n * topk, device="cuda")
        token = pair // topk
        out = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        wide = w.view(-1)[pair][:, None]
        if c["grad"]:
            dw = torch.empty(n * topk, dtype=torch.float64, device="cuda")
            dw[pair] = (s["Y"].double() * x[token]).sum(1)
            return wide * x[token], dw.view(n, topk), out.index_add_(0, token, s["drows"].double())
        return x[token], out.index_add_(0, token, s["Y"].double() * wide)
    k, n = c["k"], c["n"]
    if op == "fp8_quantize":
        return _exact_values(s["X"][:, :n].t() if c["trans"] else s["X"][:, :k], c["block"])
    m, groups = c["m"], c["groups"]
    if c["block"] == 1:
        return _exact_values(s["X"].t(), 1) @ _exact_values(s["dY"].t(), 1).t()
    x = _exact_values(s["X"], 1)
    rows, length = (m, k) if c["trans"] else (k, m)
    offsets = s["offsets"].tolist() if groups else [0, n]
    out = torch.zeros(n, m, dtype=torch.float64, device="cuda")
    for g in range(max(1, groups)):
        lo, hi = offsets[g], offsets[g + 1]
        if lo < hi:
            w = _exact_weights(s["codes"][g], s["scales"][g], rows, length)
            out[lo:hi] = x[lo:hi] @ (w.t() if c["trans"] else w)
    return out
