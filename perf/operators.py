"""The operators between a layer's activations and the next token: microscaled 4-bit floating point (quantisation and
projection) and what is done to a row of logits (rules, and the draw of a token).

Four kinds of work, each through the public entry points:

* ``quant``: rows to 4-bit codes with block scales and back (``quantize_fp4`` / ``dequantize_fp4``);
* ``linear``: a projection with both operands in 4 bits (``fp4_linear``; the activations are quantised in the call);
* ``rules``: penalties for repeated tokens, biases and a grammar mask on logits (``process_logits``);
* ``sample``: temperature, top-k, top-p, min-p and the draw, with or without the rules in front (``sample_tokens``).

Formats.  A code is E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; nearest, ties to the even code).  ``mxfp4``: 32 elements
share a power of two, 2^(floor(log2 amax) - 2).  ``nvfp4``: 16 elements share an E4M3 scale, a row shares a power of two
g = 2^(floor(log2 amax) - 10).  Two codes a byte, the even element in the low nibble.  Scales lie in tiles of 128 rows x 4
blocks, [row tile, block tile, row % 32, row % 128 / 32, block % 4].

``own`` False: elementary torch operations in 32 bits.  ``own`` True: the calls a user makes.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
VOCAB = 65536
MAX_FLOPS = 2 * 8192 * 4096 * 16384


def listed():
    return [
        # one token's activations of the small model on the way to a projection: latency is all there is
        dict(kind="quant", format="nvfp4", dtype="fp16", rows=1, k=768, name="quant-nvfp4-1x768"),
        # a prompt chunk's activations of the large model
        dict(kind="quant", format="mxfp4", dtype="bf16", rows=8192, k=4096, name="quant-mxfp4-8192x4096"),
        # FFN up-projection of one user's decode step on the large model
        dict(kind="linear", format="nvfp4", dtype="fp16", rows=1, k=4096, n=16384, epilogue="relu2", name="linear-nvfp4-1x4096x16384"),
        # output projection of 64 concurrent sequences with the residual stream added
        dict(kind="linear", format="nvfp4", dtype="fp16", rows=64, k=4096, n=4096, epilogue="residual", name="linear-nvfp4-64x4096x4096"),
        # three prompts of no particular length through the middle model's FFN
        dict(kind="linear", format="mxfp4", dtype="bf16", rows=777, k=2560, n=10240, epilogue="relu2", name="linear-mxfp4-777x2560x10240"),
        # a bulk prefill chunk through the large model's FFN: the largest product
        dict(kind="linear", format="nvfp4", dtype="fp16", rows=8192, k=4096, n=16384, epilogue="none", name="linear-nvfp4-8192x4096x16384"),
        # one chat: a few hundred tokens so far, no grammar
        dict(kind="rules", dtype="fp16", batch=1, vocab=VOCAB, history=300, bias="none", mask=False, name="rules-1x65536-h300"),
        # 64 structured answers: long histories, one bias for all rows, a grammar mask per row
        dict(kind="rules", dtype="fp16", batch=64, vocab=VOCAB, history=4096, bias="shared", mask=True, name="rules-64x65536-h4096"),
        # a vocabulary of odd size, a bias per row
        dict(kind="rules", dtype="bf16", batch=7, vocab=50277, history=777, bias="rows", mask=True, name="rules-7x50277-h777"),
        # one chat: nucleus sampling
        dict(kind="sample", dtype="fp16", batch=1, vocab=VOCAB, history=0, bias="none", mask=False, top_k=0, top_p=True, min_p=False,
             name="sample-1x65536-p"),
        # 64 requests, every filter and every rule
        dict(kind="sample", dtype="fp16", batch=64, vocab=VOCAB, history=512, bias="shared", mask=True, top_k=50, top_p=True, min_p=True,
             name="sample-64x65536-all"),
        # bulk generation from the whole distribution, fp32 logits
        dict(kind="sample", dtype="fp32", batch=256, vocab=VOCAB, history=0, bias="none", mask=False, top_k=0, top_p=False, min_p=False,
             name="sample-256x65536-plain"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("quant", "linear", "linear", "linear", "rules", "sample", "sample"))
    dtype = rng.choice(("fp16", "bf16", "fp32"))
    if kind == "quant":
        k = 32 * _log_int(rng, 1, 512)
        return dict(kind=kind, format=rng.choice(("mxfp4", "nvfp4")), dtype=dtype, rows=_log_int(rng, 1, min(8192, 16777216 // k)), k=k)
    if kind == "linear":
        if rng.random() < 0.5:
            k, n = rng.choice(((768, 768), (2560, 2560), (2560, 10240), (10240, 2560), (4096, 4096), (4096, 16384), (16384, 4096)))
        else:
            k, n = 32 * _log_int(rng, 1, 512), _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, min(8192, MAX_FLOPS // (2 * k * n)))
        return dict(kind=kind, format=rng.choice(("mxfp4", "nvfp4")), dtype=rng.choice(("fp16", "bf16")), rows=rows, k=k, n=n,
                    epilogue=rng.choice(("none", "bias", "relu2", "residual")))
    vocab = rng.choice((VOCAB, 50277, _log_int(rng, 2, 200000)))
    batch = _log_int(rng, 1, min(256, 16777216 // vocab))
    case = dict(kind=kind, dtype=dtype, batch=batch, vocab=vocab, history=rng.choice((0, 1, _log_int(rng, 1, 8192))),
                bias=rng.choice(("none", "shared", "rows")), mask=rng.random() < 0.5)
    if kind == "sample":
        case.update(top_k=rng.choice((0, 1, _log_int(rng, 1, 2 * vocab))), top_p=rng.random() < 0.6, min_p=rng.random() < 0.3)
    return case


# ---------------------------------------------------------------- inputs
def _activations(rows, k, dtype, g):
    """Normalised activations with a few channels an order of magnitude larger."""
    x = torch.randn((rows, k), device=DEV, generator=g)
    loud = 1 + 15 * (torch.rand((k,), device=DEV, generator=g) < 0.01)
    return (x * loud).to(DTYPES[dtype])


def _logits(case, g):
    """A head's logits: a broad bulk and a few dozen tokens that the context makes likely."""
    B, V = case["batch"], case["vocab"]
    z = 2.5 * torch.randn((B, V), device=DEV, generator=g) - 2
    at = torch.randint(0, V, (B, 24), device=DEV, generator=g)
    z.scatter_(1, at, 7 + 3 * torch.randn((B, 24), device=DEV, generator=g))
    return z.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "quant":
        s["x"] = _activations(case["rows"], case["k"], case["dtype"], g)
        return s
    if case["kind"] == "linear":
        rows, k, n, fmt = case["rows"], case["k"], case["n"], case["format"]
        s["x"] = _activations(rows, k, case["dtype"], g)
        # the weight as a program keeps it: codes, scale tiles, row scales
        w = torch.randn((n, k), device=DEV, generator=g) / math.sqrt(k)
        codes, scale, g_row = _encode(w, fmt)
        s["packed"] = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()
        s["scales"] = _to_tiles(_scale_bytes(scale, fmt))
        s["row_scale"] = None if fmt == "mxfp4" else g_row.reshape(-1).contiguous()
        epi = case["epilogue"]
        s["bias"] = torch.randn((n,), device=DEV, generator=g).to(DTYPES[case["dtype"]]) if epi == "bias" else None
        s["residual"] = torch.randn((rows, n), device=DEV, generator=g).to(DTYPES[case["dtype"]]) if epi == "residual" else None
        return s
    B, V, L = case["batch"], case["vocab"], case["history"]
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand((B,), device=DEV, generator=g)
    s["logits"] = _logits(case, g)
    s["tokens"] = None
    if L:
        # text repeats itself: few tokens make up most of a history; rows have their own lengths, the first row is full
        s["tokens"] = (V * torch.rand((B, L), device=DEV, generator=g) ** 4).long().clamp_(max=V - 1)
        s["lengths"] = (uniform(0, 1) * (L + 1)).int().clamp_(max=L)
        s["lengths"][0] = L
        s["prompt_lengths"] = (s["lengths"] * uniform(0, 1)).int()
        s["repetition"], s["presence"], s["frequency"] = uniform(1.0, 1.4), uniform(0.0, 0.8), uniform(0.0, 0.5)
    s["bias"] = s["allowed"] = None
    if case["bias"] != "none":
        shape = (V,) if case["bias"] == "shared" else (B, V)
        some = torch.rand(shape, device=DEV, generator=g) < 0.02
        s["bias"] = torch.where(some, 4 * torch.randn(shape, device=DEV, generator=g), 0.0)
    if case["mask"]:
        # a grammar that leaves most tokens (inside a string), some, or a handful
        share = torch.rand((B, 1), device=DEV, generator=g) ** 3
        ok = torch.rand((B, (V + 31) // 32 * 32), device=DEV, generator=g) < share
        ok[:, V // 2] = True
        bit = 2 ** torch.arange(32, device=DEV)
        word = (ok.view(B, -1, 32) * bit).sum(-1)
        s["allowed"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()
    if case["kind"] == "sample":
        s["noise"] = torch.empty((B, V), device=DEV).exponential_(generator=g)
        s["temperature"] = uniform(0.5, 1.3)
        if B >= 8:
            s["temperature"][::8] = 0  # some requests are greedy
        s["top_p"] = uniform(0.3, 0.98) if case["top_p"] else None
        s["min_p"] = uniform(0.0, 0.1) if case["min_p"] else None
        s["top_k"] = torch.full((B,), case["top_k"], device=DEV, dtype=torch.int32) if case["top_k"] else None
    return s


# ---------------------------------------------------------------- plain form: 4-bit floating point
def _blocks(x, fmt):
    return x.reshape(x.shape[0], -1, BLOCK[fmt])


def _round_e2m1(v):
    """Codes of |v| on the grid 0, 0.5, 1, 1.5, 2, 3, 4, 6: nearest, ties to the even code, 6 above."""
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    return code | (torch.signbit(v).to(torch.uint8) << 3)


def _exponent(a):
    """floor(log2(a)) of positive normal numbers."""
    return torch.frexp(a)[1] - 1


def _encode(x, fmt):
    """(codes [R,K] uint8, block scales [R,K/block], row scales [R,1]); the value of a code is grid * block scale * row scale."""
    x = x.float()
    R = x.shape[0]
    xb = _blocks(x, fmt)
    amax = xb.abs().amax(-1)
    if fmt == "mxfp4":
        e = torch.where(amax > 0, _exponent(amax) - 2, torch.full_like(amax, -127, dtype=torch.int32)).clamp(-127, 127)
        scale = torch.exp2(e.float())
        codes = _round_e2m1(xb * torch.exp2(-e.float())[..., None])
        return codes.reshape(R, -1), scale, torch.ones((R, 1), device=x.device)
    top = amax.amax(-1, keepdim=True)
    g = torch.where(top > 0, torch.exp2((_exponent(top) - 10).float()), torch.ones_like(top))
    scale = (amax / g / 6).to(torch.float8_e4m3fn).float()
    v = torch.where(scale[..., None] > 0, xb / g[..., None] / scale[..., None], torch.zeros_like(xb))
    return _round_e2m1(v).reshape(R, -1), scale, g


def _scale_bytes(scale, fmt):
    if fmt == "mxfp4":
        return (_exponent(scale) + 127).clamp(0, 254).to(torch.uint8)
    return scale.to(torch.float8_e4m3fn).view(torch.uint8)


def _to_tiles(b):
    R, C = b.shape
    rt, ct = (R + 127) // 128, (C + 3) // 4
    full = torch.zeros((rt * 128, ct * 4), device=b.device, dtype=torch.uint8)
    full[:R, :C] = b
    return full.view(rt, 4, 32, ct, 4).permute(0, 3, 2, 1, 4).contiguous()


def _from_tiles(t, R, C):
    return t.permute(0, 3, 2, 1, 4).reshape(t.shape[0] * 128, -1)[:R, :C]


def _grid(codes):
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return table[codes.long()]


def _values(codes, scale, g, fmt):
    v = _blocks(_grid(codes), fmt) * scale[..., None]
    return (v * g[..., None]).reshape(codes.shape)


def _weight(s):
    """The 32-bit values of the stored weight."""
    fmt, n, k = s["case"]["format"], s["case"]["n"], s["case"]["k"]
    codes = torch.stack((s["packed"] & 15, s["packed"] >> 4), -1).view(n, k)
    b = _from_tiles(s["scales"], n, k // BLOCK[fmt])
    if fmt == "mxfp4":
        return _values(codes, torch.exp2(b.float() - 127), torch.ones((n, 1), device=codes.device), fmt)
    return _values(codes, b.contiguous().view(torch.float8_e4m3fn).float(), s["row_scale"][:, None], fmt)


def _plain_quant(s):
    fmt = s["case"]["format"]
    return {"values": _values(*_encode(s["x"], fmt), fmt).to(s["x"].dtype)}


def _plain_linear(s):
    fmt, epi = s["case"]["format"], s["case"]["epilogue"]
    y = _values(*_encode(s["x"], fmt), fmt) @ _weight(s).t()
    if epi == "bias":
        y = y + s["bias"].float()
    elif epi == "relu2":
        y = torch.relu(y) ** 2
    elif epi == "residual":
        y = y + s["residual"].float()
    return {"y": y.to(s["x"].dtype)}


# ---------------------------------------------------------------- plain form: logits
def _ruled(s):
    """The logits after the rules, in 32 bits."""
    z = s["logits"].float()
    V = z.shape[1]
    if s["tokens"] is not None:
        ids, n, at = s["tokens"], s["lengths"][:, None], torch.arange(s["tokens"].shape[1], device=z.device)[None]
        seen = torch.zeros_like(z).scatter_add_(1, ids, (at < n).float()) > 0
        count = torch.zeros_like(z).scatter_add_(1, ids, ((at < n) & (at >= s["prompt_lengths"][:, None])).float())
        rep = s["repetition"][:, None]
        z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
        z = z - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0).float()
    if s["bias"] is not None:
        z = z + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(V, device=z.device)
        z = torch.where((s["allowed"][:, v >> 5] >> (v & 31)) & 1 == 1, z, torch.full_like(z, -math.inf))
    return z


def _plain_sample(s):
    z = _ruled(s)
    V = z.shape[1]
    T = s["temperature"][:, None]
    greedy = T <= 0
    z = z / torch.where(greedy, torch.ones_like(T), T)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    logp = z - top - torch.log(e.sum(1, keepdim=True))
    score = e / s["noise"]
    if s["top_k"] is not None or s["top_p"] is not None:
        sz, order = torch.sort(z, dim=1, descending=True, stable=True)
        keep = torch.ones_like(sz, dtype=torch.bool)
        if s["top_k"] is not None:
            keep = sz >= sz.gather(1, (s["top_k"].long()[:, None] - 1).clamp(0, V - 1))
        if s["top_p"] is not None:
            pr = torch.where(keep, torch.exp(sz - top), torch.zeros_like(sz))
            pr = pr / pr.sum(1, keepdim=True)
            keep = keep & (pr.cumsum(1) - pr < s["top_p"][:, None])
            keep[:, 0] = True
        score = torch.where(torch.zeros_like(keep).scatter(1, order, keep), score, torch.full_like(score, -1))
    if s["min_p"] is not None:
        score = torch.where(e >= s["min_p"][:, None], score, torch.full_like(score, -1))
    token = torch.where(greedy, e, score).argmax(1)
    return {"token": token, "logprob": logp.gather(1, token[:, None])[:, 0]}


# ---------------------------------------------------------------- the two sides
def _own_rules(s):
    rules = dict(bias=s["bias"], allowed=s["allowed"])
    if s["tokens"] is not None:
        rules.update(tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompt_lengths"], repetition_penalty=s["repetition"],
                     presence_penalty=s["presence"], frequency_penalty=s["frequency"])
    return rules


def _own(s):
    import hf_adapter_b200 as hb
    case = s["case"]
    if case["kind"] == "quant":
        packed, scales, row_scale = hb.quantize_fp4(s["x"], case["format"])
        return {"values": hb.dequantize_fp4(packed, scales, row_scale, format=case["format"], dtype=s["x"].dtype)}
    if case["kind"] == "linear":
        return {"y": hb.fp4_linear(s["x"], s["packed"], s["scales"], s["row_scale"], s["bias"], format=case["format"],
                                   relu2=case["epilogue"] == "relu2", residual=s["residual"])}
    if case["kind"] == "rules":
        return {"logits": hb.process_logits(s["logits"], **_own_rules(s))}
    more = {k: s[k] for k in ("top_k", "top_p", "min_p") if s[k] is not None}
    token, logprob = hb.sample_tokens(s["logits"], s["noise"], temperature=s["temperature"], return_logprobs=True, **more, **_own_rules(s))
    return {"token": token, "logprob": logprob}


@torch.no_grad()
def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "quant":
        return _plain_quant(state)
    if kind == "linear":
        return _plain_linear(state)
    if kind == "rules":
        return {"logits": _ruled(state).to(state["logits"].dtype)}
    return _plain_sample(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    es = {"fp32": 4, "fp16": 2, "bf16": 2}[case["dtype"]]
    if case["kind"] == "quant":
        n = case["rows"] * case["k"]
        return {"bytes": 2 * n * es, "flops": 4 * n}  # rows in, values out
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        weight = n * k // 2 + n * k // BLOCK[case["format"]] + (4 * n if case["format"] == "nvfp4" else 0)
        more = {"none": 0, "relu2": 0, "bias": n * es, "residual": m * n * es}[case["epilogue"]]
        return {"bytes": m * k * es + weight + m * n * es + more, "flops": 2 * m * n * k}
    B, V, L = case["batch"], case["vocab"], case["history"]
    n = B * V
    rules = B * L * 8 + {"none": 0, "shared": 4 * V, "rows": 4 * n}[case["bias"]] + (B * ((V + 31) // 32) * 4 if case["mask"] else 0)
    if case["kind"] == "rules":
        return {"bytes": 2 * n * es + rules, "flops": 4 * n}
    # the noise is needed where a token may be drawn: everywhere without a filter, at a few tokens with one
    noise = 0 if case["top_p"] or case["min_p"] or 0 < case["top_k"] < V else 4 * n
    return {"bytes": n * es + rules + noise + 12 * B, "flops": 8 * n}


# ---------------------------------------------------------------- the definition in 64 bits
def _nearest(v, grid):
    """Index of the grid value nearest to |v| (grid ascending; halfway goes to the even index, beyond the end to the last)."""
    a = v.abs().clamp(max=float(grid[-1]))
    hi = torch.searchsorted(grid, a.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = a - grid[lo], grid[hi] - a
    return torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def _exact_values(x, fmt):
    x = x.double()
    f64 = dict(dtype=torch.float64, device=x.device)
    e2m1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], **f64)
    e4m3 = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1], **f64)
    xb = x.view(x.shape[0], -1, BLOCK[fmt])
    big = xb.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        unit = torch.where(big > 0, torch.exp2(torch.frexp(big)[1].double() - 3).clamp(min=2.0 ** -127), torch.ones_like(big))
    else:
        row = big.amax(1, keepdim=True)
        g = torch.where(row > 0, torch.exp2(torch.frexp(row)[1].double() - 11), torch.ones_like(row))
        unit = e4m3[_nearest(big / (6 * g), e4m3)] * g
    q = torch.where(unit > 0, xb / torch.where(unit > 0, unit, torch.ones_like(unit)), torch.zeros_like(xb))
    return (e2m1[_nearest(q, e2m1)] * torch.sign(q) * unit).reshape(x.shape)


def _exact_weight(s):
    fmt, n, k = s["case"]["format"], s["case"]["n"], s["case"]["k"]
    codes = torch.empty((n, k), dtype=torch.long, device=DEV)
    codes[:, 0::2], codes[:, 1::2] = (s["packed"] % 16).long(), (s["packed"] // 16).long()
    mag = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)[codes % 8]
    v = torch.where(codes >= 8, -mag, mag)
    r, b = torch.arange(n, device=DEV)[:, None], torch.arange(k // BLOCK[fmt], device=DEV)[None]
    byte = s["scales"][r // 128, b // 4, r % 32, r % 128 // 32, b % 4].long()
    if fmt == "mxfp4":
        unit = torch.exp2(byte.double() - 127)
    else:
        exp, man = byte // 8, (byte % 8).double()
        unit = torch.where(exp > 0, (1 + man / 8) * torch.exp2(exp.double() - 7), man * 2.0 ** -9) * s["row_scale"].double()[:, None]
    return v * unit.repeat_interleave(BLOCK[fmt], 1)


def _exact_logits(s):
    z = s["logits"].double()
    B, V = z.shape
    if s["tokens"] is not None:
        every, made = torch.zeros_like(z), torch.zeros_like(z)
        at = torch.arange(s["tokens"].shape[1], device=DEV).expand(B, -1)
        row = torch.arange(B, device=DEV)[:, None].expand_as(at)
        here = at < s["lengths"][:, None]
        new = here & (at >= s["prompt_lengths"][:, None])
        one = torch.ones((), dtype=torch.float64, device=DEV)
        every.index_put_((row[here], s["tokens"][here]), one, accumulate=True)
        made.index_put_((row[new], s["tokens"][new]), one, accumulate=True)
        rep = s["repetition"].double()[:, None].expand_as(z)
        factor = torch.where(z > 0, 1 / rep, rep)
        z = torch.where(every > 0, z * factor, z) - made * s["frequency"].double()[:, None] - (made > 0) * s["presence"].double()[:, None]
    if s["bias"] is not None:
        z = z + s["bias"].double()
    if s["allowed"] is not None:
        bits = (s["allowed"].long()[..., None] >> torch.arange(32, device=DEV)) % 2
        z = z.masked_fill(bits.view(B, -1)[:, :V] == 0, -math.inf)
    return z


def _exact_sample(s):
    z = _exact_logits(s)
    B, V = z.shape
    tokens, logps = [], []
    for b in range(B):  # one row at a time, from the definition
        T = float(s["temperature"][b])
        row = z[b] / T if T > 0 else z[b]
        p = torch.softmax(row, 0)
        order = torch.argsort(row, descending=True, stable=True)
        kept = order[:int((row > -math.inf).sum())]
        if T <= 0:
            token = order[0]
        else:
            if s["top_k"] is not None and 0 < int(s["top_k"][b]) < len(kept):
                kept = kept[row[kept] >= row[kept[int(s["top_k"][b]) - 1]]]
            if s["top_p"] is not None:
                share = p[kept] / p[kept].sum()
                inside = share.cumsum(0) - share < s["top_p"][b].double()
                inside[0] = True
                kept = kept[inside]
            if s["min_p"] is not None:
                kept = kept[p[kept] >= s["min_p"][b].double() * p[order[0]]]
            token = kept[(p[kept] / s["noise"][b, kept].double()).argmax()]
        tokens.append(token)
        logps.append(torch.log_softmax(row, 0)[token])
    return {"token": torch.stack(tokens), "logprob": torch.stack(logps)}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        return {"values": _exact_values(s["x"], case["format"])}
    if case["kind"] == "linear":
        y = _exact_values(s["x"], case["format"]) @ _exact_weight(s).t()
        if case["epilogue"] == "bias":
            y = y + s["bias"].double()
        elif case["epilogue"] == "relu2":
            y = y.clamp(min=0).square()
        elif case["epilogue"] == "residual":
            y = y + s["residual"].double()
        return {"y": y}
    if case["kind"] == "rules":
        return {"logits": _exact_logits(s)}
    return _exact_sample(s)
