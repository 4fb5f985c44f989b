"""Rules on logits and the draw of a token against their definition in 64 bits, row by row (NumPy).

The draw has a token for an answer, so inputs are made on grids on which no decision is close: logits are multiples of 1/8 and
the noise is spread over distinct values a factor apart; where the decision between two tokens is nearer than 1e-4 (relative;
a hundred times the rounding of fp32 exp and sums) the test asks only for one of the near ones."""
import math

import numpy as np
import pytest
import torch

import hf_adapter_b200 as hb

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
F32 = np.float32


def make_logits(B, V, dtype, seed=0, step=0.125):
    rng = np.random.default_rng(seed)
    z = np.round(rng.standard_normal((B, V)) * 3 / step) * step
    hot = rng.integers(0, V, (B, min(V, 8)))
    for b in range(B):
        z[b, hot[b]] = np.round(rng.uniform(4, 12, hot.shape[1]) / step) * step
    return torch.from_numpy(z).to(DT[dtype]).cuda()


def rules64(z, tokens=None, lengths=None, prompt=None, rep=None, pres=None, freq=None, bias=None, allowed=None):
    z = z.double().cpu().numpy().copy()
    B, V = z.shape
    for b in range(B):
        if tokens is not None:
            ids = tokens[b, :int(lengths[b])]
            ok = (ids >= 0) & (ids < V)
            seen = np.unique(ids[ok])
            c = np.zeros(V)
            np.add.at(c, ids[int(prompt[b]):][ok[int(prompt[b]):]], 1)
            s = z[b, seen]
            z[b, seen] = np.where(s > 0, s / rep[b], s * rep[b])
            z[b] = z[b] - freq[b] * c - pres[b] * (c > 0)
        if bias is not None:
            z[b] = z[b] + (bias if bias.ndim == 1 else bias[b])
        if allowed is not None:
            a = allowed if allowed.ndim == 1 else allowed[b]
            v = np.arange(V)
            z[b, (a[v >> 5].astype(np.int64) >> (v & 31)) & 1 == 0] = -np.inf
    return z


def random_rules(B, V, L, seed, bias="none", mask=False, i64=True):
    rng = np.random.default_rng(seed)
    kw, ref = {}, {}
    if L:
        tok = (V * rng.random((B, L)) ** 3).astype(np.int64)
        tok[rng.random((B, L)) < 0.1] = -1  # padding
        tok[rng.random((B, L)) < 0.02] = V  # an id outside the vocabulary
        lens = rng.integers(0, L + 1, B)
        lens[0] = L
        prompt = (lens * rng.random(B)).astype(np.int64)
        pick = lambda choices: rng.choice(np.array(choices, F32), B)
        rep, pres, freq = pick([1.0, 1.25, 2.0, 0.5]), pick([0, 0.5, -0.25]), pick([0, 0.125, 0.75])
        ref.update(tokens=tok, lengths=lens, prompt=prompt, rep=rep, pres=pres, freq=freq)
        dev = lambda a, t: torch.from_numpy(a).to(t).cuda()
        kw.update(tokens=dev(tok, torch.int64 if i64 else torch.int32), lengths=dev(lens, torch.int32), prompt_lengths=dev(prompt, torch.int32),
                  repetition_penalty=dev(rep, torch.float32), presence_penalty=dev(pres, torch.float32),
                  frequency_penalty=dev(freq, torch.float32))
    if bias != "none":
        b = np.round(rng.standard_normal((V,) if bias == "shared" else (B, V)) * 8) / 8
        ref["bias"], kw["bias"] = b, torch.from_numpy(b).float().cuda()
    if mask:
        m = rng.integers(-2 ** 31, 2 ** 31, (B, (V + 31) // 32)).astype(np.int32)
        m &= rng.integers(-2 ** 31, 2 ** 31, m.shape).astype(np.int32)
        ref["allowed"], kw["allowed"] = m, torch.from_numpy(m).cuda()
    return kw, ref


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("B,V,L,bias,mask", [(1, 1, 0, "none", False), (1, 1, 3, "shared", True), (2, 7, 5, "rows", True), (3, 1000, 0, "shared", False),
                                             (3, 1001, 64, "none", True), (5, 8191, 1, "rows", False), (2, 8193, 3000, "shared", True),
                                             (1, 65536, 300, "none", False), (4, 50277, 777, "rows", True), (2, 200003, 20000, "none", True)])
def test_rules_against_64_bits(dtype, B, V, L, bias, mask):
    """fp32 steps: a quotient, a product, two differences and a sum, each off by half an ulp of a number below 2^7 (2^-18), and
    one rounding to the output type."""
    z = make_logits(B, V, dtype, seed=V)
    kw, ref = random_rules(B, V, L, V + L, bias, mask, i64=L % 2 == 0)
    want = rules64(z, **ref)
    got = hb.process_logits(z, **kw)
    assert got.dtype == z.dtype and got.shape == z.shape
    g = got.double().cpu().numpy()
    gone = np.isneginf(want)
    assert np.array_equal(np.isneginf(g), gone)
    half = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 0.0}[dtype]
    want, g = want[~gone], g[~gone]
    size = np.maximum(np.abs(want), 1.0)
    assert np.all(np.abs(g - want) <= half * np.abs(want) + 5 * 2.0 ** -24 * np.maximum(size * 4, 2.0 ** 7))
    # in place, into a wider tensor, from an unaligned view: the same bits
    wide = torch.full((B, V + 3), 7.0, device="cuda", dtype=z.dtype)
    wide[:, 1:V + 1] = z
    hb.process_logits(wide[:, 1:V + 1], **kw, out=wide[:, 1:V + 1])
    assert torch.equal(wide[:, 1:V + 1], got) and (wide[:, 0] == 7).all() and (wide[:, V + 1:] == 7).all()
    into = torch.full((B, V + 2), 7.0, device="cuda", dtype=z.dtype)
    hb.process_logits(z, **kw, out=into[:, 2:])
    assert torch.equal(into[:, 2:], got) and (into[:, :2] == 7).all()


def test_masked_places_hide_whatever_is_there():
    z = torch.zeros(2, 70, device="cuda", dtype=torch.float16)
    z[0, 3], z[0, 40], z[1, 5] = float("nan"), float("inf"), torch.finfo(torch.float16).min
    allowed = torch.full((2, 3), -1, device="cuda", dtype=torch.int32)
    allowed[0, 0] &= ~(1 << 3)
    allowed[0, 1] &= ~(1 << 8)
    allowed[1] = 0
    out = hb.process_logits(z, allowed=allowed)
    assert torch.isneginf(out[0, [3, 40]]).all() and (out[0].isinf().sum() == 2) and torch.isneginf(out[1]).all()
    bias = torch.zeros(70, device="cuda")
    bias[5], bias[6] = torch.finfo(torch.float32).min, -float("inf")
    out = hb.process_logits(z[1:], bias=bias)
    assert torch.isneginf(out[0, 5:7]).all() and (out[0, 7:] == 0).all()
    assert hb.process_logits(z[:0]).shape == (0, 70)


# ---------------------------------------------------------------- the draw
def noise_for(B, V, seed=0):
    """Distinct values a factor of at least 1.001 apart within a row, distributed about as Exp(1) variates are."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(B, V, device="cuda").exponential_(generator=g)


def candidates64(z, noise, T, k, p, mp, eps=1e-4):
    """All tokens that the definition's decisions allow when each of them may be off by ``eps`` (relative)."""
    V = z.shape[0]
    if np.all(np.isneginf(z)):
        return {-1}, None
    if T <= 0:
        return {int(np.argmax(z))}, z
    z = z / T
    order = np.argsort(-z, kind="stable")
    live = order[~np.isneginf(z[order])]
    e = np.exp(z - z[order[0]])
    kept = live
    if 0 < k < V and k < len(live):
        kept = live[z[live] >= z[live[k - 1]]]
    sure, maybe = np.ones(len(kept), bool), np.ones(len(kept), bool)
    if p < 1:
        before = np.concatenate(([0], np.cumsum(e[kept])[:-1])) / e[kept].sum()
        sure, maybe = before < p - 1e-5, before < p + 1e-5
        sure[0] = maybe[0] = True
    sure, maybe = sure & (e[kept] >= mp * (1 + eps)), maybe & (e[kept] >= mp * (1 - eps))
    sure[0] |= mp <= 1
    score = e[kept] / noise[kept]
    best = score[sure].max() if sure.any() else 0.0
    return set(int(v) for v in kept[maybe & (score >= best * (1 - eps))]), z


def check_draw(z, noise, got, logprob, T, k, p, mp, ref=None):
    zz = rules64(z, **(ref or {}))
    n = noise.double().cpu().numpy()
    for b in range(z.shape[0]):
        at = lambda v: float(v[b]) if isinstance(v, (np.ndarray, list)) else float(v)
        ok, zt = candidates64(zz[b], n[b], at(T), int(at(k)), at(p), at(mp))
        tok = int(got[b])
        assert tok in ok, (b, tok, ok)
        if tok < 0:
            assert math.isinf(float(logprob[b])) and float(logprob[b]) < 0
            continue
        top = zt.max()
        want = zt[tok] - top - np.log(np.exp(zt - top).sum())
        # z is off by an ulp of its size (2^-23 x 64 / T at most), exp and the sums by less
        assert abs(float(logprob[b]) - want) <= 2e-5 + 1e-6 * abs(want), (b, float(logprob[b]), want)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("V", [1, 2, 7, 129, 1000, 4097, 8192, 50277, 65536, 200003])
@pytest.mark.parametrize("T,k,p,mp", [(1.0, 0, 1.0, 0.0), (0.5, 50, 1.0, 0.0), (1.5, 0, 0.9, 0.0), (0.75, 40, 0.8, 0.05), (2.0, 1, 0.5, 0.0),
                                      (1.0, 100000, 0.999, 0.0), (0.0, 3, 0.5, 0.0), (8.0, 1000, 0.3, 0.0), (1.0, 0, 0.0, 0.0),
                                      (0.03125, 0, 0.99, 0.001), (1.0, 3, 1.0, 1.0)])
def test_draw_against_64_bits(dtype, V, T, k, p, mp):
    B = 5 if V < 60000 else 2
    z, noise = make_logits(B, V, dtype, seed=V), noise_for(B, V, seed=V + k)
    got, lp = hb.sample_tokens(z, noise, temperature=T, top_k=k, top_p=p, min_p=mp, return_logprobs=True)
    assert got.dtype == torch.int64 and got.shape == (B,)
    check_draw(z, noise, got, lp, T, k, p, mp)
    again = hb.sample_tokens(z, noise, temperature=T, top_k=k, top_p=p, min_p=mp)
    assert torch.equal(got, again)


@pytest.mark.parametrize("B,V,L,bias,mask", [(9, 1000, 50, "shared", True), (16, 50277, 300, "rows", True), (64, 8192, 2000, "none", False),
                                             (150, 4099, 17, "none", True), (300, 515, 0, "shared", True)])
def test_draw_with_rules_and_a_parameter_per_row(B, V, L, bias, mask):
    z, noise = make_logits(B, V, "fp16", seed=B), noise_for(B, V, seed=B)
    kw, ref = random_rules(B, V, L, B, bias, mask)
    rng = np.random.default_rng(B)
    T, p, mp = (rng.choice(np.array(c, F32), B) for c in ([0, 0.5, 1, 1.25], [0.25, 0.9, 1.0], [0, 0.01]))
    k = rng.choice([0, 1, 5, 400], B)
    dev = lambda a: torch.from_numpy(a).cuda()
    got, lp = hb.sample_tokens(z, noise, temperature=dev(T), top_k=dev(k), top_p=dev(p), min_p=dev(mp), return_logprobs=True, **kw)
    check_draw(z, noise, got, lp, T, k, p, mp, ref)
    # the rules in front as their own call: fp32 logits are not rounded on the way, so the answer is the same
    z32 = hb.process_logits(z.float(), **kw)
    two, lp2 = hb.sample_tokens(z32, noise, temperature=dev(T), top_k=dev(k), top_p=dev(p), min_p=dev(mp), return_logprobs=True)
    assert torch.equal(got, two) and torch.equal(lp, lp2)


def test_equal_values_go_by_index():
    """Ties by the thousand: the whole row, a few levels, at the cut of top-p; top-k keeps every tie."""
    V = 65536
    z = torch.zeros(4, V, device="cuda")
    z[1] = torch.arange(V, device="cuda") % 3 * -0.5
    z[2, V // 2:] = -1
    z[3, 17] = 3
    noise = noise_for(4, V)
    # temperature 0 takes the first of the largest
    assert hb.sample_tokens(z, temperature=1.0).tolist() == [0, 0, 0, 17]
    # p = 1/4 of V equal tokens: the first V / 4 of them (one more or fewer where the share is met exactly)
    t = hb.sample_tokens(z[:1], noise[:1], top_p=0.25)
    assert int(t) == int((1 / noise[0, :V // 4]).argmax())
    # the draw over row 1 at p = 0.3: all of the first level have 1 / (1 + e^-.5 + e^-1) = 0.5065 of the mass; 0.3 of it is reached after
    # a share 0.3 / 0.5065 of that level, lowest index first
    n0 = (V + 2) // 3
    keep = 3 * torch.arange(int(0.3 / (1 / (1 + math.exp(-.5) + math.exp(-1))) * n0) - 2, device="cuda")
    t = int(hb.sample_tokens(z[1:2], noise[1:2], top_p=0.3))
    scores = 1 / noise[1, keep]
    assert t == int(keep[scores.argmax()])
    # top-k = 1 among equals keeps them all
    t = hb.sample_tokens(z[:1], noise[:1], top_k=1)
    assert int(t) == int((1 / noise[0]).argmax())
    t = hb.sample_tokens(z[3:], noise[3:], top_k=2)
    s = torch.exp(z[3] - 3) / noise[3]
    assert int(t) == int(s.argmax())


def test_values_that_are_not_finite_and_empty_rows():
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[nan, nan, nan, nan], [nan, 1, -inf, 0], [inf, 0, inf, 1], [-inf, -inf, -inf, -inf], [65504, -65504, 0, -0.0],
                      [-inf, -inf, -5, -inf]], device="cuda")
    noise = torch.tensor([[1.0, 2, 0.5, 3]], device="cuda").repeat(6, 1)
    for dt in DT.values():
        tok, lp = hb.sample_tokens(z.to(dt), noise, top_k=3, top_p=0.9, return_logprobs=True)
        assert tok.tolist() == [-1, 1, 2, -1, 0, 2]
        assert torch.isneginf(lp[[0, 3]]).all() and torch.isfinite(lp[[1, 2, 4, 5]]).all() and float(lp[5]) == 0
        assert hb.sample_tokens(z.to(dt)).tolist() == [-1, 1, 0, -1, 0, 2]
    assert hb.sample_tokens(z[:0]).shape == (0,)
    allowed = torch.zeros(1, 1, device="cuda", dtype=torch.int32)
    assert hb.sample_tokens(z, noise, allowed=allowed).tolist() == [-1] * 6
    # three values that the temperature drives out of range are equal then; half of their mass is the first two, 1 / noise decides
    huge = torch.tensor([[1e38, 3e38, -3e38, 2e38]], device="cuda")
    assert int(hb.sample_tokens(huge, noise[:1], temperature=0.01, top_p=0.5)) == 0
    # one draw of noise that is zero, one that is not a number
    odd = torch.tensor([[1.0, 0.0, 1.0, nan]], device="cuda")
    assert int(hb.sample_tokens(torch.zeros(1, 4, device="cuda"), odd)) == 1
    assert int(hb.sample_tokens(torch.zeros(1, 4, device="cuda"), odd * nan)) == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_rows_of_the_lowest_value(dtype):
    """A mask of the type's lowest number instead of -inf: beside other values it takes all probability away, alone it is a row of
    equal tokens, at every temperature."""
    V, low = 5000, torch.finfo(DT[dtype]).min
    z = torch.full((3, V), low, device="cuda", dtype=DT[dtype])
    z[1, 4000:4003] = 1
    z[2, ::2] = -float("inf")
    noise = noise_for(3, V, seed=3)
    want = [int(noise[0].argmin()), 4000 + int(noise[1, 4000:4003].argmin()), 1 + 2 * int(noise[2, 1::2].argmin())]
    for T in (0.25, 1.0, 4.0):
        for kw in (dict(), dict(top_k=V - 1), dict(min_p=0.5), dict(top_p=0.9999999, min_p=0.1)):
            tok, lp = hb.sample_tokens(z, noise, temperature=T, return_logprobs=True, **kw)
            assert tok.tolist() == want, (T, kw)
            assert torch.allclose(lp.cpu(), -torch.log(torch.tensor([5000.0, 3.0, 2500.0])), atol=1e-5)
    assert hb.sample_tokens(z).tolist() == [0, 4000, 1]


def test_close_values_in_one_bin():
    """Thousands of neighbouring floats between the cuts: the search has to go down to single keys."""
    V = 30000
    g = torch.Generator(device="cuda").manual_seed(1)
    z = (10 + torch.randperm(V, device="cuda", generator=g) * 2.0 ** -20)[None]  # ulp of 8..16 is 2^-20: neighbours all
    noise = noise_for(1, V, seed=5)
    order = z[0].argsort(descending=True)
    for k in (1, 2, 100, 29999):
        keep = order[:k]
        s = torch.exp(z[0, keep].double() - float(z.max())) / noise[0, keep].double()
        assert int(hb.sample_tokens(z, noise, top_k=k)) == int(keep[s.argmax()])
    tiny = (torch.arange(V, device="cuda").float() * 1e-42)[None]  # subnormal numbers: keys near 0, all in the first bin
    order = tiny[0].argsort(descending=True)
    for k in (1, 7, 1000):
        keep = order[:k]
        assert int(hb.sample_tokens(tiny, noise, top_k=k)) == int(keep[(1 / noise[0, keep]).argmax()])


@pytest.mark.parametrize("B", [2, 40])
@pytest.mark.parametrize("dtype,width", [("fp32", 1e-3), ("fp32", 0.25), ("fp16", 0.25), ("bf16", 1.5), ("fp32", 6.0)])
@pytest.mark.parametrize("k,p,mp", [(0, 0.9, 0.0), (0, 0.1, 0.0), (3000, 1.0, 0.0), (5000, 0.5, 0.0), (0, 0.6, 0.7)])
def test_draw_of_flat_rows(B, dtype, width, k, p, mp):
    """More tokens near the cut than can be sorted, around zero (where values have the most keys), a third of them masked."""
    V = 40000
    rng = np.random.default_rng(7)
    z = rng.uniform(-0.5, 0.5, (B, V)) * width
    z[rng.random((B, V)) < 1 / 3] = -np.inf
    z = torch.from_numpy(z).to(DT[dtype]).cuda()
    noise = noise_for(B, V, seed=11)
    got, lp = hb.sample_tokens(z, noise, top_k=k, top_p=p, min_p=mp, return_logprobs=True)
    check_draw(z, noise, got, lp, 1.0, k, p, mp)


def test_next_token_is_what_tensor_code_draws():
    """``sample_next_token`` from one generator against the same steps in tensor code, the reference's order: temperature, top-k, top-p,
    a multinomial draw."""
    z = make_logits(32, 4096, "fp16", seed=3)
    for T, k, p in ((1.0, 0, 1.0), (0.7, 50, 1.0), (1.2, 0, 0.9), (0.9, 200, 0.8)):
        gen = lambda: torch.Generator(device="cuda").manual_seed(11)
        got = hb.sample_next_token(z, temperature=T, top_k=k, top_p=p, generator=gen())
        s = z.float() / T
        if k:
            s = s.masked_fill(s < torch.topk(s, k, dim=-1).values[:, -1:], float("-inf"))
        if p < 1:
            sz, idx = torch.sort(s, dim=-1, descending=True, stable=True)
            pr = torch.softmax(sz, -1)
            sz = sz.masked_fill(pr.cumsum(-1) - pr >= p, float("-inf"))
            s = torch.full_like(s, float("-inf")).scatter(-1, idx, sz)
        want = torch.multinomial(torch.softmax(s, -1), 1, generator=gen()).squeeze(-1)
        assert torch.equal(got, want)


def test_draws_follow_the_distribution():
    """100000 draws over 6 tokens: shares within 5 standard deviations of the probabilities."""
    z = torch.tensor([[2.0, 1.0, 0.0, 0.0, -1.0, -8.0]], device="cuda").repeat(100000, 1)
    g = torch.Generator(device="cuda").manual_seed(0)
    tok = hb.sample_tokens(z, torch.empty_like(z).exponential_(generator=g), temperature=1.25)
    p = torch.softmax(z[0].double() / 1.25, 0)
    share = torch.bincount(tok, minlength=6).double() / 100000
    assert ((share - p).abs() <= 5 * (p * (1 - p) / 100000).sqrt() + 1e-9).all()


def test_streams_and_strides():
    z, noise = make_logits(6, 3001, "bf16", seed=1), noise_for(6, 3001)
    want = hb.sample_tokens(z, noise, top_p=0.9)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = [hb.sample_tokens(z, noise, top_p=0.9) for _ in range(3)]
    st.synchronize()
    assert all(torch.equal(g, want) for g in got)
    wide = torch.zeros(6, 2, 3002, device="cuda", dtype=torch.bfloat16)
    wide[:, 1, 1:] = z
    assert torch.equal(hb.sample_tokens(wide[:, 1, 1:], noise, top_p=0.9), want)
    assert torch.equal(hb.sample_tokens(z.t().contiguous().t(), noise.t().contiguous().t(), top_p=0.9), want)


def test_refusals():
    z = torch.zeros(3, 40, device="cuda")
    tok = torch.zeros(3, 5, device="cuda", dtype=torch.int64)
    for bad, match in ((dict(tokens=tok[:2]), "tokens must"), (dict(tokens=tok.float()), "tokens must"), (dict(lengths=tok[:, 0].int()), "need tokens"),
                       (dict(tokens=tok, lengths=tok[:2, 0].int()), "lengths must"), (dict(tokens=tok, repetition_penalty=0.0), "positive"),
                       (dict(tokens=tok, presence_penalty=torch.zeros(2, device="cuda")), "presence_penalty must"),
                       (dict(bias=torch.zeros(41, device="cuda")), "bias must"), (dict(bias=torch.zeros(40, device="cuda").half()), "bias must"),
                       (dict(allowed=torch.zeros(3, 1, device="cuda", dtype=torch.int32)), "allowed must"),
                       (dict(allowed=torch.zeros(3, 2, device="cuda", dtype=torch.int64)), "allowed must")):
        for f in (hb.process_logits, hb.sample_tokens):
            with pytest.raises(ValueError, match=match):
                f(z, **bad)
    with pytest.raises(ValueError, match="noise must"):
        hb.sample_tokens(z, torch.zeros(3, 41, device="cuda"))
    with pytest.raises(ValueError, match="noise must"):
        hb.sample_tokens(z, torch.zeros(3, 40, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="top_k must"):
        hb.sample_tokens(z, z + 1, top_k=torch.ones(2, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError, match="logits must"):
        hb.sample_tokens(z[0])
    with pytest.raises(ValueError, match="out must"):
        hb.process_logits(z, out=torch.zeros(3, 41, device="cuda"))
    with pytest.raises(ValueError, match="dtype"):
        hb.sample_tokens(z.double())
    with pytest.raises(ValueError, match="does not fit"):
        hb.sample_tokens(torch.zeros(1, 1 << 20, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA"):
        hb.process_logits(z.cpu())
