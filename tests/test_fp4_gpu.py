"""Microscaled 4-bit floating point on the GPU: the quantiser bit for bit against the load-time one (which the CPU tests hold to
the definition), the projection against a product in 64 bits of the values that its operands stand for."""
import numpy as np
import pytest
import torch

import hf_adapter_b200 as hb
from hf_adapter_b200 import _lib

from fp4_definition import BLOCK

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def rnd(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, device="cuda", generator=g)).to(dtype)


def values64(x, fmt):
    """The values of quantised rows in 64 bits (host quantiser; every factor is exact in fp32, their product in fp64)."""
    packed, scales, rs = hb.quantize_fp4_weight(x, fmt)
    codes = torch.stack((packed & 15, packed >> 4), -1).view(x.shape).long()
    byte = hb.fp4_scale_rows(scales, x.shape[0], x.shape[1] // BLOCK[fmt])
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    v = grid[codes & 7] * torch.where(codes >= 8, -1.0, 1.0)
    s = torch.exp2(byte.double() - 127) if fmt == "mxfp4" else byte.view(torch.float8_e4m3fn).double() * rs.double()[:, None]
    return v * s.repeat_interleave(BLOCK[fmt], 1)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 768), (2, 96), (127, 64), (129, 160), (33, 4096), (5, 4128), (3, 16384), (2, 20512)])
def test_quantiser_bits(fmt, dtype, rows, k):
    x = rnd(rows, k, seed=rows + k) * torch.exp2(torch.randint(-6, 6, (rows, k // 16), device="cuda").float()).repeat_interleave(16, 1)
    x = x.to(DT[dtype])
    x[0, :16] = 0
    got, want = hb.quantize_fp4(x, fmt), hb.quantize_fp4_weight(x, fmt)
    assert torch.equal(got[1], want[1])
    assert got[2] is None if fmt == "mxfp4" else torch.equal(got[2], want[2])
    # a code of zero may carry either sign
    drop = lambda p: torch.stack([torch.where(n & 7 == 0, 0, n) for n in (p & 15, p >> 4)])
    assert torch.equal(drop(got[0]), drop(want[0]))
    back = hb.dequantize_fp4(*got, format=fmt, dtype=torch.float32)
    assert torch.equal(back.double(), values64(x, fmt))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_ties_and_their_neighbours(fmt, dtype):
    """Every half-way point between two codes, and the numbers of the type on both sides of it, under every mantissa of a scale."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    rows = []
    for e in range(-5, 6):
        for mantissa in range(8, 16):
            s = mantissa / 8 * 2.0 ** e
            exact = (ties * s).to(DT[dtype])  # (3 + 4 bits: exact)
            assert torch.equal(exact.double(), ties * s)
            up, down = torch.nextafter(exact, exact + 1000), torch.nextafter(exact, exact - 1000)
            top = torch.tensor([6 * s], dtype=DT[dtype])
            rows.append(torch.cat([torch.cat((top, v, -v, top)) for v in (exact, up, down, exact)]))
    x = torch.stack(rows).cuda()
    got, want = hb.quantize_fp4(x, fmt), hb.quantize_fp4_weight(x, fmt)
    drop = lambda p: torch.stack([torch.where(n & 7 == 0, 0, n) for n in (p & 15, p >> 4)])
    assert torch.equal(got[1], want[1]) and torch.equal(drop(got[0]), drop(want[0]))
    # and the product of few tokens, which quantises them itself: one channel a code position picks the values out
    if x.shape[1] == 64:
        w = hb.quantize_fp4(torch.eye(64, device="cuda"), fmt)
        for r in range(0, x.shape[0], 16):
            few, many = hb.fp4_linear(x[r:r + 4], *w, format=fmt), hb.fp4_linear(x, *w, format=fmt)[r:r + 4]
            assert torch.equal(few, many)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantiser_extremes(fmt):
    """Zeros, subnormals, the largest numbers, values that are not finite; strided and unaligned rows."""
    x = torch.zeros(8, 64, device="cuda")
    x[1] = 1e-42
    x[2] = 3.0e38
    x[3, 5], x[4, 6], x[5, 7] = float("inf"), float("-inf"), float("nan")
    x[6, 0], x[6, 33] = 2.0 ** -126, 1.0
    got, want = hb.quantize_fp4(x, fmt), hb.quantize_fp4_weight(x, fmt)
    assert torch.equal(got[1], want[1]) and (got[2] is None or torch.equal(got[2], want[2]))
    v = hb.dequantize_fp4(*got, format=fmt)
    bad = torch.zeros(8, 64 // BLOCK[fmt], dtype=torch.bool, device="cuda")
    for r, c in ((3, 5), (4, 6), (5, 7)):
        bad[r, c // BLOCK[fmt]] = True
    assert torch.equal(v.isnan(), bad.repeat_interleave(BLOCK[fmt], 1)) and not v.isinf().any()
    wide = rnd(6, 512, seed=3, dtype=torch.float16)
    for view in (wide[:, 64:256], wide[1::2, :96], wide[:, 1:65], wide.t()[:512, :].t()[:, :64]):
        a, b = hb.quantize_fp4(view, fmt), hb.quantize_fp4(view.contiguous().clone(), fmt)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    empty = hb.quantize_fp4(wide[:0], fmt)
    assert empty[0].shape == (0, 256) and hb.dequantize_fp4(*empty, format=fmt).shape == (0, 512)


def bound(xv, wv, y, dtype, extra=0.0):
    """Products of the operands are exact.  A chain of fp32 sums over groups of at least 16 products, each step off by at most
    2^-23 of what it holds (truncation), is off by at most (K / 16 + 16) 2^-23 of the sum of magnitudes; the epilogue rounds
    a few times in fp32 (8 x 2^-24) and once to the output type."""
    K = xv.shape[1]
    mag = xv.abs() @ wv.abs().t()
    half_ulp = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}[dtype]
    tiny = 2.0 ** -24 if dtype == "fp16" else 2.0 ** -126  # half-way between subnormals
    return (K / 16 + 16) * 2.0 ** -23 * mag + extra, half_ulp + 8 * 2.0 ** -24, tiny


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("m,k,n", [(1, 32, 1), (1, 64, 128), (2, 96, 5), (8, 768, 768), (16, 4096, 256), (17, 288, 129), (33, 2560, 130),
                                   (64, 1024, 384), (65, 320, 1000), (128, 544, 257), (130, 2560, 640), (257, 256, 512), (300, 1056, 1031),
                                   (513, 768, 2000), (777, 2560, 384), (1, 16384, 4096), (5, 10240, 2560), (1100, 32, 70), (2048, 64, 2048)])
def test_linear_against_64_bits(fmt, dtype, m, k, n):
    x = rnd(m, k, seed=m, dtype=DT[dtype])
    w = rnd(n, k, seed=n + 1, scale=k ** -0.5)
    xv, wv = values64(x, fmt), values64(w, fmt)
    weight = hb.quantize_fp4(w, fmt)
    bias, res = rnd(n, seed=5, dtype=DT[dtype]), rnd(m, n, seed=6, dtype=DT[dtype])
    z = xv @ wv.t()
    err, rel, tiny = bound(xv, wv, z, dtype)
    for kw, want, e in ((dict(), z, err),
                        (dict(bias=bias), z + bias.double(), err + 2.0 ** -23 * z.abs()),
                        (dict(relu2=True), z.clamp(min=0) ** 2, 2 * err * z.abs() + err ** 2),
                        (dict(bias=bias, residual=res), z + bias.double() + res.double(), err + 2.0 ** -22 * (z.abs() + bias.double().abs()))):
        y = hb.fp4_linear(x, *weight, format=fmt, **kw)
        assert y.shape == (m, n) and y.dtype == DT[dtype]
        off = (y.double() - want).abs() - (e + rel * want.abs() + tiny)
        assert float(off.max()) <= 0, (kw.keys(), float(off.max()))
    assert _lib.kernel_status() == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("m,k,n", [(1, 96, 130), (1, 4128, 1000), (2, 2560, 257), (3, 32, 5), (4, 800, 300), (5, 768, 768), (7, 544, 128),
                                   (9, 288, 65), (16, 96, 200), (16, 1056, 384), (4, 16384, 2048)])
def test_few_tokens_of_different_sizes(fmt, dtype, m, k, n):
    """Rows apart by orders of magnitude, one of zeros, one with a single large element at its end, a row stride that is not K; the
    weight is made right before the product that reads it."""
    x = rnd(m, k + 64, seed=m + k) * torch.exp2(torch.arange(m, device="cuda") % 5 * 2.0 - 4)[:, None]
    x[m // 2, k - 1] = 300
    if m > 2:
        x[1] = 0
    x = x.to(DT[dtype])[:, :k]
    w = rnd(n, k, seed=n, scale=k ** -0.5)
    xv, wv = values64(x.contiguous(), fmt), values64(w, fmt)
    want = xv @ wv.t()
    err, rel, tiny = bound(xv, wv, want, dtype)
    for _ in range(3):
        y = hb.fp4_linear(x, *hb.quantize_fp4(w, fmt), format=fmt)
        assert float(((y.double() - want).abs() - (err + rel * want.abs() + tiny)).max()) <= 0
    assert _lib.kernel_status() == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [3, 70, 600])
def test_a_bad_element_stays_in_its_row(fmt, m):
    """A row with a NaN or an infinity gives a row of NaN; a weight's gives a column; everything else keeps its bits."""
    x, w = rnd(m, 256, seed=1, dtype=torch.float16), rnd(200, 256, seed=2)
    clean = hb.fp4_linear(x, *hb.quantize_fp4(w, fmt), format=fmt)
    x2, w2 = x.clone(), w.clone()
    x2[1, 7], x2[2, 250], w2[150, 100] = float("nan"), float("inf"), float("-inf")
    y = hb.fp4_linear(x2, *hb.quantize_fp4(w2, fmt), format=fmt)
    assert y[1].isnan().all() and y[2].isnan().all() and y[:, 150].isnan().all()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[1], keep[2], keep[:, 150] = False, False, False
    assert torch.equal(y[keep], clean[keep])
    assert torch.equal(hb.fp4_linear(torch.zeros_like(x), *hb.quantize_fp4(w, fmt), format=fmt), torch.zeros_like(y))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_calls_repeat_bit_for_bit_and_on_another_stream(m):
    x, w = rnd(m, 2560, seed=1, dtype=torch.bfloat16), hb.quantize_fp4(rnd(1000, 2560, seed=2))
    y = hb.fp4_linear(x, *w)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        others = [hb.fp4_linear(x, *w) for _ in range(5)]
    st.synchronize()
    assert all(torch.equal(o, y) for o in others)
    # shapes and strides: a batch of sequences, a slice of a wider tensor, a given output
    assert torch.equal(hb.fp4_linear(x.view(1, m, 2560), *w), y[None])
    wide = torch.cat((x, x), 1)
    assert torch.equal(hb.fp4_linear(wide[:, 2560:], *w), y)
    out = torch.empty_like(y)
    assert hb.fp4_linear(x, *w, out=out) is out and torch.equal(out, y)
    assert hb.fp4_linear(x[:0], *w).shape == (0, 1000)


def test_refusals():
    x, w = rnd(4, 64, dtype=torch.float16), hb.quantize_fp4(rnd(40, 64))
    mx = hb.quantize_fp4(rnd(40, 64), "mxfp4")
    with pytest.raises(ValueError, match="features"):
        hb.fp4_linear(x[:, :32], *w)
    with pytest.raises(ValueError, match="takes no residual"):
        hb.fp4_linear(x, *w, relu2=True, residual=rnd(4, 40, dtype=torch.float16))
    with pytest.raises(ValueError, match="residual must"):
        hb.fp4_linear(x, *w, residual=rnd(4, 40))
    with pytest.raises(ValueError, match="bias must"):
        hb.fp4_linear(x, *w, rnd(39, dtype=torch.float16))
    with pytest.raises(ValueError, match="None for 'mxfp4'"):
        hb.fp4_linear(x, *w, format="mxfp4")
    with pytest.raises(ValueError, match="scales must"):
        hb.fp4_linear(x, mx[0], mx[1][:, :0], format="mxfp4")
    with pytest.raises(ValueError, match="row_scale must"):
        hb.fp4_linear(x, *w[:2], w[2].half())
    with pytest.raises(ValueError, match="packed must"):
        hb.dequantize_fp4(w[0].int(), *w[1:])
    with pytest.raises(ValueError, match="contiguous"):
        hb.dequantize_fp4(torch.cat((w[0], w[0]), 1)[:, ::2], *w[1:])
    with pytest.raises(ValueError, match="out must"):
        hb.fp4_linear(x, *w, out=torch.empty(4, 41, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="dtype"):
        hb.fp4_linear(x.double(), *w)
    with pytest.raises(RuntimeError, match="CUDA"):
        hb.fp4_linear(x, *(t.cpu() for t in w))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_model_decodes_with_4_bit_projections(fmt):
    """The decode graph, the eager step and the prefill of a model whose projections and head are in 4 bits: the graph replays the
    step's bits; the logits point where the dense model's do (both operands lose about a tenth of their size to the
    format, so the cosine stays far above 0.9)."""
    torch.manual_seed(2)
    cfg = hb.NativeRWKV7Config(vocab_size=512, hidden_size=256, num_hidden_layers=2, num_heads=4, head_dim=64, intermediate_size=1024,
                               decay_low_rank_dim=32, a_low_rank_dim=32, v_low_rank_dim=16, gate_low_rank_dim=32)
    model = hb.RWKV7ForCausalLM(cfg)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(0.2 * torch.randn_like(p) if p.dim() < 2 else torch.randn_like(p) * p.shape[-1] ** -0.5)
    model = model.half().cuda().eval()
    ids = torch.randint(0, 512, (3, 12), device="cuda")
    dense = model(ids, logits_to_keep=1).logits[:, -1].double()
    assert hb.quantize_model(model, fmt, min_params=1, skip=()) == 13
    prefill = model(ids, logits_to_keep=1).logits[:, -1].double()
    caches = [model.new_cache(3), model.new_cache(3)]
    for t in range(12):
        eager = model.rwkv7_forward_token(ids[:, t], caches[0], use_graph=False)
        graph = model.rwkv7_forward_token(ids[:, t], caches[1], use_graph=True)
    assert torch.equal(eager, graph)
    cos = lambda a, b: float((a * b).sum() / a.norm() / b.norm())
    assert cos(prefill, dense) > 0.9 and cos(eager.double(), dense) > 0.9 and cos(eager.double(), prefill) > 0.9
    out = model.generate(ids, max_new_tokens=4)
    assert out.shape == (3, 16) and np.array_equal(out[:, :12].cpu().numpy(), ids.cpu().numpy())
