"""The 4-bit formats on the CPU: the load-time quantiser against the definition, the scale tiles, refusals."""
import numpy as np
import pytest
import torch

import hf_adapter_b200 as hb
from hf_adapter_b200 import _lib

from fp4_definition import BLOCK, encode


def split(packed):
    p = packed.numpy().astype(np.int64)
    return np.stack((p & 15, p >> 4), -1).reshape(p.shape[0], -1)


def inputs(kind, rows, k, seed=0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, k))
    if kind == "ties":  # values on and between the grid points of a block whose scale is a power of two
        x = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 7.0], (rows, k)) * rng.choice([-1, 1], (rows, k))
        x[:, ::16] = 6.0
    elif kind == "wide":  # blocks of very different size, some too small for any scale, some of zeros
        x = x * 2.0 ** rng.integers(-14, 14, (rows, k // 16)).repeat(16, 1)
        x[0, :32] = 0
    return x.astype(np.float16)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("kind", ["normal", "ties", "wide"])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (130, 160)])
def test_load_time_quantiser_is_the_definition(fmt, kind, rows, k):
    x = inputs(kind, rows, k)
    packed, scales, row_scale = hb.quantize_fp4_weight(torch.from_numpy(x), fmt)
    codes, byte, rs = encode(x, fmt)
    got_byte = hb.fp4_scale_rows(scales, rows, k // BLOCK[fmt]).numpy()
    assert np.array_equal(got_byte, byte)
    if fmt == "nvfp4":
        assert np.array_equal(row_scale.numpy().astype(np.float64), rs)
    else:
        assert row_scale is None
    # the sign of a zero code is free
    got, zero = split(packed), (codes & 7) == 0
    assert np.array_equal(got[~zero], codes[~zero]) and not (got[zero] & 7).any()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_not_finite_elements_mark_their_block(fmt):
    x = torch.ones(2, 64)
    x[0, 3], x[1, 40] = float("inf"), float("nan")
    packed, scales, row_scale = hb.quantize_fp4_weight(x, fmt)
    byte = hb.fp4_scale_rows(scales, 2, 64 // BLOCK[fmt])
    nan = 255 if fmt == "mxfp4" else 0x7f
    marked = torch.zeros_like(byte, dtype=torch.bool)
    marked[0, 3 // BLOCK[fmt]] = marked[1, 40 // BLOCK[fmt]] = True
    assert torch.equal(byte == nan, marked)
    if row_scale is not None:
        assert torch.equal(row_scale, torch.full((2,), 2.0 ** -10))


@pytest.mark.parametrize("rows,blocks", [(1, 2), (128, 4), (129, 5), (300, 18)])
def test_scale_tiles_round_trip(rows, blocks):
    b = torch.randint(0, 255, (rows, blocks), dtype=torch.uint8)
    t = hb.fp4_scale_tiles(b)
    assert t.shape == ((rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4)
    assert torch.equal(hb.fp4_scale_rows(t, rows, blocks), b)
    r, c = rows - 1, blocks - 1
    assert int(t.reshape(-1)[((r // 128) * t.shape[1] + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4]) == int(b[r, c])
    assert int(t.long().sum()) == int(b.long().sum())  # what pads a tile is zero


def test_sizes_and_refusals_without_a_gpu():
    L = _lib.lib
    assert L.rwkv7_fp4_scale_bytes(1, 32, 0) == 512 and L.rwkv7_fp4_scale_bytes(129, 4096, 1) == 2 * 64 * 512
    assert L.rwkv7_fp4_scale_bytes(1, 33, 0) == 0 and L.rwkv7_fp4_scale_bytes(1, 32, 2) == 0
    ws = L.rwkv7_fp4_linear_workspace_bytes(3, 64, 1)
    assert ws >= 3 * 32 + 512 + 12 and L.rwkv7_fp4_linear_workspace_bytes(3, 48, 1) == 0
    assert L.rwkv7_fp4_quant(16, 64, 16, 16, 0, 1, 64, 1, 0, 0) == _lib.ERR_INVALID      # nvfp4 needs row scales
    assert L.rwkv7_fp4_quant(16, 40, 16, 16, 16, 1, 40, 1, 0, 0) == _lib.ERR_UNSUPPORTED
    assert L.rwkv7_fp4_quant(24, 64, 16, 16, 16, 1, 64, 1, 0, 0) == _lib.ERR_ALIGN
    assert L.rwkv7_fp4_quant(16, 68, 16, 16, 16, 2, 64, 1, 0, 0) == _lib.ERR_ALIGN       # rows 136 bytes apart
    assert L.rwkv7_fp4_quant(16, 32, 16, 16, 16, 2, 64, 1, 0, 0) == _lib.ERR_INVALID     # a stride shorter than a row
    assert L.rwkv7_fp4_dequant(16, 16, 0, 16, 1, 64, 3, 0, 0) == _lib.ERR_INVALID
    lin = lambda wsb, epi=0, res=0, M=3: L.rwkv7_fp4_linear(16, 64, 16, 16, 0, 0, res, 16, 128, wsb, M, 64, 8, epi, 1, 0, 0)
    assert lin(ws - 1) == _lib.ERR_WORKSPACE and lin(ws, epi=2) == _lib.ERR_INVALID and lin(ws, res=16) == _lib.ERR_INVALID
    assert lin(ws, epi=7) == _lib.ERR_INVALID and lin(ws, M=0) == _lib.ERR_INVALID
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        hb.quantize_fp4(x)
    with pytest.raises(ValueError, match="unknown 4-bit format"):
        hb.quantize_fp4(x, "fp4")
    with pytest.raises(ValueError, match="multiple of 32"):
        hb.quantize_fp4_weight(torch.zeros(2, 48))
    w = hb.quantize_fp4_weight(torch.zeros(8, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        hb.fp4_linear(x, *w)


def test_quantize_model_takes_both_formats():
    for kind in ("mxfp4", "nvfp4"):
        m = torch.nn.Sequential(torch.nn.Linear(64, 40, bias=True), torch.nn.Linear(40, 64, bias=False))
        assert hb.quantize_model(m, kind, min_params=1) == 1  # 40 features are no multiple of 32: that one stays dense
        assert isinstance(m[0], hb.FP4Linear) and isinstance(m[1], torch.nn.Linear) and m[0].bias.shape == (40,)
        again = hb.FP4Linear(torch.nn.Linear(64, 40), format=kind)
        again.load_state_dict(m[0].state_dict())
        assert torch.equal(again.packed_fp4, m[0].packed_fp4) and torch.equal(again.fp4_scales, m[0].fp4_scales)
