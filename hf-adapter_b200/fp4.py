"""Microscaled 4-bit floating point: quantisation, and projections whose operands both stay in 4 bits on the block-scaled
tensor cores (csrc/fp4.cu, csrc/fp4_umma.cu; the formats are defined in include/rwkv7_b200.h).

* ``"mxfp4"``: E2M1 elements, 32 of them share a power of two.
* ``"nvfp4"``: E2M1 elements, 16 of them share an E4M3 scale, a row shares an fp32 factor.

A quantised tensor is three tensors: ``packed [rows, K/2] uint8`` (even element in the low nibble), ``scales`` in the tiles
that the tensor cores read (``fp4_scale_tiles`` / ``fp4_scale_rows`` convert from and to ``[rows, K/block]``), and
``row_scale [rows] fp32`` (None for ``"mxfp4"``).  ``quantize_fp4_weight`` is load-time tensor code (plain torch, any device)
with the kernel's bits.  The reference has no such format; there is no CPU forward.
"""
from __future__ import annotations

import torch

from . import _lib
from ._util import dt_code, ptr, require_cuda, stream_ptr

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def _format(name) -> int:
    try:
        return FORMATS[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown 4-bit format {name!r}: 'mxfp4' or 'nvfp4'") from None


def _tile_shape(rows: int, K: int, format: str):
    return (rows + 127) // 128, (K // BLOCK[format] + 3) // 4, 32, 4, 4


def fp4_scale_tiles(scale_bytes):
    """Scale bytes ``[rows, K/block] uint8`` of a weight made elsewhere, in tiles (load-time tensor code, any device)."""
    rows, blocks = (int(v) for v in scale_bytes.shape)
    rt, kt = (rows + 127) // 128, (blocks + 3) // 4
    full = torch.zeros((rt * 128, kt * 4), device=scale_bytes.device, dtype=torch.uint8)
    full[:rows, :blocks] = scale_bytes
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous()


def fp4_scale_rows(scales, rows: int, blocks: int):
    """The bytes of scale tiles as ``[rows, blocks]``."""
    return scales.permute(0, 3, 2, 1, 4).reshape(int(scales.shape[0]) * 128, -1)[:rows, :blocks].contiguous()


def _rows2d(x, K, what):
    """``x`` as ``[rows, K]`` whose rows the kernels can load: unit stride, 16-byte aligned (a copy where they are not)."""
    if K <= 0 or K % 32:
        raise ValueError(f"{what}: the last dimension must be a positive multiple of 32 (got {tuple(x.shape)})")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    ld, unit = x2.stride()
    if unit == 1 and x2.data_ptr() % 16 == 0 and (x2.shape[0] <= 1 or (ld >= K and ld * x2.element_size() % 16 == 0)):
        return x2, ld if ld >= K else K
    return x2.clone(memory_format=torch.contiguous_format), K


def _on_gpu(what, *tensors):
    """All on one GPU; the checks of ``require_cuda`` by device index, which cost a call of one token less."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and (dev < 0 or t.get_device() != dev):
            require_cuda(*tensors, what=what)


def quantize_fp4(x, format: str = "nvfp4"):
    """``x [..., K]`` (fp16 / bf16 / fp32, K a multiple of 32) to ``(packed [rows, K/2] uint8, scales, row_scale)``."""
    f = _format(format)
    _on_gpu("quantize_fp4", x)
    dt = dt_code(x)
    K = x.shape[-1] if x.dim() else 0
    x2, ld = _rows2d(x, K, "quantize_fp4")
    rows = x2.shape[0]
    packed = x2.new_empty((rows, K // 2), dtype=torch.uint8)
    scales = packed.new_empty(_tile_shape(rows, K, format))
    row_scale = x2.new_empty(rows, dtype=torch.float32) if f else None
    if rows:
        _lib.check(_lib.lib.rwkv7_fp4_quant(x2.data_ptr(), ld, packed.data_ptr(), scales.data_ptr(), ptr(row_scale), rows, K, f, dt,
                                            stream_ptr(x2)), "quantize_fp4")
    return packed, scales, row_scale


def quantize_fp4_weight(weight, format: str = "nvfp4"):
    """``quantize_fp4`` of a ``[out, in]`` weight as plain tensor code, for weights that are not on a GPU yet."""
    f = _format(format)
    if weight.dim() != 2 or weight.shape[1] == 0 or weight.shape[1] % 32:
        raise ValueError(f"quantize_fp4_weight requires a rank-2 weight whose in_features are a positive multiple of 32, got {tuple(weight.shape)}")
    w = weight.detach().float()
    rows, K = (int(v) for v in w.shape)
    exponent = lambda a: (a.view(torch.int32) >> 23)  # biased; of a magnitude
    power = lambda e: (e << 23).view(torch.float32)   # 2^(e - 127), e in 1..254
    mag = torch.where(torch.isfinite(w), w.abs(), 0.0).view(rows, -1, BLOCK[format])
    finite = torch.isfinite(w).view_as(mag).all(-1)
    amax = mag.amax(-1)
    if f == 0:
        byte = (exponent(amax.contiguous()) - 2).clamp_(min=0)
        q = w.view_as(mag) * power(254 - byte)[..., None]
        byte, row_scale = torch.where(finite, byte, 255).to(torch.uint8), None
    else:
        top = amax.amax(-1)
        ge = torch.where(top > 0, (exponent(top).clamp(min=1) - 10).clamp(min=1), 127).int()
        row_scale, inv = power(ge), power(254 - ge)[:, None]
        e4m3 = (amax * inv * torch.tensor(1.0 / 6.0, device=w.device)).to(torch.float8_e4m3fn)
        s = e4m3.float()[..., None]
        q = torch.where(s > 0, w.view_as(mag) * inv[..., None] / s, 0.0)
        byte = torch.where(finite, e4m3.view(torch.uint8), 0x7f).to(torch.uint8)
    a = torch.where(q.isnan(), 6.0, q.abs())
    code = sum((a > t).to(torch.uint8) if strict else (a >= t).to(torch.uint8)
               for t, strict in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)))
    code = (code | (torch.signbit(q).to(torch.uint8) << 3)).view(rows, K)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), fp4_scale_tiles(byte), row_scale


def _check_quantised(packed, scales, row_scale, format, what):
    """The kernels take their sizes from ``packed``: everything else has to hold as much."""
    f = _format(format)
    shape = packed.shape
    if len(shape) != 2 or packed.dtype is not torch.uint8 or shape[1] == 0 or shape[1] % 16:
        raise ValueError(f"{what}: packed must be [rows, K/2] uint8 with K a positive multiple of 32, got {tuple(shape)} {packed.dtype}")
    rows, K = shape[0], 2 * shape[1]
    tiles = _tile_shape(rows, K, format)
    if scales.dtype is not torch.uint8 or scales.shape != tiles:
        raise ValueError(f"{what}: scales must be uint8 tiles {tiles}, got {tuple(scales.shape)} {scales.dtype}")
    if row_scale is not None and (f == 0 or row_scale.dtype is not torch.float32 or row_scale.shape != (rows,)):
        raise ValueError(f"{what}: row_scale must be [{rows}] float32, and None for 'mxfp4'")
    if not (packed.is_contiguous() and scales.is_contiguous() and (row_scale is None or row_scale.is_contiguous())):
        raise ValueError(f"{what}: packed, scales and row_scale must be contiguous")
    return f, rows, K


def dequantize_fp4(packed, scales, row_scale=None, *, format: str = "nvfp4", dtype=torch.float32):
    """The values ``[rows, K]`` in ``dtype`` (formed in fp32, rounded once)."""
    _on_gpu("dequantize_fp4", packed, scales, row_scale)
    f, rows, K = _check_quantised(packed, scales, row_scale, format, "dequantize_fp4")
    out = packed.new_empty((rows, K), dtype=dtype)
    dt = dt_code(out)
    if rows:
        _lib.check(_lib.lib.rwkv7_fp4_dequant(packed.data_ptr(), scales.data_ptr(), ptr(row_scale), out.data_ptr(), rows, K, f, dt,
                                              stream_ptr(packed)), "dequantize_fp4")
    return out


def fp4_linear(x, packed, scales, row_scale=None, bias=None, *, format: str = "nvfp4", relu2: bool = False, residual=None, out=None):
    """``x [..., K] @ weight.T (+ bias)`` then ``relu(.)**2`` or ``+ residual``, both operands in ``format``: ``x`` is
    quantised on the way, as ``quantize_fp4`` does it; the weight is ``quantize_fp4``'s three tensors.  Sums are fp32 and
    rounded once, after the epilogue."""
    _on_gpu("fp4_linear", x, packed, scales, row_scale, bias, residual, out)
    f, N, K = _check_quantised(packed, scales, row_scale, format, "fp4_linear")
    shape = x.shape
    if not shape or shape[-1] != K:
        raise ValueError(f"fp4_linear: input must end in {K} features; got {tuple(shape)}")
    if relu2 and residual is not None:
        raise ValueError("fp4_linear: the relu^2 epilogue takes no residual")
    dt, dtype = dt_code(x), x.dtype
    x2, ld = _rows2d(x, K, "fp4_linear")
    M = x2.shape[0]
    if bias is not None and (bias.dtype is not dtype or bias.shape != (N,) or not bias.is_contiguous()):
        raise ValueError(f"fp4_linear: bias must be a contiguous [{N}] in the activation dtype")
    if residual is not None:
        if residual.dtype is not dtype or residual.numel() != M * N:
            raise ValueError(f"fp4_linear: residual must be [{M}, {N}] in the activation dtype")
        if not residual.is_contiguous():
            residual = residual.contiguous()
    if out is None:
        out = x2.new_empty((*shape[:-1], N))
    elif out.dtype is not dtype or out.numel() != M * N or not out.is_contiguous():
        raise ValueError(f"fp4_linear: out must be a contiguous [{M}, {N}] in the activation dtype")
    if M and N:
        nbytes = _lib.lib.rwkv7_fp4_linear_workspace_bytes(M, K, f)
        ws = packed.new_empty(nbytes)
        epi = _lib.EPI_RELU2 if relu2 else _lib.EPI_NONE if residual is None else _lib.EPI_ADD
        _lib.check(_lib.lib.rwkv7_fp4_linear(x2.data_ptr(), ld, packed.data_ptr(), scales.data_ptr(), ptr(row_scale), ptr(bias), ptr(residual),
                                             out.data_ptr(), ws.data_ptr(), nbytes, M, K, N, epi, f, dt, stream_ptr(x2)), "fp4_linear")
    return out


class FP4Linear(torch.nn.Module):
    """``nn.Linear`` replacement with both operands in 4 bits (buffers ``packed_fp4``, ``fp4_scales``, ``fp4_row_scale``); the
    activations are quantised on the way."""

    def __init__(self, linear, *, format: str = "nvfp4"):
        super().__init__()
        self.format = format
        self.out_features, self.in_features = (int(v) for v in linear.weight.shape)
        w = linear.weight.data
        packed, scales, row_scale = (quantize_fp4 if w.is_cuda else quantize_fp4_weight)(w, format)
        self.register_buffer("packed_fp4", packed)
        self.register_buffer("fp4_scales", scales)
        self.register_buffer("fp4_row_scale", row_scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.data.clone())

    def _lin(self, x, **kw):
        return fp4_linear(x, self.packed_fp4, self.fp4_scales, self.fp4_row_scale, self.bias, format=self.format, **kw)

    def forward(self, x):
        return self._lin(x)

    def rwkv7_forward_into(self, x, out):
        self._lin(x, out=out)
        return out

    def rwkv7_forward_relu2(self, x):
        return self._lin(x, relu2=True)

    def rwkv7_forward_add(self, x, residual):
        return self._lin(x, residual=residual)

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, {self.format}"
