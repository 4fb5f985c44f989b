"""From a row of logits to the next token (csrc/logits.cu): penalties for repeated tokens, biases, grammar masks, and the draw
with temperature / top-k / top-p / min-p.  One launch each; ``sample_tokens`` takes the rules too, so that the processed
logits need not be written.  The reference does the draw in tensor code (rwkv7_hf/model_generation.py); results of
``sample_next_token`` stay what that code gives from the same generator."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._util import dt_code, require_cuda, stream_ptr


class _Rules(ctypes.Structure):  # rwkv7_logit_rules
    _fields_ = [("tokens", _lib.P), ("tokens_ld", _lib.L), ("lengths", _lib.P), ("prompt_lengths", _lib.P), ("repetition", _lib.P),
                ("presence", _lib.P), ("frequency", _lib.P), ("bias", _lib.P), ("bias_ld", _lib.L), ("allowed", _lib.P),
                ("allowed_ld", _lib.L), ("history", ctypes.c_int32), ("tokens_i64", ctypes.c_int32), ("repetition_value", _lib.F),
                ("presence_value", _lib.F), ("frequency_value", _lib.F)]


class _Draw(ctypes.Structure):  # rwkv7_draw_params
    _fields_ = [("temperature", _lib.P), ("top_p", _lib.P), ("min_p", _lib.P), ("top_k", _lib.P), ("temperature_value", _lib.F),
                ("top_p_value", _lib.F), ("min_p_value", _lib.F), ("top_k_value", ctypes.c_int32)]


def _vector(v, B, dtype, dev, name, keep):
    """``(pointer, value)`` of a parameter that is a number for all rows or a vector ``[B]`` on the device."""
    if not isinstance(v, torch.Tensor):
        return 0, v
    if v.shape != (B,):
        raise ValueError(f"{name} must be a number or a vector [{B}], got {tuple(v.shape)}")
    if v.get_device() != dev:
        raise ValueError(f"{name} must be on the device of the logits")
    if v.dtype is not dtype or not v.is_contiguous():
        v = v.to(dtype).contiguous()
        keep.append(v)
    return v.data_ptr(), 0


def _rows_of(t, B, width, name):
    """``(pointer, row stride)`` of a ``[width]`` or ``[1 | B, width]`` tensor whose rows have unit stride."""
    shape, stride = t.shape, t.stride()
    if len(shape) not in (1, 2) or shape[-1] != width or (len(shape) == 2 and shape[0] not in (1, B)):
        raise ValueError(f"{name} must be [{width}] or [{B}, {width}], got {tuple(shape)}")
    if stride[-1] != 1 and width > 1:
        raise ValueError(f"{name} must have rows of unit stride")
    return t.data_ptr(), stride[0] if len(shape) == 2 and shape[0] > 1 else 0


def _rows_in(t, B, V):
    """``t [B, V]`` with rows of unit stride that do not overlap (a copy where they do not lie so), and their distance."""
    ld, unit = t.stride()
    if (V > 1 and unit != 1) or (B > 1 and ld < V):
        t = t.contiguous()
        ld = V
    return t, ld if B > 1 else V


def _logits(logits, what):
    dev = logits.get_device()
    if dev < 0:
        require_cuda(logits, what=what)
    shape = logits.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"{what}: logits must be [rows, vocabulary], got {tuple(shape)}")
    dt = dt_code(logits)
    B, V = shape
    logits, ld = _rows_in(logits, B, V)
    return logits, ld, B, V, dt, dev


def _rules(B, V, dev, keep, what, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, allowed):
    r = _Rules()
    r.repetition_value = 1.0
    if tokens is not None:
        shape = tokens.shape
        if len(shape) != 2 or shape[0] != B or tokens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{what}: tokens must be [{B}, n] int32 or int64, got {tuple(shape)} {tokens.dtype}")
        if tokens.get_device() != dev:
            require_cuda(tokens, what=what)
            raise ValueError(f"{what}: tensors must be on the same device")
        n = shape[1]
        if n:
            rows, r.tokens_ld = _rows_in(tokens, B, n)
            if rows is not tokens:
                keep.append(rows)
            r.tokens, r.history, r.tokens_i64 = rows.data_ptr(), n, rows.dtype is torch.int64
            if lengths is not None:
                r.lengths = _vector(lengths, B, torch.int32, dev, "lengths", keep)[0]
            if prompt_lengths is not None:
                r.prompt_lengths = _vector(prompt_lengths, B, torch.int32, dev, "prompt_lengths", keep)[0]
            if not isinstance(repetition_penalty, torch.Tensor) and not repetition_penalty > 0:
                raise ValueError(f"{what}: repetition_penalty must be positive")
            r.repetition, r.repetition_value = _vector(repetition_penalty, B, torch.float32, dev, "repetition_penalty", keep)
            r.presence, r.presence_value = _vector(presence_penalty, B, torch.float32, dev, "presence_penalty", keep)
            r.frequency, r.frequency_value = _vector(frequency_penalty, B, torch.float32, dev, "frequency_penalty", keep)
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError(f"{what}: lengths need tokens")
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.get_device() != dev:
            raise ValueError(f"{what}: bias must be float32 on the device of the logits")
        r.bias, r.bias_ld = _rows_of(bias, B, V, "bias")
    if allowed is not None:
        if allowed.dtype is not torch.int32 or allowed.get_device() != dev:
            raise ValueError(f"{what}: allowed must be int32 words on the device of the logits")
        r.allowed, r.allowed_ld = _rows_of(allowed, B, (V + 31) // 32, "allowed")
    return r


def process_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition_penalty=1.0, presence_penalty=0.0,
                   frequency_penalty=0.0, bias=None, allowed=None, out=None):
    """``logits [B,V]`` (fp16 / bf16 / fp32) after the rules, in the same type; computed in fp32 and rounded once.

    ``tokens [B,n]`` (int32 / int64): each row's history, ``lengths [B]`` its valid tokens, ``prompt_lengths [B]`` how many of
    them are prompt; ids outside the vocabulary (padding: -1) are skipped.  A token of the history has its logit divided
    (positive) or multiplied by ``repetition_penalty``; a token generated c > 0 times loses ``frequency_penalty * c +
    presence_penalty``.  Then ``bias [V] | [B,V]`` (fp32) is added, and a token whose bit in ``allowed [ceil(V/32)] | [B,
    ceil(V/32)]`` (int32 words, token v at bit v % 32 of word v // 32) is 0 gets -inf, whatever its logit.  Penalties are numbers
    or vectors ``[B]``.  ``out`` may be ``logits``."""
    logits, ld, B, V, dt, dev = _logits(logits, "process_logits")
    keep = []
    r = _rules(B, V, dev, keep, "process_logits", tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias,
               allowed)
    out_ld = V
    if out is None:
        out = torch.empty_like(logits)
    else:
        out_ld = out.stride(0) if B > 1 and out.dim() == 2 else V
        if (out.shape != logits.shape or out.dtype is not logits.dtype or out.get_device() != dev or (V > 1 and out.stride(1) != 1)
                or out_ld < V):
            raise ValueError(f"process_logits: out must be like logits, [{B}, {V}] with rows of unit stride")
    if B:
        _lib.check(_lib.lib.rwkv7_process_logits(logits.data_ptr(), ld, ctypes.addressof(r), out.data_ptr(), out_ld, B, V, dt,
                                                 stream_ptr(logits)), "process_logits")
    return out


def sample_tokens(logits, noise=None, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprobs: bool = False, tokens=None,
                  lengths=None, prompt_lengths=None, repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0, bias=None,
                  allowed=None):
    """One token per row of ``logits [B,V]``: ``[B] int64``, and with ``return_logprobs`` its log-probability ``[B] fp32``.

    The rules of ``process_logits`` (same arguments), then ``z / temperature``; ``top_k`` (0: off) keeps every z at least as
    large as the k-th largest, ``top_p`` (1: off) the shortest beginning of the descending order (equal values by index) that
    reaches this share of what is left, ``min_p`` what is at least this fraction as likely as the most likely token.  The
    token is the argmax of exp(z) / noise over what is kept: with ``noise [B,V]`` of independent Exp(1) variates
    (``torch.empty(B, V).exponential_(generator=g)``) a draw from the renormalised distribution.  ``temperature <= 0``, or no
    noise: the largest logit, lowest index first.  Each parameter is a number or a vector ``[B]``.

    NaN is never drawn; a row that its mask leaves empty gives -1.  The log-probability is that of softmax(z / temperature)
    after the rules, before the filters (-inf for -1)."""
    logits, ld, B, V, dt, dev = _logits(logits, "sample_tokens")
    keep = []
    r = _rules(B, V, dev, keep, "sample_tokens", tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias,
               allowed)
    noise_ptr = noise_ld = 0
    if noise is not None:
        if noise.shape != (B, V) or noise.dtype is not torch.float32 or noise.get_device() != dev:
            raise ValueError(f"sample_tokens: noise must be [{B}, {V}] float32 on the device of the logits")
        noise, noise_ld = _rows_in(noise, B, V)
        noise_ptr = noise.data_ptr()
    d = _Draw()
    d.temperature, d.temperature_value = _vector(temperature, B, torch.float32, dev, "temperature", keep)
    d.top_p, d.top_p_value = _vector(top_p, B, torch.float32, dev, "top_p", keep)
    d.min_p, d.min_p_value = _vector(min_p, B, torch.float32, dev, "min_p", keep)
    d.top_k, d.top_k_value = _vector(top_k if isinstance(top_k, torch.Tensor) else min(int(top_k), 2 ** 31 - 1), B, torch.int32, dev, "top_k", keep)
    token = logits.new_empty(B, dtype=torch.int64)
    logprob = logits.new_empty(B, dtype=torch.float32) if return_logprobs else None
    if B:
        _lib.check(_lib.lib.rwkv7_sample_tokens(logits.data_ptr(), ld, ctypes.addressof(r), ctypes.addressof(d), noise_ptr, noise_ld,
                                                token.data_ptr(), 0 if logprob is None else logprob.data_ptr(), B, V, dt, stream_ptr(logits)),
                   "sample_tokens")
    return (token, logprob) if return_logprobs else token
