"""Processing of a step's logits before sampling, as one kernel (bd3_process_logits): penalties for
repeated tokens, a bias and a grammar mask.

``process_logits(logits, history=..., history_len=..., ...)`` goes between the backbone and
``subs_sample_step``: the penalties look at the tokens each sequence holds so far (its buffer of
tokens, as it is, with the count of valid ones), the mask at a grammar's set of allowed tokens
as bits. All arguments stay on the device, so the call can be part of a captured CUDA graph.
"""

from __future__ import annotations

import ctypes

import torch

from bd3attn._lib import LIB, check
from bd3attn.ops import _check_cuda, _check_on, _code, _raw_stream

_I64x2, _I64x4 = ctypes.c_int64 * 2, ctypes.c_int64 * 4


def _per_sequence(name, t, B, index):
    if t is None:
        return None
    _check_on(index, t)
    if t.dtype != torch.float32 or t.shape != (B,) or not t.is_contiguous():
        raise AssertionError(f"{name} must be a contiguous (batch,) fp32 tensor")
    return t.data_ptr()


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """A boolean mask (..., vocab) as the int32 words (..., ceil(vocab / 32)) process_logits takes:
    token v is bit v % 32 of word v // 32."""
    V = allowed.shape[-1]
    pad = torch.nn.functional.pad(allowed.to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (pad << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def process_logits(logits: torch.Tensor, history: torch.Tensor | None = None,
                   history_len: torch.Tensor | None = None,
                   repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   allowed: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The processed logits (batch, seq, vocab), in ``out`` (may be ``logits``) or a new tensor.

    With n the occurrences of token v among the first history_len[b] entries of history[b]:
    x = logits; if n > 0, x = (x / repetition if x > 0 else x * repetition) - (frequency * n +
    presence); x += bias; x = -inf where the mask forbids v. fp32 arithmetic, rounded once. One
    history serves the three penalties: where frequency and presence are to count the generated
    tokens only (the repetition penalty the prompt's as well), call it once for each.

    logits: bf16, f16 or fp32; history: (batch, capacity) int64 or int32 tokens (ids outside the
    vocabulary, padding for one, are ignored) with history_len (batch,) int32; repetition (> 0),
    presence, frequency: (batch,) fp32 or None; bias: (vocab,) or (batch, vocab) fp32; allowed:
    int32 words of 32 tokens (pack_mask), (batch, words) or (batch, seq, words).
    """
    _check_cuda(logits)
    dev = logits.device
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return process_logits(logits, history, history_len, repetition, presence, frequency,
                                  bias, allowed, out)
    if logits.dim() != 3:
        raise AssertionError("logits must be (batch, seq, vocab)")
    B, S, V = logits.shape
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    elif out.shape != logits.shape or out.dtype != logits.dtype or (out.stride(2) != 1 and V > 1) \
            or out.device != dev:
        raise AssertionError("out must be like logits, its vocabulary contiguous")
    h_ptr = hl_ptr = None
    h_i32 = h_stride = h_cap = 0
    if history is not None:
        if history_len is None:
            raise AssertionError("history needs history_len")
        _check_on(dev.index, history, history_len)
        if history.dtype not in (torch.int64, torch.int32) or history.dim() != 2 \
                or history.shape[0] != B or (history.stride(1) != 1 and history.shape[1] > 1):
            raise AssertionError("history must be (batch, capacity) int64 or int32 tokens")
        if history_len.dtype != torch.int32 or history_len.shape != (B,) \
                or not history_len.is_contiguous():
            raise AssertionError("history_len must be a contiguous (batch,) int32 tensor")
        h_ptr, hl_ptr = history.data_ptr(), history_len.data_ptr()
        h_i32, h_stride, h_cap = int(history.dtype == torch.int32), history.stride(0), \
            history.shape[1]
    b_ptr, b_stride = None, 0
    if bias is not None:
        _check_on(dev.index, bias)
        if bias.dtype != torch.float32 or bias.shape not in ((V,), (B, V)) \
                or (bias.stride(-1) != 1 and V > 1):
            raise AssertionError("bias must be (vocab,) or (batch, vocab) fp32")
        b_ptr, b_stride = bias.data_ptr(), bias.stride(0) if bias.dim() == 2 else 0
    a_ptr = a_strides = None
    if allowed is not None:
        _check_on(dev.index, allowed)
        words = (V + 31) // 32
        if allowed.dtype != torch.int32 or allowed.shape not in ((B, words), (B, S, words)) \
                or (allowed.stride(-1) != 1 and words > 1):
            raise AssertionError("allowed must be (batch, words) or (batch, seq, words) int32")
        a_ptr = allowed.data_ptr()
        a_strides = _I64x2(allowed.stride(0), allowed.stride(1) if allowed.dim() == 3 else 0)
    if B == 0 or S == 0:
        return out
    rc = LIB.bd3_process_logits(
        logits.data_ptr(), out.data_ptr(),
        _I64x4(logits.stride(0), logits.stride(1), out.stride(0), out.stride(1)), B, S, V,
        h_ptr, h_i32, h_stride, h_cap, hl_ptr,
        _per_sequence("repetition", repetition, B, dev.index),
        _per_sequence("presence", presence, B, dev.index),
        _per_sequence("frequency", frequency, B, dev.index), b_ptr, b_stride, a_ptr, a_strides,
        _code(logits.dtype), _raw_stream(dev))
    if rc:
        check("bd3_process_logits", rc)
    return out
