"""Logits adjusted before the next token is drawn from them (verify_tree of
model/speculative.py draws: a tree of one node, a temperature, one uniform).

On the GPU one library call (hn_adjust_logits, include/hn_int4.h); on the CPU the same
definition in torch."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_I64, _I32, _F32 = torch.int64, torch.int32, torch.float32
_MOST = torch.finfo(torch.float32).max


def _rows(x: torch.Tensor):
    """x with its last axis dense and rows that do not overlap, and their stride."""
    if x.is_contiguous():
        return x, x.shape[1]
    ld, last = x.stride()
    if last != 1 or ld < x.shape[1]:
        x = x.contiguous()
        ld = x.shape[1]
    return x, ld


def adjust_logits(logits: torch.Tensor, text: Optional[torch.Tensor] = None,
                  lens: Optional[torch.Tensor] = None, prompt: Optional[torch.Tensor] = None,
                  repetition: Union[float, torch.Tensor] = 1.0,
                  presence: Union[float, torch.Tensor] = 0.0,
                  frequency: Union[float, torch.Tensor] = 0.0,
                  bias: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                  allowed: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits [B, V] (fp16, bf16 or fp32) adjusted, in fp32, rounded once.

    text int64 [B, width]: each sequence's tokens, lens int64 [B] of them (None: all),
    of which the first prompt int64 [B] (None: 0) were given and the others generated.
    In this order: a token anywhere in the text has a positive logit divided by
    repetition, any other multiplied; one that was generated c > 0 times loses
    frequency * c + presence; bias = (ids int64 [B, n], values fp32 [B, n]) is added (of
    a token that is named twice, the last entry's; ids outside the vocabulary, such as
    -1, are padding); tokens whose bit of allowed int32 [B, ceil(V / 32)] (32 tokens to a
    word, the lowest bit first) is zero become -inf.  repetition (above 0), presence and
    frequency: numbers that fp32 holds, or fp32 [B].  out: logits itself, or another tensor of its
    shape, type and device that does not overlap it; None: a new one."""
    dt, dev, at_dev = logits.dtype, logits.device, logits.get_device()
    assert logits.dim() == 2 and dt in _DTYPES and logits.shape[1] > 0, \
        "logits: fp16, bf16 or fp32 [B, V], V > 0"
    B, V = logits.shape
    if text is not None:
        assert text.dtype is _I64 and text.dim() == 2 and text.shape[0] == B \
            and text.get_device() == at_dev, f"text: int64 [{B}, width] on {dev}"
        if lens is not None:
            assert lens.dtype is _I64 and lens.shape == (B,) and lens.get_device() == at_dev, \
                f"lens: int64 [{B}] on {dev}"
        if prompt is not None:
            assert prompt.dtype is _I64 and prompt.shape == (B,) \
                and prompt.get_device() == at_dev, f"prompt: int64 [{B}] on {dev}"
    else:
        assert lens is None and prompt is None, "lens and prompt are of a text"
    rep, rep1 = _amount(repetition, "repetition", B, at_dev)
    assert rep is not None or rep1 >= 2.0 ** -126, f"repetition {rep1}"
    pres, pres1 = _amount(presence, "presence", B, at_dev)
    freq, freq1 = _amount(frequency, "frequency", B, at_dev)
    ids, values = (None, None) if bias is None else bias
    if bias is not None:
        assert ids.dtype is _I64 and ids.dim() == 2 and ids.shape[0] == B \
            and values.dtype is _F32 and values.shape == ids.shape \
            and ids.get_device() == values.get_device() == at_dev, \
            f"bias: (int64 [{B}, n], fp32 [{B}, n]) on {dev}"
    if allowed is not None:
        assert allowed.dtype is _I32 and allowed.dim() == 2 and allowed.shape[0] == B \
            and allowed.shape[1] >= -(-V // 32) and allowed.get_device() == at_dev, \
            f"allowed: int32 [{B}, {-(-V // 32)}] on {dev}"
    if out is not None:
        assert out.shape == logits.shape and out.dtype is dt and out.device == dev \
            and out.stride(1) == 1 and (B <= 1 or out.stride(0) >= V), \
            "out: shape, type and device of logits, dense rows"
    if not logits.is_cuda:
        y = _adjust_cpu(logits, text, lens, prompt, [
            torch.full((B,), n) if x is None else x
            for x, n in ((rep, rep1), (pres, pres1), (freq, freq1))], ids, values, allowed)
        return y if out is None else out.copy_(y)
    ld_o = V if out is None else max(out.stride(0), V)
    src, ld = (logits, ld_o) if out is logits else _rows(logits)
    if out is None:
        out = src.new_empty((B, V))
    at = ld_t = width = at_lens = at_prompt = at_ids = ld_i = at_v = ld_v = n = at_a = ld_a = 0
    if text is not None:
        text, ld_t = _rows(text)
        at, width = text.data_ptr(), text.shape[1]
        if lens is not None:
            lens = lens.contiguous()
            at_lens = lens.data_ptr()
        if prompt is not None:
            prompt = prompt.contiguous()
            at_prompt = prompt.data_ptr()
    if ids is not None:
        ids, ld_i = _rows(ids)
        values, ld_v = _rows(values)
        at_ids, at_v, n = ids.data_ptr(), values.data_ptr(), ids.shape[1]
    if allowed is not None:
        allowed, ld_a = _rows(allowed)
        at_a = allowed.data_ptr()
    _lib.call_on(dev, "hn_adjust_logits", src.data_ptr(), ld, _DTYPES[dt], at, ld_t, width,
                 at_lens, at_prompt, 0 if rep is None else rep.data_ptr(),
                 0 if pres is None else pres.data_ptr(), 0 if freq is None else freq.data_ptr(),
                 rep1, pres1, freq1, at_ids, ld_i, at_v, ld_v, n, at_a, ld_a, B, V,
                 out.data_ptr(), ld_o)
    return out


def _amount(x, name, B, at_dev):
    """(fp32 [B] or None, else the number)."""
    if isinstance(x, torch.Tensor):
        assert x.dtype is _F32 and x.shape == (B,) and x.get_device() == at_dev, \
            f"{name}: a number or fp32 [{B}] on the logits' device"
        return x.contiguous(), 0.0
    x = float(x)
    assert -_MOST <= x <= _MOST, f"{name} {x}: finite in fp32"
    return None, x


def _adjust_cpu(logits, text, lens, prompt, amounts, ids, values, allowed) -> torch.Tensor:
    x = logits.float().clone()
    B, V = x.shape
    rep, pres, freq = (a.float() for a in amounts)
    for b in range(B):
        if text is not None:
            n = text.shape[1] if lens is None else min(max(int(lens[b]), 0), text.shape[1])
            first = 0 if prompt is None else min(max(int(prompt[b]), 0), n)
            t = text[b, :n]
            ok = (t >= 0) & (t < V)
            seen = t[ok].unique()
            x[b, seen] = torch.where(x[b, seen] > 0, x[b, seen] / rep[b], x[b, seen] * rep[b])
            seen, count = t[first:][ok[first:]].unique(return_counts=True)
            x[b, seen] = x[b, seen] - freq[b] * count.float() - pres[b]
        if ids is not None:
            named = {i: v for i, v in zip(ids[b].tolist(), range(ids.shape[1])) if 0 <= i < V}
            if named:
                x[b, list(named)] += values[b, list(named.values())]
        if allowed is not None:
            v = torch.arange(V)
            x[b, (allowed[b, v >> 5] >> (v & 31)) & 1 == 0] = -math.inf
    return x.to(logits.dtype)
