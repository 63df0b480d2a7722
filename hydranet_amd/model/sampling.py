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


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with its last axis dense and rows that do not overlap."""
    return x if x.stride(1) == 1 and (x.shape[0] == 1 or x.stride(0) >= x.shape[1]) \
        else x.contiguous()


def _ld(x: torch.Tensor) -> int:
    return max(x.stride(0), x.shape[1])


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
    frequency: numbers, or fp32 [B].  out: logits itself, or another tensor of its
    shape, type and device that does not overlap it; None: a new one."""
    assert logits.dim() == 2 and logits.dtype in _DTYPES, "logits: fp16, bf16 or fp32 [B, V]"
    B, V = logits.shape
    dev = logits.device
    assert V > 0, "logits: fp16, bf16 or fp32 [B, V], V > 0"
    assert text is not None or (lens is None and prompt is None), "lens and prompt are of a text"
    if text is not None:
        assert text.dtype == torch.int64 and text.dim() == 2 and text.shape[0] == B \
            and text.device == dev, f"text: int64 [{B}, width] on {dev}"
    for name, x in (("lens", lens), ("prompt", prompt)):
        assert x is None or (x.dtype == torch.int64 and tuple(x.shape) == (B,)
                             and x.device == dev), f"{name}: int64 [{B}] on {dev}"
    amounts = []
    for name, x, low in (("repetition", repetition, 0.0), ("presence", presence, None),
                         ("frequency", frequency, None)):
        if isinstance(x, torch.Tensor):
            assert x.dtype == torch.float32 and tuple(x.shape) == (B,) and x.device == dev, \
                f"{name}: a number or fp32 [{B}] on {dev}"
            amounts.append((x.contiguous(), 0.0))
        else:
            x = float(x)
            assert math.isfinite(x) and (low is None or x > low), f"{name} {x}"
            amounts.append((None, x))
    ids = values = None
    if bias is not None:
        ids, values = bias
        assert ids.dtype == torch.int64 and ids.dim() == 2 and ids.shape[0] == B \
            and values.dtype == torch.float32 and values.shape == ids.shape \
            and ids.device == values.device == dev, \
            f"bias: (int64 [{B}, n], fp32 [{B}, n]) on {dev}"
    assert allowed is None or (allowed.dtype == torch.int32 and allowed.dim() == 2
                               and allowed.shape[0] == B and allowed.shape[1] >= -(-V // 32)
                               and allowed.device == dev), \
        f"allowed: int32 [{B}, {-(-V // 32)}] on {dev}"
    if out is not None:
        assert out.shape == logits.shape and out.dtype == logits.dtype and out.device == dev \
            and out.stride(1) == 1 and (B == 1 or out.stride(0) >= V), \
            "out: shape, type and device of logits, dense rows"
    if not logits.is_cuda:
        y = _adjust_cpu(logits, text, lens, prompt, [
            torch.full((B,), n) if x is None else x for x, n in amounts], ids, values, allowed)
        return y if out is None else out.copy_(y)
    src = logits if out is logits else _rows(logits)
    out = torch.empty((B, V), dtype=logits.dtype, device=dev) if out is None else out
    t, i, v, a = (None if x is None else _rows(x) for x in (text, ids, values, allowed))
    lens, prompt = (None if x is None else x.contiguous() for x in (lens, prompt))

    def at(x):
        return None if x is None else x.data_ptr()

    def ld(x):
        return 0 if x is None else _ld(x)

    _lib.call_on(dev, "hn_adjust_logits", src.data_ptr(), _ld(src), _DTYPES[logits.dtype], at(t),
                 ld(t), 0 if t is None else t.shape[1], at(lens), at(prompt),
                 *(at(x) for x, _ in amounts), *(n for _, n in amounts), at(i), ld(i), at(v),
                 ld(v), 0 if i is None else i.shape[1], at(a), ld(a), B, V, out.data_ptr(),
                 _ld(out))
    return out


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
