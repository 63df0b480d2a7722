"""The operators of serving from a paged KV cache, in plain torch and as the
package's kernels, with their exact (64-bit) results.

Kinds of a case (``case["kind"]``):

* ``append``  paged_append: the position rotation of a step's queries and keys, each
              at its sequence's own position, and keys and values written to pages.
* ``attend``  paged_attention: a step's tokens over their sequences' pages; one token
              of each sequence, or runs of several (prompts, chunks of prompts).
* ``logits``  adjust_logits: penalties for tokens the text holds already, biases and
              the tokens a grammar allows, before the next token is drawn.

A page holds `page` positions of every KV head: keys [pages, kv_heads, page, hd],
values [pages, kv_heads, page / 8, hd, 8] (eight consecutive positions of a dimension
side by side).  table[b, i] is the page of sequence b's positions i * page on.  A
sequence of lens[b] cached positions adds rows starts[b] to starts[b + 1] of the step,
at positions lens[b] on.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # one sequence's next token: a launch's latency
        {"name": "append_b1", "kind": "append", "batch": 1, "new": 1, "low": 300, "high": 900,
         "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "type": "fp16", "layout": "half",
         "rotary": 128},
        # a serving batch's next tokens, half of each head rotated in neighbouring pairs
        {"name": "append_b64", "kind": "append", "batch": 64, "new": 1, "low": 200, "high": 8000,
         "page": 16, "heads": 96, "kv_heads": 8, "hd": 128, "type": "bf16",
         "layout": "interleaved", "rotary": 64},
        # prompts of many lengths in one step
        {"name": "append_prompts", "kind": "append", "batch": 12, "new": 1400, "low": 0, "high": 0,
         "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "type": "fp16", "layout": "half",
         "rotary": 128},
        # the next token of one short text
        {"name": "attend_b1", "kind": "attend", "batch": 1, "new": 1, "low": 701, "high": 701,
         "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "type": "fp16"},
        # the next token of one text near the model's last position: few rows, a long axis
        {"name": "attend_b1_long", "kind": "attend", "batch": 1, "new": 1, "low": 31777,
         "high": 31777, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "type": "fp16"},
        # a serving batch of ragged lengths
        {"name": "attend_b64_ragged", "kind": "attend", "batch": 64, "new": 1, "low": 150,
         "high": 8000, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "type": "fp16"},
        # twelve query heads to a KV head, small pages
        {"name": "attend_b24_rep12", "kind": "attend", "batch": 24, "new": 1, "low": 900,
         "high": 9000, "page": 16, "heads": 96, "kv_heads": 8, "hd": 128, "type": "bf16"},
        # heads of 64, a large batch of short texts
        {"name": "attend_b128_hd64", "kind": "attend", "batch": 128, "new": 1, "low": 1,
         "high": 1500, "page": 32, "heads": 32, "kv_heads": 8, "hd": 64, "type": "fp16"},
        # chunks of prompts behind what is cached of them
        {"name": "attend_chunks", "kind": "attend", "batch": 3, "new": 1000, "low": 900,
         "high": 4000, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "type": "fp16"},
        # one sequence under a grammar
        {"name": "logits_b1", "kind": "logits", "batch": 1, "vocab": 32000, "type": "fp16",
         "low": 600, "high": 600, "biases": 20, "grammar": True},
        # a serving batch with its own penalties for each text
        {"name": "logits_b64", "kind": "logits", "batch": 64, "vocab": 32000, "type": "fp16",
         "low": 50, "high": 8000, "biases": 300, "grammar": False},
        # a large, odd vocabulary in 32 bits
        {"name": "logits_b64_large", "kind": "logits", "batch": 64, "vocab": 130001,
         "type": "fp32", "low": 100, "high": 4000, "biases": 64, "grammar": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "append", "attend", "attend", "attend", "logits", "logits"))
    if kind == "logits":
        vocab = _log(rng, 500, 130000)
        batch = max(1, min(_log(rng, 1, 128), 9_000_000 // vocab))
        high = _log(rng, 1, 8000)
        return {"kind": kind, "batch": batch, "vocab": vocab,
                "type": rng.choice(("fp16", "bf16", "fp32")), "low": rng.randint(0, high),
                "high": high, "biases": rng.choice((0, _log(rng, 1, 300))),
                "grammar": rng.random() < 0.5}
    hd = rng.choice((64, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    rep = rng.choice((1, 2, 4, 6, 8, 12))
    c = {"kind": kind, "page": rng.choice((16, 32, 64, 128)), "heads": kv_heads * rep,
         "kv_heads": kv_heads, "hd": hd, "type": rng.choice(("fp16", "bf16"))}
    if kind == "append":
        c["layout"] = rng.choice(("half", "interleaved"))
        c["rotary"] = rng.choice((hd, hd, hd // 2, hd // 4))
        c["new"] = rng.choice((1, _log(rng, 2, 1200)))
        c["batch"] = min(_log(rng, 1, 64), max(1, 6000 // c["new"]))
        c["high"] = rng.choice((0, _log(rng, 1, 8000)))
        c["low"] = rng.randint(0, c["high"])
        return c
    c["new"] = rng.choice((1, 1, 1, _log(rng, 2, 600)))
    c["high"] = _log(rng, 1, 32000 if c["new"] == 1 else 4000)
    c["low"] = rng.randint(0, c["high"])
    # cached positions of the batch, and scores of its runs, below the largest listed cases'
    most = 250_000 // (c["high"] + c["new"])
    if c["new"] > 1:
        most = min(most, 60_000_000 // (c["new"] * (c["high"] + c["new"]) * rep))
    c["batch"] = max(1, min(_log(rng, 1, 64), most))
    return c


# ----------------------------------------------------------------------------- inputs
def _counts(case):
    """New tokens of each sequence, the same for every seed: `new` and shorter ones."""
    n = case["new"]
    return [max(1, n - (b * n * 5 // 16) % n) if n > 1 else 1 for b in range(case["batch"])]


def _randn(shape, g, dtype, scale=1.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, scale, generator=g)


def _tables(case, n):
    """cos, sin [n, rotary / 2] fp32, the angles in 64 bits."""
    rd = case["rotary"]
    inv = 1e6 ** (-torch.arange(0, rd, 2, device=DEV, dtype=torch.float64) / rd)
    a = torch.outer(torch.arange(n, device=DEV, dtype=torch.float64), inv)
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    B = case["batch"]
    if case["kind"] == "logits":
        V, H = case["vocab"], case["high"]
        s["logits"] = _randn((B, V), g, torch.float32, 3.0).to(TYPES[case["type"]])
        # a text repeats itself: tokens from a small part of the vocabulary, skewed
        u = torch.rand((B, H + 8), generator=g, device=DEV, dtype=torch.float64)
        s["text"] = (V * u ** 4).long().clamp(max=V - 1)
        s["lens"] = torch.randint(case["low"], H + 1, (B,), generator=g, device=DEV)
        s["prompt"] = (s["lens"] * torch.rand((B,), generator=g, device=DEV)).long()
        s["repetition"] = 1.0 + 0.3 * torch.rand((B,), generator=g, device=DEV)
        s["presence"] = torch.rand((B,), generator=g, device=DEV)
        s["frequency"] = 0.5 * torch.rand((B,), generator=g, device=DEV)
        s["bias"] = s["bits"] = None
        if case["biases"]:
            n = case["biases"]
            ids = torch.randint(0, V, (B, n), generator=g, device=DEV)
            s["bias"] = (ids, _randn((B, n), g, torch.float32, 4.0))
        if case["grammar"]:
            # a grammar leaves few tokens, as words of 32 tokens' bits
            words = -(-V // 32)
            few = torch.rand((B, words * 32), generator=g, device=DEV) < 0.05
            w = few.view(B, words, 32).long() << torch.arange(32, device=DEV)
            s["bits"] = w.sum(-1).to(torch.int32)  # (the low 32 bits)
        return s
    dt, hd, nkv, page = TYPES[case["type"]], case["hd"], case["kv_heads"], case["page"]
    counts = _counts(case)
    ends = [sum(counts[:b + 1]) for b in range(B)]
    T = ends[-1]
    s["lens"] = torch.randint(case["low"], case["high"] + 1, (B,), generator=g, device=DEV)
    P = -(-(case["high"] + case["new"]) // page)
    pool = B * P + 3
    s["table"] = torch.randperm(pool, generator=g, device=DEV)[:B * P].view(B, P).int()
    s["starts"] = torch.tensor([0] + ends, dtype=torch.int32, device=DEV)
    # of each row of the step, its sequence and its place among the sequence's new tokens
    s["seq"] = torch.tensor([b for b in range(B) for _ in range(counts[b])], device=DEV)
    s["nth"] = torch.tensor([i for b in range(B) for i in range(counts[b])], device=DEV)
    s["k"] = _randn((pool, nkv, page, hd), g, dt)
    s["v"] = _randn((pool, nkv, page // 8, hd, 8), g, dt)
    if case["kind"] == "append":
        s["qkv"] = _randn((T, (case["heads"] + 2 * nkv) * hd), g, dt)
        s["cos"], s["sin"] = _tables(case, case["high"] + case["new"])
    else:
        # queries that prefer some positions, as trained ones do: scores of deviation 2
        s["q"] = _randn((T, case["heads"] * hd), g, dt, 2.0)
    if own:
        from hydranet_amd.model.paged import PagedBatch, PagedKVCache, RotaryTable
        s["cache"] = PagedKVCache.wrap([s["k"]], [s["v"]])
        s["batch"] = PagedBatch(s["table"], s["lens"], case["high"] + case["new"],
                                s["starts"] if case["new"] > 1 else None, T, case["new"])
        if case["kind"] == "append":
            s["rope"] = RotaryTable.wrap(s["cos"], s["sin"], case["layout"])
    return s


# ----------------------------------------------------------------------------- one pass
def _append(s):
    c = s["case"]
    nh, nkv, hd, rd, page = c["heads"], c["kv_heads"], c["hd"], c["rotary"], c["page"]
    pos = s["lens"][s["seq"]] + s["nth"]
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    y = x.clone()
    if c["layout"] == "half":
        a, b = slice(0, rd // 2), slice(rd // 2, rd)
    else:
        a, b = slice(0, rd, 2), slice(1, rd, 2)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    y = y.to(s["qkv"].dtype)
    at, slot = s["table"][s["seq"], pos // page].long(), pos % page
    s["k"][at, :, slot] = y[:, nh:nh + nkv]
    s["v"][at, :, slot // 8, :, slot % 8] = s["qkv"].view(-1, nh + 2 * nkv, hd)[:, nh + nkv:]
    return y[:, :nh].reshape(-1, nh * hd), s["k"], s["v"]


def _gather(s):
    """Every sequence's pages in a row: keys and values [B, kv_heads, positions, hd] fp32."""
    c, (B, P) = s["case"], s["table"].shape
    nkv, hd, n = c["kv_heads"], c["hd"], P * c["page"]
    t = s["table"].long()
    k = s["k"][t].transpose(1, 2).reshape(B, nkv, n, hd).float()
    v = s["v"][t].permute(0, 2, 1, 3, 5, 4).reshape(B, nkv, n, hd).float()
    return k, v


def _attend(s):
    c = s["case"]
    B, nkv, hd, S = c["batch"], c["kv_heads"], c["hd"], c["new"]
    rep = c["heads"] // nkv
    k, v = _gather(s)
    n = k.shape[2]
    q = torch.zeros(B, S, nkv, rep, hd, device=DEV)
    q[s["seq"], s["nth"]] = s["q"].float().view(-1, nkv, rep, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, nkv, rep * S, hd)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, nkv, rep, S, n) / math.sqrt(hd)
    last = s["lens"][:, None] + torch.arange(S, device=DEV)
    see = torch.arange(n, device=DEV) <= last[..., None]  # [B, S, n]
    x = x.masked_fill_(~see[:, None, None], -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, nkv, rep * S, n), v).view(B, nkv, rep, S, hd)
    o = o.permute(0, 3, 1, 2, 4)[s["seq"], s["nth"]]
    return o.reshape(-1, c["heads"] * hd).to(s["q"].dtype)


def _logits(s):
    B, V = s["logits"].shape
    x = s["logits"].float()
    at = torch.arange(s["text"].shape[1], device=DEV)
    there = at < s["lens"][:, None]
    new = there & (at >= s["prompt"][:, None])
    zero = torch.zeros(B, V, device=DEV)
    seen = zero.scatter_add(1, s["text"], there.float()) > 0
    count = zero.scatter_add(1, s["text"], new.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        ids, value = s["bias"]
        # of a token that is named twice, the last entry
        nth = torch.arange(ids.shape[1], device=DEV).expand_as(ids)
        last = torch.full((B, V), -1, device=DEV).scatter_reduce(1, ids, nth, "amax")
        x = x + torch.where(last >= 0, value.gather(1, last.clamp(min=0)), 0.0)
    if s["bits"] is not None:
        v = torch.arange(V, device=DEV)
        x = torch.where((s["bits"][:, v >> 5] >> (v & 31)) & 1 > 0, x, -torch.inf)
    return x.to(s["logits"].dtype)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"append": _append, "attend": _attend, "logits": _logits}[kind](state)
    if kind == "append":
        from hydranet_amd.model.paged import paged_append
        q = paged_append(state["qkv"], state["rope"], state["batch"], state["cache"], 0,
                         case["heads"])
        return q, state["k"], state["v"]
    if kind == "attend":
        from hydranet_amd.model.paged import paged_attention
        return paged_attention(state["q"], state["batch"], state["cache"], 0)
    from hydranet_amd.model.sampling import adjust_logits
    return adjust_logits(state["logits"], state["text"], state["lens"], state["prompt"],
                         repetition=state["repetition"], presence=state["presence"],
                         frequency=state["frequency"], bias=state["bias"],
                         allowed=state["bits"])


# ----------------------------------------------------------------------------- floors
def work(case):
    B = case["batch"]
    mean = (case["low"] + case["high"]) / 2
    if case["kind"] == "logits":
        size = 4 if case["type"] == "fp32" else 2
        row = 2 * case["vocab"] * size + 8 * mean + 12 * case["biases"]
        if case["grammar"]:
            row += case["vocab"] / 8
        return {"bytes": B * row, "flops": B * 4.0 * case["vocab"]}
    counts, hd = _counts(case), case["hd"]
    T, nh, nkv = sum(counts), case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        # projections read, queries and pages written, two table rows a token
        return {"bytes": T * (2 * (nh + 2 * nkv) * hd * 2 + case["rotary"] * 4),
                "flops": 3.0 * T * (nh + nkv) * case["rotary"]}
    kv = sum(mean + n for n in counts) * nkv * hd * 2 * 2
    pairs = sum(n * mean + n * (n + 1) / 2 for n in counts)
    return {"bytes": kv + 2 * T * nh * hd * 2, "flops": 4.0 * hd * nh * pairs}


# ----------------------------------------------------------------------------- exact results
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend,
            "logits": _exact_logits}[case["kind"]](case, s)


def _exact_append(case, s):
    nh, nkv, hd, rd, page = (case[n] for n in ("heads", "kv_heads", "hd", "rotary", "page"))
    k, v = s["k"].double(), s["v"].double()
    lens, table = s["lens"].tolist(), s["table"].tolist()
    x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)
    out, row = [], 0
    for b, n in enumerate(_counts(case)):
        mine = x[row:row + n]
        row += n
        p = torch.arange(lens[b], lens[b] + n, device=DEV)
        turn = torch.complex(s["cos"][p].double(), s["sin"][p].double())[:, None]
        rot, rest = mine[:, :nh + nkv, :rd], mine[:, :nh + nkv, rd:]
        if case["layout"] == "half":
            z = torch.complex(rot[..., :rd // 2].contiguous(), rot[..., rd // 2:].contiguous())
            z = z * turn
            y = torch.cat((z.real, z.imag, rest), -1)
        else:
            z = torch.view_as_complex(rot.reshape(n, nh + nkv, rd // 2, 2).contiguous()) * turn
            y = torch.cat((torch.view_as_real(z).reshape(n, nh + nkv, rd), rest), -1)
        out.append(y[:, :nh].reshape(n, nh * hd))
        first = 0  # page by page
        while first < n:
            at = lens[b] + first
            m = min(n - first, page - at % page)
            pg, slot = table[b][at // page], at % page
            k[pg, :, slot:slot + m] = y[first:first + m, nh:].transpose(0, 1)
            flat = v[pg].transpose(1, 2).reshape(nkv, hd, page)  # [nkv, hd, slot]
            flat[:, :, slot:slot + m] = mine[first:first + m, nh + nkv:].permute(1, 2, 0)
            v[pg] = flat.view(nkv, hd, page // 8, 8).transpose(1, 2)
            first += m
    return torch.cat(out), k, v


def _exact_attend(case, s):
    nh, nkv, hd = case["heads"], case["kv_heads"], case["hd"]
    rep, out, row = nh // nkv, [], 0
    lens = s["lens"].tolist()
    for b, n in enumerate(_counts(case)):
        q = s["q"][row:row + n].double().view(n, nkv, rep, hd)
        row += n
        L = lens[b] + n
        pages = s["table"][b, :-(-L // case["page"])].long()
        hide = torch.ones(n, L, dtype=torch.bool, device=DEV).triu(lens[b] + 1)
        o = torch.empty(n, nkv, rep, hd, dtype=torch.float64, device=DEV)
        for h in range(nkv):
            k = s["k"][pages, h].reshape(-1, hd)[:L].double()
            v = s["v"][pages, h].transpose(2, 3).reshape(-1, hd)[:L].double()
            for r in range(rep):
                x = (q[:, h, r] @ k.t().contiguous()) * hd ** -0.5
                o[:, h, r] = torch.softmax(x.masked_fill(hide, -torch.inf), -1) @ v
        out.append(o.view(n, nh * hd))
    return torch.cat(out)


def _exact_logits(case, s):
    V, rows = case["vocab"], []
    for b in range(case["batch"]):
        x = s["logits"][b].double()
        L, P = int(s["lens"][b]), int(s["prompt"][b])
        words = s["text"][b, :L].unique()
        r = float(s["repetition"][b])
        x[words] = torch.where(x[words] > 0, x[words] / r, x[words] * r)
        words, many = s["text"][b, P:L].unique(return_counts=True)
        x[words] -= float(s["frequency"][b]) * many + float(s["presence"][b])
        if s["bias"] is not None:
            named = dict(zip(s["bias"][0][b].tolist(), s["bias"][1][b].tolist()))
            ids = torch.tensor(list(named), device=DEV)
            x[ids] += torch.tensor(list(named.values()), dtype=torch.float64, device=DEV)
        if s["bits"] is not None:
            lanes = torch.arange(32, device=DEV)
            on = ((s["bits"][b].long()[:, None] >> lanes) & 1).bool().view(-1)[:V]
            x[~on] = -torch.inf
        rows.append(x)
    return torch.stack(rows)
