"""64-bit forms of the paged cache's append and attention and of adjusted logits, token by
token, with the bounds that the kernels' roundings allow."""
import math

import torch

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def subnormal(dt):
    """Half the distance of the type's smallest numbers."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def make(seed, lens, counts, nkv, hd, page, dt, dev="cpu", spare=3, columns=0, poison=False):
    """Pages of random numbers (poison: NaN wherever no cached position is) in random
    order, the table, lens and starts of a step; counts None: one row each."""
    g = torch.Generator().manual_seed(seed)
    new = counts or [1] * len(lens)
    need = [-(-max(C + n, 0) // page) for C, n in zip(lens, new)]
    cols = max(need + [1]) + columns
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    k = torch.randn(pool, nkv, page, hd, generator=g)
    v = torch.randn(pool, nkv, page // 8, hd, 8, generator=g)
    if poison:
        k[:], v[:] = math.nan, math.nan
    for b, n in enumerate(need):
        for i in range(n):
            p = table[b, i] = order.pop()
            m = min(max(lens[b], 0) + new[b] - i * page, page)
            if poison:
                k[p, :, :m] = torch.randn(nkv, m, hd, generator=g)
                v[p] = torch.where(torch.arange(page).view(1, page // 8, 1, 8) < m,
                                   torch.randn(nkv, page // 8, hd, 8, generator=g), math.nan)
    starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int()
    return {"k": k.to(dt).to(dev), "v": v.to(dt).to(dev), "table": table.to(dev),
            "lens": torch.tensor(lens, dtype=torch.int64, device=dev), "starts": starts.to(dev),
            "rows": sum(new), "gen": g}


def batch(s, single, bound=None):
    """The PagedBatch of make's tensors."""
    from hydranet_amd.model.paged import PagedBatch
    new = (s["starts"][1:] - s["starts"][:-1]).max().item() if len(s["lens"]) else 1
    bound = bound or max([int(x) for x in s["lens"]] + [0]) + max(new, 1)
    if single:
        return PagedBatch(s["table"], s["lens"], bound)
    return PagedBatch(s["table"], s["lens"], bound, s["starts"], s["rows"], max(new, 1))


def tokens(s):
    """(row, sequence, position) of each row that a sequence which takes part has."""
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for b, C in enumerate(lens):
        for i in range(starts[b], starts[b + 1]):
            if C >= 0:
                yield i, b, C + i - starts[b]


def tables(dim, n, base=1e4):
    a = torch.outer(torch.arange(n).double(), base ** (-torch.arange(0, dim, 2).double() / dim))
    return a.cos().float(), a.sin().float()


def rotate(x, cos, sin, layout):
    """x [.., hd] in 64 bits at one position's angles (cos, sin [dim / 2] fp32)."""
    y, i = x.clone(), torch.arange(len(cos))
    a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + len(cos))
    y[..., a] = x[..., a] * cos.double() - x[..., b] * sin.double()
    y[..., b] = x[..., b] * cos.double() + x[..., a] * sin.double()
    return y


def attend(s, q, nh, scale=None):
    """-> (out, bound) [rows, nh, hd] in 64 bits.  The bound: a score's fp32 sum of hd
    products is off by hd 2^-24 of their magnitudes, the exponent's scaling by a few
    2^-24 of it, which moves every probability by as much; a probability is rounded to
    the type (relative to at least 2^-14 of the largest, below that by less in all than
    the sum's own rounding), the sums of fp32 by 2^-24 a term at most, and the result
    once more."""
    k, v, table = s["k"].double().cpu(), s["v"].double().cpu(), s["table"].cpu()
    dt = s["k"].dtype
    nkv, page, hd = k.shape[1:]
    rep = nh // nkv
    scale = hd ** -0.5 if scale is None else scale
    x = q.double().cpu().view(-1, nkv, rep, hd)
    out = torch.zeros(x.shape, dtype=torch.float64)
    bound = torch.zeros(x.shape, dtype=torch.float64)
    u = half_step(dt)
    last = (None, None)
    for row, b, pos in tokens({n: s[n].cpu() for n in ("starts", "lens")}):
        if last[0] != b:
            ids = table[b][:-(-(pos + s["rows"]) // page)].long()
            ids = ids[ids >= 0]
            kb = k[ids].transpose(0, 1).reshape(nkv, -1, hd)
            vb = v[ids].permute(1, 0, 2, 4, 3).reshape(nkv, -1, hd)
            last = (b, (kb, vb))
        kb, vb = (t[:, :pos + 1] for t in last[1])
        sc = x[row] @ kb.transpose(1, 2) * scale
        p = torch.softmax(sc, -1)
        out[row] = p @ vb
        size = (x[row].abs() @ kb.abs().transpose(1, 2)) * scale
        ds = (hd * size + 4 * sc.abs()).amax(-1, keepdim=True) * 2.0 ** -24
        a = p @ vb.abs()
        n = pos + 1
        bound[row] = a * (2 * u + 2 * ds + 2 * n * 2.0 ** -24) + u * out[row].abs() \
            + subnormal(dt) + 2.0 ** -22 * vb.abs().amax(1)[:, None]
    return out.view(-1, nh * hd), bound.view(-1, nh * hd)


def adjust(logits, text=None, lens=None, prompt=None, rep=1.0, pres=0.0, freq=0.0, bias=None,
           allowed=None):
    """-> (out, bound) in 64 bits, from host values (lists of tokens per row)."""
    B, V = logits.shape
    x = logits.double().clone()
    dt = logits.dtype
    size = x.abs().nan_to_num(posinf=0.0)  # the magnitudes that were added up
    for b in range(B):
        r, p, f = (float(a[b]) if isinstance(a, torch.Tensor) else a for a in (rep, pres, freq))
        row = [] if text is None else text[b].tolist()
        n = len(row) if lens is None else min(max(int(lens[b]), 0), len(row))
        first = 0 if prompt is None else int(prompt[b])
        for t in set(row[:n]):
            if 0 <= t < V:
                x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                size[b, t] = max(size[b, t], x[b, t].abs())
        new = row[max(first, 0):n]
        for t in set(new):
            if 0 <= t < V:
                x[b, t] -= f * new.count(t) + p
                size[b, t] += abs(f) * new.count(t) + abs(p)
        if bias is not None:
            for t, w in dict(zip(bias[0][b].tolist(), bias[1][b].tolist())).items():
                if 0 <= t < V:
                    x[b, t] += w
                    size[b, t] += abs(w)
        if allowed is not None:
            for t in range(V):
                if not (int(allowed[b, t >> 5]) >> (t & 31)) & 1:
                    x[b, t] = -math.inf
    # (fp32: five roundings at most before the last)
    return x, half_step(dt) * x.abs().nan_to_num(posinf=0.0, neginf=0.0) \
        + 6 * 2.0 ** -24 * size + subnormal(dt)
