"""The operators of tree-speculative decoding over the decoder's dense KV cache,
in plain torch and as the package's kernels, with their exact (64-bit) results.

Kinds of a case (``case["kind"]``):

* ``append``  tree_append: RoPE of a step's drafted tokens at each sequence's own
              positions, and their keys and values written to the cache.
* ``attend``  tree_attention: every drafted token attends over its sequence's
              cached positions and its ancestors in the tree.
* ``verify``  verify_tree: drafted tokens accepted or rejected against the
              target's probabilities, the next token drawn, from given uniforms.
* ``keep``    KVCache.keep: the accepted nodes' positions compacted, every layer.
* ``fork``    KVCache.fork: a prompt's positions copied to further sequences.

A tree of S nodes is a row of parents: node 0 is the sequence's last decided
token (parent -1), node i hangs below parents[i] < i; -2 marks padding.  Keys
are cached transposed, [B, kv_heads, 128, max_len], values [B, kv_heads,
max_len, 128]; node i of a sequence with C cached positions sits at C + i, its
rotary position is C + its depth.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HD = 128
TINY = 2.0 ** -40  # residual mass below which nothing is left to draw from
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # the drafted chain of one sequence: a launch's latency
        {"name": "append_b1_s5", "kind": "append", "batch": 1, "nodes": 5, "fan": 1, "pad": 0,
         "kv_heads": 8, "rep": 4, "max_len": 1024, "low": 300, "high": 900},
        # a batch of trees, some with fewer nodes than the widest
        {"name": "append_b32_s61", "kind": "append", "batch": 32, "nodes": 61, "fan": 3, "pad": 17,
         "kv_heads": 8, "rep": 4, "max_len": 4096, "low": 900, "high": 4000},
        # one token of one sequence: decoding without a draft
        {"name": "attend_b1_s1", "kind": "attend", "batch": 1, "nodes": 1, "fan": 1, "pad": 0,
         "kv_heads": 8, "rep": 4, "max_len": 2048, "low": 1501, "high": 1501},
        # a wide tree after a long context: few workgroups' worth of rows, a long axis
        {"name": "attend_b2_s61_long", "kind": "attend", "batch": 2, "nodes": 61, "fan": 4,
         "pad": 0, "kv_heads": 8, "rep": 4, "max_len": 32768, "low": 23001, "high": 31777},
        # a serving batch of ragged lengths, twelve query heads to a KV head
        {"name": "attend_b32_s9_ragged", "kind": "attend", "batch": 32, "nodes": 9, "fan": 2,
         "pad": 3, "kv_heads": 8, "rep": 12, "max_len": 8192, "low": 1200, "high": 8000},
        # greedy check of a short chain of one sequence
        {"name": "verify_b1_s5_greedy", "kind": "verify", "batch": 1, "nodes": 5, "fan": 1,
         "pad": 0, "vocab": 32000, "type": "fp16", "draft": False, "temperature": 0.0},
        # sampled trees whose drafter gives its probabilities
        {"name": "verify_b8_s61", "kind": "verify", "batch": 8, "nodes": 61, "fan": 4, "pad": 9,
         "vocab": 32000, "type": "fp16", "draft": True, "temperature": 0.8},
        # a serving batch of sampled chains over a large vocabulary
        {"name": "verify_b32_s6_large", "kind": "verify", "batch": 32, "nodes": 6, "fan": 1,
         "pad": 0, "vocab": 128000, "type": "fp32", "draft": True, "temperature": 1.0},
        # one sequence's accepted branch
        {"name": "keep_b1", "kind": "keep", "batch": 1, "nodes": 26, "kv_heads": 8, "layers": 32,
         "max_len": 2048, "low": 1333, "high": 1333},
        # a batch's accepted branches, each of its own length
        {"name": "keep_b32", "kind": "keep", "batch": 32, "nodes": 61, "kv_heads": 8, "layers": 32,
         "max_len": 512, "low": 100, "high": 440},
        # a short prompt continued three times
        {"name": "fork_b4", "kind": "fork", "batch": 4, "prompts": 1, "kv_heads": 8, "layers": 32,
         "max_len": 512, "length": 333},
        # two long prompts continued several times each
        {"name": "fork_b12_long", "kind": "fork", "batch": 12, "prompts": 2, "kv_heads": 8,
         "layers": 32, "max_len": 2048, "length": 1901},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "verify", "verify", "keep", "fork"))
    nodes = _log(rng, 1, 128)
    fan = rng.choice((1, 2, 3, 4, 6))
    pad = rng.randrange(nodes) if rng.random() < 0.5 else 0
    if kind in ("append", "attend"):
        high = _log(rng, 2, 32000)
        max_len = -(-(high + nodes + rng.randrange(400)) // 8) * 8
        low = rng.randint(1, high)
        # cached positions of the whole batch at most about half a million
        batch = max(1, min(_log(rng, 1, 32), 250_000 // max_len))
        return {"kind": kind, "batch": batch, "nodes": nodes, "fan": fan, "pad": pad,
                "kv_heads": rng.choice((1, 2, 4, 8)), "rep": rng.choice((1, 2, 4, 8, 12)),
                "max_len": max_len, "low": low, "high": high}
    if kind == "verify":
        vocab = _log(rng, 500, 128000)
        batch = max(1, min(_log(rng, 1, 32), 24_000_000 // (vocab * nodes)))
        return {"kind": kind, "batch": batch, "nodes": nodes, "fan": fan, "pad": pad,
                "vocab": vocab, "type": rng.choice(("fp16", "bf16", "fp32")),
                "draft": rng.random() < 0.6,
                "temperature": rng.choice((0.0, 0.5, 0.8, 1.0, 1.3))}
    layers = _log(rng, 1, 32)
    max_len = 8 * _log(rng, 18, 256)
    batch = rng.randint(1 if kind == "keep" else 2, max(2, min(32, 20_000 // max_len)))
    if kind == "keep":
        high = rng.randint(1, max_len - nodes)
        return {"kind": kind, "batch": batch, "nodes": nodes, "kv_heads": rng.choice((1, 2, 4, 8)),
                "layers": layers, "max_len": max_len, "low": rng.randint(1, high), "high": high}
    return {"kind": kind, "batch": batch, "prompts": rng.randint(1, batch - 1),
            "kv_heads": rng.choice((1, 2, 4, 8)), "layers": layers, "max_len": max_len,
            "length": rng.randint(1, max_len)}


# ----------------------------------------------------------------------------- trees
def _parents(case):
    """Rows of parents, the same for every seed: node i below node (i - 1) // fan (fan 1: a
    chain), every second sequence with the last `pad` nodes missing."""
    row = [-1] + [(i - 1) // case["fan"] for i in range(1, case["nodes"])]
    short = row[:case["nodes"] - case["pad"]] + [-2] * case["pad"]
    return [short if b % 2 else row for b in range(case["batch"])]


def _ancestors(parents):
    """Of each node, itself and the nodes above it."""
    paths = []
    for i, p in enumerate(parents):
        paths.append([] if p == -2 else [i] if p == -1 else paths[p] + [i])
    return paths


def _plan(case):
    """Per node: depth [B, S] (-1: padding) and the nodes it sees [B, S, S]."""
    rows = {}
    for r in map(tuple, _parents(case)):
        if r not in rows:
            paths = _ancestors(r)
            see = torch.zeros(len(r), len(r), dtype=torch.bool)
            for i, p in enumerate(paths):
                see[i, p] = True
            rows[r] = (torch.tensor([len(p) - 1 for p in paths]), see)
    got = [rows[tuple(r)] for r in _parents(case)]
    return (torch.stack([d for d, _ in got]).to(DEV), torch.stack([s for _, s in got]).to(DEV))


# ----------------------------------------------------------------------------- inputs
def _lens(case, g):
    return torch.randint(case["low"], case["high"] + 1, (case["batch"],), generator=g, device=DEV)


def _tables(n):
    inv = 1.0 / (1e6 ** (torch.arange(0, HD, 2, device=DEV, dtype=torch.float64) / HD))
    a = torch.outer(torch.arange(n, device=DEV, dtype=torch.float64), inv).repeat(1, 2)
    return a.cos().float(), a.sin().float()


def _randn(shape, g, dtype=torch.float16, scale=1.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, scale, generator=g)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    kind, B = case["kind"], case["batch"]
    if kind in ("append", "attend", "verify"):
        S = case["nodes"]
        s["parents"] = torch.tensor(_parents(case), dtype=torch.int32, device=DEV)
        s["depth"], s["see"] = _plan(case)
        if own:
            from hydranet_amd.model.speculative import DraftTree
            s["tree"] = DraftTree(s["parents"])
    if kind in ("append", "attend"):
        nkv, rep, L = case["kv_heads"], case["rep"], case["max_len"]
        s["lens"] = _lens(case, g)
        s["kt"] = [_randn((B, nkv, HD, L), g)]
        s["v"] = [_randn((B, nkv, L, HD), g)]
        if kind == "append":
            s["qkv"] = _randn((B * S, (nkv * rep + 2 * nkv) * HD), g)
            s["cos"], s["sin"] = _tables(L)
        else:
            # queries that prefer some positions, as trained ones do: scores of deviation 2
            s["q"] = _randn((B, nkv, rep * S, HD), g, scale=2.0)
    elif kind == "verify":
        V, dt = case["vocab"], TYPES[case["type"]]
        # a few likely tokens over a long tail; the drafter knows most of it
        base = _randn((B, S, V), g, torch.float32, 2.5)
        s["draft"] = None
        draft = base.to(dt)
        s["logits"] = (base + _randn((B, S, V), g, torch.float32, 0.7)).to(dt)
        del base
        if case["draft"]:
            s["draft"] = draft
        # each node's token is drawn from the drafter's distribution after its parent; a drafter
        # that gives no probabilities proposes its likeliest tokens
        up = s["parents"].clamp(min=0).long()
        t = max(case["temperature"], 0.25) if case["draft"] else 0.25
        gum = torch.empty((B, S, V), device=DEV).exponential_(1.0, generator=g).log_().neg_()
        best = torch.gather(draft, 1, up[..., None].expand(B, S, V)).float().div_(t).add_(gum)
        s["tokens"] = best.argmax(-1)
        s["u"] = torch.rand((B, S), generator=g, device=DEV)
    else:
        nkv, n, L = case["kv_heads"], case["layers"], case["max_len"]
        s["kt"] = _randn((n, B, nkv, HD, L), g)
        s["v"] = _randn((n, B, nkv, L, HD), g)
        if kind == "keep":
            S = case["nodes"]
            s["lens"] = _lens(case, g)
            # a branch of a drafter that lists the nodes nearest the root first: its nodes past
            # the root lie behind the positions they move to, so a second pass finds them again
            most = max(1, min(9, (S + 1) // 2))
            s["count"] = torch.randint(1, most + 1, (B,), generator=g, device=DEV).int()
            order = torch.rand((B, S), generator=g, device=DEV)
            order = order.masked_fill(torch.arange(S, device=DEV) < most, 2.0)
            order[:, 0] = -1.0
            path = order.argsort(1)[:, :most].sort(1).values
            keep = torch.arange(most, device=DEV) < s["count"][:, None]
            s["path"] = torch.full((B, S), -1, dtype=torch.int32, device=DEV)
            s["path"][:, :most] = torch.where(keep, path, -1).int()
        else:
            p = case["prompts"]
            s["dst"] = list(range(p, B))
            s["src"] = [(b * 7 + seed) % p for b in s["dst"]]
    if own and "kt" in s:
        from hydranet_amd.model.decoder import KVCache
        s["cache"] = KVCache.wrap(list(s["kt"]), list(s["v"]))
    return s


# ----------------------------------------------------------------------------- one pass
def _append(s):
    B, S = s["depth"].shape
    nkv, L = s["case"]["kv_heads"], s["case"]["max_len"]
    nh = nkv * s["case"]["rep"]
    live = s["depth"] >= 0
    pos = s["lens"][:, None] + s["depth"].clamp(min=0)
    x = s["qkv"].float().view(B, S, nh + 2 * nkv, HD)
    half = torch.cat((-x[..., HD // 2:], x[..., :HD // 2]), -1)
    y = x * s["cos"][pos][:, :, None] + half * s["sin"][pos][:, :, None]
    q = torch.where(live[..., None, None], y[:, :, :nh], 0.0).half()
    q = q.view(B, S, nkv, nh // nkv, HD).permute(0, 2, 3, 1, 4)
    slot = s["lens"][:, None] + torch.arange(S, device=DEV)
    b, i = live.nonzero(as_tuple=True)
    s["kt"][0][b, :, :, slot[b, i]] = y[b, i, nh:nh + nkv].half()
    s["v"][0][b, :, slot[b, i]] = x[b, i, nh + nkv:].half()
    return q.reshape(B, nkv, -1, HD), s["kt"][0], s["v"][0]


def _attend(s):
    B, S = s["depth"].shape
    nkv, rep, L = s["case"]["kv_heads"], s["case"]["rep"], s["case"]["high"] + s["case"]["nodes"]
    kt, v = s["kt"][0][..., :L].float(), s["v"][0][:, :, :L].float()
    at = torch.arange(L, device=DEV)[None, None] - s["lens"][:, None, None]  # [B, 1, L]
    node = at.expand(B, S, L).clamp(0, S - 1)
    see = (at < 0) | ((at < S) & torch.gather(s["see"], 2, node))
    see = (see & (s["depth"] >= 0)[..., None])[:, None, None]  # [B, 1, 1, S, L]
    x = torch.matmul(s["q"].float(), kt).view(B, nkv, rep, S, L) / math.sqrt(HD)
    x = x.masked_fill(~see, -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    x = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(x.view(B, nkv, rep * S, L), v).view(B, nkv * rep, S, HD)
    return o.transpose(1, 2).reshape(B, S, -1).half()


def _lowest(x):
    """Index of the last axis' largest value, the lowest where several are."""
    V = x.shape[-1]
    return torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device=DEV), V).amin(-1)


def _verify(s):
    B, S, V = s["logits"].shape
    T, tokens, parents, u = s["case"]["temperature"], s["tokens"], s["parents"], s["u"].double()
    rows = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.long, device=DEV)
    count = torch.ones(B, dtype=torch.int32, device=DEV)
    path = torch.full((B, S), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    if T > 0:
        p = torch.softmax(s["logits"].double() / T, -1)
        q = torch.softmax(s["draft"].double() / T, -1) if s["draft"] is not None else None
        c = torch.zeros(B, dtype=torch.float64, device=DEV)
        mass = torch.ones(B, dtype=torch.float64, device=DEV)
        gone = torch.zeros(B, V, dtype=torch.bool, device=DEV)
    else:
        top = _lowest(s["logits"])
    for i in range(1, S):  # a node's test hangs on all before it
        x = tokens[:, i]
        mine = parents[:, i] == cur
        if T == 0:
            take = mine & (top[rows, cur] == x)
        else:
            px = p[rows, cur, x]
            if q is None:
                take = mine & (mass > TINY) & ~gone[rows, x] & (u[:, i] * mass < px)
                drop = mine & ~take & ~gone[rows, x]
                gone[rows, x] |= drop
                mass = torch.where(drop, mass - px, mass)
                mass = torch.where(take, 1.0, mass)
                gone &= ~take[:, None]
            else:
                qx = q[rows, cur, x]
                take = mine & (mass > TINY) & (u[:, i] * qx * mass < px - c * qx)
                drop = mine & ~take & (mass > TINY)
                c = torch.where(take, 0.0, torch.where(drop, c + mass, c))
                left = (p[rows, cur] - c[:, None] * q[rows, cur]).clamp(min=0).sum(-1)
                mass = torch.where(take, 1.0, torch.where(drop, left, mass))
        cur = torch.where(take, i, cur)
        path[rows, torch.where(take, count, 0).long()] = torch.where(take, i, 0).int()
        count += take.int()
    if T == 0:
        return path, count, top[rows, cur]
    r = p[rows, cur]
    if q is None:
        left = torch.where(gone, 0.0, r)
    else:
        left = (r - c[:, None] * q[rows, cur]).clamp(min=0)
    r = torch.where((mass > TINY)[:, None], left, r)
    run = r.cumsum(-1)
    last = torch.where(r > 0, torch.arange(V, device=DEV), 0).amax(-1)
    token = (run <= u[:, :1] * run[:, -1:]).sum(-1).minimum(last)
    return path, count, token


def _keep(s):
    n, B, nkv, _, L = s["kt"].shape
    S = s["path"].shape[1]
    j = torch.arange(S, device=DEV)
    live = j < s["count"][:, None]
    b, j = live.nonzero(as_tuple=True)
    src, dst = s["lens"][b] + s["path"][b, j], s["lens"][b] + j
    s["kt"][:, b, :, :, dst] = s["kt"][:, b, :, :, src]
    s["v"][:, b, :, dst] = s["v"][:, b, :, src]
    return s["kt"], s["v"], s["lens"] + s["count"]


def _fork(s):
    n = s["case"]["length"]
    s["kt"][:, s["dst"], :, :, :n] = s["kt"][:, s["src"], :, :, :n]
    s["v"][:, s["dst"], :, :n] = s["v"][:, s["src"], :, :n]
    return s["kt"], s["v"]


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"append": _append, "attend": _attend, "verify": _verify, "keep": _keep,
                "fork": _fork}[kind](state)
    if kind == "append":
        from hydranet_amd.model.speculative import tree_append
        q = tree_append(state["qkv"], state["cos"], state["sin"], state["tree"], state["lens"],
                        state["cache"], 0, case["kv_heads"] * case["rep"])
        return q, state["kt"][0], state["v"][0]
    if kind == "attend":
        from hydranet_amd.model.speculative import tree_attention
        return tree_attention(state["q"], state["tree"], state["lens"], state["cache"], 0,
                              case["high"] + case["nodes"])
    if kind == "verify":
        from hydranet_amd.model.speculative import verify_tree
        return tuple(verify_tree(state["logits"], state["tokens"], state["tree"], state["u"],
                                 draft_logits=state["draft"], temperature=case["temperature"]))
    if kind == "keep":
        lens = state["cache"].keep(state["lens"], state["path"], state["count"])
        return state["kt"], state["v"], lens
    state["cache"].fork(state["src"], state["dst"], case["length"])
    return state["kt"], state["v"]


# ----------------------------------------------------------------------------- floors
def work(case):
    kind, B = case["kind"], case["batch"]
    if kind in ("append", "attend", "verify"):
        trees = [_ancestors(r) for r in _parents(case)]
        live = sum(1 for t in trees for p in t if p)
    if kind in ("append", "attend"):
        nkv, rep = case["kv_heads"], case["rep"]
        row = nkv * rep * HD * 2  # one token's queries
        mean = (case["low"] + case["high"]) / 2
    if kind == "append":
        # projections read, queries and cache entries written, two fp32 table rows a token
        one = 2 * (row + 2 * nkv * HD * 2) + 2 * HD * 4
        return {"bytes": live * one, "flops": live * 3 * (nkv * rep + nkv) * HD}
    if kind == "attend":
        pairs = sum(mean * sum(1 for p in t if p) + sum(map(len, t)) for t in trees)
        kv = (B * mean + live) * nkv * HD * 2 * 2
        return {"bytes": kv + 2 * live * row, "flops": 4 * HD * nkv * rep * pairs}
    if kind == "verify":
        size = 4 if case["type"] == "fp32" else 2
        inner = sum(len({p for p in r if p >= 0}) for r in _parents(case))
        n = live + (inner if case["draft"] and case["temperature"] > 0 else 0)
        return {"bytes": n * case["vocab"] * size, "flops": 2.0 * n * case["vocab"]}
    entry = case["kv_heads"] * HD * 2 * 2 * case["layers"]  # one position of one sequence
    if kind == "keep":
        most = max(1, min(9, (case["nodes"] + 1) // 2))
        return {"bytes": 2 * max(1, B * (most - 1) / 2) * entry, "flops": 0}
    return {"bytes": case["batch"] * case["length"] * entry, "flops": 0}


# ----------------------------------------------------------------------------- exact results
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "verify": _exact_verify,
            "keep": _exact_keep, "fork": _exact_fork}[case["kind"]](case, s)


def _exact_append(case, s):
    nkv, nh, S = case["kv_heads"], case["kv_heads"] * case["rep"], case["nodes"]
    kt, v = s["kt"][0].double(), s["v"][0].double()
    q = torch.zeros(case["batch"], S, nh, HD, dtype=torch.float64, device=DEV)
    x = s["qkv"].double().view(case["batch"], S, nh + 2 * nkv, HD)
    cos, sin = s["cos"].double(), s["sin"].double()
    for b, row in enumerate(_parents(case)):
        C = int(s["lens"][b])
        paths = _ancestors(row)
        n = sum(1 for p in paths if p)
        at = torch.tensor([C + len(p) - 1 for p in paths[:n]], device=DEV)
        lo, hi = x[b, :n, :nh + nkv, :HD // 2], x[b, :n, :nh + nkv, HD // 2:]
        c, sn = cos[at][:, None], sin[at][:, None]
        y = torch.cat((lo * c[..., :HD // 2] - hi * sn[..., :HD // 2],
                       hi * c[..., HD // 2:] + lo * sn[..., HD // 2:]), -1)
        q[b, :n] = y[:, :nh]
        kt[b, :, :, C:C + n] = y[:, nh:].permute(1, 2, 0)
        v[b, :, C:C + n] = x[b, :n, nh + nkv:].transpose(0, 1)
    q = q.view(case["batch"], S, nkv, case["rep"], HD).permute(0, 2, 3, 1, 4)
    return q.reshape(case["batch"], nkv, -1, HD), kt, v


def _exact_attend(case, s):
    nkv, rep, S = case["kv_heads"], case["rep"], case["nodes"]
    out = torch.zeros(case["batch"], S, nkv, rep, HD, dtype=torch.float64, device=DEV)
    for b, row in enumerate(_parents(case)):
        C = int(s["lens"][b])
        hide = torch.ones(S, S, dtype=torch.bool)
        for i, p in enumerate(_ancestors(row)):
            hide[i, p] = False
        live = (~hide).any(1).to(DEV)
        for h in range(nkv):
            k, v = s["kt"][0][b, h, :, :C + S].double(), s["v"][0][b, h, :C + S].double()
            x = (s["q"][b, h].double() @ k).view(rep, S, C + S) * HD ** -0.5
            x[:, :, C:].masked_fill_(hide.to(DEV), -torch.inf)
            y = (torch.softmax(x, -1).view(rep * S, -1) @ v).view(rep, S, HD)
            out[b, :, h] = torch.where(live[:, None, None], y.transpose(0, 1), 0.0)
    return out.view(case["batch"], S, -1)


def _exact_verify(case, s):
    B, S, V, T = case["batch"], case["nodes"], case["vocab"], case["temperature"]
    path = torch.full((B, S), -1, dtype=torch.int32)
    count, token = torch.zeros(B, dtype=torch.int32), torch.zeros(B, dtype=torch.long)
    tokens, u = s["tokens"].tolist(), s["u"].double().tolist()
    for b, row in enumerate(_parents(case)):
        got, here = [0], 0
        while here is not None:
            node, here = here, None
            lg = s["logits"][b, node].double()
            if T == 0:
                r = (torch.arange(V, device=DEV) == int((lg == lg.max()).nonzero()[0])).double()
            else:
                r = torch.exp(lg / T - torch.logsumexp(lg / T, 0))
            p, mass = r, 1.0
            if s["draft"] is not None and T > 0:
                d = s["draft"][b, node].double() / T
                q = torch.exp(d - torch.logsumexp(d, 0))
            for i in [i for i, up in enumerate(row) if up == node]:
                x = tokens[b][i]
                if s["draft"] is None or T == 0:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                if float(r[x]) > u[b][i] * float(q[x]):
                    got.append(i)
                    here = i
                    break
                left = (r - q).clamp(min=0)
                if T > 0:
                    mass *= float(left.sum())
                    if mass <= TINY:
                        r = p
                        break
                    r = left / left.sum()
        run_ = r.cumsum(0)
        path[b, :len(got)] = torch.tensor(got, dtype=torch.int32)
        count[b] = len(got)
        token[b] = int((run_ > u[b][0] * float(run_[-1])).nonzero()[0])
    return path, count, token


def _exact_keep(case, s):
    kt, v = s["kt"].clone(), s["v"].clone()
    for b in range(case["batch"]):
        C = int(s["lens"][b])
        for j, i in enumerate(s["path"][b, :int(s["count"][b])].tolist()):
            kt[:, b, :, :, C + j] = s["kt"][:, b, :, :, C + i]
            v[:, b, :, C + j] = s["v"][:, b, :, C + i]
    return kt, v, s["lens"] + s["count"]


def _exact_fork(case, s):
    n, kt, v = case["length"], s["kt"].clone(), s["v"].clone()
    for a, b in zip(s["src"], s["dst"]):
        kt[:, b, :, :, :n] = s["kt"][:, a, :, :, :n]
        v[:, b, :, :n] = s["v"][:, a, :, :n]
    return kt, v
