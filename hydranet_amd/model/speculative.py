"""Speculative decoding over the decoder's KV cache: several drafted tokens per
sequence, a chain or a tree, pass through the model at once and are accepted or
rejected so that the kept tokens are distributed as the target model's own
(the reference's spec/verifier.py:216-330 and inference/speculative.py:331-405,
chains there).

* ``DraftTree``       the nodes' parents, checked, with their depths and ancestors;
* ``tree_append``     RoPE at each sequence's own positions and the cache append;
* ``tree_attention``  each node over the cached positions and its ancestors;
* ``verify_tree``     acceptance from given uniforms, and the next token;
* ``KVCache.keep`` / ``KVCache.fork`` (model/decoder.py) compact the accepted
  nodes' positions and copy a prompt's to further sequences;
* ``generate``        the loop around them (MixtralDecoder.generate_speculative).

A sequence's length is an entry of a device tensor lens [B] (int64; negative: it
takes no part), so sequences advance by their own accepted counts without a host
synchronisation, and every step can be captured into a graph.  On the GPU each
function is one library call (include/hn_int4.h); on the CPU, the same
definitions in torch, also of what is no number: a position that a row does not
see has no effect on it, whatever it holds.
"""
from __future__ import annotations

import math
from typing import Callable, List, NamedTuple, Optional, Union

import numpy as np
import torch

from .. import _lib

MAX_NODES = 256
PADDING = -2
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class DraftTree:
    """Nodes of a draft: parents int32 [S] (every sequence's tree) or [B, S],
    parents[i] < i, -1 directly below the cached positions; PADDING (or any other
    value) marks a node that is not there, and everything below it.  Node 0 is
    the last decided token.  Kept with it: up (the checked parents), depth (-1:
    padding) and seen (256 bits per node: itself and its ancestors)."""

    def __init__(self, parents: torch.Tensor):
        assert parents.dtype == torch.int32 and parents.dim() in (1, 2), \
            "parents: int32 [nodes] or [batch, nodes]"
        p = parents.unsqueeze(0) if parents.dim() == 1 else parents
        n, S = p.shape
        assert n >= 1 and 1 <= S <= MAX_NODES, f"1 to {MAX_NODES} nodes, got {tuple(p.shape)}"
        self.trees, self.nodes, self.device = n, S, p.device
        if p.is_cuda:
            if p.stride(1) != 1 or p.stride(0) < S:
                p = p.contiguous()
            self.up, self.depth = torch.empty((2, n, S), dtype=torch.int32, device=p.device)
            self.seen = torch.empty((n, S, MAX_NODES // 64), dtype=torch.int64, device=p.device)
            _lib.call_on(p.device, "hn_tree_plan", p.data_ptr(), max(p.stride(0), S), n, S,
                         self.up.data_ptr(), self.depth.data_ptr(), self.seen.data_ptr())
            return
        self.up = torch.full((n, S), PADDING, dtype=torch.int32)
        self.depth = torch.full((n, S), -1, dtype=torch.int32)
        bits = np.zeros((n, S, MAX_NODES), dtype=np.uint8)
        for b, row in enumerate(p.tolist()):
            for i, at in enumerate(row):
                if at == -1 or (0 <= at < i and self.depth[b, at] >= 0):
                    self.up[b, i] = at
                    self.depth[b, i] = 0 if at < 0 else self.depth[b, at] + 1
                    bits[b, i] = 0 if at < 0 else bits[b, at]
                    bits[b, i, i] = 1
        packed = np.packbits(bits, axis=-1, bitorder="little").view(np.int64)
        self.seen = torch.from_numpy(packed.copy())

    @staticmethod
    def chain(nodes: int, device=None) -> "DraftTree":
        """Node i below node i - 1."""
        return DraftTree(torch.arange(-1, nodes - 1, dtype=torch.int32, device=device))

    def visible(self) -> torch.Tensor:
        """[trees, S, S] bool: whether node i sees node j."""
        j = torch.arange(self.nodes, device=self.device)
        return ((self.seen[:, :, j >> 6] >> (j & 63)) & 1).bool()

    def _fits(self, batch: int, device) -> None:
        assert self.trees in (1, batch), f"{self.trees} trees for {batch} sequences"
        assert self.device == device, f"the tree is on {self.device}, the call on {device}"


def _check_lens(lens: torch.Tensor, B: int, device) -> None:
    assert lens.dtype == torch.int64 and tuple(lens.shape) == (B,) and lens.device == device \
        and lens.is_contiguous(), f"lens: int64 [{B}] on {device}"


def tree_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, tree: DraftTree,
                lens: torch.Tensor, cache, layer: int, num_heads: int) -> torch.Tensor:
    """RoPE and the cache append of a step's nodes.  qkv [B * S, (heads + 2
    kv_heads) * hd]: the fused projection's rows (query heads, keys, values); cos,
    sin [positions, hd] fp32.  Node i of sequence b is rotated at position lens[b]
    + its depth and its key and value go to cache position lens[b] + i.  Returns
    the rotated queries [B, kv_heads, heads / kv_heads * S, hd].  The products
    are fp32, rounded once.  Padding nodes and sequences with a negative length
    leave the cache as it is and have zero queries; a node past the cache or the
    table writes nothing and has NaN queries."""
    kt, v = cache.kt[layer], cache.v[layer]
    B, nkv, hd, max_len = kt.shape
    S, dev = tree.nodes, qkv.device
    tree._fits(B, dev)
    _check_lens(lens, B, dev)
    assert num_heads > 0 and num_heads % nkv == 0, f"{num_heads} heads over {nkv} KV heads"
    assert tuple(qkv.shape) == (B * S, (num_heads + 2 * nkv) * hd), \
        f"qkv {tuple(qkv.shape)} vs {B} x {S} rows of {num_heads} + 2 x {nkv} heads of {hd}"
    assert cos.shape == sin.shape and cos.dim() == 2 and cos.shape[1] == hd \
        and cos.dtype == sin.dtype == torch.float32 and cos.device == sin.device == dev, \
        f"cos, sin: fp32 [positions, {hd}] on {dev}"
    rep = num_heads // nkv
    if qkv.is_cuda:
        _check_cache(kt, v, dev)
        assert qkv.dtype == torch.float16 and hd == 128, "fp16 rows of heads of 128"
        if qkv.stride(1) != 1 or qkv.stride(0) < qkv.shape[1]:
            qkv = qkv.contiguous()
        cos, sin = cos.contiguous(), sin.contiguous()
        q = torch.empty((B, nkv, rep * S, hd), dtype=qkv.dtype, device=dev)
        _lib.call_on(dev, "hn_tree_append", qkv.data_ptr(), max(qkv.stride(0), qkv.shape[1]),
                     cos.data_ptr(), sin.data_ptr(), cos.shape[0], tree.depth.data_ptr(),
                     tree.trees, lens.data_ptr(), B, S, nkv, rep, hd, q.data_ptr(),
                     kt.data_ptr(), v.data_ptr(), max_len)
        return q
    depth, at = tree.depth.expand(B, S).long(), torch.arange(S)
    live = (depth >= 0) & (lens >= 0)[:, None]
    start = lens.clamp(max=2 ** 62)[:, None]  # (no sum wraps)
    pos, slot = start + depth, start + at
    ok = live & (pos < cos.shape[0]) & (slot < max_len)
    x = qkv.view(B, S, num_heads + 2 * nkv, hd)
    x32 = x if x.dtype == torch.float64 else x.float()
    half = torch.cat((-x32[..., hd // 2:], x32[..., :hd // 2]), -1)
    p = torch.where(ok, pos, 0)
    y = x32 * cos[p][:, :, None] + half * sin[p][:, :, None]
    y = torch.where(ok[..., None, None], y, torch.where(live, math.nan, 0.0)[..., None, None])
    y = y.to(qkv.dtype)
    b, i = ok.nonzero(as_tuple=True)
    kt[b, :, :, slot[b, i]] = y[b, i, num_heads:num_heads + nkv].to(kt.dtype)
    v[b, :, slot[b, i]] = x[b, i, num_heads + nkv:].to(v.dtype)
    q = y[:, :, :num_heads].reshape(B, S, nkv, rep, hd).permute(0, 2, 3, 1, 4)
    return q.reshape(B, nkv, rep * S, hd)


def _check_cache(kt: torch.Tensor, v: torch.Tensor, dev) -> None:
    B, nkv, hd, max_len = kt.shape
    assert tuple(v.shape) == (B, nkv, max_len, hd) and kt.dtype == v.dtype == torch.float16 \
        and kt.device == v.device == dev and kt.is_contiguous() and v.is_contiguous(), \
        f"a contiguous fp16 cache on {dev}: keys [B, kv_heads, hd, len], values [B, kv_heads, len, hd]"


def tree_attention(q: torch.Tensor, tree: DraftTree, lens: torch.Tensor, cache, layer: int,
                   kv_bound: int) -> torch.Tensor:
    """Attention of a step's nodes (tree_append's queries [B, kv_heads, rep * S,
    hd], their keys and values in the cache) over the cached positions and each
    node's ancestors -> [B, S, heads * hd].  kv_bound: a host bound of lens + S
    (it sizes the launch; a longer sequence gives NaN).  Rows of padding nodes and
    of sequences with a negative length are zero."""
    kt, v = cache.kt[layer], cache.v[layer]
    B, nkv, hd, max_len = kt.shape
    S, dev = tree.nodes, q.device
    tree._fits(B, dev)
    _check_lens(lens, B, dev)
    assert q.dim() == 4 and q.shape[0] == B and q.shape[1] == nkv and q.shape[3] == hd \
        and q.shape[2] % S == 0 and q.shape[2] > 0, f"q {tuple(q.shape)} vs cache {tuple(kt.shape)}"
    assert S <= kv_bound <= max_len, f"kv_bound {kv_bound}: {S} nodes, a cache of {max_len}"
    rep = q.shape[2] // S
    if q.is_cuda:
        _check_cache(kt, v, dev)
        assert q.dtype == torch.float16 and hd == 128 and max_len % 8 == 0, \
            "fp16 heads of 128, a cache of a multiple of 8 positions"
        q = _lib.aligned_rows(q.contiguous())
        out = torch.empty((B, S, nkv * rep * hd), dtype=q.dtype, device=dev)
        n = _lib.lib().hn_tree_attention_workspace_bytes(B, nkv, rep, S, kv_bound)
        work = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        scale = float(np.float32(1.0) / np.float32(math.sqrt(hd)))
        _lib.call_on(dev, "hn_tree_attention", q.data_ptr(), kt.data_ptr(), v.data_ptr(), max_len,
                     lens.data_ptr(), tree.seen.data_ptr(), tree.trees, B, nkv, rep, hd, S,
                     kv_bound, scale, out.data_ptr(), out.stride(1),
                     None if work is None else work.data_ptr(), n)
        return out
    at = torch.arange(kv_bound) - lens[:, None]  # node at each position, negative: cached
    node = at.clamp(0, S - 1)[:, None].expand(B, S, kv_bound)
    see = torch.gather(tree.visible().expand(B, S, S), 2, node) & (at < S)[:, None]
    live = (tree.depth.expand(B, S) >= 0) & (lens >= 0)[:, None]
    see = ((see | (at < 0)[:, None]) & live[..., None])[:, None, None]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    s = torch.matmul(q.to(wide), kt[..., :kv_bound].to(wide)) / math.sqrt(hd)
    s = s.view(B, nkv, rep, S, kv_bound).masked_fill(~see, -math.inf)
    p = torch.where(see, torch.softmax(s, -1), 0.0)
    vv = v[:, :, :kv_bound].to(wide)
    vv = torch.where((at < S)[:, None, :, None], vv, 0.0)  # positions no node sees
    # a node's value that is no number reaches the rows that see it, not the product,
    # where 0 times it would reach every row
    odd = ~vv.isfinite() & (at >= 0)[:, None, :, None]
    o = torch.matmul(p.view(B, nkv, rep * S, kv_bound), torch.where(odd, 0.0, vv))
    o = o.view(B, nkv, rep, S, hd)
    for b, n in odd.any(3).any(1).nonzero().tolist():
        o[b, :, :, see[b, 0, 0, :, n]] += torch.where(odd, vv, 0.0)[b, :, n][:, None, None]
    o = torch.where(live[:, None, None, :, None], o, 0.0).view(B, nkv * rep, S, hd)
    o = torch.where((lens > kv_bound - S)[:, None, None, None] & live[:, None, :, None],
                    math.nan, o)
    return o.transpose(1, 2).reshape(B, S, nkv * rep * hd).to(q.dtype)


class Verified(NamedTuple):
    path: torch.Tensor   # [B, S] int32: node 0 and the accepted nodes, then -1
    count: torch.Tensor  # [B] int32: how many those are
    token: torch.Tensor  # [B] int64: the token after them (-1: no logit was finite)


def verify_tree(logits: torch.Tensor, tokens: torch.Tensor, tree: DraftTree,
                uniforms: torch.Tensor, draft_logits: Optional[torch.Tensor] = None,
                temperature: Union[float, torch.Tensor] = 1.0) -> Verified:
    """Accepts drafted tokens against the target's probabilities softmax(logits /
    temperature) so that what is kept is distributed as drawn from the target.

    logits [B, S, V] (fp16, bf16 or fp32): the target's after each node; tokens
    [B, S] int64: the nodes' tokens; uniforms [B, S] fp32 in [0, 1): entry i tests
    node i, entry 0 draws the token after the accepted nodes.  draft_logits, like
    logits: the drafter's after each node, from whose softmax (at the same
    temperature) its children were drawn; None: every drafted token is a certain
    proposal.  temperature: a number (rounded to fp32), or fp32 [B]; 0 takes the
    largest logit (the lowest index of equals).  Children are tested in order of
    index: accepted with probability min(1, r(x) / q(x)), r = p at first and
    norm(max(r - q, 0)) after a rejection (a certain proposal's: r without its
    token)."""
    assert logits.dim() == 3 and logits.dtype in _DTYPES, "logits: fp16, bf16 or fp32 [B, S, V]"
    B, S, V = logits.shape
    dev = logits.device
    tree._fits(B, dev)
    assert tree.nodes == S and V > 0, f"{tree.nodes} nodes, logits {tuple(logits.shape)}"
    assert tokens.dtype == torch.int64 and tuple(tokens.shape) == (B, S) and tokens.device == dev, \
        f"tokens: int64 [{B}, {S}] on {dev}"
    assert uniforms.dtype == torch.float32 and tuple(uniforms.shape) == (B, S) \
        and uniforms.device == dev, f"uniforms: fp32 [{B}, {S}] on {dev}"
    assert draft_logits is None or (draft_logits.shape == logits.shape
                                    and draft_logits.dtype == logits.dtype
                                    and draft_logits.device == dev), \
        "draft_logits: shape, type and device of logits"
    temps, temp = None, 0.0
    if isinstance(temperature, torch.Tensor):
        assert temperature.dtype == torch.float32 and tuple(temperature.shape) == (B,) \
            and temperature.device == dev, f"temperature: a number or fp32 [{B}] on {dev}"
        temps = temperature.contiguous()
    else:
        temp = float(temperature)
        assert temp >= 0.0 and math.isfinite(temp), f"temperature {temperature}"
    if not logits.is_cuda:
        return _verify_cpu(logits, tokens, tree, uniforms, draft_logits,
                           temps if temps is not None else torch.full((B,), temp))
    logits, draft = _rows(logits), None if draft_logits is None else _rows(draft_logits)
    tokens, uniforms = tokens.contiguous(), uniforms.contiguous()
    path = torch.empty((B, S), dtype=torch.int32, device=dev)
    count = torch.empty(B, dtype=torch.int32, device=dev)
    token = torch.empty(B, dtype=torch.int64, device=dev)
    n = _lib.lib().hn_verify_tree_workspace_bytes(B, S, V)
    work = torch.empty(n, dtype=torch.uint8, device=dev)
    d = (None, 0, 0) if draft is None else (draft.data_ptr(), draft.stride(0), draft.stride(1))
    _lib.call_on(dev, "hn_verify_tree", logits.data_ptr(), logits.stride(0), logits.stride(1), *d,
                 _DTYPES[logits.dtype], tokens.data_ptr(), tree.up.data_ptr(), tree.trees,
                 uniforms.data_ptr(), None if temps is None else temps.data_ptr(), temp, B, S, V,
                 path.data_ptr(), count.data_ptr(), token.data_ptr(), work.data_ptr(), n)
    return Verified(path, count, token)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with its last axis dense and rows that do not overlap."""
    return x if x.stride(2) == 1 and (x.shape[1] == 1 or x.stride(1) >= x.shape[2]) \
        else x.contiguous()


def _verify_cpu(logits, tokens, tree, uniforms, draft, temps) -> Verified:
    B, S, V = logits.shape
    tiny = 2.0 ** -40
    path = torch.full((B, S), -1, dtype=torch.int32)
    count = torch.ones(B, dtype=torch.int32)
    token = torch.empty(B, dtype=torch.int64)

    def soften(x, t):
        x = torch.where(x.isnan(), -math.inf, x.double()).clamp(max=torch.finfo(torch.float32).max)
        if x.max() == -math.inf:
            return torch.zeros(V, dtype=torch.float64)
        if not t > 0:
            return torch.nn.functional.one_hot((x == x.max()).nonzero()[0, 0], V).double()
        return torch.softmax(x / t, 0)

    for b in range(B):
        up = tree.up[b if tree.trees > 1 else 0].tolist()
        t, u = float(temps[b]), uniforms[b].double().tolist()
        cur, n = 0, 1
        path[b, 0] = 0
        p = r = soften(logits[b, 0], t)
        mass, c = 1.0, 0.0
        for i in range(1, S):
            x = int(tokens[b, i])
            if up[i] != cur or not 0 <= x < V or mass <= tiny:
                continue
            if not t > 0:
                q, take = None, bool(p[x] > 0)
            elif draft is None:
                q, take = None, u[i] * mass < float(r[x])
            else:
                q = soften(draft[b, cur], t)
                take = u[i] * float(q[x]) * mass < float(p[x] - c * q[x])
            if take:
                path[b, n] = cur = i
                n += 1
                p = r = soften(logits[b, i], t)
                mass, c = 1.0, 0.0
            elif t > 0:
                if q is None:
                    r = r.clone()
                    mass -= float(r[x])
                    r[x] = 0.0
                else:
                    c += mass
                    r = (p - c * q).clamp(min=0)
                    mass = float(r.sum())
        r = r if mass > tiny else p
        count[b] = n
        run = r.cumsum(0)
        hit = ((run > u[0] * float(run[-1])) & (r > 0)).nonzero()
        pos = (r > 0).nonzero()
        token[b] = hit[0, 0] if len(hit) else pos[-1, 0] if len(pos) else -1
    return Verified(path, count, token)


class Draft(NamedTuple):
    tokens: torch.Tensor                  # [B, S - 1] int64: of nodes 1 on (outside the
    #                                       vocabulary: never accepted)
    parents: torch.Tensor                 # int32 [S] or [B, S], node 0 (-1) the last token
    logits: Optional[torch.Tensor] = None  # [B, S, V]: the drafter's after each node


def ngram_draft(history: List[List[int]], device, nodes: int = 8, match: int = 2) -> Draft:
    """What followed the last earlier occurrence of each sequence's last `match`
    tokens, as a chain of up to nodes - 1 certain proposals (the n-gram drafters of
    the reference's inference/speculative.py); a sequence without one gets padding."""
    rows, parents = [], []
    for h in history:
        tail, got = h[-match:], []
        for at in range(len(h) - match - 1, -1, -1):
            if h[at:at + match] == tail:
                got = h[at + match:at + match + nodes - 1]
                break
        rows.append(got + [0] * (nodes - 1 - len(got)))
        parents.append(list(range(-1, len(got))) + [PADDING] * (nodes - 1 - len(got)))
    return Draft(torch.tensor(rows, dtype=torch.int64, device=device).view(len(rows), nodes - 1),
                 torch.tensor(parents, dtype=torch.int32, device=device))


@torch.no_grad()
def generate(model, input_ids: torch.Tensor, max_new_tokens: int,
             draft: Optional[Callable[[List[List[int]], torch.device], Draft]] = None,
             temperature: float = 0.0, samples: int = 1,
             generator: Optional[torch.Generator] = None, max_nodes: int = 64) -> torch.Tensor:
    """Speculative decoding of a MixtralDecoder: prompts [B, P] (one length) ->
    [samples * B, max_new_tokens], row s * B + b the s-th continuation of prompt b.
    Each prompt is prefilled once and its cache forked to its samples; a pass then
    takes the last token and the drafter's tree of each sequence, verifies, and
    compacts the cache.  draft(history, device) -> Draft, history the tokens of
    each sequence so far, at most max_nodes nodes.  A pass reads the device back once
    (beside what the drafter does)."""
    draft = draft or ngram_draft
    B, P = input_ids.shape
    assert samples >= 1 and max_new_tokens >= 1 and P >= 1, "samples, tokens and prompt >= 1"
    dev, N = input_ids.device, samples * B
    prompt = input_ids.tolist()
    history = [list(prompt[i % B]) for i in range(N)]
    longest = -(-(P + max_new_tokens + max_nodes) // 8) * 8  # a pass writes past what it keeps
    cache = model.new_cache(N, longest)
    first = type(cache).wrap([t[:B] for t in cache.kt], [t[:B] for t in cache.v])
    first_logits = model.forward(input_ids, first)[:, -1:]
    cache.fork([i % B for i in range(B, N)], list(range(B, N)), P)

    def uniforms(nodes):
        return torch.rand((N, nodes), generator=generator, device=dev)

    one = DraftTree.chain(1, dev)
    last = verify_tree(first_logits.repeat(samples, 1, 1), torch.zeros((N, 1), dtype=torch.int64,
                       device=dev), one, uniforms(1), None, temperature).token
    lens = torch.full((N,), P, dtype=torch.int64, device=dev)
    size, out = [P] * N, [[] for _ in range(N)]

    def emit(i, tokens):
        # (a draft may reach past the last position of the model: no logits there)
        tokens = tokens[:max_new_tokens - len(out[i])]
        if -1 in tokens:
            raise RuntimeError(f"sequence {i}: no logit is finite")
        out[i] += tokens
        history[i] += tokens
        return len(out[i]) >= max_new_tokens

    done, out_of = [emit(i, [t]) for i, t in enumerate(last.tolist())], 0
    while not all(done):
        if sum(done) > out_of:  # finished sequences take no part
            out_of = sum(done)
            lens = torch.where(torch.tensor(done, device=dev), -1, lens)
        d = draft(history, dev)
        tree = DraftTree(d.parents)
        tokens = torch.cat((last.clamp(min=0)[:, None], d.tokens), 1)
        assert tokens.shape[1] == tree.nodes, f"{tree.nodes} nodes, {d.tokens.shape[1]} tokens"
        assert tree.nodes <= max_nodes, f"at most {max_nodes} nodes, the draft has {tree.nodes}"
        bound = max(n for n, over in zip(size, done) if not over) + tree.nodes
        inside = tokens.clamp(0, first_logits.shape[-1] - 1)
        logits = model.forward_tree(inside, tree, lens, cache, bound)
        r = verify_tree(logits, tokens, tree, uniforms(tree.nodes), d.logits, temperature)
        lens = cache.keep(lens, r.path, r.count)
        last = r.token
        took = torch.gather(tokens, 1, r.path.clamp(min=0).long())
        back = torch.cat((r.count[:, None].long(), last[:, None], took), 1)
        for i, (n, x, *t) in enumerate(back.tolist()):
            if not done[i]:
                size[i] += n
                done[i] = emit(i, t[1:n] + [x])
    return torch.tensor(out, dtype=torch.int64, device=dev)
