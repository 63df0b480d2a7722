"""GPU tests of the tree-speculation kernels (hn_tree.hip, hn_verify.hip,
hn_cache.hip) against node-by-node 64-bit forms, at the edges of their tiles and
splits, with what a row must not see set to NaN and infinity."""
import math
import random

import pytest
import torch

from hydranet_amd import _lib
from hydranet_amd.model.decoder import KVCache
from hydranet_amd.model.speculative import DraftTree, tree_append, tree_attention, verify_tree
from tests import _tree_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HD = 128


def _tree(rows):
    return DraftTree(torch.tensor(rows, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("S,kind", [(1, "chain"), (2, "chain"), (3, "padded"), (64, "random"),
                                    (65, "padded"), (129, "roots"), (255, "padded"),
                                    (256, "chain"), (256, "random"), (256, "padded")])
def test_plan(S, kind):
    rng = random.Random(S)
    rows = torch.tensor([ref.random_tree(rng, S, kind) for _ in range(5)], dtype=torch.int32)
    wide = torch.full((5, S + 3), 77, dtype=torch.int32)
    wide[:, :S] = rows
    a, b = DraftTree(rows), DraftTree(wide.to(DEV)[:, :S])  # rows apart from each other
    for x in ("up", "depth", "seen"):
        assert torch.equal(getattr(a, x), getattr(b, x).cpu()), x


def _tables(n):
    a = torch.outer(torch.arange(n, dtype=torch.float64),
                    1e6 ** (-torch.arange(0, HD, 2, dtype=torch.float64) / HD)).repeat(1, 2)
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


def _close(got, want, mag):
    """fp32 products (2^-24 each, and their sum's) of terms up to mag, one fp16 rounding."""
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + 3 * 2.0 ** -24 * mag
    err = (got.double() - want).abs()
    assert torch.equal(got.isnan(), want.isnan())
    assert bool((err <= bound).logical_or(want.isnan()).all()), float((err / bound).nan_to_num(0).max())


@pytest.mark.parametrize("B,nkv,rep,S,lens,n,kind,shared", [
    (1, 1, 1, 1, [0], 8, "chain", False), (1, 8, 4, 5, [1001], 1024, "chain", True),
    (5, 2, 3, 33, [0, 7, -1, 500, 480], 512, "padded", False),
    (2, 1, 12, 256, [100, 1], 357, "random", False),
    (3, 2, 1, 9, [50, 3, 17], 67, "roots", True), (4, 8, 4, 61, [3000, 17, 2222, 64], 4096, "padded", False)])
def test_append(B, nkv, rep, S, lens, n, kind, shared):
    g = torch.Generator(device=DEV).manual_seed(S)
    rng = random.Random(S)
    row = ref.random_tree(rng, S, kind)
    rows = [row] * B if shared else [ref.random_tree(rng, S, kind) for _ in range(B)]
    nh = nkv * rep
    wide = torch.randn(B * S, (nh + 2 * nkv) * HD + 6, generator=g, device=DEV).half()
    qkv = wide[:, :-6]
    cos, sin = _tables(n - 2)  # the cache's last positions have no table row
    c = KVCache.wrap([torch.randn(B, nkv, HD, n, generator=g, device=DEV).half()],
                     [torch.randn(B, nkv, n, HD, generator=g, device=DEV).half()])
    ln = torch.tensor(lens, device=DEV)
    want = ref.append(qkv, cos, sin, rows, lens, nh, c.kt[0], c.v[0])
    q = tree_append(qkv, cos, sin, _tree(row if shared else rows), ln, c, 0, nh)
    mag = float(qkv.abs().max()) * 2
    _close(q, want[0], mag)
    _close(c.kt[0], want[1], mag)
    assert torch.equal(c.v[0].double(), want[2])


@pytest.mark.parametrize("B,nkv,rep,S,lens,n,kind,extra", [
    (1, 1, 1, 1, [0], 8, "chain", 0), (1, 8, 4, 5, [1001], 1024, "chain", 8),
    (5, 2, 3, 33, [0, 7, -1, 500, 480], 512, "padded", 0), (40, 1, 1, 1, list(range(40)), 45, "chain", 0),
    (2, 1, 12, 256, [100, 1], 360, "random", 16), (3, 3, 3, 31, [50, 3, 17], 88, "roots", 0)])
def test_append_aligned_rows(B, nkv, rep, S, lens, n, kind, extra):
    """16-byte aligned rows: 32 nodes per workgroup, across sequences."""
    g = torch.Generator(device=DEV).manual_seed(S)
    rng = random.Random(S)
    rows = [ref.random_tree(rng, S, kind) for _ in range(B)]
    nh = nkv * rep
    wide = torch.randn(B * S, (nh + 2 * nkv) * HD + extra, generator=g, device=DEV).half()
    qkv = wide[:, :(nh + 2 * nkv) * HD]
    cos, sin = _tables(n - 2)  # the cache's last positions have no table row
    c = KVCache.wrap([torch.randn(B, nkv, HD, n, generator=g, device=DEV).half()],
                     [torch.randn(B, nkv, n, HD, generator=g, device=DEV).half()])
    want = ref.append(qkv, cos, sin, rows, lens, nh, c.kt[0], c.v[0])
    q = tree_append(qkv, cos, sin, _tree(rows), torch.tensor(lens, device=DEV), c, 0, nh)
    mag = float(qkv.abs().max()) * 2
    _close(q, want[0], mag)
    _close(c.kt[0], want[1], mag)
    assert torch.equal(c.v[0].double(), want[2])


def _attend(B, nkv, rep, S, lens, n, kind, shared=False, bound=None, spoil=True, seed=0, scale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + S)
    rng = random.Random(seed + S)
    row = ref.random_tree(rng, S, kind)
    rows = [row] * B if shared else [ref.random_tree(rng, S, kind) for _ in range(B)]
    q = (torch.randn(B, nkv, rep * S, HD, generator=g, device=DEV) * scale).half()
    kt = torch.randn(B, nkv, HD, n, generator=g, device=DEV).half()
    v = torch.randn(B, nkv, n, HD, generator=g, device=DEV).half()
    if spoil:  # what no node sees
        for b, C in enumerate(lens):
            used = max(C, 0) + (S if C >= 0 else 0)
            kt[b, :, :, used:] = float("nan")
            v[b, :, used:] = float("inf")
            for i in range(S):
                if C >= 0 and not ref.way_up(rows[b], i):
                    kt[b, :, :, C + i] = float("nan")
                    v[b, :, C + i] = float("nan")
    c = KVCache.wrap([kt], [v])
    tree = _tree(row if shared else rows)
    got = tree_attention(q, tree, torch.tensor(lens, device=DEV), c, 0,
                         bound or max(lens) + S)
    return got.view(B, S, nkv * rep, HD), q, c, rows, tree


def _attention_close(got, q, c, rows, lens):
    want, mag, big = ref.attention(q, c.kt[0], c.v[0], rows, lens)
    # scores: 128 fp32 products and sums of terms up to `big` together, scaled (130 roundings),
    # twice (numerator and denominator); exponentials 2^-21; probabilities rounded to 16 bits
    # (2^-11) with nothing below 2^-24 / 2^8 of the largest lost; the output's rounding 2^-11
    d = 2 * 130 * 2.0 ** -24 * big + 2.0 ** -20 + 2.0 ** -11
    n = max(max(lens), 0) + len(rows[0])
    low = n * 2.0 ** -33 * c.v[0].nan_to_num(0, 0, 0).abs().max().double()
    bound = d * mag + 2.0 ** -11 * want.abs() + low + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).nan_to_num(1e9).max())


@pytest.mark.parametrize("B,nkv,rep,S,lens,n,kind", [
    (1, 1, 1, 1, [0], 8, "chain"), (1, 1, 1, 1, [7], 8, "chain"), (2, 2, 4, 1, [0, 300], 304, "chain"),
    (1, 8, 4, 5, [127], 136, "chain"), (1, 1, 1, 2, [126], 128, "chain"), (2, 1, 3, 7, [128, 121], 256, "random"),
    (3, 2, 4, 16, [0, 129, 1000], 1024, "random"), (4, 1, 5, 17, [5, -1, 640, 63], 664, "padded"),
    (2, 2, 1, 64, [1, 200], 264, "star"), (1, 1, 4, 65, [77], 144, "random"),
    (2, 1, 2, 129, [50, 255], 384, "roots"), (1, 1, 12, 9, [511], 520, "random"),
    (1, 1, 1, 256, [3], 264, "padded"), (1, 1, 3, 255, [1025], 1280, "chain"),
    (3, 1, 2, 256, [0, 130, 700], 960, "random"), (2, 1, 4, 33, [4000, 9], 4040, "padded"),
    (1, 1, 16, 8, [3333], 3344, "random"), (1, 2, 4, 3, [20001], 20008, "random"),
    (9, 4, 1, 1, [900, 3, 0, 77, 128, 64, 63, 511, 512], 904, "chain")])
def test_attention(B, nkv, rep, S, lens, n, kind):
    got, q, c, rows, _ = _attend(B, nkv, rep, S, lens, n, kind)
    _attention_close(got, q, c, rows, lens)


def test_attention_shared_tree_and_wide_bound():
    lens = [40, 0, 333, -1]
    a, q, c, rows, tree = _attend(4, 2, 4, 19, lens, 1024, "padded", shared=True)
    _attention_close(a, q, c, rows, lens)
    b = tree_attention(q, tree, torch.tensor(lens, device=DEV), c, 0, 1024)
    _attention_close(b.view_as(a), q, c, rows, lens)


def test_attention_past_the_bound_is_nan():
    lens = [100, 60]
    got, q, c, rows, tree = _attend(2, 1, 2, 9, lens, 128, "padded", bound=100)
    live = (tree.depth[0] >= 0)
    assert bool(got[0, live].isnan().all()) and bool((got[0, ~live] == 0).all())
    c.v[0][0] = 0  # (its own positions hold NaN where no node sees them)
    _attention_close(got[1:], q[1:], KVCache.wrap([c.kt[0][1:]], [c.v[0][1:]]), rows[1:], lens[1:])


@pytest.mark.parametrize("S,C", [(6, 40), (130, 127), (40, 1500)])
def test_attention_hidden_nodes_hold_nan_and_infinities(S, C):
    """A branch whose keys or values overflowed changes no row outside it, and reaches the rows
    that see it."""
    rows = [[-1] + [0] * (S - 1)]
    g = torch.Generator(device=DEV).manual_seed(4)
    n = -(-(C + S) // 8) * 8
    q = torch.randn(1, 1, 2 * S, HD, generator=g, device=DEV).half()
    kt = torch.randn(1, 1, HD, n, generator=g, device=DEV).half()
    v = torch.randn(1, 1, n, HD, generator=g, device=DEV).half()
    clean = KVCache.wrap([kt.clone()], [v.clone()])
    kt[..., 5, C + 2] = float("nan")
    v[:, :, C + 3, 7] = float("inf")
    v[:, :, C + 4, 9] = float("nan")
    v[:, :, C + 5] = -float("inf")
    c = KVCache.wrap([kt], [v])
    ln = torch.tensor([C], device=DEV)
    a = tree_attention(q, _tree(rows), ln, clean, 0, C + S).view(S, 2, HD)
    b = tree_attention(q, _tree(rows), ln, c, 0, C + S).view(S, 2, HD)
    ok = [i for i in range(S) if i not in (2, 3, 4, 5)]
    assert torch.equal(a[ok], b[ok])
    assert bool(b[2].isnan().all())
    keep = [d for d in range(HD) if d != 7]
    assert torch.equal(a[3][:, keep], b[3][:, keep]) and bool(b[3][:, 7].isposinf().all())
    keep = [d for d in range(HD) if d != 9]
    assert torch.equal(a[4][:, keep], b[4][:, keep]) and bool(b[4][:, 9].isnan().all())
    assert bool(b[5].isneginf().all())


def test_attention_scores_far_apart():
    """A first tile whose scores are hundreds below the later ones', and the reverse."""
    for order in (1, -1):
        lens, S, n = [1500], 4, 1504
        g = torch.Generator(device=DEV).manual_seed(6)
        q = torch.ones(1, 1, S, HD, device=DEV).half()
        ramp = torch.linspace(-30 * order, 30 * order, n, device=DEV)
        kt = ramp.expand(1, 1, HD, n).half().contiguous()
        v = torch.randn(1, 1, n, HD, generator=g, device=DEV).half()
        c = KVCache.wrap([kt], [v])
        rows = [[-1, 0, 0, 1]]
        got = tree_attention(q, _tree(rows), torch.tensor(lens, device=DEV), c, 0, n)
        _attention_close(got.view(1, S, 1, HD), q, c, rows, lens)


def _verify_inputs(B, S, V, dtype, soft, kind, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    rows = [ref.random_tree(rng, S, kind) for _ in range(B)]
    base = torch.randn(B, S, V, generator=g, device=DEV) * 2.5
    logits = (base + 0.7 * torch.randn(B, S, V, generator=g, device=DEV)).to(dtype)
    draft = base.to(dtype)
    up = torch.tensor(rows, device=DEV).clamp(0, S - 1).long()
    q = torch.softmax(draft.float() if soft else draft.float() * 4, -1)
    tokens = torch.multinomial(q.view(B * S, V).index_select(
        0, (up + S * torch.arange(B, device=DEV)[:, None]).flatten()), 1,
        generator=g).view(B, S)
    u = torch.rand(B, S, generator=g, device=DEV)
    return rows, logits, draft if soft else None, tokens, u


def _verify_check(got, rows, logits, draft, tokens, u, temps):
    paths, toks, margin = ref.verify(logits, tokens, rows, u, draft, temps)
    # a test nearer to its border than 64-bit sums resolve would say nothing
    assert margin > 1e-9
    S = len(rows[0])
    for b in range(len(rows)):
        assert got.path[b].tolist() == paths[b] + [-1] * (S - len(paths[b])), b
    assert got.count.tolist() == [len(p) for p in paths]
    assert got.token.tolist() == toks


@pytest.mark.parametrize("B,S,V,dtype,soft,kind", [
    (1, 1, 1, "float32", True, "chain"), (3, 2, 2, "float16", True, "chain"),
    (5, 6, 1000, "float16", True, "chain"), (7, 9, 1001, "bfloat16", True, "random"),
    (4, 33, 517, "float32", True, "star"), (6, 17, 4097, "float16", False, "random"),
    (3, 20, 32000, "float16", True, "padded"), (2, 5, 32003, "float32", False, "star"),
    (2, 4, 128001, "bfloat16", True, "chain"), (2, 256, 700, "float32", True, "padded"),
    (3, 40, 8193, "float32", True, "star"), (20, 7, 63, "float16", False, "padded")])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.0])
def test_verify(B, S, V, dtype, soft, kind, temp):
    rows, logits, draft, tokens, u = _verify_inputs(B, S, V, getattr(torch, dtype), soft, kind,
                                                    S + V)
    got = verify_tree(logits, tokens, _tree(rows), u, draft, temp)
    _verify_check(got, rows, logits, draft, tokens, u, [temp] * B)


def test_verify_strides_temperatures_and_odd_values():
    B, S, V = 6, 8, 999
    rows, logits, draft, tokens, u = _verify_inputs(B, S, V, torch.float16, True, "random", 5)
    big = torch.full((B, S + 2, V + 13), float("nan"), dtype=torch.float16, device=DEV)
    big[:, 1:-1, 6:-7] = logits
    lv = big[:, 1:-1, 6:-7]  # rows that start anywhere
    temps = torch.tensor([0.0, 0.3, 1.0, 2.0, 1e-3, 1.0], device=DEV)
    lv[2, 0, 5:] = -float("inf")
    lv[3, :, 17] = float("nan")
    lv[0, 0] = -float("inf")
    lv[5, 0] = float("nan")
    draft[2, 0, 100:] = -float("inf")
    tokens[3, 1], tokens[4, 1] = -5, V
    u[1, 0], u[2, 0] = 0.0, 1.0 - 2.0 ** -24
    got = verify_tree(lv, tokens, _tree(rows), u, draft, temps)
    _verify_check(got, rows, lv, draft, tokens, u, temps.tolist())
    assert got.token[0] == -1 and got.token[5] == -1


def test_verify_same_distributions_and_ties():
    """q = p: everything is accepted; equal largest logits: the lowest index."""
    B, S, V = 4, 5, 300
    lg = torch.randn(B, S, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    tok = torch.softmax(lg.float(), -1).argmax(-1).roll(1, 1)
    tree = DraftTree.chain(S, DEV)
    got = verify_tree(lg, tok, tree, torch.rand(B, S, device=DEV), lg)
    assert got.count.tolist() == [S] * B
    flat = torch.zeros(B, S, 4000, dtype=torch.float16, device=DEV)
    flat[..., 1234], flat[..., 3999], flat[..., 2047] = 3.0, 3.0, 3.0
    got = verify_tree(flat, torch.full((B, S), 2047, device=DEV), tree,
                      torch.zeros(B, S, device=DEV), temperature=0.0)
    assert got.token.tolist() == [1234] * B and got.count.tolist() == [1] * B


def _caches(layers, B, nkv, hd, n, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = KVCache.wrap([torch.randn(B, nkv, hd, n, generator=g, device=DEV).half() for _ in range(layers)],
                     [torch.randn(B, nkv, n, hd, generator=g, device=DEV).half() for _ in range(layers)])
    cpu = KVCache.wrap([t.cpu() for t in c.kt], [t.cpu() for t in c.v])
    return c, cpu


def _same(c, cpu):
    for a, b in zip(c.kt + c.v, cpu.kt + cpu.v):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("layers,B,nkv,hd,n,S", [(1, 1, 1, 128, 8, 1), (3, 5, 2, 128, 301, 33),
                                                  (67, 2, 1, 128, 40, 9), (2, 3, 2, 64, 77, 20),
                                                  (2, 4, 1, 200, 600, 256)])
def test_keep(layers, B, nkv, hd, n, S):
    rng = random.Random(S)
    c, cpu = _caches(layers, B, nkv, hd, n)
    lens = torch.tensor([rng.choice((0, 1, n - S, -1, rng.randint(0, n - S))) for _ in range(B)])
    path = torch.full((B, S + 2), 9, dtype=torch.int32)
    count = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        m = rng.randint(0, S)
        if m:
            way = [0] + sorted(rng.sample(range(1, S), m - 1))
            path[b, :m] = torch.tensor(way, dtype=torch.int32)
        count[b] = m
    if S > 4:  # entries that name no later position are left alone
        path[0, :4], count[0] = torch.tensor([0, 0, n, 4], dtype=torch.int32), 4
    a = c.keep(lens.to(DEV), path.to(DEV)[:, :S], count.to(DEV))
    b = cpu.keep(lens, path[:, :S], count)
    assert a.tolist() == b.tolist()
    _same(c, cpu)


@pytest.mark.parametrize("layers,B,nkv,hd,n,src,dst,length", [
    (1, 2, 1, 128, 8, [0], [1], 1), (3, 5, 2, 128, 304, [0, 0, 3], [1, 4, 2], 203),
    (66, 3, 1, 128, 40, [2, 2], [0, 1], 40), (2, 4, 2, 64, 77, [1], [3], 76),
    (1, 300, 1, 8, 16, [7] * 150, list(range(100, 250)), 9), (1, 3, 1, 128, 2056, [0], [2], 2049),
    (1, 2, 1, 128, 8, [0], [1], 0), (1, 2, 1, 128, 8, [], [], 5)])
def test_fork(layers, B, nkv, hd, n, src, dst, length):
    c, cpu = _caches(layers, B, nkv, hd, n)
    c.fork(src, dst, length)
    cpu.fork(src, dst, length)
    _same(c, cpu)


def test_caches_that_start_anywhere():
    """Views whose addresses are 2-byte aligned only."""
    B, nkv, n = 3, 2, 41
    def view(*shape):
        t = torch.randn(math.prod(shape) + 1, device=DEV).half()
        return t[1:].view(shape)
    c = KVCache.wrap([view(B, nkv, HD, n)], [view(B, nkv, n, HD)])
    cpu = KVCache.wrap([t.cpu() for t in c.kt], [t.cpu() for t in c.v])
    c.fork([0], [2], 30)
    cpu.fork([0], [2], 30)
    _same(c, cpu)
    lens, path = torch.tensor([3, 30, 9]), torch.tensor([[0, 2, 3, 7, 9]] * 3, dtype=torch.int32)
    count = torch.tensor([5, 3, 4], dtype=torch.int32)
    c.keep(lens.to(DEV), path.to(DEV), count.to(DEV))
    cpu.keep(lens, path, count)
    _same(c, cpu)


def _step(c, qkv, cos, sin, tree, lens, logits, tokens, u, nh, bound):
    q = tree_append(qkv, cos, sin, tree, lens, c, 0, nh)
    o = tree_attention(q, tree, lens, c, 0, bound)
    r = verify_tree(logits, tokens, tree, u, None, 0.8)
    return o, r, c.keep(lens, r.path, r.count)


def test_a_step_together_on_a_stream_and_replayed():
    """append, attention, verification and compaction of one step: eager on another stream, and
    captured once and replayed with other inputs, the eager result each time."""
    B, nkv, rep, S, n, V = 3, 2, 4, 11, 512, 777
    nh = nkv * rep
    rng = random.Random(3)
    tree = _tree([ref.random_tree(rng, S, "padded") for _ in range(B)])
    cos, sin = _tables(n)
    g = torch.Generator(device=DEV).manual_seed(0)

    def inputs():
        lg = torch.randn(B, S, V, generator=g, device=DEV) * 4
        return [torch.randn(B * S, (nh + 2 * nkv) * HD, generator=g, device=DEV).half(), lg,
                lg.argmax(-1).roll(1, 1), torch.rand(B, S, generator=g, device=DEV),
                torch.randint(0, 400, (B,), generator=g, device=DEV)]

    c, _ = _caches(1, B, nkv, HD, n)
    start = c.kt[0].clone(), c.v[0].clone()

    def eager(x):
        e = KVCache.wrap([start[0].clone()], [start[1].clone()])
        o, r, l = _step(e, x[0], cos, sin, tree, x[4], x[1], x[2], x[3], nh, n)
        return [o, *r, l, e.kt[0], e.v[0]]

    st = inputs()
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eager(st)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, eager(st)):
        assert torch.equal(a, b)
    with torch.cuda.stream(side):
        _step(c, st[0], cos, sin, tree, st[4], st[1], st[2], st[3], nh, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, r, l = _step(c, st[0], cos, sin, tree, st[4], st[1], st[2], st[3], nh, n)
    for _ in range(4):
        x = inputs()
        for a, b in zip(st, x):
            a.copy_(b)
        c.kt[0].copy_(start[0]), c.v[0].copy_(start[1])
        want = eager(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([o, *r, l, c.kt[0], c.v[0]], want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("B,nkv,rep,S,most,kind", [
    (150, 2, 4, 3, 700, "padded"), (70, 1, 1, 1, 2500, "chain"), (67, 1, 2, 40, 300, "random"),
    (130, 8, 4, 1, 200, "chain")])
def test_attention_many_sequences(B, nkv, rep, S, most, kind):
    """More sequences than a wave has lanes, of any lengths, some without a part."""
    rng = random.Random(B)
    lens = [rng.choice((0, -1, most, rng.randint(0, most), rng.randint(0, 130))) for _ in range(B)]
    lens[64:66] = [-1, -1]
    n = -(-(most + S) // 8) * 8
    got, q, c, rows, _ = _attend(B, nkv, rep, S, lens, n, kind)
    _attention_close(got, q, c, rows, lens)


@pytest.mark.parametrize("B,nkv,rep,S,lens", [(1, 1, 4, 256, [900]), (2, 2, 4, 200, [0, 1111]),
                                              (1, 1, 16, 100, [5000])])
def test_attention_many_row_blocks(B, nkv, rep, S, lens):
    got, q, c, rows, _ = _attend(B, nkv, rep, S, lens, -(-(max(lens) + S) // 8) * 8, "random")
    _attention_close(got, q, c, rows, lens)


def test_lengths_past_everything():
    """A length near the largest int64 counts as past the cache; the others are as ever."""
    top = 2 ** 63 - 1
    S, n, nh, nkv = 9, 128, 8, 2
    rng = random.Random(0)
    rows = [ref.random_tree(rng, S, "random") for _ in range(4)]
    tree = _tree(rows)
    lens = torch.tensor([top, 40, top - 4, 2 ** 32 + 5], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    cos, sin = _tables(n)
    for width in (0, 6):  # rows of both kinds
        qkv = torch.randn(4 * S, (nh + 2 * nkv) * HD + width, generator=g, device=DEV).half()
        qkv = qkv[:, :(nh + 2 * nkv) * HD]
        c, _ = _caches(1, 4, nkv, HD, n)
        before = c.kt[0].clone(), c.v[0].clone()
        q = tree_append(qkv, cos, sin, tree, lens, c, 0, nh)
        o = tree_attention(q, tree, lens, c, 0, n).view(4, S, nh, HD)
        for b in (0, 2, 3):
            assert bool(q[b].isnan().all()) and bool(o[b].isnan().all())
            assert torch.equal(c.kt[0][b], before[0][b]) and torch.equal(c.v[0][b], before[1][b])
        assert not bool(q[1].isnan().any()) and not bool(o[1].isnan().any())
    path = torch.arange(S, dtype=torch.int32, device=DEV).repeat(4, 1)
    path[:, 1] = 3
    before = c.kt[0].clone(), c.v[0].clone()
    c.keep(lens, path, torch.full((4,), 2, dtype=torch.int32, device=DEV))
    for b in (0, 2, 3):
        assert torch.equal(c.kt[0][b], before[0][b]) and torch.equal(c.v[0][b], before[1][b])
    assert torch.equal(c.v[0][1, :, 41], before[1][1, :, 43])


@pytest.mark.parametrize("B,S,V,soft,kind", [(2, 4, 600001, True, "star"), (1, 3, 1100000, False, "star"),
                                             (1, 9, 530000, True, "star")])
@pytest.mark.parametrize("temp", [0.0, 0.9])
def test_verify_vocabularies_of_several_blocks_per_chunk(B, S, V, soft, kind, temp):
    rows, logits, draft, tokens, u = _verify_inputs(B, S, V, torch.float16, soft, kind, V)
    u[:, 1:] = 1.0 - u[:, 1:] / 64  # rejections
    got = verify_tree(logits, tokens, _tree(rows), u, draft, temp)
    _verify_check(got, rows, logits, draft, tokens, u, [temp] * B)


@pytest.mark.parametrize("V", [90, 7000, 20001, 100003])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("near", [0.02, 1.5])
def test_verify_many_rejections_of_one_node(V, dtype, near):
    """Up to 30 children of one node, few accepted: residuals of many tokens (a drafter near the
    target) and of few, whose tokens fit on the chip or do not."""
    B, S = 6, 31
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.randn(B, S, V, generator=g, device=DEV)
    draft = (logits + near * torch.randn(B, S, V, generator=g, device=DEV)).to(dtype)
    logits = logits.to(dtype)
    q = torch.softmax(draft[:, 0].float(), -1)
    tokens = torch.cat((torch.zeros(B, 1, dtype=torch.int64, device=DEV),
                        torch.multinomial(q, S - 1, replacement=True, generator=g)), 1)
    u = torch.rand(B, S, generator=g, device=DEV)
    u[:, 1:] = 1.0 - u[:, 1:] / 1024
    rows = [[-1] + [0] * (S - 1)] * B
    got = verify_tree(logits, tokens, _tree(rows), u, draft, 1.0)
    _verify_check(got, rows, logits, draft, tokens, u, [1.0] * B)


def test_two_streams_at_once():
    """Attention and verification of different inputs on two streams, interleaved: each what it
    is alone."""
    jobs = []
    for seed, (B, S, C) in enumerate(((3, 40, 3000), (2, 7, 6000))):
        lens = [C - 100 * b for b in range(B)]
        got, q, c, rows, tree = _attend(B, 2, 4, S, lens, -(-(C + S) // 8) * 8, "random", seed=seed)
        vin = _verify_inputs(B, S, 33000, torch.float16, True, "star", seed)
        jobs.append((q, tree, torch.tensor(lens, device=DEV), c, C + S, vin, _tree(vin[0])))

    def run(j):
        q, tree, ln, c, bound, (_, lg, d, t, u), vt = j
        return [tree_attention(q, tree, ln, c, 0, bound), *verify_tree(lg, t, vt, u, d, 0.8)]

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=DEV) for _ in jobs]
    out = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, j in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                out[i].append(run(j))
    torch.cuda.synchronize()
    for i in range(2):
        for o in out[i]:
            for a, b in zip(o, want[i]):
                assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    c = KVCache.wrap([torch.zeros(2, 1, HD, 16, device=DEV).half()],
                     [torch.zeros(2, 1, 16, HD, device=DEV).half()])
    odd = KVCache.wrap([torch.zeros(2, 1, HD, 17, device=DEV).half()],
                       [torch.zeros(2, 1, 17, HD, device=DEV).half()])
    small = KVCache.wrap([torch.zeros(2, 1, 64, 16, device=DEV).half()],
                         [torch.zeros(2, 1, 16, 64, device=DEV).half()])
    full = KVCache.wrap([torch.zeros(2, 1, HD, 16, device=DEV)],
                        [torch.zeros(2, 1, 16, HD, device=DEV)])
    t, lens = _tree([-1, 0]), torch.zeros(2, dtype=torch.int64, device=DEV)
    q = torch.zeros(2, 1, 2, HD, device=DEV).half()
    for bad in (lambda: tree_attention(q, t, lens, odd, 0, 16),
                lambda: tree_attention(q[..., :64], t, lens, small, 0, 16),
                lambda: tree_attention(q, t, lens, full, 0, 16),
                lambda: tree_attention(q.float(), t, lens, c, 0, 16),
                lambda: tree_attention(q, t, lens.cpu(), c, 0, 16),
                lambda: tree_attention(q, DraftTree.chain(2), lens, c, 0, 16),
                lambda: full.keep(lens, torch.zeros(2, 2, dtype=torch.int32, device=DEV),
                                  torch.ones(2, dtype=torch.int32, device=DEV)),
                lambda: full.fork([0], [1], 4)):
        with pytest.raises(AssertionError):
            bad()
