"""CPU checks of the tree-speculation operators (hydranet_amd/model/speculative.py,
KVCache.keep / fork): the torch forms against node-by-node 64-bit ones, what is
refused, and that verification keeps the target's distribution."""
import random

import pytest
import torch

from hydranet_amd.model.decoder import KVCache
from hydranet_amd.model.speculative import (PADDING, DraftTree, tree_append, tree_attention,
                                            verify_tree)
from tests import _tree_ref as ref


def _tree(rows):
    return DraftTree(torch.tensor(rows, dtype=torch.int32))


@pytest.mark.parametrize("S,kind", [(1, "chain"), (2, "chain"), (70, "chain"), (9, "star"),
                                    (33, "random"), (40, "padded"), (65, "roots"),
                                    (256, "random"), (256, "chain")])
def test_plan(S, kind):
    rng = random.Random(S)
    rows = [ref.random_tree(rng, S, kind) for _ in range(3)]
    t = _tree(rows)
    see = t.visible()
    for b, row in enumerate(rows):
        for i in range(S):
            way = ref.way_up(row, i)
            assert t.depth[b, i] == len(way) - 1
            assert t.up[b, i] == (row[i] if way else PADDING)
            assert see[b, i].nonzero().flatten().tolist() == way


def _cache(B, nkv, hd, n, dtype=torch.float64):
    return KVCache.wrap([torch.randn(B, nkv, hd, n, dtype=dtype)],
                        [torch.randn(B, nkv, n, hd, dtype=dtype)])


@pytest.mark.parametrize("kind", ["chain", "random", "padded", "roots"])
@pytest.mark.parametrize("shared", [False, True])
def test_append_and_attention(kind, shared):
    torch.manual_seed(3)
    rng = random.Random(5)
    B, nkv, rep, S, hd, n = 4, 2, 3, 7, 16, 40
    rows = [ref.random_tree(rng, S, kind)] * B if shared else \
        [ref.random_tree(rng, S, kind) for _ in range(B)]
    tree = _tree(rows[0] if shared else rows)
    lens = torch.tensor([0, 20, -1, n - S])
    c = _cache(B, nkv, hd, n)
    a = torch.outer(torch.arange(n).float(), 0.3 ** torch.arange(hd // 2).float()).repeat(1, 2)
    cos, sin = a.cos(), a.sin()
    qkv = torch.randn(B * S, (nkv * rep + 2 * nkv) * hd, dtype=torch.float64)
    want = ref.append(qkv, cos, sin, rows, lens, nkv * rep, c.kt[0], c.v[0])
    q = tree_append(qkv, cos, sin, tree, lens, c, 0, nkv * rep)
    for got, w in zip((q, c.kt[0], c.v[0]), want):
        torch.testing.assert_close(got, w, rtol=1e-12, atol=1e-12)
    c.v[0][1, :, 20 + S:] = float("nan")  # positions nobody sees
    c.kt[0][1, :, :, 20 + S:] = float("nan")
    o = tree_attention(q, tree, lens, c, 0, n)
    w, _, _ = ref.attention(q, c.kt[0], c.v[0], rows, lens)
    torch.testing.assert_close(o.view(B, S, nkv * rep, hd), w, rtol=1e-10, atol=1e-12)
    short = tree_attention(q, tree, lens, c, 0, 20 + S)
    assert torch.equal(short[:3], o[:3])
    live = tree.depth.expand(B, S)[3] >= 0
    assert short[3, live].isnan().all() and bool((short[3, ~live] == 0).all())


@pytest.mark.parametrize("kind", ["chain", "random", "padded", "star"])
@pytest.mark.parametrize("soft", [True, False])
def test_verify_against_the_definition(kind, soft):
    rng = random.Random(11)
    g = torch.Generator().manual_seed(2)
    B, S, V = 40, 9, 23
    rows = [ref.random_tree(rng, S, kind) for _ in range(B)]
    logits = torch.randn(B, S, V, generator=g) * 2
    draft = logits + torch.randn(B, S, V, generator=g) if soft else None
    logits[3, :, 5:9] = -float("inf")
    logits[4, 0] = float("nan")
    tokens = torch.randint(0, V, (B, S), generator=g)
    up = torch.tensor(rows).clamp(0, S - 1)
    likely = logits.nan_to_num(0).gather(1, up[..., None].expand(B, S, V)).argmax(-1)
    tokens = torch.where(torch.rand(B, S, generator=g) < 0.6, likely, tokens)
    tokens[5, 1], tokens[6, 2] = -1, V
    u = torch.rand(B, S, generator=g)
    temps = torch.rand(B, generator=g)
    temps[::4] = 0
    got = verify_tree(logits, tokens, _tree(rows), u, draft, temps)
    paths, toks, _ = ref.verify(logits, tokens, rows, u, draft, temps)
    for b in range(B):
        assert got.path[b].tolist() == paths[b] + [-1] * (S - len(paths[b]))
        assert got.count[b] == len(paths[b])
    assert got.token.tolist() == toks
    assert int((got.count > 1).sum()) > 4


@pytest.mark.parametrize("soft", [True, False])
def test_verify_keeps_the_targets_distribution(soft):
    """One root with three children drawn from q (or certain): the first token after the root
    (the accepted child's, else the drawn one) is distributed as p.  N draws; a frequency's
    deviation sqrt(p (1 - p) / N) is at most 0.5 / sqrt(N); 5 deviations of it."""
    g = torch.Generator().manual_seed(8)
    N, V = 20000, 4
    p = torch.tensor([0.5, 0.3, 0.15, 0.05]).log()
    q = torch.tensor([0.1, 0.2, 0.3, 0.4]).log()
    logits = p.expand(N, 4, V).contiguous()
    draft = q.expand(N, 4, V).contiguous()
    tokens = torch.multinomial(q.exp().expand(N, V), 4, replacement=True, generator=g)
    if not soft:
        tokens[:] = torch.tensor([0, 3, 1, 3])
    got = verify_tree(logits, tokens, _tree([-1, 0, 0, 0]), torch.rand(N, 4, generator=g),
                      draft if soft else None)
    first = torch.where(got.count > 1, tokens.gather(1, got.path[:, 1:2].clamp(min=0).long())[:, 0],
                        got.token)
    freq = torch.bincount(first, minlength=V).double() / N
    assert (freq - p.double().exp()).abs().max() < 5 * 0.5 / N ** 0.5


def test_keep_and_fork():
    torch.manual_seed(1)
    B, n, S = 4, 30, 6
    c = KVCache.wrap([torch.randn(B, 2, 4, n) for _ in range(3)],
                     [torch.randn(B, 2, n, 4) for _ in range(3)])
    old = [t.clone() for t in c.kt], [t.clone() for t in c.v]
    lens = torch.tensor([5, 0, -1, n - S])
    path = torch.tensor([[0, 2, 5, -1, -1, -1], [0, 1, 2, 3, 4, 5], [0, 3, 4, -1, -1, -1],
                         [0, 0, 4, 5, -1, -1]], dtype=torch.int32)
    count = torch.tensor([3, 9, 2, 4], dtype=torch.int32)
    got = c.keep(lens, path, count)
    assert got.tolist() == [8, 6, -1, n - S + 4]
    for l in range(3):
        k, v = old[0][l].clone(), old[1][l].clone()
        for b, moves in ((0, [(1, 2), (2, 5)]), (3, [(2, 4), (3, 5)])):
            for j, i in moves:
                k[b, :, :, lens[b] + j] = old[0][l][b, :, :, lens[b] + i]
                v[b, :, lens[b] + j] = old[1][l][b, :, lens[b] + i]
        assert torch.equal(c.kt[l], k) and torch.equal(c.v[l], v)
    old = [t.clone() for t in c.kt], [t.clone() for t in c.v]
    c.fork([0, 0], [1, 2], 7)
    for l in range(3):
        assert torch.equal(c.kt[l][1, :, :, :7], old[0][l][0, :, :, :7])
        assert torch.equal(c.v[l][2, :, :7], old[1][l][0, :, :7])
        assert torch.equal(c.kt[l][1:, :, :, 7:], old[0][l][1:, :, :, 7:])
        assert torch.equal(c.v[l][3], old[1][l][3]) and torch.equal(c.v[l][0], old[1][l][0])


def test_refusals():
    c = _cache(2, 2, 8, 16)
    t = _tree([-1, 0, 1])
    lens = torch.zeros(2, dtype=torch.int64)
    qkv, tab = torch.zeros(6, 8 * 8, dtype=torch.float64), torch.zeros(16, 8)
    q = torch.zeros(2, 2, 6, 8, dtype=torch.float64)
    lg, tok, u = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    one = torch.ones(2, dtype=torch.int32)
    path = torch.zeros(2, 3, dtype=torch.int32)
    for bad in (
            lambda: DraftTree(torch.zeros(3)),
            lambda: DraftTree(torch.zeros(257, dtype=torch.int32)),
            lambda: DraftTree(torch.zeros(0, dtype=torch.int32)),
            lambda: tree_append(qkv, tab, tab, t, lens.int(), c, 0, 4),
            lambda: tree_append(qkv, tab, tab, t, lens[:1], c, 0, 4),
            lambda: tree_append(qkv, tab, tab, t, lens, c, 0, 5),
            lambda: tree_append(qkv[:5], tab, tab, t, lens, c, 0, 4),
            lambda: tree_append(qkv, tab.half(), tab, t, lens, c, 0, 4),
            lambda: tree_append(qkv, tab, tab, _tree([[-1, 0, 1]] * 3), lens, c, 0, 4),
            lambda: tree_attention(q[:, :1], t, lens, c, 0, 16),
            lambda: tree_attention(q[:, :, :5], t, lens, c, 0, 16),
            lambda: tree_attention(q, t, lens, c, 0, 2),
            lambda: tree_attention(q, t, lens, c, 0, 17),
            lambda: verify_tree(lg.double(), tok, t, u),
            lambda: verify_tree(lg[:, :2], tok, t, u),
            lambda: verify_tree(lg, tok.int(), t, u),
            lambda: verify_tree(lg, tok, t, u[:, :2]),
            lambda: verify_tree(lg, tok, t, u, lg.half()),
            lambda: verify_tree(lg, tok, t, u, temperature=-1.0),
            lambda: verify_tree(lg, tok, t, u, temperature=torch.ones(3)),
            lambda: c.keep(lens, path.long(), one),
            lambda: c.keep(lens, path[:1], one),
            lambda: c.keep(lens, path, one[:1]),
            lambda: c.fork([0], [0], 4), lambda: c.fork([0, 0], [1, 1], 4),
            lambda: c.fork([0], [2], 4), lambda: c.fork([0], [1], 17),
            lambda: c.fork([0, 1], [1], 4)):
        with pytest.raises(AssertionError):
            bad()


def test_library_refusals_without_gpu():
    """Rejected arguments return before any HIP call."""
    import ctypes
    from hydranet_amd import _lib
    P = ctypes.c_void_p(16)
    two = (ctypes.c_void_p * 2)(16, 16)
    i0, i1 = (ctypes.c_int * 2)(0, 0), (ctypes.c_int * 2)(1, 1)
    for name, args in [
            ("hn_tree_plan", (P, 257, 1, 257, P, P, P, None)),
            ("hn_tree_plan", (P, 2, 1, 3, P, P, P, None)),
            ("hn_tree_plan", (None, 3, 1, 3, P, P, P, None)),
            ("hn_tree_append", (P, 1024, P, P, 8, P, 1, P, 1, 1, 2, 4, 64, P, P, P, 8, None)),
            ("hn_tree_append", (P, 1024, P, P, 8, P, 1, P, 1, 1, 2, 4, 128, P, P, P, 8, None)),
            ("hn_tree_append", (P, 1536, P, P, 8, P, 2, P, 3, 1, 2, 4, 128, P, P, P, 8, None)),
            ("hn_tree_append", (P, 1536, P, P, 8, P, 1, None, 3, 1, 2, 4, 128, P, P, P, 8, None)),
            ("hn_tree_attention", (P, P, P, 12, P, P, 1, 1, 1, 1, 128, 1, 9, 1.0, P, 128, P, 1 << 30, None)),
            ("hn_tree_attention", (P, P, P, 16, P, P, 1, 1, 1, 1, 128, 1, 17, 1.0, P, 128, P, 1 << 30, None)),
            ("hn_tree_attention", (P, P, P, 16, P, P, 1, 1, 1, 1, 128, 4, 3, 1.0, P, 128, P, 1 << 30, None)),
            ("hn_tree_attention", (P, P, P, 16, P, P, 1, 1, 2, 1, 128, 1, 9, 1.0, P, 128, P, 1 << 30, None)),
            ("hn_tree_attention", (P, P, ctypes.c_void_p(8), 16, P, P, 1, 1, 1, 1, 128, 1, 9, 1.0, P, 128, P, 1 << 30, None)),
            ("hn_verify_tree", (P, 9, 3, None, 0, 0, 3, P, P, 1, P, None, 1.0, 1, 3, 3, P, P, P, P, 1 << 30, None)),
            ("hn_verify_tree", (P, 9, 2, None, 0, 0, 0, P, P, 1, P, None, 1.0, 1, 3, 3, P, P, P, P, 1 << 30, None)),
            ("hn_verify_tree", (P, 9, 3, P, 9, 2, 0, P, P, 1, P, None, 1.0, 1, 3, 3, P, P, P, P, 1 << 30, None)),
            ("hn_verify_tree", (P, 9, 3, None, 0, 0, 0, P, P, 1, P, None, -1.0, 1, 3, 3, P, P, P, P, 1 << 30, None)),
            ("hn_verify_tree", (P, 9, 3, None, 0, 0, 0, P, P, 1, None, None, 1.0, 1, 3, 3, P, P, P, P, 1 << 30, None)),
            ("hn_kv_keep", (two, two, 2, 8, 1, 1, 4, P, P, 2, P, 3, None, None)),
            ("hn_kv_keep", (two, two, 2, 8, 1, 1, 4, P, P, 3, P, 3, P, None)),
            ("hn_kv_keep", ((ctypes.c_void_p * 2)(16, None), two, 2, 8, 1, 1, 4, P, P, 3, P, 3, None, None)),
            ("hn_kv_fork", (two, two, 2, 8, 4, 1, 4, i0, i0, 1, 4, None)),
            ("hn_kv_fork", (two, two, 2, 8, 4, 1, 4, i0, i1, 2, 4, None)),
            ("hn_kv_fork", (two, two, 2, 8, 1, 1, 4, i0, i1, 1, 4, None)),
            ("hn_kv_fork", (two, two, 2, 8, 4, 1, 4, i0, i1, 1, 9, None))]:
        with pytest.raises(RuntimeError, match=name):
            _lib.call(name, *args)


def test_attention_module_chain_equals_one_token_steps():
    """Attention.forward_tree over a chain equals its one-token steps, float64."""
    from hydranet_amd.model.decoder import Attention, MixtralDecoderConfig, RotaryEmbedding
    torch.manual_seed(0)
    cfg = MixtralDecoderConfig(num_layers=1, hidden_dim=64, num_attention_heads=4,
                               num_kv_heads=2, head_dim=16, max_position_embeddings=32)
    att = Attention(cfg).double()
    rope = RotaryEmbedding(16, 32, 1e6)
    B, S = 2, 6
    x = torch.randn(B, S, 64, dtype=torch.float64)
    one, tree = _cache(B, 2, 16, 24), _cache(B, 2, 16, 24)
    want = [att(x[:, t:t + 1], rope, torch.tensor([t]), one, 0, t + 1) for t in range(S)]
    got = att.forward_tree(x, rope, DraftTree.chain(S), torch.zeros(B, dtype=torch.int64), tree, 0, S)
    # the one-token steps' softmax is fp32
    torch.testing.assert_close(got, torch.cat(want, 1), rtol=1e-5, atol=1e-6)


def test_ngram_draft():
    from hydranet_amd.model.speculative import ngram_draft
    d = ngram_draft([[1, 2, 3, 1, 2], [4]], "cpu", nodes=4)
    assert d.tokens.tolist() == [[3, 1, 2], [0, 0, 0]]
    assert d.parents.tolist() == [[-1, 0, 1, 2], [-1, PADDING, PADDING, PADDING]]


class _Counting:
    """A model whose next token is the last plus one; its cache holds the tokens."""

    def __init__(self, vocab):
        self.vocab, self.passes = vocab, 0

    def new_cache(self, batch, max_len):
        z = torch.zeros(batch, 1, 2, max_len, dtype=torch.float16)
        return KVCache.wrap([z], [z.transpose(2, 3).contiguous()])

    def _logits(self, ids):
        assert int(ids.min()) >= 0 and int(ids.max()) < self.vocab
        return 9.0 * torch.nn.functional.one_hot((ids + 1) % self.vocab, self.vocab).float()

    def forward(self, ids, cache):
        cache.kt[0][:, 0, :, :ids.shape[1]] = ids[:, None].half()
        return self._logits(ids)

    def forward_tree(self, tokens, tree, lens, cache, bound):
        self.passes += 1
        for b in range(tokens.shape[0]):
            C = int(lens[b])
            if C >= 0:
                assert C + tokens.shape[1] <= bound <= cache.max_len
                # what was kept is the text so far: consecutive numbers
                text = cache.kt[0][b, 0, 0, :C].long()
                assert torch.equal(text, (text[0] + torch.arange(C)) % self.vocab)
                assert int(tokens[b, 0]) == (int(text[-1]) + 1) % self.vocab
                cache.kt[0][b, 0, :, C:C + tokens.shape[1]] = tokens[b].half()
        return self._logits(tokens)


def test_generate_with_right_wrong_and_impossible_drafts():
    from hydranet_amd.model.speculative import Draft, generate
    V, n = 50, 23

    def draft(history, device):
        rows = []
        for i, h in enumerate(history):
            t = h[-1]
            right = [(t + 1) % V, (t + 2) % V, (t + 3) % V]
            rows.append([-7, V + 3] + (right if i % 2 == 0 else [right[0], V, -1]))
        return Draft(torch.tensor(rows), torch.tensor([-1, 0, 0, 0, 3, 4], dtype=torch.int32))

    prompt = torch.tensor([[3, 4, 5], [48, 49, 0]])
    for samples in (1, 2):
        model = _Counting(V)
        out = generate(model, prompt, n, draft, samples=samples, max_nodes=6)
        for i in range(2 * samples):
            want = (prompt[i % 2, -1] + 1 + torch.arange(n)) % V
            assert torch.equal(out[i], want)
        assert model.passes == 11  # two tokens a pass at the least, after the first
    assert torch.equal(generate(_Counting(V), prompt, n), out[:2])


def test_a_cache_is_copied_after_its_layers_were_passed_to_a_kernel():
    import copy
    c = KVCache.wrap([torch.zeros(1, 1, 4, 8).half()], [torch.zeros(1, 1, 8, 4).half()])
    a = c._layers()
    d = copy.deepcopy(c)
    b = d._layers()
    assert a[0][0] == c.kt[0].data_ptr() and b[0][0] == d.kt[0].data_ptr() != a[0][0]
    c.v[0] = torch.ones(1, 1, 8, 4).half()
    assert c._layers()[1][0] == c.v[0].data_ptr()


def _random_attention(rows, C, n, nkv=2, rep=2, hd=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    B, S = len(rows), len(rows[0])
    c = KVCache.wrap([torch.randn(B, nkv, hd, n, generator=g, dtype=torch.float64)],
                     [torch.randn(B, nkv, n, hd, generator=g, dtype=torch.float64)])
    q = torch.randn(B, nkv, rep * S, hd, generator=g, dtype=torch.float64)
    return q, c, torch.full((B,), C, dtype=torch.int64)


def test_attention_hidden_nodes_hold_nan_and_infinities():
    """A branch whose keys or values overflowed changes no row outside it, and reaches the rows
    that see it."""
    S, C, hd = 8, 5, 8
    rows = [[-1, 0, 0, 0, 0, 0, 3, -2]]
    q, clean, lens = _random_attention(rows, C, 16)
    c = KVCache.wrap([clean.kt[0].clone()], [clean.v[0].clone()])
    c.kt[0][:, :, 5, C + 2] = float("nan")
    c.v[0][:, :, C + 3, 7] = float("inf")
    c.v[0][:, 1, C + 4, 6] = float("nan")
    c.v[0][:, :, C + 5] = -float("inf")
    c.v[0][:, :, C + 7] = float("nan")  # padding's
    a = tree_attention(q, _tree(rows), lens, clean, 0, 16).view(S, 2, 2, hd)
    b = tree_attention(q, _tree(rows), lens, c, 0, 16).view(S, 2, 2, hd)
    # sums of 13 terms below 4, perhaps in another order: 16 roundings of 2^-53 times 4, twice
    close = dict(rtol=0, atol=2.0 ** -45)
    torch.testing.assert_close(a[[0, 1]], b[[0, 1]], **close)
    assert bool(b[2].isnan().all())
    for i in (3, 6):  # the node and its child
        torch.testing.assert_close(a[i, ..., :7], b[i, ..., :7], **close)
        assert bool(b[i, ..., 7].isposinf().all())
    torch.testing.assert_close(a[4, 0], b[4, 0], **close)
    torch.testing.assert_close(a[4, 1, :, [0, 1, 2, 3, 4, 5, 7]],
                               b[4, 1, :, [0, 1, 2, 3, 4, 5, 7]], **close)
    assert bool(b[4, 1, :, 6].isnan().all()) and bool(b[5].isneginf().all())
    assert bool((b[7] == 0).all())


def test_attention_nan_that_a_row_sees():
    """A cached key, a query: the rows that hold them are NaN; padding and inactive sequences stay
    zero whatever the cache holds."""
    rows = [[-1, 0, -2], [-1, 0, 1], [-1, 0, 1]]
    q, c, lens = _random_attention(rows, 6, 12)
    lens[2] = -1
    c.kt[0][0, 0, 3, 2] = float("nan")
    c.v[0][0, 1, 4] = float("inf")
    c.v[0][2] = float("nan")
    q.view(3, 2, 2, 3, 8)[1, 1, 0, 2, 5] = float("nan")
    o = tree_attention(q, _tree(rows), lens, c, 0, 12).view(3, 3, 2, 2, 8)
    assert bool(o[0, :2, 0].isnan().all()) and bool(o[0, :2, 1].isposinf().all())
    assert bool((o[0, 2] == 0).all()) and bool((o[2] == 0).all())
    bad = o[1].isnan()
    assert bool(bad[2, 1, 0].all()) and int(bad.sum()) == 8


def test_attention_of_a_node_past_the_table_is_nan():
    B, nkv, rep, hd, n, S = 1, 1, 2, 8, 16, 3
    c = KVCache.wrap([torch.randn(B, nkv, hd, n)], [torch.randn(B, nkv, n, hd)])
    tab, tree, lens = torch.rand(10, hd), DraftTree.chain(S), torch.tensor([8])
    q = tree_append(torch.randn(S, 4 * hd), tab, tab, tree, lens, c, 0, rep)
    o = tree_attention(q, tree, lens, c, 0, n)
    assert bool(o[0, 2].isnan().all()) and not bool(o[0, :2].isnan().any())


def test_attention_with_a_head_of_infinite_scores():
    """Every visible score at -inf, or one at +inf: no probabilities."""
    rows = [[-1, 0]]
    q, c, lens = _random_attention(rows, 3, 8, rep=1)
    q.fill_(1.0)
    c.kt[0][:, 0] = -float("inf")
    c.kt[0][:, 1, 0, 1] = float("inf")
    assert bool(tree_attention(q, _tree(rows), lens, c, 0, 8).isnan().all())


def test_lengths_past_everything():
    """A length near the largest int64 counts as past the cache; the others are as ever."""
    top, S, n, hd = 2 ** 63 - 1, 4, 16, 8
    lens = torch.tensor([top, 5, top - 2, 2 ** 32 + 5])
    tree, tab = DraftTree.chain(S), torch.rand(n, hd)
    c = _cache(4, 1, hd, n)
    kt, v = c.kt[0].clone(), c.v[0].clone()
    q = tree_append(torch.randn(4 * S, 4 * hd, dtype=torch.float64), tab, tab, tree, lens, c, 0, 2)
    o = tree_attention(q, tree, lens, c, 0, n)
    for b in (0, 2, 3):
        assert bool(q[b].isnan().all()) and bool(o[b].isnan().all())
        assert torch.equal(c.kt[0][b], kt[b]) and torch.equal(c.v[0][b], v[b])
    assert not bool(q[1].isnan().any()) and not bool(o[1].isnan().any())
    kt, v = c.kt[0].clone(), c.v[0].clone()
    path = torch.tensor([[0, 2, 3, -1]] * 4, dtype=torch.int32)
    c.keep(lens, path, torch.full((4,), 3, dtype=torch.int32))
    for b in (0, 2, 3):
        assert torch.equal(c.kt[0][b], kt[b]) and torch.equal(c.v[0][b], v[b])
    assert torch.equal(c.v[0][1, :, 6], v[1, :, 7]) and torch.equal(c.kt[0][1, ..., 7], kt[1, ..., 8])


@pytest.mark.parametrize("scale", [0.0, -0.0, -1.0, float("inf"), -float("inf"), float("nan"), 3e38])
def test_library_refuses_scales_without_gpu(scale):
    """Scores are masked before they are scaled: a scale that is not above zero, or not finite
    (also as a power of two), is refused before any HIP call."""
    import ctypes
    from hydranet_amd import _lib
    P = ctypes.c_void_p(16)
    with pytest.raises(RuntimeError, match="hn_tree_attention: scale"):
        _lib.call("hn_tree_attention", P, P, P, 16, P, P, 1, 1, 1, 1, 128, 1, 9, scale, P, 128, P,
                  1 << 30, None)


@pytest.mark.parametrize("which", [0, 1, 2, 4, 5, 14])
def test_library_refuses_null_operands_without_gpu(which):
    import ctypes
    from hydranet_amd import _lib
    P = ctypes.c_void_p(16)
    args = [P, P, P, 16, P, P, 1, 1, 1, 1, 128, 1, 9, 1.0, P, 128, P, 1 << 30, None]
    args[which] = None
    with pytest.raises(RuntimeError, match="hn_tree_attention: null operand"):
        _lib.call("hn_tree_attention", *args)


class _Short(_Counting):
    """No position from `rows` on: the nodes there have no logits."""

    def __init__(self, vocab, rows):
        super().__init__(vocab)
        self.rows = rows

    def forward_tree(self, tokens, tree, lens, cache, bound):
        logits = super().forward_tree(tokens, tree, lens, cache, bound)
        past = lens[:, None] + tree.depth >= self.rows
        return torch.where(past[..., None], float("nan"), logits)


@pytest.mark.parametrize("wide", [1, 2, 3, 5, 9])
@pytest.mark.parametrize("over", [0, 1])
def test_generate_up_to_the_models_last_position(wide, over):
    """A draft may reach past the last position; what is asked for does not."""
    from hydranet_amd.model.speculative import Draft, generate
    V, n, seen = 50, 11, []

    def draft(history, device):
        seen.append([list(h) for h in history])
        rows = [[(h[-1] + 1 + j) % V for j in range(wide)] for h in history]
        return Draft(torch.tensor(rows), torch.arange(-1, wide, dtype=torch.int32))

    prompt = torch.tensor([[3, 4, 5], [48, 49, 0]])
    # (the last token asked for is never fed: the text may be one longer than the table)
    out = generate(_Short(V, 3 + n - over), prompt, n, draft)
    want = (prompt[:, -1:] + 1 + torch.arange(n)) % V
    assert torch.equal(out, want)
    assert all(len(h) <= 3 + n and min(h) >= 0 for hs in seen for h in hs)


def test_generate_without_a_finite_logit():
    from hydranet_amd.model.speculative import generate
    with pytest.raises(RuntimeError, match="no logit is finite"):
        generate(_Short(50, 7), torch.tensor([[3, 4, 5]]), 9)


def test_generate_refuses_a_draft_wider_than_said():
    """At once, not where the cache happens to end."""
    from hydranet_amd.model.speculative import Draft, generate
    model = _Counting(50)

    def draft(history, device):
        return Draft(torch.zeros(len(history), 5, dtype=torch.int64),
                     torch.arange(-1, 5, dtype=torch.int32))
    with pytest.raises(AssertionError, match="at most 5 nodes"):
        generate(model, torch.tensor([[3, 4, 5]]), 30, draft, max_nodes=5)
    assert model.passes == 0
    assert generate(model, torch.tensor([[3, 4, 5]]), 30, draft, max_nodes=6).shape == (1, 30)


def test_generate_reads_the_device_back_once_a_pass(monkeypatch):
    from hydranet_amd.model import speculative
    from hydranet_amd.model.speculative import Draft, generate
    V, n, reads, inside = 50, 12, [0], [0]

    def draft(history, device):  # the second sequence's is wrong, so that the first ends before
        return Draft(torch.tensor([[(h[-1] + 1 + j) % V if h[0] == 3 else 0 for j in range(2)]
                                   for h in history]),
                     torch.tensor([-1, 0, 1], dtype=torch.int32))

    def tolist(self, _old=torch.Tensor.tolist):
        reads[0] += not inside[0]
        return _old(self)
    monkeypatch.setattr(torch.Tensor, "tolist", tolist)
    for owner, name in ((speculative, "verify_tree"), (DraftTree, "__init__")):  # GPU: kernels
        def kernel(*args, _old=getattr(owner, name)):
            inside[0] += 1
            try:
                return _old(*args)
            finally:
                inside[0] -= 1
        monkeypatch.setattr(owner, name, kernel)
    model = _Counting(V)
    out = generate(model, torch.tensor([[3, 4, 5], [13, 14, 15]]), n, draft)
    assert out.flatten().numpy().tolist() == [*range(6, 6 + n), *range(16, 16 + n)]
    assert model.passes == n - 1
    assert reads[0] == model.passes + 2  # and the prompt and the first tokens


class _Markov:
    """A model whose next token hangs on the last one alone."""

    def __init__(self, table):
        self.table = table

    def new_cache(self, batch, max_len):
        return KVCache.wrap([torch.zeros(batch, 1, 1, max_len)], [torch.zeros(batch, 1, max_len, 1)])

    def forward(self, ids, cache):
        return self.table[ids]

    def forward_tree(self, tokens, tree, lens, cache, bound):
        return self.table[tokens]


@pytest.mark.parametrize("soft", [True, False])
def test_generate_keeps_the_models_distribution(soft):
    """The first three tokens after a prompt, jointly, with trees of two branches drawn from
    another model (or certain).  N draws: a frequency's deviation is sqrt(p (1 - p) / N); 5 of
    it."""
    from hydranet_amd.model.speculative import Draft, generate
    g = torch.Generator().manual_seed(4)
    V, N, T = 3, 6000, 0.7
    table, other = torch.randn(V, V, generator=g), torch.randn(V, V, generator=g)
    q = torch.softmax(other / T, -1)
    parents = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32)

    def draft(history, device):
        last = torch.tensor([h[-1] for h in history])
        if not soft:
            return Draft(torch.stack((last, (last + 1) % V, last, last), 1), parents)
        a = torch.multinomial(q[last], 2, replacement=True, generator=g)
        b = torch.multinomial(q[a.flatten()], 1, generator=g).view(N, 2)
        nodes = torch.cat((last[:, None], a, b), 1)
        return Draft(nodes[:, 1:], parents, other[nodes])

    out = generate(_Markov(table), torch.tensor([[1]]), 3, draft, T, samples=N, generator=g)
    p = torch.softmax(table.double() / T, -1)
    want = p[1][:, None, None] * p[:, :, None] * p[None]
    got = torch.bincount((out * torch.tensor([V * V, V, 1])).sum(1), minlength=V ** 3).double() / N
    assert bool(((got.view(V, V, V) - want).abs() < 5 * (want * (1 - want) / N).sqrt()).all())
