"""The paged cache on the CPU: its operators' torch forms against 64-bit ones, the pages'
bookkeeping, the angles, and what is refused."""
import math

import pytest
import torch

from hydranet_amd.model.paged import (PagedBatch, PagedKVCache, RotaryTable, paged_append,
                                      paged_attention)
from hydranet_amd.model.sampling import adjust_logits
from tests import _paged_ref as ref

CASES = [
    # lens, counts (None: one row each), kv heads, query heads per KV head, hd, page
    ([0], None, 1, 1, 128, 16),
    ([15, -1, 16, 40], None, 2, 3, 8, 16),
    ([0, 20, -1, 5], [3, 0, 2, 40], 2, 2, 8, 32),
]


def _cache(s):
    return PagedKVCache.wrap([s["k"]], [s["v"]])


@pytest.mark.parametrize("dt", [torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(i, dt):
    lens, counts, nkv, rep, hd, page = CASES[i]
    s = ref.make(i, lens, counts, nkv, hd, page, dt, columns=i, poison=True)
    q = torch.randn(s["rows"], nkv * rep * hd, generator=s["gen"]).to(dt)
    want, bound = ref.attend(s, q, nkv * rep)
    got = paged_attention(q, ref.batch(s, counts is None), _cache(s), 0)
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all()


def test_attention_values_that_are_no_numbers():
    s = ref.make(1, [10], [6], 1, 8, 16, torch.float32)
    q = torch.randn(6, 16, generator=s["gen"])
    want = paged_attention(q, ref.batch(s, False), _cache(s), 0).view(6, 2, 8)
    s["v"][int(s["table"][0, 0]), 0, 1, 3, 4] = math.inf  # position 12, dimension 3
    got = paged_attention(q, ref.batch(s, False), _cache(s), 0).view(6, 2, 8)
    assert torch.equal(got[:2], want[:2]) and (got[2:, :, 3] == math.inf).all()
    got[2:, :, 3] = want[2:, :, 3]
    torch.testing.assert_close(got, want, rtol=1e-6, atol=1e-6)


def test_attention_pages_that_are_not_named():
    s = ref.make(4, [20, 30], [2, 3], 2, 8, 16, torch.float32)
    q = torch.randn(5, 32, generator=s["gen"])
    want = paged_attention(q, ref.batch(s, False), _cache(s), 0)
    for value, col in ((-1, 0), (s["k"].shape[0], 1), (-2 ** 31, 2)):
        bad = dict(s, table=s["table"].clone())
        bad["table"][1, col] = value
        got = paged_attention(q, ref.batch(bad, False), _cache(s), 0)
        first = 2 + max(0, 16 * col - 30)  # the row at the page's first position
        assert got[first:].isnan().all() and torch.equal(got[:first], want[:first])
    few = PagedBatch(s["table"], s["lens"], 50, s["starts"], 5, 2)
    got = paged_attention(q, few, _cache(s), 0)
    assert got[2:].isnan().all() and torch.equal(got[:2], want[:2])
    s["lens"][1] = 2 ** 63 - 1
    assert paged_attention(q, ref.batch(s, False, 50), _cache(s), 0)[2:].isnan().all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("i,rotary", [(0, 128), (1, 4), (2, 8), (1, 0), (2, 6)])
def test_append(i, rotary, layout):
    lens, counts, nkv, rep, hd, page = CASES[i]
    s = ref.make(i, lens, counts, nkv, hd, page, torch.float32)
    qkv = torch.randn(s["rows"], (nkv * rep + 2 * nkv) * hd, generator=s["gen"])
    cos, sin = ref.tables(rotary, 60) if rotary else (torch.zeros(60, 0),) * 2
    k, v = s["k"].clone(), s["v"].clone()
    got = paged_append(qkv, RotaryTable.wrap(cos, sin, layout), ref.batch(s, counts is None),
                       _cache(s), 0, nkv * rep)
    want = torch.zeros(s["rows"], nkv * rep, hd, dtype=torch.float64)
    for row, b, pos in ref.tokens(s):
        x = qkv[row].view(-1, hd)
        y = ref.rotate(x[:nkv * rep + nkv].double(), cos[pos], sin[pos], layout)
        want[row], p = y[:nkv * rep], int(s["table"][b, pos // page])
        k[p, :, pos % page] = y[nkv * rep:].float()
        v[p, :, pos % page // 8, :, pos % 8] = x[nkv * rep + nkv:]
    torch.testing.assert_close(got.view(want.shape).double(), want, rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(s["k"], k, rtol=1e-6, atol=1e-6)
    assert torch.equal(s["v"], v)


def test_append_outside():
    s = ref.make(2, [14, 30], [4, 4], 1, 8, 16, torch.float32)
    s["table"][0, 1] = s["k"].shape[0]
    cos, sin = ref.tables(8, 33)
    k, v = s["k"].clone(), s["v"].clone()
    q = paged_append(torch.randn(8, 24), RotaryTable.wrap(cos, sin), ref.batch(s, False),
                     _cache(s), 0, 1)
    assert q.isnan().all(1).tolist() == [False, False, True, True, False, False, False, True]
    same = torch.tensor([torch.equal(a, b) for a, b in zip(k, s["k"])])
    assert (~same).sum() == 3  # the pages of positions 14, 15; 30, 31; 32
    assert sum(not torch.equal(a, b) for a, b in zip(v, s["v"])) == 3


def test_append_then_attend_as_a_whole():
    """A text in chunks, then token by token, against all of it in one step."""
    cos, sin = ref.tables(16, 70)
    rope = RotaryTable.wrap(cos, sin, "interleaved")
    qkv = torch.randn(70, 4 * 16, generator=torch.Generator().manual_seed(1)).double()

    def run(steps):
        cache = PagedKVCache(1, 9, 1, 16, 16, dtype=torch.float64)
        pages = cache.take(5)
        out, at = [], 0
        for m in steps:
            one = PagedBatch(cache.table([pages]), torch.tensor([at]), 70,
                             torch.tensor([0, m], dtype=torch.int32), m, m)
            q = paged_append(qkv[at:at + m], rope, one, cache, 0, 2)
            out.append(paged_attention(q, one, cache, 0))
            at += m
        return torch.cat(out)
    whole = run([70])
    torch.testing.assert_close(run([33, 20] + [1] * 17), whole, rtol=1e-12, atol=1e-12)


def test_pages():
    c = PagedKVCache(2, 10, 1, 8, 16)
    a = c.take(4)
    assert c.free_pages == 6 and len(set(a)) == 4 and c.pages_for(33) == 3 and c.pages_for(0) == 0
    with pytest.raises(RuntimeError, match="KV cache full"):
        c.take(7)
    for t in c.k + c.v:
        t.normal_()
    b = c.fork(a, 40)  # two full pages and 8 positions of a third
    assert b[:2] == a[:2] and b[2] not in a and len(b) == 3 and c.free_pages == 5
    assert all(torch.equal(t[b[2]], t[a[2]]) for t in c.k + c.v)
    assert c.fork(a, 32) == a[:2] and c.free_pages == 5  # nothing to copy
    c.give(a)
    assert c.free_pages == 7  # a's own two
    c.give(a[:2])
    assert c.free_pages == 7
    with pytest.raises(AssertionError, match="free already"):
        c.give(b + b)
    assert c.free_pages == 7
    c.give(b)
    assert c.free_pages == 10
    with pytest.raises(AssertionError, match="taken"):
        c.share([0])
    with pytest.raises(AssertionError, match="taken"):
        c.fork([0, 1], 20)
    assert c.free_pages == 10
    assert c.table([[1, 2], [], [3]]).tolist() == [[1, 2], [-1, -1], [3, -1]]
    assert c.table([[1]], 3).tolist() == [[1, -1, -1]]
    for src, dst in (([0], [0]), ([0, 1], [1, 2]), ([0, 0], [3, 3]), ([10], [1]), ([0], [-1]),
                     ([0], [1, 2])):
        with pytest.raises(AssertionError):
            c.copy(src, dst)


@pytest.mark.parametrize("dim,base", [(128, 1e6), (64, 1e4), (2, 1e4), (0, 1e4)])
def test_rotary_table(dim, base):
    t = RotaryTable(dim, 40000, base)
    assert t.dim == dim and tuple(t.cos.shape) == (40000, dim // 2) and t.layout == "half"
    for p in (0, 1, 39999):
        for i in range(dim // 2):
            a = p * base ** (-2 * i / dim)
            # (the power and the product in 64 bits: 1e-11 of 4e4 turns; then one rounding)
            assert abs(float(t.cos[p, i]) - math.cos(a)) <= 2.0 ** -24 + 1e-10
            assert abs(float(t.sin[p, i]) - math.sin(a)) <= 2.0 ** -24 + 1e-10


def test_rotary_scaling():
    plain = RotaryTable(64, 4096, 1e4)
    lin = RotaryTable(64, 4096, 1e4, scaling={"type": "linear", "factor": 4.0})
    assert torch.equal(lin.cos[::4][:1000], plain.cos[:1000])

    def angle(t, i, n):  # a position's angle at index i, of small positions
        return math.atan2(float(t.sin[n, i]), float(t.cos[n, i]))
    ntk = RotaryTable(64, 64, 1e4, scaling={"type": "ntk", "factor": 8.0})
    assert abs(angle(ntk, 0, 1) - 1.0) < 1e-6
    assert abs(angle(ntk, 31, 63) * 8 / angle(plain, 31, 63) - 1) < 1e-4
    for f, n in ((4.0, 4096), (16.0, 512)):
        y = RotaryTable(64, 64, 1e4, "interleaved",
                        {"type": "yarn", "factor": f, "original": n})
        size = 0.1 * math.log(f) + 1
        r = (y.cos.double() ** 2 + y.sin.double() ** 2).sqrt()
        assert (r / size - 1).abs().max() < 1e-6
        for i in range(32):
            turns = n * 1e4 ** (-2 * i / 64) / (2 * math.pi)
            ratio = angle(y, i, 1) / angle(plain, i, 1)
            assert 1 / f - 1e-4 <= ratio <= 1 + 1e-4
            # (the borders are rounded outwards to whole indices)
            if turns > 32 * 1e4 ** (2 / 64):
                assert abs(ratio - 1) < 1e-4
            if turns < 1e4 ** (-2 / 64):
                assert abs(ratio * f - 1) < 1e-3
    for bad in ({"type": "linear", "factor": 0.5}, {"type": "other", "factor": 2.0},
                {"type": "yarn", "factor": 2.0, "original": 0},
                {"type": "yarn", "factor": 2.0, "original": 9, "fast": 1, "slow": 2}):
        with pytest.raises(AssertionError):
            RotaryTable(64, 8, 1e4, scaling=bad)
    for a in ((3, 8), (-2, 8), (8, -1), (8, 8, 0.0), (8, 8, 1e4, "other")):
        with pytest.raises(AssertionError):
            RotaryTable(*a)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_adjust_logits(dt):
    g = torch.Generator().manual_seed(3)
    T, B, V, width = ref.TYPES[dt], 3, 70, 40
    x = (torch.randn(B, V, generator=g) * 4).to(T)
    text = torch.randint(-1, V + 1, (B, width), generator=g)
    lens, prompt = torch.tensor([0, 17, 99]), torch.tensor([0, 5, 30])
    amounts = [torch.rand(B, generator=g) + 0.5 for _ in range(3)]
    ids = torch.randint(-1, V + 1, (B, 9), generator=g)
    ids[:, 8] = ids[:, 2]
    bias = (ids, torch.randn(B, 9, generator=g))
    bits = torch.randint(-2 ** 31, 2 ** 31, (B, 3), generator=g).int()
    y, bound = ref.adjust(x, text, lens, prompt, *amounts, bias, bits)
    got = adjust_logits(x, text, lens, prompt, *amounts, bias, bits)
    fin = y.isfinite()
    assert torch.equal(got.double()[~fin], y[~fin])
    assert ((got.double() - y).abs() <= bound)[fin].all()
    assert torch.equal(adjust_logits(x), x) and adjust_logits(x, out=x) is x


def _refused(match, call, *a, **kw):
    with pytest.raises(AssertionError, match=match):
        call(*a, **kw)


def test_refusals():
    s = ref.make(1, [5, 7], None, 2, 8, 16, torch.float32)
    c, one = _cache(s), ref.batch(s, True)
    t, lens = s["table"], s["lens"]
    rope = RotaryTable(8, 64)
    q, qkv = torch.randn(2, 32), torch.randn(2, 64)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32)
    _refused("table", PagedBatch, t.long(), lens, 9)
    _refused("table", PagedBatch, t[0], lens, 9)
    _refused("table", PagedBatch, torch.zeros(3, 2, dtype=torch.int32).t(), lens, 9)
    _refused("table", PagedBatch, torch.zeros(1, 3, dtype=torch.int32).expand(2, 3), lens, 9)
    _refused("sequence", PagedBatch, t[:0], lens[:0], 9, starts[:1], 4)
    _refused("lens", PagedBatch, t, lens.int(), 9)
    _refused("lens", PagedBatch, t, lens[:1], 9)
    _refused("kv_bound", PagedBatch, t, lens, 0)
    _refused("one row", PagedBatch, t, lens, 9, None, 3)
    _refused("one row", PagedBatch, t, lens, 9, None, 2, 2)
    _refused("starts", PagedBatch, t, lens, 9, starts.long(), 2)
    _refused("starts", PagedBatch, t, lens, 9, starts[:2], 2)
    _refused("rows", PagedBatch, t, lens, 9, starts)
    _refused("rows", PagedBatch, t, lens, 9, starts, 2, 0)
    _refused("layer", paged_attention, q, one, c, 1)
    _refused("heads", paged_attention, torch.randn(2, 24), one, c, 0)
    _refused("heads", paged_attention, torch.randn(2, 30), one, c, 0)
    _refused("rows", paged_attention, torch.randn(3, 32), one, c, 0)
    _refused("cache", paged_attention, q.half(), one, c, 0)
    _refused("scale", paged_attention, q, one, c, 0, 0.0)
    _refused("scale", paged_attention, q, one, c, 0, math.inf)
    _refused("scale", paged_attention, q, one, c, 0, math.nan)
    _refused("heads", paged_append, qkv, rope, one, c, 0, 3)
    _refused("qkv", paged_append, qkv[:, 1:], rope, one, c, 0, 4)
    _refused("cache", paged_append, qkv.half(), rope, one, c, 0, 4)
    _refused("rotated", paged_append, qkv, RotaryTable(10, 64), one, c, 0, 4)
    _refused("cos, sin", RotaryTable.wrap, rope.cos.double(), rope.sin.double())
    _refused("cos, sin", RotaryTable.wrap, rope.cos, rope.sin[:3])
    _refused("pages of 16", PagedKVCache, 1, 4, 1, 8, 24)
    _refused("pages of 16", PagedKVCache, 1, 4, 1, 8, 8)
    _refused("pages of 16", PagedKVCache, 1, 4, 1, 8, 2048)
    _refused("layer", PagedKVCache.wrap, [s["k"]], [])
    _refused("keys", PagedKVCache.wrap, [s["k"]], [s["v"].view(s["k"].shape)])
    _refused("keys", PagedKVCache.wrap, [s["k"]], [s["v"].half()])
    x, text = torch.zeros(2, 40), torch.zeros(2, 5, dtype=torch.int64)
    one_ = torch.ones(2)
    _refused("logits", adjust_logits, x[0])
    _refused("logits", adjust_logits, x.double())
    _refused("logits", adjust_logits, x[:, :0])
    _refused("text", adjust_logits, x, text.int())
    _refused("text", adjust_logits, x, text[:1])
    _refused("are of a text", adjust_logits, x, None, torch.tensor([1, 2]))
    _refused("lens", adjust_logits, x, text, torch.tensor([1]))
    _refused("prompt", adjust_logits, x, text, None, torch.tensor([1, 2]).int())
    _refused("repetition", adjust_logits, x, text, repetition=0.0)
    _refused("repetition", adjust_logits, x, text, repetition=one_.double())
    _refused("presence", adjust_logits, x, text, presence=math.nan)
    _refused("frequency", adjust_logits, x, text, frequency=one_[:1])
    _refused("bias", adjust_logits, x, bias=(text.int(), torch.zeros(2, 5)))
    _refused("bias", adjust_logits, x, bias=(text, torch.zeros(2, 4)))
    _refused("allowed", adjust_logits, x, allowed=torch.zeros(2, 1, dtype=torch.int32))
    _refused("allowed", adjust_logits, x, allowed=torch.zeros(2, 2, dtype=torch.int64))
    _refused("out", adjust_logits, x, out=x.half())
    _refused("out", adjust_logits, x, out=torch.zeros(40, 2).t())


def test_library_refusals():
    """The C entries refuse before any GPU work; calls over nothing succeed."""
    from hydranet_amd import _lib

    import ctypes

    def step(B=1, T=1, nh=4, nkv=1, hd=128, page=16, cols=1, ldt=1, n=1, starts=None, p=16, new=1,
             bound=1, table=16):
        s = _lib.PagedStep(p and table, ldt, cols, n, p, starts, B, T, nh, nkv, hd, page, new,
                           bound)
        step.last = s
        return ctypes.addressof(s)

    def append(dtype=0, rotary=128, ld=768, p=16, cos=16, no=False, **kw):
        at = None if no else step(p=p, **kw)
        _lib.call("hn_paged_append", at, p, ld, dtype, cos, cos, 8, rotary, 0, p, p, p, None)

    def attend(dtype=0, ld=512, p=16, scale=0.1, out=16, work=None, bytes_=0, no=False, **kw):
        at = None if no else step(p=p, **kw)
        _lib.call("hn_paged_attention", at, p, ld, dtype, p, p, scale, out, 512, work, bytes_,
                  None)
    append(B=0, T=0, p=None), append(B=2, T=0, starts=16, p=None), attend(B=0, T=0, p=None)
    sizes = (dict(dtype=2), dict(T=2), dict(B=-1, T=-1), dict(nh=3, nkv=2), dict(nkv=0),
             dict(hd=96), dict(page=24), dict(page=8), dict(page=2048), dict(cols=2),
             dict(p=None), dict(p=8), dict(n=-1), dict(table=None), dict(no=True),
             dict(B=70000, T=70000))
    for kw in sizes + (dict(rotary=130), dict(rotary=3), dict(rotary=-2), dict(ld=767),
                       dict(cos=None), dict(T=1 << 29, starts=16)):
        with pytest.raises(RuntimeError, match="hn_paged_append"):
            append(**kw)
    long = dict(cols=129, ldt=129, bound=3000)
    need = _lib.lib().hn_paged_attention_workspace_bytes(step(**long))
    assert need > 0 and _lib.lib().hn_paged_attention_workspace_bytes(step(bound=100)) == 0
    for kw in sizes + (dict(ld=504), dict(ld=514), dict(out=None), dict(out=8), dict(scale=0.0),
                       dict(scale=math.nan), dict(scale=3e38), dict(new=0), dict(bound=0),
                       dict(n=0), dict(cols=1 << 26, ldt=1 << 26), long,
                       dict(long, work=16, bytes_=need - 1), dict(long, work=8, bytes_=need),
                       dict(new=1 << 23),
                       dict(nh=1, ld=512, new=1 << 24)):
        with pytest.raises(RuntimeError, match="hn_paged_attention"):
            attend(**kw)

    def adjust(p=16, dtype=0, B=1, V=8, ld=8, width=0, n=0, allowed=None, lda=0, text=None):
        _lib.call("hn_adjust_logits", p, ld, dtype, text, width, width, None, None, None, None,
                  None, 1.0, 0.0, 0.0, None, n, None, n, n, allowed, lda, B, V, p, 8, None)
    adjust(B=0, p=None), adjust(V=0, p=None)
    for kw in (dict(dtype=3), dict(p=None), dict(ld=7), dict(width=3), dict(n=2), dict(B=-1),
               dict(V=-1), dict(V=9), dict(allowed=16), dict(n=-1), dict(width=-1),
               dict(B=70000)):
        with pytest.raises(RuntimeError, match="hn_adjust_logits"):
            adjust(**kw)
    one, ptr = (ctypes.c_int * 1)(0), (ctypes.c_void_p * 1)(16)
    two = (ctypes.c_int * 1)(5)
    for a in ((ptr, ptr, 1, 24, 4, one, one, 1), (ptr, ptr, 1, 32, 4, one, two, 1),
              (None, ptr, 1, 32, 4, one, one, 1), (ptr, ptr, -1, 32, 4, one, one, 1)):
        with pytest.raises(RuntimeError, match="hn_page_copy"):
            _lib.call("hn_page_copy", *a, None)
    _lib.call("hn_page_copy", ptr, ptr, 1, 32, 4, one, one, 0, None)
