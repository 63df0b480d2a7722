"""GPU tests of the paged cache's kernels (hn_paged_append, hn_paged_attention,
hn_page_copy) and of adjusted logits (hn_adjust_logits) against 64-bit forms."""
import math

import pytest
import torch

from tests import _paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CASES = [
    # lens, counts (None: one row each), kv heads, query heads per KV head, hd, page
    ([0], None, 1, 1, 128, 16),
    ([15], None, 8, 4, 128, 16),
    ([63, 64, 0, -1, 1], None, 2, 4, 128, 64),
    ([700, 3, 31, 33, 1000], None, 2, 12, 128, 16),
    ([257, 1023], None, 1, 16, 64, 32),
    ([128, 95], None, 2, 17, 64, 128),
    ([300, -1, 64], None, 2, 3, 256, 64),
    ([2300], None, 4, 8, 128, 1024),
    ([0, 0, 0], [1, 70, 33], 2, 4, 128, 64),
    ([100, -1, 7, 0], [3, 5, 0, 130], 2, 4, 128, 16),
    ([31, 63], [2, 1], 4, 1, 64, 32),
    ([500], [257], 1, 6, 256, 128),
    ([5, 0], [40, 300], 1, 20, 64, 16),
]


def _cache(s):
    from hydranet_amd.model.paged import PagedKVCache
    return PagedKVCache.wrap([s["k"]], [s["v"]])


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(i, dt):
    from hydranet_amd.model.paged import paged_attention
    lens, counts, nkv, rep, hd, page = CASES[i]
    s = ref.make(i, lens, counts, nkv, hd, page, ref.TYPES[dt], DEV, columns=i % 3, poison=True)
    q = torch.randn(s["rows"], nkv * rep * hd, generator=s["gen"]).mul(2).to(ref.TYPES[dt])
    want, bound = ref.attend(s, q, nkv * rep)
    one = ref.batch(s, counts is None)
    got = paged_attention(q.to(DEV), one, _cache(s), 0)
    assert torch.isfinite(got).all()
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # bounds are hints, and rows may have a stride
    wide = torch.randn(s["rows"], nkv * rep * hd + 8, device=DEV).to(q.dtype)
    wide[:, :q.shape[1]] = q
    for hint in (1, 100, 5000, 2 ** 40):
        two = paged_attention(wide[:, :q.shape[1]], ref.batch(s, counts is None, hint), _cache(s),
                              0)
        assert ((two.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,nkv,rep,page", [([9000, 40, 3000], 2, 4, 16), ([30001], 1, 2, 64),
                                               ([1500] * 7 + [0], 1, 12, 256)])
def test_attention_over_long_texts(lens, nkv, rep, page, dt):
    from hydranet_amd.model.paged import paged_attention
    s = ref.make(3, lens, None, nkv, 128, page, ref.TYPES[dt], DEV, poison=True)
    q = torch.randn(s["rows"], nkv * rep * 128, generator=s["gen"]).mul(2).to(ref.TYPES[dt])
    want, bound = ref.attend(s, q, nkv * rep)
    for hint in (None, 700, 1 << 20):
        got = paged_attention(q.to(DEV), ref.batch(s, True, hint), _cache(s), 0)
        assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("counts", [None, [1, 40, 9]])
def test_attention_large_scores(counts):
    """Scores of hundreds, and a scale of one's own: the largest takes it all."""
    from hydranet_amd.model.paged import paged_attention
    s = ref.make(8, [400, 70, 0], counts, 2, 64, 32, torch.float16, DEV, poison=True)
    q = torch.randn(s["rows"], 8 * 64, generator=s["gen"]).mul(16).half()
    want, bound = ref.attend(s, q, 8, 0.7)
    got = paged_attention(q.to(DEV), ref.batch(s, counts is None), _cache(s), 0, scale=0.7)
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("hint", [None, 5000])
@pytest.mark.parametrize("counts", [None, [1, 5, 2], [30, 40, 100]])
def test_pages_that_are_not_named(counts, hint):
    """A missing page, an id past the pages, a table too short: NaN in the rows that see the
    place, and all others as they are."""
    from hydranet_amd.model.paged import paged_attention
    s = ref.make(4, [100, 180, 90], counts, 2, 128, 16, torch.float16, DEV, poison=True)
    q = torch.randn(s["rows"], 8 * 128, generator=s["gen"]).half().to(DEV)
    want = paged_attention(q, ref.batch(s, counts is None, hint), _cache(s), 0)
    starts = s["starts"].tolist()
    assert want.isfinite().all()

    def check(bad, first):
        """NaN from position `first` of sequence 1 on."""
        got = paged_attention(q, ref.batch(bad, counts is None, hint or 300), _cache(s), 0)
        for row, b, pos in ref.tokens({n: s[n].cpu() for n in ("starts", "lens")}):
            if b == 1 and pos >= first:
                assert got[row].isnan().all()
            else:
                assert torch.equal(got[row], want[row])
    for value, col in ((-1, 0), (s["k"].shape[0], 3), (-2 ** 31, 11), (2 ** 31 - 1, 12)):
        if counts is None and col == 12:
            continue  # (positions 192 on: none of a single token's)
        if col < s["table"].shape[1]:
            bad = dict(s, table=s["table"].clone())
            bad["table"][1, col] = value
            check(bad, 16 * col)
    check(dict(s, table=s["table"][:, :12].contiguous()), 192)
    check(dict(s, table=torch.cat((s["table"][:, :12], s["table"]), 1)[:, :12]), 192)
    for C in (2 ** 63 - 1, 2 ** 31, 10 ** 6):
        far = dict(s, lens=s["lens"].clone())
        far["lens"][1] = C
        check(far, 0)
    none = dict(s, table=s["table"][:, :0])
    got = paged_attention(q, ref.batch(none, counts is None, hint), _cache(s), 0)
    assert got.isnan().all() and starts[-1] == s["rows"]


@pytest.mark.parametrize("hint", [None, 5000])
@pytest.mark.parametrize("rep,hd,n", [(4, 128, 50), (1, 64, 50), (20, 64, 50), (2, 256, 50),
                                      (4, 128, 4), (4, 64, 8), (2, 256, 8)])
def test_values_that_are_no_numbers(rep, hd, n, hint):
    """A value that is NaN or infinite reaches the rows that see it and no other."""
    from hydranet_amd.model.paged import paged_attention
    C = 1037
    s = ref.make(6, [C, 5], [n, 8], 1, hd, 16, torch.float16, DEV, poison=True)
    q = torch.randn(s["rows"], rep * hd, generator=s["gen"]).half().to(DEV)

    def run():
        return paged_attention(q, ref.batch(s, False, hint), _cache(s), 0)
    want = run()
    for at, d, x in ((C + n // 2, 3, math.nan), (C + n - 1, hd - 1, math.inf),
                     (C + 1, 0, -math.inf)):
        old = s["v"].clone()
        p = int(s["table"][0, at // 16])
        s["v"][p, 0, at % 16 // 8, d, at % 8] = x
        got = run().view(-1, rep, hd)
        s["v"].copy_(old)
        w = want.view(-1, rep, hd).clone()
        w[at - C:n, :, d] = x
        other = torch.ones_like(w, dtype=torch.bool)
        other[at - C:n, :, d] = False
        hit = got[~other]
        assert hit.isnan().all() if math.isnan(x) else (hit == x).all()
        assert torch.equal(got[other], w[other])
    # a key: its scores are no numbers, so neither are the rows that see it
    at = C + n // 2
    s["k"][int(s["table"][0, at // 16]), 0, at % 16, 1] = math.nan
    got = run()
    assert got[n // 2:n].isnan().all() and torch.equal(got[:n // 2], want[:n // 2])
    assert torch.equal(got[n:], want[n:])


@pytest.mark.parametrize("hint", [None, 9000])
@pytest.mark.parametrize("runs", [False, True])
def test_many_sequences(runs, hint):
    """Hundreds of sequences of ragged lengths, some without part, some without rows."""
    from hydranet_amd.model.paged import RotaryTable, paged_append, paged_attention
    g = torch.Generator().manual_seed(1)
    B = 210
    lens = (torch.rand(B, generator=g) ** 3 * 700).long().tolist()
    counts = (torch.rand(B, generator=g) ** 4 * 30).long().tolist() if runs else None
    for b in range(0, B, 7):
        lens[b] = -1
    s = ref.make(12, lens, counts, 1, 64, 16, torch.float16, DEV, poison=True)
    one = ref.batch(s, not runs, hint)
    q = torch.randn(s["rows"], 3 * 64, generator=s["gen"]).half()
    want, bound = ref.attend(s, q, 3)
    got = paged_attention(q.to(DEV), one, _cache(s), 0)
    assert ((got.double().cpu() - want).abs() <= bound).all()
    cos, sin = ref.tables(64, 800)
    qkv = torch.randn(s["rows"], 5 * 64, generator=s["gen"]).half()
    q = paged_append(qkv.to(DEV), RotaryTable.wrap(cos.to(DEV), sin.to(DEV)), one, _cache(s), 0, 3)
    live = torch.zeros(s["rows"], dtype=torch.bool)
    k, v, table = s["k"].cpu(), s["v"].cpu(), s["table"].cpu()
    for row, b, pos in ref.tokens({n: s[n].cpu() for n in ("starts", "lens")}):
        live[row] = True
        x = qkv[row].view(5, 64)
        y = ref.rotate(x[:4].double(), cos[pos], sin[pos], "half")
        out = torch.cat((q[row].cpu().view(3, 64), k[table[b, pos // 16], :, pos % 16])).double()
        assert ((out - y).abs() <= 2.0 ** -11 * y.abs() + 2.0 ** -20).all()
        assert torch.equal(v[table[b, pos // 16], 0, pos % 16 // 8, :, pos % 8], x[4])
    assert not q[~live.to(DEV)].any()


def test_two_calls_at_once():
    """Attention of two batches on two streams, each with its own workspace."""
    from hydranet_amd.model.paged import paged_attention
    work = []
    for seed, lens in ((1, [9000, 100]), (2, [3000, 5000, 7000])):
        s = ref.make(seed, lens, None, 2, 128, 64, torch.float16, DEV)
        q = torch.randn(len(lens), 8 * 128, generator=s["gen"]).half().to(DEV)
        work.append((q, ref.batch(s, True), _cache(s), torch.cuda.Stream()))
    want = [paged_attention(q, one, cache, 0) for q, one, cache, _ in work]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for q, one, cache, stream in work:
            with torch.cuda.stream(stream):
                got.append(paged_attention(q, one, cache, 0))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("i,rotary", [(0, 128), (1, 64), (2, 128), (3, 32), (4, 64), (5, 20),
                                      (6, 256), (7, 2), (8, 128), (9, 0), (10, 34), (11, 128),
                                      (12, 64)])
@pytest.mark.parametrize("offset", [0, 1])
def test_append(i, rotary, dt, layout, offset):
    """offset: rows that start anywhere, with a stride."""
    from hydranet_amd.model.paged import RotaryTable, paged_append
    lens, counts, nkv, rep, hd, page = CASES[i]
    T = ref.TYPES[dt]
    s = ref.make(i, lens, counts, nkv, hd, page, T, DEV, columns=1)
    nh = nkv * rep
    wide = torch.randn(s["rows"], (nh + 2 * nkv) * hd + 3 * offset, generator=s["gen"]).to(T)
    qkv = wide[:, offset:offset + (nh + 2 * nkv) * hd]
    cos, sin = ref.tables(rotary, max(lens) + s["rows"] + 1) if rotary else \
        (torch.zeros(5000, 0),) * 2
    k, v = s["k"].clone().cpu(), s["v"].clone().cpu()
    rope = RotaryTable.wrap(cos.to(DEV), sin.to(DEV), layout)
    got = paged_append(wide.to(DEV)[:, offset:offset + (nh + 2 * nkv) * hd], rope,
                       ref.batch(s, counts is None), _cache(s), 0, nh).cpu()
    table, u = s["table"].cpu(), ref.half_step(T)
    kd, vd = s["k"].cpu(), s["v"].cpu()
    live = set()
    for row, b, pos in ref.tokens({n: s[n].cpu() for n in ("starts", "lens")}):
        live.add(row)
        x = qkv[row].view(nh + 2 * nkv, hd)
        y = ref.rotate(x[:nh + nkv].double(), cos[pos], sin[pos], layout)
        # two products and a sum in fp32, of magnitudes up to twice the row's largest
        bound = u * y.abs() + 3 * 2.0 ** -24 * 2 * x.double().abs().max() + ref.subnormal(T)
        p = int(table[b, pos // page])
        out = torch.cat((got[row].view(nh, hd), kd[p, :, pos % page])).double()
        assert ((out - y).abs() <= bound).all(), (row, float(((out - y).abs() / bound).max()))
        assert torch.equal(out[:, rotary:], y[:, rotary:])
        k[p, :, pos % page] = kd[p, :, pos % page]
        v[p, :, pos % page // 8, :, pos % 8] = x[nh + nkv:]
    assert torch.equal(v, vd) and torch.equal(k, kd)  # all else as it was
    assert all(row in live or not got[row].any() for row in range(s["rows"]))


@pytest.mark.parametrize("counts", [None, [9, 20, 33, 1]])
def test_append_outside(counts):
    """Past the table of angles, past the table of pages, on no page: NaN queries, nothing
    written."""
    from hydranet_amd.model.paged import RotaryTable, paged_append
    s = ref.make(2, [40, 20, 300, 2], counts, 2, 128, 16, torch.float16, DEV)
    s["table"][0, 2] = 10 ** 6  # positions 32 to 47
    s["table"][1, 1] = -1       # 16 to 31
    cos, sin = ref.tables(128, 310)
    qkv = torch.randn(s["rows"], 8 * 128, generator=s["gen"]).half().to(DEV)
    s["lens"][3] = 2 ** 63 - 1
    k, v = s["k"].clone(), s["v"].clone()
    q = paged_append(qkv, RotaryTable.wrap(cos.to(DEV), sin.to(DEV)),
                     ref.batch(s, counts is None, 400), _cache(s), 0, 4)
    starts = s["starts"].tolist()
    for row, b, pos in ref.tokens({n: s[n].cpu() for n in ("starts", "lens")}):
        bad = b == 3 or pos >= 310 or b == 0 and 32 <= pos < 48 or b == 1 and 16 <= pos < 32
        assert bool(q[row].isnan().all()) == bad and bool(q[row].isfinite().all()) != bad
        if not bad:
            p = int(s["table"][b, pos // 16])
            assert not torch.equal(s["k"][p, :, pos % 16], k[p, :, pos % 16])
            k[p, :, pos % 16] = s["k"][p, :, pos % 16]
            v[p, :, pos % 16 // 8, :, pos % 8] = s["v"][p, :, pos % 16 // 8, :, pos % 8]
    assert torch.equal(k, s["k"]) and torch.equal(v, s["v"]) and starts[-1] == s["rows"]


def test_rows_of_no_sequence():
    """Rows behind the last sequence (and before the first) come back zero and write
    nothing; a run longer than max_new has NaN rows."""
    from hydranet_amd.model.paged import PagedBatch, RotaryTable, paged_append, paged_attention
    s = ref.make(9, [30, 5], [100, 7], 2, 128, 16, torch.float16, DEV)
    rows = s["rows"] + 13
    cos, sin = ref.tables(128, 200)
    rope = RotaryTable.wrap(cos.to(DEV), sin.to(DEV))
    qkv = torch.randn(rows, 8 * 128, generator=s["gen"]).half().to(DEV)
    one = PagedBatch(s["table"], s["lens"], 50, s["starts"], rows, 100)
    q = paged_append(qkv, rope, one, _cache(s), 0, 4)
    out = paged_attention(q, one, _cache(s), 0)
    for x in (q, out):
        assert not x[s["rows"]:].any() and x[:s["rows"]].any(1).all()
    want, bound = ref.attend(s, q[:s["rows"]], 4)
    assert ((out[:s["rows"]].double().cpu() - want).abs() <= bound).all()
    late = PagedBatch(s["table"], s["lens"], 50, s["starts"] + 4, rows, 100)
    q2 = torch.cat((q[:4], q[:rows - 4]))
    out2 = paged_attention(q2, late, _cache(s), 0)
    assert not out2[:4].any() and torch.equal(out2[4:4 + s["rows"]], out[:s["rows"]])
    for hint in (50, 5000):
        few = PagedBatch(s["table"], s["lens"], hint, s["starts"], rows, 7)
        out3 = paged_attention(q, few, _cache(s), 0)
        assert out3[:100].isnan().all() and not out3[s["rows"]:].any()
        assert ((out3[100:s["rows"]].double().cpu() - want[100:]).abs() <= bound[100:]).all()


def test_page_copy():
    from hydranet_amd.model.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(0)
    c = PagedKVCache(70, 90, 2, 64, 16, DEV)
    for t in c.k + c.v:
        t.normal_(generator=g)
    src = [3] * 56 + list(range(4, 18))
    dst = list(range(89, 19, -1))
    want = [t.clone() for t in c.k + c.v]
    for t in want:
        t[dst] = t[src].clone()
    c.copy(src, dst)
    assert all(torch.equal(a, b) for a, b in zip(want, c.k + c.v))


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("B,V,width", [(1, 1, 0), (1, 31, 5), (3, 1000, 70), (2, 4097, 3000),
                                       (5, 2048, 1), (2, 9001, 12000)])
def test_adjust_logits(B, V, width, dt):
    from hydranet_amd.model.sampling import adjust_logits
    g = torch.Generator().manual_seed(V)
    T = ref.TYPES[dt]
    x = (torch.randn(B, V, generator=g) * 4).to(T)
    x[0, V // 2] = -math.inf
    x[-1, V - 1] = math.inf
    text = (torch.rand(B, width, generator=g) ** 3 * (V + 3)).long() - 1  # (some outside)
    lens = torch.randint(-1, width + 2, (B,), generator=g)
    prompt = (lens.clamp(min=0) * torch.rand(B, generator=g)).long()
    amounts = [torch.rand(B, generator=g) + lo for lo in (0.6, -0.5, -0.3)]
    n = min(V, 37) + 3
    ids = torch.randint(-2, V + 1, (B, n), generator=g)
    ids[:, -1] = ids[:, 0]  # the same token twice
    bias = (ids, torch.randn(B, n, generator=g) * 5)
    bits = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32 + 1), generator=g).int()
    bits[0] = 0  # nothing is allowed
    on = lambda a: tuple(map(on, a)) if isinstance(a, tuple) else a.to(DEV)  # noqa: E731
    for use in ("all", "text", "bias", "bits", "numbers"):
        kw, want = {}, {}
        if use in ("all", "text"):
            kw = dict(text=on(text), lens=on(lens), prompt=on(prompt), repetition=on(amounts[0]),
                      presence=on(amounts[1]), frequency=on(amounts[2]))
            want = dict(text=text, lens=lens, prompt=prompt, rep=amounts[0], pres=amounts[1],
                        freq=amounts[2])
        if use == "numbers":
            kw = dict(text=on(text), repetition=1.25, presence=0.5, frequency=-0.25)
            want = dict(text=text, rep=1.25, pres=0.5, freq=-0.25)
        if use in ("all", "bias"):
            kw["bias"], want["bias"] = on(bias), bias
        if use in ("all", "bits"):
            kw["allowed"], want["allowed"] = on(bits), bits
        y, bound = ref.adjust(x, **want)
        got = adjust_logits(on(x), **kw).cpu()
        wide = torch.zeros(B, V + 5, dtype=T, device=DEV)[:, 3:3 + V]
        wide.copy_(x)
        assert adjust_logits(wide, out=wide, **kw) is wide and torch.equal(wide.cpu(), got)
        fin = y.isfinite() & (y.abs() < torch.finfo(T).max)
        assert torch.equal(got.double()[~fin], y[~fin])
        assert ((got.double() - y).abs() <= bound)[fin].all()


def test_adjust_logits_keeps_nan():
    from hydranet_amd.model.sampling import adjust_logits
    x = torch.zeros(1, 64, device=DEV)
    x[0, 3] = x[0, 40] = math.nan
    bits = torch.tensor([[-1, 0]], dtype=torch.int32, device=DEV)
    y = adjust_logits(x, torch.tensor([[3, 40]], device=DEV), repetition=2.0, allowed=bits)
    assert y[0, 3].isnan() and (y[0, 32:] == -math.inf).all() and not y[0, :3].any()


def test_other_streams_and_graphs():
    """A step on another stream, and captured and replayed as the sequences grow, beside
    eager calls of the same batch."""
    from hydranet_amd.model.paged import RotaryTable, paged_append, paged_attention
    from hydranet_amd.model.sampling import adjust_logits
    s = ref.make(5, [90, 511, -1, 0], None, 2, 128, 16, torch.float16, DEV, columns=3)
    s["table"] = torch.randperm(200, generator=s["gen"])[:4 * 40].view(4, 40).int().to(DEV)
    s["k"] = torch.randn(200, 2, 16, 128, device=DEV).half()
    s["v"] = torch.randn(200, 2, 2, 128, 8, device=DEV).half()
    cache, one = _cache(s), ref.batch(s, True, 600)
    cos, sin = ref.tables(128, 700)
    rope = RotaryTable.wrap(cos.to(DEV), sin.to(DEV))
    qkv = torch.randn(4, 12 * 128, device=DEV).half()
    lg = torch.randn(4, 1000, device=DEV)
    text = torch.randint(0, 1000, (4, 700), device=DEV)

    def step():
        q = paged_append(qkv, rope, one, cache, 0, 8)
        return paged_attention(q, one, cache, 0), adjust_logits(lg, text, s["lens"],
                                                                frequency=0.3)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        s["lens"].add_((s["lens"] >= 0) * 17)
        qkv.normal_()
        eager = [t.clone() for t in step()]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
    assert not held[0][2].any()


def test_offsets_past_32_bits():
    """Pages whose addresses and a table whose entries lie past 4 GiB."""
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache, RotaryTable, paged_append, \
        paged_attention
    n, nkv, hd, page = 9000, 8, 128, 512  # 1 MiB a page, 9.4 GB of keys, as much of values
    k = torch.zeros(n, nkv, page, hd, dtype=torch.float16, device=DEV)
    v = torch.zeros(n, nkv, page // 8, hd, 8, dtype=torch.float16, device=DEV)
    table = torch.tensor([[8999, 4097], [0, 8998]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([600, 511], device=DEV)
    small = torch.tensor([0, 1, 2, 3], device=DEV)
    for t in (k, v):
        t[table.view(-1).long()] = torch.randn((4,) + t.shape[1:], device=DEV).half()
    kk, vv = k[table.view(-1).long()].contiguous(), v[table.view(-1).long()].contiguous()
    cos, sin = ref.tables(hd, 1024)
    rope = RotaryTable.wrap(cos.to(DEV), sin.to(DEV))
    qkv = torch.randn(2, 48 * hd, device=DEV).half()
    res = []
    for keys, vals, t in ((k, v, table), (kk, vv, small.view(2, 2).int())):
        cache, one = PagedKVCache.wrap([keys], [vals]), PagedBatch(t, lens, 601)
        q = paged_append(qkv, rope, one, cache, 0, 32)
        res.append((q, paged_attention(q, one, cache, 0), keys[t.view(-1).long()],
                    vals[t.view(-1).long()]))
    assert all(torch.equal(a, b) for a, b in zip(*res))
