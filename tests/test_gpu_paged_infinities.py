"""GPU tests of paged attention over values that are infinite or NaN anywhere in a sequence:
the rows that see one have it in that dimension, whatever its weight, in every form."""
import math

import pytest
import torch

from tests import _paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _cache(s):
    from hydranet_amd.model.paged import PagedKVCache
    return PagedKVCache.wrap([s["k"]], [s["v"]])


def _place(s, at, g=0):
    """(page, KV head, slot / 8, slice of dimensions, slot % 8) of sequence 0's position."""
    page = s["k"].shape[2]
    return int(s["table"][0, at // page]), g, at % page // 8, slice(None), at % page % 8


def _check(s, counts, hint, nh, hd, values):
    """values: {position: (dimension, value)} of sequence 0, KV head 0."""
    from hydranet_amd.model.paged import paged_attention
    q = torch.randn(s["rows"], nh * hd, generator=s["gen"]).to(s["k"].dtype).to(DEV)
    nkv, C = s["k"].shape[1], int(s["lens"][0])
    n, rep = (counts or [1])[0], nh // nkv

    def run():
        return paged_attention(q, ref.batch(s, counts is None, hint), _cache(s), 0)
    want = run().view(s["rows"], nh, hd)
    assert want.isfinite().all()
    extra = torch.zeros_like(want, dtype=torch.float32)
    for at, (d, x) in values.items():
        p, g, i, _, j = _place(s, at)
        s["v"][p, g, i, d, j] = x
        extra[max(at - C, 0):n, :rep, d] += x
    got = run().view(s["rows"], nh, hd)
    odd = ~extra.isfinite()
    assert odd.any() and torch.equal(got[~odd], want[~odd])
    assert torch.equal(got[odd].isnan(), extra[odd].isnan())
    fin = ~extra[odd].isnan()
    assert torch.equal(got[odd][fin].float(), extra[odd][fin])


FORMS = [
    # lens, counts (None: one row each), kv heads, query heads per KV head, hd, page
    ([21], None, 2, 4, 128, 16),
    ([300, 5], None, 1, 4, 64, 64),
    ([1037, 70], None, 2, 8, 128, 16),
    ([700], None, 1, 3, 256, 32),
    ([150, 9], None, 1, 20, 128, 16),
    ([1037, 5], [4, 8], 1, 4, 128, 16),
    ([900], [2], 2, 12, 64, 32),
    ([300, 20], [50, 7], 2, 4, 128, 64),
    ([1500], [40], 1, 4, 64, 16),
    ([400], [33], 1, 2, 256, 16),
]


@pytest.mark.parametrize("hint", [None, 5000])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_infinities_among_cached_positions(form, dt, hint):
    lens, counts, nkv, rep, hd, page = FORMS[form]
    C, n = lens[0], (counts or [1])[0]
    for values in ({0: (3, math.inf)}, {C // 2: (hd - 1, -math.inf)}, {C - 1: (0, math.nan)},
                   {C: (7, math.inf)}, {C + n - 1: (8, -math.inf), C // 3: (8, -math.inf)},
                   {1: (5, math.inf), C - 2: (5, -math.inf), C + n // 2: (6, math.inf)}):
        s = ref.make(form, lens, counts, nkv, hd, page, ref.TYPES[dt], DEV, poison=True)
        _check(s, counts, hint, nkv * rep, hd, values)


@pytest.mark.parametrize("hint", [None, 5000])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_infinities_of_no_weight(form, hint):
    """A weight too small for any type: the softmax's is above 0 all the same."""
    lens, counts, nkv, rep, hd, page = FORMS[form]
    s = ref.make(form, lens, counts, nkv, hd, page, torch.float16, DEV, poison=True)
    from hydranet_amd.model.paged import paged_attention
    C, nh = lens[0], nkv * rep
    q = torch.randn(s["rows"], nh * hd, generator=s["gen"]).half().to(DEV).abs() + 0.5
    for at in (0, C // 2, C - 1):  # scores of -50 sqrt(hd) or less, of others about +-sqrt(hd)
        p, g, i, _, j = _place(s, at)
        s["k"][p, 0, at % page] = -100.0
        for d, x in ((1, math.inf), (2, -math.inf), (4, math.nan)):
            old = s["v"].clone()
            s["v"][p, g, i, d, j] = x
            got = paged_attention(q, ref.batch(s, counts is None, hint), _cache(s), 0)
            s["v"].copy_(old)
            got = got.view(-1, nh, hd)[:(counts or [1])[0], :rep]
            hit = got[..., d]
            assert hit.isnan().all() if math.isnan(x) else (hit == x).all()
            got[..., d] = 0
            assert got.isfinite().all()


def test_every_value_infinite_and_a_page_missing():
    """A dimension without a finite value; and rows that see a missing page are NaN as ever."""
    from hydranet_amd.model.paged import paged_attention
    for counts in (None, [40, 3]):
        s = ref.make(2, [500, 64], counts, 1, 128, 16, torch.float16, DEV, poison=True)
        q = torch.randn(s["rows"], 4 * 128, generator=s["gen"]).half().to(DEV)
        n = (counts or [1])[0]
        want = paged_attention(q, ref.batch(s, counts is None), _cache(s), 0).view(-1, 4, 128)
        s["v"][s["table"][0, :31].long(), :, :, 9] = math.inf
        got = paged_attention(q, ref.batch(s, counts is None), _cache(s), 0).view(-1, 4, 128)
        assert (got[:n, :, 9] == math.inf).all()
        got[:n, :, 9] = want[:n, :, 9]
        assert torch.equal(got, want)
        s["table"][0, 3] = -1
        got = paged_attention(q, ref.batch(s, counts is None), _cache(s), 0).view(-1, 4, 128)
        assert got[:n].isnan().all() and torch.equal(got[n:], want[n:])
