"""GPU tests of how exactly paged attention adds up: probabilities are not rounded to the
cache's type in any of its forms, so what is left is the result's own rounding."""
import math

import pytest
import torch

from tests import _paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _cache(s):
    from hydranet_amd.model.paged import PagedKVCache
    return PagedKVCache.wrap([s["k"]], [s["v"]])


def _tight(s, q, nh):
    """-> (out, bound) in 64 bits.  A score is off by hd 2^-24 of its products' magnitudes and
    a few 2^-24 of itself, which moves its probability by as much.  A probability is the sum
    of two numbers of the type (each rounding leaves u of what it rounds: u^2; in fp16 not
    below 2^-25 / 2^8 of the largest), an exponential's own error is 2^-23.  Sums of fp32: a
    product passes one addition per tile of 32 positions, 32 within one and some 30 of the
    waves and shares.  The result is rounded once."""
    k, v, table = s["k"].double().cpu(), s["v"].double().cpu(), s["table"].cpu().long()
    nkv, page, hd = k.shape[1:]
    u, dt = ref.half_step(s["k"].dtype), s["k"].dtype
    x = q.double().view(-1, nkv, nh // nkv, hd)
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    for row, b, pos in ref.tokens({n: s[n].cpu() for n in ("starts", "lens")}):
        n = pos + 1
        ids = table[b][:-(-n // page)]
        kb = k[ids].transpose(0, 1).reshape(nkv, -1, hd)[:, :n]
        vb = v[ids].permute(1, 0, 2, 4, 3).reshape(nkv, -1, hd)[:, :n]
        sc = x[row] @ kb.transpose(1, 2) * hd ** -0.5
        p = torch.softmax(sc, -1)
        size = x[row].abs() @ kb.abs().transpose(1, 2) * hd ** -0.5
        ds = (hd * size + 4 * sc.abs()).amax(-1, keepdim=True) * 2.0 ** -24
        out[row] = p @ vb
        bound[row] = (p @ vb.abs()) * (2 * u * u + 2 * ds + (n / 32 + 64) * 2.0 ** -23) \
            + u * out[row].abs() + ref.subnormal(dt) + n * 2.0 ** -33 * vb.abs().amax(1)[:, None]
    return out.view(-1, nh * hd), bound.view(-1, nh * hd)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("hint", [None, 5000])
@pytest.mark.parametrize("lens,counts,nkv,rep,hd,page", [
    ([40, 21, 30], None, 2, 16, 128, 16),
    ([33], None, 4, 4, 64, 32),
    ([50], None, 1, 12, 256, 16),
    ([40, 30], None, 2, 20, 128, 16),    # 17 to 24 rows a KV head
    ([25, 60], [2, 3], 1, 8, 64, 16),
    ([20, 0], [30, 13], 2, 4, 128, 16),  # blocks of rows
    ([9], [50], 2, 3, 64, 32),
    ([0], [40], 1, 2, 256, 64),
])
def test_short_texts(lens, counts, nkv, rep, hd, page, hint, dt):
    """Few positions of like weight: a probability rounded to the type would move a result
    near 0 by more than its own rounding and the sums' errors."""
    from hydranet_amd.model.paged import paged_attention
    s = ref.make(11, lens, counts, nkv, hd, page, ref.TYPES[dt], DEV, poison=True)
    q = torch.randn(s["rows"], nkv * rep * hd, generator=s["gen"]).mul(0.05).to(ref.TYPES[dt])
    want, bound = _tight(s, q, nkv * rep)
    got = paged_attention(q.to(DEV), ref.batch(s, counts is None, hint), _cache(s), 0)
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("hint", [None, 20000])
@pytest.mark.parametrize("lens,counts,nkv,rep,hd", [
    ([2500, 700], None, 1, 8, 128),
    ([1900], None, 1, 20, 128),
    ([2000], None, 2, 4, 256),
    ([2400], [40], 1, 4, 128),
    ([1500], [33], 2, 4, 64),
    ([1300], [40], 1, 2, 256),
])
def test_long_texts(lens, counts, nkv, rep, hd, hint):
    """The same over shares of the positions, in the type of fewer bits."""
    from hydranet_amd.model.paged import paged_attention
    s = ref.make(12, lens, counts, nkv, hd, 64, torch.bfloat16, DEV, poison=True)
    q = torch.randn(s["rows"], nkv * rep * hd, generator=s["gen"]).mul(0.05).bfloat16()
    want, bound = _tight(s, q, nkv * rep)
    got = paged_attention(q.to(DEV), ref.batch(s, counts is None, hint), _cache(s), 0)
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert math.isfinite(float(err.max()))
