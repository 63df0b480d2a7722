"""GPU tests of the paged append at 256 rows and more (a thread takes several heads of a
token), row by row against the 64-bit form."""
import pytest
import torch

from tests import _paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,counts,nkv,rep,hd,page,rotary", [
    ([0, 0, 0], [200, 55, 1], 2, 4, 128, 64, 128),          # 256 rows
    ([13, -1, 100, 7, 0], [150, 9, 0, 131, 17], 1, 5, 128, 16, 64),
    ([5] * 40, [8] * 40, 2, 1, 128, 32, 128),               # runs across groups of 8 slots
    ([3 * i for i in range(300)], None, 1, 3, 128, 16, 32),  # single tokens
    ([9, 50], [300, 14], 2, 4, 64, 128, 64),
    ([31, 0], [123, 140], 1, 2, 256, 16, 128),
    ([0], [255], 2, 2, 128, 16, 128),                       # one row less
])
def test_many_rows(lens, counts, nkv, rep, hd, page, rotary, dt, layout):
    from hydranet_amd.model.paged import PagedKVCache, RotaryTable, paged_append
    T, nh = ref.TYPES[dt], nkv * rep
    s = ref.make(21, lens, counts, nkv, hd, page, T, DEV, columns=1)
    qkv = torch.randn(s["rows"], (nh + 2 * nkv) * hd, generator=s["gen"]).to(T)
    cos, sin = ref.tables(rotary, max(lens) + s["rows"] + 1)
    k, v = s["k"].cpu(), s["v"].cpu()
    got = paged_append(qkv.to(DEV), RotaryTable.wrap(cos.to(DEV), sin.to(DEV), layout),
                       ref.batch(s, counts is None), PagedKVCache.wrap([s["k"]], [s["v"]]), 0,
                       nh).cpu()
    table, kd, vd, u = s["table"].cpu(), s["k"].cpu(), s["v"].cpu(), ref.half_step(T)
    live = torch.zeros(s["rows"], dtype=torch.bool)
    for row, b, pos in ref.tokens({n: s[n].cpu() for n in ("starts", "lens")}):
        live[row] = True
        x = qkv[row].view(nh + 2 * nkv, hd)
        y = ref.rotate(x[:nh + nkv].double(), cos[pos], sin[pos], layout)
        # two products and a sum in fp32, of magnitudes up to twice the row's largest
        bound = u * y.abs() + 3 * 2.0 ** -24 * 2 * x.double().abs().max() + ref.subnormal(T)
        p = int(table[b, pos // page])
        out = torch.cat((got[row].view(nh, hd), kd[p, :, pos % page])).double()
        assert ((out - y).abs() <= bound).all(), row
        assert torch.equal(out[:, rotary:], y[:, rotary:])
        k[p, :, pos % page] = kd[p, :, pos % page]
        v[p, :, pos % page // 8, :, pos % 8] = x[nh + nkv:]
    assert torch.equal(v, vd) and torch.equal(k, kd)  # all else as it was
    assert not got[~live].any()
