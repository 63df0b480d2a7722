"""GPU tests of paged attention over bf16 values near the type's largest: means of them are
finite, though 2^14 times one is not a number of fp32."""
import pytest
import torch

from tests import _paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("hint", [None, 5000])
@pytest.mark.parametrize("lens,counts,nkv,rep,hd", [
    ([21, 0], None, 2, 4, 128), ([1037], None, 1, 4, 64), ([300], None, 1, 20, 128),
    ([500], None, 1, 2, 256), ([400, 9], [40, 2], 2, 4, 128), ([1500], [40], 1, 2, 64)])
def test_means_of_large_values(lens, counts, nkv, rep, hd, hint):
    from hydranet_amd.model.paged import PagedKVCache, paged_attention
    s = ref.make(31, lens, counts, nkv, hd, 16, torch.bfloat16, DEV, poison=True)
    cache = PagedKVCache.wrap([s["k"]], [s["v"]])
    q = torch.randn(s["rows"], nkv * rep * hd, generator=s["gen"]).bfloat16()
    plain = paged_attention(q.to(DEV), ref.batch(s, counts is None, hint), cache, 0)
    # values of one text's one head, to 1.7e38; and one large value among small ones
    big = s["v"][:, 0].abs().nan_to_num().amax()
    s["v"][:, 0] *= 2.0 ** 127 / big.float().log2().ceil().exp2()
    at = lens[0] // 3
    s["v"][int(s["table"][0, at // 16]), -1, at % 16 // 8, 5, at % 8] = 3.0e38
    want, bound = ref.attend(s, q, nkv * rep)
    got = paged_attention(q.to(DEV), ref.batch(s, counts is None, hint), cache, 0)
    assert got.isfinite().all()
    # (where a head's values are small all but one, the products' errors are of the large one's
    # weight: the bound says so)
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    if nkv > 1:  # dimensions of the other head without a large value: as before
        same = got.view(-1, nkv, rep, hd)[:, 1:].clone()
        old = plain.view(-1, nkv, rep, hd)[:, 1:].clone()
        same[..., 5] = old[..., 5] = 0
        torch.testing.assert_close(same.float(), old.float(), rtol=2.0 ** -7, atol=1e-5)
