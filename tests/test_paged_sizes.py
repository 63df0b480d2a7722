"""Paged attention's workspace for sizes that the call refuses, and at the largest that it
takes: a number, whatever the struct says (the process ended in a division by 0)."""
import ctypes
import itertools

import pytest

from hydranet_amd import _lib


def _need(**kw):
    sizes = dict(B=4, T=4, nh=32, nkv=8, hd=128, page=64, max_new=1, bound=1000)
    sizes.update(kw)
    step = _lib.PagedStep(16, 1 << 20, 1 << 20, 10, 16, None, *sizes.values())
    return _lib.lib().hn_paged_attention_workspace_bytes(ctypes.addressof(step))


@pytest.mark.parametrize("kw", [
    dict(max_new=1 << 40), dict(max_new=1 << 39), dict(max_new=(1 << 38) + 1),
    dict(max_new=1 << 62, nh=8), dict(max_new=2 ** 63 - 1), dict(max_new=0), dict(max_new=-1),
    dict(B=1 << 32, T=1 << 32, nkv=1 << 32, nh=1 << 32), dict(B=1 << 40), dict(B=-1), dict(T=-1),
    dict(nkv=0), dict(nh=0), dict(nh=33), dict(nh=-32), dict(nkv=-8), dict(hd=0), dict(hd=96),
    dict(hd=1 << 40), dict(page=0), dict(page=24), dict(bound=0), dict(bound=-5),
    dict(bound=-2 ** 63)])
def test_sizes_that_the_call_refuses(kw):
    assert _need(**kw) == 0


def test_sizes_that_it_takes():
    assert _need() > 0
    for B, (nh, nkv), hd, new, bound in itertools.product(
            (1, 65535), ((1, 1), (65535, 65535), (128, 1)), (64, 128, 256),
            (1, 7, 256, (1 << 24) // 65535), (1, 4000, 1 << 62, 2 ** 63 - 1)):
        assert 0 <= _need(B=B, T=B, nh=nh, nkv=nkv, hd=hd, max_new=new, bound=bound) < 1 << 50
    assert _need(nh=1, nkv=1, max_new=65535 * 128) >= 0
