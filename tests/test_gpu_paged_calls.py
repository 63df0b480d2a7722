"""GPU tests of paged calls around their kernels: what a call holds while it runs."""
import gc
import weakref

import pytest
import torch

from tests import _paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("which", ["append", "attention"])
def test_a_step_lives_as_long_as_the_call_that_reads_it(which, monkeypatch):
    """Another thread may use the batch with another cache while a call reads its struct."""
    from hydranet_amd import _lib
    from hydranet_amd.model import paged
    s = ref.make(1, [20, 5], None, 2, 128, 16, torch.float16, DEV)
    one, cache = ref.batch(s, True), paged.PagedKVCache.wrap([s["k"]], [s["v"]])
    other = paged.PagedKVCache.wrap([s["k"].clone()], [s["v"].clone()])
    cos, sin = ref.tables(128, 40)
    rope = paged.RotaryTable.wrap(cos.to(DEV), sin.to(DEV))
    x = torch.randn(2, (8 if which == "append" else 4) * 128, device=DEV).half()
    call_on, alive = _lib.call_on, []

    def between(device, name, *args):
        step = weakref.ref(one._made[2][0])
        one._step(other, 4)  # what another thread does
        gc.collect()
        alive.append(step() is not None)
        if alive[-1]:
            call_on(device, name, *args)
    monkeypatch.setattr(_lib, "call_on", between)
    if which == "append":
        paged.paged_append(x, rope, one, cache, 0, 4)
    else:
        paged.paged_attention(x, one, cache, 0)
    assert alive == [True]
