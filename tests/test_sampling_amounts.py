"""Penalties given as numbers that fp32 does not hold are refused."""
import math

import pytest
import torch

from hydranet_amd.model.sampling import adjust_logits

X = torch.linspace(-3, 3, 8)[None]
TEXT = torch.tensor([[1, 6, 6]])


@pytest.mark.parametrize("name,value", [
    ("repetition", 1e-50), ("repetition", 1e39), ("repetition", -1.0), ("repetition", math.inf),
    ("presence", 1e39), ("presence", -math.inf), ("frequency", -1e39), ("frequency", 10 ** 400)])
def test_refused(name, value):
    with pytest.raises((AssertionError, OverflowError)):
        adjust_logits(X, TEXT, **{name: value})


def test_the_smallest_and_largest():
    y = adjust_logits(X, TEXT, repetition=2.0 ** -126)
    assert y.isfinite().all() and float(y[0, 6]) == float(X[0, 6]) * 2.0 ** 126
    y = adjust_logits(X, TEXT, presence=3e38, frequency=1e37)
    assert y.isfinite().all() and float(y[0, 6]) < -3e38
