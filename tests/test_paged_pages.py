"""Forks of a text that ends at a page's end."""
import torch

from hydranet_amd.model.paged import PagedKVCache


def test_a_fork_looks_at_no_page_past_the_length():
    c = PagedKVCache(1, 6, 1, 8, 16)
    a = c.take(2)
    for t in c.k + c.v:
        t.normal_()
    assert c.fork(a + [-1], 32) == a          # (a row of a table, with its padding)
    assert c.fork(a + [5], 32) == a           # (5 is nobody's)
    assert c.fork([-1], 0) == [] and c.free_pages == 4
    b = c.fork(a + [-1], 20)
    assert b[0] == a[0] and b[1] not in a and torch.equal(c.k[0][b[1]], c.k[0][a[1]])
