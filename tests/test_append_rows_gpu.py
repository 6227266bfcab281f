"""Appends of more rows than one launch takes (a grid has fewer than 2^32 threads, a wave a row)."""
import pytest
import torch

from qengine_amd import ops

pytestmark = pytest.mark.gpu


def test_rows_past_one_launch(dev):
    """2^26 + 9 rows in the memory of one, of which the sequences name some at the ends of the launches"""
    t, cut = (1 << 26) + 9, 1 << 25
    c = ops.KVCache.empty(1, 12, 16, 1, 64, 4, 48, device=dev)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    seqs = ints(2, 0, 3)
    assert c.reserve(seqs, ints(5, 20, 7)).tolist() == [1, 1, 1]
    k = torch.randn(1, 1, 64, device=dev).to(torch.bfloat16)
    v = torch.randn(1, 1, 64, device=dev).to(torch.bfloat16)
    wide = lambda x: x.expand(t, 1, 64)
    for cu in ((cut - 3, cut + 2, cut + 2, cut + 2), (2 * cut - 1, 2 * cut - 1, 2 * cut + 9, 2 * cut + 9), (t - 7, t - 7, t - 7, t)):
        c.k.zero_(), c.v.zero_()
        c.append(0, wide(k), wide(v), seqs, ints(*cu))
        for b, s in enumerate(seqs.tolist()):
            n = cu[b + 1] - cu[b]
            pages = c.table[s, :c.held[s]].long()
            for pool, row in ((c.k, k), (c.v, v)):
                got = pool[0, pages, 0].reshape(-1, 64)
                assert (got[:n] == row[0, 0]).all() and not got[n:].any(), (cu, s)
        free = (c.ref == 0).nonzero()[:, 0]
        assert not c.k[:, free].any() and not c.v[:, free].any()
