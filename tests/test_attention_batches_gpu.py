"""Batches at the limits of what attention takes: starts far outside the rows, many sequences on every tile, rows past 2^32
bytes, one workspace for batches of every size."""
import ctypes

import pytest
import torch

from qengine_amd import call, lib, ops
from test_attn_prompt_gpu import compare as compare_prompt
from test_attn_prompt_gpu import inputs
from test_attn_tree_gpu import attend, ints, setup
from test_attn_tree_gpu import compare as compare_tree

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [2, 64])
def test_prompt_starts_at_the_ends_of_int(dev, heads, d):
    """the same rows as with starts inside, and nothing before or behind them"""
    q, k, v, cu = inputs(dev, [130, 170], heads, 1, d, BF, seed=d)
    buf = torch.full((900, heads, d), 7.0, dtype=BF, device=dev)
    out, lse = ops.attn_prompt(q, k, v, ints([200, LOW, LOW, 130, HIGH, HIGH, LOW + 1], dev), out=buf[300:600], lse=True)
    for h in (0, heads - 1):
        compare_prompt(q[:, h:h + 1], k, v, cu, out[:, h:h + 1], lse[:, h:h + 1])
    assert (buf[:300] == 7).all() and (buf[600:] == 7).all()


@pytest.mark.parametrize("parts", [1, 0])
@pytest.mark.parametrize("d,heads", [(64, 1), (64, 8), (64, 40), (128, 1), (128, 8), (128, 40), (256, 1), (256, 8), (256, 40)])
def test_tree_starts_at_the_ends_of_int(dev, d, heads, parts):
    c, q, seqs, cu, mask, words = setup(dev, [900, 50], [3, 5], heads, 1, d, 16, BF, seed=d, tree="tree")
    call("qe_attn_tree_set_split", parts)
    try:
        want, wl = attend(c, q, seqs, cu, 5, mask, lse=True)
        buf = torch.full((300, heads, d), 7.0, dtype=BF, device=dev)
        named = ints([seqs[0], seqs[0], seqs[1], seqs[1], seqs[0]], dev)
        out, lse = attend(c, q, named, ints([5, LOW, 3, HIGH, HIGH, LOW], dev), 5, mask, lse=True, out=buf[100:108])
    finally:
        call("qe_attn_tree_set_split", 1)
    # the split into parts depends on the batch's entries, so sums may be joined in another order
    compare_tree(c, q, seqs, cu, words, want, wl)
    compare_tree(c, q, seqs, cu, words, out, lse)
    assert (buf[:100] == 7).all() and (buf[108:] == 7).all()


# more than 64 sequences on blocks of 128 rows in steps of 32 keys, of 64, and on groups
@pytest.mark.parametrize("nseq,most,heads,kv,d", [(300, 90, 8, 2, 128), (70, 90, 4, 1, 128), (200, 90, 8, 1, 64), (66, 4200, 2, 1, 64),
                                                  (100, 300, 8, 2, 256), (65, 3, 2, 1, 256), (65, 3, 2, 1, 128)])
def test_many_sequences(dev, nseq, most, heads, kv, d):
    lens = [(i * 37) % most if i % 7 else 0 for i in range(nseq)]
    lens[nseq // 2] = 4 * most
    if most > 4000:
        lens = [2000 + i for i in range(nseq)]
    q, k, v, cu = inputs(dev, lens, heads, kv, d, F16, seed=nseq)
    out, lse = ops.attn_prompt(q, k, v, cu, lse=True)
    for h in (0, heads - 1):
        m = h // (heads // kv)
        compare_prompt(q[:, h:h + 1], k[:, m:m + 1], v[:, m:m + 1], cu, out[:, h:h + 1], lse[:, h:h + 1])


@pytest.mark.parametrize("nseq,rows,d", [(300, 3, 128), (70, 20, 128), (257, 20, 64), (70, 5, 256), (300, 1, 256)])
def test_many_sequences_over_the_cache(dev, nseq, rows, d):
    ctx = [(i * 53) % 200 for i in range(nseq)]
    c, q, seqs, cu, _, _ = setup(dev, ctx, [rows if i % 5 else 0 for i in range(nseq)], 2, 1, d, 16, BF, seed=nseq)
    compare_tree(c, q, seqs, cu, None, *attend(c, q, seqs, cu, rows, lse=True))


def test_rows_past_32_bits(dev):
    """rows of q, k, v and out that lie 1.2 MB apart: those from the 3580th on start past 2^32 bytes"""
    t, wide = 4200, 600000
    x = torch.empty(t, wide, dtype=BF, device=dev)
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    x[:, :384] = torch.randn(t, 384, device=dev, generator=g).to(BF)
    x[:, 384:640] = 7
    q, k, v, out = (x[:, i:i + 128].view(t, 1, 128) for i in (0, 128, 256, 384))
    assert q.stride(0) * 2 * t > 2 ** 32
    cu = ints([0, 50, t], dev)
    _, lse = ops.attn_prompt(q, k, v, cu, out=out, lse=True)
    compare_prompt(q, k, v, cu, out, lse)
    assert (x[:, 512:640] == 7).all()


def test_one_workspace_for_batches_of_any_size(dev):
    """calls of one kernel ask for the same workspace whatever the batch, so one that grows keeps its buffer: the calls of a
    capture take a buffer of the graph's"""
    lib().qe_workspace_count.restype = ctypes.c_int
    c, q, seqs, cu, _, _ = setup(dev, [200] * 48, [1] * 48, 4, 2, 128, 16, BF, seed=1)
    want = attend(c, q, seqs, cu, 1)
    out = torch.zeros_like(q)
    before = call("qe_workspace_count", 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for n in range(1, 49):
            attend(c, q[:n], seqs[:n], cu[:n + 1], 1, out=out[:n])
    assert call("qe_workspace_count", 5) - before == 1
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
