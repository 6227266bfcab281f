"""Attention over tens of thousands of tokens, in parts over all compute units, on values that show a unit left out, repeated or
misplaced (long_context.py; test_long_contexts.py plants such mistakes), and on single keys that decide a row."""
import pytest
import torch

import attention_ref as ref
from long_context import values
from test_attn_tree_gpu import attend, compare, setup

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
SHAPES = [(128, 8, 2, 1), (256, 8, 1, 5), (64, 16, 1, 64), (128, 5, 1, 40), (128, 40, 8, 32), (64, 8, 1, 4)]


def at_tokens(c, s, n, dev):
    """page and row in it of a slot's first n tokens"""
    at = torch.arange(n, device=dev)
    return c.table[s].long()[at // c.page], at % c.page


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d,heads,kv,new", SHAPES)
def test_every_unit_once(dev, d, heads, kv, new, page):
    for ctx, dtype in (([70001], BF), ([20001, 3, 500, 9000], F16)):
        rows = [new if x > 10000 else 1 for x in ctx]
        c, q, seqs, cu, _, _ = setup(dev, ctx, rows, heads, kv, d, page, dtype, seed=d)
        for s, n in zip(seqs.tolist(), [x + y for x, y in zip(ctx, rows)]):
            pg, off = at_tokens(c, s, n, dev)
            for m in range(kv):
                c.v[0, pg, m, off] = values(n, d, dtype, dev)
        compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, new, lse=True))


@pytest.mark.parametrize("d,heads,kv,new", SHAPES)
def test_single_keys(dev, d, heads, kv, new):
    """every row of every head looks for one key of its own, at the ends of pages, waves' stretches, units and blocks' ranges"""
    n, dtype = 40000, BF
    c, q, seqs, cu, _, _ = setup(dev, [n], [new], heads, kv, d, 64, dtype, seed=d)
    s, group = seqs.item(), heads // kv
    g = torch.Generator(device=dev)
    g.manual_seed(d)
    sign = torch.randint(0, 2, q.shape, device=dev, generator=g) * 2.0 - 1
    q.copy_(sign)
    pg, off = at_tokens(c, s, n + new, dev)
    edges = sorted({e + x for e in range(0, n, 2048) for x in (0, 15, 16, 31, 32, 63, 64, 127, 128, 1023) if e + x < n})
    edges = torch.tensor(edges)[torch.randperm(len(edges), generator=torch.Generator().manual_seed(d))].tolist()
    step = new * group  # needles of a kv head at a time
    for first in range(0, min(len(edges), 6 * step), step):
        keep = c.k.clone()
        for m in range(kv):
            for r, e in enumerate(edges[first:first + step]):
                i, h = r // group, m * group + r % group
                c.k[0, pg[e], m, off[e]] = (sign[i, h] * 64 / d ** 0.5).to(dtype)
        compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, new, lse=True))
        c.k.copy_(keep)
