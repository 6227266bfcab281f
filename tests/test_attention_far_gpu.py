"""Attention where scores times the scale are far from zero, on every tile choice of the kernels. The exponent of a row's largest
score has to come out as 0 there, however large the score is."""
import pytest
import torch

import attention_far as far
from qengine_amd import call, ops
from test_attn_prompt_gpu import inputs
from test_attn_tree_gpu import attend, setup

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16

# lengths, heads, kv heads, head size of every tile choice of attn_prompt: blocks of 64 rows in groups, of 128 rows in steps of
# 64 and of 32 keys
PROMPTS = [([300], 2, 1, 64), ([400, 31, 33, 257], 64, 8, 64), ([3000], 32, 4, 64), ([300, 70], 2, 1, 128), ([700], 40, 8, 128),
           ([900, 1, 255, 64], 40, 8, 128), ([300, 5], 2, 1, 256), ([1100, 40], 32, 2, 256)]
# rows of a kv head: attn_tree.hip's and attn_wide.hip's choices
ROWS = [(64, 5), (64, 17), (64, 33), (64, 129), (128, 5), (128, 17), (128, 129), (256, 5), (256, 17), (256, 129)]
POWERS = [-100, 2, 4, 6, 40, 100]


def compare_prompt(q, k, v, cu, out, lse, power):
    heads, c = q.shape[1], cu.tolist()
    group = heads // k.shape[1]
    for b, (a, e) in enumerate(zip(c[:-1], c[1:])):
        seen = torch.ones(e - a, e - a, dtype=torch.bool, device=q.device).tril()
        for h in {0, heads // 2, heads - 1}:
            want = far.rows(q[a:e, h], k[a:e, h // group], v[a:e, h // group], seen, power)
            far.check(out[a:e, h], lse[a:e, h], want, f"sequence {b} head {h}")


def ranks(shape, order, g, dev):
    """whole numbers 0 .. 7 for keys along the first dimension: mixed, or up by one every 64 keys (128: a wave's steps of
    attn_tree.hip)"""
    if order == "mixed":
        return torch.randint(0, 8, shape, device=dev, generator=g)
    return (torch.arange(shape[0], device=dev) // (128 if order == "up by 128" else 64) % 8).view(-1, *[1] * (len(shape) - 1)).expand(shape)


@pytest.mark.parametrize("order,sign", [("mixed", 1), ("mixed", -1), ("up", 1)])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lens,heads,kv,d", PROMPTS, ids=str)
def test_prompt(dev, lens, heads, kv, d, dtype, order, sign):
    q, k, v, cu = inputs(dev, lens, heads, kv, d, dtype, seed=d)
    g = torch.Generator(device=dev)
    g.manual_seed(sum(lens))
    far.fill_queries(q, g)
    far.fill_keys(k, ranks(k.shape[:2], order, g, dev), sign)
    for power in POWERS:
        out, lse = ops.attn_prompt(q, k, v, cu, scale=far.scale_of(power), lse=True)
        compare_prompt(q, k, v, cu, out, lse, power)


@pytest.mark.parametrize("parts", [1, 0])
@pytest.mark.parametrize("order,sign", [("mixed", 1), ("mixed", -1), ("up", 1), ("up by 128", 1)])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d,rows", ROWS)
def test_tree(dev, d, rows, dtype, order, sign, parts):
    n = min(rows, 16)
    heads = -(-rows // n)
    ctx, new = [3000, 0, 70], [n, n, 1]
    c, q, seqs, cu, mask, words = setup(dev, ctx, new, heads, 1, d, 16, dtype, seed=rows, tree="tree")
    g = torch.Generator(device=dev)
    g.manual_seed(rows + d)
    far.fill_queries(q, g)
    table, length = c.table.tolist(), c.length.tolist()
    far.fill_keys(c.k, torch.zeros(c.k.shape[:-1], device=dev))
    keys = []
    for b, s in enumerate(seqs.tolist()):
        t = ranks((ctx[b] + new[b],), order, g, dev)
        at = torch.arange(ctx[b] + new[b], device=dev)
        pg = torch.tensor(table[s], device=dev)[at // 16]
        far_k = torch.zeros(len(at), d, dtype=dtype, device=dev)
        far.fill_keys(far_k, t, sign)
        c.k[0, pg, 0, at % 16] = far_k
        keys.append((far_k, c.v[0, pg, 0, at % 16]))
        assert length[s] == ctx[b]
    call("qe_attn_tree_set_split", parts)
    try:
        got = [attend(c, q, seqs, cu, n, mask, lse=True, scale=far.scale_of(p)) for p in POWERS]
    finally:
        call("qe_attn_tree_set_split", 1)
    first = cu.tolist()
    for power, (out, lse) in zip(POWERS, got):
        for b, (k, v) in enumerate(keys):
            a, e = first[b], first[b + 1]
            seen = torch.ones(e - a, len(k), dtype=torch.bool)
            for i in range(e - a):
                seen[i, ctx[b]:] = torch.tensor([bool(words[a + i] >> j & 1) for j in range(new[b])])
            for h in {0, heads - 1}:
                want = far.rows(q[a:e, h], k, v, seen.to(dev), power)
                far.check(out[a:e, h], lse[a:e, h], want, f"sequence {b} head {h} scale 2^{power}")


CONSTANTS = [5736, 5808, 3000, 20000, 60000]


def check_means(out, lse, mean, size, counts, score, dtype, what):
    """keys of one score each: a row's output is the mean of its keys' values, its lse that score and the log of their number"""
    n = counts.max()
    u = far.HALF_STEP[dtype]
    assert torch.isfinite(out).all() and torch.isfinite(lse).all(), what
    bound = (n + 8) * 2.0 ** -24 * size + u * mean.abs() * 1.02 + 2.0 ** -25
    assert ((out.double() - mean).abs() <= bound).all(), what
    # the score: an fp32 sum of at most 256 products, times the scale with log2(e), a sum, times ln 2
    assert ((lse.double() - score - torch.log(counts)).abs() <= 270 * 2.0 ** -24 * score + 2.0 ** -18).all(), what


@pytest.mark.parametrize("lens,heads,kv,d", PROMPTS, ids=str)
def test_prompt_of_equal_large_keys(dev, lens, heads, kv, d):
    """fp16 numbers of ordinary size at the usual scale"""
    q, k, v, cu = inputs(dev, lens, heads, kv, d, F16, seed=d)
    c = cu.tolist()
    for x in CONSTANTS:
        q.fill_(x), k.fill_(x)
        x = float(q.flatten()[0])
        out, lse = ops.attn_prompt(q, k, v, cu, lse=True)
        for a, e in zip(c[:-1], c[1:]):
            counts = torch.arange(1, e - a + 1, device=dev, dtype=torch.float64)
            for h in {0, heads - 1}:
                vd = v[a:e, h // (heads // kv)].double()
                mean, size = vd.cumsum(0) / counts[:, None], vd.abs().cumsum(0) / counts[:, None]
                check_means(out[a:e, h], lse[a:e, h], mean, size, counts, d ** 0.5 * x * x, F16, f"{x} head {h}")


@pytest.mark.parametrize("d,rows", ROWS)
def test_decode_of_equal_large_keys(dev, d, rows):
    ctx = [3000, 0, 70]
    c, q, seqs, cu, _, _ = setup(dev, ctx, [1] * 3, rows, 1, d, 16, F16, seed=rows)
    table = c.table.tolist()
    for x in CONSTANTS:
        q.fill_(x), c.k.fill_(x)
        x = float(q.flatten()[0])
        out, lse = attend(c, q, seqs, cu, 1, lse=True)
        for b, s in enumerate(seqs.tolist()):
            at = torch.arange(ctx[b] + 1, device=dev)
            vd = c.v[0, torch.tensor(table[s], device=dev)[at // 16], 0, at % 16].double()
            counts = torch.full((rows,), len(at), device=dev, dtype=torch.float64)
            check_means(out[b], lse[b], vd.mean(0)[None], vd.abs().mean(0)[None], counts, d ** 0.5 * x * x, F16, f"{x} sequence {b}")
