"""Attention over values at the ends of their type: sums that pass fp32 though the result does not, infinities under weights that
underflow, log-sum-exps of rows that see values which are not finite. Against the formula in 64 bits (bounds: attention_ref.py)."""
import math

import pytest
import torch

import attention_far as far
import attention_ref as ref
from qengine_amd import call, ops
from test_attention_far_gpu import PROMPTS, ROWS
from test_attn_prompt_gpu import compare as compare_prompt
from test_attn_prompt_gpu import inputs
from test_attn_tree_gpu import attend, setup
from test_attn_tree_gpu import compare as compare_tree

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
LARGEST = torch.finfo(BF).max
INF, NAN = math.inf, math.nan


def large_columns(v, g):
    """columns of large values of one sign, of both, of the type's largest alone, between ordinary ones"""
    x = torch.rand(v.shape[:-1], device=v.device, generator=g)
    v[..., 1] = ((0.5 + x / 4) * 2.0 ** 127).to(v.dtype)
    v[..., 2] = ((x - 0.5) * 2.0 ** 127).to(v.dtype)
    v[..., 3] = LARGEST
    v[..., 4] = -LARGEST
    v[..., 5] = ((0.5 + x / 4) * 2.0 ** 118).to(v.dtype)
    v[..., -1] = (x * 2.0 ** -60).to(v.dtype)


@pytest.mark.parametrize("lens,heads,kv,d", PROMPTS, ids=str)
def test_prompt_sums_past_fp32(dev, lens, heads, kv, d):
    q, k, v, cu = inputs(dev, lens, heads, kv, d, BF, seed=d)
    g = torch.Generator(device=dev)
    g.manual_seed(d)
    large_columns(v, g)
    out, lse = ops.attn_prompt(q, k, v, cu, lse=True)
    for h in (0, heads - 1):
        m = h // (heads // kv)
        compare_prompt(q[:, h:h + 1], k[:, m:m + 1], v[:, m:m + 1], cu, out[:, h:h + 1], lse[:, h:h + 1])


@pytest.mark.parametrize("parts", [1, 0])
@pytest.mark.parametrize("d,rows", ROWS)
def test_tree_sums_past_fp32(dev, d, rows, parts):
    n = min(rows, 16)
    heads = -(-rows // n)
    c, q, seqs, cu, mask, words = setup(dev, [9000, 0, 70], [n, n, 1], heads, 1, d, 16, BF, seed=rows, tree="tree")
    g = torch.Generator(device=dev)
    g.manual_seed(rows)
    large_columns(c.v, g)
    call("qe_attn_tree_set_split", parts)
    try:
        compare_tree(c, q, seqs, cu, words, *attend(c, q, seqs, cu, n, mask, lse=True))
    finally:
        call("qe_attn_tree_set_split", 1)


def test_some_parts_alone_pass_fp32(dev):
    """one stretch of a long context holds the large values, its neighbours ordinary ones: parts of both kinds are joined"""
    c, q, seqs, cu, _, _ = setup(dev, [40000], [2], 8, 1, 128, 64, BF, seed=3)
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    table = torch.tensor(c.table[seqs.item()].tolist(), device=dev)
    for first, rows in ((10000, 3000), (39000, 40)):
        at = torch.arange(first, first + rows, device=dev)
        x = torch.rand(rows, device=dev, generator=g)
        c.v[0, table[at // 64], 0, at % 64, 7] = ((0.5 + x / 4) * 2.0 ** 127).to(BF)
    compare_tree(c, q, seqs, cu, None, *attend(c, q, seqs, cu, 2, lse=True))


# where the key with the large score and the infinity under a weight that underflows lie: in two waves of a block, two steps,
# two parts
PLACES = [(100, 5, 40), (100, 40, 5), (700, 3, 690), (9000, 8990, 5), (9000, 5, 8990), (9000, 4000, 4040)]


@pytest.mark.parametrize("parts", [1, 0])
@pytest.mark.parametrize("context,top,far_key", PLACES)
@pytest.mark.parametrize("d,rows", ROWS)
def test_infinities_under_small_weights(dev, d, rows, context, top, far_key, parts):
    """a row that sees an infinity gets it, wherever the key is and whatever its weight; other columns are what the formula says"""
    n = min(rows, 16)
    heads = -(-rows // n)
    c, q, seqs, cu, _, _ = setup(dev, [context], [n], heads, 1, d, 16, BF, seed=rows)
    s = seqs.item()
    table = c.table[s].tolist()
    q.mul_(0.125)
    q[..., 0] = 16
    c.k.mul_(0.125)
    c.k[..., 0] = 0
    put = lambda x, i, col, y: x[0, table[i // 16], 0, i % 16].__setitem__(col, y)
    put(c.k, top, 0, 16.0)
    put(c.k, far_key, 0, -16.0)  # exponents 256 + 256 apart
    for col, y in ((1, INF), (2, -INF), (3, NAN)):
        put(c.v, far_key, col, y)
    put(c.v, far_key, 4, INF), put(c.v, top, 4, -INF)
    put(c.v, far_key, 5, -INF), put(c.v, top, 5, 3.0)
    call("qe_attn_tree_set_split", parts)
    try:
        out, lse = attend(c, q, seqs, cu, n, scale=far.LN2, lse=True)
    finally:
        call("qe_attn_tree_set_split", 1)
    for col, y in ((1, INF), (2, -INF), (5, -INF)):
        assert (out[..., col].float() == y).all(), col
    assert torch.isnan(out[..., 3]).all() and torch.isnan(out[..., 4]).all()
    at = torch.arange(context + n, device=dev)
    pg = torch.tensor(table, device=dev)[at // 16]
    k, v = c.k[0, pg, 0, at % 16], c.v[0, pg, 0, at % 16].clone()
    v[:, 1:6] = 0
    seen = torch.ones(n, context + n, dtype=torch.bool, device=dev).tril(context)
    rest = [0] + list(range(6, d))
    for h in range(heads):
        o, l, ob, lb = ref.rows(q[:, h], k, v, seen, far.LN2)
        ref.check(out[:, h][:, rest], lse[:, h], o[:, rest], l, ob[:, rest], lb)


@pytest.mark.parametrize("lens,heads,kv,d", PROMPTS, ids=str)
def test_prompt_infinities_and_their_lse(dev, lens, heads, kv, d):
    q, k, v, cu = inputs(dev, lens, heads, kv, d, BF, seed=d)
    q.mul_(0.125), k.mul_(0.125)
    q[..., 0], k[..., 0] = 16, 0
    n = lens[0]
    k[3, :, 0], k[n - 60, :, 0] = 16, -16
    v[n - 60, :, 1], v[n - 60, :, 2], v[n - 60, :, 3] = INF, -INF, NAN
    out, lse = ops.attn_prompt(q, k, v, cu, scale=far.LN2, lse=True)
    sees = out[n - 60:n]
    assert (sees[..., 1].float() == INF).all() and (sees[..., 2].float() == -INF).all() and torch.isnan(sees[..., 3]).all()
    clean = v.clone()
    clean[n - 60, :, 1:4] = 0
    out[n - 60:n, :, 1:4] = 0
    hole = slice(n - 60, n)
    for h in (0, heads - 1):
        m = h // (heads // kv)
        seen = torch.ones(n, n, dtype=torch.bool, device=dev).tril()
        o, l, ob, lb = ref.rows(q[:n, h], k[:n, m], clean[:n, m], seen, far.LN2)
        o[hole, 1:4] = 0
        ref.check(out[:n, h], lse[:n, h], o, l, ob, lb)


@pytest.mark.parametrize("d,rows", ROWS)
def test_tree_lse_beside_values_that_are_not_finite(dev, d, rows):
    n = min(rows, 16)
    heads = -(-rows // n)
    c, q, seqs, cu, mask, words = setup(dev, [3000, 40], [n, n], heads, 1, d, 16, F16, seed=rows, tree="tree")
    want, lse = attend(c, q, seqs, cu, n, mask, lse=True)
    for b, s in enumerate(seqs.tolist()):
        for i, (col, y) in ((7, (1, INF)), (30, (2, -INF)), (33, (3, NAN))):
            c.v[0, c.table[s, i // 16], 0, i % 16, col] = y
    out, again = attend(c, q, seqs, cu, n, mask, lse=True)
    assert torch.equal(lse, again)
    assert (out[..., 1].float() == INF).all() and (out[..., 2].float() == -INF).all() and torch.isnan(out[..., 3]).all()
    rest = [0] + list(range(4, d))
    assert torch.equal(out[..., rest], want[..., rest])
